// Penalties for repeated tokens, biases and grammar masks on the logits of a decoding step.
#include "common.h"

// For class v of row r with c = how often v occurs in the row's history:
//   x = logit;  c > 0: x = x > 0 ? x / repetition : x * repetition;  x -= frequency c + presence [c > 0];
//   x += bias;  -inf where the row's mask does not allow v.
// A workgroup takes one tile of classes of one row: occurrences of the tile's classes are counted in LDS from
// the history (whole-number atomics: their order does not matter), classes with a bias of their own carry a
// flag in the counter's top bit, and the tile's logits then pass once.  Bound by the logits' way in and out;
// the history is read again by every tile of a row, from the L2.
struct LogitsArgs {
    const void* logits;
    void* out;
    const int32_t *history, *history_len, *bias_ids, *allowed;
    const float *repetition, *presence, *frequency, *bias, *bias_values;
    long ldl, ldo, ld_history, ld_bias, ld_bias_ids, ld_bias_values, ld_allowed;
    int R, V, L, nb, tile;
};

#define LOGITS_TILE 8192
#define LOGITS_BIASED 0x80000000u

template <typename T>
__device__ __forceinline__ float logits_one(const LogitsArgs& a, int r, int v, float x, unsigned c, float rep, float pres, float freq,
                                            unsigned mask_word) {
    const unsigned n = c & ~LOGITS_BIASED;
    if (n) {
        x = x > 0.f ? x / rep : x * rep;
        x = x - freq * (float)n - pres;
    }
    if (a.bias) x += a.bias[(long)r * a.ld_bias + v];
    if (c & LOGITS_BIASED) {
        float own = 0.f;                        // entries of one class add up in their order
        for (int j = 0; j < a.nb; ++j)
            if (a.bias_ids[(long)r * a.ld_bias_ids + j] == v) own += a.bias_values[(long)r * a.ld_bias_values + j];
        x += own;
    }
    return (mask_word >> (v & 31)) & 1u ? x : -INFINITY;
}

template <typename T>
__global__ __launch_bounds__(256) void logits_process_kernel(LogitsArgs a) {
    extern __shared__ unsigned count[];
    const int r = blockIdx.y, v0 = blockIdx.x * a.tile, nv = min(a.tile, a.V - v0), tid = threadIdx.x;
    for (int i = tid; i < nv; i += 256) count[i] = 0;
    __syncthreads();
    if (a.history) {
        const int n = a.history_len ? min(max(a.history_len[r], 0), a.L) : a.L;
        for (int i = tid; i < n; i += 256) {
            const unsigned at = (unsigned)a.history[(long)r * a.ld_history + i] - (unsigned)v0;
            if (at < (unsigned)nv) atomicAdd(&count[at], 1u);
        }
    }
    for (int j = tid; j < a.nb; j += 256) {
        const unsigned at = (unsigned)a.bias_ids[(long)r * a.ld_bias_ids + j] - (unsigned)v0;
        if (at < (unsigned)nv) atomicOr(&count[at], LOGITS_BIASED);
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[r] : 1.f, pres = a.presence ? a.presence[r] : 0.f,
                freq = a.frequency ? a.frequency[r] : 0.f;
    const T* in = (const T*)a.logits + (long)r * a.ldl + v0;
    T* out = (T*)a.out + (long)r * a.ldo + v0;
    const int32_t* allowed = a.allowed ? a.allowed + (long)r * a.ld_allowed : nullptr;
    for (int i = tid; i < nv; i += 256) {
        const unsigned m = allowed ? (unsigned)allowed[(v0 + i) >> 5] : ~0u;
        out[i] = from_f32<T>(logits_one<T>(a, r, v0 + i, to_f32<T>(in[i]), count[i], rep, pres, freq, m));
    }
}

extern "C" int athena_logits_process(const void* logits, long ldl, int dtype, int R, int V, const int32_t* history, long ld_history,
                                     int L, const int32_t* history_len, const float* repetition, const float* presence,
                                     const float* frequency, const float* bias, long ld_bias, const int32_t* bias_ids,
                                     long ld_bias_ids, const float* bias_values, long ld_bias_values, int nb,
                                     const int32_t* allowed, long ld_allowed, void* out, long ldo, athena_stream_t stream) {
    ATHENA_REQUIRE(R >= 0 && R <= 65535 && V > 0 && L >= 0 && nb >= 0, ATHENA_E_SHAPE,
                   "athena_logits_process: bad shape R=%d V=%d L=%d biases=%d", R, V, L, nb);
    ATHENA_REQUIRE(dtype == ATHENA_F32 || dtype == ATHENA_BF16, ATHENA_E_UNSUPPORTED, "athena_logits_process: dtype");
    if (R == 0) return ATHENA_OK;
    ATHENA_REQUIRE(logits && out && (nb == 0 || (bias_ids && bias_values)), ATHENA_E_SHAPE, "athena_logits_process: null operand");
    ATHENA_REQUIRE(ldl >= V && ldo >= V, ATHENA_E_SHAPE, "athena_logits_process: leading dimension too small");
    LogitsArgs a = {logits, out, history, history_len, bias_ids, allowed, repetition, presence, frequency, bias, bias_values,
                    ldl, ldo, ld_history, ld_bias, ld_bias_ids, ld_bias_values, ld_allowed, R, V, history ? L : 0, nb, LOGITS_TILE};
    const dim3 grid((V + a.tile - 1) / a.tile, R);
    if (dtype == ATHENA_BF16) ATHENA_LAUNCH(logits_process_kernel<bf16_t>, grid, dim3(256), a.tile * 4, (hipStream_t)stream, a);
    else ATHENA_LAUNCH(logits_process_kernel<float>, grid, dim3(256), a.tile * 4, (hipStream_t)stream, a);
    ATHENA_CHECK_LAUNCH("athena_logits_process");
    return ATHENA_OK;
}
