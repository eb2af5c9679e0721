// Penalties for repeated tokens, biases and grammar masks on the logits of a decoding step.
#include "common.h"

// For class v of row r with c = how often v occurs in the row's history:
//   x = logit;  c > 0: x = x > 0 ? x / repetition : x * repetition;  x -= frequency c + presence [c > 0];
//   x += bias;  -inf where the row's mask does not allow v.
// A workgroup takes one tile of classes of one row.  Its logits are requested first; while they travel, occurrences of
// the tile's classes are counted in LDS from the history (whole-number atomics: their order does not matter) and classes with
// a bias of their own get a flag in the counter's top bit.  Then the tile passes once, 16 bytes a lane.  Bound by the
// logits' way in and out; the history is read again by every tile of a row, from the L2, so tiles are large (4096: 16 KB of
// counters, eight workgroups a CU; 8192 took 57 us where 4096 take 43) where there are enough of them to fill the chip, and
// 1024 (fp32) / 2048 (bf16) where there are not.
// Measured: 256 rows of 131072 classes in bf16 with 2000 ids, 100 biases and a mask each 41 us for 140 MB, 3.4 TB/s, in fp32 57 us
// for 275 MB, 4.8 TB/s; 10 rows of 4233 classes in fp32 4.1 us (a launch).
struct LogitsArgs {
    const void* logits;
    void* out;
    const int32_t *history, *history_len, *bias_ids, *allowed;
    const float *repetition, *presence, *frequency, *bias, *bias_values;
    long ldl, ldo, ld_history, ld_bias, ld_bias_ids, ld_bias_values, ld_allowed;
    int R, V, L, nb, wide;
};

#define LOGITS_BIASED 0x80000000u
#define LOGITS_LIST 256         // biases of one tile kept in LDS; more are looked up in memory

// Where the counter of a tile's class i lies: a thread reads E of them, four at a time, and the fours that are read
// together stand side by side.
template <int E, int TILE>
__device__ __forceinline__ unsigned logits_place(unsigned i) {
    return E == 8 ? (i >> 3) * 4 + (i & 3) + ((i >> 2) & 1) * (TILE / 2) : i;
}

// NB vectors of 16 bytes per thread
template <typename T, int NB>
__global__ __launch_bounds__(256) void logits_process_kernel(LogitsArgs a) {
    constexpr int E = 16 / sizeof(T), TILE = 256 * E * NB;
    __shared__ __attribute__((aligned(16))) unsigned count[TILE];
    __shared__ unsigned list_at[LOGITS_LIST];
    __shared__ float list_value[LOGITS_LIST];
    __shared__ int listed;
    struct alignas(16) Vec { T e[E]; };
    const int r = blockIdx.y, v0 = blockIdx.x * TILE, nv = min(TILE, a.V - v0), tid = threadIdx.x;
    const T* in = (const T*)a.logits + (long)r * a.ldl + v0;
    T* out = (T*)a.out + (long)r * a.ldo + v0;
    Vec x[NB];
    unsigned mask[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int i = (b * 256 + tid) * E;
        mask[b] = a.allowed && i < nv ? (unsigned)a.allowed[(long)r * a.ld_allowed + ((v0 + i) >> 5)] : ~0u;
        if (a.wide && i + E <= nv) x[b] = *(const Vec*)(in + i);
        else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[b].e[e] = i + e < nv ? in[i + e] : from_f32<T>(0.f);
        }
    }
#pragma unroll
    for (int i = tid * 4; i < TILE; i += 1024) *(uint4*)&count[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (a.history) {
        const int n = a.history_len ? min(max(a.history_len[r], 0), a.L) : a.L;
        const int32_t* ids = a.history + (long)r * a.ld_history;
#pragma unroll 4
        for (int i = tid; i < n; i += 256) {
            const unsigned at = (unsigned)ids[i] - (unsigned)v0;
            if (at < (unsigned)nv) atomicAdd(&count[logits_place<E, TILE>(at)], 1u);
        }
    }
    if (tid < 64) {                             // the tile's own biases, in their order
        int n = 0;
        for (int j0 = 0; j0 < a.nb; j0 += 64) {
            const int j = j0 + tid;
            const unsigned at = j < a.nb ? (unsigned)a.bias_ids[(long)r * a.ld_bias_ids + j] - (unsigned)v0 : ~0u;
            const unsigned long long found = __ballot(at < (unsigned)nv);
            if (at < (unsigned)nv) {
                atomicOr(&count[logits_place<E, TILE>(at)], LOGITS_BIASED);
                const int k = n + __popcll(found & ((1ull << tid) - 1));
                if (k < LOGITS_LIST) {
                    list_at[k] = at;
                    list_value[k] = a.bias_values[(long)r * a.ld_bias_values + j];
                }
            }
            n += __popcll(found);
        }
        if (tid == 0) listed = n;
    }
    __syncthreads();
    const int biased = listed;
    const float rep = a.repetition ? a.repetition[r] : 1.f, pres = a.presence ? a.presence[r] : 0.f,
                freq = a.frequency ? a.frequency[r] : 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int i = (b * 256 + tid) * E;
        if (i >= nv) continue;
        unsigned c[E], any = 0;
#pragma unroll
        for (int q = 0; q < E; q += 4) {
            const uint4 four = *(const uint4*)&count[logits_place<E, TILE>(i + q)];
            c[q] = four.x, c[q + 1] = four.y, c[q + 2] = four.z, c[q + 3] = four.w;
            any |= (four.x | four.y) | (four.z | four.w);
        }
        if (any || a.bias) {                    // (most vectors hold no class of the history and none with a bias)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int v = v0 + i + e;
                const unsigned n = c[e] & ~LOGITS_BIASED;
                float y = to_f32<T>(x[b].e[e]);
                if (n) {
                    y = y > 0.f ? y / rep : y * rep;
                    y = y - freq * (float)n - pres;
                }
                if (a.bias && i + e < nv) y += a.bias[(long)r * a.ld_bias + v];
                if (c[e] & LOGITS_BIASED) {
                    float own = 0.f;            // entries of one class add up in their order
                    if (biased <= LOGITS_LIST) {
                        for (int j = 0; j < biased; ++j) own += list_at[j] == (unsigned)(i + e) ? list_value[j] : 0.f;
                    } else {
                        for (int j = 0; j < a.nb; ++j)
                            if (a.bias_ids[(long)r * a.ld_bias_ids + j] == v) own += a.bias_values[(long)r * a.ld_bias_values + j];
                    }
                    y += own;
                }
                x[b].e[e] = from_f32<T>(y);
            }
        }
        if (mask[b] != ~0u) {
            const unsigned bits = mask[b] >> ((v0 + i) & 31);
#pragma unroll
            for (int e = 0; e < E; ++e) x[b].e[e] = (bits >> e) & 1u ? x[b].e[e] : from_f32<T>(-INFINITY);
        }
        if (a.wide && i + E <= nv) *(Vec*)(out + i) = x[b];
        else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (i + e < nv) out[i + e] = x[b].e[e];
        }
    }
}

extern "C" int athena_logits_process(const athena_logits_desc* d, athena_stream_t stream) {
    ATHENA_REQUIRE(d, ATHENA_E_SHAPE, "athena_logits_process: null descriptor");
    const int R = d->R, V = d->V;
    ATHENA_REQUIRE(R >= 0 && R <= 65535 && V > 0 && d->L >= 0 && d->L <= (1 << 30) && d->nb >= 0 && d->nb <= (1 << 30), ATHENA_E_SHAPE,
                   "athena_logits_process: bad shape R=%d V=%d L=%d biases=%d", R, V, d->L, d->nb);
    ATHENA_REQUIRE(d->dtype == ATHENA_F32 || d->dtype == ATHENA_BF16, ATHENA_E_UNSUPPORTED, "athena_logits_process: dtype");
    if (R == 0) return ATHENA_OK;
    ATHENA_REQUIRE(d->logits && d->out && (d->nb == 0 || (d->bias_ids && d->bias_values)), ATHENA_E_SHAPE,
                   "athena_logits_process: null operand");
    ATHENA_REQUIRE(d->ldl >= V && d->ldo >= V, ATHENA_E_SHAPE, "athena_logits_process: leading dimension too small");
    LogitsArgs a = {d->logits, d->out, d->history, d->history_len, d->bias_ids, d->allowed, d->repetition, d->presence, d->frequency,
                    d->bias, d->bias_values, d->ldl, d->ldo, d->ld_history, d->ld_bias, d->ld_bias_ids, d->ld_bias_values,
                    d->ld_allowed, R, V, d->history ? d->L : 0, d->nb, 0};
    const int e = d->dtype == ATHENA_BF16 ? 2 : 4;
    a.wide = athena_aligned16(d->logits) && athena_aligned16(d->out) && (R == 1 || (d->ldl * e % 16 == 0 && d->ldo * e % 16 == 0));
    const bool large = R * (((long)V + 4095) / 4096) >= 512;
    const int tile = large ? 4096 : 4096 / e;
    const dim3 grid((unsigned)(((long)V + tile - 1) / tile), R);
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == ATHENA_BF16) {
        if (large) ATHENA_LAUNCH((logits_process_kernel<bf16_t, 2>), grid, dim3(256), 0, s, a);
        else ATHENA_LAUNCH((logits_process_kernel<bf16_t, 1>), grid, dim3(256), 0, s, a);
    } else {
        if (large) ATHENA_LAUNCH((logits_process_kernel<float, 4>), grid, dim3(256), 0, s, a);
        else ATHENA_LAUNCH((logits_process_kernel<float, 1>), grid, dim3(256), 0, s, a);
    }
    ATHENA_CHECK_LAUNCH("athena_logits_process");
    return ATHENA_OK;
}
