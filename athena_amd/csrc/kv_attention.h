// Attention over the 8-bit paged cache on the matrix cores (fp16 operands, fp32 softmax and accumulation).
//
// A wave owns RT tiles of 16 query rows (row = new token x query head of one kv head) and walks tokens in tiles of 64.
// Sequences with few rows (single new tokens) and with many (chunks of prompts) have a kernel each, see there.
//   S^T = K Q^T   A = 16 keys x 32 columns, B = 32 columns x 16 queries.  Which keys make a tile's rows is free:
//                 tile t (of 4) takes keys 16 (m >> 2) + 4 t + (m & 3), so that lane group g = lane >> 4 ends up
//                 with the 16 consecutive keys 16 g .. 16 g + 15 of its query (lane & 15).  The order of the
//                 contracted columns is free too: a lane reads 16 consecutive columns at once.
//   O^T = V^T P^T A = 16 columns x 32 keys, B = 32 keys x 16 queries: the probabilities a lane holds are the
//                 operand already, and the same 16 consecutive tokens of one column are one 16-byte load, as
//                 the values lie column by column.
// The 16 keys of a lane group lie in one block (block sizes are multiples of 16), so a lane needs ONE key scale, one
// value scale and one table entry for its part of a tile.  The key scale multiplies scores, the value
// scale probabilities; codes are whole numbers below 128 and exact in fp16.
//
// Rounding.  Queries are scaled by a power of two to [2^14, 2^15), where fp16 ends, and held in fp16: bf16 queries fit (8 bits of 11; columns
// more than 2^-31 below a row's largest lose bits), fp32 queries take two fp16 numbers (22 bits; fewer from 2^-17 on).  Probability
// times value scale is held relative to the largest such product of its query so far (see KvSoftmax):
// 11 bits for bf16 results, 22 bits in two numbers for fp32 results, fewer far below it (KV_RAISE).  Sums stay in fp32.
#pragma once
#include "common.h"

typedef _Float16 f16_t;
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

struct KvAttn {
    const void* q;
    long ldq, ldq_head;
    const int8_t *k_codes, *v_codes;
    const float *k_scale, *v_scale;
    const int32_t* tables;
    long ld_tables;
    const int32_t *lens, *cu_rows;
    void* out;
    long ldo, ldo_head;
    float* lse;             // [N][h] or null
    float *part, *part_lse; // [splits][N][h][dk], [splits][N][h]: used where the key axis is split
    int table_width, num_blocks, B, N, h, hk, dk, block_size, block_shift, causal, splits, row_tiles, few, longest_first, q_wide, out_wide;     // few: rows up to which a sequence's key axis is divided
    float scale;
};

#define KV_KEYS 64          // tokens of a tile
#define KV_MIN_TILES 8      // tiles of a split at least
#define KV_FEW 64           // rows of a (sequence, kv head) up to which the key axis is what is divided

// eight codes as fp16: bytes b of code + 128 become 1024 + b (0x6400 | b), less 1152
__device__ __forceinline__ f16x8_t kv_widen(unsigned lo, unsigned hi) {
    union { unsigned u[4]; f16x2_t h[4]; f16x8_t v; } x;
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    x.u[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
    x.u[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
    x.u[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
    x.u[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
    const f16x2_t less = {(f16_t)1152.f, (f16_t)1152.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) x.h[i] -= less;
    return x.v;
}

template <int W> struct KvKeys {            // a lane's codes of one tile of 64 keys
    uint4 c[4][W / 64];
    __device__ __forceinline__ void load(const int8_t* p) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < W / 64; ++i) c[t][i] = *(const uint4*)(p + t * 4 * W + 64 * i);
    }
    __device__ __forceinline__ f16x8_t frag(int t, int f) const {
        const uint4 w = c[t][f >> 1];
        return (f & 1) ? kv_widen(w.z, w.w) : kv_widen(w.x, w.y);
    }
};
template <> struct KvKeys<32> {
    uint2 c[4];
    __device__ __forceinline__ void load(const int8_t* p) {
#pragma unroll
        for (int t = 0; t < 4; ++t) c[t] = *(const uint2*)(p + t * 4 * 32);
    }
    __device__ __forceinline__ f16x8_t frag(int t, int) const { return kv_widen(c[t].x, c[t].y); }
};
// first column of fragment f for lane group g
template <int W> __device__ __forceinline__ int kv_column(int f, int g) {
    return W == 32 ? 8 * g : 64 * (f >> 1) + 16 * g + 8 * (f & 1);
}

// Queries of RT tiles of 16 rows from row ``row0`` of a (sequence, kv head), scaled by a power of two to [2^14, 2^15), as operands;
// what the power and the softmax's scale come to (``qs``, for exponents of two); how many tokens each row sees.
template <typename T, int W, int RT> struct KvQueries {
    static constexpr bool TWO = sizeof(T) == 4;             // fp32: queries and probabilities in two fp16 numbers
    static constexpr int F = W / 32;
    f16x8_t q[RT][F], ql[TWO ? RT : 1][TWO ? F : 1];
    float qs[RT];
    int limit[RT], least, most;                             // of a lane's rows; the fewest and the most of the wave's
    __device__ __forceinline__ void load(const KvAttn& a, int kvh, int G, int lo, int n, int len, int row0, int qc, int g) {
        least = 0x7fffffff;
        most = 0;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = row0 + 16 * r + qc;
            const bool in = row < n * G;
            const int token = in ? row / G : 0, head = kvh * G + (in ? row - token * G : 0);
            limit[r] = !in ? 0 : a.causal ? min(max(len - n + token + 1, 0), len) : len;
            const T* p = (const T*)a.q + (long)(lo + token) * a.ldq + (long)head * a.ldq_head;
            float v[F][8], top = 0.f;
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const int c = kv_column<W>(f, g);
                if (in && a.q_wide && c < a.dk) {
                    struct alignas(16) Eight { T e[8]; };
                    const Eight x = *(const Eight*)(p + c);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[f][i] = to_f32<T>(x.e[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[f][i] = in && c + i < a.dk ? to_f32<T>(p[c + i]) : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[f][i]));
            }
            // (15: powers of two and their reciprocals stay normal numbers)
            const unsigned e = min(max(__float_as_uint(rows4_max(top)) >> 23, 15u), 253u);
            // (the softmax's scale leaves its sign here, so that ``qs`` is not negative)
            const float down = copysignf(__uint_as_float((268u - e) << 23), a.scale);
            qs[r] = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((e - 14u) << 23);
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = v[f][i] * down;
                    q[r][f][i] = (f16_t)x;
                    if (TWO) ql[r][f][i] = (f16_t)(x - (float)q[r][f][i]);
                }
            least = min(least, in ? limit[r] : 0x7fffffff);
            most = max(most, limit[r]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            least = min(least, __shfl_xor(least, o, 64));
            most = max(most, __shfl_xor(most, o, 64));
        }
        least = __builtin_amdgcn_readfirstlane(least);
        most = __builtin_amdgcn_readfirstlane(most);
    }
    __device__ __forceinline__ void score(f32x4_t& s, f16x8_t k, int r, int f) const {
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[r][f], s, 0, 0, 0);
        if (TWO) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[r][f], s, 0, 0, 0);
    }
};

// One tile of 16 rows: the running maximum m of the scores (exponents of two), the sum l of exponentials relative to 2^m, and the sums o
// of values relative to 2^(m + unit()).  ``w`` is log2 of the largest product of probability and value scale relative to m -- by itself,
// as m + w would lose w's bits where scores are large; the unit is made of its next whole number, so that changes of it are exact.
// ``ksq`` (not negative) brings scores to exponents of two, ``vs`` is the lane's value scale, ``vl`` its logarithm to base 2.
// Products go to the matrix units raised by 2^15, up to where fp16 ends: its numbers end at 2^-24, so that relative to a row's largest
// product one fp16 number keeps 11 bits down to 2^-29 and something down to 2^-40, two keep 22 bits down to 2^-18 (and a bit less with
// every further power of two).
#define KV_RAISE 15
#define KV_NO_WEIGHT -300.f     // nothing yet; products below 2^-300 of 2^m do not show in fp32
template <int W, bool TWO> struct KvSoftmax {
    f32x4_t o[W / 16];
    float m, l, w;
    float lim;                  // m + ceil(w) where m is small enough for weigh(), -inf elsewhere
    __device__ __forceinline__ void begin() {
        m = lim = -INFINITY;
        w = KV_NO_WEIGHT;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < W / 16; ++d) o[d] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ int unit() const { return (int)ceilf(w) - KV_RAISE; }     // of o
    // Steps of a tile; each is called for all of a wave's row tiles before the next, so that their chains of dependent
    // instructions run side by side.  1: the largest of the lane's sixteen scores
    __device__ __forceinline__ float peak(f32x4_t (&s)[4], float ksq, bool whole, int seen) {
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][e] = 4 * i + e < seen ? s[i][e] : -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, s[i][e]);
        // (a scale of 0 beside a score of -inf, which is "hidden": still hidden)
        return top == -INFINITY ? top : top * ksq;
    }
    __device__ __forceinline__ bool grows(float top, float vl) const { return top > m || top + vl > lim; }
    // 2, where it grows for any row: the new maxima, and what is there already relative to them.  From some size of m on a difference
    // from it may be above 0 by a number that counts (fp32: steps of 1/16), or the sum with a scale's logarithm be too coarse (bf16: see weigh)
    __device__ __forceinline__ void grow(float top, float vl) {
        const float mn = fmaxf(m, rows4_max(top)), base = mn == -INFINITY ? 0.f : mn, dm = m - base;
        const float wn = fmaxf(fmaxf(w + dm, KV_NO_WEIGHT), rows4_max(top - base + vl));
        l *= __builtin_amdgcn_exp2f(dm);
        const float down = __builtin_amdgcn_exp2f(dm + (ceilf(w) - ceilf(wn)));
#pragma unroll
        for (int d = 0; d < W / 16; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][e] *= down;
        m = mn;
        w = wn;
        lim = fabsf(m) < (TWO ? 1048576.f : 1024.f) ? m + ceilf(w) : -INFINITY;
    }
    // 3: probabilities, their sum, and their products with the value scales, relative to the unit.
    // fp32: by themselves.  bf16: in one exponential, and the sum of the lane's sixteen divided by the scale again.  There the exponent's
    // constant ``at`` is rounded at the size of m (below 1024: by 2^-14, results have 2^-9); the sum is divided by what is left of
    // the scale in it (sixteen multiplications less: 474 against 488 us for chunks of 512 rows, 158 against 163 us for prompts).
    // Not where the value scale is 0, not finite or far from the largest product, nor where m is large.
    __device__ __forceinline__ bool far(float vl) const { return !(fabsf(vl - lim + m) <= 40.f); }
    __device__ __forceinline__ void weigh(f32x4_t (&s)[4], float ksq, float vs, float vl, f16x8_t (&p)[2], f16x8_t (&pl)[2]) {
        const float vf = __builtin_ldexpf(vs, -unit()), at = TWO ? -m : vl + KV_RAISE - lim;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[i][e], ksq, at));
                sum += x;
                s[i][e] = TWO ? x * vf : x;
            }
        l = TWO ? l + sum : fmaf(sum, __builtin_amdgcn_exp2f(-(at + m)), l);
        pack(s, p, pl);
    }
    // the same, one after the other, for tiles with hidden keys (scales that are 0 or not finite must not reach them) and where weigh() would
    // not do.  (A scale more than 2^126 above the largest product has no probability above fp32's least number beside it: any finite factor
    // does.)
    __device__ __forceinline__ void weigh_apart(f32x4_t (&s)[4], float ksq, float vs, float vl, f16x8_t (&p)[2], f16x8_t (&pl)[2]) {
        const float base = m == -INFINITY ? 0.f : m;
        const float vf = __builtin_ldexpf(vs, vl - ceilf(w) > 126.f ? 126 - (int)ceilf(vl) : -(int)ceilf(w));
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool hidden = s[i][e] == -INFINITY;
                float d = fmaf(s[i][e], ksq, -base);
                d = d > 0.f ? 0.f : d;                      // (NaN stays)
                const float x = __builtin_amdgcn_exp2f(d);
                l += hidden ? 0.f : x;
                s[i][e] = hidden ? 0.f : x * vf * (float)(1 << KV_RAISE);
            }
        pack(s, p, pl);
    }
    __device__ __forceinline__ void pack(const f32x4_t (&s)[4], f16x8_t (&p)[2], f16x8_t (&pl)[2]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f16_t h = (f16_t)s[i][e];
                p[i >> 1][4 * (i & 1) + e] = h;
                if (TWO) pl[i >> 1][4 * (i & 1) + e] = (f16_t)(s[i][e] - (float)h);
            }
    }
    __device__ __forceinline__ void add(int d, f16x8_t v, const f16x8_t& p, const f16x8_t& pl) {
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p, o[d], 0, 0, 0);
        if (TWO) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[d], 0, 0, 0);
    }
};

// The softmax's part of one tile of keys, for all row tiles of a wave.
template <typename T, int W, int RT>
__device__ __forceinline__ void kv_weights(const KvQueries<T, W, RT>& q, KvSoftmax<W, sizeof(T) == 4> (&x)[RT], f32x4_t (&s)[RT][4], float ks,
                                           float vs, bool ok, bool whole, int j0, f16x8_t (&p)[RT][2], f16x8_t (&pl)[RT][2]) {
    // log2 |vs| (the instruction takes numbers below fp32's least normal one for 0)
    const float vl = __builtin_amdgcn_logf(fabsf(__builtin_amdgcn_frexp_mantf(vs))) + (float)__builtin_amdgcn_frexp_expf(vs);
    float top[RT];
    bool grows = false, far = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        top[r] = x[r].peak(s[r], ks * q.qs[r], whole, ok ? q.limit[r] - j0 : 0);
        grows = grows || x[r].grows(top[r], vl);
    }
    if (__any(grows)) {
#pragma unroll
        for (int r = 0; r < RT; ++r) x[r].grow(top[r], vl);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) far = far || x[r].far(vl);
    if (whole && !__any(far)) {
#pragma unroll
        for (int r = 0; r < RT; ++r) x[r].weigh(s[r], ks * q.qs[r], vs, vl, p[r], pl[r]);
    } else {
#pragma unroll
        for (int r = 0; r < RT; ++r) x[r].weigh_apart(s[r], ks * q.qs[r], vs, vl, p[r], pl[r]);
    }
}

// rows of a sequence that the kernel of few rows takes; the others go to the kernel of many
__device__ __forceinline__ bool kv_few(const KvAttn& a, int n) { return (long)n * (a.h / a.hk) <= a.few; }

// four columns of a row's result: sum ``y`` over the sum of exponentials ``l`` relative to 2^base; with a split key axis to that
// split's part of the workspace.
template <typename T>
__device__ __forceinline__ void kv_finish(const KvAttn& a, long token, long head, int c, float base, float l, f32x4_t y, int split) {
    // nothing seen: zeros; NaN stays
    const float inv = l > 0.f ? 1.f / l : l != l ? l : 0.f;
    const float lse = l > 0.f ? base + __builtin_amdgcn_logf(l) : l != l ? l : -INFINITY;
    if (a.splits > 1) {
        const long at = ((long)split * a.N + token) * a.h + head;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < a.dk) a.part[at * a.dk + c + j] = y[j] * inv;
        if (c == 0) a.part_lse[at] = lse;
        return;
    }
    T* out = (T*)a.out + token * a.ldo + head * a.ldo_head + c;
    if (a.out_wide && c + 4 <= a.dk) {
        struct alignas(4 * sizeof(T)) Four { T e[4]; } four;
#pragma unroll
        for (int j = 0; j < 4; ++j) four.e[j] = from_f32<T>(y[j] * inv);
        *(Four*)out = four;
    } else {
        for (int j = 0; j < 4; ++j)
            if (c + j < a.dk) out[j] = from_f32<T>(y[j] * inv);
    }
    if (a.lse && c == 0) a.lse[token * a.h + head] = lse * 0.6931471805599453f;
}

// ---------------------------------------------------------------- few rows: bound by the cache's way in
// The four waves of a workgroup take every fourth tile of its share of the keys and meet once, at the end; a lane's codes go
// from memory straight into operands, one tile ahead of their use (two waves per SIMD keep 64 KB of a CU's loads under way).
// Measured (bf16, 32 heads over 8 kv heads of 128, blocks of 64): 8 contexts of 120 to 131 K tokens 355 us for 2.07 GB,
// 5.8 TB/s; 64 requests of 60 to 8192 tokens 116 us for 543 MB, 4.7 TB/s (fp32 118 us) -- a large copy moves 4.8 TB/s here.  The
// smallest calls (a beam of ten, a few dozen tokens) take 6.2 us, most of it the launch and the chain table -> codes -> result.
// One tile of 16 rows per wave: two (17 to 32 rows in one workgroup) spilled registers with heads of 128 and took 89 us where
// two workgroups of one take 71 (40 rows, 32 requests of 3 to 9 K tokens), and the same time with heads of 64.
template <typename T, int W>
__global__ __launch_bounds__(256, 2) void kv8_attention_kernel(KvAttn a) {
    constexpr bool TWO = sizeof(T) == 4;
    constexpr int RT = 1, F = W / 32, D = W / 16, ROWS = 16 * RT;
    __shared__ float s_m[4][ROWS], s_l[4][ROWS];
    __shared__ int s_unit[4][ROWS];
    __shared__ float s_o[4][ROWS][W + 4];
    // (what is the same in all lanes of a wave is said to be, or the compiler keeps it per lane)
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, qc = lane & 15;
    // workgroups of one (sequence, kv head) lie eight apart, on one XCD: they share its L2
    const int inner = a.row_tiles * a.splits, unit = blockIdx.x / 8;
    const int pair = unit / inner * 8 + blockIdx.x % 8, part = unit % inner;
    if (pair >= a.B * a.hk) return;
    const int b = pair / a.hk, kvh = pair % a.hk, split = part % a.splits, G = a.h / a.hk;
    const int lo = min(max(a.cu_rows ? a.cu_rows[b] : b, 0), a.N), hi = min(max(a.cu_rows ? a.cu_rows[b + 1] : b + 1, lo), a.N);
    const int n = hi - lo;
    const int len = (int)min((long long)max(a.lens[b], 0), (long long)a.table_width * a.block_size);
    const int32_t* table = a.tables + (long)b * a.ld_tables;
    if (!kv_few(a, n)) return;

    // (rows of all heads together are below 2^31; 64 bits for the step past the end)
    for (long first = (long)(part / a.splits) * ROWS; first < (long)n * G; first += (long)a.row_tiles * ROWS) {
        const int tile0 = (int)first;
        KvQueries<T, W, RT> q;
        q.load(a, kvh, G, lo, n, len, tile0, qc, g);
        // ---- this workgroup's tiles of keys
        const int tiles = (q.most + KV_KEYS - 1) / KV_KEYS;
        const int per = a.splits > 1 ? max((tiles + a.splits - 1) / a.splits, KV_MIN_TILES) : tiles;
        const int t_end = min((split + 1) * per, tiles);
        KvSoftmax<W, TWO> x[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) x[r].begin();
        KvKeys<W> k;
        uint4 v[D];
        float ks, vs;
        bool ok;                                            // this lane group's keys lie in a block of the pool
        int kb, vb;                                         // blocks of this lane's keys and values, of the tile to load next
        const int kc = 16 * (qc >> 2), vc = 16 * g;         // where in a tile they begin
        auto find = [&](int t) {
            const int jk = t * KV_KEYS + kc, jv = t * KV_KEYS + vc;
            kb = t < t_end && jk < q.most ? table[jk >> a.block_shift] : -1;
            vb = t < t_end && jv < q.most ? table[jv >> a.block_shift] : -1;
        };
        auto load_keys = [&](int t) {
            const int at = ((t * KV_KEYS + kc) & (a.block_size - 1)) + (qc & 3);
            const int block = (unsigned)kb < (unsigned)a.num_blocks ? kb : 0;
            k.load(a.k_codes + ((((long)block * a.hk + kvh) << a.block_shift) + at) * W + (W == 32 ? 8 : 16) * g);
            ok = (unsigned)vb < (unsigned)a.num_blocks;
            const long scale_at = (long)(ok ? vb : 0) * a.hk + kvh;
            ks = a.k_scale[scale_at];
            vs = a.v_scale[scale_at];
        };
        auto load_values = [&](int t, int block) {
            const int at = (t * KV_KEYS + vc) & (a.block_size - 1);
            const int8_t* p = a.v_codes + ((((long)((unsigned)block < (unsigned)a.num_blocks ? block : 0) * a.hk + kvh) * W + qc) << a.block_shift) + at;
#pragma unroll
            for (int d = 0; d < D; ++d) v[d] = *(const uint4*)(p + d * 16 * a.block_size);
        };
        int t = split * per + w;
        if (t < t_end) {
            find(t);
            load_keys(t);
            load_values(t, vb);
            find(t + 4);
        }
        for (; t < t_end; t += 4) {
            const bool next = t + 4 < t_end;
            const float ks_now = ks, vs_now = vs;
            const bool ok_now = ok;
            f32x4_t s[RT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int r = 0; r < RT; ++r) s[r][i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    const f16x8_t kf = k.frag(i, f);
#pragma unroll
                    for (int r = 0; r < RT; ++r) q.score(s[r][i], kf, r, f);
                }
            }
            const int block_next = vb;
            if (next) load_keys(t + 4);
            const bool whole = !__any(!ok_now) && (t + 1) * KV_KEYS <= q.least;
            const int j0 = t * KV_KEYS + vc;
            f16x8_t p[RT][2], pl[RT][2];
            kv_weights<T, W, RT>(q, x, s, ks_now, vs_now, ok_now, whole, j0, p, pl);
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const f16x8_t v0 = kv_widen(v[d].x, v[d].y), v1 = kv_widen(v[d].z, v[d].w);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    x[r].add(d, v0, p[r][0], pl[r][0]);
                    x[r].add(d, v1, p[r][1], pl[r][1]);
                }
            }
            if (next) {
                load_values(t + 4, block_next);
                find(t + 8);
            }
        }
        // ---- the four waves meet
        __syncthreads();                                    // (the rows before are done with the shared memory)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const float l = rows4_sum(x[r].l);
            if (g == 0) {
                s_m[w][16 * r + qc] = x[r].m;
                s_l[w][16 * r + qc] = l;
                s_unit[w][16 * r + qc] = x[r].unit();
            }
#pragma unroll
            for (int d = 0; d < D; ++d) *(f32x4_t*)&s_o[w][16 * r + qc][16 * d + 4 * g] = x[r].o[d];
        }
        __syncthreads();
        constexpr int CG = W / 4;                           // groups of four columns
        for (int e = threadIdx.x; e < ROWS * CG; e += 256) {
            const int rr = e / CG, c = 4 * (e % CG);
            const int row = tile0 + rr;
            if (row >= n * G) continue;
            float mt = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) mt = fmaxf(mt, s_m[i][rr]);
            const float base = mt == -INFINITY ? 0.f : mt;
            float lt = 0.f;
            f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lt += s_l[i][rr] * __builtin_amdgcn_exp2f(s_m[i][rr] - base);
                // (2^(m - base) may be below fp32's least number where 2^(m - base + unit) is not: whole powers apart)
                const float d = fmaxf(s_m[i][rr] - base, -1000.f), down = __builtin_amdgcn_exp2f(d - floorf(d));
                const int power = (int)floorf(d) + s_unit[i][rr];
                const f32x4_t z = *(const f32x4_t*)&s_o[i][rr][c];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] += __builtin_ldexpf(z[j] * down, power);
            }
            kv_finish<T>(a, lo + row / G, kvh * G + row % G, c, base, lt, y, split);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- many rows: bound by the vector and matrix units
// A wave owns 16 RT rows, the NW waves of a workgroup walk its share of the keys together: a tile is loaded once (each thread a few
// 16-byte pieces), widened once and left in LDS as fp16, double-buffered, one barrier a tile.  Widening took more
// vector instructions than the softmax when every wave did it for itself.
// Measured (bf16, causal): chunks of 128 to 512 rows x 4 heads behind 2 to 16 K tokens (heads of 128) 403 us for 269 GFLOP, 668
// TFLOP/s, and 22 us for the join of three splits; three prompts of 1501 to 4001 rows, 16 heads of 64, 148 us for 68.7 GFLOP, 464
// TFLOP/s.  fp32 (two fp16 numbers each) 649 and 217 us.  A large library product reaches 1330 TFLOP/s.  What bounds it: 16 rows x 64
// keys are 175 vector instructions, 16 of them exponentials at a quarter rate, beside 512 clocks of matrix instructions (heads of 128),
// and two or three waves per SIMD overlap them in part only (vector units busy 47 % of the time, matrix units 26 %, waves waiting 30 %;
// prompts 68, 19 and 30 %).
// LDS images in 16-byte chunks (8 numbers), placed so that the 8 lanes that read side by side hit 8 different groups of
// banks: keys [64][W], chunk ^ swz(key); values [W][64], chunk ^ (column & 7).
template <int W> __device__ __forceinline__ int kv_swz(int key) {
    return W == 32 ? (key >> 4) & 3 : (key & 3) | ((key >> 4) & 1) << 2;
}

template <typename T, int W, int RT, int NW>
__global__ __launch_bounds__(64 * NW, (W < 128 && sizeof(T) == 2 ? 3 : 2)) void kv8_attention_rows_kernel(KvAttn a) {
    constexpr bool TWO = sizeof(T) == 4;
    constexpr int F = W / 32, D = W / 16, NT = 64 * NW, ROWS = 16 * NW * RT, NC = W / 8, PIECES = 4 * W, NP = (PIECES + NT - 1) / NT;
    __shared__ __attribute__((aligned(16))) f16_t s_k[2][64 * W], s_v[2][64 * W];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, qc = lane & 15;
    // A (sequence, kv head) stays on one XCD (workgroups eight apart).  Where the caches of all that share an XCD fit its L2, the
    // longest row tiles of all of them come first, or one that begins late makes the chip wait (three causal prompts of 4001
    // rows: 149 against 186 us); elsewhere the tiles of one come together, or its cache is read from memory again and again
    // (chunks of 512 rows behind 16 K tokens: 431 against 686 us).
    const int inner = a.row_tiles * a.splits, eights = (a.B * a.hk + 7) / 8, unit = blockIdx.x / 8;
    const int part = a.longest_first ? unit / eights : unit % inner;
    const int pair = (a.longest_first ? unit % eights : unit / inner) * 8 + blockIdx.x % 8;
    if (pair >= a.B * a.hk) return;
    const int b = pair / a.hk, kvh = pair % a.hk, split = part % a.splits, G = a.h / a.hk;
    const int lo = min(max(a.cu_rows ? a.cu_rows[b] : b, 0), a.N), hi = min(max(a.cu_rows ? a.cu_rows[b + 1] : b + 1, lo), a.N);
    const int n = hi - lo;
    const int len = (int)min((long long)max(a.lens[b], 0), (long long)a.table_width * a.block_size);
    const int32_t* table = a.tables + (long)b * a.ld_tables;
    if (kv_few(a, n)) return;
    // where this lane's fragments lie in the images: keys 16 (qc >> 2) + (qc & 3) + 4 i, columns qc + 16 d
    const int key0 = 16 * (qc >> 2) + (qc & 3), z = kv_swz<W>(key0);
    const int at_k0 = key0 * W + (((W == 32 ? g : 2 * g) ^ z) * 8), at_k1 = key0 * W + (((2 * g + 1) ^ z) * 8);
    const int at_v0 = qc * 64 + (((2 * g) ^ (qc & 7)) * 8), at_v1 = qc * 64 + (((2 * g + 1) ^ (qc & 7)) * 8);
    const int row_tiles = (n * G - 1) / ROWS + 1;
    for (int i = part / a.splits; i < row_tiles; i += a.row_tiles) {
        const int tile0 = (row_tiles - 1 - i) * ROWS, row0 = tile0 + w * 16 * RT;     // causal: the longest rows begin first
        KvQueries<T, W, RT> q;
        q.load(a, kvh, G, lo, n, len, row0, qc, g);
        const int last = (int)min((long)tile0 + ROWS, (long)n * G) - 1, most = a.causal ? min(max(len - n + last / G + 1, 0), len) : len;
        const int all = (most + KV_KEYS - 1) / KV_KEYS, per = a.splits > 1 ? max((all + a.splits - 1) / a.splits, KV_MIN_TILES) : all;
        const int begin = min(split * per, all), tiles = min(begin + per, all);         // this workgroup's tiles of keys
        KvSoftmax<W, TWO> x[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) x[r].begin();
        // ---- staging: this thread's pieces of 16 codes
        uint4 kr[NP], vr[NP];
        int kb[NP], vb, sb;                                 // blocks of the tile to load next: keys, values, scales
        float ks = 0.f, vs = 0.f;
        bool ok = false;
        const auto lookup = [&](int t, int j) { return t < tiles && t * KV_KEYS + j < most ? table[(t * KV_KEYS + j) >> a.block_shift] : -1; };
        const auto inside = [&](int block) { return (unsigned)block < (unsigned)a.num_blocks ? block : 0; };
        auto find = [&](int t) {
#pragma unroll
            for (int p = 0; p < NP; ++p) kb[p] = lookup(t, (tid + NT * p) / (W / 16) & 63);
            vb = lookup(t, 16 * (tid & 3));
            sb = lookup(t, 16 * g);
        };
        auto load = [&](int t) {
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const int e = tid + NT * p, key = e / (W / 16), d = e >> 2;
                if (PIECES < NT && e >= PIECES) continue;
                kr[p] = *(const uint4*)(a.k_codes + ((((long)inside(kb[p]) * a.hk + kvh) << a.block_shift) + ((t * KV_KEYS + key) & (a.block_size - 1))) * W + 16 * (e % (W / 16)));
                vr[p] = *(const uint4*)(a.v_codes + ((((long)inside(vb) * a.hk + kvh) * W + d) << a.block_shift) + ((t * KV_KEYS + 16 * (e & 3)) & (a.block_size - 1)));
            }
        };
        auto load_scales = [&] {
            ok = (unsigned)sb < (unsigned)a.num_blocks;
            const long at = (long)(ok ? sb : 0) * a.hk + kvh;
            ks = a.k_scale[at];
            vs = a.v_scale[at];
        };
        auto stage = [&](int buf) {
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const int e = tid + NT * p, key = e / (W / 16), c = 2 * (e % (W / 16)), d = e >> 2, cv = 2 * (e & 3);
                if (PIECES < NT && e >= PIECES) continue;
                *(f16x8_t*)&s_k[buf][(key * NC + (c ^ kv_swz<W>(key))) * 8] = kv_widen(kr[p].x, kr[p].y);
                *(f16x8_t*)&s_k[buf][(key * NC + ((c + 1) ^ kv_swz<W>(key))) * 8] = kv_widen(kr[p].z, kr[p].w);
                *(f16x8_t*)&s_v[buf][(d * 8 + (cv ^ (d & 7))) * 8] = kv_widen(vr[p].x, vr[p].y);
                *(f16x8_t*)&s_v[buf][(d * 8 + ((cv + 1) ^ (d & 7))) * 8] = kv_widen(vr[p].z, vr[p].w);
            }
        };
        __syncthreads();                                    // (the rows before are done with the shared memory)
        if (begin < tiles) {
            find(begin);
            load(begin);
            load_scales();
            find(begin + 1);
            stage(begin & 1);
        }
        __syncthreads();
        for (int t = begin; t < tiles; ++t) {
            const float ks_now = ks, vs_now = vs;
            const bool ok_now = ok, next = t + 1 < tiles;
            if (next) {
                load(t + 1);
                load_scales();
                find(t + 2);
            }
            if (t * KV_KEYS < q.most) {                     // (a causal wave is done before the workgroup's last rows are)
                // (the XORs depend on the lane alone: everything else is a constant distance from these four places)
                const f16_t *sk0 = s_k[t & 1] + at_k0, *sk1 = s_k[t & 1] + at_k1, *sv0 = s_v[t & 1] + at_v0, *sv1 = s_v[t & 1] + at_v1;
                // (fragments are asked for one step ahead, and the compiler is kept from moving the requests down to their use)
                f32x4_t s[RT][4];
                f16x8_t kf[2][F];
#pragma unroll
                for (int f = 0; f < F; ++f) kf[0][f] = *(const f16x8_t*)((f & 1 ? sk1 : sk0) + (f >> 1) * 64);
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    if (i4 < 3) {
#pragma unroll
                        for (int f = 0; f < F; ++f) kf[(i4 + 1) & 1][f] = *(const f16x8_t*)((f & 1 ? sk1 : sk0) + (i4 + 1) * 4 * W + (f >> 1) * 64);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int r = 0; r < RT; ++r) s[r][i4] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int f = 0; f < F; ++f)
#pragma unroll
                        for (int r = 0; r < RT; ++r) q.score(s[r][i4], kf[i4 & 1][f], r, f);
                }
                const bool whole = !__any(!ok_now) && (t + 1) * KV_KEYS <= q.least;
                const int j0 = t * KV_KEYS + 16 * g;
                f16x8_t p[RT][2], pl[RT][2];
                kv_weights<T, W, RT>(q, x, s, ks_now, vs_now, ok_now, whole, j0, p, pl);
                f16x8_t vf[2][2];
                vf[0][0] = *(const f16x8_t*)sv0;
                vf[0][1] = *(const f16x8_t*)sv1;
#pragma unroll
                for (int d = 0; d < D; ++d) {
                    if (d + 1 < D) {
                        vf[(d + 1) & 1][0] = *(const f16x8_t*)(sv0 + (d + 1) * 16 * 64);
                        vf[(d + 1) & 1][1] = *(const f16x8_t*)(sv1 + (d + 1) * 16 * 64);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int r = 0; r < RT; ++r) x[r].add(d, vf[d & 1][0], p[r][0], pl[r][0]);
#pragma unroll
                    for (int r = 0; r < RT; ++r) x[r].add(d, vf[d & 1][1], p[r][1], pl[r][1]);
                }
            }
            if (next) stage((t + 1) & 1);
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = row0 + 16 * r + qc;
            const float l = rows4_sum(x[r].l), base = x[r].m == -INFINITY ? 0.f : x[r].m;
            const int unit = x[r].unit();
            if (row >= n * G) continue;
#pragma unroll
            for (int d = 0; d < D; ++d) {
                f32x4_t y;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = __builtin_ldexpf(x[r].o[d][j], unit);
                kv_finish<T>(a, lo + row / G, kvh * G + row % G, 16 * d + 4 * g, base, l, y, split);
            }
        }
    }
}

// out = the splits' results weighted by their share of the sum of exponentials; one wave per (row, head).  Bound by the
// latency of its loads: the weights are worked out by the lanes side by side, the results then requested eight at a time
// (24 splits of 256 rows 6.4 us; 27 us with one request after the other).
template <typename T>
__global__ __launch_bounds__(256) void kv8_join_kernel(KvAttn a) {
    const int lane = threadIdx.x & 63, head = blockIdx.y * 4 + (threadIdx.x >> 6), b = blockIdx.z;
    if (head >= a.h) return;
    const int lo = min(max(a.cu_rows ? a.cu_rows[b] : b, 0), a.N), hi = min(max(a.cu_rows ? a.cu_rows[b + 1] : b + 1, lo), a.N);
    const int c0 = lane < a.dk ? lane : 0, c1 = lane + 64 < a.dk ? lane + 64 : c0;
    for (long t = lo + blockIdx.x; t < hi; t += gridDim.x) {
        const long at = t * a.h + head, step = (long)a.N * a.h;
        float top = -INFINITY;
        for (int i = lane; i < a.splits; i += 64) top = fmaxf(top, a.part_lse[at + i * step]);
        top = wave_max(top);
        const float base = top == -INFINITY ? 0.f : top;
        float o0 = 0.f, o1 = 0.f, sum = 0.f;
        for (int i0 = 0; i0 < a.splits; i0 += 64) {
            const float mine = i0 + lane < a.splits ? __builtin_amdgcn_exp2f(a.part_lse[at + (i0 + lane) * step] - base) : 0.f;
            sum += mine;
            for (int i = 0; i < 64 && i0 + i < a.splits; i += 8) {
                float x0[8], x1[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float* p = a.part + (at + (long)min(i0 + i + j, a.splits - 1) * step) * a.dk;
                    x0[j] = p[c0];
                    x1[j] = p[c1];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float weight = __shfl(mine, i + j, 64);       // 0: a split without tokens leaves no result
                    o0 += weight != 0.f ? weight * x0[j] : 0.f;
                    o1 += weight != 0.f ? weight * x1[j] : 0.f;
                }
            }
        }
        sum = wave_sum(sum);
        const float inv = sum > 0.f ? 1.f / sum : sum != sum ? sum : 0.f;
        T* out = (T*)a.out + t * a.ldo + (long)head * a.ldo_head;
        if (lane < a.dk) out[lane] = from_f32<T>(o0 * inv);
        if (lane + 64 < a.dk) out[lane + 64] = from_f32<T>(o1 * inv);
        if (a.lse && lane == 0)
            a.lse[at] = sum > 0.f ? (base + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f : sum != sum ? sum : -INFINITY;
    }
}
