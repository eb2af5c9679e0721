// Attention over the 8-bit paged cache on the matrix cores (fp16 operands, fp32 softmax and accumulation).
//
// A wave owns RT tiles of 16 query rows (row = new token x query head of one kv head) and walks its share of the
// sequence in tiles of 64 tokens; the four waves of a workgroup take every fourth tile and meet once, at the end.
// Nothing is staged: codes go from memory into registers, are widened there, and are the matrix operands.
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
// Rounding.  Queries are scaled by a power of two to [1, 2) and held in fp16: bf16 queries fit (8 bits of 11; columns
// more than 2^-17 below a row's largest lose bits), fp32 queries take two fp16 numbers (22 bits).  Probability
// times value scale is held relative to the largest such product of its query so far (M2, beside the softmax's
// own running maximum m): 11 bits for bf16 results, 22 bits in two numbers for fp32 results.  Sums stay in fp32.
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
    int table_width, num_blocks, B, N, h, hk, dk, block_size, causal, splits, row_tiles, q_wide, out_wide;
    float scale;
};

#define KV_KEYS 64          // tokens of a tile
#define KV_MIN_TILES 16     // tiles of a split at least

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

template <typename T, int W, int RT>
__global__ __launch_bounds__(256, 2) void kv8_attention_kernel(KvAttn a) {
    constexpr bool TWO = sizeof(T) == 4;    // fp32: queries and probabilities in two fp16 numbers
    constexpr int F = W / 32, D = W / 16, ROWS = 16 * RT;
    __shared__ float s_m[4][ROWS], s_l[4][ROWS], s_m2[4][ROWS];
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

    for (long tile0 = (long)(part / a.splits) * ROWS; tile0 < (long)n * G; tile0 += (long)a.row_tiles * ROWS) {
        // ---- this wave's queries
        f16x8_t qf[RT][F], ql[TWO ? RT : 1][TWO ? F : 1];
        float qs[RT];
        int limit[RT], least = 0x7fffffff, most = 0;        // tokens a row sees; the fewest and the most of the tile
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const long row = tile0 + 16 * r + qc;
            const bool in = row < (long)n * G;
            const int token = in ? (int)(row / G) : 0, head = kvh * G + (in ? (int)(row % G) : 0);
            limit[r] = !in ? 0 : a.causal ? min(max(len - n + token + 1, 0), len) : len;
            const T* q = (const T*)a.q + (long)(lo + token) * a.ldq + (long)head * a.ldq_head;
            float v[F][8], top = 0.f;
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const int c = kv_column<W>(f, g);
                if (in && a.q_wide && c < a.dk) {
                    struct alignas(16) Eight { T e[8]; };
                    const Eight x = *(const Eight*)(q + c);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[f][i] = to_f32<T>(x.e[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[f][i] = in && c + i < a.dk ? to_f32<T>(q[c + i]) : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[f][i]));
            }
            const unsigned e = min(max(__float_as_uint(rows4_max(top)) >> 23, 1u), 253u);
            const float down = __uint_as_float((254u - e) << 23);
            qs[r] = a.scale * 1.4426950408889634f * __uint_as_float(e << 23);
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = v[f][i] * down;
                    qf[r][f][i] = (f16_t)x;
                    if (TWO) ql[r][f][i] = (f16_t)(x - (float)qf[r][f][i]);
                }
            least = min(least, limit[r]);
            most = max(most, limit[r]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            least = min(least, __shfl_xor(least, o, 64));
            most = max(most, __shfl_xor(most, o, 64));
        }
        least = __builtin_amdgcn_readfirstlane(least);
        most = __builtin_amdgcn_readfirstlane(most);
        // ---- this workgroup's tiles of keys
        const int tiles = (most + KV_KEYS - 1) / KV_KEYS;
        const int per = a.splits > 1 ? max((tiles + a.splits - 1) / a.splits, KV_MIN_TILES) : tiles;
        const int t_end = min((split + 1) * per, tiles);
        f32x4_t o[RT][D];
        float m[RT], l[RT], m2[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            m[r] = m2[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int d = 0; d < D; ++d) o[r][d] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        }
        KvKeys<W> k;
        uint4 v[D];
        float ks, vs;
        bool ok;                                            // this lane group's keys lie in a block of the pool
        int kb, vb;                                         // blocks of this lane's keys and values, of the tile to load next
        const int kc = 16 * (qc >> 2), vc = 16 * g;         // where in a tile they begin
        auto find = [&](int t) {
            const int jk = t * KV_KEYS + kc, jv = t * KV_KEYS + vc;
            kb = t < t_end && jk < most ? table[jk / a.block_size] : -1;
            vb = t < t_end && jv < most ? table[jv / a.block_size] : -1;
        };
        auto load_keys = [&](int t) {
            const int at = (t * KV_KEYS + kc) % a.block_size + (qc & 3);
            const int block = (unsigned)kb < (unsigned)a.num_blocks ? kb : 0;
            k.load(a.k_codes + (((long)block * a.hk + kvh) * a.block_size + at) * W + (W == 32 ? 8 : 16) * g);
            ok = (unsigned)vb < (unsigned)a.num_blocks;
            const long scale_at = (long)(ok ? vb : 0) * a.hk + kvh;
            ks = a.k_scale[scale_at];
            vs = a.v_scale[scale_at];
        };
        auto load_values = [&](int t, int block) {
            const int at = (t * KV_KEYS + vc) % a.block_size;
            const int8_t* p = a.v_codes + (((long)((unsigned)block < (unsigned)a.num_blocks ? block : 0) * a.hk + kvh) * W + qc) * a.block_size + at;
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
            // ---- scores
            f32x4_t s[RT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int r = 0; r < RT; ++r) s[r][i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    const f16x8_t kf = k.frag(i, f);
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        s[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[r][f], s[r][i], 0, 0, 0);
                        if (TWO) s[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[r][f], s[r][i], 0, 0, 0);
                    }
                }
            }
            const int block_next = vb;
            if (next) load_keys(t + 4);
            const bool whole = !__any(!ok_now) && (t + 1) * KV_KEYS <= least;
            const int j0 = t * KV_KEYS + vc;
            const float vl = __builtin_amdgcn_logf(fabsf(vs_now));          // log2
            // ---- softmax
            f16x8_t p[RT][2], pl[TWO ? RT : 1][2];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const float ksq = ks_now * qs[r];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r][i][e] *= ksq;
                if (!whole) {
                    const int seen = ok_now ? limit[r] - j0 : 0;            // this lane's keys below it are visible
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[r][i][e] = 4 * i + e < seen ? s[r][i][e] : -INFINITY;
                }
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, s[r][i][e]);
                const float mn = fmaxf(m[r], rows4_max(top)), mn2 = fmaxf(m2[r], rows4_max(top + vl));
                const float base = mn == -INFINITY ? 0.f : mn, base2 = mn2 == -INFINITY ? 0.f : mn2;
                if (__any(mn > m[r] || mn2 > m2[r])) {
                    l[r] *= __builtin_amdgcn_exp2f(m[r] - base);
                    const float down = __builtin_amdgcn_exp2f(m2[r] - base2);
#pragma unroll
                    for (int d = 0; d < D; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[r][d][e] *= down;
                    m[r] = mn;
                    m2[r] = mn2;
                }
                const float vf = fminf(vs_now * __builtin_amdgcn_exp2f(base - base2), 3.4e38f);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[r][i][e] = __builtin_amdgcn_exp2f(s[r][i][e] - base);
                        sum += s[r][i][e];
                    }
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[r][i][e] *= vf;
                } else {                                    // a scale that is not finite must not reach hidden keys
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[r][i][e] = s[r][i][e] == 0.f ? 0.f : s[r][i][e] * vf;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const f16_t h = (f16_t)s[r][i][e];
                        p[r][i >> 1][4 * (i & 1) + e] = h;
                        if (TWO) pl[r][i >> 1][4 * (i & 1) + e] = (f16_t)(s[r][i][e] - (float)h);
                    }
                l[r] += sum;
            }
            // ---- values
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const f16x8_t v0 = kv_widen(v[d].x, v[d].y), v1 = kv_widen(v[d].z, v[d].w);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[r][0], o[r][d], 0, 0, 0);
                    o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[r][1], o[r][d], 0, 0, 0);
                    if (TWO) {
                        o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[r][0], o[r][d], 0, 0, 0);
                        o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[r][1], o[r][d], 0, 0, 0);
                    }
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
            l[r] = rows4_sum(l[r]);
            if (g == 0) {
                s_m[w][16 * r + qc] = m[r];
                s_l[w][16 * r + qc] = l[r];
                s_m2[w][16 * r + qc] = m2[r];
            }
#pragma unroll
            for (int d = 0; d < D; ++d) *(f32x4_t*)&s_o[w][16 * r + qc][16 * d + 4 * g] = o[r][d];
        }
        __syncthreads();
        constexpr int CG = W / 4;                           // groups of four columns
        for (int e = threadIdx.x; e < ROWS * CG; e += 256) {
            const int rr = e / CG, c = 4 * (e % CG);
            const long row = tile0 + rr;
            if (row >= (long)n * G) continue;
            float mt = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) mt = fmaxf(mt, s_m[i][rr]);
            const float base = mt == -INFINITY ? 0.f : mt;
            float lt = 0.f;
            f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lt += s_l[i][rr] * __builtin_amdgcn_exp2f(s_m[i][rr] - base);
                const float up = s_m2[i][rr] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m2[i][rr] - base);
                const f32x4_t y = *(const f32x4_t*)&s_o[i][rr][c];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] += y[j] * up;
            }
            // nothing seen: zeros; NaN stays
            const float inv = lt > 0.f ? 1.f / lt : lt != lt ? lt : 0.f;
            const float lse = lt > 0.f ? base + __builtin_amdgcn_logf(lt) : lt != lt ? lt : -INFINITY;
            const long token = lo + row / G, head = kvh * G + row % G;
            if (a.splits > 1) {
                const long at = ((long)split * a.N + token) * a.h + head;
                for (int j = 0; j < 4; ++j)
                    if (c + j < a.dk) a.part[at * a.dk + c + j] = x[j] * inv;
                if (c == 0) a.part_lse[at] = lse;
            } else {
                T* out = (T*)a.out + token * a.ldo + head * a.ldo_head + c;
                if (a.out_wide && c + 4 <= a.dk) {
                    struct alignas(4 * sizeof(T)) Four { T e[4]; } four;
#pragma unroll
                    for (int j = 0; j < 4; ++j) four.e[j] = from_f32<T>(x[j] * inv);
                    *(Four*)out = four;
                } else {
                    for (int j = 0; j < 4; ++j)
                        if (c + j < a.dk) out[j] = from_f32<T>(x[j] * inv);
                }
                if (a.lse && c == 0) a.lse[token * a.h + head] = lse * 0.6931471805599453f;
            }
        }
        __syncthreads();
    }
}

// out = the splits' results weighted by their share of the sum of exponentials; one wave per (row, head).  Bound by the
// latency of its loads: the weights are worked out by the lanes side by side, the results then requested eight at a time.
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
