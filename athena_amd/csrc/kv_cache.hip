// Paged key/value cache in 8 bits for decoding: block plans (which blocks a request gets, where its new
// tokens go), the write of new keys and values, and attention over the cache.
//
// The cache of one attention layer, in blocks of ``block_size`` tokens:
//   k_codes int8 [blocks][kv_heads][block_size][width]   k_scale fp32 [blocks][kv_heads]
//   v_codes int8 [blocks][kv_heads][width][block_size]   v_scale fp32 [blocks][kv_heads]
// An element stands for code * scale.  Keys are contracted over the head's columns and lie row by row, values
// are contracted over the tokens and lie column by column: both are then read from memory straight into
// matrix-core operands, without a transposition on the way.
#include "common.h"
#include "kv_attention.h"

// ---------------------------------------------------------------- block plans
// One workgroup sums over the requests (new rows, blocks taken, blocks given back), decides whether the
// plan fits, and leaves the running sums; rows, table entries and returned blocks are then filled in by
// ``plan_fill``, in the same workgroup or in a launch of many.  Whole numbers throughout.
// Bound by latency: 16 requests 6.0 us in one launch; 2048 requests, half of them giving back some 250 blocks each, 11.8 K new
// rows 6.8 + 7.0 us in two (318 us when one workgroup filled them; 8.2 us for the filling when a row searched for its request
// instead of a request's wave laying out its rows).
#define PLAN_THREADS 1024

struct PlanArgs {
    const int32_t* lens;
    const int32_t* new_rows;
    int32_t* tables;
    long ld_tables;
    int32_t* free_blocks;
    const int32_t* free_count;
    int32_t *cu_rows, *slots, *positions, *lens_out, *free_count_out, *status;
    int32_t* work;          // [2][B] first block taken / given back by a request, then {blocks in the stack, level, fits}
    int32_t* before;        // [B] lengths before the plan
    int B, table_width, free_capacity, block_size, rows;
};

struct PlanSum {
    long long rows;
    long long taken, given;
};

__device__ __forceinline__ long long shfl_up64(long long v, int o) { return __shfl_up(v, o, 64); }

// blocks of n tokens
__device__ __forceinline__ int blocks_of(long long n, int bs) { return (int)((n + bs - 1) / bs); }

// entry ``at`` of the stack of free blocks with the given-back ones on top of it; ``given`` [B]: given-back blocks in front
// of a request (in LDS where they fit)
__device__ __forceinline__ int plan_stack(const PlanArgs& a, const int32_t* given, int count, int at) {
    if (at < count) return a.free_blocks[at];
    const int f = at - count;
    int lo = 0, hi = a.B - 1;                   // last request whose first given-back block is <= f
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (given[mid] <= f) lo = mid;
        else hi = mid - 1;
    }
    return a.tables[(long)lo * a.ld_tables + (f - given[lo])];
}

// a wave per request: its rows, its new table entries or its returned blocks; threads [first, first + step, ...)
__device__ __forceinline__ void plan_fill(const PlanArgs& a, const int32_t* given, int first, int step) {
    const int32_t* end = a.work + 2 * a.B;
    const int count = end[0], level = end[1], fits = end[2], bs = a.block_size;
    for (int t = (fits ? a.cu_rows[a.B] : 0) + first; t < a.rows; t += step) {      // behind the last row
        a.slots[t] = -1;
        a.positions[t] = 0;
    }
    if (!fits) return;
    const int lane = first & 63;
    for (int b = first >> 6; b < a.B; b += step >> 6) {
        const int len = a.before[b], n = a.new_rows[b], have = blocks_of(len, bs);
        int32_t* row = a.tables + (long)b * a.ld_tables;
        if (n < 0) {
            const int at = count + a.work[a.B + b];
            for (int j = lane; j < have; j += 64) a.free_blocks[at + j] = row[j];
            continue;
        }
        const int row0 = a.cu_rows[b], taken = a.work[b];
        // 64 blocks at a time: a lane finds one of them, then the rows look their block up in the lanes
        const int last = blocks_of((long long)len + n, bs);
        for (int j0 = len / bs; j0 < last; j0 += 64) {
            const int j = j0 + lane;
            int block = -1;
            if (j < have) block = row[j];
            else if (j < last) {
                block = plan_stack(a, given, count, level - 1 - (taken + j - have));
                row[j] = block;
            }
            const int from = max(j0 * bs, len), to = (int)min((long long)(j0 + 64) * bs, (long long)len + n);
            for (int p0 = from; p0 < to; p0 += 64) {
                const int p = p0 + lane, mine = __shfl(block, min(p / bs - j0, 63), 64);
                if (p < to) {
                    a.slots[row0 + p - len] = mine < 0 ? -1 : mine * bs + p % bs;
                    a.positions[row0 + p - len] = p;
                }
            }
        }
    }
}

__global__ __launch_bounds__(PLAN_THREADS) void kv_plan_kernel(PlanArgs a, int fill) {
    __shared__ PlanSum part[PLAN_THREADS / 64];
    __shared__ int s_long, s_fits;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int per = (a.B + PLAN_THREADS - 1) / PLAN_THREADS, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    if (tid == 0) s_long = 0;
    __syncthreads();
    PlanSum mine = {0, 0, 0};
    int too_long = 0;
    const long long top = (long long)a.table_width * a.block_size;
    for (int b = b0; b < b1; ++b) {
        const int len = a.lens[b], n = a.new_rows[b];
        if (len < 0 || (long long)len + max(n, 0) > top) {
            ++too_long;
            continue;
        }
        const int have = blocks_of(len, a.block_size);
        if (n < 0) mine.given += have;
        else {
            mine.rows += n;
            mine.taken += blocks_of((long long)len + n, a.block_size) - have;
        }
    }
    if (too_long) atomicAdd(&s_long, too_long);
    PlanSum run = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long r = shfl_up64(run.rows, o), t = shfl_up64(run.taken, o), g = shfl_up64(run.given, o);
        if (lane >= o) { run.rows += r; run.taken += t; run.given += g; }
    }
    if (lane == 63) part[w] = run;
    __syncthreads();
    PlanSum base = {0, 0, 0}, all = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < PLAN_THREADS / 64; ++i) {
        if (i < w) { base.rows += part[i].rows; base.taken += part[i].taken; base.given += part[i].given; }
        all.rows += part[i].rows; all.taken += part[i].taken; all.given += part[i].given;
    }
    int32_t* end = a.work + 2 * a.B;
    if (tid == 0) {
        const int count = min(max(a.free_count[0], 0), a.free_capacity);
        const long long level = count + all.given;
        const long long missing = max(all.taken - level, 0ll), rows_over = max(all.rows - a.rows, 0ll),
                        stack_over = max(level - a.free_capacity, 0ll);
        const int fits = !(s_long || missing || rows_over || stack_over);
        const long long most = 0x7fffffff;
        a.status[0] = (int)min(missing, most);
        a.status[1] = s_long;
        a.status[2] = (int)min(rows_over, most);
        a.status[3] = (int)min(stack_over, most);
        end[0] = count;
        end[1] = fits ? (int)level : count;
        end[2] = fits;
        s_fits = fits;
        a.cu_rows[a.B] = fits ? (int)all.rows : 0;
        a.free_count_out[0] = fits ? (int)(level - all.taken) : a.free_count[0];
    }
    __syncthreads();
    const int fits = s_fits;
    long long rows = base.rows + run.rows - mine.rows, taken = base.taken + run.taken - mine.taken,
              given = base.given + run.given - mine.given;
    for (int b = b0; b < b1; ++b) {
        const int len = a.lens[b], n = a.new_rows[b];
        a.before[b] = len;
        a.cu_rows[b] = fits ? (int)rows : 0;
        a.work[b] = (int)taken;
        a.work[a.B + b] = (int)given;
        a.lens_out[b] = !fits ? len : n < 0 ? 0 : len + n;
        if (!fits) continue;
        const int have = blocks_of(len, a.block_size);
        if (n < 0) given += have;
        else {
            rows += n;
            taken += blocks_of((long long)len + n, a.block_size) - have;
        }
    }
    if (!fill) return;
    __threadfence_block();
    __syncthreads();
    plan_fill(a, a.work + a.B, tid, PLAN_THREADS);
}

#define PLAN_LDS 8192       // requests whose running sums a workgroup keeps in LDS
__global__ __launch_bounds__(256) void kv_plan_fill_kernel(PlanArgs a) {
    __shared__ int32_t sums[PLAN_LDS];
    const int32_t* given = a.work + a.B;
    if (a.B <= PLAN_LDS) {
        for (int b = threadIdx.x; b < a.B; b += 256) sums[b] = given[b];
        __syncthreads();
        given = sums;
    }
    plan_fill(a, given, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

extern "C" int athena_kv_plan(const athena_kv_plan_desc* d, athena_stream_t stream) {
    ATHENA_REQUIRE(d, ATHENA_E_SHAPE, "athena_kv_plan: null descriptor");
    ATHENA_REQUIRE(d->B > 0 && d->table_width > 0 && d->free_capacity > 0 && d->rows >= 0 && d->ld_tables >= d->table_width,
                   ATHENA_E_SHAPE, "athena_kv_plan: bad shape B=%d table_width=%d free_capacity=%d rows=%d ld=%ld", d->B,
                   d->table_width, d->free_capacity, d->rows, (long)d->ld_tables);
    const int bs = d->block_size;
    ATHENA_REQUIRE(bs == 16 || bs == 32 || bs == 64 || bs == 128, ATHENA_E_UNSUPPORTED,
                   "athena_kv_plan: block size %d not in {16, 32, 64, 128}", bs);
    // (steps of 64 places past the last one stay below 2^31)
    ATHENA_REQUIRE((long)d->table_width * bs < (1L << 31) - KV_KEYS * 8, ATHENA_E_SHAPE, "athena_kv_plan: table too wide");
    ATHENA_REQUIRE(d->lens && d->new_rows && d->tables && d->free_blocks && d->free_count && d->cu_rows &&
                       ((d->slots && d->positions) || !d->rows) && d->lens_out && d->free_count_out && d->status && d->work,
                   ATHENA_E_SHAPE, "athena_kv_plan: null operand");
    PlanArgs a = {d->lens, d->new_rows, d->tables, d->ld_tables, d->free_blocks, d->free_count, d->cu_rows, d->slots, d->positions,
                  d->lens_out, d->free_count_out, d->status, d->work, d->work + 2L * d->B + 3, d->B, d->table_width,
                  d->free_capacity, bs, d->rows};
    hipStream_t s = (hipStream_t)stream;
    // one workgroup fills the rows of a few requests a wave itself; beyond that a launch of many is faster
    const int fill = d->rows <= 4 * PLAN_THREADS && d->B <= 8 * (PLAN_THREADS / 64);
    ATHENA_LAUNCH(kv_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, s, a, fill);
    ATHENA_CHECK_LAUNCH("athena_kv_plan");
    if (!fill) {
        const int wgs = (d->B + 3) / 4;
        ATHENA_LAUNCH(kv_plan_fill_kernel, dim3(wgs < 1024 ? wgs : 1024), dim3(256), 0, s, a);
        ATHENA_CHECK_LAUNCH("athena_kv_plan (fill)");
    }
    return ATHENA_OK;
}

// ---------------------------------------------------------------- writing new keys and values
// Consecutive rows that go to the same block are one run: the block's scale grows to the largest magnitude of
// the run / 127 (from nothing where the run begins the block), codes in front of the run are brought to a grown
// scale, and the run's codes are written.  A run, kv head and side (keys or values) belongs to one wave, or to a
// team of four that divide its places and exchange their largest magnitudes; the workgroup that finds a run's first
// row takes all of it, so two never meet in a block.
//
// Codes are round-half-to-even(x / scale) exactly.  (bf16 values and a scale made of one of them have few distinct
// quotients: one in 300 lies on or next to a border.)  The quotient in fp32 gives a whole number next to the right one,
// and the remainder x - code * scale, which one fused multiply-add leaves exactly (a multiple of 2^-24 of the scale's power
// of two, at most half the scale or so), decides.  Rounding in fp32 is an addition of 1.5 * 2^23, whose lowest byte is the code.
//
// A lane holds two columns of 16 consecutive places, so that the values' codes (16 bytes of one column) leave
// in one store.  Bound by latency: slots -> rows -> largest magnitude -> codes is a chain of four trips to memory, about 5 us a
// run.  8192 rows of 8 heads of 128 in bf16 26 us (50 MB, 1.9 TB/s; fp32 31 us), 256 single rows 9.8 us, ten of 4 heads of 64 4.9 us.
// Where every run makes its block's scale grow, 35 and 25 us: the codes in front of it are read and written again, four at a time.
template <typename T> struct AppendSide {
    const T* x;
    long ld_row, ld_head;
    int8_t* codes;
    float* scale;
};

#define KV_ROUND 12582912.f         // 1.5 * 2^23
#define KV_DOUBT 1.3e-7f            // a product in fp32 of a rounded ratio is off by at most 2^-23 of itself
// code of a number, in the lowest byte; ``s`` at least 1e-30 (see tiny below)
__device__ __forceinline__ unsigned code_of(float x, float s, float inv) {
    const float y = fmaf(x, inv, KV_ROUND), r = fmaf(-(y - KV_ROUND), s, x);
    // beyond half the scale, or at it with an odd code: one further (the bound is 0 for odd codes, the least number for even)
    const float beyond = fmaf(2.f, fabsf(r), -s), bound = __uint_as_float((__float_as_uint(y) & 1u) ^ 1u);
    return __float_as_uint(y + (beyond >= bound ? copysignf(1.f, r) : 0.f));
}
// a code brought from scale s0 to s1: products of both sides of a border are compared in 64 bits, where they are exact
__device__ __forceinline__ float kv_recode_border(float q, float c, float s0, float s1) {
    const double num = (double)q * (double)s0, up = (c + 0.5) * (double)s1, down = (c - 0.5) * (double)s1;
    const bool odd = (int)c & 1;
    return num > up || (odd && num == up) ? c + 1.f : num < down || (odd && num == down) ? c - 1.f : c;
}
// scales below 1e-30 have reciprocals that do not fit: both sides are multiplied by 2^100 first, and what a scale rounded to
// few bits leaves beyond 127 is cut
#define KV_TINY 1e-30f
#define KV_LIFT 1.2676506002282294e30f
__device__ __forceinline__ float kv_lift(float x, float lifted) { return fminf(fmaxf(x * KV_LIFT, -127.f * lifted), 127.f * lifted); }
// the first ``keep`` of four codes in a word, brought from scale s0 to s1
__device__ __forceinline__ unsigned recode4(unsigned w, int keep, float s0, float s1, float ratio) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = (float)(int8_t)(w >> (8 * i)), f = q * ratio;
        float y = f + KV_ROUND;
        if (fmaf(fabsf(f), KV_DOUBT, fabsf(f - (y - KV_ROUND))) > 0.5f) y = kv_recode_border(q, y - KV_ROUND, s0, s1) + KV_ROUND;
        if (i < keep) w = (w & ~(0xffu << (8 * i))) | ((__float_as_uint(y) & 0xffu) << (8 * i));
    }
    return w;
}
// the lowest bytes of four words
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

template <typename T, int W, bool VALUES>
__device__ __forceinline__ void append_run(const AppendSide<T>& a, const int32_t* __restrict__ slots, long slots_end, int t, int n,
                                           int first, bool straight, int block, int head, int hk, int dk, int block_size, bool pairs,
                                           int lane, int rank, int team, unsigned* tops) {
    constexpr int LR = W / 2, SUB = 64 / LR;                // lanes of a row, groups of 16 places side by side
    const int sub = lane / LR, c = 2 * (lane % LR);
    const T* x = a.x + (long)t * a.ld_row + (long)head * a.ld_head;
    const int ld = (int)a.ld_row;
    const long at = (long)block * hk + head;
    int8_t* codes = a.codes + at * W * block_size;
    const int step = 16 * SUB, begin = first & ~15, end = first + n;
    const float s0 = first == 0 ? 0.f : a.scale[at];
    struct alignas(2 * sizeof(T)) Pair { T e[2]; };
    // Runs of more than a few rows: two columns of 16 places at once, all requests out before the first is waited for.  Places
    // outside the run read the run's nearest row (which leaves the largest magnitude as it is) and are not written.
    const bool fast = pairs && n > 4;
    Pair raw[16];
    auto load = [&](int base) {
        const int r0 = base + 16 * sub - first;
        const unsigned col = (c < dk ? c : 0) * (unsigned)sizeof(T), pitch = ld * (unsigned)sizeof(T);
#pragma unroll
        for (int i = 0; i < 16; ++i) raw[i] = *(const Pair*)((const char*)x + (min(max(r0 + i, 0), n - 1) * pitch + col));
        if (c >= dk) {
#pragma unroll
            for (int i = 0; i < 16; ++i) raw[i].e[0] = raw[i].e[1] = from_f32<T>(0.f);
        }
    };
    // others (single rows, odd columns): four places at a time, each looked at by itself
    auto load4 = [&](int p0, float (&f)[4][2]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = p0 + i - first;
            T e0 = from_f32<T>(0.f), e1 = e0;
            if ((unsigned)r < (unsigned)n && c < dk) e0 = x[r * ld + c];
            if ((unsigned)r < (unsigned)n && c + 1 < dk) e1 = x[r * ld + c + 1];
            f[i][0] = to_f32<T>(e0);
            f[i][1] = to_f32<T>(e1);
        }
    };
    // runs that are not straight: their rows one after the other, in order, with their slots; any number of skipped rows may stand between
    auto each_row = [&](auto f) {
#pragma unroll 1
        for (int r0 = 0; r0 < n; r0 += 64) {
            const int s = r0 + lane < n ? slots[t + r0 + lane] : -1;
#pragma unroll 1
            for (unsigned long long left = __ballot(s >= 0 && s < slots_end); left; left &= left - 1) {
                const int at = __ffsll((long long)left) - 1;
                f(r0 + at, __builtin_amdgcn_readlane(s, at));
            }
        }
    };
    unsigned top = 0;                                       // largest magnitude, as bits: NaN over infinity over numbers
    const auto mag = [](float f) { return __float_as_uint(f) & 0x7fffffffu; };
    if (straight) {
#pragma unroll 1
        for (int base = begin + rank * step; base < end; base += team * step) {
            if (fast) {
                load(base);
#pragma unroll
                for (int i = 0; i < 16; ++i) top = max(top, max(mag(to_f32<T>(raw[i].e[0])), mag(to_f32<T>(raw[i].e[1]))));
            } else {
#pragma unroll 1
                for (int g = 0; g < 16; g += 4) {
                    const int p0 = base + 16 * sub + g;
                    if (!__any(p0 + 4 > first && p0 < end)) continue;
                    float f[4][2];
                    load4(p0, f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = max(top, max(mag(f[i][0]), mag(f[i][1])));
                }
            }
        }
    } else if (rank == 0) {
        each_row([&](int r, int) {
            for (int col = lane; col < dk; col += 64) top = max(top, mag(to_f32<T>(x[(long)r * a.ld_row + col])));
        });
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    if (team > 1) {
        if (lane == 0) tops[rank] = top;
        __syncthreads();                                    // (every wave of the workgroup is here: teams go through runs together)
        for (int i = 0; i < team; ++i) top = max(top, tops[i]);
    }
    top = __builtin_amdgcn_readfirstlane(top);
    // (as whole numbers, so that a scale that is not finite stays; it is kept as NaN)
    const unsigned bits = max(mag(s0), mag(__uint_as_float(top) / 127.f));
    const float s1 = __uint_as_float(bits < 0x7f800000u ? bits : 0x7fc00000u);
    if (s1 > s0 && first > 0) {
        const float ratio = s0 / s1;
        // four codes at a time; those of the 16 places that ``first`` cuts belong to the wave that writes the others of them
        const int whole = VALUES ? first / 16 * 4 : first * W / 4, columns = VALUES ? W : 1;
#pragma unroll 1
        for (int e = lane + 64 * rank; e < whole * columns; e += 64 * team) {
            const int col = e / whole, k = e - col * whole;
            unsigned* p = (unsigned*)(codes + col * block_size + 4 * k);
            *p = recode4(*p, 4, s0, s1, ratio);
        }
        if (VALUES && rank == 0 && (first & 15)) {
#pragma unroll 1
            for (int e = lane; e < 4 * W; e += 64) {
                const int keep = (first & 15) - 4 * (e & 3);
                unsigned* p = (unsigned*)(codes + (e >> 2) * block_size + 4 * whole + 4 * (e & 3));
                if (keep > 0) *p = recode4(*p, keep, s0, s1, ratio);
            }
        }
    }
    const bool tiny = s1 > 0.f && s1 < KV_TINY;
    // (a block of zeros has scale 0, and codes 0 beside any scale)
    const float sd = tiny ? s1 * KV_LIFT : s1 == 0.f ? 3e38f : s1, inv = s1 > 0.f ? 1.f / sd : 0.f;
    if (straight) {
#pragma unroll 1
        for (int base = begin + rank * step; base < end; base += team * step) {
            if (fast && !tiny) {
                if (end - begin > team * step) load(base);  // (otherwise the registers hold the rows still)
                const int p0 = base + 16 * sub;
                const bool whole = p0 >= first && p0 + 16 <= end;
                unsigned w[2][4];                           // codes of a column, four places to a word
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    unsigned q[4][2];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int k = 0; k < 2; ++k) q[i][k] = code_of(to_f32<T>(raw[4 * g + i].e[k]), sd, inv);
                    if (VALUES) {
                        w[0][g] = low_bytes(q[0][0], q[1][0], q[2][0], q[3][0]);
                        w[1][g] = low_bytes(q[0][1], q[1][1], q[2][1], q[3][1]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (whole || (p0 + 4 * g + i >= first && p0 + 4 * g + i < end))
                                *(uint16_t*)(codes + (p0 + 4 * g + i) * W + c) = (uint16_t)__builtin_amdgcn_perm(q[i][1], q[i][0], 0x0c0c0400u);
                    }
                }
                if (VALUES) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        int8_t* p = codes + (c + k) * block_size + p0;
                        if (whole) *(uint4*)p = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
                        else {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (p0 + i >= first && p0 + i < end) p[i] = (int8_t)(w[k][i >> 2] >> (8 * (i & 3)));
                        }
                    }
                }
            } else {
#pragma unroll 1
                for (int g = 0; g < 16; g += 4) {
                    const int p0 = base + 16 * sub + g;
                    if (!__any(p0 + 4 > first && p0 < end)) continue;
                    float f[4][2];
                    load4(p0, f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (p0 + i < first || p0 + i >= end) continue;
                        const unsigned q0 = code_of(tiny ? kv_lift(f[i][0], sd) : f[i][0], sd, inv),
                                       q1 = code_of(tiny ? kv_lift(f[i][1], sd) : f[i][1], sd, inv);
                        if (VALUES) {
                            codes[c * block_size + p0 + i] = (int8_t)q0;
                            codes[(c + 1) * block_size + p0 + i] = (int8_t)q1;
                        } else *(uint16_t*)(codes + (p0 + i) * W + c) = (uint16_t)__builtin_amdgcn_perm(q1, q0, 0x0c0c0400u);
                    }
                }
            }
        }
    } else if (rank == 0) {
        each_row([&](int r, int s) {                        // (of two rows for one place the later stays)
            for (int col = lane; col < W; col += 64) {
                float f = col < dk ? to_f32<T>(x[(long)r * a.ld_row + col]) : 0.f;
                if (tiny) f = kv_lift(f, sd);
                codes[VALUES ? col * block_size + s % block_size : (s % block_size) * W + col] = (int8_t)code_of(f, sd, inv);
            }
        });
    }
    if (lane == 0 && rank == 0) a.scale[at] = s1;
}

#define KV_TEAM 4
template <typename T, int W, bool VALUES>
__device__ __forceinline__ void append_rows(const AppendSide<T>& a, const int32_t* __restrict__ slots, int N, int rows_per_wg, int hk,
                                            int dk, int shift, bool pairs, long slots_end, unsigned (*tops)[KV_TEAM]) {
    // (what is the same in all lanes of a wave is said to be, or the compiler keeps it per lane)
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6, head = blockIdx.y;
    const int t0 = blockIdx.x * rows_per_wg, block_size = 1 << shift;
    const auto good = [&](int s) { return s >= 0 && s < slots_end; };
    // the slots of these rows and of the 64 behind them, in one trip to memory
    const int sa = t0 + lane < N ? slots[t0 + lane] : -1, sb = t0 + 64 + lane < N ? slots[t0 + 64 + lane] : -1;
    const int before = t0 > 0 ? slots[t0 - 1] : -1;
    // first rows of runs among the workgroup's rows; skipped rows do not end a run
    int p = __shfl_up(sa, 1, 64);
    if (lane == 0) p = before;
    const bool mine = lane < rows_per_wg && good(sa);
    for (unsigned long long gaps = __ballot(mine && !good(p) && t0 + lane > 0); gaps; gaps &= gaps - 1) {
        const int at = __ffsll((long long)gaps) - 1;        // the row behind a skipped one: back to the last that was not
        int seen = -1;
        for (int r0 = t0 + at - 1; r0 >= 0 && seen < 0; r0 -= 64) {
            const int s = r0 - lane >= 0 ? slots[r0 - lane] : -1;
            const unsigned long long any = __ballot(good(s));
            if (any) seen = __builtin_amdgcn_readlane(s, __ffsll((long long)any) - 1);
        }
        if (lane == at) p = seen;
    }
    const bool leads = mine && (!good(p) || p >> shift != sa >> shift);
    unsigned long long found = __ballot(leads);             // (the same in every wave)
    // few runs (chunks of prompts): teams of four waves; many (single tokens): a wave each
    const int team = nw == KV_TEAM && __popcll(found) <= 2 ? KV_TEAM : 1, rank = team > 1 ? w : 0;
    for (int run = 0; found; ++run) {
        const int at = __ffsll((long long)found) - 1, t = t0 + at;
        found &= found - 1;
        if (team == 1 && run % nw != w) continue;
        const int s0 = __builtin_amdgcn_readlane(sa, at), block = s0 >> shift;
        // rows up to the run's last one, first place; straight: no row skipped, places in order (the usual run, and one that
        // ends among the slots at hand)
        const int ra = lane - at, rb = 64 - at + lane;
        const unsigned long long stop_a = __ballot(ra >= 0 && sa != s0 + ra), stop_b = __ballot(sb != s0 + rb);
        int n = min(stop_a ? __ffsll((long long)stop_a) - 1 - at : stop_b ? 64 - at + __ffsll((long long)stop_b) - 1 : 128 - at,
                    block_size - (s0 & (block_size - 1)));
        int first = s0 & (block_size - 1);
        bool straight = t + n >= N;
        if (!straight && at + n < 128) {                    // what stands behind decides: another block
            const int behind = at + n < 64 ? __builtin_amdgcn_readlane(sa, at + n) : __builtin_amdgcn_readlane(sb, at + n - 64);
            straight = good(behind) && behind >> shift != block;
        }
        if (!straight) {
            n = 0;
            first = block_size;
            bool more = true, order = true;
            for (int r1 = 0; more; r1 += 256) {             // (skipped rows behind the last run are a padded batch's usual end)
                int four[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) four[i] = t + r1 + 64 * i + lane < N ? slots[t + r1 + 64 * i + lane] : -1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r0 = r1 + 64 * i, r = r0 + lane, s = four[i];
                    const unsigned long long same = __ballot(good(s) && s >> shift == block),
                                             other = __ballot(t + r >= N || (good(s) && s >> shift != block));
                    const unsigned long long in = !more ? 0 : other ? same & ((other & -other) - 1) : same;
                    if (in) {
                        const int last = 63 - __clzll((long long)in);
                        order = order && n == r0 && __ballot(lane <= last && s != s0 + r) == 0;
                        n = r0 + last + 1;
                        int q = (in >> lane) & 1 ? s & (block_size - 1) : block_size;
#pragma unroll
                        for (int o = 32; o > 0; o >>= 1) q = min(q, __shfl_xor(q, o, 64));
                        first = min(first, __builtin_amdgcn_readfirstlane(q));
                    }
                    more = more && !other;
                }
            }
            straight = order;
        }
        append_run<T, W, VALUES>(a, slots, slots_end, t, n, first, straight, block, head, hk, dk, block_size, pairs, lane, rank, team,
                                 tops[run & 1]);
    }
}

template <typename T, int W>
__global__ __launch_bounds__(64 * KV_TEAM) void kv8_append_kernel(AppendSide<T> ks, AppendSide<T> vs, const int32_t* __restrict__ slots,
                                                                 int N, int rows_per_wg, int hk, int dk, int shift, int k_pairs,
                                                                 int v_pairs, long slots_end) {
    __shared__ unsigned tops[2][KV_TEAM];
    if (blockIdx.z) append_rows<T, W, true>(vs, slots, N, rows_per_wg, hk, dk, shift, v_pairs, slots_end, tops);
    else append_rows<T, W, false>(ks, slots, N, rows_per_wg, hk, dk, shift, k_pairs, slots_end, tops);
}

static int kv8_check(const char* name, int num_blocks, int hk, int block_size, int dk, int width) {
    ATHENA_REQUIRE(num_blocks > 0 && hk > 0 && hk <= 65535 && dk > 0 && dk <= width, ATHENA_E_SHAPE,
                   "%s: bad shape blocks=%d kv_heads=%d head=%d width=%d", name, num_blocks, hk, dk, width);
    ATHENA_REQUIRE(block_size == 16 || block_size == 32 || block_size == 64 || block_size == 128, ATHENA_E_UNSUPPORTED,
                   "%s: block size %d not in {16, 32, 64, 128}", name, block_size);
    ATHENA_REQUIRE(width == 32 || width == 64 || width == 128, ATHENA_E_UNSUPPORTED, "%s: width %d not in {32, 64, 128}", name,
                   width);
    ATHENA_REQUIRE((long)num_blocks * block_size < (1L << 31), ATHENA_E_SHAPE, "%s: more than 2^31 places", name);
    return ATHENA_OK;
}

extern "C" int athena_kv8_append(const athena_kv8_append_desc* d, athena_stream_t stream) {
    ATHENA_REQUIRE(d, ATHENA_E_SHAPE, "athena_kv8_append: null descriptor");
    const int num_blocks = d->num_blocks, hk = d->hk, block_size = d->block_size, dk = d->dk, width = d->width, N = d->N;
    int rc = kv8_check("athena_kv8_append", num_blocks, hk, block_size, dk, width);
    if (rc) return rc;
    // (64 rows a workgroup of 256 threads: fewer than 2^32 threads)
    ATHENA_REQUIRE(N >= 0 && N <= (1 << 30) - 64, ATHENA_E_SHAPE, "athena_kv8_append: N=%d (2^30 - 64 at most)", N);
    ATHENA_REQUIRE(d->dtype == ATHENA_F32 || d->dtype == ATHENA_BF16, ATHENA_E_UNSUPPORTED, "athena_kv8_append: dtype");
    if (N == 0) return ATHENA_OK;
    const void *k = d->k, *v = d->v;
    const long ldk = d->ldk, ldk_head = d->ldk_head, ldv = d->ldv, ldv_head = d->ldv_head;
    const int32_t* slots = d->slots;
    int8_t *k_codes = d->k_codes, *v_codes = d->v_codes;
    float *k_scale = d->k_scale, *v_scale = d->v_scale;
    ATHENA_REQUIRE(k && v && slots && k_codes && v_codes && k_scale && v_scale, ATHENA_E_SHAPE, "athena_kv8_append: null operand");
    ATHENA_REQUIRE(athena_aligned16(k_codes) && athena_aligned16(v_codes), ATHENA_E_ALIGN, "athena_kv8_append: codes must lie on 16 bytes");
    ATHENA_REQUIRE(ldk >= 0 && ldv >= 0 && ldk < (1 << 22) && ldv < (1 << 22), ATHENA_E_SHAPE,
                   "athena_kv8_append: rows %ld / %ld elements apart (2^22 at most)", ldk, ldv);
    // Rows of a workgroup.  The host does not see the runs: single rows want a wave each, chunks a team per run and few workgroups that
    // leave at once.  1 / 8 / 64 rows a workgroup, heads of 128 in bf16, blocks of 64, us: single rows 256 x 8 heads 9.6 / 11.1 / 46.8,
    // 513 x 8 15.9 / 17.3 / 48.6, 1024 x 8 25.7 / 25.9 / 50.2, 2048 x 8 45.5 / 46.4 / 58.2; chunks of 512 rows, 512 x 4 heads
    // 18.5 / 5.7 / 8.4, 512 x 8 20.3 / 8.1 / 8.5, 2048 x 4 35.7 / 14.3 / 8.8, 8192 x 8 237 / 81 / 28.
    const int per = (long)N * hk <= 2048 ? 1 : (long)N * hk <= 8192 ? 8 : 64;
    const dim3 grid((N + per - 1) / per, hk, 2), block(per == 1 ? 64 : 64 * KV_TEAM);
    const long end = (long)num_blocks * block_size;
    const int shift = __builtin_ctz(block_size);
    const size_t two = d->dtype == ATHENA_BF16 ? 4 : 8;        // two elements in one load where rows and heads begin on them
    const int kp = (uintptr_t)k % two == 0 && ldk % 2 == 0 && ldk_head % 2 == 0 && dk % 2 == 0;
    const int vp = (uintptr_t)v % two == 0 && ldv % 2 == 0 && ldv_head % 2 == 0 && dk % 2 == 0;
#define KV_APPEND(T, W)                                                                                                     \
    do {                                                                                                                    \
        AppendSide<T> ks = {(const T*)k, ldk, ldk_head, k_codes, k_scale}, vs = {(const T*)v, ldv, ldv_head, v_codes, v_scale}; \
        ATHENA_LAUNCH((kv8_append_kernel<T, W>), grid, block, 0, (hipStream_t)stream, ks, vs, slots, N, per, hk, dk, shift,      \
                      kp, vp, end);                                                                                         \
    } while (0)
#define KV_APPEND_W(T)                     \
    do {                                   \
        if (width == 32) KV_APPEND(T, 32); \
        else if (width == 64) KV_APPEND(T, 64); \
        else KV_APPEND(T, 128);            \
    } while (0)
    if (d->dtype == ATHENA_BF16) KV_APPEND_W(bf16_t);
    else KV_APPEND_W(float);
#undef KV_APPEND_W
#undef KV_APPEND
    ATHENA_CHECK_LAUNCH("athena_kv8_append");
    return ATHENA_OK;
}

// ---------------------------------------------------------------- attention over the cache
struct KvShape {
    int row_tiles;                  // sequences of few rows: tiles of 16 rows
    int waves, row_tiles_many;      // sequences of many rows: waves of a workgroup (0: there are none), row tiles
    int splits;                     // shares of the key axis
};
// tiles of 16 rows per wave of the kernel of many rows: what fits the registers
static constexpr int kv8_rt_many(int bytes, int width) { return bytes == 4 && width == 128 ? 1 : 2; }

// A split costs a second launch (the join, 4 us and more) and the partial results' way out and in, so none has fewer than
// KV_MIN_TILES tiles, and there are as many as fill the chip about three times over: 768 / 1536 / 2560 / 6000 workgroups took
// 125 / 121 / 124 / 148 us for 64 requests of up to 8192 tokens and 358 / 361 / 366 / 385 us for 8 contexts of 131 K; of many
// rows 1024 / 1536 / 2048 took 466 / 446 / 463 us for chunks of 512 rows behind 16 K.  At least 16 / 8 / 4 tiles a split: 21.2 /
// 15.8 / 14.9 us for 8 rows on 3.7 to 7.5 K tokens, 61 / 49 / 63 us for 13 chunks of 412 rows behind 1500.
static KvShape kv8_shape(const athena_kv8_attention_desc* d) {
    KvShape s;
    const long G = d->h / d->hk, most = (long)(d->cu_rows ? d->max_rows : 1) * G, few = G > KV_FEW ? G : KV_FEW, rows = most < few ? most : few;
    s.row_tiles = (int)((rows + 15) / 16);
    const int rt = kv8_rt_many(d->dtype == ATHENA_F32 ? 4 : 2, d->width);
    // (heads of 128: two waves fit a SIMD either way, and eight share a tile's widening, 440 against 475 us for chunks of 512 rows
    // x 4 heads behind 16 K tokens; smaller heads: three workgroups of four fit a CU and hide each other's barriers, 195 against
    // 230 us for prompts of 4001 rows)
    s.waves = most <= few ? 0 : most > 512 && d->width == 128 ? 8 : 4;
    const long tiles = s.waves ? (most + 16 * rt * s.waves - 1) / (16 * rt * s.waves) : 0;
    s.row_tiles_many = (int)(tiles < 65536 ? tiles : 65536);
    const long pairs = (long)d->B * d->hk, units = pairs * s.row_tiles, units_many = pairs * s.row_tiles_many * (s.waves / 4);
    const long cap = (long)d->table_width * d->block_size / (KV_KEYS * KV_MIN_TILES);      // below 1024 places: 1
    // (at least what N rows take however they are spread over the sequences, or a max_rows below the truth would have a workspace of
    // hundreds of splits for all of them; as it is no call needs more than 204 MB)
    const long wg_rows = s.waves ? 64 * rt : 16, all = d->hk * ((d->N * G + wg_rows - 1) / wg_rows), named = s.waves ? units_many : units;
    const long work = all > named ? all : named;
    long splits = (1535 + work) / work;
    if (splits > cap) splits = cap;
    s.splits = (int)(splits < 1 ? 1 : splits > 256 ? 256 : splits);
    return s;
}

extern "C" int64_t athena_kv8_attention_workspace_bytes(const athena_kv8_attention_desc* d) {
    if (!d || d->B <= 0 || d->max_rows <= 0 || d->N <= 0 || d->hk <= 0 || d->h < d->hk || d->table_width <= 0 || d->block_size <= 0 ||
        d->dk <= 0)
        return 0;
    const KvShape s = kv8_shape(d);
    return s.splits > 1 ? (int64_t)s.splits * d->N * d->h * (d->dk + 1) * 4 : 0;
}

template <typename T, int W>
static void kv8_launch(KvAttn a, const KvShape& sh, hipStream_t s) {
    const long pairs = ((long)a.B * a.hk + 7) / 8 * 8;
    const dim3 block(256);
    if (sh.waves) {
        a.row_tiles = sh.row_tiles_many;
        const dim3 grid((unsigned)(pairs * sh.row_tiles_many * sh.splits));
        constexpr int RT = kv8_rt_many(sizeof(T), W);
        if (sh.waves == 8) {
            if constexpr (W == 128) ATHENA_LAUNCH((kv8_attention_rows_kernel<T, W, RT, 8>), grid, dim3(512), 0, s, a);
        } else ATHENA_LAUNCH((kv8_attention_rows_kernel<T, W, RT, 4>), grid, block, 0, s, a);
    }
    a.row_tiles = sh.row_tiles;
    const dim3 grid((unsigned)(pairs * sh.row_tiles * sh.splits));
    ATHENA_LAUNCH((kv8_attention_kernel<T, W>), grid, block, 0, s, a);
}

extern "C" int athena_kv8_attention(const athena_kv8_attention_desc* d, athena_stream_t stream) {
    ATHENA_REQUIRE(d, ATHENA_E_SHAPE, "athena_kv8_attention: null descriptor");
    int rc = kv8_check("athena_kv8_attention", d->num_blocks, d->hk, d->block_size, d->dk, d->width);
    if (rc) return rc;
    const int B = d->B, N = d->N, h = d->h, hk = d->hk, e = d->dtype == ATHENA_BF16 ? 2 : 4;
    ATHENA_REQUIRE(B > 0 && B <= 65535 && N >= 0 && d->max_rows > 0 && h > 0 && h <= 65535 && h % hk == 0 && d->table_width > 0 &&
                       (long)d->table_width * d->block_size < (1L << 31) - KV_KEYS * 8,
                   ATHENA_E_SHAPE, "athena_kv8_attention: bad shape B=%d N=%d max_rows=%d heads=%d kv_heads=%d table_width=%d", B, N,
                   d->max_rows, h, hk, d->table_width);
    ATHENA_REQUIRE(d->dtype == ATHENA_F32 || d->dtype == ATHENA_BF16, ATHENA_E_UNSUPPORTED, "athena_kv8_attention: dtype");
    if (N == 0) return ATHENA_OK;
    ATHENA_REQUIRE(d->q && d->k_codes && d->v_codes && d->k_scale && d->v_scale && d->tables && d->lens && d->out, ATHENA_E_SHAPE,
                   "athena_kv8_attention: null operand");
    // (the rows of the last tile stay below 2^31)
    ATHENA_REQUIRE((long)N * (h / hk) < (1L << 31) - 512, ATHENA_E_SHAPE, "athena_kv8_attention: %d rows of %d heads are too many", N, h);
    ATHENA_REQUIRE(d->cu_rows || N == B, ATHENA_E_SHAPE, "athena_kv8_attention: %d rows for %d sequences need cu_rows", N, B);
    ATHENA_REQUIRE(athena_aligned16(d->k_codes) && athena_aligned16(d->v_codes), ATHENA_E_ALIGN,
                   "athena_kv8_attention: codes must lie on 16 bytes");
    const KvShape sh = kv8_shape(d);
    // (a launch has fewer than 2^32 threads)
    const long pairs = ((long)B * hk + 7) / 8 * 8;
    ATHENA_REQUIRE(pairs * sh.row_tiles * sh.splits < (1L << 24) && pairs * sh.row_tiles_many * sh.splits < (1L << 26) / (sh.waves ? sh.waves : 4),
                   ATHENA_E_SHAPE, "athena_kv8_attention: too many workgroups");
    const int64_t need = athena_kv8_attention_workspace_bytes(d);
    ATHENA_REQUIRE(need == 0 || (d->workspace && d->workspace_bytes >= need), ATHENA_E_SHAPE,
                   "athena_kv8_attention: workspace of %ld bytes, %ld needed", (long)d->workspace_bytes, (long)need);
    float* part = (float*)d->workspace;
    // whole 16-byte (queries) / four-element (results) accesses where rows, heads and columns allow them
    const int q_wide = athena_aligned16(d->q) && d->ldq * e % 16 == 0 && d->ldq_head * e % 16 == 0 && d->dk % 8 == 0;
    const int out_wide = (uintptr_t)d->out % (4 * e) == 0 && d->ldo % 4 == 0 && d->ldo_head % 4 == 0;
    KvAttn a = {d->q, d->ldq, d->ldq_head, d->k_codes, d->v_codes, d->k_scale, d->v_scale, d->tables, d->ld_tables, d->lens, d->cu_rows,
                d->out, d->ldo, d->ldo_head, d->lse, part, part + (sh.splits > 1 ? (long)sh.splits * N * h * d->dk : 0), d->table_width,
                d->num_blocks, B, N, h, hk, d->dk, d->block_size, __builtin_ctz(d->block_size), d->causal, sh.splits, sh.row_tiles, sh.waves ? (h / hk > KV_FEW ? h / hk : KV_FEW) : 0x7fffffff,
                ((long)B * hk + 7) / 8 * d->table_width * d->block_size * 2 * d->width <= (4L << 20), q_wide, out_wide, d->scale};
    hipStream_t s = (hipStream_t)stream;
#define KV_LAUNCH(T)                                      \
    do {                                                  \
        if (d->width == 32) kv8_launch<T, 32>(a, sh, s);  \
        else if (d->width == 64) kv8_launch<T, 64>(a, sh, s); \
        else kv8_launch<T, 128>(a, sh, s);                \
    } while (0)
    if (d->dtype == ATHENA_BF16) KV_LAUNCH(bf16_t);
    else KV_LAUNCH(float);
#undef KV_LAUNCH
    ATHENA_CHECK_LAUNCH("athena_kv8_attention");
    if (sh.splits > 1) {
        const int rows = d->cu_rows ? d->max_rows : 1;
        const dim3 grid(rows < 4096 ? rows : 4096, (h + 3) / 4, B);
        if (d->dtype == ATHENA_BF16) ATHENA_LAUNCH(kv8_join_kernel<bf16_t>, grid, dim3(256), 0, s, a);
        else ATHENA_LAUNCH(kv8_join_kernel<float>, grid, dim3(256), 0, s, a);
        ATHENA_CHECK_LAUNCH("athena_kv8_attention (join)");
    }
    return ATHENA_OK;
}
