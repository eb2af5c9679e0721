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
    ATHENA_REQUIRE((long)d->table_width * bs < (1L << 31), ATHENA_E_SHAPE, "athena_kv_plan: table too wide");
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
// scale, and the run's codes are written.  One wave per (run, kv head, keys or values); the wave that finds a
// run's first row takes all of it, so waves of one block never meet.
//
// Codes are round-half-to-even(x / scale) exactly: the product with the reciprocal in fp32 is off by less
// than 127 * 2^-23, so a quotient within 1e-4 of a border is divided again in 64 bits, where quotients of
// fp32 operands of this size cannot come closer than 2^-34 to a border without lying on it.
//
// A lane holds two columns of 16 consecutive places, so that the values' codes (16 bytes of one column) leave
// in one store.  Bound by the rows' way in and the codes' way out; a run of more places than the wave holds at
// once reads its rows twice, the second time from the caches.
template <typename T> struct AppendSide {
    const T* x;
    long ld_row, ld_head;
    int8_t* codes;
    float* scale;
};

__device__ __forceinline__ int code_of(float x, float s, float inv) {
    const float f = x * inv;
    float q = rintf(f);
    if (fabsf(fabsf(f - q) - 0.5f) < 1e-4f || s < 1e-30f) q = s > 0.f ? (float)rint((double)x / (double)s) : 0.f;
    return (int)fminf(fmaxf(q, -127.f), 127.f);
}
__device__ __forceinline__ int recode(int q, float s0, float s1, float ratio) {
    const float f = (float)q * ratio;
    float r = rintf(f);
    if (fabsf(fabsf(f - r) - 0.5f) < 1e-4f || s0 < 1e-30f) r = (float)rint((double)q * (double)s0 / (double)s1);
    return (int)r;
}
// the first ``keep`` of four codes in a word
__device__ __forceinline__ unsigned recode4(unsigned w, int keep, float s0, float s1, float ratio) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned q = (unsigned)recode((int8_t)(w >> (8 * i)), s0, s1, ratio) & 0xffu;
        if (i < keep) w = (w & ~(0xffu << (8 * i))) | (q << (8 * i));
    }
    return w;
}

template <typename T, int W>
__device__ __forceinline__ void append_run(const AppendSide<T>& a, bool values, const int32_t* __restrict__ slots, long slots_end,
                                           int t, int n, int first, bool straight, int block, int head, int hk, int dk,
                                           int block_size, bool pairs, int lane) {
    constexpr int LR = W / 2, SUB = 64 / LR;                // lanes of a row, groups of 16 places side by side
    const int sub = lane / LR, c = 2 * (lane % LR);
    const T* x = a.x + (long)t * a.ld_row + (long)head * a.ld_head;
    const long at = (long)block * hk + head;
    int8_t* codes = a.codes + at * W * block_size;
    const int step = 16 * SUB, begin = first & ~15, end = first + n;
    float v[16][2];
    struct alignas(2 * sizeof(T)) Pair { T e[2]; };
    // the two columns of places base + 16 sub ...: all sixteen requests go out before the first is waited for, so rows and
    // columns that are not there are read from ones that are, and dropped afterwards
    auto load = [&](int base) {
        const int p0 = base + 16 * sub;
        const int c0 = c < dk ? c : 0, c1 = c + 1 < dk ? c + 1 : 0;
        Pair raw[16];
        if (pairs && (dk & 1) == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) raw[i] = *(const Pair*)(x + (long)min(max(p0 + i - first, 0), n - 1) * a.ld_row + c0);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const T* p = x + (long)min(max(p0 + i - first, 0), n - 1) * a.ld_row;
                raw[i].e[0] = p[c0];
                raw[i].e[1] = p[c1];
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const bool in = p0 + i >= first && p0 + i < end;
            v[i][0] = in && c < dk ? to_f32<T>(raw[i].e[0]) : 0.f;
            v[i][1] = in && c + 1 < dk ? to_f32<T>(raw[i].e[1]) : 0.f;
        }
    };
    unsigned top = 0;                                       // largest magnitude, as bits: NaN over infinity over numbers
    const auto mag = [](float f) { return __float_as_uint(f) & 0x7fffffffu; };
    if (straight) {
        for (int base = begin; base < end; base += step) {
            load(base);
#pragma unroll
            for (int i = 0; i < 16; ++i) top = max(top, max(mag(v[i][0]), mag(v[i][1])));
        }
    } else {
        for (int e = lane; e < n * dk; e += 64) {
            const int r = e / dk, s = slots[t + r];
            if (s >= 0 && s < slots_end) top = max(top, mag(to_f32<T>(x[(long)r * a.ld_row + (e - r * dk)])));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    const float s0 = first == 0 ? 0.f : a.scale[at];
    // (as whole numbers, so that a scale that is not finite stays; it is kept as NaN)
    const unsigned bits = max(mag(s0), mag(__uint_as_float(top) / 127.f));
    const float s1 = __uint_as_float(bits < 0x7f800000u ? bits : 0x7fc00000u);
    if (s1 > s0 && first > 0) {
        const float ratio = s0 / s1;
        const int words = values ? (first + 15) / 16 : first * W / 16, columns = values ? W : 1;
        for (int e = lane; e < words * columns; e += 64) {
            const int col = e / words, k = e - col * words;
            uint4* p = (uint4*)(codes + (values ? col * block_size : 0) + 16 * k);
            const int keep = values ? first - 16 * k : 16;
            uint4 w = *p;
            w.x = recode4(w.x, keep, s0, s1, ratio);
            w.y = recode4(w.y, keep - 4, s0, s1, ratio);
            w.z = recode4(w.z, keep - 8, s0, s1, ratio);
            w.w = recode4(w.w, keep - 12, s0, s1, ratio);
            *p = w;
        }
    }
    const float inv = s1 > 0.f ? 1.f / s1 : 0.f;
    if (straight) {
        for (int base = begin; base < end; base += step) {
            if (end - begin > step) load(base);             // (otherwise the registers hold the rows still)
            const int p0 = base + 16 * sub;
            if (values) {
                if (p0 >= first && p0 + 16 <= end) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        unsigned w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            w[i] = 0;
#pragma unroll
                            for (int r = 0; r < 4; ++r) w[i] |= ((unsigned)code_of(v[4 * i + r][k], s1, inv) & 0xffu) << (8 * r);
                        }
                        *(uint4*)(codes + (c + k) * block_size + p0) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (p0 + i >= first && p0 + i < end) {
                            codes[c * block_size + p0 + i] = (int8_t)code_of(v[i][0], s1, inv);
                            codes[(c + 1) * block_size + p0 + i] = (int8_t)code_of(v[i][1], s1, inv);
                        }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (p0 + i >= first && p0 + i < end) {
                        const unsigned two = ((unsigned)code_of(v[i][0], s1, inv) & 0xffu) | ((unsigned)code_of(v[i][1], s1, inv) & 0xffu) << 8;
                        *(uint16_t*)(codes + (p0 + i) * W + c) = (uint16_t)two;
                    }
            }
        }
    } else {
        for (int r = 0; r < n; ++r) {                       // in the rows' order: of two rows for one place the later stays
            const int s = slots[t + r];
            if (s < 0 || s >= slots_end) continue;
            for (int col = lane; col < W; col += 64) {
                const float f = col < dk ? to_f32<T>(x[(long)r * a.ld_row + col]) : 0.f;
                codes[values ? col * block_size + s % block_size : (s % block_size) * W + col] = (int8_t)code_of(f, s1, inv);
            }
        }
    }
    if (lane == 0) a.scale[at] = s1;
}

template <typename T, int W>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendSide<T> ks, AppendSide<T> vs, const int32_t* __restrict__ slots,
                                                         int N, int rows_per_wg, int hk, int dk, int block_size, int k_pairs,
                                                         int v_pairs, long slots_end) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6, head = blockIdx.y;
    const int t0 = blockIdx.x * rows_per_wg;
    const auto good = [&](int s) { return s >= 0 && s < slots_end; };
    // first rows of runs among the workgroup's rows; skipped rows do not end a run
    bool leads = false;
    if (lane < rows_per_wg && t0 + lane < N) {
        const int s = slots[t0 + lane];
        if (good(s)) {
            int p = t0 + lane - 1;
            while (p >= 0 && !good(slots[p])) --p;
            leads = p < 0 || slots[p] / block_size != s / block_size;
        }
    }
    unsigned long long found = __ballot(leads);
    for (int job = 0; found; job += 2) {
        const int t = t0 + __ffsll((long long)found) - 1;
        found &= found - 1;
        // both sides of a run go to neighbouring waves
        for (int side = 0; side < 2; ++side) {
            if ((job + side) % nw != w) continue;
            const int s0 = slots[t], block = s0 / block_size;
            int n = 0, first = block_size;                  // rows up to the run's last one, first place
            bool straight = true, more = true;              // straight: no row skipped, places in order
            for (int r0 = 0; more; r0 += 64) {
                const int r = r0 + lane, s = t + r < N ? slots[t + r] : -1;
                const unsigned long long mine = __ballot(good(s) && s / block_size == block),
                                         other = __ballot(t + r >= N || (good(s) && s / block_size != block));
                const unsigned long long in = other ? mine & ((other & -other) - 1) : mine;
                more = !other;
                if (in) {
                    const int last = 63 - __clzll((long long)in);
                    straight = straight && n == r0 && __ballot(lane <= last && s != s0 + r) == 0;
                    n = r0 + last + 1;
                    int p = (in >> lane) & 1 ? s % block_size : block_size;
#pragma unroll
                    for (int o = 32; o > 0; o >>= 1) p = min(p, __shfl_xor(p, o, 64));
                    first = min(first, p);
                }
            }
            if (side) append_run<T, W>(vs, true, slots, slots_end, t, n, first, straight, block, head, hk, dk, block_size, v_pairs, lane);
            else append_run<T, W>(ks, false, slots, slots_end, t, n, first, straight, block, head, hk, dk, block_size, k_pairs, lane);
        }
    }
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
    ATHENA_REQUIRE(N >= 0, ATHENA_E_SHAPE, "athena_kv8_append: N=%d", N);
    ATHENA_REQUIRE(d->dtype == ATHENA_F32 || d->dtype == ATHENA_BF16, ATHENA_E_UNSUPPORTED, "athena_kv8_append: dtype");
    if (N == 0) return ATHENA_OK;
    const void *k = d->k, *v = d->v;
    const long ldk = d->ldk, ldk_head = d->ldk_head, ldv = d->ldv, ldv_head = d->ldv_head;
    const int32_t* slots = d->slots;
    int8_t *k_codes = d->k_codes, *v_codes = d->v_codes;
    float *k_scale = d->k_scale, *v_scale = d->v_scale;
    ATHENA_REQUIRE(k && v && slots && k_codes && v_codes && k_scale && v_scale, ATHENA_E_SHAPE, "athena_kv8_append: null operand");
    ATHENA_REQUIRE(athena_aligned16(k_codes) && athena_aligned16(v_codes), ATHENA_E_ALIGN, "athena_kv8_append: codes must lie on 16 bytes");
    const int per = (long)N * hk <= 4096 ? 1 : 16;
    const dim3 grid((N + per - 1) / per, hk), block(per == 1 ? 128 : 256);
    const long end = (long)num_blocks * block_size;
    const size_t two = d->dtype == ATHENA_BF16 ? 4 : 8;        // two elements in one load where rows and heads begin on them
    const int kp = (uintptr_t)k % two == 0 && ldk % 2 == 0 && ldk_head % 2 == 0;
    const int vp = (uintptr_t)v % two == 0 && ldv % 2 == 0 && ldv_head % 2 == 0;
#define KV_APPEND(T, W)                                                                                                     \
    do {                                                                                                                    \
        AppendSide<T> ks = {(const T*)k, ldk, ldk_head, k_codes, k_scale}, vs = {(const T*)v, ldv, ldv_head, v_codes, v_scale}; \
        ATHENA_LAUNCH((kv8_append_kernel<T, W>), grid, block, 0, (hipStream_t)stream, ks, vs, slots, N, per, hk, dk, block_size, \
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
    int rt, row_tiles, splits;
};

// Query rows per wave and how far the key axis is split.  A split costs a second launch (the join, about 2 us), so
// none has fewer than KV_MIN_TILES tiles, and there are as many as fill the chip about three times over.
static KvShape kv8_shape(const athena_kv8_attention_desc* d) {
    KvShape s;
    const long rows = (long)(d->cu_rows ? d->max_rows : 1) * (d->h / d->hk);
    const int most = d->dtype == ATHENA_F32 ? (d->width == 128 ? 1 : 2) : d->width == 128 ? 2 : 4;     // what fits the registers
    s.rt = rows <= 16 || most == 1 ? 1 : rows <= 32 || most == 2 ? 2 : 4;
    const long tiles = (rows + 16 * s.rt - 1) / (16 * s.rt);
    s.row_tiles = (int)(tiles < 65536 ? tiles : 65536);
    const long units = (long)d->B * d->hk * s.row_tiles, key_tiles = ((long)d->table_width * d->block_size + KV_KEYS - 1) / KV_KEYS;
    long splits = (1536 + units - 1) / units;
    const long cap = key_tiles / KV_MIN_TILES;
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
static void kv8_launch(const KvAttn& a, const KvShape& sh, hipStream_t s) {
    const long units = ((long)a.B * a.hk + 7) / 8 * 8 * sh.row_tiles * sh.splits;
    const dim3 grid((unsigned)units), block(256);
    if (sh.rt == 4) {
        if constexpr (W < 128 && sizeof(T) == 2) ATHENA_LAUNCH((kv8_attention_kernel<T, W, 4>), grid, block, 0, s, a);
    } else if (sh.rt == 2) {
        if constexpr (W < 128 || sizeof(T) == 2) ATHENA_LAUNCH((kv8_attention_kernel<T, W, 2>), grid, block, 0, s, a);
    } else ATHENA_LAUNCH((kv8_attention_kernel<T, W, 1>), grid, block, 0, s, a);
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
    ATHENA_REQUIRE(d->cu_rows || N == B, ATHENA_E_SHAPE, "athena_kv8_attention: %d rows for %d sequences need cu_rows", N, B);
    ATHENA_REQUIRE(athena_aligned16(d->k_codes) && athena_aligned16(d->v_codes), ATHENA_E_ALIGN,
                   "athena_kv8_attention: codes must lie on 16 bytes");
    const KvShape sh = kv8_shape(d);
    ATHENA_REQUIRE(((long)B * hk + 7) / 8 * 8 * sh.row_tiles * sh.splits < (1L << 31), ATHENA_E_SHAPE, "athena_kv8_attention: too many workgroups");
    const int64_t need = athena_kv8_attention_workspace_bytes(d);
    ATHENA_REQUIRE(need == 0 || (d->workspace && d->workspace_bytes >= need), ATHENA_E_SHAPE,
                   "athena_kv8_attention: workspace of %ld bytes, %ld needed", (long)d->workspace_bytes, (long)need);
    float* part = (float*)d->workspace;
    // whole 16-byte (queries) / four-element (results) accesses where rows, heads and columns allow them
    const int q_wide = athena_aligned16(d->q) && d->ldq * e % 16 == 0 && d->ldq_head * e % 16 == 0 && d->dk % 8 == 0;
    const int out_wide = (uintptr_t)d->out % (4 * e) == 0 && d->ldo % 4 == 0 && d->ldo_head % 4 == 0;
    KvAttn a = {d->q, d->ldq, d->ldq_head, d->k_codes, d->v_codes, d->k_scale, d->v_scale, d->tables, d->ld_tables, d->lens, d->cu_rows,
                d->out, d->ldo, d->ldo_head, d->lse, part, part + (sh.splits > 1 ? (long)sh.splits * N * h * d->dk : 0), d->table_width,
                d->num_blocks, B, N, h, hk, d->dk, d->block_size, d->causal, sh.splits, sh.row_tiles, q_wide, out_wide, d->scale};
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
