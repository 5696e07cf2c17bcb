/*
 * uocr_sample.hip - sampling a token of each row of logits on gfx950.
 */
#include "uocr_serve.h"

#include <math.h>

typedef uint32_t u32;
typedef unsigned long long u64;

namespace {

constexpr u32 NT = 1024, WAVES = NT / 64; /* a block has one row */
constexpr u32 E = 8, STEP = 64 * E;       /* values of a lane and of a wavefront per step */
constexpr u32 BINS = 2048;                /* two a thread */
constexpr u32 LIST = 1024;                /* values that are ordered by comparing all pairs */
constexpr u32 GROUPS = 64;                /* partial sums of a wavefront's run in the last pass */
constexpr u32 IDX_BITS = 24;

/* Weights are integers in units of 2^-shift, shift = 62 - log2(vocab) rounded
 * up: their sums neither overflow nor depend on the order of addition (the
 * atomics below are integer ones).  A unit is 2^-45 for 129,280 tokens: sums of
 * that many are off by 2^-29 of the largest weight at most, by 2^-37 as a rule. */
struct Row {
    double c;      /* log2(e) / temperature */
    double unit;   /* 2^shift */
    float top;     /* the largest logit */
    float scale;   /* bins per logit */
    double min_w;
};

/* Order-preserving key of a logit; NaN as -inf, -0 as 0. */
__device__ __forceinline__ u32 key_of(float x) {
    x = x != x ? -INFINITY : x == 0.0f ? 0.0f : x;
    const u32 b = __float_as_uint(x);
    return (b >> 31) != 0u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(u32 k) {
    return __uint_as_float((k >> 31) != 0u ? k & 0x7fffffffu : ~k);
}

/* Larger logits first, equal ones by lowest id: all different. */
__device__ __forceinline__ u64 rank_of(float x, u32 id) {
    return ((u64)key_of(x) << IDX_BITS) | ((1u << IDX_BITS) - 1u - id);
}

__device__ __forceinline__ double weight(const Row &r, float x) {
    if (x == r.top) return 1.0;
    const double d = (double)x - (double)r.top;
    return d > -INFINITY ? exp2(d * r.c) : 0.0; /* NaN is not above -inf either */
}
__device__ __forceinline__ u64 units(const Row &r, double w) {
    return (u64)(w * r.unit + 0.5);
}

/* Bins of equal width below the largest logit, over the range where a weight
 * has a unit; the last one holds what has none. */
__device__ __forceinline__ u32 bin_of(const Row &r, float x) {
    return x == r.top ? 0u : (u32)fminf((r.top - x) * r.scale, (float)(BINS - 1u)); /* NaN: the last */
}

/* f(logit, id) for the E values of the lane at id0, those inside the row. */
template <bool F32, typename F>
__device__ __forceinline__ void lane_values(const void *row, u32 id0, u32 vocab, F &&f) {
    float x[E];
    if (id0 + E <= vocab) {
        if constexpr (F32) {
            const f32x4_any4 a = *(const f32x4_any4 *)((const float *)row + id0), b = *(const f32x4_any4 *)((const float *)row + id0 + 4);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
            union {
                uint4 u;
                _Float16 h[8];
            } v;
            v.u = load_any((const uint16_t *)row + id0);
#pragma unroll
            for (u32 e = 0; e < E; ++e) x[e] = (float)v.h[e];
        }
#pragma unroll
        for (u32 e = 0; e < E; ++e) f(x[e], id0 + e);
    } else {
        for (u32 id = id0; id < vocab; ++id) f(F32 ? ((const float *)row)[id] : (float)((const _Float16 *)row)[id], id);
    }
}

/* f over the whole row, by all threads. */
template <bool F32, typename F>
__device__ __forceinline__ void row_values(const void *row, u32 vocab, F &&f) {
    for (u32 id0 = threadIdx.x * E; id0 < vocab; id0 += NT * E) lane_values<F32>(row, id0, vocab, f);
}

__device__ __forceinline__ u64 shfl64(u64 v, int src) {
    return ((u64)(u32)__shfl((int)(v >> 32), src) << 32) | (u32)__shfl((int)v, src);
}
__device__ __forceinline__ u64 shfl_xor64(u64 v, int m) {
    return ((u64)(u32)__shfl_xor((int)(v >> 32), m) << 32) | (u32)__shfl_xor((int)v, m);
}

/* Sums of what earlier lanes hold. */
__device__ __forceinline__ u64 wave_before(u64 v) {
    u64 s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = shfl64(s, (int)(threadIdx.x & 63u) - d);
        if ((int)(threadIdx.x & 63u) >= d) s += o;
    }
    return s - v;
}

struct Shared {
    u64 weight[BINS];
    u32 count[BINS];
    u64 list[LIST];
    u64 list_w[LIST];
    u64 red[WAVES];
    u64 red2[WAVES];
    u64 out[4];
    u32 n;
};

/* Sums of what earlier threads hold, and all of it. */
__device__ __forceinline__ u64 block_before(u64 v, u64 *red, u64 &all) {
    const u64 b = wave_before(v);
    if ((threadIdx.x & 63u) == 63u) red[threadIdx.x >> 6] = b + v;
    __syncthreads();
    u64 before = b;
    all = 0;
    for (u32 w = 0; w < WAVES; ++w) {
        if (w < (threadIdx.x >> 6)) before += red[w];
        all += red[w];
    }
    __syncthreads();
    return before;
}

/* What is known of the value that ends a kept set: it lies in bin `bin`, its
 * rank begins with `prefix` from bit `sh` on (64: nothing known), `n` values
 * are left to choose from, and `before` is what stands in front of them (a
 * count, or a sum of units). */
struct Region {
    u32 bin, n;
    u64 prefix;
    u32 sh;
    u64 before;
};

/* The rank of the last value that is kept: of the values in the region, largest
 * first, those in front of which there is less than `limit` (values, or units
 * of weight where WEIGHTED) and whose rank is at least `floor`.  Crowded
 * regions are divided by the next bits of the rank first.  kept_w: the kept
 * values' units. */
template <bool F32, bool WEIGHTED>
__device__ u64 last_kept(const void *row, u32 vocab, const Row &r, Region g, double limit, u64 floor, Shared &sm, u64 &kept_w) {
    const u32 t = threadIdx.x;
    auto inside = [&](float x, u64 rank) {
        return bin_of(r, x) == g.bin && rank >= floor && (g.sh == 64u || (rank >> g.sh) == g.prefix);
    };
    kept_w = 0;
    while (g.n > LIST) {
        const u32 sh = g.sh == 64u ? 45u : g.sh > 11u ? g.sh - 11u : 0u;
        for (u32 i = t; i < BINS; i += NT) sm.weight[i] = 0ull, sm.count[i] = 0u;
        __syncthreads();
        row_values<F32>(row, vocab, [&](float x, u32 id) {
            const u64 rank = rank_of(x, id);
            if (!inside(x, rank)) return;
            const u32 i = BINS - 1u - ((u32)(rank >> sh) & (BINS - 1u));
            atomicAdd(&sm.count[i], 1u);
            atomicAdd(&sm.weight[i], units(r, weight(r, x)));
        });
        __syncthreads();
        const u64 n0 = sm.count[2 * t], n1 = sm.count[2 * t + 1], w0 = sm.weight[2 * t], w1 = sm.weight[2 * t + 1];
        u64 all;
        const u64 nb = block_before(n0 + n1, sm.red, all), wb = block_before(w0 + w1, sm.red2, all);
        for (u32 k = 0; k < 2u; ++k) {
            const u64 n = k ? n1 : n0, bw = wb + (k ? w0 : 0ull), bn = nb + (k ? n0 : 0ull);
            const u64 b = g.before + (WEIGHTED ? bw : bn), e = b + (WEIGHTED ? (k ? w1 : w0) : n);
            /* the last one with a value that is kept */
            if (n != 0ull && (double)b < limit && !((double)e < limit)) sm.out[0] = 2u * t + k, sm.out[1] = b, sm.out[2] = n, sm.out[3] = bw;
        }
        __syncthreads();
        const u32 digit = BINS - 1u - (u32)sm.out[0];
        /* the bits above this digit are the known ones, or none where this is the first */
        g.prefix = g.sh == 64u ? digit : (g.prefix << (g.sh - sh)) | (digit & ((1u << (g.sh - sh)) - 1u));
        g.sh = sh;
        g.before = sm.out[1];
        g.n = (u32)sm.out[2];
        kept_w += sm.out[3];
        __syncthreads();
    }
    if (t == 0u) sm.n = 0u;
    __syncthreads();
    row_values<F32>(row, vocab, [&](float x, u32 id) {
        const u64 rank = rank_of(x, id);
        if (!inside(x, rank)) return;
        const u32 at = atomicAdd(&sm.n, 1u);
        sm.list[at] = rank;
        sm.list_w[at] = units(r, weight(r, x));
    });
    __syncthreads();
    const u32 n = sm.n;
    u64 mine = ~0ull, w = 0;
    if (t < n) {
        const u64 rank = sm.list[t];
        u64 before = g.before;
        for (u32 i = 0; i < n; ++i)
            if (sm.list[i] > rank) before += WEIGHTED ? sm.list_w[i] : 1ull;
        if ((double)before < limit) mine = rank, w = sm.list_w[t];
    }
    u64 sum;
    (void)block_before(w, sm.red, sum);
    kept_w += sum;
    for (int o = 32; o > 0; o >>= 1) {
        const u64 v = shfl_xor64(mine, o);
        mine = v < mine ? v : mine;
    }
    if ((t & 63u) == 0u) sm.red[t >> 6] = mine;
    __syncthreads();
    for (u32 i = 0; i < WAVES; ++i) mine = sm.red[i] < mine ? sm.red[i] : mine;
    __syncthreads();
    return mine;
}

/* A row in one block.  The kept set of top-k and top-p is all values from some
 * rank on: a histogram over bins below the maximum (counts, and units of weight
 * for top-p) finds the bin of the last kept value, the bin's few values are
 * then ordered by comparing them.  Bound by the block's vector units: a pass
 * over a row costs them more than its reading from the L2. */
template <bool F32>
__global__ __launch_bounds__(NT) void k_sample(uocr_sample_args a, u32 shift) {
    __shared__ Shared sm;
    const u32 t = threadIdx.x, lane = t & 63u, wave = t >> 6, b = blockIdx.x, vocab = a.vocab;
    const void *row = (const uint8_t *)a.logits + (uint64_t)b * a.stride * (F32 ? 4u : 2u);

    float best = -INFINITY;
    u32 best_id = 0xffffffffu;
    row_values<F32>(row, vocab, [&](float x, u32 id) {
        if (x > best) best = x, best_id = id;
    });
    u64 rank = best_id == 0xffffffffu ? 0ull : rank_of(best, best_id);
    for (int o = 32; o > 0; o >>= 1) {
        const u64 v = shfl_xor64(rank, o);
        rank = v > rank ? v : rank;
    }
    if (lane == 0u) sm.red[wave] = rank;
    __syncthreads();
    for (u32 i = 0; i < WAVES; ++i) rank = sm.red[i] > rank ? sm.red[i] : rank;
    __syncthreads();
    const u64 max_rank = rank;
    const float temp = a.temperature != nullptr ? a.temperature[b] : 1.0f;
    if (max_rank == 0ull || !(temp > 0.0f)) {
        if (t == 0u) {
            a.tokens[b] = max_rank == 0ull ? 0 : (int32_t)((1u << IDX_BITS) - 1u - (u32)(max_rank & ((1u << IDX_BITS) - 1u)));
            if (a.probs != nullptr) a.probs[b] = max_rank == 0ull ? 0.0f : 1.0f;
        }
        return;
    }
    Row r;
    r.top = of_key((u32)(max_rank >> IDX_BITS));
    r.c = 1.4426950408889634 / (double)temp;
    r.unit = (double)(1ull << shift);
    r.scale = (float)((double)(BINS - 1u) * r.c / (double)(shift + 1u));
    r.min_w = a.min_p != nullptr && a.min_p[b] > 0.0f ? fmin((double)a.min_p[b], 1.0) : 0.0;
    const u32 k = a.top_k != nullptr && a.top_k[b] > 0 ? (u32)a.top_k[b] : 0u;
    const float p = a.top_p != nullptr ? a.top_p[b] : 1.0f;
    const bool use_k = k != 0u && k < vocab, use_p = p < 1.0f;

    u64 thr = 0; /* kept: ranks from here on */
    if (use_k || use_p) {
        for (u32 i = t; i < BINS; i += NT) sm.weight[i] = 0ull, sm.count[i] = 0u;
        __syncthreads();
        row_values<F32>(row, vocab, [&](float x, u32 id) {
            const u32 i = bin_of(r, x);
            if (i == BINS - 1u) return; /* no weight */
            atomicAdd(&sm.count[i], 1u);
            if (use_p) atomicAdd(&sm.weight[i], units(r, weight(r, x)));
        });
        __syncthreads();
        const u32 n0 = sm.count[2 * t], n1 = sm.count[2 * t + 1];
        const u64 w0 = sm.weight[2 * t], w1 = sm.weight[2 * t + 1];
        u64 all_n, all_w;
        const u64 nb = block_before(n0 + n1, sm.red, all_n), wb = block_before(w0 + w1, sm.red2, all_w);
        u64 w_in = 0;
        if (use_k && (u64)k < all_n) {
            for (u32 i = 0; i < 2u; ++i) {
                const u64 c0 = nb + (i ? n0 : 0u), c1 = c0 + (i ? n1 : n0);
                if (c0 < k && k <= c1) sm.out[0] = 2u * t + i, sm.out[1] = c0, sm.out[2] = c1 - c0, sm.out[3] = wb + (i ? w0 : 0ull);
            }
            __syncthreads();
            const Region g = {(u32)sm.out[0], (u32)sm.out[2], 0ull, 64u, sm.out[1]};
            const u64 above = sm.out[3];
            __syncthreads();
            thr = last_kept<F32, false>(row, vocab, r, g, (double)k, 0ull, sm, w_in);
            all_w = above + w_in;
        }
        if (use_p && !(p > 0.0f)) {
            thr = max_rank;
        } else if (use_p) {
            const double target = (double)p * (double)all_w;
            for (u32 i = 0; i < 2u; ++i) {
                const u64 c0 = wb + (i ? w0 : 0ull), c1 = c0 + (i ? w1 : w0);
                if ((i ? n1 : n0) != 0u && (double)c0 < target && !((double)c1 < target)) sm.out[0] = 2u * t + i, sm.out[1] = c0, sm.out[2] = i ? n1 : n0;
            }
            __syncthreads();
            const Region g = {(u32)sm.out[0], (u32)sm.out[2], 0ull, 64u, sm.out[1]};
            __syncthreads();
            thr = last_kept<F32, true>(row, vocab, r, g, target, thr, sm, w_in);
        }
    }

    /* the kept weights by id: a run of the row for each wavefront, a sum for each group of its steps */
    const u32 steps = (vocab + STEP - 1u) / STEP, run = (steps + WAVES - 1u) / WAVES, per = (run + GROUPS - 1u) / GROUPS;
    auto kept = [&](float x, u32 id) {
        if (rank_of(x, id) < thr || bin_of(r, x) == BINS - 1u) return 0ull;
        const double w = weight(r, x);
        return w >= r.min_w ? units(r, w) : 0ull;
    };
    u64 *sums = sm.weight; /* [WAVES][GROUPS] */
    sums[t] = 0ull;
    __syncthreads();
    for (u32 g = 0; g * per < run; ++g) {
        u64 s = 0;
        for (u32 i = g * per; i < min(g * per + per, run); ++i)
            lane_values<F32>(row, min((wave * run + i) * STEP + lane * E, vocab), vocab, [&](float x, u32 id) { s += kept(x, id); });
        for (int o = 32; o > 0; o >>= 1) s += shfl_xor64(s, o);
        if (lane == 0u) sums[wave * GROUPS + g] = s;
    }
    __syncthreads();
    const u64 mine = sums[t];
    u64 all;
    const u64 before = block_before(mine, sm.red, all);
    const float u = a.uniform[b];
    const double target = (double)(u > 0.0f ? fminf(u, 0.99999994f) : 0.0f) * (double)all;
    /* the group that holds the first id whose running sum is over the target */
    if (mine != 0ull && !((double)before > target) && (double)(before + mine) > target) sm.out[0] = t, sm.out[1] = before;
    __syncthreads();
    if (wave == 0u) {
        const u32 w = (u32)sm.out[0] / GROUPS, g = (u32)sm.out[0] % GROUPS;
        u64 sum = sm.out[1];
        for (u32 i = g * per; i < min(g * per + per, run); ++i) {
            const u32 id0 = min((w * run + i) * STEP + lane * E, vocab);
            u64 s = 0;
            lane_values<F32>(row, id0, vocab, [&](float x, u32 id) { s += kept(x, id); });
            u64 at = sum + wave_before(s);
            const u64 found = __ballot(s != 0ull && !((double)at > target) && (double)(at + s) > target);
            if (found != 0ull) {
                if (lane == (u32)__ffsll((long long)found) - 1u) {
                    bool done = false;
                    lane_values<F32>(row, id0, vocab, [&](float x, u32 id) {
                        const u64 v = kept(x, id);
                        at += v;
                        if (!done && v != 0ull && (double)at > target) {
                            done = true;
                            a.tokens[b] = (int32_t)id;
                            if (a.probs != nullptr) a.probs[b] = (float)((double)v / (double)all);
                        }
                    });
                }
                break;
            }
            sum = shfl64(at + s, 63);
        }
    }
}

}  // namespace

size_t uocr_sample_ws_bytes(uint32_t rows, uint32_t vocab) {
    (void)rows;
    (void)vocab;
    return 16u;
}

hipError_t uocr_launch_sample(hipStream_t st, const uocr_sample_args *a) {
    u32 bits = 0;
    while ((1u << bits) < a->vocab) ++bits;
    const u32 shift = 62u - bits < 52u ? 62u - bits : 52u;
    if (a->f32) hipLaunchKernelGGL((k_sample<true>), dim3(a->rows), dim3(NT), 0, st, *a, shift);
    else hipLaunchKernelGGL((k_sample<false>), dim3(a->rows), dim3(NT), 0, st, *a, shift);
    return hipGetLastError();
}
