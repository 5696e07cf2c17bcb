/*
 * uocr_sample.hip - sampling a token of each row of logits on gfx950.
 */
#include "uocr_serve.h"

#include <math.h>

typedef uint32_t u32;
typedef unsigned long long u64;

namespace {

constexpr u32 NT = 1024, WAVES = NT / 64; /* a block that has a row of its own */
constexpr u32 CT = 512, CWAVES = CT / 64; /* a block that has a part of a row */
constexpr u32 E = 8, STEP = 64 * E;       /* values of a lane and of a wavefront per step */
constexpr u32 BINS = 2048;
constexpr u32 LIST = 1024;                /* values that are ordered by comparing all pairs */
constexpr u32 GROUPS = 64;                /* partial sums of a wavefront's run in the last pass */
constexpr u32 IDX_BITS = 24, IDX_MASK = (1u << IDX_BITS) - 1u;
constexpr u32 TAB = 1024;                 /* 2^(i / TAB) */
constexpr u32 MAX_CHUNKS = 64;

/* Weights are integers in units of 2^-shift, shift = 62 - log2(vocab) rounded
 * up (50 at most): their sums neither overflow nor depend on the order of
 * addition (the atomics below are integer ones).  A unit is 2^-45 for 129,280
 * tokens: a sum of that many is off by 2^-29 of the largest weight at most, by
 * 2^-37 as a rule. */
struct Row {
    double c;      /* TAB log2(e) / temperature */
    double min_w;  /* min_p in units */
    float top;     /* the largest logit */
    float scale;   /* bins per logit */
    float cut;     /* logits below are lighter than min_p */
    u32 shift, k;
    float p;
    bool inf, use_k, use_p;
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
    return ((u64)key_of(x) << IDX_BITS) | (IDX_MASK - id);
}

/* A weight in units, not yet rounded: 2^shift exp((x - top) / temperature), as
 * 2^(n / TAB) from the table, a third-degree sum for the rest of |r| <= 1/2
 * (off by 2^-50) and the exponent.  fp64: next to a limit the last bits decide
 * which token it is, and fp64 runs at the rate of fp32 here. */
__device__ __forceinline__ double weight(const Row &r, const double *tab, float x) {
    constexpr double L = 0.6931471805599453 / TAB;
    const double y = fmax(((double)x - (double)r.top) * r.c, -65536.0); /* NaN, too: no weight */
    const double big = y + 6755399441055744.0, f = y - (big - 6755399441055744.0);
    const int n = (int)(u32)__double_as_longlong(big);
    const double p = fma(fma(fma(L * L * L / 6.0, f, L * L / 2.0), f, L), f, 1.0);
    return ldexp(tab[(u32)n & (TAB - 1u)] * p, (n >> 10) + (int)r.shift);
}
__device__ __forceinline__ u64 units(double w) {
    return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
}
__device__ __forceinline__ void fill_table(double *tab) {
    for (u32 i = threadIdx.x; i < TAB; i += blockDim.x) tab[i] = exp2((double)i / TAB);
}

/* Bins of equal width below the largest logit, over the range where a weight
 * has a unit; the last one holds what has none. */
__device__ __forceinline__ u32 bin_of(const Row &r, float x) {
    return x == r.top ? 0u : (u32)fminf((r.top - x) * r.scale, (float)(BINS - 1u)); /* NaN: the last */
}

/* The settings of row b whose largest logit has rank max_rank.  With a +inf
 * one, logits are taken as 0 there and -inf elsewhere (value_of). */
__device__ __forceinline__ Row row_of(const uocr_sample_args &a, u32 b, u64 max_rank, float temp, u32 shift) {
    Row r;
    r.top = of_key((u32)(max_rank >> IDX_BITS));
    r.inf = r.top == INFINITY;
    if (r.inf) r.top = 0.0f;
    r.shift = shift;
    r.c = (double)TAB * 1.4426950408889634 / (double)temp;
    r.scale = (float)((double)(BINS - 1u) / TAB * r.c / (double)(shift + 1u));
    const float m = a.min_p != nullptr && a.min_p[b] > 0.0f ? fminf(a.min_p[b], 1.0f) : 0.0f;
    r.min_w = ldexp((double)m, (int)shift);
    /* below: lighter than min_p by more than the roundings here (2^-20 of the distance, and of the logit) */
    const float far = temp * logf(m); /* -inf without min_p */
    r.cut = r.top + far - 1e-6f * (fabsf(r.top) + fabsf(far));
    if (!(r.cut > -INFINITY)) r.cut = -INFINITY;
    r.k = a.top_k != nullptr && a.top_k[b] > 0 ? (u32)a.top_k[b] : 0u;
    r.p = a.top_p != nullptr ? a.top_p[b] : 1.0f;
    r.use_k = r.k != 0u && r.k < a.vocab;
    r.use_p = r.p < 1.0f;
    return r;
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

__device__ __forceinline__ float value_of(const Row &r, float x) {
    return !r.inf ? x : x == INFINITY ? 0.0f : -INFINITY;
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
__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += shfl_xor64(v, o);
    return v;
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
    double tab[TAB];
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
    for (u32 w = 0; w < blockDim.x / 64u; ++w) {
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
        row_values<F32>(row, vocab, [&](float raw, u32 id) {
            const float x = value_of(r, raw);
            const u64 rank = rank_of(x, id);
            if (!inside(x, rank)) return;
            const u32 i = BINS - 1u - ((u32)(rank >> sh) & (BINS - 1u));
            atomicAdd(&sm.count[i], 1u);
            atomicAdd(&sm.weight[i], units(weight(r, sm.tab, x)));
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
    row_values<F32>(row, vocab, [&](float raw, u32 id) {
        const float x = value_of(r, raw);
        const u64 rank = rank_of(x, id);
        if (!inside(x, rank)) return;
        const u32 at = atomicAdd(&sm.n, 1u);
        sm.list[at] = rank;
        sm.list_w[at] = units(weight(r, sm.tab, x));
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

/* The first id whose running sum of kept units is over the target, in the
 * STEP values from id0 in front of which `sum` stands; by one wavefront.
 * Returns whether it is there, and what stands in front of the next values. */
template <bool F32, typename K>
__device__ __forceinline__ bool pick(const uocr_sample_args &a, u32 b, const void *row, u32 id0, double target, u64 all, u64 &sum, K &&kept) {
    const u32 lane = threadIdx.x & 63u;
    id0 = min(id0 + lane * E, a.vocab);
    u64 s = 0;
    lane_values<F32>(row, id0, a.vocab, [&](float x, u32 id) { s += kept(x, id); });
    u64 at = sum + wave_before(s);
    const u64 found = __ballot(s != 0ull && !((double)at > target) && (double)(at + s) > target);
    sum = shfl64(at + s, 63);
    if (found == 0ull) return false;
    if (lane == (u32)__ffsll((long long)found) - 1u) {
        bool done = false;
        lane_values<F32>(row, id0, a.vocab, [&](float x, u32 id) {
            const u64 v = kept(x, id);
            at += v;
            if (!done && v != 0ull && (double)at > target) {
                done = true;
                a.tokens[b] = (int32_t)id;
                if (a.probs != nullptr) a.probs[b] = (float)((double)v / (double)all);
            }
        });
    }
    return true;
}

__device__ __forceinline__ double target_of(const uocr_sample_args &a, u32 b, u64 all) {
    const float u = a.uniform[b];
    return (double)(u > 0.0f ? fminf(u, 0.99999994f) : 0.0f) * (double)all;
}

/* Rows that are decided by their largest logit; true where this one is. */
__device__ __forceinline__ bool greedy(const uocr_sample_args &a, u32 b, u64 max_rank, float temp) {
    if (max_rank != 0ull && temp > 0.0f) return false;
    if (threadIdx.x == 0u) {
        a.tokens[b] = max_rank == 0ull ? 0 : (int32_t)(IDX_MASK - (u32)(max_rank & IDX_MASK));
        if (a.probs != nullptr) a.probs[b] = max_rank == 0ull ? 0.0f : 1.0f;
    }
    return true;
}

__device__ __forceinline__ float temperature_of(const uocr_sample_args &a, u32 b) {
    return a.temperature != nullptr ? a.temperature[b] : 1.0f;
}

/* The largest logit's rank, of the values that `each` goes over. */
template <typename G>
__device__ __forceinline__ u64 largest(u64 *red, G &&each) {
    float best = -INFINITY;
    u32 best_id = 0xffffffffu;
    each([&](float x, u32 id) {
        if (x > best) best = x, best_id = id;
    });
    u64 rank = best_id == 0xffffffffu ? 0ull : rank_of(best, best_id);
    for (int o = 32; o > 0; o >>= 1) {
        const u64 v = shfl_xor64(rank, o);
        rank = v > rank ? v : rank;
    }
    if ((threadIdx.x & 63u) == 0u) red[threadIdx.x >> 6] = rank;
    __syncthreads();
    for (u32 i = 0; i < blockDim.x / 64u; ++i) rank = red[i] > rank ? red[i] : rank;
    __syncthreads();
    return rank;
}

/* Units that a value brings to the kept sum: ranks from thr on, not below min_p. */
__device__ __forceinline__ u64 kept_units(const Row &r, const double *tab, float least, u64 thr, float x, u32 id) {
    if (!(x >= least) || (x == least && rank_of(x, id) < thr)) return 0ull;
    const double w = weight(r, tab, x);
    return w >= r.min_w ? units(w) : 0ull;
}
/* The logit below which nothing is kept. */
__device__ __forceinline__ float least_of(const Row &r, u64 thr) {
    return thr == 0ull ? r.cut : fmaxf(r.cut, of_key((u32)(thr >> IDX_BITS)));
}

/* A row in one block (max_rank: 0 where it is not known yet).  The kept set of
 * top-k and top-p is all values from some rank on: a histogram over bins below
 * the maximum (counts, and units of weight for top-p) finds the bin of the last
 * kept value, the bin's few values are then ordered by comparing them. */
template <bool F32>
__device__ void whole_row(const uocr_sample_args &a, u32 b, const void *row, u32 shift, Shared &sm) {
    const u32 t = threadIdx.x, lane = t & 63u, wave = t >> 6, vocab = a.vocab;
    const u64 max_rank = largest(sm.red, [&](auto f) { row_values<F32>(row, vocab, f); });
    const float temp = temperature_of(a, b);
    if (greedy(a, b, max_rank, temp)) return;
    const Row r = row_of(a, b, max_rank, temp, shift);
    fill_table(sm.tab);

    u64 thr = 0; /* kept: ranks from here on */
    if (r.use_k || r.use_p) {
        for (u32 i = t; i < BINS; i += NT) sm.weight[i] = 0ull, sm.count[i] = 0u;
        __syncthreads();
        row_values<F32>(row, vocab, [&](float raw, u32 id) {
            const float x = value_of(r, raw);
            const u32 i = bin_of(r, x);
            if (i == BINS - 1u) return; /* no weight */
            atomicAdd(&sm.count[i], 1u);
            if (r.use_p) atomicAdd(&sm.weight[i], units(weight(r, sm.tab, x)));
        });
        __syncthreads();
        const u32 n0 = sm.count[2 * t], n1 = sm.count[2 * t + 1];
        const u64 w0 = sm.weight[2 * t], w1 = sm.weight[2 * t + 1];
        u64 all_n, all_w;
        const u64 nb = block_before(n0 + n1, sm.red, all_n), wb = block_before(w0 + w1, sm.red2, all_w);
        u64 w_in = 0;
        if (r.use_k && (u64)r.k < all_n) {
            for (u32 i = 0; i < 2u; ++i) {
                const u64 c0 = nb + (i ? n0 : 0u), c1 = c0 + (i ? n1 : n0);
                if (c0 < r.k && r.k <= c1) sm.out[0] = 2u * t + i, sm.out[1] = c0, sm.out[2] = c1 - c0, sm.out[3] = wb + (i ? w0 : 0ull);
            }
            __syncthreads();
            const Region g = {(u32)sm.out[0], (u32)sm.out[2], 0ull, 64u, sm.out[1]};
            const u64 above = sm.out[3];
            __syncthreads();
            thr = last_kept<F32, false>(row, vocab, r, g, (double)r.k, 0ull, sm, w_in);
            all_w = above + w_in;
        }
        if (r.use_p && !(r.p > 0.0f)) {
            thr = ((u64)key_of(r.top) << IDX_BITS) | (max_rank & IDX_MASK);
        } else if (r.use_p) {
            const double target = (double)r.p * (double)all_w;
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
    const float least = least_of(r, thr);
    auto kept = [&](float raw, u32 id) { return kept_units(r, sm.tab, least, thr, value_of(r, raw), id); };
    u64 *sums = sm.weight; /* [WAVES][GROUPS] */
    __syncthreads();
    sums[t] = 0ull;
    __syncthreads();
    for (u32 g = 0; g * per < run; ++g) {
        u64 s = 0;
        for (u32 i = g * per; i < min(g * per + per, run); ++i)
            lane_values<F32>(row, min((wave * run + i) * STEP + lane * E, vocab), vocab, [&](float x, u32 id) { s += kept(x, id); });
        s = wave_sum64(s);
        if (lane == 0u) sums[wave * GROUPS + g] = s;
    }
    __syncthreads();
    const u64 mine = sums[t];
    u64 all;
    const u64 before = block_before(mine, sm.red, all);
    const double target = target_of(a, b, all);
    /* the group that holds the first id whose running sum is over the target */
    if (mine != 0ull && !((double)before > target) && (double)(before + mine) > target) sm.out[0] = t, sm.out[1] = before;
    __syncthreads();
    if (wave == 0u) {
        const u32 w = (u32)sm.out[0] / GROUPS, g = (u32)sm.out[0] % GROUPS;
        u64 sum = sm.out[1];
        for (u32 i = g * per; i < min(g * per + per, run); ++i)
            if (pick<F32>(a, b, row, min((w * run + i) * STEP, vocab), target, all, sum, kept)) break;
    }
}

template <bool F32>
__device__ __forceinline__ const void *row_at(const uocr_sample_args &a, u32 b) {
    return (const uint8_t *)a.logits + (uint64_t)b * a.stride * (F32 ? 4u : 2u);
}

template <bool F32>
__global__ __launch_bounds__(NT) void k_sample_row(uocr_sample_args a, u32 shift) {
    __shared__ Shared sm;
    whole_row<F32>(a, blockIdx.x, row_at<F32>(a, blockIdx.x), shift, sm);
}

/* ---- a row over several blocks --------------------------------------------------- */

/* What the histogram says of a row: whether its kept set ends (any), in a list
 * of n values that base_n values and base_w units stand in front of; crowded
 * lists are not made. */
struct Found {
    u64 base_n, base_w, all_w;
    u32 n, any, use_k, crowded;
};

/* What the launches of a row leave for each other, in the workspace. */
struct Plan {
    uocr_sample_args a;
    u32 shift, steps, chunks, run; /* of a row; run: steps of a chunk */
    u64 *max_rank;                 /* [rows][chunks] */
    u64 *weight;                   /* [rows][BINS] */
    u32 *count;                    /* [rows][BINS] */
    u64 *list;                     /* [rows][LIST] */
    u32 *n;                        /* [rows]: the list's length so far */
    Found *found;                  /* [rows] */
    u64 *thr;                      /* [rows]: the rank that ends the kept set */
    u64 *sums;                     /* [rows][steps] */
    bool cut;                      /* some row has top-k or top-p */
};

template <bool F32, typename F>
__device__ __forceinline__ void chunk_values(const Plan &g, const void *row, u32 chunk, F &&f) {
    const u32 s1 = min(chunk * g.run + g.run, g.steps);
    for (u32 s = chunk * g.run + (threadIdx.x >> 6); s < s1; s += CWAVES)
        lane_values<F32>(row, min(s * STEP + (threadIdx.x & 63u) * E, g.a.vocab), g.a.vocab, f);
}

/* 1: the chunk's largest logit; the row's histogram is cleared. */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_max(Plan g) {
    __shared__ u64 red[CWAVES];
    const u32 b = blockIdx.x / g.chunks, chunk = blockIdx.x % g.chunks;
    for (u32 i = chunk * CT + threadIdx.x; i < BINS; i += CT * g.chunks) g.weight[(u64)b * BINS + i] = 0ull, g.count[(u64)b * BINS + i] = 0u;
    if (chunk == 0u && threadIdx.x == 0u) {
        g.n[b] = 0u;
        g.found[b] = Found{};
    }
    const void *row = row_at<F32>(g.a, b);
    const u64 rank = largest(red, [&](auto f) { chunk_values<F32>(g, row, chunk, f); });
    if (threadIdx.x == 0u) g.max_rank[(u64)b * g.chunks + chunk] = rank;
}

__device__ __forceinline__ u64 row_max(const Plan &g, u32 b) {
    u64 rank = (threadIdx.x & 63u) < g.chunks ? g.max_rank[(u64)b * g.chunks + (threadIdx.x & 63u)] : 0ull;
    for (int o = 32; o > 0; o >>= 1) {
        const u64 v = shfl_xor64(rank, o);
        rank = v > rank ? v : rank;
    }
    return rank;
}

/* 2: the histogram, in LDS and from there into the row's. */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_bins(Plan g) {
    __shared__ double tab[TAB];
    __shared__ u64 weights[BINS];
    __shared__ u32 counts[BINS];
    const u32 b = blockIdx.x / g.chunks, chunk = blockIdx.x % g.chunks;
    const u64 max_rank = row_max(g, b);
    const float temp = temperature_of(g.a, b);
    if (max_rank == 0ull || !(temp > 0.0f)) return;
    const Row r = row_of(g.a, b, max_rank, temp, g.shift);
    if (!r.use_k && !r.use_p) return;
    for (u32 i = threadIdx.x; i < BINS; i += CT) weights[i] = 0ull, counts[i] = 0u;
    if (r.use_p) fill_table(tab);
    __syncthreads();
    chunk_values<F32>(g, row_at<F32>(g.a, b), chunk, [&](float raw, u32 id) {
        const float x = value_of(r, raw);
        const u32 i = bin_of(r, x);
        if (i == BINS - 1u) return;
        atomicAdd(&counts[i], 1u);
        if (r.use_p) atomicAdd(&weights[i], units(weight(r, tab, x)));
    });
    __syncthreads();
    for (u32 i = threadIdx.x; i < BINS; i += CT) {
        if (counts[i] == 0u) continue;
        atomicAdd(&g.count[(u64)b * BINS + i], counts[i]);
        if (r.use_p) atomicAdd(&g.weight[(u64)b * BINS + i], weights[i]);
    }
}

/* The bins whose values decide: those up to `last` (from `first`), in front of
 * which base_n values and base_w units stand, n values in all. */
struct Deciding {
    u32 first, last, n;
    u64 base_n, base_w, all_w;
    bool use_k, any;
};

__device__ __forceinline__ Deciding deciding(const Plan &g, u32 b, const Row &r, u64 *red, u64 *red2, u64 *out) {
    constexpr u32 PER = BINS / CT;
    const u32 t = threadIdx.x;
    u32 n[PER];
    u64 w[PER], sn = 0, sw = 0;
#pragma unroll
    for (u32 i = 0; i < PER; ++i) {
        n[i] = g.count[(u64)b * BINS + PER * t + i];
        w[i] = g.weight[(u64)b * BINS + PER * t + i];
        sn += n[i];
        sw += w[i];
    }
    u64 all_n, all_w;
    u64 nb = block_before(sn, red, all_n), wb = block_before(sw, red2, all_w);
    Deciding d;
    d.all_w = all_w;
    d.use_k = r.use_k && (u64)r.k < all_n;
    d.any = d.use_k || r.use_p;
    if (!d.any) return d;
    const double target = (double)r.p * (double)all_w;
#pragma unroll
    for (u32 i = 0; i < PER; ++i) {
        const bool here = d.use_k ? nb < r.k && r.k <= nb + n[i] : n[i] != 0u && (!(r.p > 0.0f) ? nb == 0ull : (double)wb < target && !((double)(wb + w[i]) < target));
        if (here) out[0] = PER * t + i, out[1] = nb, out[2] = wb, out[3] = n[i];
        nb += n[i];
        wb += w[i];
    }
    __syncthreads();
    d.last = (u32)out[0];
    /* with both, top-p decides within top-k's values: all of them are looked at */
    const bool both = d.use_k && r.use_p;
    d.first = both ? 0u : d.last;
    d.base_n = both ? 0ull : out[1];
    d.base_w = both ? 0ull : out[2];
    const u64 count = both ? out[1] + out[3] : out[3];
    d.n = count > LIST ? LIST + 1u : (u32)count;
    return d;
}

/* 3: the values in the deciding bins, listed (in any order). */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_list(Plan g) {
    __shared__ u64 red[CWAVES], red2[CWAVES], out[4], list[LIST];
    __shared__ u32 n, first;
    const u32 b = blockIdx.x / g.chunks, chunk = blockIdx.x % g.chunks;
    const u64 max_rank = row_max(g, b);
    const float temp = temperature_of(g.a, b);
    if (max_rank == 0ull || !(temp > 0.0f)) return;
    const Row r = row_of(g.a, b, max_rank, temp, g.shift);
    if (!r.use_k && !r.use_p) return;
    if (threadIdx.x == 0u) n = 0u;
    const Deciding d = deciding(g, b, r, red, red2, out);
    if (chunk == 0u && threadIdx.x == 0u) {
        Found &f = g.found[b];
        f.crowded = d.any && d.n > LIST ? 1u : 0u;
        f.any = d.any ? 1u : 0u;
        f.use_k = d.use_k ? 1u : 0u;
        f.n = d.any ? d.n : 0u;
        f.base_n = d.any ? d.base_n : 0ull;
        f.base_w = d.any ? d.base_w : 0ull;
        f.all_w = d.all_w;
    }
    if (!d.any || d.n > LIST) return;
    /* most values are well below the deciding bins: a comparison tells (two bins' margin for the bins' roundings) */
    float floor = r.top - ((float)d.last + 3.0f) / r.scale;
    if (!(floor > -INFINITY) || r.inf) floor = -INFINITY;
    chunk_values<F32>(g, row_at<F32>(g.a, b), chunk, [&](float raw, u32 id) {
        if (!(raw >= floor)) return;
        const float x = value_of(r, raw);
        const u32 i = bin_of(r, x);
        if (i < d.first || i > d.last) return;
        const u32 at = atomicAdd(&n, 1u);
        if (at < LIST) list[at] = rank_of(x, id); /* at most d.n: the bins were counted by the same arithmetic */
    });
    __syncthreads();
    const u32 mine = min(n, LIST);
    if (threadIdx.x == 0u && mine != 0u) first = atomicAdd(&g.n[b], mine);
    __syncthreads();
    for (u32 i = threadIdx.x; i < mine; i += CT)
        if (first + i < LIST) g.list[(u64)b * LIST + first + i] = list[i];
}

/* 4: the rank that ends the kept set: the listed values in order (a bitonic
 * sort of one value a thread, by lane exchange within wavefronts), what stands
 * in front of each, and the last one that is kept. */
template <bool F32>
__global__ __launch_bounds__(LIST) void k_sample_cut(Plan g) {
    __shared__ double tab[TAB];
    __shared__ u64 red[LIST / 64], list[LIST];
    const u32 b = blockIdx.x, t = threadIdx.x;
    const u64 max_rank = row_max(g, b);
    const float temp = temperature_of(g.a, b);
    if (max_rank == 0ull || !(temp > 0.0f)) return;
    const Row r = row_of(g.a, b, max_rank, temp, g.shift);
    const Found f = g.found[b];
    if ((!r.use_k && !r.use_p) || f.any == 0u || f.crowded != 0u) {
        if (t == 0u) g.thr[b] = 0ull;
        return;
    }
    u64 rank = t < f.n ? g.list[(u64)b * LIST + t] : 0ull; /* 0: behind all */
    fill_table(tab);
    __syncthreads();
    u32 size = 64u;
    while (size < f.n) size <<= 1;
    for (u32 k = 2u; k <= size; k <<= 1) {
        for (u32 j = k >> 1; j > 0u; j >>= 1) {
            u64 other;
            if (j >= 64u) {
                list[t] = rank;
                __syncthreads();
                other = list[t ^ j];
                __syncthreads();
            } else {
                other = shfl_xor64(rank, (int)j);
            }
            /* descending: the lower place of a pair keeps the larger value in runs that descend */
            const bool larger = ((t & j) == 0u) == ((t & k) == 0u);
            rank = (other > rank) == larger ? other : rank;
        }
    }
    const bool in = t < f.n;
    const u64 bn = f.base_n + t, w = in ? units(weight(r, tab, of_key((u32)(rank >> IDX_BITS)))) : 0ull;
    const bool in_k = in && (f.use_k == 0u || bn < r.k);
    u64 all;
    const u64 bw = f.base_w + block_before(in_k ? w : 0ull, red, all);
    if (!(f.use_k != 0u && r.use_p)) all = f.all_w;
    const double target = (double)r.p * (double)all;
    const bool kept = in_k && (!r.use_p || bn == 0ull || (double)bw < target);
    const u32 n = (u32)__syncthreads_count(kept);
    if (kept && t == n - 1u) g.thr[b] = rank;
}

/* 5: the kept units of each step. */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_sums(Plan g) {
    __shared__ double tab[TAB];
    const u32 b = blockIdx.x / g.chunks, chunk = blockIdx.x % g.chunks, t = threadIdx.x;
    const u64 max_rank = row_max(g, b);
    const float temp = temperature_of(g.a, b);
    if (max_rank == 0ull || !(temp > 0.0f) || (g.cut && g.found[b].crowded != 0u)) return;
    const Row r = row_of(g.a, b, max_rank, temp, g.shift);
    const u64 thr = g.cut ? g.thr[b] : 0ull;
    fill_table(tab);
    __syncthreads();
    const void *row = row_at<F32>(g.a, b);
    const float least = least_of(r, thr);
    const u32 s1 = min(chunk * g.run + g.run, g.steps);
    for (u32 s = chunk * g.run + (t >> 6); s < s1; s += CWAVES) {
        u64 sum = 0;
        lane_values<F32>(row, min(s * STEP + (t & 63u) * E, g.a.vocab), g.a.vocab,
                         [&](float raw, u32 id) { sum += kept_units(r, tab, least, thr, value_of(r, raw), id); });
        if (__any(sum != 0ull)) sum = wave_sum64(sum);
        if ((t & 63u) == 0u) g.sums[(u64)b * g.steps + s] = sum;
    }
}

/* 6: the step that the target falls into, and its token.  Rows with crowded
 * bins are done here from the start. */
template <bool F32>
__global__ __launch_bounds__(NT) void k_sample_pick(Plan g) {
    __shared__ Shared sm;
    const u32 b = blockIdx.x, t = threadIdx.x;
    const void *row = row_at<F32>(g.a, b);
    const u64 max_rank = row_max(g, b);
    const float temp = temperature_of(g.a, b);
    if (greedy(g.a, b, max_rank, temp)) return;
    if (g.cut && g.found[b].crowded != 0u) {
        whole_row<F32>(g.a, b, row, g.shift, sm);
        return;
    }
    const Row r = row_of(g.a, b, max_rank, temp, g.shift);
    fill_table(sm.tab);
    const u64 thr = g.cut ? g.thr[b] : 0ull;
    const u32 per = (g.steps + NT - 1u) / NT, s0 = min(t * per, g.steps), s1 = min(s0 + per, g.steps);
    u64 mine = 0;
    for (u32 s = s0; s < s1; ++s) mine += g.sums[(u64)b * g.steps + s];
    u64 all;
    const u64 before = block_before(mine, sm.red, all);
    const double target = target_of(g.a, b, all);
    if (mine != 0ull && !((double)before > target) && (double)(before + mine) > target) sm.out[0] = s0, sm.out[1] = before;
    __syncthreads();
    if (t >= 64u) return;
    const float least = least_of(r, thr);
    auto kept = [&](float raw, u32 id) { return kept_units(r, sm.tab, least, thr, value_of(r, raw), id); };
    u64 sum = sm.out[1];
    for (u32 s = (u32)sm.out[0]; s < g.steps; ++s)
        if (pick<F32>(g.a, b, row, s * STEP, target, all, sum, kept)) break;
}

u32 shift_of(u32 vocab) {
    u32 bits = 0;
    while ((1u << bits) < vocab) ++bits;
    return 62u - bits < 50u ? 62u - bits : 50u;
}

/* Rows of up to this many tokens are done by one block each, in one launch. */
constexpr u32 ONE_BLOCK = 8192;

size_t lay_out(Plan &g, u32 rows, u32 vocab, uint8_t *ws) {
    g.steps = (vocab + STEP - 1u) / STEP;
    /* about 2,048 blocks (192 rows of 129,280 fp16: 94.9 us, with 1,024 103.1; blocks of 256 threads 99.2); a wavefront
     * has at least a step */
    const u32 most = (g.steps + CWAVES - 1u) / CWAVES, want = rows < 2048u ? 2048u / rows : 1u;
    g.chunks = want < most ? want : most;
    if (g.chunks > MAX_CHUNKS) g.chunks = MAX_CHUNKS;
    g.run = (g.steps + g.chunks - 1u) / g.chunks;
    g.shift = shift_of(vocab);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t *p = ws + at;
        at += (bytes + 255u) & ~(size_t)255u;
        return (void *)p;
    };
    g.max_rank = (u64 *)take((size_t)rows * MAX_CHUNKS * 8u);
    g.weight = (u64 *)take((size_t)rows * BINS * 8u);
    g.count = (u32 *)take((size_t)rows * BINS * 4u);
    g.list = (u64 *)take((size_t)rows * LIST * 8u);
    g.n = (u32 *)take((size_t)rows * 4u);
    g.found = (Found *)take((size_t)rows * sizeof(Found));
    g.thr = (u64 *)take((size_t)rows * 8u);
    g.sums = (u64 *)take((size_t)rows * g.steps * 8u);
    return at;
}

template <bool F32>
hipError_t launch(hipStream_t st, const uocr_sample_args &a) {
    if (a.vocab <= ONE_BLOCK) {
        hipLaunchKernelGGL((k_sample_row<F32>), dim3(a.rows), dim3(NT), 0, st, a, shift_of(a.vocab));
        return hipGetLastError();
    }
    Plan g;
    g.a = a;
    (void)lay_out(g, a.rows, a.vocab, (uint8_t *)a.ws);
    g.cut = a.top_k != nullptr || a.top_p != nullptr;
    const dim3 grid(a.rows * g.chunks), block(CT);
    hipLaunchKernelGGL((k_sample_max<F32>), grid, block, 0, st, g);
    if (g.cut) {
        hipLaunchKernelGGL((k_sample_bins<F32>), grid, block, 0, st, g);
        hipLaunchKernelGGL((k_sample_list<F32>), grid, block, 0, st, g);
        hipLaunchKernelGGL((k_sample_cut<F32>), dim3(a.rows), dim3(LIST), 0, st, g);
    }
    hipLaunchKernelGGL((k_sample_sums<F32>), grid, block, 0, st, g);
    hipLaunchKernelGGL((k_sample_pick<F32>), dim3(a.rows), dim3(NT), 0, st, g);
    return hipGetLastError();
}

}  // namespace

size_t uocr_sample_ws_bytes(uint32_t rows, uint32_t vocab) {
    if (vocab <= ONE_BLOCK || rows == 0u) return 16u;
    Plan g;
    return lay_out(g, rows, vocab, nullptr);
}

hipError_t uocr_launch_sample(hipStream_t st, const uocr_sample_args *a) {
    return a->f32 ? launch<true>(st, *a) : launch<false>(st, *a);
}
