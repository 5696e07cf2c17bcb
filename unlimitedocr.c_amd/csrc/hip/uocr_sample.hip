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
constexpr u32 ROW_U = 1;                  /* steps that it loads at a time: its registers hold no more */
constexpr u32 E = 8, STEP = 64 * E;       /* values of a lane and of a wavefront per step */
constexpr u32 BINS = 2048;
constexpr u32 LIST = 1024;                /* values that are ordered at once, one a thread */
constexpr u32 GROUPS = 64;                /* partial sums of a wavefront's run in the last pass */
constexpr u32 IDX_BITS = 24, IDX_MASK = (1u << IDX_BITS) - 1u;
constexpr u32 TAB = 1024;                 /* 2^(i / TAB) */
constexpr u32 MAX_CHUNKS = 64;
constexpr u32 TOPS = 512;                 /* groups of steps whose largest logits bound top-k */

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

/* 2^(i / TAB) by the exponential series: 24 terms of at most ln 2 leave less than 2^-90. */
struct Powers {
    double v[TAB];
};
constexpr Powers powers() {
    Powers p = {};
    for (u32 i = 0; i < TAB; ++i) {
        const double x = 0.6931471805599453 * i / TAB;
        double sum = 1.0;
        for (int n = 24; n > 0; --n) sum = 1.0 + x / n * sum;
        p.v[i] = sum;
    }
    return p;
}
__device__ const Powers g_powers = powers();

__device__ __forceinline__ void fill_table(double *tab) {
    for (u32 i = threadIdx.x; i < TAB; i += blockDim.x) tab[i] = g_powers.v[i];
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

/* The E values of the lane at id0; NaN, which takes part in nothing, outside the row. */
template <bool F32, bool INSIDE>
__device__ __forceinline__ void lane_load(const void *row, u32 id0, u32 vocab, float *x) {
    if (INSIDE || id0 + E <= vocab) {
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
    } else {
#pragma unroll
        for (u32 e = 0; e < E; ++e) x[e] = id0 + e >= vocab ? __builtin_nanf("") : F32 ? ((const float *)row)[id0 + e] : (float)((const _Float16 *)row)[id0 + e];
    }
}
__device__ __forceinline__ float largest_of(const float *x) {
    return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
}

/* f(step, values) for the steps s0, s0 + stride, .. below s1, by a wavefront:
 * U steps' loads at a time, or a pass over a row would be a chain of
 * memory latencies. */
template <bool F32, u32 U, typename F>
__device__ __forceinline__ void each_step(const void *row, u32 vocab, u32 s0, u32 s1, u32 stride, F &&f) {
    const u32 lane = threadIdx.x & 63u;
    u32 s = s0;
    if constexpr (U > 1)
    for (; s + (U - 1u) * stride < s1 && (s + (U - 1u) * stride + 1u) * STEP <= vocab; s += U * stride) {
        float x[U][E];
#pragma unroll
        for (u32 u = 0; u < U; ++u) lane_load<F32, true>(row, (s + u * stride) * STEP + lane * E, vocab, x[u]);
#pragma unroll
        for (u32 u = 0; u < U; ++u) f(s + u * stride, x[u]);
    }
    for (; s < s1; s += stride) {
        float x[E];
        lane_load<F32, false>(row, min(s * STEP + lane * E, vocab), vocab, x);
        f(s, x);
    }
}

/* g(logit, id) for the lane's values of step s that are at least `least` (not
 * NaN): few lanes have one where few values are kept. */
template <typename G>
__device__ __forceinline__ void values_from(float least, u32 s, const float *x, G &&g) {
    if (!(largest_of(x) >= least)) return;
    const u32 id0 = s * STEP + (threadIdx.x & 63u) * E;
#pragma unroll
    for (u32 e = 0; e < E; ++e)
        if (x[e] >= least) g(x[e], id0 + e);
}

/* The step's largest logit, in every lane; best and best_id of the lane. */
__device__ __forceinline__ float step_largest(u32 s, const float *x, float &best, u32 &best_id) {
    float m = largest_of(x);
    if (m > best) {
        best = m;
        const u32 id0 = s * STEP + (threadIdx.x & 63u) * E;
#pragma unroll
        for (int e = E - 1; e >= 0; --e) best_id = x[e] == m ? id0 + e : best_id;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    return m;
}

__device__ __forceinline__ float value_of(const Row &r, float x) {
    return !r.inf ? x : x == INFINITY ? 0.0f : -INFINITY;
}

/* f over the whole row's values from `least` on, by all threads. */
template <bool F32, typename F>
__device__ __forceinline__ void row_values(const void *row, u32 vocab, float least, F &&f) {
    each_step<F32, ROW_U>(row, vocab, threadIdx.x >> 6, (vocab + STEP - 1u) / STEP, WAVES, [&](u32 s, const float *x) { values_from(least, s, x, f); });
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
    u32 tops[TOPS], place[512];
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

/* The ranks of the block's LIST threads, largest first; the first n threads have
 * one, the others 0.  Few are counted against each other, by all threads (256:
 * 1 us); from about 400 on a bitonic sort, by lane exchange within wavefronts,
 * is the faster one (7 us). */
__device__ __forceinline__ u64 sorted(u64 rank, u32 n, u64 *buf, u32 *place) {
    const u32 t = threadIdx.x;
    u32 size = 64u;
    while (size < n) size <<= 1;
    if (n <= 384u) {
        const u32 parts = LIST / size, part = t / size, e = t % size;
        if (t < size) {
            buf[t] = rank;
            place[t] = 0u;
        }
        __syncthreads();
        if (e < n) {
            const u64 mine = buf[e];
            const u32 i1 = n * (part + 1u) / parts;
            u32 before = 0;
#pragma unroll 4
            for (u32 i = n * part / parts; i < i1; ++i) before += buf[i] > mine ? 1u : 0u;
            if (before != 0u) atomicAdd(&place[e], before);
        }
        __syncthreads();
        if (t < n) buf[place[t]] = rank;
        __syncthreads();
        rank = t < n ? buf[t] : 0ull;
        __syncthreads();
        return rank;
    }
    for (u32 k = 2u; k <= size; k <<= 1) {
        for (u32 j = k >> 1; j > 0u; j >>= 1) {
            u64 other;
            if (j >= 64u) {
                buf[t] = rank;
                __syncthreads();
                other = buf[t ^ j];
                __syncthreads();
            } else {
                other = shfl_xor64(rank, (int)j);
            }
            /* the lower place of a pair keeps the larger value in runs that descend */
            const bool larger = ((t & j) == 0u) == ((t & k) == 0u);
            rank = (other > rank) == larger ? other : rank;
        }
    }
    return rank;
}

/* Top-k of up to 7/8 of the groups: k values are at least the k-th largest of
 * the groups' largest, so what is below cannot be kept. */
__device__ __forceinline__ bool bounded(const Row &r, u32 groups) {
    return r.use_k && r.k <= groups * 7u / 8u;
}
/* tops[i] of lane l: group 64 i + l's, 0 where there is none; by each wavefront
 * for itself, from the key's highest bit on.  To 20 bits: a bound may be lower. */
template <u32 N>
__device__ __forceinline__ u32 kth_key(const u32 *tops, u32 k) {
    u32 key = 0;
    for (u32 bit = 1u << 31; bit >= 1u << 12; bit >>= 1) {
        u32 n = 0;
#pragma unroll
        for (u32 i = 0; i < N; ++i) n += (u32)__popcll(__ballot(tops[i] >= (key | bit)));
        if (n >= k) key |= bit;
    }
    return key;
}
__device__ __forceinline__ float kth_largest(const u32 *tops, u32 groups, u32 k) {
    const u32 key = groups <= 64u ? kth_key<1>(tops, k) : groups <= 256u ? kth_key<4>(tops, k) : kth_key<TOPS / 64>(tops, k);
    return of_key(max(key, key_of(-INFINITY)));
}

/* The rank of the last value that is kept, of the n listed ones in order (one a
 * thread), in front of which base_n values and base_w units stand; all: units
 * of all values that top-p sums. */
__device__ __forceinline__ u64 cut(const Row &r, const double *tab, u64 rank, u32 n, bool use_k, u64 base_n, u64 base_w, u64 all, u64 *red, u64 *out) {
    const u32 t = threadIdx.x;
    const bool in = t < n;
    const u64 bn = base_n + t, w = in ? units(weight(r, tab, of_key((u32)(rank >> IDX_BITS)))) : 0ull;
    const bool in_k = in && (!use_k || bn < r.k);
    u64 sum;
    const u64 bw = base_w + block_before(in_k ? w : 0ull, red, sum);
    const double target = (double)r.p * (double)(use_k ? sum : all);
    const bool kept = in_k && (!r.use_p || bn == 0ull || (double)bw < target);
    const u32 last = (u32)__syncthreads_count(kept);
    if (t + 1u == last) *out = rank;
    __syncthreads();
    return *out;
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
        row_values<F32>(row, vocab, -INFINITY, [&](float raw, u32 id) {
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
    row_values<F32>(row, vocab, -INFINITY, [&](float raw, u32 id) {
        const float x = value_of(r, raw);
        const u64 rank = rank_of(x, id);
        if (!inside(x, rank)) return;
        sm.list[atomicAdd(&sm.n, 1u)] = rank;
    });
    __syncthreads();
    const u32 n = sm.n;
    const u64 rank = sorted(t < n ? sm.list[t] : 0ull, n, sm.list, sm.place);
    const u64 w = t < n ? units(weight(r, sm.tab, of_key((u32)(rank >> IDX_BITS)))) : 0ull;
    u64 all;
    const u64 before = g.before + block_before(t >= n ? 0ull : WEIGHTED ? w : 1ull, sm.red, all);
    const bool kept = t < n && (double)before < limit;
    (void)block_before(kept ? w : 0ull, sm.red, all);
    kept_w += all;
    const u32 last = (u32)__syncthreads_count(kept);
    if (t + 1u == last) sm.out[0] = rank;
    __syncthreads();
    const u64 thr = sm.out[0];
    __syncthreads();
    return thr;
}

/* The first id whose running sum of kept units is over the target, in the step
 * that `sum` stands in front of; by one wavefront.
 * Returns whether it is there, and what stands in front of the next values. */
template <bool F32, typename K>
__device__ __forceinline__ bool pick(const uocr_sample_args &a, u32 b, const void *row, u32 step, float least, double target, u64 all, u64 &sum, K &&kept) {
    const u32 lane = threadIdx.x & 63u;
    float x[E];
    lane_load<F32, false>(row, min(step * STEP + lane * E, a.vocab), a.vocab, x);
    u64 s = 0;
    values_from(least, step, x, [&](float v, u32 id) { s += kept(v, id); });
    u64 at = sum + wave_before(s);
    const u64 found = __ballot(s != 0ull && !((double)at > target) && (double)(at + s) > target);
    sum = shfl64(at + s, 63);
    if (found == 0ull) return false;
    if (lane == (u32)__ffsll((long long)found) - 1u) {
        bool done = false;
        values_from(least, step, x, [&](float y, u32 id) {
            const u64 v = kept(y, id);
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

/* The rank of the block's largest logit, from its lanes'. */
__device__ __forceinline__ u64 largest(float best, u32 best_id, u64 *red) {
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
    if (x == least && rank_of(x, id) < thr) return 0ull;
    const double w = weight(r, tab, x);
    return w >= r.min_w ? units(w) : 0ull;
}
/* The logit below which nothing is kept (with +inf ones, as they stand in the
 * row: those alone). */
__device__ __forceinline__ float least_of(const Row &r, u64 thr) {
    return thr == 0ull ? r.cut : fmaxf(r.cut, of_key((u32)(thr >> IDX_BITS)));
}
__device__ __forceinline__ float least_raw(const Row &r, float least) {
    return r.inf ? INFINITY : least;
}

/* A row in one block.  The kept set of top-k and top-p is all values from some
 * rank on.  For a small k the values that can be in it are those from the k-th
 * largest of 512-value steps' maxima on, some k to 2 k of them, which are listed
 * and ordered.  Else a histogram over bins below the maximum (counts, and units
 * of weight for top-p) finds the bin of the last kept value, and the bin's few
 * values are ordered. */
template <bool F32>
__device__ void whole_row(const uocr_sample_args &a, u32 b, const void *row, u32 shift, Shared &sm) {
    const u32 t = threadIdx.x, lane = t & 63u, wave = t >> 6, vocab = a.vocab;
    const u32 steps = (vocab + STEP - 1u) / STEP, groups = min(steps, TOPS);
    float best = -INFINITY;
    u32 best_id = 0xffffffffu;
    sm.tops[t % TOPS] = 0u;
    __syncthreads();
    each_step<F32, ROW_U>(row, vocab, wave, steps, WAVES, [&](u32 s, const float *x) {
        const u32 top = key_of(step_largest(s, x, best, best_id));
        if (lane == 0u) sm.tops[s % TOPS] = max(sm.tops[s % TOPS], top); /* a group's steps are one wavefront's: TOPS is a multiple of WAVES */
    });
    const u64 max_rank = largest(best, best_id, sm.red);
    const float temp = temperature_of(a, b);
    if (greedy(a, b, max_rank, temp)) return;
    const Row r = row_of(a, b, max_rank, temp, shift);
    fill_table(sm.tab);
    if (t == 0u) sm.n = 0u;
    __syncthreads();

    u64 thr = 0; /* kept: ranks from here on */
    bool found = false;
    if (bounded(r, groups)) {
        u32 tops[TOPS / 64];
#pragma unroll
        for (u32 i = 0; i < TOPS / 64; ++i) tops[i] = sm.tops[64u * i + lane];
        const float floor = kth_largest(tops, groups, r.k);
        row_values<F32>(row, vocab, floor, [&](float raw, u32 id) {
            const u32 at = atomicAdd(&sm.n, 1u);
            if (at < LIST) sm.list[at] = rank_of(value_of(r, raw), id);
        });
        __syncthreads();
        const u32 n = sm.n;
        found = n <= LIST;
        if (found) thr = cut(r, sm.tab, sorted(t < n ? sm.list[t] : 0ull, n, sm.list, sm.place), n, true, 0ull, 0ull, 0ull, sm.red, &sm.out[0]);
        __syncthreads();
    }
    if (!found && (r.use_k || r.use_p)) {
        for (u32 i = t; i < BINS; i += NT) sm.weight[i] = 0ull, sm.count[i] = 0u;
        __syncthreads();
        row_values<F32>(row, vocab, -INFINITY, [&](float raw, u32 id) {
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
    const u32 run = (steps + WAVES - 1u) / WAVES, per = (run + GROUPS - 1u) / GROUPS;
    const float least = least_of(r, thr), raw_least = least_raw(r, least);
    auto kept = [&](float raw, u32 id) { return kept_units(r, sm.tab, least, thr, value_of(r, raw), id); };
    u64 *sums = sm.weight; /* [WAVES][GROUPS] */
    __syncthreads();
    sums[t] = 0ull;
    __syncthreads();
    each_step<F32, ROW_U>(row, vocab, min(wave * run, steps), min(wave * run + run, steps), 1u, [&](u32 s, const float *x) {
        u64 sum = 0;
        values_from(raw_least, s, x, [&](float v, u32 id) { sum += kept(v, id); });
        if (!__any(sum != 0ull)) return;
        sum = wave_sum64(sum);
        if (lane == 0u) sums[wave * GROUPS + (s - wave * run) / per] += sum;
    });
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
            if (w * run + i < steps && pick<F32>(a, b, row, w * run + i, raw_least, target, all, sum, kept)) break;
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
 * of n values that base_n values and base_w units stand in front of. */
struct Found {
    u64 base_n, base_w, all_w;
    u32 n, any, use_k, pad;
};

/* What the launches of a row leave for each other, in the workspace. */
struct Plan {
    uocr_sample_args a;
    u32 shift, steps, chunks;      /* of a row; chunks: of the first launch */
    u32 parts, run;                /* of this launch: blocks of a row, steps of each */
    u64 *max_rank;                 /* [rows][chunks] */
    u32 *tops;                     /* [rows][steps]: keys of the steps' largest logits */
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
__device__ __forceinline__ void chunk_steps(const Plan &g, const void *row, u32 chunk, F &&f) {
    each_step<F32, 4>(row, g.a.vocab, chunk * g.run + (threadIdx.x >> 6), min(chunk * g.run + g.run, g.steps), CWAVES, f);
}
template <bool F32, typename F>
__device__ __forceinline__ void chunk_values(const Plan &g, const void *row, u32 chunk, float least, F &&f) {
    chunk_steps<F32>(g, row, chunk, [&](u32 s, const float *x) { values_from(least, s, x, f); });
}

/* 1: the steps' and the chunk's largest logit; the row's histogram is cleared. */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_max(Plan g) {
    __shared__ u64 red[CWAVES];
    const u32 b = blockIdx.x / g.parts, chunk = blockIdx.x % g.parts, lane = threadIdx.x & 63u;
    if (g.cut)
        for (u32 i = chunk * CT + threadIdx.x; i < BINS; i += CT * g.parts) g.weight[(u64)b * BINS + i] = 0ull, g.count[(u64)b * BINS + i] = 0u;
    if (chunk == 0u && threadIdx.x == 0u) {
        g.n[b] = 0u;
        g.found[b] = Found{};
    }
    const void *row = row_at<F32>(g.a, b);
    float best = -INFINITY;
    u32 best_id = 0xffffffffu;
    chunk_steps<F32>(g, row, chunk, [&](u32 s, const float *x) {
        const float top = step_largest(s, x, best, best_id);
        if (lane == 0u) g.tops[(u64)b * g.steps + s] = key_of(top);
    });
    const u64 rank = largest(best, best_id, red);
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
    const u32 b = blockIdx.x / g.parts, chunk = blockIdx.x % g.parts;
    const u64 max_rank = row_max(g, b);
    const float temp = temperature_of(g.a, b);
    if (max_rank == 0ull || !(temp > 0.0f)) return;
    const Row r = row_of(g.a, b, max_rank, temp, g.shift);
    if ((!r.use_k && !r.use_p) || bounded(r, min(g.steps, TOPS))) return;
    for (u32 i = threadIdx.x; i < BINS; i += CT) weights[i] = 0ull, counts[i] = 0u;
    if (r.use_p) fill_table(tab);
    __syncthreads();
    chunk_values<F32>(g, row_at<F32>(g.a, b), chunk, -INFINITY, [&](float raw, u32 id) {
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

/* 3: the values that decide, listed (in any order): those from top-k's bound on,
 * or those in the deciding bins. */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_list(Plan g) {
    __shared__ u64 red[CWAVES], red2[CWAVES], out[4], list[LIST];
    __shared__ u32 n, first;
    const u32 b = blockIdx.x / g.parts, chunk = blockIdx.x % g.parts, t = threadIdx.x;
    const u64 max_rank = row_max(g, b);
    const float temp = temperature_of(g.a, b);
    if (max_rank == 0ull || !(temp > 0.0f)) return;
    const Row r = row_of(g.a, b, max_rank, temp, g.shift);
    if (!r.use_k && !r.use_p) return;
    if (t == 0u) n = 0u;
    const u32 groups = min(g.steps, TOPS);
    const void *row = row_at<F32>(g.a, b);
    Found f = {};
    f.any = 1u;
    if (bounded(r, groups)) {
        u32 tops[TOPS / 64] = {};
        for (u32 s0 = 0; s0 < g.steps; s0 += TOPS) {
#pragma unroll
            for (u32 i = 0; i < TOPS / 64; ++i) {
                const u32 s = s0 + 64u * i + (t & 63u);
                if (s < g.steps) tops[i] = max(tops[i], g.tops[(u64)b * g.steps + s]);
            }
        }
        const float floor = kth_largest(tops, groups, r.k);
        __syncthreads();
        f.use_k = 1u;
        f.n = LIST;
        if (chunk == 0u && t == 0u) g.found[b] = f;
        chunk_values<F32>(g, row, chunk, floor, [&](float raw, u32 id) {
            const u32 at = atomicAdd(&n, 1u);
            if (at < LIST) list[at] = rank_of(value_of(r, raw), id);
        });
    } else {
        const Deciding d = deciding(g, b, r, red, red2, out);
        f.any = d.any ? 1u : 0u;
        if (d.any) {
            f.use_k = d.use_k ? 1u : 0u;
            f.n = d.n;
            f.base_n = d.base_n;
            f.base_w = d.base_w;
        }
        f.all_w = d.all_w;
        if (chunk == 0u && t == 0u) {
            g.found[b] = f;
            if (d.any && d.n > LIST) g.n[b] = LIST + 1u; /* too many */
        }
        if (!d.any || d.n > LIST) return;
        /* most values are well below the deciding bins: a comparison tells (three bins' margin for the bins' roundings) */
        float floor = r.top - ((float)d.last + 3.0f) / r.scale;
        if (!(floor > -INFINITY) || r.inf) floor = -INFINITY;
        chunk_values<F32>(g, row, chunk, floor, [&](float raw, u32 id) {
            const float x = value_of(r, raw);
            const u32 i = bin_of(r, x);
            if (i < d.first || i > d.last) return;
            const u32 at = atomicAdd(&n, 1u);
            if (at < LIST) list[at] = rank_of(x, id); /* at most d.n: the bins were counted by the same arithmetic */
        });
    }
    __syncthreads();
    if (t == 0u && n != 0u) first = atomicAdd(&g.n[b], n); /* of a crowded list: past LIST */
    __syncthreads();
    for (u32 i = t; i < min(n, LIST); i += CT)
        if (first + i < LIST) g.list[(u64)b * LIST + first + i] = list[i];
}

/* 4: the rank that ends the kept set: the listed values in order, what stands in
 * front of each, and the last one that is kept. */
template <bool F32>
__global__ __launch_bounds__(LIST) void k_sample_cut(Plan g) {
    __shared__ double tab[TAB];
    __shared__ u64 red[LIST / 64], list[LIST], out;
    __shared__ u32 place[512];
    const u32 b = blockIdx.x, t = threadIdx.x;
    const u64 max_rank = row_max(g, b);
    const float temp = temperature_of(g.a, b);
    if (max_rank == 0ull || !(temp > 0.0f)) return;
    const Row r = row_of(g.a, b, max_rank, temp, g.shift);
    const Found f = g.found[b];
    const u32 n = g.n[b];
    u64 thr = 0;
    if ((r.use_k || r.use_p) && f.any != 0u && n <= LIST) {
        const u64 rank = t < n ? g.list[(u64)b * LIST + t] : 0ull;
        fill_table(tab);
        __syncthreads();
        thr = cut(r, tab, sorted(rank, n, list, place), n, f.use_k != 0u, f.base_n, f.base_w, f.all_w, red, &out);
    }
    if (t == 0u) g.thr[b] = thr;
}

/* 5: the kept units of each step. */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_sums(Plan g) {
    __shared__ double tab[TAB];
    const u32 b = blockIdx.x / g.parts, chunk = blockIdx.x % g.parts, t = threadIdx.x;
    const u64 max_rank = row_max(g, b);
    const float temp = temperature_of(g.a, b);
    if (max_rank == 0ull || !(temp > 0.0f) || (g.cut && g.n[b] > LIST)) return;
    const Row r = row_of(g.a, b, max_rank, temp, g.shift);
    const u64 thr = g.cut ? g.thr[b] : 0ull;
    fill_table(tab);
    __syncthreads();
    const void *row = row_at<F32>(g.a, b);
    const float least = least_of(r, thr);
    chunk_steps<F32>(g, row, chunk, [&](u32 s, const float *x) {
        u64 sum = 0;
        values_from(least_raw(r, least), s, x, [&](float raw, u32 id) { sum += kept_units(r, tab, least, thr, value_of(r, raw), id); });
        if (__any(sum != 0ull)) sum = wave_sum64(sum);
        if ((t & 63u) == 0u) g.sums[(u64)b * g.steps + s] = sum;
    });
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
    if (g.cut && g.n[b] > LIST) {
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
        if (pick<F32>(g.a, b, row, s, least_raw(r, least), target, all, sum, kept)) break;
}

u32 shift_of(u32 vocab) {
    u32 bits = 0;
    while ((1u << bits) < vocab) ++bits;
    return 62u - bits < 50u ? 62u - bits : 50u;
}

/* Rows of up to ONE_BLOCK tokens are done by a block each, in one launch, and
 * with MANY_ROWS or more up to twice that: us by one launch and by several, fp16,
 * top-k alone and top-p alone, were 19 and 28 against 29 and 33 for 1 row of
 * 16,000, 23 and 39 against 29 and 34 for 1 of 32,000, 34 and 48 against 38 and
 * 47 for 64 of those, 49 and 80 against 55 and 80 for 192 of 64,000, 58 and 148
 * against 64 and 124 for 192 of 129,280. */
constexpr u32 ONE_BLOCK = 16384, MANY_ROWS = 64;
bool by_one_block(u32 rows, u32 vocab) { return vocab <= (rows < MANY_ROWS ? ONE_BLOCK : 2u * ONE_BLOCK); }

/* Blocks of a launch, all rows: where all values take little each, more of them
 * only have their own beginnings to pay for; where some rows' values take an
 * exponential and atomics each and others' nothing, the rows are cut finer.  192
 * mixed rows of 129,280 fp16 took 93.9 us so, 95.4 with 768 everywhere, 98.2 and
 * 96.8 with 1,400 and 4,096 for the heavy ones. */
constexpr u32 LIGHT_BLOCKS = 768, HEAVY_BLOCKS = 2048;

u32 parts_of(const Plan &g, u32 rows, u32 blocks) {
    const u32 most = (g.steps + CWAVES - 1u) / CWAVES, want = rows < blocks ? blocks / rows : 1u; /* a wavefront has at least a step */
    const u32 parts = want < most ? want : most;
    return parts < MAX_CHUNKS ? parts : MAX_CHUNKS;
}

size_t lay_out(Plan &g, u32 rows, u32 vocab, uint8_t *ws) {
    g.steps = (vocab + STEP - 1u) / STEP;
    g.chunks = parts_of(g, rows, LIGHT_BLOCKS);
    g.shift = shift_of(vocab);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t *p = ws + at;
        at += (bytes + 255u) & ~(size_t)255u;
        return (void *)p;
    };
    g.max_rank = (u64 *)take((size_t)rows * MAX_CHUNKS * 8u);
    g.tops = (u32 *)take((size_t)rows * g.steps * 4u);
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
    if (by_one_block(a.rows, a.vocab)) {
        hipLaunchKernelGGL((k_sample_row<F32>), dim3(a.rows), dim3(NT), 0, st, a, shift_of(a.vocab));
        return hipGetLastError();
    }
    Plan g;
    g.a = a;
    (void)lay_out(g, a.rows, a.vocab, (uint8_t *)a.ws);
    g.cut = a.top_k != nullptr || a.top_p != nullptr;
    auto go = [&](void (*kernel)(Plan), u32 blocks) {
        g.parts = parts_of(g, a.rows, blocks);
        g.run = (g.steps + g.parts - 1u) / g.parts;
        hipLaunchKernelGGL(kernel, dim3(a.rows * g.parts), dim3(CT), 0, st, g);
    };
    go(k_sample_max<F32>, LIGHT_BLOCKS);
    if (g.cut) {
        go(k_sample_bins<F32>, HEAVY_BLOCKS);
        go(k_sample_list<F32>, LIGHT_BLOCKS);
        hipLaunchKernelGGL((k_sample_cut<F32>), dim3(a.rows), dim3(LIST), 0, st, g);
    }
    go(k_sample_sums<F32>, HEAVY_BLOCKS);
    hipLaunchKernelGGL((k_sample_pick<F32>), dim3(a.rows), dim3(NT), 0, st, g);
    return hipGetLastError();
}

}  // namespace

size_t uocr_sample_ws_bytes(uint32_t rows, uint32_t vocab) {
    if (rows == 0u || by_one_block(rows, vocab)) return 16u;
    Plan g;
    return lay_out(g, rows, vocab, nullptr);
}

hipError_t uocr_launch_sample(hipStream_t st, const uocr_sample_args *a) {
    return a->f32 ? launch<true>(st, *a) : launch<false>(st, *a);
}
