/*
 * uocr_sample.hip - sampling a token of each row of logits on gfx950.
 */
#include "uocr_dev.h"
#include "uocr_serve.h"


namespace {

constexpr u32 NT = 1024, WAVES = NT / 64; /* a block that has a row of its own */
constexpr u32 CT = 512, CWAVES = CT / 64; /* a block that has a part of a row */
constexpr u32 ROW_U = 1;                  /* steps that it loads at a time: its registers hold no more */
constexpr u32 E = 8, STEP = 64 * E;       /* values of a lane and of a wavefront per step */
constexpr u32 ILP = 4;                     /* of them that are weighed side by side */
constexpr u32 BINS = 2048;
constexpr u32 LIST = 1024;                /* values that are ordered at once, one a thread */
constexpr u32 GROUPS = 64;                /* partial sums of a wavefront's run in the last pass */
constexpr u32 IDX_BITS = 24, IDX_MASK = (1u << IDX_BITS) - 1u;
constexpr u32 TAB = 64;                   /* 2^(i / TAB): 64 doubles, two to a pair of LDS banks */
constexpr u32 MAX_CHUNKS = 64;
constexpr u32 TOPS = 512;                 /* groups of steps whose largest logits bound top-k */
constexpr u32 FEW = 128;                  /* values that are all counted against each other */
constexpr float COUNTED = 8.0f;           /* values of top-p alone are counted to this distance, in temperatures */
constexpr u64 DONE = ~0ull;               /* instead of a rank: the row has its token */

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
    float near;    /* distance to which values are counted */
    float most;    /* the last bin that a logit above -inf can be in */
    u32 shift, k;
    float p;
    bool inf, use_k, use_p;
    bool hot;      /* a temperature above 0 */
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
 * 2^(n / TAB) from the table, a fifth-degree sum for the rest, f <= 1/2 (off by
 * 2^-54), and the exponent (never below -986).  fp64: next to a limit the last
 * bits decide which token it is. */
__device__ __forceinline__ double weight(const Row &r, const double *tab, float x) {
    constexpr double L = 0.6931471805599453 / TAB;
    const double y = fmax(((double)x - (double)r.top) * r.c, -65536.0); /* NaN, too: no weight */
    const double big = y + 6755399441055744.0, f = y - (big - 6755399441055744.0);
    const int n = (int)(u32)__double_as_longlong(big);
    const double p = fma(fma(fma(fma(fma(L * L * L * L * L / 120.0, f, L * L * L * L / 24.0), f, L * L * L / 6.0), f, L * L / 2.0), f, L), f, 1.0);
    const u64 w = (u64)__double_as_longlong(tab[(u32)n & (TAB - 1u)] * p);
    return __longlong_as_double((long long)(w + ((u64)(u32)((n >> 6) << 20) << 32)));
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

/* In units. */
__device__ __forceinline__ void fill_table(double *tab, u32 shift) {
    if (threadIdx.x < TAB) tab[threadIdx.x] = ldexp(g_powers.v[threadIdx.x], (int)shift);
}

/* Bins of equal width below the largest logit, over the range where a weight
 * has a unit, or down to the least of the row's first logits if that is less
 * than half as far: flat rows would crowd few bins, and a crowded one takes 220
 * us instead of 30.  The bin before the last then holds all from there down.
 * The last one holds what has no unit. */
__device__ __forceinline__ u32 bin_of(const Row &r, float x) {
    return x == r.top ? 0u : (u32)fminf((r.top - x) * r.scale, x > -INFINITY ? r.most : (float)(BINS - 1u)); /* NaN: the last */
}

/* The settings of row b; cut: the distance from the largest logit. */
__device__ __forceinline__ Row settings_of(const uocr_sample_args &a, u32 b, u32 shift) {
    Row r;
    const float temp = a.temperature != nullptr ? a.temperature[b] : 1.0f;
    r.hot = temp > 0.0f;
    r.top = 0.0f;
    r.inf = false;
    r.shift = shift;
    r.c = (double)TAB * 1.4426950408889634 / (double)temp;
    r.scale = (float)((double)(BINS - 1u) / TAB * r.c / (double)(shift + 1u));
    const float m = a.min_p != nullptr && a.min_p[b] > 0.0f ? fminf(a.min_p[b], 1.0f) : 0.0f;
    r.min_w = ldexp((double)m, (int)shift);
    r.cut = temp * logf(m); /* -inf without min_p */
    r.near = COUNTED * temp;
    r.most = (float)(BINS - 1u);
    r.k = a.top_k != nullptr && a.top_k[b] > 0 ? (u32)a.top_k[b] : 0u;
    r.p = a.top_p != nullptr ? a.top_p[b] : 1.0f;
    r.use_k = r.k != 0u && r.k < a.vocab;
    r.use_p = r.p < 1.0f;
    return r;
}

/* With the rank of the row's largest logit, and the least that is known (+inf:
 * none).  Where the largest is +inf, logits are taken as 0 there and -inf elsewhere
 * (value_of). */
__device__ __forceinline__ void set_top(Row &r, u64 max_rank, float least) {
    r.top = of_key((u32)(max_rank >> IDX_BITS));
    r.inf = r.top == INFINITY;
    if (r.inf) r.top = 0.0f;
    const float span = r.top - least;
    if (!r.inf && span > 0.0f && span * r.scale < (float)(BINS / 2u)) {
        r.scale = fminf(((float)BINS - 1.5f) / span, 1e30f);
        r.most = (float)(BINS - 2u);
    }
    /* below: lighter than min_p by more than the roundings here (2^-20 of the distance, and of the logit) */
    const float far = r.cut;
    r.cut = r.top + far - 1e-6f * (fabsf(r.top) + fabsf(far));
    if (!(r.cut > -INFINITY)) r.cut = -INFINITY;
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

/* The least of the lane's logits that are not -inf, and `least`. */
__device__ __forceinline__ float least_of(const float *x, float least) {
#pragma unroll
    for (u32 e = 0; e < E; ++e) least = fminf(least, x[e] > -INFINITY ? x[e] : INFINITY);
    return least;
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
    return wave_max_dpp(m);
}

__device__ __forceinline__ float value_of(const Row &r, float x) {
    return !r.inf ? x : x == INFINITY ? 0.0f : -INFINITY;
}

/* f over the whole row's values from `least` on, by all threads. */
template <bool F32, typename F>
__device__ __forceinline__ void row_values(const void *row, u32 vocab, float least, F &&f) {
    each_step<F32, ROW_U>(row, vocab, threadIdx.x >> 6, (vocab + STEP - 1u) / STEP, WAVES, [&](u32 s, const float *x) { values_from(least, s, x, f); });
}

/* Sum and maximum of all lanes (all of them active), as wave_sum. */
__device__ __forceinline__ u64 wave_sum64(u64 v) {
    v += dpp64<0xB1>(v);
    v += dpp64<0x4E>(v);
    v += dpp64<0x141>(v);
    v += dpp64<0x140>(v);
    return (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
}
__device__ __forceinline__ u64 wave_max64(u64 v) {
    v = max(v, dpp64<0xB1>(v));
    v = max(v, dpp64<0x4E>(v));
    v = max(v, dpp64<0x141>(v));
    v = max(v, dpp64<0x140>(v));
    return max(max(lane64(v, 0), lane64(v, 16)), max(lane64(v, 32), lane64(v, 48)));
}

struct Shared {
    double tab[TAB];
    u64 weight[BINS];
    u32 count[BINS];
    u64 list[LIST];
    u32 tops[TOPS], place[LIST], start[LIST];
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

/* The ranks of the first n threads, largest first.  Few are counted against each
 * other, by all threads.  More go to LIST buckets of equal width first, and are
 * counted within them (equal logits share a bucket, at worst all of them): the
 * launch of 192 rows' lists took 14.8 us with a bitonic sort, 11.1 so. */
__device__ __forceinline__ u64 sorted(u64 rank, u32 n, Shared &sm) {
    const u32 t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    u64 *buf = sm.list;
    u32 *place = sm.place;
    if (n <= FEW) {
        const u32 size = n <= 64u ? 64u : FEW, parts = LIST / size, part = t / size, e = t % size;
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
    } else {
        const float x = of_key((u32)(rank >> IDX_BITS));
        const bool in = t < n, finite = in && x > -INFINITY;
        const float hi = wave_max_dpp(finite ? x : -INFINITY), lo = -wave_max_dpp(finite ? -x : -INFINITY);
        float *ends = (float *)sm.red; /* [WAVES][2] */
        if (lane == 0u) ends[2u * wave] = hi, ends[2u * wave + 1u] = -lo;
        place[t] = 0u;
        __syncthreads();
        const float end = wave_max_dpp(lane < 2u * WAVES && lane % 2u == 0u ? ends[lane] : -INFINITY);
        const float low = -wave_max_dpp(lane < 2u * WAVES && lane % 2u == 1u ? ends[lane] : -INFINITY);
        const float scale = end > low ? ((float)LIST - 0.5f) / (end - low) : 0.0f;
        const u32 bucket = x == end ? 0u : (u32)fminf((end - x) * scale, (float)(LIST - 1u)); /* -inf: the last */
        u32 index = 0;
        if (in) index = atomicAdd(&place[bucket], 1u);
        __syncthreads();
        u64 all;
        sm.start[t] = (u32)block_before(place[t], sm.red, all);
        __syncthreads();
        u32 at = 0, many = 0;
        if (in) {
            at = sm.start[bucket];
            many = place[bucket];
            buf[at + index] = rank;
        }
        __syncthreads();
        u32 before = at;
        for (u32 i = 0; i < many; ++i) before += buf[at + i] > rank ? 1u : 0u;
        __syncthreads();
        if (in) buf[before] = rank;
    }
    __syncthreads();
    rank = t < n ? buf[t] : 0ull;
    __syncthreads();
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
 * thread, with its weight), in front of which base_n values and base_w units
 * stand; all: units of all values that top-p sums.  last: how many of the
 * listed ones are kept. */
__device__ __forceinline__ u64 cut(const Row &r, u64 rank, double wd, u32 n, bool use_k, u64 base_n, u64 base_w, u64 all, u64 *red, u64 *out, u32 &last) {
    const u32 t = threadIdx.x;
    const bool in = t < n;
    const u64 bn = base_n + t, w = in ? units(wd) : 0ull;
    const bool in_k = in && (!use_k || bn < r.k);
    u64 sum;
    const u64 bw = base_w + block_before(in_k ? w : 0ull, red, sum);
    const double target = (double)r.p * (double)(use_k ? sum : all);
    const bool kept = in_k && (!r.use_p || bn == 0ull || (double)bw < target);
    last = (u32)__syncthreads_count(kept);
    if (t + 1u == last) *out = rank;
    __syncthreads();
    return *out;
}

__device__ __forceinline__ double target_of(const uocr_sample_args &a, u32 b, u64 all) {
    const float u = a.uniform[b];
    return (double)(u > 0.0f ? fminf(u, 0.99999994f) : 0.0f) * (double)all;
}

/* The token, where the n values of largest rank (one a thread) are all that
 * top-k and top-p keep: in front of each stands the weight of lower ids, summed
 * as `sorted` counts: over all of few, else by buckets of ids. */
__device__ __forceinline__ void pick_listed(const uocr_sample_args &a, u32 b, const Row &r, u64 rank, double wd, u32 n, Shared &sm) {
    const u32 t = threadIdx.x, id = IDX_MASK - (u32)(rank & IDX_MASK);
    const u64 w = t < n && wd >= r.min_w ? units(wd) : 0ull;
    const u32 bits = 32u - (u32)__builtin_clz(a.vocab | 1u), bucket = id >> (bits > 10u ? bits - 10u : 0u);
    u32 *count = sm.place, *ids = sm.count;
    u64 *sums = sm.weight, *ws = sm.weight + LIST;
    static_assert(LIST == 1024 && BINS >= 2 * LIST, "buckets of ten bits");
    count[t] = 0u;
    sums[t] = 0ull;
    u64 all, sum = 0;
    if (n <= FEW) {
        const u32 size = n <= 64u ? 64u : FEW, parts = LIST / size, part = t / size, e = t % size;
        if (t < n) ids[t] = id, ws[t] = w;
        (void)block_before(w, sm.red, all);
        if (e < n) {
            const u32 mine = ids[e], i1 = n * (part + 1u) / parts;
            u64 here = 0;
#pragma unroll 4
            for (u32 i = n * part / parts; i < i1; ++i) here += ids[i] < mine ? ws[i] : 0ull;
            if (here != 0ull) atomicAdd(&sums[e], here);
        }
        __syncthreads();
        sum = sums[t];
    } else {
        __syncthreads();
        u32 index = 0;
        if (w != 0ull) {
            index = atomicAdd(&count[bucket], 1u);
            atomicAdd(&sums[bucket], w);
        }
        __syncthreads();
        u64 kept;
        const u64 in_front = block_before(sums[t], sm.red, all);
        sm.start[t] = (u32)block_before(count[t], sm.red2, kept);
        sums[t] = in_front;
        __syncthreads();
        u32 at = 0, many = 0;
        if (w != 0ull) {
            at = sm.start[bucket];
            many = count[bucket];
            sum = sums[bucket];
            ids[at + index] = id;
            ws[at + index] = w;
        }
        __syncthreads();
        for (u32 i = 0; i < many; ++i) sum += ids[at + i] < id ? ws[at + i] : 0ull;
    }
    const double target = target_of(a, b, all);
    if (w != 0ull && !((double)sum > target) && (double)(sum + w) > target) {
        a.tokens[b] = (int32_t)id;
        if (a.probs != nullptr) a.probs[b] = (float)((double)w / (double)all);
    }
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
    const u64 rank = sorted(t < n ? sm.list[t] : 0ull, n, sm);
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

/* A row that is decided by its largest logit. */
__device__ __forceinline__ void greedy(const uocr_sample_args &a, u32 b, u64 max_rank) {
    a.tokens[b] = max_rank == 0ull ? 0 : (int32_t)(IDX_MASK - (u32)(max_rank & IDX_MASK));
    if (a.probs != nullptr) a.probs[b] = max_rank == 0ull ? 0.0f : 1.0f;
}

/* The rank of the block's largest logit, and the least of its lanes'. */
__device__ __forceinline__ u64 largest(float best, u32 best_id, float &least, u64 *red, u64 *red2) {
    u64 rank = wave_max64(best_id == 0xffffffffu ? 0ull : rank_of(best, best_id));
    least = -wave_max_dpp(-least);
    if ((threadIdx.x & 63u) == 0u) red[threadIdx.x >> 6] = rank, red2[threadIdx.x >> 6] = __float_as_uint(least);
    __syncthreads();
    for (u32 i = 0; i < blockDim.x / 64u; ++i) {
        rank = red[i] > rank ? red[i] : rank;
        least = fminf(least, __uint_as_float((u32)red2[i]));
    }
    __syncthreads();
    return rank;
}

/* What is kept: logits above `least`, and of those equal to it the ids up to
 * `id`, if their weights are not below min_p.  raw: `least` as it stands in the
 * row (with +inf logits, which are taken as 0, those alone). */
struct Keep {
    float least, raw;
    u32 id;
};
__device__ __forceinline__ Keep keep_from(const Row &r, u64 thr) {
    Keep k = {r.cut, 0.0f, IDX_MASK};
    const float last = of_key((u32)(thr >> IDX_BITS));
    if (thr != 0ull && last >= r.cut) k.least = last, k.id = IDX_MASK - (u32)(thr & IDX_MASK);
    k.raw = r.inf ? INFINITY : k.least;
    return k;
}
__device__ __forceinline__ bool is_kept(const Keep &k, float x, u32 id) {
    return (x > k.least) | ((x == k.least) & (id <= k.id)); /* no branches */
}

/* Units that a value brings to the kept sum. */
__device__ __forceinline__ u64 kept_units(const Row &r, const double *tab, const Keep &k, float raw, u32 id) {
    const float x = value_of(r, raw);
    if (!is_kept(k, x, id)) return 0ull;
    const double w = weight(r, tab, x);
    return w >= r.min_w ? units(w) : 0ull;
}
/* Those of the lane's values, of ids from id0 on.  Without branches: where few
 * lanes have one the step is one of few, where many have one it takes half the
 * instructions.  A loop: the code of a kernel is fetched by every CU. */
__device__ __forceinline__ u64 lane_units(const Row &r, const double *tab, const Keep &k, u32 id0, const float *values) {
    float x[E];
#pragma unroll
    for (u32 e = 0; e < E; ++e) x[e] = values[e];
    if (r.inf) {
#pragma unroll
        for (u32 e = 0; e < E; ++e) x[e] = value_of(r, x[e]);
    }
    u64 sum = 0;
#pragma unroll 1
    for (u32 e = 0; e < E; e += ILP) {
#pragma unroll
        for (u32 i = 0; i < ILP; ++i) {
            const double w = weight(r, tab, is_kept(k, x[i], id0 + e + i) ? x[i] : -INFINITY);
            sum += units(w >= r.min_w ? w : 0.0);
        }
#pragma unroll
        for (u32 i = 0; i + ILP < E; ++i) x[i] = x[i + ILP];
    }
    return sum;
}

/* The lane's values into the histogram (the last bin's have no weight): counts
 * from `counted` bins, weights for top-p.  Without EXACT, NaN and -inf of a flat
 * row go to the bin before the last, where their weights and places at the end
 * change nothing. */
template <bool EXACT>
__device__ __forceinline__ void into_bins(const Row &r, const double *tab, const float *x, u32 counted, u32 *counts, u64 *weights) {
    float v[E];
#pragma unroll
    for (u32 e = 0; e < E; ++e) v[e] = x[e];
    if (r.inf) {
#pragma unroll
        for (u32 e = 0; e < E; ++e) v[e] = value_of(r, v[e]);
    }
#pragma unroll 1
    for (u32 e = 0; e < E; e += ILP) {
        u32 bin[ILP];
        u64 w[ILP];
#pragma unroll
        for (u32 i = 0; i < ILP; ++i) bin[i] = EXACT ? bin_of(r, v[i]) : v[i] == r.top ? 0u : (u32)fminf((r.top - v[i]) * r.scale, r.most);
        if (r.use_p) {
#pragma unroll
            for (u32 i = 0; i < ILP; ++i) w[i] = units(weight(r, tab, v[i]));
#pragma unroll
            for (u32 i = 0; i < ILP; ++i)
                if (bin[i] != BINS - 1u) atomicAdd(&weights[bin[i]], w[i]);
        }
#pragma unroll
        for (u32 i = 0; i < ILP; ++i)
            if (bin[i] < counted) atomicAdd(&counts[bin[i]], 1u);
#pragma unroll
        for (u32 i = 0; i + ILP < E; ++i) v[i] = v[i + ILP];
    }
}

/* The first id whose running sum of kept units is over the target, in the step
 * that `sum` stands in front of; by one wavefront: its lane by the steps' order,
 * then that lane's values by a lane each.  Returns whether it is there, and what
 * stands in front of the next values. */
template <bool F32>
__device__ __forceinline__ bool pick(const uocr_sample_args &a, u32 b, const Row &r, const double *tab, const Keep &k, const void *row, u32 step, double target, u64 all, u64 &sum) {
    const u32 lane = threadIdx.x & 63u, id0 = step * STEP + lane * E;
    float x[E];
    lane_load<F32, false>(row, min(id0, a.vocab), a.vocab, x);
    const u64 s = lane_units(r, tab, k, id0, x);
    const u64 at = sum + wave_before(s);
    const u64 found = __ballot(s != 0ull && !((double)at > target) && (double)(at + s) > target);
    sum = lane64(at + s, 63);
    if (found == 0ull) return false;
    const u32 from = (u32)__builtin_ctzll(found), id = step * STEP + from * E + lane;
    u64 w = 0;
    if (lane < E && id < a.vocab) w = kept_units(r, tab, k, F32 ? ((const float *)row)[id] : (float)((const _Float16 *)row)[id], id);
    const u64 before = lane64(at, (int)from) + wave_before(w);
    if (w != 0ull && !((double)before > target) && (double)(before + w) > target) {
        a.tokens[b] = (int32_t)id;
        if (a.probs != nullptr) a.probs[b] = (float)((double)w / (double)all);
    }
    return true;
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
    float least = INFINITY;
    u32 best_id = 0xffffffffu;
    sm.tops[t % TOPS] = 0u;
    __syncthreads();
    each_step<F32, ROW_U>(row, vocab, wave, steps, WAVES, [&](u32 s, const float *x) {
        const u32 top = key_of(step_largest(s, x, best, best_id));
        if (s == wave) least = least_of(x, least); /* of the wavefront's first step */
        if (lane == 0u) sm.tops[s % TOPS] = max(sm.tops[s % TOPS], top); /* a group's steps are one wavefront's: TOPS is a multiple of WAVES */
    });
    const u64 max_rank = largest(best, best_id, least, sm.red, sm.red2);
    Row r = settings_of(a, b, shift);
    if (max_rank == 0ull || !r.hot) {
        if (t == 0u) greedy(a, b, max_rank);
        return;
    }
    set_top(r, max_rank, least);
    fill_table(sm.tab, r.shift);
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
        if (found) {
            const u64 rank = sorted(t < n ? sm.list[t] : 0ull, n, sm);
            const double wd = weight(r, sm.tab, of_key((u32)(rank >> IDX_BITS)));
            u32 last;
            thr = cut(r, rank, wd, n, true, 0ull, 0ull, 0ull, sm.red, &sm.out[0], last);
            pick_listed(a, b, r, rank, wd, last, sm);
            return;
        }
        __syncthreads();
    }
    if (!found && (r.use_k || r.use_p)) {
        for (u32 i = t; i < BINS; i += NT) sm.weight[i] = 0ull, sm.count[i] = 0u;
        __syncthreads();
        each_step<F32, ROW_U>(row, vocab, wave, steps, WAVES, [&](u32, const float *x) { into_bins<true>(r, sm.tab, x, BINS - 1u, sm.count, sm.weight); });
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
    const Keep keep = keep_from(r, thr);
    u64 *sums = sm.weight; /* [WAVES][GROUPS] */
    __syncthreads();
    sums[t] = 0ull;
    __syncthreads();
    each_step<F32, ROW_U>(row, vocab, min(wave * run, steps), min(wave * run + run, steps), 1u, [&](u32 s, const float *x) {
        if (!__any(largest_of(x) >= keep.raw)) return;
        const u64 sum = wave_sum64(lane_units(r, sm.tab, keep, s * STEP + lane * E, x));
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
            if (w * run + i < steps && pick<F32>(a, b, r, sm.tab, keep, row, w * run + i, target, all, sum)) break;
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

/* What is known of a row before its list is made: whether its kept set ends
 * (any), in the values from `floor` on that lie in the bins first .. last (all
 * for a bounded row), in front of which base_n values and base_w units stand;
 * all_w: units of all values; crowded: more than LIST values, as far as they
 * were counted. */
struct Found {
    u64 base_n, base_w, all_w;
    u32 first, last;
    float floor;
    bool any, use_k, crowded;
};

/* What the launches of a row leave for each other, in the workspace. */
struct Plan {
    uocr_sample_args a;
    u32 shift, steps, chunks;      /* of a row; chunks: of the first launch */
    u32 parts, run;                /* of this launch, [parts][rows] blocks: steps of each */
    Row *settings;                 /* [rows] */
    u64 *max_rank;                 /* [rows][chunks] */
    float *least;                  /* [rows][chunks] */
    u32 *tops;                     /* [rows][steps]: keys of the steps' largest logits */
    u64 *weight;                   /* [rows][BINS] */
    u32 *count;                    /* [rows][BINS] */
    u64 *list;                     /* [rows][LIST] */
    u32 *n;                        /* [rows]: the list's length so far */
    Found *found;                  /* [rows] */
    u64 *thr;                      /* [rows]: the rank that ends the kept set, or DONE */
    u64 *sums;                     /* [rows][steps] */
    u32 *arrived;                  /* [rows]: blocks that have written their sums */
    bool cut;                      /* some row has top-k or top-p */
};

/* The lane's values of a step, as they stand in memory.  The row's last lanes,
 * whose values may not be E, begin at its last E ones instead. */
template <bool F32>
struct Raw {
    uint4 w[F32 ? 2 : 1];
};
__device__ __forceinline__ u32 lane_id0(u32 step, u32 vocab) { return min(step * STEP + (threadIdx.x & 63u) * E, vocab - E); }
template <bool F32>
__device__ __forceinline__ Raw<F32> raw_load(const void *row, u32 id0) {
    Raw<F32> q;
    if constexpr (F32) {
        const f32x4_any4 a = *(const f32x4_any4 *)((const float *)row + id0), b = *(const f32x4_any4 *)((const float *)row + id0 + 4);
        q.w[0] = __builtin_bit_cast(uint4, a);
        q.w[1] = __builtin_bit_cast(uint4, b);
    } else {
        q.w[0] = load_any((const uint16_t *)row + id0);
    }
    return q;
}
/* NaN, which takes part in nothing, for those that are not of the lane. */
template <bool F32>
__device__ __forceinline__ void raw_values(const Raw<F32> &q, u32 step, u32 vocab, float *x) {
    if constexpr (F32) {
        const uint4 a = q.w[0], b = q.w[1];
        const u32 v[E] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (u32 e = 0; e < E; ++e) x[e] = __uint_as_float(v[e]);
    } else {
        union {
            uint4 u;
            _Float16 h[E];
        } v;
        v.u = q.w[0];
#pragma unroll
        for (u32 e = 0; e < E; ++e) x[e] = (float)v.h[e];
    }
    if ((step + 1u) * STEP > vocab) {
        const u32 first = step * STEP + (threadIdx.x & 63u) * E - lane_id0(step, vocab);
#pragma unroll
        for (u32 e = 0; e < E; ++e) x[e] = e < first ? __builtin_nanf("") : x[e];
    }
}

/* The steps of a wavefront (every CWAVES-th of its chunk's), a lane each.  The
 * first 64 are asked for their largest logits before anything else is known of
 * the row: the launches below are chains of loads that wait for each other. */
struct Steps {
    const u32 *tops;
    u32 s0, s1, key;
};
__device__ __forceinline__ Steps steps_of(const Plan &g, u32 b, u32 chunk) {
    Steps c;
    c.tops = g.tops + (u64)b * g.steps;
    c.s0 = chunk * g.run + (u32)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    c.s1 = min(chunk * g.run + g.run, g.steps);
    const u32 mine = c.s0 + CWAVES * (threadIdx.x & 63u);
    c.key = mine < c.s1 ? c.tops[mine] : 0u;
    return c;
}

/* f(step, first id, values) for the steps that hold a value from `least` on,
 * four steps' loads at a time; skip(step) for the others, by a lane each. */
template <bool F32, typename F, typename S>
__device__ __forceinline__ void chunk_steps(const Plan &g, const void *row, const Steps &c, float least, F &&f, S &&skip) {
    constexpr u32 U = 4;
    const u32 lane = threadIdx.x & 63u, vocab = g.a.vocab, key = key_of(least), s1 = c.s1;
#pragma unroll 1
    for (u32 first = c.s0; first < s1; first += 64u * CWAVES) {
        const u32 mine = first + CWAVES * lane;
        const bool in = mine < s1, look = in && (first == c.s0 ? c.key : c.tops[mine]) >= key;
        if (in && !look) skip(mine);
        u64 left = __ballot(look);
#pragma unroll 1
        while (left != 0ull) {
            u32 s[U], n = 0;
            Raw<F32> q[U];
#pragma unroll
            for (u32 u = 0; u < U; ++u) {
                s[u] = left != 0ull ? first + CWAVES * (u32)__builtin_ctzll(left) : s[u > 0u ? u - 1u : 0u]; /* the last one again */
                n += left != 0ull ? 1u : 0u;
                left &= left - 1ull;
                q[u] = raw_load<F32>(row, lane_id0(s[u], vocab));
            }
#pragma unroll 1
            for (u32 u = 0; u < n; ++u) {
                float x[E];
                raw_values<F32>(q[0], s[0], vocab, x);
                f(s[0], lane_id0(s[0], vocab), x);
#pragma unroll
                for (u32 i = 0; i + 1u < U; ++i) q[i] = q[i + 1u], s[i] = s[i + 1u];
            }
        }
    }
}
/* g(logit, id) for those values, up to `most`. */
template <bool F32, typename G>
__device__ __forceinline__ void chunk_values(const Plan &g, const void *row, const Steps &c, float least, float most, G &&each) {
    chunk_steps<F32>(g, row, c, least, [&](u32, u32 id0, const float *x) {
        u32 here = 0;
#pragma unroll
        for (u32 e = 0; e < E; ++e) here |= ((x[e] >= least) & (x[e] <= most)) ? 1u << e : 0u;
        while (here != 0u) {
            const u32 e = (u32)__builtin_ctz(here);
            here &= here - 1u;
            const float a0 = e & 1u ? x[1] : x[0], a1 = e & 1u ? x[3] : x[2], a2 = e & 1u ? x[5] : x[4], a3 = e & 1u ? x[7] : x[6];
            const float c0 = e & 2u ? a1 : a0, c1 = e & 2u ? a3 : a2;
            each(e & 4u ? c1 : c0, id0 + e);
        }
    }, [](u32) {});
}

/* 1: the steps' and the chunk's largest logit; the row's histogram is cleared. */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_max(Plan g) {
    __shared__ u64 red[CWAVES], red2[CWAVES];
    const u32 b = blockIdx.x, chunk = blockIdx.y, lane = threadIdx.x & 63u;
    if (g.cut)
        for (u32 i = chunk * CT + threadIdx.x; i < BINS; i += CT * g.parts) g.weight[(u64)b * BINS + i] = 0ull, g.count[(u64)b * BINS + i] = 0u;
    if (chunk == 0u && threadIdx.x == 0u) {
        g.settings[b] = settings_of(g.a, b, g.shift);
        g.n[b] = g.arrived[b] = 0u;
        g.found[b] = Found{};
    }
    const void *row = row_at<F32>(g.a, b);
    float best = -INFINITY;
    float least = INFINITY;
    u32 best_id = 0xffffffffu;
    const u32 s0 = chunk * g.run + (u32)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    each_step<F32, 4>(row, g.a.vocab, s0, min(chunk * g.run + g.run, g.steps), CWAVES, [&](u32 s, const float *x) {
        const float top = step_largest(s, x, best, best_id);
        if (s == s0) least = least_of(x, least); /* of the wavefront's first step */
        if (lane == 0u) g.tops[(u64)b * g.steps + s] = key_of(top);
    });
    const u64 rank = largest(best, best_id, least, red, red2);
    if (threadIdx.x == 0u) g.max_rank[(u64)b * g.chunks + chunk] = rank, g.least[(u64)b * g.chunks + chunk] = least;
}

__device__ __forceinline__ u64 row_max(const Plan &g, u32 b) {
    return wave_max64((threadIdx.x & 63u) < g.chunks ? g.max_rank[(u64)b * g.chunks + (threadIdx.x & 63u)] : 0ull);
}
__device__ __forceinline__ float row_least(const Plan &g, u32 b) {
    return -wave_max_dpp((threadIdx.x & 63u) < g.chunks ? -g.least[(u64)b * g.chunks + (threadIdx.x & 63u)] : -INFINITY);
}

/* Bins whose values are counted: all for top-k; for top-p alone only so many as a
 * list might hold. */
__device__ __forceinline__ u32 counted_bins(const Row &r) {
    return r.use_k ? BINS - 1u : (u32)fminf(r.near * r.scale, (float)(BINS - 1u));
}

/* Below: in bins behind `last`, as a comparison tells (three bins' margin for
 * their roundings). */
__device__ __forceinline__ float floor_of(const Row &r, u32 last) {
    const float floor = r.top - ((float)last + 3.0f) / r.scale;
    return floor > -INFINITY && !r.inf && !(last >= BINS - 2u && r.most < (float)(BINS - 1u)) ? floor : -INFINITY;
}
/* Above: in bins before `first`. */
__device__ __forceinline__ float ceiling_of(const Row &r, u32 first) {
    const float ceiling = r.top - ((float)first - 3.0f) / r.scale;
    return first > 3u && !r.inf && ceiling == ceiling ? ceiling : INFINITY;
}

__device__ __forceinline__ u64 agent_load(const u64 *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

/* Whether this block is the last of its row to come here; what the others have
 * written (with agent scope) is there for it. */
__device__ __forceinline__ bool comes_last(u32 *count, u32 parts, u32 *shared) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (parts == 1u) return true;
    if (threadIdx.x == 0u) *shared = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const bool last = *shared == parts - 1u;
    asm volatile("" ::: "memory");
    return last;
}

/* The bins whose values decide, from the row's histogram; by each block for
 * itself (done once, by the last block to add to it, it took 3 us more). */
__device__ __forceinline__ Found find_bins(const Plan &g, u32 b, const Row &r, u64 *red, u64 *red2, u64 *out) {
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
    Found f = {};
    u64 all_n;
    u64 nb = block_before(sn, red, all_n), wb = block_before(sw, red2, f.all_w);
    f.use_k = r.use_k && (u64)r.k < all_n;
    f.any = f.use_k || r.use_p;
    if (!f.any) return f; /* all are kept */
    const double target = (double)r.p * (double)f.all_w;
#pragma unroll
    for (u32 i = 0; i < PER; ++i) {
        const bool here = f.use_k ? nb < r.k && r.k <= nb + n[i] : w[i] != 0ull && (!(r.p > 0.0f) ? wb == 0ull : (double)wb < target && !((double)(wb + w[i]) < target));
        if (here) out[0] = PER * t + i, out[1] = nb, out[2] = wb, out[3] = n[i];
        nb += n[i];
        wb += w[i];
    }
    __syncthreads();
    f.last = (u32)out[0];
    f.floor = floor_of(r, f.last);
    /* With both, top-p decides within top-k's values: all of them are looked at.  As many as a list holds are listed from
     * the first on: then nothing else needs to be looked at for the token. */
    const bool known = f.last < counted_bins(r), all = (f.use_k && r.use_p) || (known && out[1] + out[3] <= LIST);
    f.first = all ? 0u : f.last;
    f.base_n = all ? 0ull : out[1];
    f.base_w = all ? 0ull : out[2];
    f.crowded = known && (all ? out[1] + out[3] : out[3]) > LIST;
    return f;
}

/* 2: the histogram, in LDS and from there into the row's.  A bounded row only
 * needs its bound. */
template <bool F32>
__global__ __launch_bounds__(CT, F32 ? 5 : 7) void k_sample_bins(Plan g) {
    __shared__ double tab[TAB];
    __shared__ u64 weights[BINS];
    __shared__ u32 counts[BINS];
    const u32 b = blockIdx.x, chunk = blockIdx.y, t = threadIdx.x, groups = min(g.steps, TOPS);
    const Steps mine = steps_of(g, b, chunk);
    Row r = g.settings[b];
    fill_table(tab, g.shift);
    if (!r.hot || (!r.use_k && !r.use_p)) return;
    const bool listed = bounded(r, groups);
    if (listed && (chunk != 0u || t >= 64u)) return;
    const u64 max_rank = row_max(g, b);
    const float least = listed ? INFINITY : row_least(g, b);
    if (max_rank == 0ull) return;
    set_top(r, max_rank, least);
    if (listed) {
        u32 tops[TOPS / 64] = {};
        for (u32 s0 = 0; s0 < g.steps; s0 += TOPS) {
#pragma unroll
            for (u32 i = 0; i < TOPS / 64; ++i) {
                const u32 s = s0 + 64u * i + t;
                if (s < g.steps) tops[i] = max(tops[i], g.tops[(u64)b * g.steps + s]);
            }
        }
        Found f = {};
        f.any = f.use_k = true;
        f.last = BINS;
        f.floor = kth_largest(tops, groups, r.k);
        if (t == 0u) g.found[b] = f;
        return;
    }
    for (u32 i = t; i < BINS; i += CT) weights[i] = 0ull, counts[i] = 0u;
    __syncthreads();
    const u32 counted = counted_bins(r);
    chunk_steps<F32>(g, row_at<F32>(g.a, b), mine, floor_of(r, BINS - 1u), [&](u32, u32, const float *x) { into_bins<false>(r, tab, x, counted, counts, weights); }, [](u32) {});
    __syncthreads();
    for (u32 i = t; i < BINS; i += CT) {
        if (counts[i] != 0u) atomicAdd(&g.count[(u64)b * BINS + i], counts[i]);
        if (weights[i] != 0ull) atomicAdd(&g.weight[(u64)b * BINS + i], weights[i]);
    }
}

/* 3: the values that decide, listed in any order. */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_list(Plan g) {
    __shared__ u64 red[CWAVES], red2[CWAVES], out[4], list[LIST];
    __shared__ u32 n, first;
    const u32 b = blockIdx.x, chunk = blockIdx.y, t = threadIdx.x;
    const Steps mine = steps_of(g, b, chunk);
    Row r = g.settings[b];
    if (!r.hot || (!r.use_k && !r.use_p)) return;
    const bool listed = bounded(r, min(g.steps, TOPS));
    const u64 max_rank = row_max(g, b);
    const float least = listed ? INFINITY : row_least(g, b);
    if (max_rank == 0ull) return;
    set_top(r, max_rank, least);
    if (t == 0u) n = 0u;
    Found f;
    if (listed) {
        f = g.found[b];
        __syncthreads();
    } else {
        f = find_bins(g, b, r, red, red2, out);
        if (chunk == 0u && t == 0u) g.found[b] = f;
        if (!f.any || f.crowded) return;
    }
    chunk_values<F32>(g, row_at<F32>(g.a, b), mine, f.floor, ceiling_of(r, f.first), [&](float raw, u32 id) {
        const float x = value_of(r, raw);
        const u32 i = bin_of(r, x);
        if (f.last != BINS && (i < f.first || i > f.last)) return;
        const u32 at = atomicAdd(&n, 1u);
        if (at < LIST) list[at] = rank_of(x, id);
    });
    __syncthreads();
    if (n == 0u) return;
    if (t == 0u) first = atomicAdd(&g.n[b], n); /* of a crowded list: past LIST */
    __syncthreads();
    for (u32 i = t; i < min(n, LIST); i += CT)
        if (first + i < LIST) g.list[(u64)b * LIST + first + i] = list[i];
}

/* 4: the rank that ends the kept set: the listed values in order, what stands in
 * front of each, and the last one that is kept.  Where all of the kept set is
 * listed, its token too; rows whose lists ran over are done from
 * their beginning. */
template <bool F32>
__global__ __launch_bounds__(NT) void k_sample_cut(Plan g) {
    static_assert(LIST == NT, "a listed value for each thread");
    __shared__ Shared sm;
    const u32 b = blockIdx.x, t = threadIdx.x;
    Row r = g.settings[b];
    const Found f = g.found[b];
    const u32 n = g.n[b];
    const u64 max_rank = row_max(g, b), listed = g.list[(u64)b * LIST + t];
    if (max_rank == 0ull || !r.hot) return;
    set_top(r, max_rank, -INFINITY); /* no bins here */
    u64 thr = 0;
    if (f.any) {
        if (f.crowded || n > LIST) {
            whole_row<F32>(g.a, b, row_at<F32>(g.a, b), g.shift, sm);
            thr = DONE;
        } else {
            fill_table(sm.tab, r.shift);
            __syncthreads();
            const u64 rank = sorted(t < n ? listed : 0ull, n, sm);
            const double wd = weight(r, sm.tab, of_key((u32)(rank >> IDX_BITS)));
            u32 last;
            thr = cut(r, rank, wd, n, f.use_k, f.base_n, f.base_w, f.all_w, sm.red, &sm.out[0], last);
            if (f.base_n == 0ull) {
                pick_listed(g.a, b, r, rank, wd, last, sm);
                thr = DONE;
            }
        }
    }
    if (t == 0u) g.thr[b] = thr;
}

/* 5: the kept units of each step, from block to block with agent scope; the last
 * block of a row finds the step, and in it the token. */
template <bool F32>
__global__ __launch_bounds__(CT) void k_sample_sums(Plan g) {
    __shared__ double tab[TAB];
    __shared__ u64 red[CWAVES], at[2];
    __shared__ u32 arrived;
    const u32 b = blockIdx.x, chunk = blockIdx.y, t = threadIdx.x;
    const Steps mine_steps = steps_of(g, b, chunk);
    Row r = g.settings[b];
    fill_table(tab, g.shift);
    const u64 max_rank = row_max(g, b), thr = g.cut ? g.thr[b] : 0ull;
    if (max_rank == 0ull || !r.hot) {
        if (chunk == 0u && t == 0u) greedy(g.a, b, max_rank);
        return;
    }
    if (thr == DONE) return;
    set_top(r, max_rank, -INFINITY); /* no bins here */
    const void *row = row_at<F32>(g.a, b);
    __syncthreads();
    const Keep keep = keep_from(r, thr);
    u64 *sums = g.sums + (u64)b * g.steps;
    auto put = [&](u32 s, u64 sum) { __hip_atomic_store(sums + s, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    chunk_steps<F32>(g, row, mine_steps, keep.raw, [&](u32 s, u32 id0, const float *x) {
        const u64 sum = wave_sum64(lane_units(r, tab, keep, id0, x));
        if ((t & 63u) == 0u) put(s, sum);
    }, [&](u32 s) { put(s, 0ull); });
    if (!comes_last(g.arrived + b, g.parts, &arrived)) return;
    const u32 per = (g.steps + CT - 1u) / CT, s0 = min(t * per, g.steps), s1 = min(s0 + per, g.steps);
    u64 mine = 0;
    for (u32 s = s0; s < s1; ++s) mine += agent_load(sums + s);
    u64 all;
    const u64 before = block_before(mine, red, all);
    const double target = target_of(g.a, b, all);
    if (mine != 0ull && !((double)before > target) && (double)(before + mine) > target) at[0] = s0, at[1] = before;
    __syncthreads();
    if (t >= 64u) return;
    u64 sum = at[1];
    for (u32 s = (u32)at[0]; s < g.steps; ++s)
        if (pick<F32>(g.a, b, r, tab, keep, row, s, target, all, sum)) break;
}

u32 shift_of(u32 vocab) {
    u32 bits = 0;
    while ((1u << bits) < vocab) ++bits;
    return 62u - bits < 50u ? 62u - bits : 50u;
}

/* Rows of up to ONE_BLOCK tokens are done by a block each, in one launch, and
 * with MANY_ROWS or more up to twice that: us by one launch and by several, fp16,
 * top-k alone and top-p alone, were 16 and 25 against 20 and 25 for 1 row of
 * 16,000, 24 and 29 against 33 and 43 for 192; 19 and 36 against 21 and 25 for 1
 * of 32,000, 33 and 44 against 29 and 41 for 64, 34 and 45 against 39 and 56 for
 * 192; 51 and 74 against 46 and 74 for 192 of 64,000. */
constexpr u32 ONE_BLOCK = 16384, MANY_ROWS = 128;
bool by_one_block(u32 rows, u32 vocab) { return vocab <= (rows < MANY_ROWS ? ONE_BLOCK : 2u * ONE_BLOCK); }

/* Blocks of a launch, all rows: where all values take little each, more of them
 * only have their own beginnings to pay for; where some rows' values take an
 * exponential and atomics each and others' nothing, the rows are cut finer.  192
 * mixed rows of 129,280 fp16 took 88.7 us so, 91.1 and 91.7 with 1,536 and 3,000
 * for the heavy ones (80.5 since the lists are ordered by buckets). */
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
    g.settings = (Row *)take((size_t)rows * sizeof(Row));
    g.max_rank = (u64 *)take((size_t)rows * MAX_CHUNKS * 8u);
    g.least = (float *)take((size_t)rows * MAX_CHUNKS * 4u);
    g.tops = (u32 *)take((size_t)rows * g.steps * 4u);
    g.weight = (u64 *)take((size_t)rows * BINS * 8u);
    g.count = (u32 *)take((size_t)rows * BINS * 4u);
    g.list = (u64 *)take((size_t)rows * LIST * 8u);
    g.n = (u32 *)take((size_t)rows * 4u);
    g.found = (Found *)take((size_t)rows * sizeof(Found));
    g.thr = (u64 *)take((size_t)rows * 8u);
    g.sums = (u64 *)take((size_t)rows * g.steps * 8u);
    g.arrived = (u32 *)take((size_t)rows * 4u);
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
        hipLaunchKernelGGL(kernel, dim3(a.rows, g.parts), dim3(CT), 0, st, g);
    };
    go(k_sample_max<F32>, LIGHT_BLOCKS);
    if (g.cut) {
        /* a block adds up to 2,048 bins to its row's: 16 blocks a row where that fills the chip (64 rows with top-p: 17.8
         * us, 24.2 with 32 a row; 1 row 7.0, so 5.7) */
        go(k_sample_bins<F32>, a.rows * 16u < 256u ? 256u : a.rows * 16u < HEAVY_BLOCKS ? a.rows * 16u : HEAVY_BLOCKS);
        go(k_sample_list<F32>, LIGHT_BLOCKS);
        hipLaunchKernelGGL((k_sample_cut<F32>), dim3(a.rows), dim3(NT), 0, st, g);
    }
    go(k_sample_sums<F32>, HEAVY_BLOCKS);
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
