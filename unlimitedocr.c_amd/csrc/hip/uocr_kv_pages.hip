/*
 * uocr_kv_pages.hip - the paged KV cache on gfx950: appending tokens with the
 * position rotation applied, reading them back as rows, and the attention of
 * one new token of each sequence.
 */
#include "uocr_gemm.h"
#include "uocr_serve.h"

#include <math.h>

typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

typedef u32 u32x4 __attribute__((ext_vector_type(4)));

/* Cached rows are read once: non-temporal loads, 154 against 285 us at 876 MB
 * of fp16 cache and 18.6 against 24.6 at 41 MB that the caches hold
 * from call to call; Q8_0 pages, which need half the lines, 70 against 71. */
__device__ __forceinline__ uint4 load_once(const uint8_t *p) {
    const u32x4 v = __builtin_nontemporal_load((const u32x4 *)p);
    return make_uint4(v.x, v.y, v.z, v.w);
}

constexpr u32 APPEND_TOKENS = 8; /* most tokens of a block */
constexpr u32 GATHER_NT = 1024;  /* threads of a block */

/* The largest of a row's N lanes (4 or 8). */
template <u32 N>
__device__ __forceinline__ u32 row_max(u32 v) {
    v = max(v, (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true)); /* quad_perm [1,0,3,2] */
    v = max(v, (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true)); /* quad_perm [2,3,0,1] */
    if (N == 8u) v = max(v, (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true)); /* row_half_mirror */
    return v;
}

/* ---- append ----------------------------------------------------------------- */

/* y1 = x1 cos - x2 sin, y2 = x1 sin + x2 cos on the pairs (i, i + D/2) of a
 * head.  A row is D/16 lanes, each 8 values of the low half and their partners.
 * Bound by HBM: every row is read and written once.  A thread's rows are loaded
 * before the block finds its tokens' pages and angles, so that the two chains
 * of loads run side by side.  The angle is formed in turns in fp64 and reduced
 * to half a turn before the fp32 sine and cosine (position 10^6 in fp32 would
 * be off by 0.06 radians); a block computes them once per token, in LDS, for
 * all its heads. */
/* 8 blocks of a CU: with the registers that the compiler takes by itself (3 blocks) 16,000 fp16 tokens of 32 + 8 heads
 * take 128 us, so 82 (5.2 TB/s, a large copy's rate); blocks of 512 threads 88.  4,988 Q8_0 tokens of 10 + 20 heads take
 * 22.9 (3.4 TB/s). */
template <int D, bool Q8>
__global__ __launch_bounds__(256, 8) void k_kv_append(uocr_append_args a, u32 tpb) {
    constexpr u32 LPR = D / 16;
    __shared__ float2 cs[APPEND_TOKENS][D / 2];
    __shared__ int page_of[APPEND_TOKENS], pos_of[APPEND_TOKENS];
    const u32 t = threadIdx.x, t0 = blockIdx.x * tpb, nt = min(tpb, a.tokens - t0);
    const u32 kvh = a.kv.heads, rows = a.heads + 2u * kvh, items = nt * rows * LPR;
    auto source = [&](u32 tok, u32 r) {
        const bool is_q = r < a.heads, is_v = r >= a.heads + kvh;
        const u32 h = is_q ? r : r - a.heads - (is_v ? kvh : 0u);
        return (is_q ? a.q + (t0 + tok) * a.qs : is_v ? a.v + (t0 + tok) * a.vs : a.k + (t0 + tok) * a.ks) + h * D;
    };
    uint4 raw0, raw1;
    auto load = [&](u32 i) {
        if (i >= items) return;
        const uint16_t *src = source(i / LPR / rows, i / LPR % rows) + 8u * (i % LPR);
        raw0 = load_any(src);
        raw1 = load_any(src + D / 2);
    };
    load(t);
    if (a.rotate) {
#pragma unroll 1
        for (u32 i = t; i < nt * (D / 2); i += 256u) {
            const u32 tok = i / (D / 2), d = i % (D / 2);
            const double turns = (double)a.pos[t0 + tok] * (exp2((double)d * (-2.0 / D) * a.log2_theta) * 0.15915494309189535);
            float2 v;
            sincospif((float)(2.0 * (turns - rint(turns))), &v.y, &v.x);
            cs[tok][d] = v;
        }
    }
    if (t < nt) {
        const int seq = a.seqs != nullptr ? a.seqs[t0 + t] : (int)(t0 + t), pos = a.pos[t0 + t];
        const bool in = seq >= 0 && (u32)seq < a.kv.n_seqs && pos >= 0 && ((u32)pos >> a.kv.shift) < a.kv.table_stride;
        pos_of[t] = in ? pos : -1;
        page_of[t] = in ? kv_page(a.kv, seq, (u32)pos) : -1;
    }
    __syncthreads();
#pragma unroll 1
    for (u32 i = t; i < items; i += 256u) {
        if (i != t) load(i);
        const u32 lane = i % LPR, tok = i / LPR / rows, r = i / LPR % rows;
        const int pos = pos_of[tok];
        if (pos < 0) continue; /* a padding row: the whole row's lanes leave together */
        const bool is_q = r < a.heads, is_v = r >= a.heads + kvh;
        const u32 h = is_q ? r : r - a.heads - (is_v ? kvh : 0u);
        U4H8 lo, hi;
        lo.u = raw0;
        hi.u = raw1;
        float y[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x1 = (float)lo.h[e], x2 = (float)hi.h[e];
            if (a.rotate && !is_v) {
                const float2 w = cs[tok][8u * lane + e];
                y[e] = fmaf(x1, w.x, -(x2 * w.y));
                y[8 + e] = fmaf(x1, w.y, x2 * w.x);
            } else {
                y[e] = x1;
                y[8 + e] = x2;
            }
            lo.h[e] = (h16)y[e];
            hi.h[e] = (h16)y[8 + e];
        }
        uint16_t *rows_out = is_q ? a.q_out + (t0 + tok) * a.qos : is_v || a.k_out == nullptr ? nullptr : a.k_out + (t0 + tok) * a.kos;
        if (rows_out != nullptr) {
            store_any(rows_out + h * D + 8u * lane, lo.u);
            store_any(rows_out + h * D + 8u * lane + D / 2, hi.u);
        }
        if (is_q || page_of[tok] < 0) continue;
        const u32 slot = (h << a.kv.shift) + ((u32)pos & ((1u << a.kv.shift) - 1u)); /* row of the page */
        const uint64_t at = (uint64_t)page_of[tok] * a.kv.page_stride + (uint64_t)slot * D + 8u * lane;
        if constexpr (!Q8) {
            uint16_t *dst = (uint16_t *)(is_v ? a.kv.v : a.kv.k) + at;
            *(uint4 *)dst = lo.u;
            *(uint4 *)(dst + D / 2) = hi.u;
        } else {
            /* the quantiser's rule from the fp32 values: scale = max / 127 (1 for zeros), q = rint(y / scale), the
             * scale then rounded to fp16 (2^-11; below 6e-5, values of under 0.008, to the subnormals' 3e-8).  The
             * largest magnitudes go by their bits: what is not finite is above all others. */
            u32 b0 = 0u, b1 = 0u;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                b0 = max(b0, __float_as_uint(y[e]) & 0x7fffffffu);
                b1 = max(b1, __float_as_uint(y[8 + e]) & 0x7fffffffu);
            }
            if (D == 64) b0 = b1 = max(b0, b1); /* both halves are one group */
            b0 = row_max<LPR>(b0);
            b1 = row_max<LPR>(b1);
            const bool f0 = b0 < 0x7f800000u, f1 = b1 < 0x7f800000u;
            const float m0 = __uint_as_float(b0), m1 = __uint_as_float(b1);
            const float s0 = b0 == 0u ? 1.0f : m0 / 127.0f, s1 = b1 == 0u ? 1.0f : m1 / 127.0f;
            /* y / s rounded as a division is: the product with the rounded reciprocal, corrected by its residual
             * (Markstein's method), then to the nearest integer by adding 1.5 2^23, in whose last byte it is left.  It
             * is 127 at most: scales are no subnormals (y is 0 or more than 2^-100), so their rounding adds 2^-23. */
            const float i0 = 1.0f / s0, i1 = 1.0f / s1;
            auto quantised = [](float v, float sc, float inv) {
                const float x = v * inv;
                return __float_as_uint(fmaf(fmaf(-x, sc, v), inv, x) + 12582912.0f);
            };
            auto bytes = [&](const float *v, float sc, float inv) {
                u32 w[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const u32 q01 = __builtin_amdgcn_perm(quantised(v[4 * k + 1], sc, inv), quantised(v[4 * k], sc, inv), 0x0c0c0400u);
                    const u32 q23 = __builtin_amdgcn_perm(quantised(v[4 * k + 3], sc, inv), quantised(v[4 * k + 2], sc, inv), 0x04000c0cu);
                    w[k] = q01 | q23;
                }
                return make_uint2(w[0], w[1]);
            };
            /* a group that is not finite: 0 times its NaN scale */
            const uint2 q0 = f0 ? bytes(y, s0, i0) : make_uint2(0u, 0u), q1 = f1 ? bytes(y + 8, s1, i1) : make_uint2(0u, 0u);
            int8_t *dst = (int8_t *)(is_v ? a.kv.v : a.kv.k) + at;
            *(uint2 *)dst = q0;
            *(uint2 *)(dst + D / 2) = q1;
            if (lane == 0u) {
                uint16_t *sc = (is_v ? a.kv.vs : a.kv.ks) + (uint64_t)page_of[tok] * (a.kv.page_stride / 64u) + slot * (D / 64u);
                sc[0] = f0 ? __builtin_bit_cast(uint16_t, (h16)s0) : (uint16_t)0x7e00u;
                if (D == 128) sc[1] = f1 ? __builtin_bit_cast(uint16_t, (h16)s1) : (uint16_t)0x7e00u;
            }
        }
    }
}

/* ---- gather ------------------------------------------------------------------- */

/* A copy (Q8_0: fp16(q * scale)), bound by HBM: 8 or 16 values a lane, one item
 * a thread.  Each item is a chain of loads (position, page, row) that only other
 * wavefronts can hide, so no thread waits for a second one: 18,569 Q8_0 tokens of
 * 8 heads took 34.0 us with four items a thread, 24.4 so (4.7 TB/s; 25.6 in
 * blocks of 512 threads, 26.8 of 256). */
template <int D, bool Q8>
__global__ __launch_bounds__(GATHER_NT) void k_kv_gather(uocr_gather_args a, u32 tpb, bool once) {
    constexpr u32 E = Q8 ? 16 : 8, LPR = D / E;
    const u32 t0 = blockIdx.x * tpb, nt = min(tpb, a.tokens - t0);
    const u32 kvh = a.kv.heads, first = a.k_out == nullptr ? kvh : 0u, rows = (a.v_out == nullptr ? kvh : 2u * kvh) - first;
    const u32 items = nt * rows * LPR;
    for (u32 i = threadIdx.x; i < items; i += GATHER_NT) {
        const u32 lane = i % LPR, tok = t0 + i / LPR / rows, r = i / LPR % rows + first;
        const bool is_v = r >= kvh;
        const u32 h = is_v ? r - kvh : r;
        const int seq = a.seqs != nullptr ? a.seqs[tok] : (int)tok, pos = a.pos[tok];
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        u32 sc = 0u;
        int page = -1;
        if (seq >= 0 && (u32)seq < a.kv.n_seqs && pos >= 0 && ((u32)pos >> a.kv.shift) < a.kv.table_stride) page = kv_page(a.kv, seq, (u32)pos);
        if (page >= 0) {
            const u32 slot = (h << a.kv.shift) + ((u32)pos & ((1u << a.kv.shift) - 1u));
            const uint64_t at = (uint64_t)page * a.kv.page_stride + (uint64_t)slot * D + E * lane;
            const uint8_t *src = (const uint8_t *)(is_v ? a.kv.v : a.kv.k) + (Q8 ? at : 2u * at);
            w = once ? load_once(src) : *(const uint4 *)src;
            if (Q8) sc = (is_v ? a.kv.vs : a.kv.ks)[(uint64_t)page * (a.kv.page_stride / 64u) + slot * (D / 64u) + lane / 4u];
        }
        uint16_t *dst = (is_v ? a.v_out + tok * a.vos : a.k_out + tok * a.kos) + h * D + E * lane;
        if constexpr (!Q8) {
            store_any(dst, w);
        } else {
            U4H8 lo, hi;
            /* an absent token's zeros are zeros with any scale: its payload 0 and scale 0 */
            lo.v = dequant_q8(w.x, w.y, sc);
            hi.v = dequant_q8(w.z, w.w, sc);
            store_any(dst, lo.u);
            store_any(dst + 8u, hi.u);
        }
    }
}

/* ---- attention of one token ---------------------------------------------------- */

constexpr u32 PA_TILE = 128;   /* tokens of a block's tile: 32 of each of its 4 wavefronts */
constexpr u32 PA_BLOCKS = 512; /* 2 per CU: what the registers of a wavefront allow */
constexpr u32 ALIGNED = 4;     /* most tiles of a block that has one set alone */
constexpr u32 FUSED_ROWS = 512; /* most rows of partials that the last block of a set joins */

struct PagedGrid {
    uocr_paged_args a;
    u32 group, chunks; /* query heads of a KV head; sets of up to 16 of them */
    u32 rows;          /* of a partial: min(group, 16) */
    float c;           /* scale * log2(e) */
    u32 *count;        /* [PA_BLOCKS]: partials of the set that goes on behind a block, which is one at most, that have
                        * arrived; 0 between launches, at the same place whatever the heads */
    bool fused;        /* the last block of a set joins it */
    bool aligned;      /* few enough sets for a block each */
};

__device__ const uint4 g_zero_row[16] = {};

/* Partials go from block to block within a launch: stores and loads that pass
 * the L2 of an XCD by (sc1), counted in by an atomic once they have arrived. */
__device__ __forceinline__ __amdgpu_buffer_rsrc_t device_buffer(const void *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, 0x7fffffff, 0x00020000);
}
__device__ __forceinline__ void store_through(float *base, u32 at, f32x4 v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), device_buffer(base), at * 4u, 0, 16);
}
__device__ __forceinline__ f32x4 load_through(const float *base, u32 at) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(device_buffer(base), at * 4u, 0, 16));
}

/* Tokens of sequence s, and the tiles of each of its head sets. */
__device__ __forceinline__ u32 seq_len(const uocr_paged_args &a, u32 s) {
    return (u32)min(max(a.lengths[s], 0), (int)(a.kv.table_stride << a.kv.shift));
}
__device__ __forceinline__ u32 len_tiles(u32 len) {
    return max((len + PA_TILE - 1u) / PA_TILE, 1u); /* an empty sequence has its zeros to write */
}

/* Which block takes which tiles.  Tiles are numbered by sequence, head set and
 * position.  Where a block has many, block b takes [N b / B, N (b + 1) / B) of
 * all N, whatever sequences these belong to: no length of one sequence leaves
 * CUs idle.  Where it has few (q of them, at most ALIGNED + 1), a set's tiles
 * are padded to a multiple of q, if the blocks still run at once, and none
 * begins a second set, whose loads would wait for the first one's end (16 sequences of about 1,044 tokens, Q8_0,
 * 10 heads: 19.1 us, else 19.9; of 500 tokens fp16 17.3, else 19.8; with up to 9 tiles a
 * block 2,000 tokens took 38.7 us against 35.6). */
struct Split {
    uint64_t total;
    u32 q, blocks; /* q 0: any tiles */
};
__device__ __forceinline__ u32 padded(const Split &p, u32 nt) {
    return p.q == 0u ? nt : (nt + p.q - 1u) / p.q * p.q;
}
__device__ __forceinline__ uint64_t share(const Split &p, u32 b) {
    return p.q == 0u ? p.total * b / p.blocks : (uint64_t)b * p.q;
}
__device__ __forceinline__ u32 block_of(const Split &p, uint64_t tile) {
    return (u32)(p.q == 0u ? ((tile + 1u) * p.blocks - 1u) / p.total : tile / p.q);
}
/* Place of a block's partial of the set that begins at tile T0: only without
 * padding can it have two, of its first set and of its last. */
__device__ __forceinline__ u32 place(const Split &p, u32 b, uint64_t T0) {
    return p.q != 0u ? b : 2u * b + (share(p, b) >= T0 ? 0u : 1u);
}

/* The split, and the tiles (padded) before the lane's run of sequences, by each
 * wavefront for itself. */
__device__ __forceinline__ uint64_t make_split(const PagedGrid &g, u32 run, Split &p) {
    const u32 lane = threadIdx.x & 63u, sets = g.a.kv.heads * g.chunks, s0 = lane * run, s1 = min(s0 + run, g.a.kv.n_seqs);
    const u32 nt0 = s0 < s1 ? len_tiles(seq_len(g.a, s0)) : 0u; /* mostly the only one */
    auto sum = [&](uint64_t &own) {
        own = padded(p, nt0);
        for (u32 s = s0 + 1u; s < s1; ++s) own += padded(p, len_tiles(seq_len(g.a, s)));
        own *= sets;
        const uint64_t all = wave_before(own);
        p.total = lane64(own + all, 63);
        return all;
    };
    p.q = 0u;
    uint64_t own, before = sum(own);
    const uint64_t n = p.total, q = (n + PA_BLOCKS - 1u) / PA_BLOCKS;
    if (g.aligned && q <= ALIGNED) {
        for (p.q = (u32)q; p.q <= (u32)q + 1u; ++p.q) {
            const uint64_t with = p.q == 1u ? before : sum(own);
            if (p.total > (uint64_t)PA_BLOCKS * p.q) continue; /* a second round of blocks would cost more */
            p.blocks = (u32)(p.total / p.q);
            return with;
        }
        p.q = 0u;
        p.total = n;
    }
    p.blocks = (u32)min(n, (uint64_t)PA_BLOCKS); /* none without a tile */
    return before;
}

/* The scale of group j, of two in a word. */
__device__ __forceinline__ float scale_of(u32 pair, u32 j) {
    return (float)__builtin_bit_cast(h16, (unsigned short)(j == 0u ? pair & 0xffffu : pair >> 16));
}

/* What a state with maximum m counts for beside one with maximum M >= m.  Only
 * scores that are all NaN leave weight without a maximum: their NaN goes on. */
__device__ __forceinline__ float state_factor(float m, float M, float c) {
    return m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - M) * c);
}

/* Joins the partials of n heads (rows row0 .. of their set) that blocks b0 .. b1
 * had tiles of (the set's tiles begin at T0): out = sum_b o_b 2^((m_b - M) c) /
 * sum_b l_b 2^((m_b - M) c).  A group of n D / 4 threads reads every par-th
 * partial, with the running maximum; the groups are joined through LDS. */
template <int D>
__device__ __forceinline__ void join_heads(const PagedGrid &g, const Split &sp, uint64_t T0, u32 b0, u32 b1, u32 row0, u32 n, uint16_t *out, uint8_t *sm) {
    constexpr u32 LN = D / 4;
    f32x4 *acc = (f32x4 *)sm;               /* [256] */
    float2 *state = (float2 *)(acc + 256);  /* [256] */
    const u32 t = threadIdx.x, lanes = n * LN, par = 256u / lanes, p = t / lanes, h = t % lanes / LN, ln = t % LN;
    float m = -INFINITY, l = 0.0f;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](float m2, float l2, f32x4 v2) {
        if (l2 == 0.0f) return; /* no weight there */
        const float M = fmaxf(m, m2), f = l == 0.0f ? 0.0f : state_factor(m, M, g.c), f2 = state_factor(m2, M, g.c);
        m = M;
        l = fmaf(l2, f2, l * f);
#pragma unroll
        for (u32 e = 0; e < 4; ++e) v[e] = fmaf(v2[e], f2, v[e] * f);
    };
    if (p < par) {
#pragma unroll 4
        for (u32 b = b0 + p; b <= b1; b += par) {
            const u32 at = (place(sp, b, T0) * g.rows + row0 + h) * (D + 4);
            const f32x4 ml = load_through(g.a.part, at + D), o = load_through(g.a.part, at + 4u * ln);
            add(ml.x, ml.y, o);
        }
    }
    acc[t] = v;
    state[t] = make_float2(m, l);
    __syncthreads();
    if (t < lanes) {
        for (u32 x = 1; x < par; ++x) {
            const float2 s2 = state[x * lanes + t];
            add(s2.x, s2.y, acc[x * lanes + t]);
        }
        const float li = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (u32 e = 0; e < 4; ++e) out[h * D + 4u * ln + e] = __builtin_bit_cast(uint16_t, (h16)(v[e] * li));
    }
    __syncthreads();
}

/* One pass over the cache with the running maximum and sum of the softmax.
 * Bound by HBM on long caches and by the chain of dependent loads (lengths,
 * page, rows) on short ones.
 *
 * The query heads of a KV head are one side of the MFMA tiles (up to 16; a
 * group of one leaves 15 columns idle, which costs nothing: 16 MFMAs per 16 KB
 * of cache are an eighth of what the CU could do meanwhile), so a cache row is
 * read once for all of them.  A wavefront takes 32 tokens of the block's tile:
 *   S^T = K Q^T, 16x16x32: lane l holds head l % 16 and tokens
 *   16 n + 4 (l / 16) + i; K goes from memory straight into the operand (lane
 *   l: token l % 16, 16 bytes at (l / 16));
 *   O^T += V^T P^T: the probabilities stay where S^T left them, V goes through
 *   LDS, row-major, and is transposed by the LDS read.
 * Q8_0: K enters the MFMA as its integers (exact in fp16), a sum for each group
 * of 64 dims, the fp32 sums times the scales; V as its integers, too, and its
 * scales, over a power of two above the largest so far, with the probabilities
 * (one rounding to fp16 for both).
 * Tokens past the length or in absent pages are read from a row of zeros: what
 * stands there never enters a product.
 *
 * The wavefronts' states are merged in LDS; a head set that one block covers is
 * written at once, else its fp32 state goes to the block's partials (at most
 * two: its first and its last set), which the last block to come, or
 * k_paged_join, joins. */
template <int D, bool Q8>
__global__ __launch_bounds__(256, 2) void k_paged_attention(PagedGrid g) {
    constexpr u32 ROW = D * (Q8 ? 1 : 2);      /* bytes of a cached row */
    constexpr u32 NK = ROW / 64;               /* 16-byte loads of a lane per 16 keys */
    constexpr u32 VL = ROW / 16;               /* lanes of a V row */
    constexpr u32 NV = 32 * VL / 64;           /* V loads of a lane per 32 tokens */
    constexpr u32 ORS = D + 4;                 /* floats from a head's row to the next, in LDS */
    constexpr u32 WLDS = 16 * ORS * 4 > 64 * D ? 16 * ORS * 4 : 64 * D; /* V tile, later the state */
    __shared__ __attribute__((aligned(1024))) uint8_t sm[4 * WLDS];
    __shared__ float sml[4][2][16];
    __shared__ __attribute__((aligned(16))) float scales[4][2][32 * (D / 64)]; /* Q8_0: of the tokens' groups, those of V in units */
    __shared__ u32 arrived;
    const u32 t = threadIdx.x, lane = t & 63u, wave = t >> 6, col = lane & 15u, gr = lane >> 4;
    const uocr_kv &kv = g.a.kv;
    const u32 sets = kv.heads * g.chunks;

    Split sp;
    const u32 run = (kv.n_seqs + 63u) / 64u;
    const uint64_t before = make_split(g, run, sp);
    if (blockIdx.x >= sp.blocks) return;
    const uint64_t lo = share(sp, blockIdx.x), hi = share(sp, blockIdx.x + 1u);
    /* the last lane whose run begins at or before tile lo has its sequence (each has a tile) */
    const u32 at_lane = 63u - (u32)__builtin_clzll(__ballot(before <= lo && lane * run < kv.n_seqs));
    u32 s = at_lane * run;
    uint64_t base = lane64(before, (int)at_lane), at = lo;
    uint8_t *vt = sm + wave * WLDS;
    while (at < hi) {
        const u32 len = seq_len(g.a, s), nt = len_tiles(len), ntp = padded(sp, nt);
        if (at >= base + (uint64_t)ntp * sets) {
            base += (uint64_t)ntp * sets;
            ++s;
            continue;
        }
        const u32 set = (u32)((at - base) / ntp), ta = (u32)((at - base) % ntp);
        const u32 tb = (u32)min((uint64_t)nt, (uint64_t)ta + (hi - at)); /* the block's tiles of this set: [ta, tb) */
        const u32 kvh = set / g.chunks, h0 = kvh * g.group + 16u * (set % g.chunks);
        const u32 nh = min(16u, kvh * g.group + g.group - h0); /* query heads of the set */
        const int32_t *table = kv.table + (uint64_t)s * kv.table_stride;

        /* the query operand: head `col`, the dims that the K operand has in the same place */
        U4H8 qr[D / 32];
#pragma unroll
        for (u32 x = 0; x < D / 32; ++x) {
            const u32 d = Q8 ? 64u * (x / 2u) + 16u * gr + 8u * (x % 2u) : 32u * x + 8u * gr;
            qr[x].u = make_uint4(0u, 0u, 0u, 0u);
            if (col < nh) qr[x].u = load_any(g.a.q + (uint64_t)s * g.a.qs + (h0 + col) * D + d);
        }
        f32x4 o[D / 16];
#pragma unroll
        for (u32 n = 0; n < D / 16; ++n) o[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        float unit = 0x1p30f; /* Q8_0: sums are in units of 1 / unit, a power of two */

        uint4 kr[2 * NK], vr[NV];
        u32 ksc = 0, vsc = 0; /* scales of token lane % 32 */
        u32 valid;            /* bit i: token i of the wavefront's 32 */
        /* the page of token lane % 32 of the wavefront's part of tile x (-1: none) */
        auto page = [&](u32 x) {
            const u32 tok = x * PA_TILE + 32u * wave + (lane & 31u);
            int p = -1;
            if (x < tb && tok < len) {
                p = table[tok >> kv.shift];
                if ((u32)p >= kv.n_pages) p = -1;
            }
            return p;
        };
        auto load = [&](u32 x, int p) {
            const u32 tok0 = x * PA_TILE + 32u * wave;
            valid = (u32)__ballot(p >= 0);
            const uint8_t *k = (const uint8_t *)kv.k, *v = (const uint8_t *)kv.v;
            /* Where the row of token lane % 32 stands in k and v.  V rows' places go from lane to lane, K rows' are formed anew
             * from their pages: 146 us at 876 MB of fp16 cache, 154 with all formed anew; 53.3 at 272 MB of Q8_0, so 54.7, and
             * 56.4 with all from lane to lane.  An absent token's scores count nothing, so a row of page 0 does for its key,
             * but its value is read from a row of zeros. */
            const u32 mask = (1u << kv.shift) - 1u, hrow = kvh << kv.shift, in_head = hrow + ((tok0 + (lane & 31u)) & mask);
            const uint64_t values = p >= 0 ? (uint64_t)(u32)p * kv.page_stride + (uint64_t)in_head * D : 0u, bytes = values * (Q8 ? 1u : 2u);
#pragma unroll
            for (u32 n = 0; n < 2; ++n) {
                const int pk = max(__shfl(p, (int)(16u * n + col)), 0);
                const uint8_t *r = k + ((uint64_t)(u32)pk * kv.page_stride + (uint64_t)(hrow + ((tok0 + 16u * n + col) & mask)) * D) * (Q8 ? 1u : 2u) + 16u * gr;
#pragma unroll
                for (u32 x2 = 0; x2 < NK; ++x2) kr[n * NK + x2] = load_once(r + 64u * x2);
            }
#pragma unroll
            for (u32 y = 0; y < NV; ++y) {
                const u32 i = (64u / VL) * y + lane / VL;
                const uint8_t *r = v + (((uint64_t)(u32)__shfl((int)(bytes >> 32), (int)i) << 32) | (u32)__shfl((int)bytes, (int)i));
                vr[y] = load_once(((valid >> i) & 1u ? r : (const uint8_t *)g_zero_row) + 16u * (lane % VL));
            }
            if constexpr (Q8) {
                ksc = vsc = 0u;
                if (p >= 0) {
                    const uint64_t sat = values / 64u;
                    if (D == 128) {
                        ksc = *(const u32 *)(kv.ks + sat);
                        vsc = *(const u32 *)(kv.vs + sat);
                    } else {
                        ksc = kv.ks[sat];
                        vsc = kv.vs[sat];
                    }
                }
            }
        };
        load(ta, page(ta));
        int pn = page(ta + 1u);
        for (u32 x = ta; x < tb; ++x) {
            const u32 now = valid;
            float sc[8];
            float sv[8][D / 64]; /* Q8_0: the scales of V, where the scores are */
            if (now != 0u) {
                /* V to LDS, rows swizzled by pairs of 16-byte pieces so that the transposing reads touch all banks */
                __builtin_amdgcn_wave_barrier();
                if constexpr (Q8) {
                    const float top = fmaxf(fabsf(scale_of(vsc, 0)), fabsf(scale_of(vsc, 1)));
                    if (__any(top * unit > 1.0f)) {
                        float all = top;
#pragma unroll
                        for (int x2 = 32; x2 > 0; x2 >>= 1) all = fmaxf(all, __shfl_xor(all, x2));
                        const float to = all < 65536.0f ? ldexpf(1.0f, -ilogbf(all) - 1) : 0x1p-16f, by = to / unit;
                        unit = to;
#pragma unroll
                        for (u32 n = 0; n < D / 16; ++n)
#pragma unroll
                            for (u32 i = 0; i < 4; ++i) o[n][i] *= by;
                    }
                    if (lane < 32u) {
#pragma unroll
                        for (u32 j = 0; j < D / 64; ++j) {
                            scales[wave][0][lane * (D / 64) + j] = scale_of(ksc, j);
                            scales[wave][1][lane * (D / 64) + j] = scale_of(vsc, j) * unit;
                        }
                    }
                }
                auto swz = [](u32 key, u32 pc) { return key * (2u * D) + 16u * (pc ^ (D == 128 ? (key & 7u) << 1 : ((key >> 1) & 3u) << 1)); };
#pragma unroll
                for (u32 y = 0; y < NV; ++y) {
                    const u32 key = (64u / VL) * y + lane / VL, pc = lane % VL;
                    if constexpr (Q8) {
                        U4H8 a, b;
                        a.v = dequant_q8(vr[y].x, vr[y].y, 0x3c00u);
                        b.v = dequant_q8(vr[y].z, vr[y].w, 0x3c00u);
                        *(uint4 *)(vt + swz(key, 2u * pc)) = a.u;
                        *(uint4 *)(vt + swz(key, 2u * pc + 1u)) = b.u;
                    } else {
                        *(uint4 *)(vt + swz(key, pc)) = vr[y];
                    }
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (u32 n = 0; n < 2; ++n) {
                    if constexpr (Q8) {
                        f32x4 part[D / 64];
#pragma unroll
                        for (u32 j = 0; j < D / 64; ++j) {
                            part[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                            part[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(dequant_q8(kr[n * NK + j].x, kr[n * NK + j].y, 0x3c00u), qr[2 * j].v, part[j], 0, 0, 0);
                            part[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(dequant_q8(kr[n * NK + j].z, kr[n * NK + j].w, 0x3c00u), qr[2 * j + 1].v, part[j], 0, 0, 0);
                        }
                        const float *ks = &scales[wave][0][(16u * n + 4u * gr) * (D / 64)], *vs = &scales[wave][1][(16u * n + 4u * gr) * (D / 64)];
#pragma unroll
                        for (u32 i = 0; i < 4; ++i) {
                            float v = part[0][i] * ks[i * (D / 64)];
                            if (D == 128) v = fmaf(part[D / 64 - 1][i], ks[i * (D / 64) + D / 64 - 1], v);
                            sc[4 * n + i] = v;
#pragma unroll
                            for (u32 j = 0; j < D / 64; ++j) sv[4 * n + i][j] = vs[i * (D / 64) + j];
                        }
                    } else {
                        f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (u32 x2 = 0; x2 < NK; ++x2) {
                            U4H8 kk;
                            kk.u = kr[n * NK + x2];
                            a = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk.v, qr[x2].v, a, 0, 0, 0);
                        }
#pragma unroll
                        for (u32 i = 0; i < 4; ++i) sc[4 * n + i] = a[i];
                    }
                }
            }
            if (x + 1u < tb) {
                load(x + 1u, pn);
                pn = page(x + 2u);
            }
            if (now == 0u) continue;
            if (now != 0xffffffffu) {
#pragma unroll
                for (u32 i = 0; i < 8; ++i)
                    if (!((now >> (16u * (i / 4u) + 4u * gr + i % 4u)) & 1u)) sc[i] = -INFINITY;
            }
            float tm = sc[0];
#pragma unroll
            for (u32 i = 1; i < 8; ++i) tm = fmaxf(tm, sc[i]);
            tm = fmaxf(tm, __shfl_xor(tm, 16));
            tm = fmaxf(tm, __shfl_xor(tm, 32));
            if (__any(tm > m)) {
                const float mn = fmaxf(m, tm), corr = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * g.c);
                m = mn;
                l *= corr;
#pragma unroll
                for (u32 n = 0; n < D / 16; ++n)
#pragma unroll
                    for (u32 i = 0; i < 4; ++i) o[n][i] *= corr;
            }
            const float mc = m == -INFINITY ? 0.0f : m * g.c;
            constexpr u32 NP = Q8 ? D / 64 : 1;
            U4H8 p[NP];
#pragma unroll
            for (u32 i = 0; i < 8; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(sc[i], g.c, -mc));
                l += e;
#pragma unroll
                for (u32 j = 0; j < NP; ++j) p[j].h[i] = Q8 ? (h16)(e * sv[i][j]) : (h16)e;
            }
#pragma unroll
            for (u32 n = 0; n < D / 16; ++n) {
                /* the lane's key of the transposing read: 4 gr + lane / 4 % 4 (and + 16), its dims 16 n + 4 (lane % 4) */
                const u32 key = 4u * gr + ((lane >> 2) & 3u);
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
                auto tr = [&](u32 kk) {
                    const u32 pc = 2u * n + ((lane >> 1) & 1u);
                    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4 *)(vt + kk * (2u * D) + 16u * (pc ^ (D == 128 ? (kk & 7u) << 1 : ((kk >> 1) & 3u) << 1)) + 8u * (lane & 1u))));
                };
                const uint2 a0 = tr(key), a1 = tr(key + 16u);
                U4H8 vv;
                vv.u = make_uint4(a0.x, a0.y, a1.x, a1.y);
                o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv.v, p[Q8 ? n / 4u : 0u].v, o[n], 0, 0, 0);
            }
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        /* the four states: lane holds head col, dims 16 n + 4 gr + i */
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (u32 n = 0; n < D / 16; ++n) {
            if constexpr (Q8) {
#pragma unroll
                for (u32 i = 0; i < 4; ++i) o[n][i] *= 1.0f / unit;
            }
            *(f32x4 *)(vt + (col * ORS + 16u * n + 4u * gr) * 4u) = o[n];
        }
        if (lane < 16u) {
            sml[wave][0][col] = m;
            sml[wave][1][col] = l;
        }
        __syncthreads();
        const bool whole = ta == 0u && tb == nt;
        const u32 slot = place(sp, blockIdx.x, base + (uint64_t)set * ntp);
        for (u32 i = t; i < nh * (D / 4); i += 256u) {
            const u32 h = i / (D / 4), d = 4u * (i % (D / 4));
            const float M = fmaxf(fmaxf(sml[0][0][h], sml[1][0][h]), fmaxf(sml[2][0][h], sml[3][0][h]));
            float L = 0.0f;
            f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (u32 w = 0; w < 4; ++w) {
                const float mw = sml[w][0][h], lw = sml[w][1][h];
                const f32x4 x = *(const f32x4 *)(sm + w * WLDS + (h * ORS + d) * 4u);
                if (lw == 0.0f) continue; /* no weight in this wavefront's tokens */
                const float f = state_factor(mw, M, g.c);
                L = fmaf(lw, f, L);
#pragma unroll
                for (u32 e = 0; e < 4; ++e) v[e] = fmaf(x[e], f, v[e]);
            }
            if (whole) {
                const float li = L == 0.0f ? 0.0f : 1.0f / L;
                uint16_t *dst = g.a.out + (uint64_t)s * g.a.os + (h0 + h) * D + d;
#pragma unroll
                for (u32 e = 0; e < 4; ++e) dst[e] = __builtin_bit_cast(uint16_t, (h16)(v[e] * li));
            } else {
                const u32 to = (slot * g.rows + h) * (D + 4);
                store_through(g.a.part, to + d, v);
                if (d == 0u) store_through(g.a.part, to + D, f32x4{M, L, 0.0f, 0.0f});
            }
        }
        if (!whole && g.fused) {
            /* the block that comes last joins the set's partials */
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const uint64_t T0 = base + (uint64_t)set * ntp;
            const u32 b0 = block_of(sp, T0), b1 = block_of(sp, T0 + ntp - 1u);
            if (t == 0u) {
                u32 *count = g.count + b0;
                arrived = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (arrived == b1 - b0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (arrived == b1 - b0) {
                asm volatile("" ::: "memory");
                constexpr u32 MOST = 256 / (D / 4);
                for (u32 h = 0; h < nh; h += MOST)
                    join_heads<D>(g, sp, T0, b0, b1, h, min(nh - h, MOST), g.a.out + (uint64_t)s * g.a.os + (h0 + h) * D, sm);
            }
        }
        if (sp.q != 0u) break;
        __syncthreads();
        at += tb - ta;
    }
}

/* The join as a launch of its own, a block for each sequence and head. */
template <int D>
__global__ __launch_bounds__(256) void k_paged_join(PagedGrid g) {
    __shared__ __attribute__((aligned(16))) uint8_t sm[256 * 24];
    const u32 s = blockIdx.x / g.a.hq, h = blockIdx.x % g.a.hq;
    const uocr_kv &kv = g.a.kv;
    const u32 kvh = h / g.group, set = kvh * g.chunks + h % g.group / 16u, row = h % g.group % 16u, sets = kv.heads * g.chunks;
    Split sp;
    const u32 run = (kv.n_seqs + 63u) / 64u;
    const uint64_t before = make_split(g, run, sp);
    const u32 ntp = padded(sp, len_tiles(seq_len(g.a, s)));
    uint64_t T0 = lane64(before, (int)(s / run)) + (uint64_t)set * ntp;
    for (u32 i = s / run * run; i < s; ++i) T0 += (uint64_t)padded(sp, len_tiles(seq_len(g.a, i))) * sets;
    const u32 b0 = block_of(sp, T0), b1 = block_of(sp, T0 + ntp - 1u);
    if (b0 != b1) join_heads<D>(g, sp, T0, b0, b1, row, 1u, g.a.out + (uint64_t)s * g.a.os + h * D, sm);
}

}  // namespace

hipError_t uocr_launch_kv_append(hipStream_t st, const uocr_append_args *a) {
    /* a block for at least 256 lanes' work, so that few heads do not leave most of it idle */
    const u32 lanes = (a->heads + 2u * a->kv.heads) * (a->kv.dim / 16u);
    const u32 tpb = lanes >= 256u ? 1u : (256u / lanes < APPEND_TOKENS ? 256u / lanes : APPEND_TOKENS);
    const dim3 grid((a->tokens + tpb - 1u) / tpb);
    if (a->kv.dim == 128u) {
        if (a->kv.q8) hipLaunchKernelGGL((k_kv_append<128, true>), grid, dim3(256), 0, st, *a, tpb);
        else hipLaunchKernelGGL((k_kv_append<128, false>), grid, dim3(256), 0, st, *a, tpb);
    } else {
        if (a->kv.q8) hipLaunchKernelGGL((k_kv_append<64, true>), grid, dim3(256), 0, st, *a, tpb);
        else hipLaunchKernelGGL((k_kv_append<64, false>), grid, dim3(256), 0, st, *a, tpb);
    }
    return hipGetLastError();
}

hipError_t uocr_launch_kv_gather(hipStream_t st, const uocr_gather_args *a) {
    const u32 sides = (a->k_out != nullptr ? 1u : 0u) + (a->v_out != nullptr ? 1u : 0u);
    const u32 lanes = sides * a->kv.heads * a->kv.dim / (a->kv.q8 ? 16u : 8u);
    const u32 tpb = lanes >= GATHER_NT ? 1u : GATHER_NT / lanes;
    /* Pages of many tokens are read past the caches (16,000 tokens of 8 heads of 128, eight caches in turn: fp16 27.5
     * against 27.9 us, Q8_0 24.2 against 25.4; 18,569 Q8_0 ones of 8: 25.6 against 28.4), those of few may be there still
     * (4,000 of 10: 8.8 against 11.3, 8.4 against 9.6). */
    const bool once = (uint64_t)a->tokens * lanes * 16u > (24u << 20);
    const dim3 grid((a->tokens + tpb - 1u) / tpb);
    if (a->kv.dim == 128u) {
        if (a->kv.q8) hipLaunchKernelGGL((k_kv_gather<128, true>), grid, dim3(GATHER_NT), 0, st, *a, tpb, once);
        else hipLaunchKernelGGL((k_kv_gather<128, false>), grid, dim3(GATHER_NT), 0, st, *a, tpb, once);
    } else {
        if (a->kv.q8) hipLaunchKernelGGL((k_kv_gather<64, true>), grid, dim3(GATHER_NT), 0, st, *a, tpb, once);
        else hipLaunchKernelGGL((k_kv_gather<64, false>), grid, dim3(GATHER_NT), 0, st, *a, tpb, once);
    }
    return hipGetLastError();
}

size_t uocr_paged_attention_ws_bytes(uint32_t heads, uint32_t kv_heads, uint32_t dim) {
    const u32 group = heads / kv_heads, rows = group < 16u ? group : 16u;
    return PA_BLOCKS * sizeof(u32) + (size_t)2u * PA_BLOCKS * rows * (dim + 4u) * sizeof(float);
}

hipError_t uocr_launch_paged_attention(hipStream_t st, const uocr_paged_args *a) {
    PagedGrid g;
    g.a = *a;
    g.group = a->hq / a->kv.heads;
    g.chunks = (g.group + 15u) / 16u;
    g.rows = g.group < 16u ? g.group : 16u;
    g.c = a->scale * 1.4426950408889634f;
    g.count = (u32 *)a->part;
    g.a.part = a->part + PA_BLOCKS;
    /* A set has at most PA_BLOCKS / sets + 2 partials (all sets of a sequence have as many tiles).  One block reads them
     * one after another, the launch of its own with a block for each head: that pays where they are many. */
    g.fused = (PA_BLOCKS / (a->kv.heads * g.chunks) + 2u) * g.rows <= FUSED_ROWS;
    const uint64_t most = ((uint64_t)(a->kv.table_stride << a->kv.shift) + PA_TILE - 1u) / PA_TILE; /* tiles of a set */
    const uint64_t tiles = most * a->kv.n_seqs * a->kv.heads * g.chunks;
    g.aligned = (uint64_t)a->kv.n_seqs * a->kv.heads * g.chunks <= PA_BLOCKS;
    const u32 blocks = tiles < PA_BLOCKS ? (u32)tiles : PA_BLOCKS;
    if (a->kv.dim == 128u) {
        if (a->kv.q8) hipLaunchKernelGGL((k_paged_attention<128, true>), dim3(blocks), dim3(256), 0, st, g);
        else hipLaunchKernelGGL((k_paged_attention<128, false>), dim3(blocks), dim3(256), 0, st, g);
    } else {
        if (a->kv.q8) hipLaunchKernelGGL((k_paged_attention<64, true>), dim3(blocks), dim3(256), 0, st, g);
        else hipLaunchKernelGGL((k_paged_attention<64, false>), dim3(blocks), dim3(256), 0, st, g);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || g.fused || most == 1u) return e; /* one tile a set: nothing to join */
    const dim3 grid(a->kv.n_seqs * a->hq);
    if (a->kv.dim == 128u) hipLaunchKernelGGL((k_paged_join<128>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_paged_join<64>), grid, dim3(256), 0, st, g);
    return hipGetLastError();
}
