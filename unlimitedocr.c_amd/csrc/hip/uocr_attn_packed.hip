/*
 * uocr_attn_packed.hip - causal attention of packed prompts on gfx950: rows of
 * several sequences behind each other, query heads grouped over key heads,
 * queries that continue a prefix of keys.
 */
#include "uocr_async.h"
#include "uocr_serve.h"

#include <math.h>

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint2 lds_read_tr4(const uint8_t *p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p));
}

struct PackedGrid {
    uocr_packed_args a;
    u32 slots, group;
    float c; /* scale * log2(e) */
};

/* Not-finite values of V: 0 times them is NaN, whether a row does not see them
 * or their weight rounds to 0.  They are taken out of the product and counted by
 * a second one, of 0 / 1 visibilities and these codes.  At most 64 keys a tile:
 * the counts of the three kinds do not run into each other, and all fit fp32
 * and fp16 exactly. */
constexpr float CODE_PLUS = 1.0f, CODE_MINUS = 128.0f, CODE_NAN = 16384.0f;

__device__ __forceinline__ void split_special(uint4 v, U4H8 &fin, U4H8 &code) {
    fin.u = v;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = (float)fin.h[i];
        code.h[i] = (h16)(x != x ? CODE_NAN : x == INFINITY ? CODE_PLUS : x == -INFINITY ? CODE_MINUS : 0.0f);
        if (x != x || fabsf(x) == INFINITY) fin.h[i] = (h16)0.0f;
    }
}

/* What a sum with n (the decoded counts) of not-finite terms is. */
__device__ __forceinline__ float with_special(float o, float n) {
    if (n == 0.0f) return o;
    const u32 k = (u32)n;
    const bool nan = k >= 16384u, minus = (k & 16383u) >= 128u, plus = (k & 127u) != 0u;
    return nan || (minus && plus) ? __builtin_nanf("") : o + (plus ? INFINITY : -INFINITY);
}

/* The first slot (query tile) of sequence s.  A sequence of n rows from row a
 * has ceil(n / B) tiles, at most (a + n) / B - a / B + 1: with slots from
 * a / B + s on, no two sequences share one, and a block finds its sequence
 * from the starts alone, without a sum over all of them. */
__device__ __forceinline__ u32 start_of(const int32_t *starts, u32 s, u32 tokens) {
    return (u32)min(max(starts[s], 0), (int)tokens);
}

/* Bound by the power that the matrix unit may draw: 4 x 4,001 rows of 32 heads
 * run at 894 TFLOP/s and 2.0 GHz, the library's fp16 product of 8,192 x 8,192
 * x 8,192 at 1,134 and 1.84 GHz.  Multiplying the next tile's K beside this
 * one's exponentials, or reading K operands further ahead, changed nothing.
 *
 * Block: WQ x 32 query rows of one sequence and head; its wavefronts are WG key
 * groups of WQ wavefronts, group g takes the key tiles g, g + WG, .. of the
 * visible range and the groups' softmax states are merged through LDS.
 * A wavefront keeps its 32 rows' scores, statistics and sums in registers
 * (32x32x16 MFMAs): S^T = K Q^T leaves lane l query l % 32 and keys
 * 8 q + 4 (l / 32) + i, which is where O^T += V^T P^T wants the probabilities.
 * K and V tiles go straight to LDS, row-major, NB tiles of a group with NB - 1
 * in flight; V is transposed by the LDS read.  Both are swizzled by 16-byte
 * pieces so that the reads touch all banks.  DMA = false (k or v rows off
 * 16-byte boundaries): through registers. */
template <int D, int WQ, int WG, int KT, int NB, bool DMA>
__global__ __launch_bounds__(64 * WQ * WG, 2) void k_packed_attention(PackedGrid g) {
    constexpr u32 RB = 2 * D, PPR = RB / 16, RPL = 64 / PPR; /* bytes and pieces of a row, rows of a load */
    constexpr u32 TILE = KT * RB, GB = NB * 2u * TILE;
    constexpr int LD = (int)(2u * TILE / 1024u) / WQ;
    constexpr u32 SLOT = 32u * D * 4u + 512u, MERGE = (WG - 1u) * WQ * SLOT, STAGE = WQ * 32u * RB;
    constexpr u32 LDS0 = WG * GB > MERGE ? WG * GB : MERGE, LDS = LDS0 > STAGE ? LDS0 : STAGE;
    constexpr u32 BQ = WQ * 32u;
    static_assert(KT <= 64, "counts of not-finite values");
    __shared__ __attribute__((aligned(1024))) uint8_t sm[LDS];
    const uocr_packed_args &a = g.a;
    const u32 t = threadIdx.x, lane = t & 63u, r = lane & 31u, hf = lane >> 5;
    const u32 wave = uni(t >> 6), wq = wave % WQ, gi = wave / WQ;
    /* the last tiles of a sequence first: they see most keys.  The heads of a KV head run on one XCD (every eighth
     * block), so its rows are fetched into one L2. */
    const u32 slot = g.slots - 1u - blockIdx.x / a.heads, hx = blockIdx.x % a.heads;
    const u32 kvh = hx % a.kv_heads, h = kvh * g.group + hx / a.kv_heads;

    u32 count = 0; /* sequences that begin at or before the slot */
    for (u32 s = lane; s < a.n_seqs; s += 64u) count += start_of(a.q_starts, s, a.q_tokens) / BQ + s <= slot ? 1u : 0u;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) count += (u32)__shfl_xor((int)count, o);
    count = uni(count);
    if (count == 0u) return;
    const u32 s = count - 1u;
    const u32 qa = start_of(a.q_starts, s, a.q_tokens), qb = start_of(a.q_starts, s + 1u, a.q_tokens);
    const u32 ka = start_of(a.k_starts, s, a.k_tokens), kb = start_of(a.k_starts, s + 1u, a.k_tokens);
    const u32 nq = qb > qa ? qb - qa : 0u, nk = kb > ka ? kb - ka : 0u;
    if (qa / BQ + s > slot) return; /* starts that decrease */
    const u32 q0 = (slot - (qa / BQ + s)) * BQ;
    if (q0 >= nq) return;

    const int lead = (int)nk - (int)nq;                        /* row i sees keys up to i + lead */
    const u32 qw = q0 + 32u * wq, qmax = min(qw + r, nq - 1u); /* the wavefront's first row, the lane's row */
    const int limit = (int)qmax + lead, klast = (int)min(q0 + BQ, nq) - 1 + lead;
    const u32 nt = klast < 0 ? 0u : (u32)klast / KT + 1u, iters = (nt + WG - 1u) / WG;
    const uint16_t *kp = a.k + ka * a.ks + kvh * D, *vp = a.v + ka * a.vs + kvh * D;
    uint8_t *gsm = sm + gi * GB;
    const u32 lds0 = uni((u32)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)gsm);

    auto swz_k = [](u32 key, u32 pc) { return pc ^ (D == 128 ? key & 15u : (key >> 1) & 7u); };
    auto swz_v = [](u32 key, u32 pc) { return pc ^ (D == 128 ? (key & 7u) << 1 : ((key >> 1) & 3u) << 1); };
    /* load x of a tile (the first KT / RPL: K, else V) covers its rows RPL (x % (KT / RPL)) .. */
    auto issue = [&](u32 tile, u32 buf) {
        const u32 left = nk - 1u - tile * KT; /* rows past the last key re-read it */
#pragma unroll
        for (int y = 0; y < LD; ++y) {
            const u32 x = wq * LD + y, kr = RPL * (x % (KT / RPL)) + lane / PPR, pc = lane % PPR;
            const bool is_k = x < KT / RPL;
            const uint16_t *base = is_k ? kp + (uint64_t)(tile * KT) * a.ks : vp + (uint64_t)(tile * KT) * a.vs;
            const u32 row = min(kr, left) * (u32)(is_k ? a.ks : a.vs);
            const u32 piece = is_k ? swz_k(kr, pc) : swz_v(kr, pc);
            if constexpr (DMA) lds_load16(base, 2u * row + 16u * piece, lds0 + buf * 2u * TILE + 1024u * x);
            else *(uint4 *)(gsm + buf * 2u * TILE + 1024u * x + 16u * lane) = load_any(base + row + 8u * piece);
        }
    };

    U4H8 qreg[D / 16];
    f32x16 o[D / 32];
    float m, l; /* m in units of the raw scores; l: this lane's half of the sum */
    auto attend = [&](auto special) {
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
        m = -INFINITY;
        l = 0.0f;
        if (nt != 0u) {
#pragma unroll
            for (u32 b = 0; b + 1u < NB; ++b) issue(min(b * WG + gi, nt - 1u), b);
        }
#pragma unroll
        for (u32 x = 0; x < D / 16; ++x) qreg[x].u = load_any(a.q + (uint64_t)(qa + qmax) * a.qs + h * D + 16u * x + 8u * hf);
        /* The queries are waited for here.  Left to their first use, in the loop, the compiler's wait counts the tiles'
         * loads, which it does not know of, and stops every pass until the next tile has come as well. */
#pragma unroll
        for (u32 x = 0; x < D / 16; ++x) asm volatile("" : "+v"(qreg[x].v));
        u32 buf = 0;
        for (u32 it = 0; it < iters; ++it) {
            /* tile it has landed for all wavefronts; its predecessor's buffer is free */
            wait_barrier<LD * (NB - 2)>();
            issue(min((it + NB - 1u) * WG + gi, nt - 1u), buf == 0u ? NB - 1u : buf - 1u);
            const u32 tile = it * WG + gi, k0 = tile * KT;
            const uint8_t *kt = gsm + buf * 2u * TILE, *vt = kt + TILE;
            buf = buf + 1u == NB ? 0u : buf + 1u;
            if (tile >= nt || (int)k0 > (int)qw + 31 + lead) continue; /* no key of the tile is visible to these rows */
            const bool masked = (int)(k0 + KT - 1u) > (int)qw + lead;
            f32x16 sc[KT / 32];
            float tm = -INFINITY;
#pragma unroll
            for (u32 n = 0; n < KT / 32; ++n) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[n][i] = 0.0f;
#pragma unroll
                for (u32 x = 0; x < D / 16; ++x) {
                    U4H8 kk;
                    kk.u = *(const uint4 *)(kt + (32u * n + r) * RB + 16u * swz_k(32u * n + r, 2u * x + hf));
                    sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kk.v, qreg[x].v, sc[n], 0, 0, 0);
                }
                if (masked) {
#pragma unroll
                    for (u32 i = 0; i < 16; ++i) {
                        const int key = (int)(k0 + 32u * n + 8u * (i / 4u) + 4u * hf + i % 4u);
                        if (key > limit) sc[n][i] = -INFINITY;
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) tm = fmaxf(tm, sc[n][i]);
            }
            tm = fmaxf(tm, __shfl_xor(tm, 32));
            /* The reference point follows a row's maximum at a distance of up to 2^8 (weights of up to 256 round to fp16
             * as those up to 1 do): most tiles then rescale nothing, 470 -> 452 us for 10,216 rows of 32 heads. */
            if (__any((tm - m) * g.c > 8.0f)) {
                const float mn = fmaxf(m, tm), corr = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * g.c);
                m = mn;
                l *= corr;
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= corr;
            }
            const float mc = m == -INFINITY ? 0.0f : m * g.c;
            U4H8 p[KT / 16];
#pragma unroll
            for (int i = 0; i < KT / 2; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(sc[i >> 4][i & 15], g.c, -mc));
                l += e;
                p[i >> 3].h[i & 7] = (h16)e;
            }
            /* the lane's key of the transposing read: 16 y + 4 hf + lane / 4 % 4 (and + 8), its dims
             * 32 d + 16 (lane / 16 % 2) + 4 (lane % 4) */
            auto v_operand = [&](u32 y, u32 d) {
                const u32 key = 16u * y + 4u * hf + ((lane >> 2) & 3u), pc = 4u * d + 2u * ((lane >> 4) & 1u) + ((lane >> 1) & 1u);
                const uint2 lo = lds_read_tr4(vt + key * RB + 16u * swz_v(key, pc) + 8u * (lane & 1u));
                const uint2 hi = lds_read_tr4(vt + (key + 8u) * RB + 16u * swz_v(key + 8u, pc) + 8u * (lane & 1u));
                return make_uint4(lo.x, lo.y, hi.x, hi.y);
            };
            if (special) {
                for (u32 d = 0; d < D / 32; ++d) {
                    f32x16 n;
#pragma unroll
                    for (int i = 0; i < 16; ++i) n[i] = 0.0f;
#pragma unroll
                    for (u32 y = 0; y < KT / 16; ++y) {
                        U4H8 fin, code, seen;
                        split_special(v_operand(y, d), fin, code);
#pragma unroll
                        for (u32 i = 0; i < 8; ++i) {
                            const int key = (int)(k0 + 16u * y + 8u * (i / 4u) + 4u * hf + i % 4u);
                            seen.h[i] = (h16)(key > limit ? 0.0f : 1.0f);
                        }
                        n = __builtin_amdgcn_mfma_f32_32x32x16_f16(code.v, seen.v, n, 0, 0, 0);
#pragma unroll
                        for (u32 dd = 0; dd < D / 32; ++dd)
                            if (dd == d) o[dd] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fin.v, p[y].v, o[dd], 0, 0, 0);
                    }
#pragma unroll
                    for (u32 dd = 0; dd < D / 32; ++dd)
                        if (dd == d)
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[dd][i] = with_special(o[dd][i], n[i]);
                }
            } else {
#pragma unroll
                for (u32 y = 0; y < KT / 16; ++y) {
#pragma unroll
                    for (u32 d = 0; d < D / 32; ++d) {
                        U4H8 vv;
                        vv.u = v_operand(y, d);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv.v, p[y].v, o[d], 0, 0, 0);
                    }
                }
            }
        }
        l += __shfl_xor(l, 32);
        wait_barrier<0>(); /* the tiles' LDS is free (loads past the last tile have landed) */
        if constexpr (WG > 1) {
            if (gi > 0u) {
                uint8_t *dst = sm + ((gi - 1u) * WQ + wq) * SLOT;
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *(float4 *)(dst + (4u * d + q) * 1024u + 16u * lane) = make_float4(o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]);
                *(float2 *)(dst + 32u * D * 4u + 8u * lane) = make_float2(m, l);
            }
            __syncthreads();
            if (gi == 0u) {
                float mg[WG], lg[WG];
                mg[0] = m;
                lg[0] = l;
                float M = m;
#pragma unroll
                for (u32 x = 1; x < WG; ++x) {
                    const float2 v = *(const float2 *)(sm + ((x - 1u) * WQ + wq) * SLOT + 32u * D * 4u + 8u * lane);
                    mg[x] = v.x;
                    lg[x] = v.y;
                    M = fmaxf(M, v.x);
                }
                l = 0.0f;
#pragma unroll
                for (u32 x = 0; x < WG; ++x) {
                    /* a group without weight counts nothing; weight without a maximum is NaN, which goes on */
                    const float w = lg[x] == 0.0f ? 0.0f : mg[x] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((mg[x] - M) * g.c);
                    l += lg[x] * w;
#pragma unroll
                    for (int d = 0; d < D / 32; ++d)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            if (x == 0u) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) o[d][4 * q + i] *= w;
                            } else {
                                const float4 v = *(const float4 *)(sm + ((x - 1u) * WQ + wq) * SLOT + (4u * d + q) * 1024u + 16u * lane);
                                o[d][4 * q] = fmaf(v.x, w, o[d][4 * q]);
                                o[d][4 * q + 1] = fmaf(v.y, w, o[d][4 * q + 1]);
                                o[d][4 * q + 2] = fmaf(v.z, w, o[d][4 * q + 2]);
                                o[d][4 * q + 3] = fmaf(v.w, w, o[d][4 * q + 3]);
                            }
                        }
                }
            }
            __syncthreads();
        }
    };
    attend(std::false_type{});
    /* 0 times a value that is not finite is NaN: a result that is not may hold one that its row does not see, and the
     * tile is done again with such values apart.  (Told from the results the first pass needs nothing for it: looking
     * for them in every tile of mixed visibility took 830 us instead of 476 for 10,216 rows of 32 heads, in registers.) */
    bool odd = false;
    if (gi == 0u) {
        const float li = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) odd |= !(fabsf(o[d][i] * li) < INFINITY);
    }
    if (__syncthreads_or(odd)) attend(std::true_type{});
    if (gi == 0u) {
        const float li = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (u32 d = 0; d < D / 32; ++d)
#pragma unroll
            for (u32 q = 0; q < 4; ++q) {
                union {
                    h16 x[4];
                    uint2 u;
                } v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v.x[i] = (h16)(o[d][4 * q + i] * li);
                *(uint2 *)(sm + (32u * wq + r) * RB + 16u * swz_k(r, 4u * d + q) + 8u * hf) = v.u;
            }
    }
    __syncthreads();
    for (u32 x = t; x < BQ * PPR; x += 64u * WQ * WG) {
        const u32 row = x / PPR, pc = x % PPR;
        if (q0 + row >= nq) break;
        store_any(a.out + (uint64_t)(qa + q0 + row) * a.os + h * D + 8u * pc, *(const uint4 *)(sm + row * RB + 16u * swz_k(row & 31u, pc)));
    }
}

template <int D, int WQ, int WG, int KT, int NB>
hipError_t launch(hipStream_t st, const uocr_packed_args &a) {
    PackedGrid g;
    g.a = a;
    g.slots = a.q_tokens / (WQ * 32u) + a.n_seqs;
    g.group = a.heads / a.kv_heads;
    g.c = a.scale * 1.4426950408889634f;
    const u32 blocks = g.slots * a.heads; /* the operator's limit keeps it in range */
    const bool dma = ((((uintptr_t)a.k | (uintptr_t)a.v) & 15u) | ((a.ks | a.vs) & 7u)) == 0u;
    if (dma) hipLaunchKernelGGL((k_packed_attention<D, WQ, WG, KT, NB, true>), dim3(blocks), dim3(64 * WQ * WG), 0, st, g);
    else hipLaunchKernelGGL((k_packed_attention<D, WQ, WG, KT, NB, false>), dim3(blocks), dim3(64 * WQ * WG), 0, st, g);
    return hipGetLastError();
}

/* Measured (us; wavefronts along queries x along keys, keys per tile; head_dim
 * 128; x: tiles of 128 rows, all heads, and one more for each sequence):
 *   heads x sequences x rows     x     4 x 1, 64   2 x 4, 32   4 x 2, 64
 *   10 x 1 x 64                  10         7.4         9.4         8.7
 *   10 x 1 x 932                 80        23.1        18.2        21.2
 *   32 x 1 x 700                192        18.9        20.9        17.5
 *   10 x 1 x 2500               200        51.3        38.6        42.3
 *   10 x 3 x 932                240        24.1        30.9        22.6
 *   10 x 12 x 200               300        15.6        22.4        22.1
 *   10 x 2 x 2000               330        46.9        53.0        39.8
 *   32 x 1 x 2000               512        53.1        71.9        49.9
 *   32 x 4 x 4001              4128       599.6       865.4       649.4   (894 TFLOP/s)
 * Few tiles leave CUs or their second block idle: then wavefronts share the
 * walk over long keys; many want the tile with the fewest passes over K and V.
 * head_dim 64 goes alike (512 tiles: 35.2, 47.8, 33.0). */
template <int D>
hipError_t choose(hipStream_t st, const uocr_packed_args &a) {
    const uint64_t x = ((uint64_t)a.q_tokens / 128u + a.n_seqs) * a.heads, keys = a.k_tokens / a.n_seqs;
    if (keys >= 256u && (x <= 160u || (x <= 240u && keys >= 1000u))) return launch<D, 2, 4, 32, 2>(st, a);
    if (x <= 512u && keys >= 320u) return launch<D, 4, 2, 64, 2>(st, a);
    return launch<D, 4, 1, 64, 2>(st, a);
}

}  // namespace

hipError_t uocr_launch_packed_attention(hipStream_t st, const uocr_packed_args *a) {
    return a->dim == 128u ? choose<128>(st, *a) : choose<64>(st, *a);
}
