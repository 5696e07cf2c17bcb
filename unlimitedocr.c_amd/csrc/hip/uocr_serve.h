/*
 * uocr_serve.h - launch interface of the operators that serve several
 * sequences: the paged KV cache (uocr_kv_pages.hip), the attention of packed
 * prompts (uocr_attn_packed.hip) and sampling (uocr_sample.hip).
 *
 * Internal to libunlimitedocr.so.  The operator ABI has checked the arguments.
 */
#ifndef UOCR_SERVE_H
#define UOCR_SERVE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#define UOCR_TENSOR_F32 2u /* as in uocr_format.h */

#define UOCR_SERVE_MAX_SEQS 65536u /* keeps grids and counts of tiles well inside their types */
#define UOCR_SERVE_MAX_HEADS 1024u
#define UOCR_SERVE_MAX_TOKENS 8388607u /* blocks of a launch, of up to 512 threads each: below 2^32 threads */

/* A paged cache: page_stride in values; pages of 2^shift tokens. */
struct uocr_kv {
    void *k, *v;
    uint16_t *ks, *vs;
    const int32_t *table;
    uint64_t page_stride;
    uint32_t table_stride, n_pages, n_seqs, heads, shift, dim;
    bool q8;
};

/* Strides in values. */
struct uocr_append_args {
    uocr_kv kv;
    const int32_t *seqs, *pos;
    uint32_t tokens, heads; /* heads 0: no queries */
    double log2_theta;
    bool rotate;
    const uint16_t *q, *k, *v;
    uint16_t *q_out, *k_out;
    uint64_t qs, ks, vs, qos, kos;
};

struct uocr_gather_args {
    uocr_kv kv;
    const int32_t *seqs, *pos;
    uint32_t tokens;
    uint16_t *k_out, *v_out;
    uint64_t kos, vos;
};

struct uocr_paged_args {
    uocr_kv kv;
    const int32_t *lengths;
    uint32_t hq;
    float scale;
    const uint16_t *q;
    uint16_t *out;
    uint64_t qs, os;
    float *part;
};

struct uocr_packed_args {
    const int32_t *q_starts, *k_starts;
    uint32_t n_seqs, q_tokens, k_tokens, heads, kv_heads, dim;
    float scale;
    const uint16_t *q, *k, *v;
    uint16_t *out;
    uint64_t qs, ks, vs, os;
};

struct uocr_sample_args {
    const void *logits;
    uint64_t stride;
    bool f32;
    uint32_t rows, vocab;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p, *uniform;
    void *ws;
    int32_t *tokens;
    float *probs;
};

hipError_t uocr_launch_kv_append(hipStream_t st, const uocr_append_args *a);
hipError_t uocr_launch_kv_gather(hipStream_t st, const uocr_gather_args *a);
size_t uocr_paged_attention_ws_bytes(uint32_t heads, uint32_t kv_heads, uint32_t dim);
hipError_t uocr_launch_paged_attention(hipStream_t st, const uocr_paged_args *a);
hipError_t uocr_launch_packed_attention(hipStream_t st, const uocr_packed_args *a);
size_t uocr_sample_ws_bytes(uint32_t rows, uint32_t vocab);
hipError_t uocr_launch_sample(hipStream_t st, const uocr_sample_args *a);

#ifdef __HIPCC__
/* Where a token stands: its page, or -1 where it has none. */
__device__ __forceinline__ int kv_page(const uocr_kv &c, int32_t seq, uint32_t pos) {
    const int p = c.table[(uint64_t)(uint32_t)seq * c.table_stride + (pos >> c.shift)];
    return (uint32_t)p < c.n_pages ? p : -1;
}

typedef unsigned long long u64;

__device__ __forceinline__ u64 lane64(u64 v, int lane) {
    return ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
template <int CTRL>
__device__ __forceinline__ u64 dpp64(u64 v) {
    return ((u64)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xf, 0xf, true) << 32) |
           (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}

/* Sums of what earlier lanes hold (all lanes are active): row_shr by 1, 2, 4, 8
 * within 16 lanes, where zeros come in, then the rows'. */
__device__ __forceinline__ u64 wave_before(u64 v) {
    u64 s = v;
    s += dpp64<0x111>(s);
    s += dpp64<0x112>(s);
    s += dpp64<0x114>(s);
    s += dpp64<0x118>(s);
    const u64 a = lane64(s, 15), b = a + lane64(s, 31), c = b + lane64(s, 47);
    const uint32_t row = (threadIdx.x & 63u) >> 4;
    return s - v + (row == 0u ? 0ull : row == 1u ? a : row == 2u ? b : c);
}

/* Rows that no alignment above a value's is known of: 16-byte loads and stores
 * at any value's boundary, which global memory instructions take. */
typedef uint32_t u32x4_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ uint4 load_any(const uint16_t *p) {
    const u32x4_any2 v = *(const u32x4_any2 *)p;
    return make_uint4(v.x, v.y, v.z, v.w);
}

__device__ __forceinline__ void store_any(uint16_t *p, uint4 v) {
    *(u32x4_any2 *)p = u32x4_any2{v.x, v.y, v.z, v.w};
}
#endif

#endif /* UOCR_SERVE_H */
