// p8x_kv.h -- what the cache, attention and norm kernels share: the cache and the drafted tokens as kernel arguments
// (the structs of p8x.h after the host's checks), slot addresses, conversions.
#pragma once
#include "p8x_internal.h"

namespace p8x {

struct KvDev {
    uint16_t *k, *v;
    size_t page_stride, head_stride, slot_stride;
    const int32_t *pages; size_t ld_pages;
    const int32_t *len;
    int page_size, n_pages, max_len, n_seq, n_kv, bf16;
};

struct DraftDev {
    const int32_t *first;
    const void *k, *v; size_t ld_kv, hs_kv; int kv_f32;
    const uint64_t *mask;
    const void *q; size_t ld_q, hs_q; int q_f32;
    int n_tokens, max_tokens, G;   // G: query heads of a key/value head
    float scale;
};

// launchers (p8x_norm.hip, p8x_attn.hip, p8x_kv.hip); arguments checked by p8x_kv_host.cpp
int launch_norm_residual(const p8x_norm_args &a, hipStream_t st);
int launch_attn_tree(const KvDev &c, const DraftDev &d, int head_dim, void *out, size_t ldo, size_t hso, float *lse, void *ws, size_t ws_bytes,
                     hipStream_t st);
size_t attn_workspace(const KvDev &c, const DraftDev &d, int head_dim);
int launch_kv_score(const KvDev &c, const DraftDev &d, int head_dim, const uint64_t *accept, const float *lse, float decay, const float *score,
                    float *score_out, hipStream_t st);
int launch_kv_append(const KvDev &c, const DraftDev &d, int head_dim, const uint64_t *accept, const int32_t *at, int32_t *pos, int32_t *len_out,
                     hipStream_t st);
int launch_kv_evict(const KvDev &c, int head_dim, const p8x_evict_args &a, hipStream_t st);
size_t kv_evict_workspace(const KvDev &c, int budget);

__device__ __forceinline__ int seq_len(const KvDev &c, int s) { return min(max(c.len[s], 0), c.max_len); }

// element offset of a slot's row of head 0 in the pool, or -1 where the table has no page for it
__device__ __forceinline__ int64_t slot_offset(const KvDev &c, int s, int slot) {
    if (!c.pages) return (int64_t)((size_t)s * c.page_stride + (size_t)slot * c.slot_stride);
    const int pg = slot / c.page_size;
    const int page = c.pages[(size_t)s * c.ld_pages + pg];
    if ((unsigned)page >= (unsigned)c.n_pages) return -1;
    return (int64_t)((size_t)page * c.page_stride + (size_t)(slot - pg * c.page_size) * c.slot_stride);
}

// tokens of sequence s: the first one's row, how many (0 where `first` is out of order or range)
__device__ __forceinline__ int seq_tokens(const DraftDev &d, int s, int &a) {
    a = d.first[s];
    const int b = d.first[s + 1];
    return a < 0 || b < a || b > d.n_tokens ? 0 : min(b - a, d.max_tokens);
}

__device__ __forceinline__ float from_f16(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ __forceinline__ float from_bf16(uint16_t h) { return __builtin_bit_cast(float, (uint32_t)h << 16); }
__device__ __forceinline__ uint16_t to_f16(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
// round to nearest even; a NaN stays one
__device__ __forceinline__ uint16_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
__device__ __forceinline__ float from16(uint16_t h, int bf16) { return bf16 ? from_bf16(h) : from_f16(h); }
__device__ __forceinline__ uint16_t to16(float f, int bf16) { return bf16 ? to_bf16(f) : to_f16(f); }

// element i of a P8X_F32 / P8X_F16 / P8X_BF16 array as f32
__device__ __forceinline__ float load_as_f32(const void *p, int dtype, size_t i) {
    if (dtype == P8X_F32) return ((const float *)p)[i];
    return from16(((const uint16_t *)p)[i], dtype == P8X_BF16);
}

}  // namespace p8x
