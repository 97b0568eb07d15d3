// p8x_attn.h -- operands of the matrix-core products with queries and cached keys (p8x_attn.hip, p8x_score.hip, p8x_prompt.hip).
#pragma once
#include "p8x_kv.h"

namespace p8x {

__device__ __forceinline__ uint64_t token_mask(const DraftDev &d, int tok, int i) {
    return d.mask ? d.mask[tok] : i == 63 ? ~0ull : (2ull << i) - 1;
}

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bhalf2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));

template <bool BF>
__device__ __forceinline__ float4v mfma(uint4v a, uint4v b, float4v c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
// two f32 rounded to 16 bits, to nearest even
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x, y}, bhalf2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x, y}, half2v));
}
template <bool BF>
__device__ __forceinline__ float part_lo(uint32_t w) { return BF ? __builtin_bit_cast(float, w << 16) : from_f16((uint16_t)w); }
template <bool BF>
__device__ __forceinline__ float part_hi(uint32_t w) { return BF ? __builtin_bit_cast(float, w & 0xFFFF0000u) : from_f16((uint16_t)(w >> 16)); }

// 8 f32 as N operands of 16 bits that sum to them: N x 11 (fp16) or N x 8 (bf16) bits
template <bool BF, int N>
__device__ __forceinline__ void split8(const float *f, uint4v *o) {
    float r[8];
    for (int e = 0; e < 8; ++e) r[e] = f[e];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = pack2<BF>(r[2 * e], r[2 * e + 1]);
            o[n][e] = w;
            if (n + 1 < N) {
                r[2 * e] -= part_lo<BF>(w);
                r[2 * e + 1] -= part_hi<BF>(w);
            }
        }
}

// A lane's pieces of an f32 query row, 8 elements at 32 k, for splitting: fp16 parts need the row scaled to 2^13 (the lanes
// 16 apart hold the rest of the row). Returns the factor of a product, f with that power taken back out.
template <int C, bool BF>
__device__ __forceinline__ float load_split(const float *q, bool on, float f, float (&x)[C][8]) {
    float mx = 0.0f;
#pragma unroll
    for (int k = 0; k < C; ++k) {
        const float4v lo = on ? *(const float4v *)(q + 32 * k) : float4v{0, 0, 0, 0}, hi = on ? *(const float4v *)(q + 32 * k + 4) : float4v{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[k][e] = lo[e];
            x[k][e + 4] = hi[e];
            mx = fmaxf(mx, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
        }
    }
    if constexpr (!BF) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const int ex = mx > 0.0f && mx < INFINITY ? 13 - (int)((__builtin_bit_cast(uint32_t, mx) >> 23) - 127) : 0;
        const int e1 = min(ex, 100);   // in two steps: 2^ex may be beyond f32
        const float s1 = ldexpf(1.0f, e1), s2 = ldexpf(1.0f, ex - e1);
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[k][e] = x[k][e] * s1 * s2;
        f = ldexpf(f, -ex);
    }
    return f;
}

// Whether a dword holds a 16-bit infinity or NaN, and the dword without them.
template <bool BF>
__device__ __forceinline__ bool take_odd(uint32_t &w) {
    constexpr uint32_t inf = BF ? 0x7F80u : 0x7C00u;
    const bool lo = (w & inf) == inf, hi = (w >> 16 & inf) == inf;
    w &= (lo ? 0 : 0xFFFFu) | (hi ? 0 : 0xFFFF0000u);
    return lo || hi;
}

// 16 bytes a lane from base + off to LDS at `to` + 16 lane, without a wait. Written by hand: the compiler, which knows no other
// wait than for all of these, would put one before every read of LDS. M0 holds `to` while the load is issued; five wait
// states lie between it, or a VALU write of the base, and the load. Nothing is loaded into registers.
__device__ __forceinline__ void load_lds(const uint16_t *base, uint32_t off, uint32_t to) {
    uint32_t m0;
    __asm__ volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0" : "=&s"(m0) : "v"(off), "s"(base), "s"(to) : "memory");
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 8 elements of a draft row as the cache holds them
__device__ __forceinline__ uint4v draft8(const void *p, size_t at, int f32, int bf16) {
    if (!f32) return *(const uint4v *)((const uint16_t *)p + at);
    const float4v lo = *(const float4v *)((const float *)p + at), hi = *(const float4v *)((const float *)p + at + 4);
    uint4v o;
    for (int e = 0; e < 2; ++e) {
        o[e] = to16(lo[2 * e], bf16) | (uint32_t)to16(lo[2 * e + 1], bf16) << 16;
        o[e + 2] = to16(hi[2 * e], bf16) | (uint32_t)to16(hi[2 * e + 1], bf16) << 16;
    }
    return o;
}

}  // namespace p8x
