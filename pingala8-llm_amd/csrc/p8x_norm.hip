// p8x_norm.hip -- the end of one block and the start of the next (p8x_norm_residual): h' = h + alpha a(gate) N_post(y),
// x = N_pre(h').
//
// One workgroup a row, the row in registers between its one read and its one write; two sums through LDS (three or four
// with layer norms: mean, then the sum of squares about it). Bound by HBM for many rows and by the launch and
// three memory round trips for few: 1500 rows of 5120 with a gate (138 MB) 31.8 us, 4.35 TB/s, of 8192 (221 MB) 48.5 us, 4.6 TB/s; one row of
// 4096 4.0 us.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_kv.h"

namespace p8x {

struct NormDev {
    p8x_norm_args a;
};

// Four elements of a row of C, raw. VEC: i .. i + 3, all of them there, as they lie in memory, so that a load is not waited for
// before the next is issued (a choice of the type at run time would end each with moves of what it loaded); else i, i + d,
// i + 2 d, i + 3 d as f32, 0 past the row (d the workgroup's threads: neighbours in neighbouring lanes).
template <bool VEC, bool WIDE>
struct Four {
    uint4 r;
    __device__ __forceinline__ void load(const void *p, int dtype, size_t row, int i, int d, int C) {
        if constexpr (VEC && WIDE) r = *(const uint4 *)((const float *)p + row + i);
        else if constexpr (VEC) {
            const uint2 v = *(const uint2 *)((const uint16_t *)p + row + i);
            r.x = v.x, r.y = v.y;
        } else {
            float o[4];
            for (int e = 0; e < 4; ++e) o[e] = i + e * d < C ? load_as_f32(p, dtype, row + i + e * d) : 0.0f;
            r = __builtin_bit_cast(uint4, o);
        }
    }
    __device__ __forceinline__ void get(int dtype, float (&o)[4]) const {
        if constexpr (VEC && !WIDE) {
            const int bf = dtype == P8X_BF16;
            o[0] = from16((uint16_t)r.x, bf), o[1] = from16((uint16_t)(r.x >> 16), bf), o[2] = from16((uint16_t)r.y, bf), o[3] = from16((uint16_t)(r.y >> 16), bf);
        } else {
            o[0] = __builtin_bit_cast(float, r.x), o[1] = __builtin_bit_cast(float, r.y), o[2] = __builtin_bit_cast(float, r.z), o[3] = __builtin_bit_cast(float, r.w);
        }
    }
};
template <bool VEC>
__device__ __forceinline__ void store4(void *p, int dtype, size_t row, int i, int d, int C, const float (&v)[4]) {
    const int bf = dtype == P8X_BF16;
    if constexpr (VEC) {
        if (dtype == P8X_F32) *(float4 *)((float *)p + row + i) = make_float4(v[0], v[1], v[2], v[3]);
        else *(uint2 *)((uint16_t *)p + row + i) = make_uint2(to16(v[0], bf) | (uint32_t)to16(v[1], bf) << 16, to16(v[2], bf) | (uint32_t)to16(v[3], bf) << 16);
    } else {
        for (int e = 0; e < 4; ++e) {
            if (i + e * d >= C) break;
            if (dtype == P8X_F32) ((float *)p)[row + i + e * d] = v[e];
            else ((uint16_t *)p)[row + i + e * d] = to16(v[e], bf);
        }
    }
}

// sum over the workgroup, in every thread; red: used by no other call of the launch
__device__ __forceinline__ float block_sum(float v, float *red) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if (nw == 1) return v;
    if (lane == 0) red[w] = v;
    __syncthreads();
    float t = 0;
    for (int i = 0; i < nw; ++i) t += red[i];
    return t;
}

// 1 / (1 + e^-g) to a few units in the last place: 2^(t + r), t + r = -g log2 e to more than f32. Where 2^t is 0 or infinite, r is
// of no use, and infinite or NaN where t itself has overflowed.
__device__ __forceinline__ float sigmoid(float g) {
    const float t = g * -1.44269502f, r = fmaf(g, -1.44269502f, -t) + g * -1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_amdgcn_rcpf(1.0f + (e > 0.0f && e < INFINITY ? fmaf(e, r * 0.693147182f, e) : e));
}

// NV groups of four elements a thread, strided by the workgroup's width; Y32, H32, G32: y, h, gate are f32 (VEC).
template <int NV, bool VEC, bool Y32, bool H32, bool G32>
__global__ __launch_bounds__(1024) void k_norm(NormDev J) {
    // h and gate are loaded with y where all three fit the 128 registers of 1024 threads, else after the first norm (all at once: 50
    // registers through memory, 300 rows of 24576 74 us for 42)
    constexpr bool LATE = NV * (VEC ? 1 : 2) > 5;
    __shared__ float red[4][16];
    const p8x_norm_args &a = J.a;
    const size_t row = blockIdx.x;
    const int C = a.C, d = VEC ? 1 : blockDim.x, step = 4 * blockDim.x, c0 = VEC ? 4 * threadIdx.x : threadIdx.x;
    const bool gated = a.y && a.gate;
    Four<VEC, Y32> ry[NV];
    Four<VEC, H32> rh[NV];
    Four<VEC, G32> rg[NV];
    float u[NV][4], h[NV][4];
    // groups past the row load its last ones again, and count as zeros
    auto place = [&](int i) { return VEC ? min(i * step + c0, C - 4) : i * step + c0; };
    auto load_h = [&](int i) { rh[i].load(a.h, a.h_dtype, row * a.ldh, place(i), d, C); };
    auto load_g = [&](int i) {
        if (gated) rg[i].load(a.gate, a.gate_dtype, row * a.ld_gate, place(i), d, C);
    };
    auto value = [&](const auto &r, int dtype, int i, float (&v)[4]) {
        r.get(dtype, v);
        if (i * step + c0 >= C)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = 0.0f;
    };
    if (a.y)
#pragma unroll
        for (int i = 0; i < NV; ++i) ry[i].load(a.y, a.y_dtype, row * a.ldy, place(i), d, C);
    if (!LATE || !a.y)
#pragma unroll
        for (int i = 0; i < NV; ++i) load_h(i), load_g(i);
    auto norm = [&](float (&v)[NV][4], int kind, const float *w, const float *b, float eps, int r) {
        if (kind == P8X_NORM_NONE) return;
        float mean = 0.0f, s = 0.0f;
        if (kind == P8X_NORM_LAYER) {
#pragma unroll
            for (int i = 0; i < NV; ++i) s += v[i][0] + v[i][1] + v[i][2] + v[i][3];
            mean = block_sum(s, red[2 * r]) / (float)C;
            s = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[i][e] = i * step + c0 + e * d < C ? v[i][e] - mean : 0.0f;
                s = fmaf(v[i][e], v[i][e], s);
            }
        const float inv = 1.0f / sqrtf(block_sum(s, red[2 * r + 1]) / (float)C + eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = place(i);
            float wv[4] = {1, 1, 1, 1}, bv[4] = {};
            Four<VEC, true> rw;
            if (w) rw.load(w, P8X_F32, 0, c, d, C), rw.get(P8X_F32, wv);
            if (b) rw.load(b, P8X_F32, 0, c, d, C), rw.get(P8X_F32, bv);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = v[i][e] * inv * wv[e] + bv[e];
        }
    };
    if (a.y) {
#pragma unroll
        for (int i = 0; i < NV; ++i) value(ry[i], a.y_dtype, i, u[i]);
        norm(u, a.post, a.w_post, a.b_post, a.eps_post, 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float g[4] = {1, 1, 1, 1};
            if (LATE) load_h(i), load_g(i);
            value(rh[i], a.h_dtype, i, h[i]);
            if (gated) rg[i].get(a.gate_dtype, g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (gated && a.gate_act == P8X_GATE_SIGMOID) g[e] = sigmoid(g[e]);
                if (i * step + c0 + e * d < C) h[i][e] += a.alpha * (g[e] * u[i][e]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) value(rh[i], a.h_dtype, i, h[i]);
    }
    if (a.h_out)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * step + c0 < C) store4<VEC>(a.h_out, a.h_dtype, row * a.ldho, i * step + c0, d, C, h[i]);
    if (!a.x) return;
    norm(h, a.pre, a.w_pre, a.b_pre, a.eps_pre, 1);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (i * step + c0 < C) store4<VEC>(a.x, a.x_dtype, row * a.ldx, i * step + c0, d, C, h[i]);
}

template <int NV>
static void norm_run(const NormDev &J, int nt, bool vec, hipStream_t st) {
    const p8x_norm_args &a = J.a;
    if (!vec) k_norm<NV, false, true, true, true><<<a.n, nt, 0, st>>>(J);
    else {
        const bool y = !a.y || a.y_dtype == P8X_F32, h = a.h_dtype == P8X_F32, g = !a.y || !a.gate || a.gate_dtype == P8X_F32;
        const int k = y * 4 + h * 2 + g;
        (k == 0 ? k_norm<NV, true, false, false, false> : k == 1 ? k_norm<NV, true, false, false, true> : k == 2 ? k_norm<NV, true, false, true, false> :
         k == 3 ? k_norm<NV, true, false, true, true> : k == 4 ? k_norm<NV, true, true, false, false> : k == 5 ? k_norm<NV, true, true, false, true> :
         k == 6 ? k_norm<NV, true, true, true, false> : k_norm<NV, true, true, true, true>)<<<a.n, nt, 0, st>>>(J);
    }
}

int launch_norm_residual(const p8x_norm_args &a, hipStream_t st) {
    const NormDev J{a};
    // four at a time where rows and pointers allow it (one at a time, 1500 rows of 5121: 35 us for 32 at 5120; one of 4097 6.6 for 4.0)
    bool vec = a.C % 4 == 0;
    auto four = [&](const void *p, int dtype, size_t ld) {
        if (p && ((uintptr_t)p % (dtype == P8X_F32 ? 16 : 8) || (a.n > 1 && ld % 4))) vec = false;
    };
    four(a.y, a.y_dtype, a.ldy);
    four(a.h, a.h_dtype, a.ldh);
    four(a.h_out, a.h_dtype, a.ldho);
    four(a.x, a.x_dtype, a.ldx);
    if (a.y) four(a.gate, a.gate_dtype, a.ld_gate);
    for (const float *w : {a.w_post, a.b_post, a.w_pre, a.b_pre}) four(w, P8X_F32, 0);
    // few rows: as many threads as groups of four, for the shortest chain (256 rows of 4096: 4.7 us, 5.7 with 256 threads); many:
    // 256 threads, so that several rows' loads and sums overlap on a compute unit (1500 rows of 5120: 33.3 us, 36.8 with 1024), and
    // twice or four times that from six groups a thread on (eight groups took 128 registers and memory for 50 more: 74 us for 35 at
    // 1500 rows of 6144, 83 for 48 at 8192)
    const int groups = (a.C + 3) / 4, most = a.n <= num_cus() ? 1024 : 256;
    int nt = std::min(most, (groups + 63) / 64 * 64);
    while ((groups + nt - 1) / nt > 5 && nt < 1024) nt *= 2;
    switch ((groups + nt - 1) / nt) {
    case 1: norm_run<1>(J, nt, vec, st); break;
    case 2: norm_run<2>(J, nt, vec, st); break;
    case 3: norm_run<3>(J, nt, vec, st); break;
    case 4:
    case 5: norm_run<5>(J, nt, vec, st); break;
    default: norm_run<8>(J, nt, vec, st); break;
    }
    return hip_check(hipGetLastError(), "p8x_norm_residual launch");
}

}  // namespace p8x
