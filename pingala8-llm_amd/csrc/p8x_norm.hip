// p8x_norm.hip -- the end of one block and the start of the next (p8x_norm_residual): h' = h + alpha a(gate) N_post(y),
// x = N_pre(h').
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_kv.h"

namespace p8x {

struct NormDev {
    p8x_norm_args a;
};

__device__ __forceinline__ void store_from_f32(void *p, int dtype, size_t i, float v) {
    if (dtype == P8X_F32) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = to16(v, dtype == P8X_BF16);
}

// sum over the workgroup, in every thread; `at`: a slot of red that no earlier call of the launch used
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

// One workgroup a row, NV elements a thread in registers, strided by the workgroup's width.
template <int NV>
__global__ __launch_bounds__(1024) void k_norm(NormDev J) {
    __shared__ float red[4][16];
    const p8x_norm_args &a = J.a;
    const size_t row = blockIdx.x;
    const int C = a.C, nt = blockDim.x;
    float u[NV], h[NV];
    for (int i = 0; i < NV; ++i) {
        const int c = i * nt + threadIdx.x;
        h[i] = c < C ? load_as_f32(a.h, a.h_dtype, row * a.ldh + c) : 0.0f;
        u[i] = c < C && a.y ? load_as_f32(a.y, a.y_dtype, row * a.ldy + c) : 0.0f;
    }
    auto norm = [&](float (&v)[NV], int kind, const float *w, const float *b, float eps, int r) {
        if (kind == P8X_NORM_NONE) return;
        float mean = 0.0f;
        if (kind == P8X_NORM_LAYER) {
            float s = 0;
            for (int i = 0; i < NV; ++i) s += v[i];
            mean = block_sum(s, red[2 * r]) / (float)C;
        }
        float s = 0;
        for (int i = 0; i < NV; ++i) {
            v[i] = i * nt + (int)threadIdx.x < C ? v[i] - mean : 0.0f;
            s += v[i] * v[i];
        }
        const float inv = 1.0f / sqrtf(block_sum(s, red[2 * r + 1]) / (float)C + eps);
        for (int i = 0; i < NV; ++i) {
            const int c = i * nt + threadIdx.x;
            if (c < C) v[i] = v[i] * inv * (w ? w[c] : 1.0f) + (b ? b[c] : 0.0f);
        }
    };
    if (a.y) {
        norm(u, a.post, a.w_post, a.b_post, a.eps_post, 0);
        for (int i = 0; i < NV; ++i) {
            const int c = i * nt + threadIdx.x;
            if (c >= C) continue;
            float g = 1.0f;
            if (a.gate) {
                g = load_as_f32(a.gate, a.gate_dtype, row * a.ld_gate + c);
                if (a.gate_act == P8X_GATE_SIGMOID) g = 1.0f / (1.0f + expf(-g));
            }
            h[i] += a.alpha * (g * u[i]);
        }
    }
    if (a.h_out)
        for (int i = 0; i < NV; ++i) {
            const int c = i * nt + threadIdx.x;
            if (c < C) store_from_f32(a.h_out, a.h_dtype, row * a.ldho + c, h[i]);
        }
    if (!a.x) return;
    norm(h, a.pre, a.w_pre, a.b_pre, a.eps_pre, 1);
    for (int i = 0; i < NV; ++i) {
        const int c = i * nt + threadIdx.x;
        if (c < C) store_from_f32(a.x, a.x_dtype, row * a.ldx + c, h[i]);
    }
}

int launch_norm_residual(const p8x_norm_args &a, hipStream_t st) {
    const NormDev J{a};
    const int nt = std::min(1024, (a.C + 63) / 64 * 64), nv = (a.C + nt - 1) / nt;
    if (nv <= 4) k_norm<4><<<a.n, nt, 0, st>>>(J);
    else if (nv <= 8) k_norm<8><<<a.n, nt, 0, st>>>(J);
    else if (nv <= 16) k_norm<16><<<a.n, nt, 0, st>>>(J);
    else k_norm<32><<<a.n, nt, 0, st>>>(J);
    return hip_check(hipGetLastError(), "p8x_norm_residual launch");
}

}  // namespace p8x
