// p8x_prompt.hip -- causal attention of new tokens over the cache that holds them (p8x_attn_prompt).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_attn.h"

namespace p8x {

struct PromptJob {
    KvDev c;
    DraftDev d;
    void *out; size_t ldo, hso; int out_dtype;
    float *lse;
    int D;
};

// One workgroup a token and head, 256 slots at a time: a thread the score of one slot, then an element of the sums.
__global__ __launch_bounds__(256) void k_prompt_simple(PromptJob J) {
    __shared__ float q[256], p[256], red[4];
    __shared__ int64_t at[256];
    const KvDev &c = J.c;
    const DraftDev &d = J.d;
    const int t = threadIdx.x, D = J.D, head = blockIdx.y, h = head / d.G, s = blockIdx.z;
    int first;
    const int nt = seq_tokens(d, s, first), n = seq_len(c, s);
    auto across = [&](float v, bool top) {
        for (int o = 32; o; o >>= 1) v = top ? fmaxf(v, __shfl_xor(v, o)) : v + __shfl_xor(v, o);
        __syncthreads();
        if ((t & 63) == 0) red[t >> 6] = v;
        __syncthreads();
        return top ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : red[0] + red[1] + red[2] + red[3];
    };
    for (int i = blockIdx.x; i < nt; i += gridDim.x) {
        const int see = max(0, n - nt + i + 1);   // slots
        __syncthreads();
        if (t < D) q[t] = load_as_f32(d.q, d.q_f32 ? P8X_F32 : c.bf16 ? P8X_BF16 : P8X_F16, (size_t)(first + i) * d.ld_q + (size_t)head * d.hs_q + t);
        float m = -INFINITY, l = 0, o = 0;
        for (int j0 = 0; j0 < see; j0 += 256) {
            __syncthreads();
            const int j = j0 + t;
            const int64_t off = j < see ? slot_offset(c, s, j) : -1;
            float x = -INFINITY;
            if (off >= 0) {
                x = 0;
                const uint16_t *k = c.k + off + (size_t)h * c.head_stride;
                for (int e = 0; e < D; ++e) x = fmaf(q[e], from16(k[e], c.bf16), x);
                x *= d.scale;
            }
            at[t] = off;
            const float mx = fmaxf(m, across(x, true)), f = mx == -INFINITY ? 1.0f : expf(m - mx);
            p[t] = x == -INFINITY ? 0.0f : expf(x - mx);
            l = l * f + across(p[t], false);
            o *= f;
            m = mx;
            if (t < D)
                for (int k = 0; k < min(256, see - j0); ++k)
                    if (at[k] >= 0) o = fmaf(p[k], from16(c.v[at[k] + (size_t)h * c.head_stride + t], c.bf16), o);
        }
        const size_t to = (size_t)(first + i) * J.ldo + (size_t)head * J.hso + t;
        const float r = l == 0.0f ? 0.0f : o / l;
        if (t < D) {
            if (J.out_dtype == P8X_F32) ((float *)J.out)[to] = r;
            else ((uint16_t *)J.out)[to] = to16(r, J.out_dtype == P8X_BF16);
        }
        if (t == 0 && J.lse) J.lse[(size_t)(first + i) * c.n_kv * d.G + head] = l == 0.0f ? -INFINITY : m + logf(l);
    }
}

size_t attn_prompt_workspace(const KvDev &, const DraftDev &, int) { return 0; }

int launch_attn_prompt(const KvDev &c, const DraftDev &d, int D, void *out, int out_dtype, size_t ldo, size_t hso, float *lse, void *, size_t, hipStream_t st) {
    const PromptJob J{c, d, out, ldo, hso, out_dtype, lse, D};
    k_prompt_simple<<<dim3(std::min(d.max_tokens, 65535), c.n_kv * d.G, c.n_seq), 256, 0, st>>>(J);
    return hip_check(hipGetLastError(), "p8x_attn_prompt launch");
}

}  // namespace p8x
