// p8x_attn.hip -- attention of drafted tokens over the cache and each other (p8x_attn_tree), and the attention weight
// that accepted tokens gave (p8x_kv_score).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_kv.h"

namespace p8x {

// 8 elements of a query or draft row as f32; drafts in f32 are rounded to the cache's type
__device__ __forceinline__ void load8(const void *p, size_t i, bool f32, int bf16, bool round, float *o) {
    for (int e = 0; e < 8; ++e) {
        o[e] = f32 ? ((const float *)p)[i + e] : from16(((const uint16_t *)p)[i + e], bf16);
        if (round) o[e] = from16(to16(o[e], bf16), bf16);
    }
}

__device__ __forceinline__ uint64_t token_mask(const DraftDev &d, int tok, int i) {
    return d.mask ? d.mask[tok] : i == 63 ? ~0ull : (2ull << i) - 1;
}

template <int D>
__global__ __launch_bounds__(256) void k_attn(KvDev c, DraftDev d, void *out, size_t ldo, size_t hso, float *lse) {
    __shared__ float q[D], p[256], red[8], acc[256];
    const int s = blockIdx.z, head = blockIdx.y, i = blockIdx.x, t = threadIdx.x;
    int first;
    const int nt = seq_tokens(d, s, first);
    if (i >= nt) return;
    const int tok = first + i, h = head / d.G;
    const uint64_t mask = token_mask(d, tok, i);
    if (t < D) q[t] = d.q_f32 ? ((const float *)d.q)[(size_t)tok * d.ld_q + head * d.hs_q + t] : from16(((const uint16_t *)d.q)[(size_t)tok * d.ld_q + head * d.hs_q + t], c.bf16);
    const int n = seq_len(c, s), total = n + nt;
    float m = -INFINITY, l = 0, o = 0;
    const int part = t / D, e = t % D;   // PV: 256 / D parts of the slots
    for (int j0 = 0; j0 < total; j0 += 256) {
        __syncthreads();
        const int j = j0 + t;
        float x = -INFINITY;
        if (j < n) {
            const int64_t at = slot_offset(c, s, j);
            if (at >= 0) {
                float a = 0;
                for (int k = 0; k < D; ++k) a = fmaf(q[k], from16(c.k[at + h * c.head_stride + k], c.bf16), a);
                x = a * d.scale;
            }
        } else if (j < total && (mask >> (j - n) & 1)) {
            float a = 0, r[8];
            for (int k = 0; k < D; k += 8) {
                load8(d.k, (size_t)(first + j - n) * d.ld_kv + h * d.hs_kv + k, d.kv_f32, c.bf16, d.kv_f32, r);
                for (int u = 0; u < 8; ++u) a = fmaf(q[k + u], r[u], a);
            }
            x = a * d.scale;
        }
        float mx = x;
        for (int b = 32; b; b >>= 1) mx = fmaxf(mx, __shfl_xor(mx, b));
        if ((t & 63) == 0) red[t >> 6] = mx;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float base = mn == -INFINITY ? 0.0f : mn, al = expf(m - base);
        const float w = x == -INFINITY ? 0.0f : expf(x - base);
        p[t] = x == -INFINITY ? -1.0f : w;   // -1: not seen
        float sum = w;
        for (int b = 32; b; b >>= 1) sum += __shfl_xor(sum, b);
        if ((t & 63) == 0) red[4 + (t >> 6)] = sum;
        __syncthreads();
        l = l * al + (red[4] + red[5] + red[6] + red[7]);
        o *= al;
        m = mn;
        for (int jj = part; jj < 256 && j0 + jj < total; jj += 256 / D) {
            const float w2 = p[jj];
            if (w2 < 0.0f) continue;
            const int j2 = j0 + jj;
            float v;
            if (j2 < n) v = from16(c.v[slot_offset(c, s, j2) + h * c.head_stride + e], c.bf16);
            else {
                const size_t at = (size_t)(first + j2 - n) * d.ld_kv + h * d.hs_kv + e;
                v = d.kv_f32 ? from16(to16(((const float *)d.v)[at], c.bf16), c.bf16) : from16(((const uint16_t *)d.v)[at], c.bf16);
            }
            o = fmaf(w2, v, o);
        }
    }
    __syncthreads();
    acc[t] = o;
    __syncthreads();
    if (t < D) {
        for (int k = 1; k < 256 / D; ++k) o += acc[t + k * D];
        const float r = l == 0.0f ? 0.0f : o / l;
        const size_t at = (size_t)tok * ldo + head * hso + t;
        if (d.q_f32) ((float *)out)[at] = r;
        else ((uint16_t *)out)[at] = to16(r, c.bf16);
    }
    if (t == 0 && lse) lse[(size_t)tok * c.n_kv * d.G + head] = m == -INFINITY ? -INFINITY : m + logf(l);
}

size_t attn_workspace(const KvDev &, const DraftDev &, int) { return 0; }

int launch_attn_tree(const KvDev &c, const DraftDev &d, int D, void *out, size_t ldo, size_t hso, float *lse, void *, size_t, hipStream_t st) {
    const dim3 grid(d.max_tokens, c.n_kv * d.G, c.n_seq);
    if (D == 64) k_attn<64><<<grid, 256, 0, st>>>(c, d, out, ldo, hso, lse);
    else if (D == 128) k_attn<128><<<grid, 256, 0, st>>>(c, d, out, ldo, hso, lse);
    else k_attn<256><<<grid, 256, 0, st>>>(c, d, out, ldo, hso, lse);
    return hip_check(hipGetLastError(), "p8x_attn_tree launch");
}

// One thread a slot or accepted token of a key/value head.
template <int D>
__global__ __launch_bounds__(256) void k_score(KvDev c, DraftDev d, const uint64_t *accept, const float *lse, float decay, const float *score, float *score_out) {
    const int s = blockIdx.z, h = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
    int first = 0;
    const int nt = d.n_tokens ? seq_tokens(d, s, first) : 0, n = seq_len(c, s);
    const uint64_t all = nt >= 64 ? ~0ull : (1ull << nt) - 1, acc = accept ? accept[s] & all : all;
    const int cnt = __popcll(acc);
    if (j >= min(n + cnt, c.max_len)) return;
    int tj = -1;   // the accepted token that becomes slot j
    if (j >= n) {
        uint64_t b = acc;
        for (int r = j - n; r; --r) b &= b - 1;
        tj = __ffsll((unsigned long long)b) - 1;
    }
    const int64_t at = tj < 0 ? slot_offset(c, s, j) : 0;
    float sum = 0;
    if (at >= 0)
        for (uint64_t b = acc; b; b &= b - 1) {
            const int i = __ffsll((unsigned long long)b) - 1, tok = first + i;
            if (tj >= 0 && !(token_mask(d, tok, i) >> tj & 1)) continue;
            for (int g = 0; g < d.G; ++g) {
                const int head = h * d.G + g;
                float a = 0;
                for (int k = 0; k < D; k += 8) {
                    float q[8], r[8];
                    load8(d.q, (size_t)tok * d.ld_q + head * d.hs_q + k, d.q_f32, c.bf16, false, q);
                    if (tj < 0) load8(c.k, at + h * c.head_stride + k, false, c.bf16, false, r);
                    else load8(d.k, (size_t)(first + tj) * d.ld_kv + h * d.hs_kv + k, d.kv_f32, c.bf16, d.kv_f32, r);
                    for (int u = 0; u < 8; ++u) a = fmaf(q[u], r[u], a);
                }
                sum += expf(a * d.scale - lse[(size_t)tok * c.n_kv * d.G + head]);
            }
        }
    const size_t o = ((size_t)s * c.n_kv + h) * c.max_len + j;
    score_out[o] = tj < 0 ? decay * score[o] + sum : sum;
}

int launch_kv_score(const KvDev &c, const DraftDev &d, int D, const uint64_t *accept, const float *lse, float decay, const float *score,
                    float *score_out, hipStream_t st) {
    const dim3 grid((c.max_len + 255) / 256, c.n_kv, c.n_seq);
    if (D == 64) k_score<64><<<grid, 256, 0, st>>>(c, d, accept, lse, decay, score, score_out);
    else if (D == 128) k_score<128><<<grid, 256, 0, st>>>(c, d, accept, lse, decay, score, score_out);
    else k_score<256><<<grid, 256, 0, st>>>(c, d, accept, lse, decay, score, score_out);
    return hip_check(hipGetLastError(), "p8x_kv_score launch");
}

}  // namespace p8x
