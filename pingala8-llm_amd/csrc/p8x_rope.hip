// p8x_rope.hip -- rotary positions: heads of queries and keys, normed where the model does, rotated in place or to other rows
// (p8x_rope), or with the keys and values going to the cache (p8x_kv_append_rope).
//
// A head takes L lanes, 8 elements each: four pairs of it (elements 4 l .. of either half, or 8 l .. as neighbours) or 8
// elements that pass; a wave takes 64 / L heads of one token at a time, and several such groups in turn, two at a time. The angle of a pair is p freq mod 2^64, a wrapping integer product: its upper 32 bits
// are the turn to 2^-32 whatever the position (as an f32 product, position 131071 would be off by 0.008 radians). Sine and
// cosine by their series over an eighth of a turn either way, once for all heads of a wave.
//
// What bounds it: HBM where rows are many, the launch where they are few. 1500 tokens of 48 normed heads of 128, f32 to bf16, 55 MB: 13.4
// us, 4.1 TB/s, where a large copy reaches 4.9; appended (16 bits throughout, 37 MB) 12.0 us: a wave's requests go out in turn (length, position,
// page, then the rows of one group after those of the other: below). One token of 40 heads 3.3 to 4.1 us, 24 tokens of 48 appended 4.8. A prompt of
// 8000 tokens appended alone 37 us, beside 255 single tokens 291: each sequence has as many workgroups as the longest.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_kv.h"

namespace p8x {

typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));

struct RopeJob {
    TurnDev r;
    HeadsDev q, k;          // k: also the input of keys that go to the cache
    const void *v;          // append: values, rows and heads apart as keys
    int n, D, groups, each; // tokens (append: most of a sequence), groups of 64 / L heads a token, groups of a wave
    const int32_t *at;
    KvDev c;
    DraftDev d;
    int32_t *pos, *len_out;
};

// cosine and sine of f / 2^64 turns
__device__ __forceinline__ void turn_of(uint64_t f, float &c, float &s) {
    const uint32_t u = (uint32_t)(f >> 32), quarter = (u + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(u - (quarter << 30)) * 1.4629180792671596e-9f, x2 = x * x;   // 2 pi / 2^32; |x| <= pi / 4
    // the next terms are below 2^-28
    const float sn = fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
    const float cs = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const bool odd = quarter & 1;
    c = odd ? sn : cs, s = odd ? cs : sn;
    if (quarter == 1 || quarter == 2) c = -c;
    if (quarter >= 2) s = -s;
}

template <bool F32>
__device__ __forceinline__ float4v load4(const void *p, size_t i, int bf16) {
    if constexpr (F32) return *(const float4v *)((const float *)p + i);
    const uint2v w = *(const uint2v *)((const uint16_t *)p + i);
    return float4v{from16((uint16_t)w[0], bf16), from16((uint16_t)(w[0] >> 16), bf16), from16((uint16_t)w[1], bf16), from16((uint16_t)(w[1] >> 16), bf16)};
}
__device__ __forceinline__ void store4(void *p, size_t i, int dtype, float4v v) {
    if (dtype == P8X_F32) {
        *(float4v *)((float *)p + i) = v;
    } else {
        const int b = dtype == P8X_BF16;
        *(uint2v *)((uint16_t *)p + i) = uint2v{to16(v[0], b) | (uint32_t)to16(v[1], b) << 16, to16(v[2], b) | (uint32_t)to16(v[3], b) << 16};
    }
}

// groups of heads that a wave has in registers together (1500 tokens of 48 heads, and appended: 13.8 and 12.7 us; with 1, 13.5 and 12.9; with 4,
// 14.6 and 14.9). Only the append of f32 rows has both groups' rows on their way at once: 16-bit rows are converted where they are
// loaded, and without the append the place of q or k is read from the arguments in memory, so that either waits for one group before it
// requests the next
constexpr int kAtOnce = 2;

// F32: of the rows that come in
template <int L, bool F32, bool APPEND>
__global__ __launch_bounds__(256) void k_rope(RopeJob J) {
    constexpr int HP = 64 / L;
    const int lane = threadIdx.x & 63, l = lane % L, D = J.D, rot = J.r.n_rot;
    const int parts = (J.groups + J.each - 1) / J.each;   // of a token
    const int s = APPEND ? blockIdx.y : 0;
    int first = 0, nt = J.n, len = 0;
    if constexpr (APPEND) {
        nt = seq_tokens(J.d, s, first);
        len = seq_len(J.c, s);
    }
    const uint32_t items = (uint32_t)nt * parts;   // (below 2^31: rope_plan)
    const bool on = 8 * l < D, turned = 8 * l < rot;
    // the lane's two fours of a head
    const int e0 = turned && !J.r.pairs ? 4 * l : 8 * l, e1 = turned && !J.r.pairs ? rot / 2 + 4 * l : 8 * l + 4;
    u64x2 f0 = {0, 0}, f1 = {0, 0};
    if (turned) f0 = *(const u64x2 *)(J.r.freq + 4 * l), f1 = *(const u64x2 *)(J.r.freq + 4 * l + 2);
    for (uint32_t x = blockIdx.x * 4 + (threadIdx.x >> 6); x < items; x += gridDim.x * 4) {
        const int i = __builtin_amdgcn_readfirstlane(x / parts), g0 = __builtin_amdgcn_readfirstlane(x - (uint32_t)i * parts) * J.each;
        const int tok = first + i, slot = len + i, p = J.at ? J.at[tok] : slot;
        const int64_t to = APPEND && slot < J.c.max_len ? slot_offset(J.c, s, slot) : -1;
        float4v co, si;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float c, sn;
            turn_of((uint64_t)(int64_t)p * (j < 2 ? f0[j & 1] : f1[j & 1]), c, sn);
            co[j] = J.r.amp * c, si[j] = J.r.amp * sn;
        }
        const int g1 = min(J.groups, g0 + J.each);
        for (int g = g0; g < g1; g += kAtOnce) {
            float4v a[kAtOnce], b[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int h = (g + u) * HP + lane / L;   // of queries, then keys, then (append) values
                const bool q = h < J.q.n, k = !q && h < J.q.n + J.k.n, v = APPEND && !q && !k && h < J.q.n + 2 * J.k.n;
                a[u] = b[u] = float4v{0, 0, 0, 0};
                if (!on || g + u >= g1 || !(q || k || v)) continue;
                const HeadsDev &w = q ? J.q : J.k;
                const size_t at = (size_t)tok * w.ld + (size_t)(h - (q ? 0 : k ? J.q.n : J.q.n + J.k.n)) * w.hs;
                const void *src = v ? J.v : w.x;
                a[u] = load4<F32>(src, at + e0, w.dtype == P8X_BF16);
                b[u] = load4<F32>(src, at + e1, w.dtype == P8X_BF16);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int h = (g + u) * HP + lane / L;
                const bool q = h < J.q.n, k = !q && h < J.q.n + J.k.n, v = APPEND && !q && !k && h < J.q.n + 2 * J.k.n;
                const float *w = q ? J.r.w_q : k ? J.r.w_k : nullptr;
                if (J.r.w_q || J.r.w_k) {   // (all lanes: the sum is over a head's)
                    float sum = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum = fmaf(a[u][j], a[u][j], fmaf(b[u][j], b[u][j], sum));
#pragma unroll
                    for (int o = 1; o < L; o <<= 1) sum += __shfl_xor(sum, o);
                    if (w && on) {
                        const float ms = fmaf(sum, 1.0f / D, J.r.eps), r = ms < 0x1p-100f ? 1.0f / sqrtf(ms) : __builtin_amdgcn_rsqf(ms);   // (which takes no subnormals)
                        a[u] = a[u] * r * *(const float4v *)(w + e0);
                        b[u] = b[u] * r * *(const float4v *)(w + e1);
                    }
                }
                if (!on || g + u >= g1 || !(q || k || v)) continue;
                float4v ya = a[u], yb = b[u];
                if (turned && !v) {
                    if (J.r.pairs) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            ya[2 * j] = fmaf(a[u][2 * j], co[j], -(a[u][2 * j + 1] * si[j]));
                            ya[2 * j + 1] = fmaf(a[u][2 * j + 1], co[j], a[u][2 * j] * si[j]);
                            yb[2 * j] = fmaf(b[u][2 * j], co[j + 2], -(b[u][2 * j + 1] * si[j + 2]));
                            yb[2 * j + 1] = fmaf(b[u][2 * j + 1], co[j + 2], b[u][2 * j] * si[j + 2]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            ya[j] = fmaf(a[u][j], co[j], -(b[u][j] * si[j]));
                            yb[j] = fmaf(b[u][j], co[j], a[u][j] * si[j]);
                        }
                    }
                }
                if (APPEND && !q) {
                    if (to < 0 || slot >= J.c.max_len) continue;
                    const int hd = h - J.q.n - (v ? J.k.n : 0);
                    uint16_t *dst = (v ? J.c.v : J.c.k) + to + (size_t)hd * J.c.head_stride;
                    store4(dst, e0, J.c.bf16 ? P8X_BF16 : P8X_F16, ya);
                    store4(dst, e1, J.c.bf16 ? P8X_BF16 : P8X_F16, yb);
                } else {
                    const HeadsDev &o = q ? J.q : J.k;
                    const size_t at = (size_t)tok * o.ldo + (size_t)(q ? h : h - J.q.n) * o.hso;
                    store4(o.out, at + e0, o.out_dtype, ya);
                    store4(o.out, at + e1, o.out_dtype, yb);
                }
            }
        }
        if (APPEND && J.pos && slot < J.c.max_len && g0 == 0)
            for (int h = lane; h < J.c.n_kv; h += 64) J.pos[((size_t)s * J.c.n_kv + h) * J.c.max_len + slot] = p;
    }
    if (APPEND && J.len_out && blockIdx.x == 0) {
        __syncthreads();
        if (threadIdx.x == 0) J.len_out[s] = len + min(nt, J.c.max_len - len);
    }
}

// tokens of a launch, or of a sequence at most; returns the workgroups of it (of a sequence)
template <bool APPEND>
static int rope_plan(RopeJob &J, int seqs) {
    const int L = J.D <= 64 ? 8 : J.D <= 128 ? 16 : 32, HP = 64 / L;
    J.groups = (J.q.n + (APPEND ? 2 : 1) * J.k.n + HP - 1) / HP;
    // groups of a wave: one until there are waves for all compute units, then up to all of a token
    const int64_t all = (int64_t)J.n * J.groups * seqs;
    J.each = (int)std::min<int64_t>(J.groups, std::max<int64_t>(1, all / (16 * num_cus())));
    while ((int64_t)J.n * ((J.groups + J.each - 1) / J.each) > INT32_MAX) J.each *= 2;
    const int64_t waves = (int64_t)J.n * ((J.groups + J.each - 1) / J.each);
    // (workgroups go on with further tokens. Each sequence has as many as the longest may need: 65535 of one token and one of 200000 would
    // be a launch of 3.3e9, nearly all of which find nothing)
    return (int)std::min<int64_t>((waves + 3) / 4, std::max(8, (1 << 20) / seqs));
}

template <bool F32, bool APPEND>
static void rope_run(const RopeJob &J, int nb, int seqs, hipStream_t st) {
    const dim3 grid(nb, seqs);
    if (J.D <= 64) k_rope<8, F32, APPEND><<<grid, 256, 0, st>>>(J);
    else if (J.D <= 128) k_rope<16, F32, APPEND><<<grid, 256, 0, st>>>(J);
    else k_rope<32, F32, APPEND><<<grid, 256, 0, st>>>(J);
}

int launch_rope(const TurnDev &r, int n, int D, const int32_t *pos, const HeadsDev &q, const HeadsDev &k, hipStream_t st) {
    auto go = [&](const HeadsDev &hq, const HeadsDev &hk) {   // rows of f32, or of 16 bits
        RopeJob J{};
        J.r = r, J.q = hq, J.k = hk, J.n = n, J.D = D, J.at = pos;
        const int nb = rope_plan<false>(J, 1);
        if ((hq.n ? hq : hk).dtype == P8X_F32) rope_run<true, false>(J, nb, 1, st);
        else rope_run<false, false>(J, nb, 1, st);
    };
    if (q.n && k.n && (q.dtype == P8X_F32) != (k.dtype == P8X_F32)) {
        go(q, HeadsDev{});
        go(HeadsDev{}, k);
    } else {
        go(q, k);
    }
    return hip_check(hipGetLastError(), "p8x_rope launch");
}

int launch_kv_append_rope(const KvDev &c, const DraftDev &d, int D, const TurnDev &r, const int32_t *at, const HeadsDev &q, int kv_dtype,
                          int32_t *pos, int32_t *len_out, hipStream_t st) {
    bool own_len = len_out != nullptr;   // the length by a launch of its own
    if (d.n_tokens && d.max_tokens) {
        RopeJob J{};
        J.r = r, J.n = std::min(d.max_tokens, d.n_tokens), J.D = D, J.at = at, J.c = c, J.d = d, J.v = d.v;
        J.k = HeadsDev{d.k, d.ld_kv, d.hs_kv, nullptr, 0, 0, c.n_kv, kv_dtype, 0};
        if (q.n && (q.dtype == P8X_F32) != (kv_dtype == P8X_F32)) {   // queries of another width: theirs first
            RopeJob Q = J;
            Q.q = q, Q.k.n = 0;
            const int nb = rope_plan<true>(Q, c.n_seq);
            if (q.dtype == P8X_F32) rope_run<true, true>(Q, nb, c.n_seq, st);
            else rope_run<false, true>(Q, nb, c.n_seq, st);
        } else {
            J.q = q;
        }
        J.pos = pos;
        const int nb = rope_plan<true>(J, c.n_seq);
        own_len = len_out && len_out == c.len && nb > 1;   // other workgroups read it
        J.len_out = own_len ? nullptr : len_out;
        if (kv_dtype == P8X_F32) rope_run<true, true>(J, nb, c.n_seq, st);
        else rope_run<false, true>(J, nb, c.n_seq, st);
    }
    if (own_len) return launch_append_len(c, d, nullptr, len_out, st);
    return hip_check(hipGetLastError(), "p8x_kv_append_rope launch");
}

}  // namespace p8x
