// p8x_score.hip -- the attention weight that accepted tokens gave (p8x_kv_score):
// sum over the accepted tokens' rows of exp(scale q k - lse) per slot. S [row][slot] = Q K^T with K as the B operand (lane
// n = slot) straight from memory, each slot's keys read by one wave once, and Q as A from LDS, where the workgroup
// leaves its rows in operand order; a lane's four rows of every tile are added in place, the four lane groups at the end.
// Keys come one tile ahead of the products. Bound by HBM: some 16 rows over 93000 slots x 8 heads (4 sequences, 197 MB) 48.3 us,
// 4.07 TB/s; by latency for one sequence (1001 slots: 5.4 us).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_attn.h"

namespace p8x {

constexpr int kScoreWaves = 4;
// rows that LDS holds at a time (64 of 256 f32 elements would leave no room for a second workgroup); more of them take the
// slots again
__host__ __device__ constexpr int score_rows(int D) { return D == 256 ? 32 : 64; }

struct ScoreJob {
    KvDev c;
    DraftDev d;
    const uint64_t *accept;
    const float *lse, *score;
    float *score_out;
    float decay;
};

// token of accepted rank r
__device__ __forceinline__ int nth_bit(uint64_t b, int r) {
    for (; r; --r) b &= b - 1;
    return __ffsll((unsigned long long)b) - 1;
}

template <int D, bool BF, bool QF>
__global__ __launch_bounds__(64 * kScoreWaves) void k_score(ScoreJob J) {
    constexpr int C = D / 32, QP = QF ? (BF ? 3 : 2) : 1, RB = score_rows(D);
    __shared__ uint4v sq[RB / 16][QP][C][64];
    __shared__ float4v sl[RB / 4], sc[RB / 4];   // lse and factor of a product, by row (rows that are not there: 0)
    __shared__ uint64_t see[RB];
    const KvDev &c = J.c;
    const DraftDev &d = J.d;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, ln = lane & 15;
    const int s = blockIdx.z, h = blockIdx.y;
    int first = 0;
    const int nt = __builtin_amdgcn_readfirstlane(d.n_tokens ? seq_tokens(d, s, first) : 0), n = __builtin_amdgcn_readfirstlane(seq_len(c, s));
    const uint64_t all = nt >= 64 ? ~0ull : (1ull << nt) - 1, acc = J.accept ? J.accept[s] & all : all;
    const int cnt = __popcll(acc), rows = cnt * d.G;
    // the workgroup's tiles of 32 slots; the drafts' are the last ones
    const int ctx = (n + 31) / 32, tiles = ctx + (min(cnt, c.max_len - n) + 31) / 32, per = (tiles + (int)gridDim.x - 1) / (int)gridDim.x;
    const int t0 = blockIdx.x * per, t1 = min(tiles, t0 + per);
    if (t0 >= t1) return;
    const size_t base = ((size_t)s * c.n_kv + h) * c.max_len;
    const uint16_t *kp = c.k + (size_t)h * c.head_stride;
    const uint32_t ko = (uint32_t)ln * (uint32_t)c.slot_stride + 8 * g;

    int rb = 0;
    do {   // once without rows: scores decay
        const int rt = min(RB / 16, (rows - rb + 15) / 16);
        // the wave's tiles from tb on: offsets of its next 64 halves, a lane each, and keys one tile ahead, the first before
        // the rows are laid out
        int tb = t0 + wave, lo = 0, hi = 0, many = 0;
        uint4v kf[2][C], kn[2][C];
        float next = 0.0f;
        auto half = [&](int i) { return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, i)); };
        // tile i's keys into kn; a lane past the last slot reads the half's first, whose column is then not written
        auto fetch = [&](int i) {
            const int slot = 32 * (tb + kScoreWaves * i);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int64_t o = half(2 * i + x);
                if (o >= 0) {
                    const uint16_t *at = kp + o + (slot + 16 * x + ln < n ? ko : 8 * g);
#pragma unroll
                    for (int k = 0; k < C; ++k) kn[x][k] = *(const uint4v *)(at + 32 * k);
                }
            }
            if (lane < 32 && slot + lane < n && !rb) next = J.score[base + slot + lane];
        };
        auto ahead = [&](int tb) {
            if (tb >= min(t1, ctx)) return;
            const int t = tb + kScoreWaves * (lane >> 1), slot = 32 * t + 16 * (lane & 1);
            const int64_t off = t < min(t1, ctx) && slot < n ? slot_offset(c, s, slot) : -1;
            lo = (int)off, hi = (int)(off >> 32), many = min(32, (min(t1, ctx) - tb + kScoreWaves - 1) / kScoreWaves);
            fetch(0);
        };
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int k = 0; k < C; ++k) kn[x][k] = uint4v{0, 0, 0, 0};
        ahead(tb);
        if (rb) __syncthreads();
        for (int r = threadIdx.x; r < 16 * rt; r += 64 * kScoreWaves) {
            const int row = rb + r, i = row / d.G;
            see[r] = 0;
            ((float *)sl)[r] = 0.0f;
            if (row < rows) {
                const int ti = nth_bit(acc, i);
                see[r] = token_mask(d, first + ti, ti);
                ((float *)sl)[r] = J.lse[(size_t)(first + ti) * c.n_kv * d.G + h * d.G + row - i * d.G];
            }
        }
        for (int r = wave; r < rt; r += kScoreWaves) {
            const int row = rb + 16 * r + ln, i = row / d.G;
            const bool on = row < rows;
            const size_t at = on ? (size_t)(first + nth_bit(acc, i)) * d.ld_q + (size_t)(h * d.G + row - i * d.G) * d.hs_q + 8 * g : 0;
            float f = d.scale;
            if constexpr (QF) {
                float x[C][8];
                f = load_split<C, BF>((const float *)d.q + at, on, f, x);
#pragma unroll
                for (int k = 0; k < C; ++k) {
                    uint4v p[QP];
                    split8<BF, QP>(x[k], p);
#pragma unroll
                    for (int u = 0; u < QP; ++u) sq[r][u][k][lane] = p[u];
                }
            } else {
#pragma unroll
                for (int k = 0; k < C; ++k) sq[r][0][k][lane] = on ? *(const uint4v *)((const uint16_t *)d.q + at + 32 * k) : uint4v{0, 0, 0, 0};
            }
            if (g == 0) ((float *)sc)[16 * r + ln] = f;
        }
        __syncthreads();

        // the tile's weights, summed over the rows: lane l < 32 has slot l's. draft: the slots are drafted tokens, of which a row
        // counts those that its mask shows; tj0, tj1: the token of the lane's slot in either half
        auto sum_rows = [&](bool draft, int tj0, int tj1) {
            float w0 = 0.0f, w1 = 0.0f;
            for (int r = 0; r < rt; ++r) {
                const float4v l = sl[4 * r + g], f = sc[4 * r + g];
                float4v s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
                for (int u = QP - 1; u >= 0; --u)
#pragma unroll
                    for (int k = 0; k < C; ++k) {
                        const uint4v q = sq[r][u][k][lane];
                        s0 = mfma<BF>(q, kf[0][k], s0);
                        s1 = mfma<BF>(q, kf[1][k], s1);
                    }
                const int left = rows - rb - 16 * r - 4 * g;   // rows of the lane's four that are there
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float e0 = __builtin_amdgcn_exp2f(fmaf(s0[i], f[i], -l[i]) * kLog2e), e1 = __builtin_amdgcn_exp2f(fmaf(s1[i], f[i], -l[i]) * kLog2e);
                    if (draft) {
                        const uint64_t m = see[16 * r + 4 * g + i];
                        if (!(m >> tj0 & 1)) e0 = 0.0f;
                        if (!(m >> tj1 & 1)) e1 = 0.0f;
                    }
                    w0 += i < left ? e0 : 0.0f;
                    w1 += i < left ? e1 : 0.0f;
                }
            }
            w0 += __shfl_xor(w0, 16);
            w0 += __shfl_xor(w0, 32);
            w1 += __shfl_xor(w1, 16);
            w1 += __shfl_xor(w1, 32);
            return lane < 16 ? w0 : w1;
        };
        auto put = [&](int slot, int end, bool old, float w, float before) {
            if (lane < 32 && slot + lane < end) {
                float *o = J.score_out + base + slot + lane;
                *o = rb ? *o + w : old ? J.decay * before + w : w;
            }
        };

        for (; tb < min(t1, ctx); ahead(tb += 32 * kScoreWaves)) {
            for (int i = 0; i < many; ++i) {
                const int slot = 32 * (tb + kScoreWaves * i);
                const float before = next;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int k = 0; k < C; ++k) kf[x][k] = kn[x][k];
                if (i + 1 < many) fetch(i + 1);
                float w = rt > 0 ? sum_rows(false, 0, 0) : 0.0f;
                if ((lane < 16 ? half(2 * i) : half(2 * i + 1)) < 0) w = 0.0f;
                put(slot, n, true, w, before);
            }
        }
        for (int t = max(t0, ctx) + wave; t < t1; t += kScoreWaves) {   // accepted tokens
            const int r0 = 32 * (t - ctx), j0 = r0 + ln < cnt ? nth_bit(acc, r0 + ln) : 0, j1 = r0 + 16 + ln < cnt ? nth_bit(acc, r0 + 16 + ln) : 0;
#pragma unroll
            for (int k = 0; k < C; ++k) {
                kf[0][k] = draft8(d.k, (size_t)(first + j0) * d.ld_kv + (size_t)h * d.hs_kv + 32 * k + 8 * g, d.kv_f32, BF);
                kf[1][k] = draft8(d.k, (size_t)(first + j1) * d.ld_kv + (size_t)h * d.hs_kv + 32 * k + 8 * g, d.kv_f32, BF);
            }
            put(n + r0, min(n + cnt, c.max_len), false, sum_rows(true, j0, j1), 0.0f);
        }
        rb += RB;
    } while (rb < rows);
}

template <int D>
static void score_types(const ScoreJob &J, dim3 grid, hipStream_t st) {
    if (J.d.q_f32 && J.d.n_tokens) {
        if (J.c.bf16) k_score<D, true, true><<<grid, 64 * kScoreWaves, 0, st>>>(J);
        else k_score<D, false, true><<<grid, 64 * kScoreWaves, 0, st>>>(J);
    } else {
        if (J.c.bf16) k_score<D, true, false><<<grid, 64 * kScoreWaves, 0, st>>>(J);
        else k_score<D, false, false><<<grid, 64 * kScoreWaves, 0, st>>>(J);
    }
}

int launch_kv_score(const KvDev &c, const DraftDev &d, int D, const uint64_t *accept, const float *lse, float decay, const float *score,
                    float *score_out, hipStream_t st) {
    if (c.slot_stride >= (1u << 26)) return set_error(P8X_ERR_UNSUPPORTED, "p8x_kv_score: slot_stride %zu (below 2^26)", c.slot_stride);
    const ScoreJob J{c, d, accept, lse, score, score_out, decay};
    const int64_t heads = (int64_t)c.n_seq * c.n_kv, tiles = (c.max_len + 31) / 32 + 2;
    // two workgroups a compute unit: each lays out the rows again (4, 2 and 1: 16.5, 13.6 and 18.0 us at 4 sequences x 8 heads
    // of 8190 slots at most, 49.0, 48.5 and 65.0 at 32767)
    const int nb = (int)std::max<int64_t>(1, std::min<int64_t>((tiles + kScoreWaves - 1) / kScoreWaves, (2 * num_cus() + heads - 1) / heads));
    const dim3 grid(nb, c.n_kv, c.n_seq);
    if (D == 64) score_types<64>(J, grid, st);
    else if (D == 128) score_types<128>(J, grid, st);
    else score_types<256>(J, grid, st);
    return hip_check(hipGetLastError(), "p8x_kv_score launch");
}

}  // namespace p8x
