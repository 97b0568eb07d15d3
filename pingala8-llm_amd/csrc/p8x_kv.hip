// p8x_kv.hip -- the cache's own calls: append of accepted tokens (p8x_kv_append), eviction to a budget by accumulated
// attention weight (p8x_kv_evict).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_kv.h"

namespace p8x {

// ---- append -----------------------------------------------------------------------------------------------
// Pieces of 8 elements: (token, key or value, head, piece of the row), the last fastest; the workgroups of a sequence
// take them in turn. len_out may be the len that the other workgroups read: one workgroup alone (after its barrier) or a
// launch of its own (k_append_len) writes it then.
__device__ __forceinline__ int accepted(const DraftDev &d, const uint64_t *accept, int s, int &first, uint64_t &acc) {
    const int nt = seq_tokens(d, s, first);
    if (!accept) return nt;
    acc = accept[s] & (nt >= 64 ? ~0ull : (1ull << nt) - 1);
    return __popcll(acc);
}

__global__ __launch_bounds__(1024) void k_append(KvDev c, DraftDev d, int D, const uint64_t *accept, const int32_t *at, int32_t *pos, int32_t *len_out) {
    const int s = blockIdx.y, nb = gridDim.x;
    int first;
    uint64_t acc = 0;
    const int cnt = accepted(d, accept, s, first, acc), n = seq_len(c, s);
    const int row = D / 8, per = 2 * c.n_kv * row, slots = min(cnt, c.max_len - n);
    for (int64_t x = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; x < (int64_t)slots * per; x += (int64_t)nb * blockDim.x) {
        const int r = (int)(x / per);
        int y = (int)(x - (int64_t)r * per);
        const bool val = y >= c.n_kv * row;
        if (val) y -= c.n_kv * row;
        const int h = y / row, e = y % row * 8;
        int i = r;
        if (accept) {
            uint64_t b = acc;
            for (int k = r; k; --k) b &= b - 1;
            i = __ffsll((unsigned long long)b) - 1;
        }
        const int tok = first + i, slot = n + r;
        const int64_t to = slot_offset(c, s, slot);
        if (to >= 0) {
            const void *src = val ? d.v : d.k;
            const size_t from = (size_t)tok * d.ld_kv + h * d.hs_kv + e;
            uint4 o;
            if (d.kv_f32) {
                const float4 lo = *(const float4 *)((const float *)src + from), hi = *(const float4 *)((const float *)src + from + 4);
                const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                uint32_t w[4];
                for (int k = 0; k < 4; ++k) w[k] = to16(f[2 * k], c.bf16) | (uint32_t)to16(f[2 * k + 1], c.bf16) << 16;
                o = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                o = *(const uint4 *)((const uint16_t *)src + from);
            }
            *(uint4 *)((val ? c.v : c.k) + to + h * c.head_stride + e) = o;
        }
        if (!val && e == 0 && pos && at) pos[((size_t)s * c.n_kv + h) * c.max_len + slot] = at[tok];
    }
    if (len_out && blockIdx.x == 0) {
        __syncthreads();
        if (threadIdx.x == 0) len_out[s] = n + slots;
    }
}

__global__ void k_append_len(KvDev c, DraftDev d, const uint64_t *accept, int32_t *len_out) {
    const int s = blockIdx.x * 64 + threadIdx.x;
    if (s >= c.n_seq) return;
    int first;
    uint64_t acc = 0;
    const int cnt = accepted(d, accept, s, first, acc), n = seq_len(c, s);
    len_out[s] = n + min(cnt, c.max_len - n);
}

int launch_kv_append(const KvDev &c, const DraftDev &d, int D, const uint64_t *accept, const int32_t *at, int32_t *pos, int32_t *len_out,
                     hipStream_t st) {
    const bool in_place = len_out == c.len;
    const int64_t pieces = (int64_t)(D / 8) * 2 * c.n_kv * d.max_tokens;
    const int nb = (int)std::max<int64_t>(1, std::min<int64_t>((pieces + 1023) / 1024, 1024));
    if (d.n_tokens && d.max_tokens) k_append<<<dim3(nb, c.n_seq), 1024, 0, st>>>(c, d, D, accept, at, pos, in_place && nb > 1 ? nullptr : len_out);
    if (len_out && ((in_place && nb > 1) || !(d.n_tokens && d.max_tokens))) k_append_len<<<(c.n_seq + 63) / 64, 64, 0, st>>>(c, d, accept, len_out);
    return hip_check(hipGetLastError(), "p8x_kv_append launch");
}

// ---- evict ------------------------------------------------------------------------------------------------
// workspace of a key/value head: [0] moves, [1] slots in use before, [4 ..] the moves' sources, then their destinations
__host__ __device__ inline size_t evict_most(int max_len, int budget) { return max_len > budget ? (size_t)(budget < max_len - budget ? budget : max_len - budget) : 0; }
__host__ __device__ inline size_t evict_words(int max_len, int budget) { return (4 + 2 * evict_most(max_len, budget) + 3) / 4 * 4; }

size_t kv_evict_workspace(const KvDev &c, int budget) { return 4 * evict_words(c.max_len, budget) * c.n_seq * c.n_kv; }

struct EvictDev {
    int budget, n_sink, n_recent;
    const float *score; float *score_out;
    const int32_t *pos; int32_t *pos_out;
    int32_t *len_out;
    int *ws;
};

// A slot's key: kept slots are those of the largest keys. Protected ones are above every score, NaN below.
__device__ __forceinline__ uint32_t evict_key(const EvictDev &a, size_t base, int j, int64_t recent) {
    if (a.pos) {
        const int p = a.pos[base + j];
        if (p < a.n_sink || p >= recent) return 0xFFFFFFFFu;
    }
    const float f = a.score[base + j];
    if (f != f) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, f + 0.0f);   // -0 becomes +0
    return b >> 31 ? ~b : b | 0x80000000u;
}

// sum of v over the workgroup's threads before this one, and over all (1024 threads)
__device__ __forceinline__ int block_scan(int v, int *red, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x = v;
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) red[w] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < 16; ++i) {
        if (i < w) before += red[i];
        total += red[i];
    }
    return before + x - v;
}

// One workgroup a key/value head: the budget-th largest key by four passes of 8 bits, then every slot's fate in slot
// order, a contiguous range of slots a thread.
__global__ __launch_bounds__(1024) void k_evict_select(KvDev c, EvictDev a) {
    __shared__ int hist[256], red[16], pick[2];
    const int h = blockIdx.x, s = blockIdx.y, t = threadIdx.x;
    const size_t hd = (size_t)s * c.n_kv + h, base = hd * c.max_len;
    const int n = seq_len(c, s), keep = min(n, a.budget);
    int *ws = a.ws + hd * evict_words(c.max_len, a.budget);
    if (a.score_out != a.score)
        for (int j = t; j < keep; j += 1024) a.score_out[base + j] = a.score[base + j];
    if (a.pos && a.pos_out != a.pos)
        for (int j = t; j < keep; j += 1024) a.pos_out[base + j] = a.pos[base + j];
    if (t == 0) ws[1] = n;
    if (n <= a.budget) {
        if (t == 0) ws[0] = 0;
        return;
    }
    int64_t recent = INT64_MAX;   // positions from here on are protected
    if (a.pos && a.n_recent) {
        int m = INT32_MIN;
        for (int j = t; j < n; j += 1024) m = max(m, a.pos[base + j]);
        for (int o = 32; o; o >>= 1) m = max(m, __shfl_xor(m, o));
        if ((t & 63) == 0) red[t >> 6] = m;
        __syncthreads();
        m = red[0];
        for (int i = 1; i < 16; ++i) m = max(m, red[i]);
        recent = (int64_t)m + 1 - a.n_recent;
    }
    uint32_t key = 0, known = 0;
    int want = keep;   // of the keys that agree with `key` in the known bits, how many of the largest stay
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (t < 256) hist[t] = 0;
        __syncthreads();
        for (int j = t; j < n; j += 1024) {
            const uint32_t k = evict_key(a, base, j, recent);
            if ((k & known) == key) atomicAdd(&hist[k >> shift & 255], 1);
        }
        __syncthreads();
        if (t < 64) {   // from the largest digit down: the digit in which the count passes `want`
            int v[4], sum = 0;
            for (int i = 0; i < 4; ++i) sum += v[i] = hist[255 - 4 * t - i];
            int x = sum;
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(x, o);
                if (t >= o) x += y;
            }
            int above = x - sum;
            if (above < want && x >= want)
                for (int i = 0; i < 4; ++i) {
                    if (above + v[i] >= want) {
                        pick[0] = 255 - 4 * t - i;
                        pick[1] = want - above;
                        break;
                    }
                    above += v[i];
                }
        }
        __syncthreads();
        key |= (uint32_t)pick[0] << shift;
        known |= 255u << shift;
        want = pick[1];
    }
    // want: how many slots of exactly `key` stay, the lowest ones
    const int per = (n + 1023) / 1024, j0 = min(n, t * per), j1 = min(n, j0 + per);
    int ties = 0, total;
    for (int j = j0; j < j1; ++j) ties += evict_key(a, base, j, recent) == key;
    const int tie0 = block_scan(ties, red, total);
    int holes = 0, movers = 0, tie = tie0;
    for (int j = j0; j < j1; ++j) {
        const uint32_t k = evict_key(a, base, j, recent);
        const bool stay = k > key || (k == key && tie++ < want);
        holes += !stay && j < a.budget;
        movers += stay && j >= a.budget;
    }
    int hole = block_scan(holes, red, total), mover = block_scan(movers, red, total);
    if (t == 0) ws[0] = total;
    int *src = ws + 4, *dst = src + evict_most(c.max_len, a.budget);
    tie = tie0;
    for (int j = j0; j < j1; ++j) {
        const uint32_t k = evict_key(a, base, j, recent);
        const bool stay = k > key || (k == key && tie++ < want);
        if (!stay && j < a.budget) dst[hole++] = j;
        if (stay && j >= a.budget) src[mover++] = j;
    }
}

// The moves: sources are slots >= budget and destinations slots < budget, so no row is both.
__global__ __launch_bounds__(256) void k_evict_move(KvDev c, EvictDev a, int D) {
    const int h = blockIdx.y, s = blockIdx.z;
    const size_t hd = (size_t)s * c.n_kv + h, base = hd * c.max_len;
    const int *ws = a.ws + hd * evict_words(c.max_len, a.budget);
    const int moves = ws[0], *src = ws + 4, *dst = src + evict_most(c.max_len, a.budget);
    if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.len_out[s] = min(ws[1], a.budget);
    const int row = D / 8;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < (int64_t)moves * row; x += (int64_t)gridDim.x * 256) {
        const int i = (int)(x / row), e = (int)(x % row) * 8, j0 = src[i], j1 = dst[i];
        const int64_t from = slot_offset(c, s, j0), to = slot_offset(c, s, j1);
        if (from >= 0 && to >= 0) {
            const size_t o = (size_t)h * c.head_stride + e;
            const uint4 k = *(const uint4 *)(c.k + from + o), v = *(const uint4 *)(c.v + from + o);
            *(uint4 *)(c.k + to + o) = k;
            *(uint4 *)(c.v + to + o) = v;
        }
        if (e == 0) {
            a.score_out[base + j1] = a.score[base + j0];
            if (a.pos) a.pos_out[base + j1] = a.pos[base + j0];
        }
    }
}

int launch_kv_evict(const KvDev &c, int D, const p8x_evict_args &p, hipStream_t st) {
    const EvictDev a{p.budget, p.n_sink, p.n_recent, p.score, p.score_out, p.pos, p.pos_out, p.len_out, (int *)p.workspace};
    k_evict_select<<<dim3(c.n_kv, c.n_seq), 1024, 0, st>>>(c, a);
    const int64_t pieces = (int64_t)evict_most(c.max_len, a.budget) * (D / 8);
    const int nb = (int)std::max<int64_t>(1, std::min<int64_t>((pieces + 255) / 256, 512));
    k_evict_move<<<dim3(nb, c.n_kv, c.n_seq), 256, 0, st>>>(c, a, D);
    return hip_check(hipGetLastError(), "p8x_kv_evict launch");
}

}  // namespace p8x
