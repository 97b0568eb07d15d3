// p8x_kv.hip -- the cache's own calls: append of accepted tokens (p8x_kv_append), eviction to a budget by accumulated
// attention weight (p8x_kv_evict).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_kv.h"

namespace p8x {

// ---- append -----------------------------------------------------------------------------------------------
// Pieces of 8 elements: (token, key or value, head, piece of the row), the last fastest; the workgroups of a sequence
// take them in turn. len_out may be the len that the other workgroups read: one workgroup alone (after its barrier) or a
// launch of its own (k_append_len) writes it then. Bound by HBM and the launch: 1500 tokens of 8 heads x 128 from f32 (18.5 MB) 6.6
// us, 8 tokens 4.2.
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
    if (len_out && ((in_place && nb > 1) || !(d.n_tokens && d.max_tokens))) return launch_append_len(c, d, accept, len_out, st);
    return hip_check(hipGetLastError(), "p8x_kv_append launch");
}

int launch_append_len(const KvDev &c, const DraftDev &d, const uint64_t *accept, int32_t *len_out, hipStream_t st) {
    k_append_len<<<(c.n_seq + 63) / 64, 64, 0, st>>>(c, d, accept, len_out);
    return hip_check(hipGetLastError(), "append length launch");
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

constexpr uint32_t kSafeKey = 0xFFFFFFFFu;
// A slot's key: kept slots are those of the largest keys. Protected ones are above every score, NaN below.
__device__ __forceinline__ uint32_t score_key(float f) {
    if (f != f) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, f + 0.0f);   // -0 becomes +0
    return b >> 31 ? ~b : b | 0x80000000u;
}

// sums of v over the waves before this one, and over all; v is the wave's
constexpr int kSelectWaves = 16;
__device__ __forceinline__ int wave_scan(int v, int *red, int &total) {
    constexpr int WAVES = kSelectWaves;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 0) red[wave] = v;
    __syncthreads();
    int r = lane < WAVES ? red[lane] : 0, before = lane < wave ? r : 0;
    for (int o = WAVES / 2; o; o >>= 1) before += __shfl_xor(before, o), r += __shfl_xor(r, o);
    total = __builtin_amdgcn_readfirstlane(r);
    return __builtin_amdgcn_readfirstlane(before);
}

// One workgroup of 16 waves a key/value head. Each wave has a contiguous range of the slots, in groups of 64, a slot a lane:
// the budget-th largest key by three passes of 11, 11 and 10 bits over counts in LDS (protected slots are counted apart), then
// every slot's fate in slot order, by ballots. KEEP: up to 64 KEEP slots a wave, whose keys stay in LDS, each lane its own;
// else (0) every pass makes them again from scores and positions. Loops are rolled, U groups a turn: a workgroup runs each
// pass once, and with all groups unrolled it waited for instructions most of the time. Bound by the latency of the passes on
// one compute unit a head: 32767 slots 43 us (memory 13, counts 15, fates 10).
template <int U, int KEEP>
__global__ __launch_bounds__(64 * kSelectWaves) void k_evict_select(KvDev c, EvictDev a) {
    constexpr int WAVES = kSelectWaves, BINS = 2048 / (64 * WAVES);   // of a thread
    __shared__ int hist[2048], red[WAVES], pick[2];
    extern __shared__ uint32_t kept[];   // KEEP: [wave][group][lane]
    const int h = blockIdx.x, s = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const size_t hd = (size_t)s * c.n_kv + h, base = hd * c.max_len;
    const int n = __builtin_amdgcn_readfirstlane(seq_len(c, s)), keep = min(n, a.budget);
    int *ws = a.ws + hd * evict_words(c.max_len, a.budget);
    if (t == 0) ws[1] = n;
    if (n == 0) {
        if (t == 0) ws[0] = 0;
        return;
    }
    const int groups = (n + 64 * WAVES - 1) / (64 * WAVES);   // of a wave
    const uint32_t first = wave * groups * 64 + lane, end = n - 1;   // the lane's first slot; the last slot
    const float *score = a.score + base;
    const int *pos = a.pos ? a.pos + base : nullptr;
    const bool copy_s = a.score_out != a.score, copy_p = pos && a.pos_out != a.pos;
    uint32_t *const mine = kept + wave * KEEP * 64 + lane;
    // v[u] of group g0 + u, all loads before the first use; a lane past the last slot reads that one
    auto fetch = [&](int g0, const uint32_t *from, uint32_t (&v)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = from[min(first + 64 * (g0 + u), end)];
    };
    int m = INT32_MIN;   // the largest position; positions of slots that stay in place to pos_out
    if (pos)
#pragma unroll 1
        for (int g0 = 0; g0 < groups; g0 += U) {
            uint32_t v[U];
            fetch(g0, (const uint32_t *)pos, v);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t j = first + 64 * (g0 + u);
                m = max(m, (int)v[u]);
                if (KEEP && g0 + u < groups) mine[64 * (g0 + u)] = v[u];
                if (copy_p && g0 + u < groups && j < (uint32_t)keep) a.pos_out[base + j] = (int)v[u];
            }
        }
    int64_t recent = INT64_MAX;   // positions from here on are protected
    if (pos && a.n_recent && n > a.budget) {
        for (int o = 32; o; o >>= 1) m = max(m, __shfl_xor(m, o));
        if (lane == 0) red[wave] = m;
        __syncthreads();
        m = red[lane & (WAVES - 1)];
        for (int o = WAVES / 2; o; o >>= 1) m = max(m, __shfl_xor(m, o));
        recent = (int64_t)m + 1 - a.n_recent;
    }
    // keys of groups g0 .. g0 + U - 1 from scores, and positions from LDS or memory
    auto make = [&](int g0, uint32_t (&k)[U], uint32_t (&sc)[U], bool kept_pos) {
        uint32_t p[U];
        fetch(g0, (const uint32_t *)score, sc);
        if (pos) {
            if (kept_pos)
#pragma unroll
                for (int u = 0; u < U; ++u) p[u] = mine[64 * min(g0 + u, groups - 1)];
            else fetch(g0, (const uint32_t *)pos, p);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool safe = pos && ((int)p[u] < a.n_sink || (int)p[u] >= recent);
            k[u] = safe ? kSafeKey : score_key(__builtin_bit_cast(float, sc[u]));
        }
    };
    int guarded = 0;   // protected slots; the scores of slots that stay in place go to score_out
#pragma unroll 1
    for (int g0 = 0; g0 < groups; g0 += U) {
        uint32_t k[U], sc[U];
        make(g0, k, sc, KEEP > 0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (g0 + u < groups) {
                const uint32_t j = first + 64 * (g0 + u);
                if (KEEP) mine[64 * (g0 + u)] = k[u];
                if (copy_s && j < (uint32_t)keep) a.score_out[base + j] = __builtin_bit_cast(float, sc[u]);
                guarded += __popcll(__ballot(k[u] == kSafeKey && j <= end));
            }
    }
    if (n <= a.budget) {
        if (t == 0) ws[0] = 0;
        return;
    }
    // f(group, slot, key, whether there is one) over groups g0 .. g1 - 1 of the wave in order
    auto each = [&](int g0, int g1, auto f) {
#pragma unroll 1
        for (; g0 < g1; g0 += U) {
            uint32_t k[U], sc[U];
            if constexpr (KEEP) {
#pragma unroll
                for (int u = 0; u < U; ++u) k[u] = mine[64 * min(g0 + u, groups - 1)];
            } else {
                make(g0, k, sc, false);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t j = first + 64 * (g0 + u);
                f(g0 + u, j, k[u], g0 + u < g1 && j <= end);
            }
        }
    };
    int all;
    wave_scan(guarded, red, all);
    uint32_t key = kSafeKey;
    int want = keep;   // how many slots of exactly `key` stay, the lowest ones; all with a larger key stay
    if (all < keep) {
        want = keep - all;
        key = 0;
        uint32_t known = 0;
#pragma unroll 1
        for (int p = 0; p < 3; ++p) {
            const int shift = p == 0 ? 21 : p == 1 ? 10 : 0, mask = p == 2 ? 1023 : 2047;
            __syncthreads();
#pragma unroll
            for (int b = 0; b < BINS; ++b) hist[64 * WAVES * b + t] = 0;
            __syncthreads();
            each(0, groups, [&](int, uint32_t, uint32_t k, bool in) {
                if (in && k != kSafeKey && (k & known) == key) atomicAdd(&hist[k >> shift & mask], 1);
            });
            __syncthreads();
            // from the largest digit down, BINS of them a thread: the digit in which the count passes `want`
            const int d0 = 2047 - BINS * t;
            int v[BINS], sum = 0;
#pragma unroll
            for (int b = 0; b < BINS; ++b) sum += v[b] = hist[d0 - b];
            int x = sum;
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(x, o);
                if (lane >= o) x += y;
            }
            int total;
            int above = wave_scan(__builtin_amdgcn_readlane(x, 63), red, total) + x - sum;
            if (above < want && above + sum >= want) {
                int d = d0;
#pragma unroll
                for (int b = 0; b + 1 < BINS; ++b)
                    if (d == d0 - b && above + v[b] < want) above += v[b], --d;
                pick[0] = d;
                pick[1] = want - above;
            }
            __syncthreads();
            key |= (uint32_t)pick[0] << shift;
            known |= (uint32_t)mask << shift;
            want = pick[1];
        }
    }
    // Every slot's fate, 64 groups at a time: lane i has the ballots of group c0 + i, so that what goes on in the slots' order
    // is a scan over lanes.
    uint64_t more, same;   // keys above and at `key`
    auto sweep = [&](int c0) {
        more = same = 0;
        each(c0, min(groups, c0 + 64), [&](int g, uint32_t, uint32_t k, bool in) {
            const uint64_t up = __ballot(in && k > key), eq = __ballot(in && k == key);
            if (lane == g - c0) more = up, same = eq;
        });
    };
    auto scan = [&](int v) {   // over lanes, own included
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(v, o);
            if (lane >= o) v += y;
        }
        return v;
    };
    const bool once = groups <= 64;   // the ballots stay
    int ties = 0, total;
#pragma unroll 1
    for (int c0 = 0; c0 < groups; c0 += 64) {
        sweep(c0);
        ties += __builtin_amdgcn_readlane(scan(__popcll(same)), 63);
    }
    const int tie0 = wave_scan(ties, red, total);
    int tie, holes = 0, movers = 0;
    uint64_t ho, mo;   // of the lane's group: slots below the budget that go, slots above it that stay
    auto fates = [&](int c0) {
        if (!once) sweep(c0);
        const int cnt = __popcll(same), upto = tie + scan(cnt), left = want - (upto - cnt);
        tie = __builtin_amdgcn_readlane(upto, 63);
        uint64_t go = left >= cnt ? 0 : same;   // of the slots at `key`: all but the lowest `left`
        for (int i = 0; i < left && go; ++i) go &= go - 1;
        const uint64_t stay = more | (same & ~go);
        const int64_t j = ((int64_t)wave * groups + c0 + lane) * 64, in = n - j, low = a.budget - j;   // the group's first slot
        const uint64_t there = c0 + lane >= groups || in <= 0 ? 0 : in >= 64 ? ~0ull : (1ull << in) - 1;
        const uint64_t below = low <= 0 ? 0 : low >= 64 ? ~0ull : (1ull << low) - 1;
        ho = there & below & ~stay;
        mo = there & stay & ~below;
    };
    tie = tie0;
#pragma unroll 1
    for (int c0 = 0; c0 < groups; c0 += 64) {
        fates(c0);
        holes += __builtin_amdgcn_readlane(scan(__popcll(ho)), 63), movers += __builtin_amdgcn_readlane(scan(__popcll(mo)), 63);
    }
    holes = wave_scan(holes, red, total);
    movers = wave_scan(movers, red, total);
    if (t == 0) ws[0] = total;
    int *src = ws + 4, *dst = src + evict_most(c.max_len, a.budget);
    const uint64_t lower = (1ull << lane) - 1;
    tie = tie0;
#pragma unroll 1
    for (int c0 = 0; c0 < groups; c0 += 64) {
        if (!once) fates(c0);
        const int hs = holes + scan(__popcll(ho)), ms = movers + scan(__popcll(mo)), h0 = hs - __popcll(ho), m0 = ms - __popcll(mo);
        holes = __builtin_amdgcn_readlane(hs, 63), movers = __builtin_amdgcn_readlane(ms, 63);
        for (int i = 0; i < min(64, groups - c0); ++i) {
            auto of = [&](uint64_t v) { return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, i); };
            const uint64_t gh = of(ho), gm = of(mo);
            const uint32_t j = first + 64 * (c0 + i);
            if (gh >> lane & 1) dst[__builtin_amdgcn_readlane(h0, i) + __popcll(gh & lower)] = j;
            if (gm >> lane & 1) src[__builtin_amdgcn_readlane(m0, i) + __popcll(gm & lower)] = j;
        }
    }
}

// The same for rows of at most 64 K slots a wave and 16 waves, whose keys stay in registers, K a lane: four digits of 8 bits, each
// with counts of its own and one barrier (every wave finds the digit for itself), then ties and fates by ballots. Bound by the
// latency of its seven barriers and of the scans between them: 1008 slots 12.2 us with the moves, 4000 16.7.
template <int K>
__global__ __launch_bounds__(1024) void k_evict_short(KvDev c, EvictDev a) {
    __shared__ int hist[4][256], red[3][16];
    const int h = blockIdx.x, s = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), waves = blockDim.x >> 6;
    const size_t hd = (size_t)s * c.n_kv + h, base = hd * c.max_len;
    const int n = __builtin_amdgcn_readfirstlane(seq_len(c, s)), keep = min(n, a.budget);
    int *ws = a.ws + hd * evict_words(c.max_len, a.budget);
    if (t == 0) ws[1] = n;
    if (n == 0) {
        if (t == 0) ws[0] = 0;
        return;
    }
    const int j0 = wave * K * 64 + lane;   // the lane's slots: j0 + 64 g
    int p[K] = {};
    float sc[K];
#pragma unroll
    for (int g = 0; g < K; ++g) {
        const int j = min(j0 + 64 * g, n - 1);
        sc[g] = a.score[base + j];
        if (a.pos) p[g] = a.pos[base + j];
    }
    for (int i = t; i < 1024; i += blockDim.x) hist[i >> 8][i & 255] = 0;
    // slots that stay in place, to the outputs
#pragma unroll
    for (int g = 0; g < K; ++g)
        if (j0 + 64 * g < keep) {
            if (a.score_out != a.score) a.score_out[base + j0 + 64 * g] = sc[g];
            if (a.pos && a.pos_out != a.pos) a.pos_out[base + j0 + 64 * g] = p[g];
        }
    if (n <= a.budget) {
        if (t == 0) ws[0] = 0;
        return;
    }
    // sum of the values that the waves put into r, before this wave's and of all
    auto across = [&](const int *r, int &total) {
        int v = lane < waves ? r[lane & 15] : 0, before = lane < wave ? v : 0;
        for (int o = 8; o; o >>= 1) before += __shfl_xor(before, o), v += __shfl_xor(v, o);
        total = __builtin_amdgcn_readfirstlane(v);
        return __builtin_amdgcn_readfirstlane(before);
    };
    const bool latest = a.pos && a.n_recent;
    if (latest) {
        int m = p[0];
#pragma unroll
        for (int g = 1; g < K; ++g) m = max(m, p[g]);
        for (int o = 32; o; o >>= 1) m = max(m, __shfl_xor(m, o));
        if (lane == 0) red[0][wave] = m;
    }
    __syncthreads();
    int64_t recent = INT64_MAX;   // positions from here on are protected
    if (latest) {
        int m = red[0][min(lane & 15, waves - 1)];
        for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor(m, o));
        recent = (int64_t)m + 1 - a.n_recent;
    }
    uint32_t k[K];
#pragma unroll
    for (int g = 0; g < K; ++g) k[g] = a.pos && (p[g] < a.n_sink || p[g] >= recent) ? kSafeKey : score_key(sc[g]);
    uint32_t key = 0;
    int want = keep;   // of the keys that agree with `key` in the digits known, how many of the largest stay
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int shift = 24 - 8 * d;
#pragma unroll
        for (int g = 0; g < K; ++g) {
            const uint32_t dig = k[g] >> shift & 255;
            if (j0 + 64 * g < n && (d == 0 || k[g] >> (shift + 8 & 31) == key >> (shift + 8 & 31))) {
                // the first lane adds all that have its digit (many slots have the same score, of nothing)
                const uint64_t same = __ballot(dig == (uint32_t)__builtin_amdgcn_readfirstlane(dig));
                if (!(same >> lane & 1)) atomicAdd(&hist[d][dig], 1);
                else if (!(same & ((1ull << lane) - 1))) atomicAdd(&hist[d][dig], __popcll(same));
            }
        }
        __syncthreads();
        // from the largest digit down, four of them a lane: the one in which the count passes `want`
        const int4 v = *(const int4 *)&hist[d][252 - 4 * lane];
        const int sum = v.x + v.y + v.z + v.w;
        int x = sum;
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        int above = x - sum, dig = 255 - 4 * lane;
        const int f = __ffsll((unsigned long long)__ballot(x >= want)) - 1;
        if (above + v.w < want) {
            above += v.w, --dig;
            if (above + v.z < want) {
                above += v.z, --dig;
                if (above + v.y < want) above += v.y, --dig;
            }
        }
        key |= (uint32_t)__builtin_amdgcn_readlane(dig, f) << shift;
        want -= __builtin_amdgcn_readlane(above, f);
    }
    // want: how many slots of exactly `key` stay, the lowest ones
    uint64_t same[K];
    int ties = 0, total;
#pragma unroll
    for (int g = 0; g < K; ++g) same[g] = __ballot(j0 + 64 * g < n && k[g] == key), ties += __popcll(same[g]);
    if (lane == 0) red[1][wave] = ties;
    __syncthreads();
    int tie = across(red[1], total);
    const uint64_t lower = (1ull << lane) - 1;
    uint64_t ho[K], mo[K];   // slots below the budget that go, slots above it that stay
    int counts = 0;          // of the former, and of the latter in the upper half
#pragma unroll
    for (int g = 0; g < K; ++g) {
        const int j = j0 + 64 * g;
        const bool stay = k[g] > key || (k[g] == key && tie + __popcll(same[g] & lower) < want);
        tie += __popcll(same[g]);
        ho[g] = __ballot(j < n && !stay && j < a.budget), mo[g] = __ballot(j < n && stay && j >= a.budget);
        counts += __popcll(ho[g]) + (__popcll(mo[g]) << 16);
    }
    if (lane == 0) red[2][wave] = counts;
    __syncthreads();
    const int before = across(red[2], total);
    if (t == 0) ws[0] = total & 0xFFFF;
    int *src = ws + 4, *dst = src + evict_most(c.max_len, a.budget);
    int hole = before & 0xFFFF, mover = before >> 16;
#pragma unroll
    for (int g = 0; g < K; ++g) {
        if (ho[g] >> lane & 1) dst[hole + __popcll(ho[g] & lower)] = j0 + 64 * g;
        if (mo[g] >> lane & 1) src[mover + __popcll(mo[g] & lower)] = j0 + 64 * g;
        hole += __popcll(ho[g]), mover += __popcll(mo[g]);
    }
}

template <int U, int KEEP>
static int evict_select(const KvDev &c, const EvictDev &a, hipStream_t st) {
    constexpr int lds = 4 * 64 * kSelectWaves * KEEP;
    static OncePerDevice once;
    if (int rc = allow_lds(once, (const void *)k_evict_select<U, KEEP>, lds, "p8x_kv_evict LDS")) return rc;
    k_evict_select<U, KEEP><<<dim3(c.n_kv, c.n_seq), 64 * kSelectWaves, lds, st>>>(c, a);
    return P8X_OK;
}
template <int K>
static int evict_short(const KvDev &c, const EvictDev &a, hipStream_t st) {
    k_evict_short<K><<<dim3(c.n_kv, c.n_seq), (c.max_len + 64 * K - 1) / (64 * K) * 64, 0, st>>>(c, a);
    return P8X_OK;
}

// The moves: sources are slots >= budget and destinations slots < budget, so no row is both. D / 8 lanes a row, four rows at a
// time: their places, then eight loads, then the stores. Bound by HBM on rows of 2 D bytes: 39 to 42 us for 167 MB (24 heads, 9000 slots
// at most), 4 TB/s.
template <int D>
__global__ __launch_bounds__(256) void k_evict_move(KvDev c, EvictDev a) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    constexpr int PC = D / 8, ROWS = 256 / PC;
    const int h = blockIdx.y, s = blockIdx.z;
    const size_t hd = (size_t)s * c.n_kv + h, base = hd * c.max_len;
    const int *ws = a.ws + hd * evict_words(c.max_len, a.budget);
    const int moves = ws[0], *src = ws + 4, *dst = src + evict_most(c.max_len, a.budget);
    if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.len_out[s] = min(ws[1], a.budget);
    const int r0 = threadIdx.x / PC, e = threadIdx.x % PC;
    const size_t o = (size_t)h * c.head_stride + 8 * e;
    for (int i0 = 4 * ROWS * blockIdx.x + r0; i0 < moves; i0 += 4 * ROWS * gridDim.x) {
        int j0[4], j1[4];
        int64_t from[4], to[4];
        u4 k[4], v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = min(i0 + u * ROWS, moves - 1);   // (the last one once more is harmless)
            j0[u] = src[i], j1[u] = dst[i];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) from[u] = slot_offset(c, s, j0[u]), to[u] = slot_offset(c, s, j1[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t f = max(from[u], (int64_t)0);
            k[u] = *(const u4 *)(c.k + f + o);
            v[u] = *(const u4 *)(c.v + f + o);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (from[u] >= 0 && to[u] >= 0) {
                *(u4 *)(c.k + to[u] + o) = k[u];
                *(u4 *)(c.v + to[u] + o) = v[u];
            }
        if (e == 0) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                a.score_out[base + j1[u]] = a.score[base + j0[u]];
                if (a.pos) a.pos_out[base + j1[u]] = a.pos[base + j0[u]];
            }
        }
    }
}

int launch_kv_evict(const KvDev &c, int D, const p8x_evict_args &p, hipStream_t st) {
    const EvictDev a{p.budget, p.n_sink, p.n_recent, p.score, p.score_out, p.pos, p.pos_out, p.len_out, (int *)p.workspace};
    // Keys in registers up to 8 a lane, as few as fit (both calls, us): 2, 4 and 8 a lane 13.4, 13.7 and 16.1 at 2000 slots; 4 and 8
    // 15.4 and 16.8 at 3000; 1 and 2 the same at 1008. With k_evict_select instead 14.6 at 1008 slots, 18.1 at 2000, 20.8 at 4000, 24.5 for 19.7
    // at 6000. There keys in LDS 86 and read again 100 at 32767.
    const int rc = c.max_len <= 1024 * 2       ? evict_short<2>(c, a, st)
                   : c.max_len <= 1024 * 4     ? evict_short<4>(c, a, st)
                   : c.max_len <= 1024 * 8     ? evict_short<8>(c, a, st)
                   : c.max_len <= 16 * 32 * 64 ? evict_select<16, 32>(c, a, st)
                                               : evict_select<8, 0>(c, a, st);
    if (rc) return rc;
    const int64_t rows = 4 * (256 / (D / 8));   // of a workgroup at a time
    const int nb = (int)std::max<int64_t>(1, std::min<int64_t>(((int64_t)evict_most(c.max_len, a.budget) + rows - 1) / rows, 1024));
    const dim3 grid(nb, c.n_kv, c.n_seq);
    if (D == 64) k_evict_move<64><<<grid, 256, 0, st>>>(c, a);
    else if (D == 128) k_evict_move<128><<<grid, 256, 0, st>>>(c, a);
    else k_evict_move<256><<<grid, 256, 0, st>>>(c, a);
    return hip_check(hipGetLastError(), "p8x_kv_evict launch");
}

}  // namespace p8x
