// p8x_prompt.hip -- causal attention of new tokens over the cache that holds them (p8x_attn_prompt).
//
// Rows: the (token, head of the group) pairs of a sequence and key/value head, token-major, so that the rows of a workgroup
// end at about the same slot and share K and V. A wave has 32 rows; tiles of 64 slots (32 where 64 do not fit) come to LDS
// asynchronously, once for the workgroup, in a ring of stages. Products on v_mfma_f32_32x32x16, transposed throughout so that
// nothing passes through LDS between the two:
//   S^T [slot][row] = K Q^T: A = K (lane m = lane % 32 is the slot, 8 elements at 8 (lane / 32)), B = Q, kept in registers; of its
//   result lane (row, g) has slots 8 (i / 4) + 4 g + i % 4 of 32. The weights in that place are, as they are, B operands of
//   O^T [element][row] = V^T P^T when the operand's k index 8 g + j stands for slot 4 g + j (j < 4) or 8 + 4 g + j - 4 of 16;
//   A = V^T by ds_read_b64_tr_b16, which transposes blocks of 4 slots by 16 elements.
// Softmax: the weights of a tile are relative to the row's reference m of the tiles before. Their sum, which is needed anyway,
// tells whether that was good: where it is beyond 2^8 (or NaN, or there is no reference yet) the tile's largest score becomes the
// reference, the sums are scaled and the weights made again, so that the usual tile needs no maximum and no exchange between lanes.
// 16-bit queries take weights of one 16-bit part: a second would be half as many products again where the matrix units bound the call, for
// an error beside that of the result's own rounding (together 0.0020 to 0.0023 of the largest for bf16, 0.0016 to 0.0017 by the
// rounding alone; fp16 0.00027, 0.0002). Callers who need more pass f32 queries, with weights of two parts (fp16) or three (bf16). Sums are
// f32, of the unrounded weights. fp16
// parts end at 2^-24: weights stand there times 2^7, and where a tile's largest is below 2^-10, as in a tail beside slots that
// take nearly all, m moves down to it, as far as f32 sums have the range for: until what was summed stands at 2^64 (kRoom), m 2^57 below it
// (a weight's 2^7 apart). Steps of 2^-24 there are 2^-88 of the sum so far, and where a much larger score follows, the factor 2^(m - its m)
// ends at 2^-126: what is below 2^-69 of the row's sum may be lost.
//
// What bounds it: the matrix units, at the clock that the card's power leaves. 8190 tokens of 32 heads on 8 of 128 elements, fp16: 550
// GFLOP in 541 to 592 us by card, 930 to 1017 TFLOP/s, where a large library product reaches 1191; K, V and queries together would take 20 us
// from HBM. The matrix units are busy for 51% of the cycles (63% with f32 queries, which have twice the products to an exponential), the
// clock is about 1.85 GHz meanwhile. f32 queries, fp16 cache, 999 tokens over 16000 slots: 254 GFLOP, products of two parts, in 497 to 507 us,
// 1022 to 1000 TFLOP/s counting both; on a bf16 cache, three parts, 590. 4096 tokens of 64 elements, 69 GFLOP: fp16 99 us, bf16 93, f32 queries
// 159 and 189. Rows of 256 elements, bf16: 471 GFLOP in 537 us, 877 TFLOP/s: segments are as many as compute units, the longest of 320 tiles where
// the mean is 253, and the registers do not suffice: with 16-bit queries 16 (eight waves) or 19 (four) go to scratch, of which a turn of the
// steady loop reads none, one or two back and waits for all loads in flight, the ring's too. With f32 queries on bf16 60 do, and a turn reads
// 13: 2 x 700 tokens over 8190 slots, 16 heads, 1108 us, on fp16 (none) 839, with 16-bit queries 211 to 219. What else was tried at 8190 tokens:
// operands of LDS eight products ahead instead of four (slower: reads in flight beyond about eight delay each other), two barriers a turn (605
// against 541 us for 256 elements), the loads among the products (nothing). Few rows are bound by what is done in turn, 10 us at least: the
// tables, the first K, the products of a tile, the sums. Each workgroup reads `first` and `len` of all sequences to find its own: one token of 256
// sequences of <= 201 slots 95 us, of 1024 477, of 4096 3.6 ms (floors 25, 98, 392).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_attn.h"

namespace p8x {

typedef float float16v __attribute__((ext_vector_type(16)));

template <bool BF>
__device__ __forceinline__ float16v mfma32(uint4v a, uint4v b, float16v c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// log2 of how far a tile's weights may add up beyond 1 before the reference moves up, and of how large the f32 sums may become
// by its moving down
constexpr float kUp = 8.0f, kRoom = 64.0f;
constexpr int kStages = 4;   // in LDS: two in use (K of the next tile, V of this one), the others on their way
// slots of a tile: fewer where the operands of 64 do not fit the registers, or two rings of stages LDS
__host__ __device__ constexpr int tile_slots(int D, bool bf, bool qf, bool halves) { return D == 256 || (D == 128 && ((bf && qf) || halves)) ? 32 : 64; }

struct PromptJob {
    KvDev c;
    DraftDev d;
    void *out; size_t ldo, hso; int out_dtype;
    float *lse;
    float *part;   // a record of each workgroup of a split segment: rows x D sums, then rows x (m, l)
    int heads_wg;  // workgroups of a key/value head
    int split;     // segments may be split over workgroups
};

// A sequence's share of a head's workgroups: it has rts row tiles (segments) of at most `tiles` tiles of slots, each cut into
// `parts`.
struct PromptSeq { int nt, n, first, rts, tiles, parts; };

// sum and largest of what the first n lanes have (n at most 64; the others 0)
__device__ __forceinline__ float first_total(float v, int n) {
    for (int o = 1; o < min(n, 64); o <<= 1) v += __shfl_xor(v, o);
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
__device__ __forceinline__ int first_most(int v, int n) {
    for (int o = 1; o < min(n, 64); o <<= 1) v = max(v, __shfl_xor(v, o));
    return __builtin_amdgcn_readfirstlane(v);
}

template <int ROWS, int TS>
__device__ __forceinline__ PromptSeq prompt_seq(const PromptJob &J, int s, int per) {
    PromptSeq q{};
    if (s >= J.c.n_seq) return q;
    q.nt = seq_tokens(J.d, s, q.first);
    q.n = seq_len(J.c, s);
    q.rts = (int)(((int64_t)q.nt * J.d.G + ROWS - 1) / ROWS);
    q.tiles = (q.n + TS - 1) / TS;
    q.parts = per ? max(1, (q.tiles + per - 1) / per) : 1;
    return q;
}

// Tiles of a part: as few as a head's workgroups allow, but the join costs what kRecord slots do for each record that it reads, so
// that a longest segment of n slots is done first in parts of about sqrt(n * kRecord). Where no segment would get shorter by more
// than kJoin, 0: they stay whole, and nothing is joined. COST: what a slot takes against one of 128 elements.
constexpr int kRecord = 32, kLeast = 128, kJoin = 384;
__host__ __device__ constexpr int slot_cost(int D) { return D == 256 ? 2 : 1; }
template <int COST, int ROWS, int TS>
__device__ __forceinline__ int prompt_per(const PromptJob &J) {
    if (!J.split) return 0;
    const int lane = threadIdx.x & 63;
    auto least = [](int tiles) { return max(max(2, kLeast / COST / TS), (int)(__builtin_amdgcn_sqrtf((float)tiles * kRecord / COST / TS) + 0.5f)); };
    int most = 0, per;
    if (J.c.n_seq == 1) {
        const PromptSeq q = prompt_seq<ROWS, TS>(J, 0, 0);
        if (q.rts == 0) return 0;
        const int parts = J.heads_wg / q.rts;
        most = q.tiles, per = max(least(most), (q.tiles + parts - 1) / parts);
    } else {
        auto over = [&](auto f) {   // f(sequence) summed; in f32: products of long sequences pass 31 bits
            float t = 0.0f;
            for (int s0 = 0; s0 < J.c.n_seq; s0 += 64) t += first_total(f(s0 + lane), J.c.n_seq);
            return t;
        };
        const float tiles = over([&](int s) {
            const PromptSeq q = prompt_seq<ROWS, TS>(J, s, 0);
            most = max(most, q.rts ? q.tiles : 0);
            return (float)q.rts * (float)q.tiles;
        });
        most = first_most(most, J.c.n_seq);
        per = max(least(most), (int)(tiles / (float)J.heads_wg) + 1);
        // (there are at least twice as many workgroups as segments: twice the first `per` fits, or, of sequences that overlap in
        // `first` and so may have more segments than that, none)
        while (per < most && over([&](int s) { const PromptSeq q = prompt_seq<ROWS, TS>(J, s, per); return (float)q.rts * (float)q.parts; }) > (float)J.heads_wg) per += (per + 7) / 8;
    }
    return most - per <= kJoin / COST / TS ? 0 : per;
}

// The segment x (of a head's, all sequences' in a row; `part` of it when they are counted in parts): its sequence's numbers, s = -1
// behind the last
template <int ROWS, int TS>
__device__ __forceinline__ PromptSeq prompt_find(const PromptJob &J, int per, bool in_parts, int x, int &s, int &rt, int &part) {
    const int lane = threadIdx.x & 63;
    PromptSeq r{};
    int i = x;   // among the sequence's
    s = -1, rt = part = 0;
    if (J.c.n_seq == 1) {
        r = prompt_seq<ROWS, TS>(J, 0, per);
        if (x < r.rts * (in_parts ? r.parts : 1)) s = 0;
    } else {
        for (int s0 = 0, base = 0; s0 < J.c.n_seq && s < 0; s0 += 64) {
            PromptSeq q = prompt_seq<ROWS, TS>(J, s0 + lane, per);
            int id = s0 + lane;
            if (!per && J.c.n_seq <= 64) {   // whole segments: those of the longest sequence first (16 of 400 to 4400 slots 165 us, in their order 195)
                const int mine = q.rts ? q.tiles : 0;
                int at = 0;
                for (int j = 0; j < J.c.n_seq; ++j) {
                    const int its = __builtin_amdgcn_readlane(mine, j);
                    at += its > mine || (its == mine && j < lane);
                }
                if (lane >= J.c.n_seq) at = lane;
                auto to = [&](int a) { return __builtin_amdgcn_ds_permute(4 * at, a); };
                q = PromptSeq{to(q.nt), to(q.n), to(q.first), to(q.rts), to(q.tiles), to(q.parts)};
                id = to(lane);
            }
            const int v = q.rts * (in_parts ? q.parts : 1);
            int y = v;
            for (int o = 1; o < min(J.c.n_seq, 64); o <<= 1) {   // (lanes behind the last sequence add nothing)
                const int z = __shfl_up(y, o);
                if (lane >= o) y += z;
            }
            const uint64_t in = __ballot(base + y > x);
            if (in) {
                const int f = __ffsll((unsigned long long)in) - 1;
                auto of = [&](int a) { return __builtin_amdgcn_readlane(a, f); };
                r = PromptSeq{of(q.nt), of(q.n), of(q.first), of(q.rts), of(q.tiles), of(q.parts)};
                s = of(id);
                i = x - base - of(y - v);
            }
            base += __builtin_amdgcn_readlane(y, min(J.c.n_seq - s0, 64) - 1);
        }
    }
    if (s < 0) return r;
    if (in_parts && r.parts > 1) {
        part = i % r.parts;
        i /= r.parts;
    }
    rt = r.rts - 1 - i;   // the longest first
    return r;
}

__device__ __forceinline__ float lse_of(float m, float l, float bias) { return l == 0.0f ? -INFINITY : (m - bias + __log2f(l)) * kLn2; }

// four elements of the result, from the joined sums
__device__ __forceinline__ void store_out(const PromptJob &J, int first, int h, int row, int e, float4v v, float m, float l, float bias) {
    const int G = J.d.G, i = row / G, head = h * G + row - i * G;
    v *= l == 0.0f ? 0.0f : 1.0f / l;
    const size_t at = (size_t)(first + i) * J.ldo + (size_t)head * J.hso + e;
    if (J.out_dtype == P8X_F32) *(float4v *)((float *)J.out + at) = v;
    else if (J.out_dtype == P8X_BF16) *(uint2v *)((uint16_t *)J.out + at) = uint2v{pack2<true>(v[0], v[1]), pack2<true>(v[2], v[3])};
    else *(uint2v *)((uint16_t *)J.out + at) = uint2v{pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3])};
    if (e == 0 && J.lse) J.lse[(size_t)(first + i) * J.c.n_kv * G + head] = lse_of(m, l, bias);
}

// HALVES: the second four waves have the rows of the first, over the second half of the tiles, in a ring of stages of their own; the sums
// of both meet in LDS at the end.
template <int D, bool BF, bool QF, int WAVES, bool HALVES>
__global__ __launch_bounds__(64 * WAVES, QF && D == 256 ? 1 : 2) void k_prompt(PromptJob J) {
    constexpr int TS = tile_slots(D, BF, QF, HALVES), GW = HALVES ? WAVES / 2 : WAVES, SUB = TS / 32, C = D / 16, DT = D / 32, KS = TS / 16, PC = D / 8, ROW = 2 * D, ROWS = 32 * GW;
    constexpr int QP = QF ? (BF ? 3 : 2) : 1, PP = QP;
    constexpr float kBias = BF ? 0.0f : 7.0f;
    // (fp16) log2 of a lane's sum of weights below which the tile's largest is looked up, and of that one below which m moves down
    constexpr float kLow = QF ? 5.0f : 10.0f, kDown = 10.0f;
    extern __shared__ float4v sh4[];
    constexpr bool PING = WAVES == 8;
    __shared__ int odd_rows[HALVES ? 2 : 1][8][TS], any_odds[HALVES ? 2 : 1][8][GW];   // slots with infinities or NaN among their values, of stages that some rows see in part; whether a wave found any
    const KvDev &c = J.c;
    const DraftDev &d = J.d;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5, ln = lane & 31;
    const int h = blockIdx.x % c.n_kv;
    int s, rt, part;
    const int per = prompt_per<slot_cost(D), ROWS, TS>(J);
    const PromptSeq q = prompt_find<ROWS, TS>(J, per, true, blockIdx.x / c.n_kv, s, rt, part);
    if (s < 0) return;
    const int G = d.G, rows = q.nt * G, rows_here = min(ROWS, rows - rt * ROWS), ahead = q.n - q.nt;   // slots before the tokens
    // tiles of the row tile's last token, and this part's
    const int tiles = (max(0, ahead + (rt * ROWS + rows_here - 1) / G + 1) + TS - 1) / TS;
    const int share = q.parts == 1 ? tiles : tiles / q.parts, more = tiles - share * q.parts;
    const int p0 = part * share + min(part, more), p1 = p0 + share + (part < more), turns = HALVES ? (p1 - p0 + 1) / 2 : p1 - p0;
    // the waves' half, and their number in it
    const int half = HALVES ? wave >> 2 : 0, gw = HALVES ? wave & 3 : wave;
    const int t0 = half ? p0 + turns : p0, t1 = half ? p1 : p0 + turns;
    auto &odd_row = odd_rows[half];
    auto &any_odd = any_odds[half];
    const uint16_t *kp = c.k + (size_t)h * c.head_stride, *vp = c.v + (size_t)h * c.head_stride;
    const uint32_t ss = (uint32_t)c.slot_stride;
    const int td = max(0, ahead + rt * ROWS / G + 1) / TS;   // the first tile that some row sees in part only

    // ---- K and V of stage t to LDS: straight there where all of the wave's rows are in use and have a page, else through
    // registers, rows that are not there as zeros
    constexpr int RWV = 64 / PC, RP = GW * RWV, PASS = TS / RP;   // rows of a wave and of the workgroup in a pass
    constexpr int STAGE = TS * ROW;                                  // bytes of a stage's K; its V follows
    static_assert(PASS >= 1 && TS % RP == 0 && RWV <= 16, "passes");
    // 16-byte pieces of a row lie at p ^ fk(row) (K), p ^ fv(row) (V), so that a read's rows are in other banks
    auto fk = [](int row) { return PC < 16 ? row >> 1 & 7 : row & 15; };
    auto fv = [](int row) { return PC < 16 ? (row >> 1 & 1) << 2 : (row & 3) << 2; };
    char *const lds = (char *)sh4 + half * kStages * 2 * STAGE;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const int rl = lane / PC, pl = lane % PC;
    uint32_t kl[2], vl[2];   // the lane's bytes from its 16 slots' first
#pragma unroll
    for (int p = 0; p < (RP % 16 ? 2 : 1); ++p) {
        const int r15 = (p * RP + gw * RWV + rl) & 15;
        kl[p] = 2 * (r15 * ss + 8 * (pl ^ fk(r15)));
        vl[p] = 2 * (r15 * ss + 8 * (pl ^ fv(r15)));
    }
    // Of CH stages from c0 on, the lanes hold where their groups of 16 slots lie; bit KS i + k: group k of stage c0 + i has a page
    constexpr int CH = 64 / KS;
    int lo = 0, hi = 0, c0 = 0;
    uint64_t here = 0, before = 0;   // of these stages, of the CH before them
    auto pages = [&](int st) {
        const int slot = TS * (t0 + st + lane / KS) + 16 * (lane % KS);
        int64_t off = -1;
        if (t0 + st + lane / KS < t1 && slot < q.n) off = slot_offset(c, s, slot);
        lo = (int)off, hi = (int)(off >> 32), c0 = st;
        before = here;
        here = __ballot(off >= 0);
    };
    auto group = [&](int st, int p) {   // where the 16 slots of the wave's rows of a pass lie
        const int from = (st - c0) * KS + (p * RP + gw * RWV) / 16;
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, from) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, from));
    };
    auto load_direct = [&](int t, int i) {   // load i of 2 PASS
        const int p = i / 2;
        const uint32_t to = lds0 + (uint32_t)(t - t0) % kStages * 2 * STAGE + (p * RP + gw * RWV) * ROW;
        const int64_t off = group(t - t0, p);
        if (i % 2) load_lds(vp + off, vl[RP % 16 ? p & 1 : 0], to + STAGE);
        else load_lds(kp + off, kl[RP % 16 ? p & 1 : 0], to);
    };
    auto load = [&](int t) {
        if ((t - t0) % CH == 0) pages(t - t0);
        bool direct = true;
#pragma unroll
        for (int p = 0; p < PASS; ++p) direct = direct && group(t - t0, p) >= 0 && TS * t + p * RP + gw * RWV + RWV <= q.n;
        if (direct) {
#pragma unroll
            for (int i = 0; i < 2 * PASS; ++i) load_direct(t, i);
            return;
        }
        const uint32_t buf = (uint32_t)(t - t0) % kStages * 2 * STAGE;
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the stages before have arrived
#pragma unroll 1
        for (int p = 0; p < PASS; ++p) {
            const int r = p * RP + gw * RWV + rl;
            const int64_t off = group(t - t0, p);
            uint4v k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
            if (off >= 0 && TS * t + r < q.n) {
                const size_t at = (size_t)off + (size_t)(r % 16) * ss + 8 * pl;
                k = *(const uint4v *)(kp + at);
                v = *(const uint4v *)(vp + at);
            }
            *(uint4v *)(lds + buf + r * ROW + (pl ^ fk(r)) * 16) = k;
            *(uint4v *)(lds + buf + STAGE + r * ROW + (pl ^ fv(r)) * 16) = v;
        }
    };
    // which groups of tile t have a page
    auto present = [&](int t) { return (uint32_t)(t - t0 >= c0 ? here >> (t - t0 - c0) * KS : before >> (t - t0 - c0 + CH) * KS) & ((1u << KS) - 1); };
    // Waits until the wave's part of stage t has arrived; a barrier then tells of the others'. Loads come back in order, 2 PASS of
    // each stage: younger stages may be on their way (a stage through registers has waited for all before it; other loads make
    // the wait longer, never shorter).
    int loaded = t0;
    auto arrive = [&](int t) {
        if (loaded > t + 2) __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * PASS) : "memory");
        else if (loaded > t + 1) __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PASS) : "memory");
        else __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (t >= td && t < t1) {   // some of the slots may be hidden from some rows: infinities and NaN among the wave's values
            bool any = false;
#pragma unroll 1
            for (int p = 0; p < PASS; ++p) {
                const int r = p * RP + gw * RWV + rl;
                uint4v *at = (uint4v *)(lds + (uint32_t)(t - t0) % kStages * 2 * STAGE + STAGE + r * ROW + pl * 16);
                uint4v v = *at;
                bool has = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t w = v[e];
                    has |= take_odd<BF>(w);
                    v[e] = w;
                }
                const uint64_t by = __ballot(has);
                if (by) *at = v;
                if (pl == 0) odd_row[(uint32_t)(t - t0) % 8][r] = (by >> (rl * PC) & (PC == 64 ? ~0ull : (1ull << PC) - 1)) != 0;
                any |= by != 0;
            }
            if (lane == 0) any_odd[(uint32_t)(t - t0) % 8][gw] = any;
        }
        __syncthreads();
    };
    const int grp = PING ? wave >> 2 : 0, next = 2 + grp;   // a turn loads the stage so many behind its own
#pragma unroll 1
    for (; loaded < min(t1, t0 + next); ++loaded) load(loaded);

    // ---- the wave's rows: queries, last slot that each sees
    uint4v qf[QP][C];
    float16v o[DT];
    float m, l, c2;
    int lim;
    const int row0 = rt * ROWS + gw * 32, wrows = min(32, rows - row0);   // of the wave (0 or less: none)
    const int last = ahead + (row0 + max(wrows, 1) - 1) / G, least = ahead + row0 / G;   // slots of the wave's last and first token
    const int tw = wrows > 0 ? min(t1, (max(0, last + 1) + TS - 1) / TS) : t0;
    {
        const int r = row0 + ln, i = min(r, rows - 1) / G;
        const bool on = r < rows;   // the others have queries of zeros and see what the last one does
        lim = ahead + i;
        m = -INFINITY;
        l = 0.0f;
        c2 = fabsf(d.scale) * kLog2e;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[t][e] = 0.0f;
        const size_t at = on ? (size_t)(q.first + i) * d.ld_q + (size_t)(h * G + r - i * G) * d.hs_q + 8 * g : 0;
        if constexpr (QF) {
            // fp16 parts need the row scaled to 2^13 (the lane 32 apart holds the other half of it)
            const float *p = (const float *)d.q + at;
            float f[C][8], mx = 0.0f;
#pragma unroll
            for (int k = 0; k < C; ++k) {
                const float4v x = on ? *(const float4v *)(p + 16 * k) : float4v{0, 0, 0, 0}, y = on ? *(const float4v *)(p + 16 * k + 4) : float4v{0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[k][e] = x[e], f[k][e + 4] = y[e];
                    mx = fmaxf(mx, fmaxf(fabsf(x[e]), fabsf(y[e])));
                }
            }
            float s1 = d.scale < 0 ? -1.0f : 1.0f, s2 = 1.0f;
            if constexpr (!BF) {
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const int ex = mx > 0.0f && mx < INFINITY ? 13 - (int)((__builtin_bit_cast(uint32_t, mx) >> 23) - 127) : 0;
                const int e1 = min(ex, 100);   // in two steps: 2^ex may be beyond f32
                s1 *= ldexpf(1.0f, e1), s2 = ldexpf(1.0f, ex - e1);
                c2 = ldexpf(c2, -ex);
            }
#pragma unroll
            for (int k = 0; k < C; ++k) {
                uint4v w[QP];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[k][e] = f[k][e] * s1 * s2;
                split8<BF, QP>(f[k], w);
#pragma unroll
                for (int n = 0; n < QP; ++n) qf[n][k] = w[n];
            }
        } else {
#pragma unroll
            for (int k = 0; k < C; ++k) {
                uint4v w = on ? *(const uint4v *)((const uint16_t *)d.q + at + 16 * k) : uint4v{0, 0, 0, 0};
                if (d.scale < 0) w ^= uint4v{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};   // its sign goes into the queries
                qf[0][k] = w;
            }
        }
        c2 = fmaxf(c2, 0x1p-149f);   // of a scale of 0, or one that underflows: hidden scores, -inf, stay so
    }

    const int k_at = ln * ROW + ((g ^ fk(ln)) * 16);   // pieces 2 c + g: c only flips higher bits
    const int tl = lane & 15, v_row = 4 * g + (tl >> 2), v_at = v_row * ROW + ((((lane >> 4 & 1) * 2 + (tl >> 1 & 1)) ^ fv(v_row)) * 16) + 8 * (tl & 1);
    auto place = [&](int t) { return lds + (uint32_t)(t - t0) % kStages * 2 * STAGE; };
    auto qk = [&](const char *k, float16v (&x)[SUB]) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[u][e] = 0.0f;
#pragma unroll
        for (int n = 0; n < C; ++n)
#pragma unroll
            for (int u = 0; u < SUB; ++u) {   // (sums in turn: a product waits for the one before on its own)
                const uint4v kf = *(const uint4v *)(k + (k_at ^ 32 * n) + 32 * u * ROW);
#pragma unroll
                for (int p = QP - 1; p >= 0; --p)   // small parts first
                    x[u] = mfma32<BF>(kf, qf[p][n], x[u]);
            }
    };
    // scores to weights, in parts; returns the lane's sum of them
    auto weights = [&](const float16v (&x)[SUB], float c2, float m, uint4v (&p)[KS][PP]) {
        const float base = (m == -INFINITY ? 0.0f : m) - kBias;
        float sum = 0;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f[e] = __builtin_amdgcn_exp2f(fmaf(x[u][8 * half + e], c2, -base));
                    sum += f[e];
                }
                uint4v w[PP];
                split8<BF, PP>(f, w);
#pragma unroll
                for (int n = 0; n < PP; ++n) p[2 * u + half][n] = w[n];
            }
        return sum;
    };
    bool settled = false;   // every row has a reference
    auto softmax = [&](float16v (&x)[SUB], uint4v (&p)[KS][PP]) {
        float sum;
        bool bad = !settled;
        if (settled) {
            sum = weights(x, c2, m, p);
            bad |= !(sum <= __builtin_exp2f(kUp + kBias));
            if (!BF) bad |= sum < __builtin_exp2f(kBias - kLow);
            bad = __any(bad);
        } else {
            sum = INFINITY;
        }
        if (bad) {
            settled = true;
            float v = -INFINITY;
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) v = fmaxf(v, x[u][e]);
            v = fmaxf(v, __shfl_xor(v, 32)) * c2;   // log2 of the tile's largest (-inf: the row sees none of it)
            float to = m;
            if (v > m && (m == -INFINITY || !(sum <= __builtin_exp2f(kUp + kBias)))) {
                to = v;
            } else if (!BF && v < m - kDown && v > -INFINITY) {
                const float ls = l + __shfl_xor(l, 32);
                to = fmaxf(v, fminf(m, m - (kRoom - __log2f(ls))));
            }
            to = fmaxf(to, __shfl_xor(to, 32));   // where one of the row's two lanes moves up so does the other
            const float al = m == -INFINITY || to == m ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            settled = settled && !__any(to == -INFINITY);
            l *= al;
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] *= al;
            sum = weights(x, c2, m, p);
        }
        l += sum;
    };
    // hides what a row does not see: later tokens' slots, those without a page
    auto hide = [&](int t, uint32_t pg, float16v (&x)[SUB]) {
        const int see = lim - TS * t - 4 * g;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int upto = pg >> (2 * u + half) & 1 ? see : -1;
#pragma unroll
                for (int e = 8 * half; e < 8 * half + 8; ++e) x[u][e] = 32 * u + 8 * (e / 4) + e % 4 > upto ? -INFINITY : x[u][e];
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    typedef short s4 __attribute__((ext_vector_type(4)));
    auto vt = [&](const char *v, int t, int ks) {   // V^T operand: elements 32 t .., slots 16 ks ..
        uint2v e[2];
#pragma unroll
        for (int half = 0; half < 2; ++half)
            e[half] = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(v + (v_at ^ 64 * t) + (16 * ks + 8 * half) * ROW)));
        return uint4v{e[0][0], e[0][1], e[1][0], e[1][1]};
    };
    constexpr int AHEAD = 4, EARLY = 4;   // operands that are read ahead of their products; of V before the barrier in front of them
    uint4v first[EARLY];
    auto pv = [&](const char *v, const uint4v (&p)[KS][PP]) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const uint4v e = ks * DT + t < EARLY ? first[ks * DT + t] : vt(v, t, ks);
#pragma unroll
                for (int n = PP - 1; n >= 0; --n)
                    o[t] = mfma32<BF>(e, p[ks][n], o[t]);
            }
    };
    // Adds the odd values of a stage's slots, which are zeros there, to the rows that see them.
    auto add_odd = [&](int t) {
        for (int j = 0; j < TS; ++j) {
            if (!__builtin_amdgcn_readfirstlane(odd_row[(uint32_t)(t - t0) % 8][j])) continue;
            const int slot = TS * t + j;
            const uint16_t *p = vp + slot_offset(c, s, slot) + 4 * g;
#pragma unroll
            for (int k = 0; k < DT; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint2v w = *(const uint2v *)(p + 32 * k + 8 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t word = e < 2 ? w[0] : w[1];
                        const float v = e & 1 ? part_hi<BF>(word) : part_lo<BF>(word);
                        o[k][4 * i + e] += !(v - v == 0.0f) && slot <= lim ? v : 0.0f;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    };

    float16v x[SUB];
    uint4v p[KS][PP];
    auto weigh = [&](int t) {
        softmax(x, p);
#pragma unroll
        for (int i = 0; i < EARLY; ++i) first[i] = vt(place(t) + STAGE, i % DT, i / DT);
    };
    // products of the tile's weights and values, then the scores of the next
    auto multiply = [&](int t, int next) {
        __builtin_amdgcn_s_setprio(1);
        pv(place(t) + STAGE, p);
        qk(place(next), x);
        if constexpr (QP == 1) {   // operands from LDS some products ahead, no more of them than registers
            constexpr int NV = KS * DT, NK = SUB * C;
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * (AHEAD - EARLY), 0);
#pragma unroll
            for (int i = 0; i < NV + NK; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                if (i + AHEAD < NV) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                else if (i + AHEAD < NV + NK) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
    };
    // A turn is weights, then products. One barrier a turn: at that of turn t stage t + 1 has arrived and t - 1 is no longer read. Where
    // two waves share a SIMD it lies between weights and products for the first four waves and before the weights for the
    // others, so that from one barrier to the next one of the two multiplies first and then makes weights, the other the other
    // way round. The place of stage t - 1 takes stage t + 3 with the weights that follow the barrier, those of turn t + 1 of the first
    // four waves and of turn t of the others.
    auto start = [&](int t) {
        if (grp) arrive(t + 1);
        if (t + next < t1) load(t + next), loaded = t + next + 1;
    };
    auto middle = [&](int t) {
        if (!grp) arrive(t + 1);
    };
    auto arrive_full = [&]() {
        __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PASS) : "memory");
        __syncthreads();
    };
    if (p0 < p1) {
        arrive(t0);
        if (t0 < tw) qk(place(t0), x);
        int t = t0;
#pragma unroll 1
        while (t < tw) {
            start(t);
            const uint32_t pg = present(t);
            if (TS * t + TS - 1 > least || pg != (1u << KS) - 1) hide(t, pg, x);
            weigh(t);
            middle(t);
            multiply(t, min(t + 1, tw - 1));   // (of the last tile its own scores once more: not used)
            if (t >= td) {
                int any = 0;
#pragma unroll
                for (int w = 0; w < GW; ++w) any |= any_odd[(uint32_t)(t - t0) % 8][w];
                if (__builtin_amdgcn_readfirstlane(any)) add_odd(t);
            }
            ++t;
            // The turns without any of that: all rows have a reference and see all of the tile, pages are there, and there is a stage
            // that goes straight to LDS with each.
            if (!settled || (t - t0 < c0 && ~before)) continue;
            const int run = min(min(td - 2, min(t1, q.n / TS) - next), t0 + c0 - next + (~here ? __builtin_ctzll(~here) : 64) / KS);
#pragma unroll 1
            for (; t < run; ++t) {
                if (grp) arrive_full();
#pragma unroll
                for (int i = 0; i < 2 * PASS; ++i) load_direct(t + next, i);
                loaded = t + next + 1;
                weigh(t);
                if (!grp) arrive_full();
                multiply(t, t + 1);
            }
        }
#pragma unroll 1
        for (; t < t1; ++t) {
            start(t);
            middle(t);
        }
        if constexpr (HALVES) {
            for (int k = t1 - t0; k <= turns; ++k) __syncthreads();   // as many as the other half's, and one: LDS is free
            l += __shfl_xor(l, 32);
            // a lane's sums lie in the same places in both
            float4v *po = sh4 + (size_t)gw * DT * 4 * 64 + lane;
            float2 *pm = (float2 *)(sh4 + (size_t)GW * DT * 4 * 64) + (size_t)gw * 64 + lane;
            if (half) {
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) po[(t * 4 + i) * 64] = float4v{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
                *pm = make_float2(m, l);
            }
            __syncthreads();
            if (half) return;
            const float2 ml = *pm;
            const float mn = fmaxf(m, ml.x), f0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn), f1 = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn);
            m = mn;
            l = l * f0 + ml.y * f1;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4v w = po[(t * 4 + i) * 64];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[t][4 * i + e] = o[t][4 * i + e] * f0 + w[e] * f1;
                }
        }
    }
    if constexpr (HALVES)
        if (half) return;

    // (the cases around the pieces, not in each: what is fetched and run once a workgroup took 3 us of the 20.4 of 512 tokens otherwise, 1.7 so)
    const int r = row0 + ln;
    if constexpr (!HALVES) l += __shfl_xor(l, 32);
    if (r >= rows) return;
    auto pieces = [&](auto f) {   // f(element, four sums from there)
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) f(32 * t + 8 * i + 4 * g, float4v{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]});
    };
    if (q.parts > 1) {
        float *rec = J.part + (size_t)blockIdx.x * ROWS * (D + 2) + (size_t)(r - rt * ROWS) * D;
        if (g == 0) *(float2 *)(J.part + (size_t)blockIdx.x * ROWS * (D + 2) + (size_t)ROWS * D + 2 * (r - rt * ROWS)) = make_float2(m, l);
        pieces([&](int e, float4v v) { *(float4v *)(rec + e) = v; });
        return;
    }
    const int i = r / G, head = h * G + r - i * G;
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    const size_t at = (size_t)(q.first + i) * J.ldo + (size_t)head * J.hso;
    if (g == 0 && J.lse) J.lse[(size_t)(q.first + i) * c.n_kv * G + head] = lse_of(m, l, kBias);
    if (J.out_dtype == P8X_BF16) {
        pieces([&](int e, float4v v) { v *= by; *(uint2v *)((uint16_t *)J.out + at + e) = uint2v{pack2<true>(v[0], v[1]), pack2<true>(v[2], v[3])}; });
    } else if (!QF || J.out_dtype == P8X_F16) {
        pieces([&](int e, float4v v) { v *= by; *(uint2v *)((uint16_t *)J.out + at + e) = uint2v{pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3])}; });
    } else {
        pieces([&](int e, float4v v) { *(float4v *)((float *)J.out + at + e) = v * by; });
    }
}

// The records of split segments: a thread four elements of a row, over all parts in order.
template <int D, int TS, int ROWS, int COST>
__global__ __launch_bounds__(256) void k_prompt_join(PromptJob J) {
    const KvDev &c = J.c;
    const float bias = c.bf16 ? 0.0f : 7.0f;
    const int h = blockIdx.x % c.n_kv, x = blockIdx.x / c.n_kv;
    const int per = prompt_per<COST, ROWS, TS>(J);
    int s, rt, part;
    const PromptSeq q = prompt_find<ROWS, TS>(J, per, false, x, s, rt, part);
    if (s < 0 || q.parts < 2) return;
    // the workgroups of the segment's parts: those of the sequences before, then of the longer row tiles
    int before = 0;
    for (int s0 = 0; s0 < s; s0 += 64) {
        const PromptSeq p = prompt_seq<ROWS, TS>(J, s0 + (threadIdx.x & 63), per);
        before += first_total(s0 + (int)(threadIdx.x & 63) < s ? p.rts * p.parts : 0, J.c.n_seq);
    }
    const int b0 = before + (q.rts - 1 - rt) * q.parts;
    const int rows = min(ROWS, q.nt * J.d.G - rt * ROWS);
    for (int i = blockIdx.y * 256 + threadIdx.x; i < rows * (D / 4); i += gridDim.y * 256) {
        const int r = i / (D / 4), e = i % (D / 4) * 4;
        float4v v = {0, 0, 0, 0};
        float m = -INFINITY, l = 0.0f;
        for (int b = 0; b < q.parts; ++b) {
            const float *rec = J.part + (size_t)((b0 + b) * c.n_kv + h) * ROWS * (D + 2);
            const float2 ml = *(const float2 *)(rec + (size_t)ROWS * D + 2 * r);
            const float4v w = *(const float4v *)(rec + (size_t)r * D + e);
            // (a part without a reference is not left out: of scores of NaN alone its sums are NaN, and else zeros)
            const float mn = fmaxf(m, ml.x), mb = mn == -INFINITY ? 0.0f : mn, f0 = __builtin_amdgcn_exp2f(m - mb), f1 = __builtin_amdgcn_exp2f(ml.x - mb);
            v = v * f0 + w * f1;
            l = l * f0 + ml.y * f1;
            m = mn;
        }
        store_out(J, q.first, h, rt * ROWS + r, e, v, m, l, bias);
    }
}

// Rows of a workgroup: 256, or 128 where sequences have no more rows than those, where contexts are short and too few compute units
// would get a workgroup of 256 (long ones are cut: 2 x 325 tokens of 8 heads a group over 49909 slots 533 us with 128, 386 with
// 256), and where rows of 256 elements and queries of several parts together take more than 256 registers a lane. Segments are split
// where a head has at most half as many as workgroups for it. (Equal shares of all tiles in a row, cut anywhere, balance better but
// read K and V at as many places at once as there are workgroups, which the L2s do not hold: 95 against 72 us at 2048 tokens, 1086
// against 604 at 2 x 8190 slots of 256 elements.) The host knows of a sequence's slots only that they are max_len at most: in a cache with
// room for 2048 or more, 512 tokens take workgroups of 256 rows and a join that finds nothing to do, 26.5 us instead of 19.3 where max_len is
// 512; 19 tokens 13.3 instead of 10.9.
struct PromptPlan { int rows, segs, heads_wg; bool split; size_t rec_bytes; };
static PromptPlan prompt_plan(const KvDev &c, const DraftDev &d, int D) {
    PromptPlan p;
    auto segs = [&](int rows) {   // of a head: row tiles of all sequences, at most
        const int64_t each = ((int64_t)d.max_tokens * d.G + rows - 1) / rows, all = (int64_t)d.n_tokens * d.G / rows + std::min(c.n_seq, d.n_tokens);
        return std::min(each * c.n_seq, all);
    };
    const int cus = num_cus();
    p.rows = (D == 256 && d.q_f32) || (int64_t)d.max_tokens * d.G <= 128 || (c.max_len < 2048 && segs(256) * c.n_kv < cus) ? 128 : 256;
    const int64_t n = segs(p.rows);
    p.segs = (int)n;
    // A round of the compute units; of rows whose records are small two, where one is too few to cut all segments, so that long and
    // short ones even out (24 sequences of one token and 400 to 4000 slots, 8 heads of 128: whole 97 us, so 64; 8 of 1600 to 16000
    // slots in one round 66, in two 76, in three 90), or where a compute unit has room for two workgroups (64 elements: 35 to 28).
    p.heads_wg = cus / c.n_kv;
    if ((D == 64 || p.heads_wg < 2 * n) && (int64_t)d.max_tokens * d.G <= 64) p.heads_wg *= 2;
    p.split = p.heads_wg >= 2 * n && c.max_len > (kJoin + kLeast) / slot_cost(D);
    p.rec_bytes = 4 * (size_t)p.rows * (D + 2);
    return p;
}

size_t attn_prompt_workspace(const KvDev &c, const DraftDev &d, int D) {
    const PromptPlan p = prompt_plan(c, d, D);
    return p.split ? (size_t)p.heads_wg * c.n_kv * p.rec_bytes : 0;
}

template <int D, bool BF, bool QF, int WAVES, bool HALVES>
static int prompt_run(const PromptJob &J, int segs, hipStream_t st) {
    constexpr int TS = tile_slots(D, BF, QF, HALVES), lds = (HALVES ? 2 : 1) * kStages * 2 * TS * 2 * D, ROWS = 32 * (HALVES ? WAVES / 2 : WAVES);
    static OncePerDevice once;
    if (int rc = allow_lds(once, (const void *)k_prompt<D, BF, QF, WAVES, HALVES>, lds, "p8x_attn_prompt LDS")) return rc;
    k_prompt<D, BF, QF, WAVES, HALVES><<<J.heads_wg * J.c.n_kv, 64 * WAVES, lds, st>>>(J);
    if (J.split) {   // a pass of 256 threads for a row tile's pieces, up to 8 of them side by side
        const int64_t pieces = std::min<int64_t>(ROWS, (int64_t)J.d.max_tokens * J.d.G) * (D / 4);
        k_prompt_join<D, TS, ROWS, slot_cost(D)><<<dim3(segs * J.c.n_kv, (unsigned)std::min<int64_t>(8, (pieces + 255) / 256)), 256, 0, st>>>(J);
    }
    return hip_check(hipGetLastError(), "p8x_attn_prompt launch");
}

template <int D, bool BF, bool QF>
static int prompt_form(const PromptJob &J, const PromptPlan &p, hipStream_t st) {
    if constexpr (D == 256 && QF) return prompt_run<D, BF, QF, 4, false>(J, p.segs, st);
    else if (p.rows == 256) return prompt_run<D, BF, QF, 8, false>(J, p.segs, st);
    else if constexpr (D != 128) return prompt_run<D, BF, QF, 4, false>(J, p.segs, st);
    else return prompt_run<D, BF, QF, 8, true>(J, p.segs, st);
}

template <int D, bool BF>
static int prompt_types(const PromptJob &J, const PromptPlan &p, hipStream_t st) {
    return J.d.q_f32 ? prompt_form<D, BF, true>(J, p, st) : prompt_form<D, BF, false>(J, p, st);
}

int launch_attn_prompt(const KvDev &c, const DraftDev &d, int D, void *out, int out_dtype, size_t ldo, size_t hso, float *lse, void *ws, size_t ws_bytes,
                       hipStream_t st) {
    if (c.slot_stride >= (1u << 26)) return set_error(P8X_ERR_UNSUPPORTED, "p8x_attn_prompt: slot_stride %zu (below 2^26)", c.slot_stride);
    const PromptPlan p = prompt_plan(c, d, D);
    PromptJob J{c, d, out, ldo, hso, out_dtype, lse, (float *)ws, p.segs, 0};
    const int room = (int)std::min<size_t>(p.heads_wg, ws_bytes / p.rec_bytes / c.n_kv);
    if (p.split && room >= 2 * p.segs) J.split = 1, J.heads_wg = room;
    if (D == 64) return c.bf16 ? prompt_types<64, true>(J, p, st) : prompt_types<64, false>(J, p, st);
    if (D == 128) return c.bf16 ? prompt_types<128, true>(J, p, st) : prompt_types<128, false>(J, p, st);
    return c.bf16 ? prompt_types<256, true>(J, p, st) : prompt_types<256, false>(J, p, st);
}

}  // namespace p8x
