// p8x_attn.hip -- attention of drafted tokens over the cache and each other (p8x_attn_tree).
//
// Rows: the (token, head of the group) pairs of a sequence and key/value head, token-major; they share K and V. A wave
// multiplies tiles of 32 slots with its 16 NT rows on v_mfma_f32_16x16x32, transposed throughout so that nothing passes
// through LDS between the two products:
//   S^T [slot][row] = K Q^T: A = K (lane m = slot, 8 elements of the row at 8 (lane / 16)), B = Q, kept in registers;
//   its result has, in lane (row, g), slots 4 g + i of each 16: the weights p in that place are, as they are, the B operand
//   of O^T [element][row] = V^T P^T when the operand's k index 8 g + j stands for slot 4 g + j (j < 4) or 16 + 4 g + j - 4.
//   A = V^T: from memory, lane (m, g) takes D / 16 elements of its group's 8 slots and transposes them in registers (one
//   v_perm a dword), output tile t's row m then is element (D / 16) m + t; from LDS, ds_read_b64_tr_b16 transposes blocks
//   of 4 slots by 16 elements, and row m is element 16 t + m.
// Softmax: the reference m of a row, to which its weights are relative, only moves when a score exceeds it by 2^8 in the weight, seen
// by each lane for itself, so that the usual tile needs no exchange between lanes and no rescaling; sums l stay in their
// lanes until the end. Weights enter the product as two 16-bit parts (three for f32 queries on a bf16 cache). bf16 parts have
// the range of f32: a weight keeps 16 bits or more. fp16 parts end at 2^-24: weights stand there times 2^7, and where the largest
// of a row's weights in a tile is below 2^-12 (2^-10 for f32 queries), as in a tail beside slots that take nearly all, m
// moves down to it, as far as the f32 sums have the range for (up to 2^64: what is further below is below 2^-64 of the row's sum).
// So a weight is held to 2^-17 of itself or 2^-19 (2^-22) of the largest of its tile. (Without moving down, weights e^-15 below
// the largest were off by 1.4e-3 of themselves, at e^-26 by 10%. Moving from 2^-8 on, the usual spread of scores moves it back and
// forth: 138 to 146 us at 256 rows of 64, 2 x 65535 slots.)
//
// Work: the 32-slot tiles of all (sequence, head, row tile) segments in a row, an equal share for each of one workgroup a
// compute unit. Where the shares can be cut at the segments' ends without more workgroups or longer shares they are (each
// segment that a workgroup visits costs it some 8 us of latency: queries, sums through LDS, records); else a share may
// span segments. A segment of several workgroups leaves records (sums, maximum, sum of weights) that the last of them
// joins in order, or, where they are many, a second launch. (Shares that always span segments: 118 to 125 us at one sequence of
// 131071 slots, 106 to 111 at four trees of 64, 73 either way at 16 sequences.)
//
// What bounds it: HBM for few rows (8 tokens x 4 heads over 131071 slots x 8 heads, 537 MB: 117 us, 4.6 TB/s with the join; 16
// sequences, 301 MB: 73 us, 4.1 TB/s, the ends of 128 segments included). For many rows the VALU and matrix instructions
// of a tile: 256 rows by 32 slots take a compute unit 1.8 us, where K and V would take 1 from HBM (4 x 64 tokens x 32
// heads over 46484 slots, 43.7 GFLOP: 101 us, 430 TFLOP/s). One token over 1001 slots: 14.5 us of latency: 2 the shares, 3.5 the
// first tile, 2.5 its products (instructions come from memory too), 4 the waves' sums, 3 the join.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_attn.h"

namespace p8x {

// Waves of a workgroup, one of which a compute unit holds: 8 of 256 registers a lane, or 4 of 512 for rows of 256 elements.
// SHARE: the waves that share K and V through LDS, 0 for none.
__host__ __device__ constexpr int attn_waves(int D, int share) { return share ? share : D == 256 ? 4 : 8; }
// log2 of how far a weight may exceed 1 before its row's reference moves up (0: 106 to 116 us at 256 rows a workgroup), and of the
// sums beyond which it does not move down
constexpr float kUp = 8.0f, kRoom = 64.0f;
// tiles that a workgroup's waves share through LDS at a time
__host__ __device__ constexpr int stage_tiles(int D) { return D == 256 ? 1 : 2; }
constexpr int kStages = 4;   // stages in LDS: one in use, the others on their way

struct AttnJob {
    KvDev c;
    DraftDev d;
    void *out; size_t ldo, hso;
    float *lse;
    unsigned *count;   // arrivals of a segment's workgroups, 0 between calls
    float *part;       // two records a workgroup: rows x D sums, then rows x (m, l)
    int2 *where;       // of a segment: first workgroup, workgroups (for a join launch)
    int rw, rt, least; // row waves of a workgroup; row tiles of a sequence at most; units a workgroup takes at least: a tile a wave (twice or
                       // four times that: 15.4 to 18.2 and 20.6 us for one token over 1001 slots)
    int split;         // unit: a tile; 0: a whole segment (no records)
    int join;          // records are joined by a launch of their own
    int nwg;
};

struct Seq { int nt, n, first, rts, tiles; };   // tokens, slots, first token's row, row tiles, tiles of slots and drafts
__device__ __forceinline__ Seq seq_of(const AttnJob &J, int s, int rows_wg) {
    Seq q;
    q.nt = seq_tokens(J.d, s, q.first);
    q.n = seq_len(J.c, s);
    q.rts = (q.nt * J.d.G + rows_wg - 1) / rows_wg;
    q.tiles = q.nt ? (q.n + 31) / 32 + (q.nt + 31) / 32 : 0;
    return q;
}

__device__ __forceinline__ int wave_sum(int v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return __builtin_amdgcn_readfirstlane(v);
}

// How the tiles are shared out: `per` units a workgroup, units of a segment of `tiles` tiles. The same in every wave. A lane
// holds the numbers of one of the first 64 sequences; those of others are read again.
struct Shares {
    int per, aligned, split, total;
    int tiles, segs;   // of the lane's sequence: tiles of a segment, segments
    Seq q;             // and its numbers
    __device__ __forceinline__ int units(int tiles) const { return !split ? tiles > 0 : aligned ? (tiles + per - 1) / per * per : tiles; }
};
// f(tiles, segments) for the lane's sequence of s0 .. s0 + 63
template <typename F>
__device__ __forceinline__ int lane_seq(const AttnJob &J, int rows_wg, const Shares &h, int s0, F f) {
    const int s = s0 + (threadIdx.x & 63);
    if (s0 == 0) return f(h.tiles, h.segs);
    if (s >= J.c.n_seq) return 0;
    const Seq q = seq_of(J, s, rows_wg);
    return f(q.tiles, J.c.n_kv * q.rts);
}
__device__ __forceinline__ Shares share_out(const AttnJob &J, int rows_wg) {
    const int lane = threadIdx.x & 63, n_seq = J.c.n_seq;
    Shares h;
    h.tiles = h.segs = 0;
    if (lane < n_seq) {
        h.q = seq_of(J, lane, rows_wg);
        h.tiles = h.q.tiles, h.segs = J.c.n_kv * h.q.rts;
    }
    auto over = [&](auto f) {   // f(tiles) summed over all segments
        int t = 0;
        for (int s0 = 0; s0 < n_seq; s0 += 64) {
            const int v = lane_seq(J, rows_wg, h, s0, [&](int tiles, int segs) { return segs * f(tiles); });
            t += n_seq > 1 ? wave_sum(v) : __builtin_amdgcn_readfirstlane(v);
        }
        return t;
    };
    h.split = J.split;
    h.aligned = 0;
    if (!J.split) {
        h.total = over([](int t) { return t > 0 ? 1 : 0; });
        h.per = max(1, (h.total + J.nwg - 1) / J.nwg);
        return h;
    }
    h.total = over([](int t) { return t; });
    h.per = max(J.least, (h.total + J.nwg - 1) / J.nwg);
    for (int k = 0; k < 2; ++k) {   // shares cut at segments' ends, of this length or a sixteenth more
        const int per = k ? h.per + (h.per + 15) / 16 : h.per;
        const int parts = over([&](int t) { return (t + per - 1) / per; });
        if (parts <= J.nwg) {
            h.per = per;
            h.aligned = 1;
            h.total = parts * per;
            break;
        }
    }
    return h;
}

template <int D, bool BF, bool QF, int NT, int SHARE>
struct Wave {
    static constexpr int C = D / 32, DV = D / 16, VW = DV / 2;       // K operands a row; elements and dwords of V a lane and slot
    // 16-byte pieces of a row. In LDS a row's pieces lie at p ^ fk(row) (K) or p ^ fv(row) (V), so that the rows of a read are in
    // other banks: 16 rows by 16 bytes of K (ds_read_b128), 8 rows by 32 bytes of V (ds_read_b64_tr_b16).
    static constexpr int PC = D / 8, ROW = 2 * D;
    static __device__ __forceinline__ int fk(int row) { return row & (PC < 16 ? PC - 1 : 15); }
    static __device__ __forceinline__ int fv(int row) { return PC < 16 ? (row >> 1 & 3) << 1 : (row & 7) << 1; }
    static constexpr int QP = QF ? (BF ? 3 : 2) : 1, PP = QF && BF ? 3 : 2;   // 16-bit parts of a query and of a weight
    static constexpr float kBias = BF ? 0.0f : 7.0f;
    static constexpr float kDown = QF ? 10.0f : 12.0f;   // (fp16) log2 of how far below 1 a tile's largest weight may be
    uint4v q[NT][QP][C];
    float4v o[NT][DV];
    float m[NT], l[NT], c2[NT];
    uint4v kf[2][C];
    uint32_t vf[SHARE ? 1 : 8][VW];
    uint4v ve[SHARE ? DV : 1];

    // the lane's rows' queries; a negative scale's sign goes into them
    __device__ __forceinline__ void load_q(const DraftDev &d, int first, int h, int row0, int rows, int lane) {
        const float sc = fabsf(d.scale) * kLog2e;
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            const int r = row0 + 16 * a + (lane & 15), g = lane >> 4;
            const bool on = r < rows;
            const int i = r / d.G;
            const size_t at = on ? (size_t)(first + i) * d.ld_q + (size_t)(h * d.G + r - i * d.G) * d.hs_q + 8 * g : 0;
            m[a] = -INFINITY;
            l[a] = 0.0f;
            c2[a] = sc;
#pragma unroll
            for (int t = 0; t < DV; ++t) o[a][t] = float4v{0, 0, 0, 0};
            if constexpr (QF) {
                float f[C][8];
                c2[a] = load_split<C, BF>((const float *)d.q + at, on, sc, f);
#pragma unroll
                for (int k = 0; k < C; ++k) {
                    uint4v p[QP];
                    if (d.scale < 0)
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[k][e] = -f[k][e];
                    split8<BF, QP>(f[k], p);
#pragma unroll
                    for (int n = 0; n < QP; ++n) q[a][n][k] = p[n];
                }
            } else {
#pragma unroll
                for (int k = 0; k < C; ++k) {
                    uint4v w = on ? *(const uint4v *)((const uint16_t *)d.q + at + 32 * k) : uint4v{0, 0, 0, 0};
                    if (d.scale < 0) w ^= uint4v{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
                    q[a][0][k] = w;
                }
            }
            c2[a] = fmaxf(c2[a], 0x1p-149f);   // of a scale of 0, or one that underflows: hidden scores, -inf, stay so
        }
    }

    // K and V of a 32-slot tile whose two halves of 16 slots start at element offsets h0, h1 of the pools; ko, vo: the
    // lane's own offsets
    __device__ __forceinline__ void load_k(const uint16_t *k, int64_t h0, int64_t h1, uint32_t ko) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            kf[0][c] = *(const uint4v *)(k + h0 + ko + 32 * c);
            kf[1][c] = *(const uint4v *)(k + h1 + ko + 32 * c);
        }
    }
    __device__ __forceinline__ void load_v1(const uint16_t *p, uint32_t *o) {
        if constexpr (VW == 2) *(uint2v *)o = *(const uint2v *)p;
        else
#pragma unroll
            for (int w = 0; w < VW; w += 4) *(uint4v *)(o + w) = *(const uint4v *)(p + 2 * w);
    }
    __device__ __forceinline__ void load_v(const uint16_t *v, int64_t h0, int64_t h1, uint32_t vo, uint32_t ss) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            load_v1(v + h0 + vo + j * ss, vf[j]);
            load_v1(v + h1 + vo + j * ss, vf[j + 4]);
        }
    }
    // the same operands from a tile in LDS; ve: V^T operands of the output tiles
    __device__ __forceinline__ void lds_k(const char *k) {
        const int lane = threadIdx.x & 63, ln = lane & 15, at = ln * ROW + ((lane >> 4) ^ fk(ln)) * 16;   // pieces 4 c + g: c only flips higher bits
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int t = 0; t < 2; ++t) kf[t][c] = *(const uint4v *)(k + (at ^ 64 * c) + 16 * t * ROW);
    }
    __device__ __forceinline__ void lds_v(const char *v) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        const int lane = threadIdx.x & 63, ln = lane & 15, row = 4 * (lane >> 4) + ln / 4, at = row * ROW + fv(row) * 16 + 8 * (ln & 3);
#pragma unroll
        for (int t = 0; t < DV; ++t) {
            uint2v e[2];
#pragma unroll
            for (int half = 0; half < 2; ++half)
                e[half] = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(v + (at ^ 32 * t) + 16 * half * ROW)));
            ve[t] = uint4v{e[0][0], e[0][1], e[1][0], e[1][1]};
        }
    }

    // scores x[a][j] of slot j of the lane's eight
    __device__ __forceinline__ void qk(float (&x)[NT][8]) {
        float4v s[2][NT];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int a = 0; a < NT; ++a) s[t][a] = float4v{0, 0, 0, 0};
#pragma unroll
        for (int n = QP - 1; n >= 0; --n)   // small parts first
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int a = 0; a < NT; ++a) s[t][a] = mfma<BF>(kf[t][c], q[a][n][c], s[t][a]);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[a][4 * t + i] = s[t][a][i];
    }

    // (NaN propagates; fmaxf would quiet each operand first, an instruction apiece)
    static __device__ __forceinline__ float top(float a, float b) { return __builtin_elementwise_maximum(a, b); }
    // scores to weights: x[a][j] of slot j of the lane's eight (-inf: hidden)
    __device__ __forceinline__ void softmax(float (&x)[NT][8]) {
        float mx[NT];
        bool far = false;   // one comparison a tile and row, what follows from it only then
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            mx[a] = top(top(top(top(x[a][0], x[a][1]), x[a][2]), top(x[a][3], x[a][4])), top(top(x[a][5], x[a][6]), x[a][7]));
            const float d = fmaf(mx[a], c2[a], -m[a]);
            far |= BF ? d > kUp : fabsf(d + 0.5f * (kDown - kUp)) > 0.5f * (kDown + kUp);
        }
        bool move = __any(far);
        uint64_t down = 0;
        if (!BF && move) {   // up where one of a row's lanes is, down where all four are (or see nothing, but one does)
            uint64_t up = 0;
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                const float d = fmaf(mx[a], c2[a], -m[a]);
                const uint64_t low = __ballot(d < -kDown), two = low & low >> 32, some = __ballot(d > -INFINITY), of2 = some | some >> 32;
                up |= __ballot(d > kUp);
                down |= two & two >> 16 & (of2 | of2 >> 16) & 0xFFFF;
            }
            move = up | down;
        }
        if (move) {
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                float v = mx[a] * c2[a];
                v = fmaxf(v, __shfl_xor(v, 16));
                v = fmaxf(v, __shfl_xor(v, 32));
                float least = m[a];   // what the reference may become
                if (down) {
                    float s = fmaxf(l[a], __shfl_xor(l[a], 16));
                    s = fmaxf(s, __shfl_xor(s, 32));
                    if (v - m[a] < -kDown && v > -INFINITY) least = fminf(m[a], m[a] - (kRoom - __log2f(s)));
                }
                v = fmaxf(v, least);
                const float al = v == -INFINITY || m[a] == v ? 1.0f : __builtin_amdgcn_exp2f(m[a] - v);
                m[a] = v;
                l[a] *= al;
#pragma unroll
                for (int t = 0; t < DV; ++t) o[a][t] *= al;
            }
        }
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            const float base = (m[a] == -INFINITY ? 0.0f : m[a]) - kBias;
            float s = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[a][j] = __builtin_amdgcn_exp2f(fmaf(x[a][j], c2[a], -base));
                s += x[a][j];
            }
            l[a] += s;
        }
    }

    // the weights' parts; of two fp16 parts the first may be rounded toward zero, the second holds what is left
    __device__ __forceinline__ void parts(const float *x, uint4v *p) {
        if constexpr (!BF && PP == 2 && !QF) {
            float minus1 = -1.0f;
            __asm__("" : "+s"(minus1));   // not known to be -1: x - hi is one v_fma_mix, not a conversion and a subtraction
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[2 * e], x[2 * e + 1]));
                p[0][e] = w;
                p[1][e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf(part_lo<BF>(w), minus1, x[2 * e]), fmaf(part_hi<BF>(w), minus1, x[2 * e + 1])));
            }
        } else {
            split8<BF, PP>(x, p);
        }
    }

    __device__ __forceinline__ void pv(const float (&x)[NT][8]) {
        uint4v p[NT][PP];
#pragma unroll
        for (int a = 0; a < NT; ++a) parts(x[a], p[a]);
#pragma unroll
        for (int w = 0; w < VW; ++w) {   // output tiles 2 w and 2 w + 1
            uint4v e0, e1;
            if constexpr (SHARE) {
                e0 = ve[2 * w], e1 = ve[2 * w + 1];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    e0[j] = __builtin_amdgcn_perm(vf[2 * j + 1][w], vf[2 * j][w], 0x05040100u);
                    e1[j] = __builtin_amdgcn_perm(vf[2 * j + 1][w], vf[2 * j][w], 0x07060302u);
                }
            }
#pragma unroll
            for (int n = PP - 1; n >= 0; --n)
#pragma unroll
                for (int a = 0; a < NT; ++a) {
                    o[a][2 * w] = mfma<BF>(e0, p[a][n], o[a][2 * w]);
                    o[a][2 * w + 1] = mfma<BF>(e1, p[a][n], o[a][2 * w + 1]);
                }
        }
    }
    // hides from the lane's rows the slots whose bit of see[a] (j: slot j of the 32) is not set
    __device__ __forceinline__ void hide(float (&x)[NT][8], const uint32_t (&see)[NT]) {
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            const uint32_t lo = see[a] >> (4 * ((threadIdx.x & 63) >> 4)), hi = lo >> 16;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!((j < 4 ? lo >> j : hi >> (j - 4)) & 1)) x[a][j] = -INFINITY;
        }
    }
    // A drafted token's infinities and NaN, which must not meet the zero weight of a row that does not see the token, are
    // zeros in the product; here they are added to the rows that do. odd: the tokens of the tile (from row tok0 on) that have any.
    __device__ __forceinline__ void add_odd(uint32_t odd, const uint32_t (&see)[NT], const DraftDev &d, int tok0, int h, int lane) {
        const int g = lane >> 4;
        for (; odd; odd &= odd - 1) {
            const int j = __ffs(odd) - 1;
            const size_t at = (size_t)(tok0 + j) * d.ld_kv + (size_t)h * d.hs_kv;
#pragma unroll 1
            for (int t = 0; t < DV; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const size_t e = at + (SHARE ? 16 * t + 4 * g + i : DV * (4 * g + i) + t);
                    const float v = d.kv_f32 ? from16(to16(((const float *)d.v)[e], BF), BF) : from16(((const uint16_t *)d.v)[e], BF);
#pragma unroll
                    for (int a = 0; a < NT; ++a) {
                        const float put = !(v - v == 0.0f) && (see[a] >> j & 1) ? v : 0.0f;
#pragma unroll
                        for (int k = 0; k < DV; ++k) o[a][k][i] += k == t ? put : 0.0f;   // (constant indices keep o in registers)
                    }
                }
        }
    }
};

// which of the drafted tokens j0 .. j0 + 31 the lane's rows see
template <int NT>
__device__ __forceinline__ void draft_mask(const DraftDev &d, const Seq &q, int j0, int row0, int rows, int ln, uint32_t (&see)[NT]) {
    const int left = q.nt - j0;
#pragma unroll
    for (int a = 0; a < NT; ++a) {
        const int r = row0 + 16 * a + ln, i = r / d.G;
        see[a] = r < rows ? (uint32_t)(token_mask(d, q.first + i, i) >> j0) & (left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1) : 0;
    }
}

__device__ __forceinline__ float2 load2_agent(const float *p) {
    const uint64_t v = __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__builtin_bit_cast(float, (uint32_t)v), __builtin_bit_cast(float, (uint32_t)(v >> 32)));
}
__device__ __forceinline__ void store2_agent(float *p, float a, float b) {
    __hip_atomic_store((uint64_t *)p, (uint64_t)__builtin_bit_cast(uint32_t, b) << 32 | __builtin_bit_cast(uint32_t, a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct Part { float4v v; float m, l; };   // four elements of a row
__device__ __forceinline__ void add_part(Part &a, const Part &b) {
    const float mn = fmaxf(a.m, b.m), mb = mn == -INFINITY ? 0.0f : mn;
    const float f0 = __builtin_amdgcn_exp2f(a.m - mb), f1 = __builtin_amdgcn_exp2f(b.m - mb);
    a.m = mn;
    a.l = a.l * f0 + b.l * f1;
    a.v = a.v * f0 + b.v * f1;
}

// Elements e .. e + 3 of row r over records b0 .. b1 - 1 of a segment (of workgroups p0 ..), in order, eight loads in flight
// at a time; AGENT: written in this launch by other workgroups.
template <int D, bool AGENT>
__device__ __forceinline__ Part join_records(const float *part, size_t rec, int rows_wg, int p0, int b0, int b1, int r, int e) {
    Part s{float4v{0, 0, 0, 0}, -INFINITY, 0.0f};
    for (int b = b0; b < b1; b += 8) {
        Part x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int p = min(b + k, b1 - 1);
            const float *q = part + (2 * (size_t)(p0 + p) + (p == 0 ? 1 : 0)) * rec;
            float2 ml;
            if constexpr (AGENT) {
                ml = load2_agent(q + (size_t)rows_wg * D + 2 * r);
                const float2 lo = load2_agent(q + (size_t)r * D + e), hi = load2_agent(q + (size_t)r * D + e + 2);
                x[k].v = float4v{lo.x, lo.y, hi.x, hi.y};
            } else {
                ml = *(const float2 *)(q + (size_t)rows_wg * D + 2 * r);
                x[k].v = *(const float4v *)(q + (size_t)r * D + e);
            }
            x[k].m = ml.x, x[k].l = ml.y;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (b + k < b1) add_part(s, x[k]);
    }
    return s;
}

template <int D, bool BF, bool QF>
__device__ __forceinline__ void store_row(const AttnJob &J, int first, int h, int row, int e, Part p) {
    constexpr float bias = BF ? 0.0f : 7.0f;
    p.v *= p.l == 0.0f ? 0.0f : 1.0f / p.l;
    const int G = J.d.G, i = row / G, head = h * G + row - i * G;
    const size_t at = (size_t)(first + i) * J.ldo + (size_t)head * J.hso + e;
    if constexpr (QF) *(float4v *)((float *)J.out + at) = p.v;
    else *(uint2v *)((uint16_t *)J.out + at) = uint2v{pack2<BF>(p.v[0], p.v[1]), pack2<BF>(p.v[2], p.v[3])};
    if (e == 0 && J.lse) J.lse[(size_t)(first + i) * J.c.n_kv * G + head] = p.l == 0.0f ? -INFINITY : (p.m - bias + __log2f(p.l)) * kLn2;
}

// The records of split segments in a launch of their own: a thread four elements of a row, over all records of its segment
// (SUB 1), or, where they are many and the rows few, over one of eight ranges of them.
template <int D, bool BF, bool QF, int SUB>
__global__ __launch_bounds__(256) void k_attn_join(AttnJob J, int rows_wg) {
    constexpr int PIECES = 256 / SUB;
    __shared__ Part sh[SUB > 1 ? SUB : 1][SUB > 1 ? PIECES : 1];
    const int s = blockIdx.z / J.c.n_kv, h = blockIdx.z % J.c.n_kv, rt = blockIdx.y;
    const int sub = threadIdx.x / PIECES, x4 = blockIdx.x * PIECES + threadIdx.x % PIECES, r = x4 / (D / 4), e = x4 % (D / 4) * 4;
    const int2 at = J.where[(size_t)blockIdx.z * J.rt + rt];
    const Seq q = seq_of(J, s, rows_wg);
    const int p0 = at.x, np = at.y;
    if (rt >= q.rts || q.tiles == 0 || np < 2) return;
    const bool on = r < min(rows_wg, q.nt * J.d.G - rt * rows_wg);
    const int each = (np + SUB - 1) / SUB;
    Part p{float4v{0, 0, 0, 0}, -INFINITY, 0.0f};
    if (on) p = join_records<D, false>(J.part, (size_t)rows_wg * (D + 2), rows_wg, p0, min(np, sub * each), min(np, (sub + 1) * each), r, e);
    if constexpr (SUB > 1) {
        sh[sub][threadIdx.x % PIECES] = p;
        __syncthreads();
        if (sub) return;
        for (int k = 1; k < SUB; ++k) add_part(p, sh[k][threadIdx.x % PIECES]);
    }
    if (on) store_row<D, BF, QF>(J, q.first, h, rt * rows_wg + r, e, p);
}

// SHARE: the waves' rows are many; each tile of K and V is brought to LDS once for all of them, three stages of tiles
// ahead. Else each wave loads its tiles straight into operands.
template <int D, bool BF, bool QF, int NT, int SHARE>
__global__ __launch_bounds__(64 * attn_waves(D, SHARE)) void k_attn(AttnJob J) {
    constexpr int kWaves = attn_waves(D, SHARE);
    typedef Wave<D, BF, QF, NT, SHARE> W;
    constexpr int R16 = 16 * NT, DV = W::DV, PC = W::PC;
    extern __shared__ float4v sh4[];   // SHARE: stages of K, V; then [wave][row][D + 4] sums, [wave][row] m, l
    __shared__ unsigned last;
    __shared__ int paged[8][2 * stage_tiles(D)];   // SHARE: whether a stage's halves have a page
    __shared__ int odd_row[8][32 * stage_tiles(D)];   // SHARE: drafted tokens with infinities or NaN among their values
    float *sh = (float *)sh4;
    const KvDev &c = J.c;
    const DraftDev &d = J.d;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, ln = lane & 15;
    const int RW = J.rw, SW = kWaves / RW, rwi = wave % RW, swi = wave / RW, rows_wg = R16 * RW;
    // consecutive units on one XCD: workgroups go round robin over the eight
    const int nwg = gridDim.x, wg = nwg % 8 ? (int)blockIdx.x : (int)(blockIdx.x % 8) * (nwg / 8) + (int)(blockIdx.x / 8);

    const Shares share = share_out(J, rows_wg);
    const int per = share.per, u0 = wg * per, u1 = min(share.total, u0 + per);
    if (u0 >= u1) return;
    // the sequence of unit u0
    int s = 0, base = 0;
    if (c.n_seq > 1)
        for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
            const int v = lane_seq(J, rows_wg, share, s0, [&](int tiles, int segs) { return segs * share.units(tiles); });
            int x = v;
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(x, o);
                if (lane >= o) x += y;
            }
            const uint64_t in = __ballot(base + x > u0);
            if (in) {
                const int f = __ffsll((unsigned long long)in) - 1;
                s = s0 + f;
                base += __builtin_amdgcn_readlane(x - v, f);
                break;
            }
            base += __builtin_amdgcn_readlane(x, 63);
        }

    W w;
    const uint32_t ss = (uint32_t)c.slot_stride, ko = (uint32_t)ln * ss + 8 * g, vo = 4 * g * ss + DV * ln;
    for (int u = u0; u < u1;) {
        Seq q = share.q;
        if (s >= 64) q = seq_of(J, s, rows_wg);
        const int from = s < 64 ? s : 0;
        q.nt = __builtin_amdgcn_readlane(q.nt, from), q.n = __builtin_amdgcn_readlane(q.n, from), q.first = __builtin_amdgcn_readlane(q.first, from);
        q.rts = __builtin_amdgcn_readlane(q.rts, from), q.tiles = __builtin_amdgcn_readlane(q.tiles, from);
        const int ps = share.units(q.tiles), units = c.n_kv * q.rts * ps;
        if (u >= base + units) {   // past this sequence (or none of its units)
            base += units;
            ++s;
            continue;
        }
        const int seg = (u - base) / ps, t0 = (u - base) - seg * ps, h = seg / q.rts, rt = seg - h * q.rts;
        const int t1 = share.split ? min(q.tiles, t0 + (u1 - u)) : q.tiles, ctx = (q.n + 31) / 32;
        const int sa = u - t0, sb = sa + ps;   // the segment's units
        u = min(u1, sb);
        const int rows = q.nt * d.G, row0 = rt * rows_wg + rwi * R16;
        const uint16_t *kp = c.k + (size_t)h * c.head_stride, *vp = c.v + (size_t)h * c.head_stride;

        if constexpr (SHARE) {
            constexpr int ST = stage_tiles(D), RWV = 64 / PC, RP = kWaves * RWV, PASS = 32 * ST / RP;   // rows of a wave and of the workgroup in a pass
            constexpr int STAGE = 32 * ST * W::ROW;   // bytes of a stage's K; its V follows
            const int rl = lane / PC, pl = lane % PC;
            char *const lds = (char *)sh4;
            const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
            int lo = 0, hi = 0;
            const int stages = (t1 - t0 + ST - 1) / ST;
            // Brings the wave's rows of stage st to LDS: straight there, asynchronously, where all of them are in use and have a
            // page, else through registers, rows that are not there as zeros.
            auto load = [&](int st) {
                constexpr int CH = 64 / PASS;   // stages whose row offsets the lanes hold
                if (st % CH == 0) {
                    const int r0 = (lane % PASS) * RP + wave * RWV, t = t0 + (st + lane / PASS) * ST + r0 / 32, slot = 32 * t + r0 % 32;
                    int64_t off = -1;
                    if (t < min(t1, ctx) && slot < q.n) off = slot_offset(c, s, slot & ~15);
                    lo = (int)off, hi = (int)(off >> 32);
                }
                const int buf = (st % kStages) * 2 * STAGE;
                bool direct = true;
                int64_t off[PASS];
#pragma unroll
                for (int p = 0; p < PASS; ++p) {
                    const int r0 = p * RP + wave * RWV, t = t0 + st * ST + r0 / 32, from = st % CH * PASS + p;
                    off[p] = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, from) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, from));
                    direct = direct && t < min(t1, ctx) && off[p] >= 0 && 32 * t + r0 % 32 + RWV <= q.n;
                    if (lane == 0 && r0 % 16 == 0) paged[st % 8][r0 / 16] = off[p] >= 0;
                }
                if (direct) {
#pragma unroll
                    for (int p = 0; p < PASS; ++p) {
                        const uint32_t to = lds0 + buf + (p * RP + wave * RWV) * W::ROW;
                        const uint16_t *kf = kp + off[p], *vf = vp + off[p];
                        const int r15 = (p * RP + wave * RWV + rl) & 15;   // the lane's row; its bytes from the half's first slot:
                        const uint32_t kl = 2 * (r15 * ss + 8 * (pl ^ W::fk(r15))), vl = 2 * (r15 * ss + 8 * (pl ^ W::fv(r15)));
                        load_lds(kf, kl, to);
                        load_lds(vf, vl, to + STAGE);
                    }
                    return;
                }
                __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the stages before have arrived (see the stage loop)
#pragma unroll 1
                for (int p = 0; p < PASS; ++p) {
                    const int r0 = p * RP + wave * RWV, t = t0 + st * ST + r0 / 32, from = st % CH * PASS + p, r = r0 + rl;
                    const int64_t offs = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, from) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, from));
                    uint4v k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
                    if (t < min(t1, ctx)) {
                        if (offs >= 0 && 32 * t + r % 32 < q.n) {
                            const size_t at = (size_t)offs + (r % 16) * ss + 8 * pl;
                            k = *(const uint4v *)(kp + at);
                            v = *(const uint4v *)(vp + at);
                        }
                    } else if (t < t1) {
                        const int j = 32 * (t - ctx) + r % 32;
                        bool has = false;
                        if (j < q.nt) {
                            const size_t at = (size_t)(q.first + j) * d.ld_kv + (size_t)h * d.hs_kv + 8 * pl;
                            k = draft8(d.k, at, d.kv_f32, BF);
                            v = draft8(d.v, at, d.kv_f32, BF);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                uint32_t w4 = v[e];
                                has |= take_odd<BF>(w4);
                                v[e] = w4;
                            }
                        }
                        const uint64_t by = __ballot(has);
                        if (pl == 0) odd_row[st % 8][r] = (by >> (rl * PC) & (PC == 64 ? ~0ull : (1ull << PC) - 1)) != 0;
                    }
                    *(uint4v *)(lds + buf + r * W::ROW + (pl ^ W::fk(r)) * 16) = k;
                    *(uint4v *)(lds + buf + STAGE + r * W::ROW + (pl ^ W::fv(r)) * 16) = v;
                }
            };
            w.load_q(d, q.first, h, row0, rows, lane);
            // Waits until stage st has arrived; the stage before it is no longer read then, and its place takes stage st +
            // kStages - 1. Loads come back in order, 2 PASS of each stage: the younger ones may be on their way (a stage that went
            // through registers has waited for all before it; other loads make the wait longer, never shorter).
            int loaded = 0;
            auto arrive = [&](int st) {
                const int young = min(kStages - 2, stages - 1 - st);
                if (young == 2) __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * PASS) : "memory");
                else if (young == 1) __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PASS) : "memory");
                else __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
#pragma unroll 1
                for (; loaded < min(stages, st + kStages); ++loaded) load(loaded);
            };
            auto place = [&](int t) { return lds + ((t - t0) / ST % kStages) * 2 * STAGE + 32 * ((t - t0) % ST) * W::ROW; };
#pragma unroll 1
            for (int st = -1; st < 1; ++st) arrive(st);   // (-1: the first loads)
            // the next tile's pages, read with its K: a wait for them after V's reads would be one for V
            int pg[2];
            auto pages = [&](int t) {
                const int *p = paged[(t - t0) / ST % 8] + 2 * ((t - t0) % ST);
                pg[0] = p[0], pg[1] = p[1];
            };
            pages(t0);
            w.lds_k(place(t0));
            uint32_t odd[2] = {0, 0};
            // One body for all tiles, so that the sums stay in their registers. V of a tile and K of the next come from LDS while the
            // scores become weights (the barriers to the scheduler keep it from moving the reads to their uses).
#pragma unroll 1
            for (int t = t0; t < t1; ++t) {
                const int st = (t - t0) / ST, i = (t - t0) % ST, left = q.n - 32 * t;
                float x[NT][8];
                w.qk(x);
                __builtin_amdgcn_sched_barrier(0);
                w.lds_v(place(t) + STAGE);
                uint32_t in = (pg[0] ? 0xFFFFu : 0) | (pg[1] ? 0xFFFF0000u : 0);
                in = t < ctx ? __builtin_amdgcn_readfirstlane(in) & (left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1) : 0;
                if (t >= ctx) {
                    const uint32_t o = (uint32_t)__ballot(lane < 32 && odd_row[st % 8][32 * i + lane]);
                    if (t == ctx) odd[0] = o;
                    else odd[1] = o;
                }
                if (t + 1 < t1) {
                    if (i == ST - 1) arrive(st + 1);
                    pages(t + 1);
                    w.lds_k(place(t + 1));
                }
                __builtin_amdgcn_sched_barrier(0);
                if (in != 0xFFFFFFFFu) {
                    uint32_t see[NT];
                    if (t >= ctx) draft_mask<NT>(d, q, 32 * (t - ctx), row0, rows, ln, see);
                    else
                        for (int a = 0; a < NT; ++a) see[a] = in;
                    w.hide(x, see);
                }
                w.softmax(x);
                w.pv(x);
            }
#pragma unroll 1
            for (int j = 0; j < 2; ++j)
                if (const uint32_t o = j ? odd[1] : odd[0]) {
                    uint32_t see[NT];
                    draft_mask<NT>(d, q, 32 * j, row0, rows, ln, see);
                    w.add_odd(o, see, d, q.first + 32 * j, h, lane);
                }
            __syncthreads();   // the stages' place is free
        } else {
            const int full = min(t1, q.n / 32);   // tiles of 32 slots in use
            bool have_q = false;
            for (int tb = t0 + swi; tb < full; tb += 32 * SW) {
                // offsets of the wave's next 64 halves, a lane each: tile tb + SW (lane / 2), half lane & 1
                int64_t off = -1;
                {
                    const int t = tb + SW * (lane >> 1);
                    if (t < full) off = slot_offset(c, s, 32 * t + 16 * (lane & 1));
                }
                const int lo = (int)off, hi = (int)(off >> 32), many = min(32, (full - tb + SW - 1) / SW);
                auto half = [&](int i) { return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, i)); };
                int64_t h0 = half(0), h1 = half(1);
                w.load_k(kp, max(h0, (int64_t)0), max(h1, (int64_t)0), ko);
                w.load_v(vp, max(h0, (int64_t)0), max(h1, (int64_t)0), vo, ss);
                if (!have_q) w.load_q(d, q.first, h, row0, rows, lane);   // behind the loads of the first tile
                have_q = true;
                for (int i = 0; i < many; ++i) {
                    const int64_t n0 = half(2 * min(i + 1, many - 1)), n1 = half(2 * min(i + 1, many - 1) + 1);
                    float x[NT][8];
                    w.qk(x);
                    if (i + 1 < many) w.load_k(kp, max(n0, (int64_t)0), max(n1, (int64_t)0), ko);
                    if ((h0 | h1) < 0) {   // a half without a page: hidden, its values zeros
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if ((j < 4 ? h0 : h1) >= 0) continue;
#pragma unroll
                            for (int a = 0; a < NT; ++a) x[a][j] = -INFINITY;
                            for (int e = 0; e < W::VW; ++e) w.vf[j][e] = 0;
                        }
                    }
                    w.softmax(x);
                    w.pv(x);
                    if (i + 1 < many) w.load_v(vp, max(n0, (int64_t)0), max(n1, (int64_t)0), vo, ss);
                    h0 = n0, h1 = n1;
                }
            }
            if (!have_q) w.load_q(d, q.first, h, row0, rows, lane);
            // the cache's last, partial tile and the drafted tokens
            const int t_rest = max(t0, q.n / 32);
            for (int t = t_rest + (swi - (t_rest - t0) % SW + SW) % SW; t < t1; t += SW) {
                const bool draft = t >= ctx;
                uint32_t see[NT];
                const int j0 = 32 * (t - ctx), left = draft ? q.nt - j0 : q.n - 32 * t;
                int64_t h0 = 0, h1 = 0;
                if (draft) {
                    draft_mask<NT>(d, q, j0, row0, rows, ln, see);
                } else {
                    h0 = slot_offset(c, s, 32 * t);
                    h1 = left > 16 ? slot_offset(c, s, 32 * t + 16) : -1;
                    for (int a = 0; a < NT; ++a) see[a] = ((1u << left) - 1) & ((h0 >= 0 ? 0xFFFFu : 0) | (h1 >= 0 ? 0xFFFF0000u : 0));
                }
                // slots that are not there: the tile's first, hidden, and zeros among the values
                auto put_v = [&](int j, bool on, const uint32_t *v) {
#pragma unroll
                    for (int e = 0; e < W::VW; ++e) w.vf[j][e] = on ? v[e] : 0;
                };
                if (draft) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int jj = 16 * b + ln < left ? 16 * b + ln : 0;
                        const size_t at = (size_t)(q.first + j0 + jj) * d.ld_kv + (size_t)h * d.hs_kv + 8 * g;
#pragma unroll
                        for (int k = 0; k < W::C; ++k) w.kf[b][k] = draft8(d.k, at + 32 * k, d.kv_f32, BF);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int jj = (j < 4 ? 0 : 12) + 4 * g + j;
                        const size_t at = (size_t)(q.first + j0 + (jj < left ? jj : 0)) * d.ld_kv + (size_t)h * d.hs_kv + DV * ln;
                        uint32_t v[W::VW];
                        if constexpr (W::VW == 2) {
                            if (d.kv_f32) {
                                const float4v f = *(const float4v *)((const float *)d.v + at);
                                v[0] = pack2<BF>(f[0], f[1]), v[1] = pack2<BF>(f[2], f[3]);
                            } else {
                                *(uint2v *)v = *(const uint2v *)((const uint16_t *)d.v + at);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < W::VW; e += 4) *(uint4v *)(v + e) = draft8(d.v, at + 2 * e, d.kv_f32, BF);
                        }
                        put_v(j, jj < left, v);
                    }
                } else {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int64_t hb = b ? h1 : h0;
                        const uint32_t o = 16 * b + ln < left ? ko : 8 * g;
#pragma unroll
                        for (int k = 0; k < W::C; ++k) w.kf[b][k] = *(const uint4v *)(kp + max(hb, (int64_t)0) + o + 32 * k);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int jj = (j < 4 ? 0 : 12) + 4 * g + j;
                        const int64_t hb = j < 4 ? h0 : h1;
                        uint32_t v[W::VW];
                        w.load_v1(vp + max(hb, (int64_t)0) + (jj < left ? vo + (j & 3) * ss : DV * ln), v);
                        put_v(j, jj < left && hb >= 0, v);
                    }
                }
                uint32_t odd = 0;
                if (draft)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        bool has = false;
#pragma unroll
                        for (int e = 0; e < W::VW; ++e) has |= take_odd<BF>(w.vf[j][e]);
                        const uint64_t by = __ballot(has);
                        for (int k = 0; k < 4; ++k)
                            if (by >> (16 * k) & 0xFFFF) odd |= 1u << ((j < 4 ? 0 : 12) + 4 * k + j);
                    }
                float x[NT][8];
                w.qk(x);
                w.hide(x, see);
                w.softmax(x);
                w.pv(x);
                if (odd) w.add_odd(odd, see, d, q.first + j0, h, lane);
            }
        }

        const bool whole = t0 == 0 && t1 == q.tiles;
        const int here = min(rows_wg, rows - rt * rows_wg);
        const int p0 = sa / per, np = (sb - 1) / per - p0 + 1;   // the segment's workgroups p0 .. p0 + np - 1
        const size_t rec = (size_t)rows_wg * (D + 2);
        if (J.join && t0 == 0 && threadIdx.x == 0) J.where[((size_t)s * c.n_kv + h) * J.rt + rt] = make_int2(p0, np);
        float *mine = whole ? nullptr : J.part + (2 * (size_t)wg + (sa < wg * per ? 0 : 1)) * rec;
        auto leave = [&](int r, int e, const Part &p) {   // row r of the row tile
            if (whole) {
                store_row<D, BF, QF>(J, q.first, h, rt * rows_wg + r, e, p);
            } else if (SHARE || J.join) {
                *(float4v *)(mine + (size_t)r * D + e) = p.v;
                if (e == 0) *(float2 *)(mine + (size_t)rows_wg * D + 2 * r) = make_float2(p.m, p.l);
            } else {
                store2_agent(mine + (size_t)r * D + e, p.v[0], p.v[1]);
                store2_agent(mine + (size_t)r * D + e + 2, p.v[2], p.v[3]);
                if (e == 0) store2_agent(mine + (size_t)rows_wg * D + 2 * r, p.m, p.l);
            }
        };
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            w.l[a] += __shfl_xor(w.l[a], 16);
            w.l[a] += __shfl_xor(w.l[a], 32);
        }
        // f(element, four of the row's sums) over what the lane has of row tile a
        auto pieces = [&](int a, auto f) {
            if constexpr (SHARE) {
#pragma unroll
                for (int t = 0; t < DV; ++t) f(16 * t + 4 * g, w.o[a][t]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < DV; t += 4) f(DV * (4 * g + i) + t, float4v{w.o[a][t][i], w.o[a][t + 1][i], w.o[a][t + 2][i], w.o[a][t + 3][i]});
            }
        };
        if (SW == 1) {   // the wave's sums are the workgroup's
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                const int r = rwi * R16 + 16 * a + ln;
                if (r < here) pieces(a, [&](int e, float4v v) { leave(r, e, Part{v, w.m[a], w.l[a]}); });
            }
        } else {   // the workgroup's waves of the same rows meet in LDS
            constexpr int LD = D + 4;
            float *po = sh + (size_t)wave * R16 * LD, *pm = sh + (size_t)kWaves * R16 * LD, *pl = pm + kWaves * R16;
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                const int r = 16 * a + ln;
                if (row0 + r >= rows) continue;
                if (g == 0) {
                    pm[wave * R16 + r] = w.m[a];
                    pl[wave * R16 + r] = w.l[a];
                }
                pieces(a, [&](int e, float4v v) { *(float4v *)(po + r * LD + e) = v; });
            }
            __syncthreads();
            for (int x4 = threadIdx.x; x4 < here * (D / 4); x4 += 64 * kWaves) {
                const int r = x4 / (D / 4), e = x4 % (D / 4) * 4, rg = r / R16, rr = r % R16;
                float m = -INFINITY;
                for (int k = 0; k < SW; ++k) m = fmaxf(m, pm[(k * RW + rg) * R16 + rr]);
                const float mb = m == -INFINITY ? 0.0f : m;
                Part p{float4v{0, 0, 0, 0}, m, 0.0f};
                for (int k = 0; k < SW; ++k) {
                    const int wv = k * RW + rg;
                    const float f = __builtin_amdgcn_exp2f(pm[wv * R16 + rr] - mb);
                    p.l += f * pl[wv * R16 + rr];
                    p.v += f * *(const float4v *)(sh + ((size_t)wv * R16 + rr) * LD + e);
                }
                leave(r, e, p);
            }
        }
        if (!SHARE && !whole && !J.join) {
            // the segment's last workgroup adds the records in the workgroups' order
            unsigned *ctr = J.count + ((size_t)s * c.n_kv + h) * J.rt + rt;
            __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the wave's record stores complete before the arrival
            __syncthreads();
            if (threadIdx.x == 0) {
                const unsigned old = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last = old + 1 == (unsigned)np;
                if (last) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (last) {
                // ranges of records side by side where the threads are more than the row pieces
                Part *ps4 = (Part *)sh4;
                const int items = here * (D / 4), subs = max(1, min(8, 64 * kWaves / items)), each = (np + subs - 1) / subs;
                for (int x0 = 0; x0 < items; x0 += 64 * kWaves) {
                    const int xi = x0 + (int)threadIdx.x, sub = subs > 1 ? xi / items : 0, x4 = xi - sub * items, r = x4 / (D / 4), e = x4 % (D / 4) * 4;
                    const bool on = sub < subs && x4 < items;
                    Part p{float4v{0, 0, 0, 0}, -INFINITY, 0.0f};
                    if (on) p = join_records<D, true>(J.part, rec, rows_wg, p0, min(np, sub * each), min(np, (sub + 1) * each), r, e);
                    if (subs > 1) {
                        if (on && sub) ps4[xi] = p;
                        __syncthreads();
                        if (on && !sub)
                            for (int k = 1; k < subs; ++k) add_part(p, ps4[k * items + x4]);
                    }
                    if (on && !sub) store_row<D, BF, QF>(J, q.first, h, rt * rows_wg + r, e, p);
                }
            }
        }
        __syncthreads();   // sh and last are free again
    }
}

// Rows of a wave and row waves of a workgroup. Few rows: 16 or 32 in every wave (16 with queries of several parts or rows of
// 256 elements, whose operands fill the registers), at most two row waves, the other waves take slots in turn; up to two
// such row tiles, each reading K and V for itself. More rows: 8 waves (4 of twice the registers for rows of 256) share K and V
// through LDS, each with 16 or 32 of the rows. us, few-rows form then sharing (2 sequences x 32767 slots x 8 heads, 65535 for
// head_dim 64, 16383 for 256; bf16, in brackets f32 queries):
//   head_dim   64: 64 rows 78 (101) and 104 (116), 96 rows 105 (146) and 107 (123)
//   head_dim  128: 64 rows 77 (88) and 78 (91), 96 rows 98 (125) and 79 (93), 256 rows 174 (310) and 117 (171)
//   head_dim  256: 64 rows (86.5) and (83.5), 96 rows (121) and (109)
// hence above 64 rows, above 32 of 256 elements. 32 rows a wave against 16 where both fit: 105 to 130 us at 512 rows, 4
// sequences x 16383 slots.
// Records of a segment of more than kJoinBytes are joined by a launch of their own, else by the segment's last
// workgroup: 118.8 to 126.5 us at 32 rows and 32 records (530 KB), 22.5 to 32.6 at 8190 slots; the other way 14.8 to
// 16.3 at 4 rows and 5 records (10 KB).
constexpr size_t kJoinBytes = 96 << 10;
// The workspace starts with as many counters whatever the shape, so that calls of other shapes, which write
// places and records behind them, leave them zero; more segments are joined by a launch.
constexpr size_t kCounters = 4096;
struct AttnPlan { int nt, rw, rows_wg, rt, share; size_t segs, rec_bytes, head_bytes; };
static AttnPlan attn_plan(const KvDev &c, const DraftDev &d, int D) {
    AttnPlan p;
    const int rows = d.max_tokens * d.G;
    if (rows > (D == 256 ? 32 : 64)) {
        p.share = D == 256 ? 4 : 8;
        p.nt = rows > 16 * p.share && !d.q_f32 && D < 256 ? 2 : 1;
        p.rw = p.share;
    } else {
        p.share = 0;
        p.nt = rows <= 16 || d.q_f32 || D == 256 ? 1 : 2;
        p.rw = rows > 16 * p.nt ? 2 : 1;
    }
    p.rows_wg = 16 * p.nt * p.rw;
    p.rt = (rows + p.rows_wg - 1) / p.rows_wg;
    p.segs = (size_t)c.n_seq * c.n_kv * p.rt;
    p.head_bytes = 4 * kCounters + (8 * p.segs + 255) / 256 * 256;   // counters, then places
    p.rec_bytes = 4 * (size_t)p.rows_wg * (D + 2);
    return p;
}

size_t attn_workspace(const KvDev &c, const DraftDev &d, int D) {
    const AttnPlan p = attn_plan(c, d, D);
    return p.head_bytes + 2 * (size_t)num_cus() * p.rec_bytes;
}

template <int D, bool BF, bool QF, int NT, int SHARE>
static int attn_run(const AttnJob &J, int rows_wg, hipStream_t st) {
    constexpr int waves = attn_waves(D, SHARE);
    constexpr int lds = SHARE ? kStages * 2 * 32 * stage_tiles(D) * 2 * D : waves * 16 * NT * (D + 4 + 2) * 4;
    static OncePerDevice once;
    if (int rc = allow_lds(once, (const void *)k_attn<D, BF, QF, NT, SHARE>, lds, "p8x_attn_tree LDS")) return rc;
    k_attn<D, BF, QF, NT, SHARE><<<J.nwg, 64 * waves, lds, st>>>(J);
    const dim3 heads(0, J.rt, J.c.n_seq * J.c.n_kv);
    // eight threads to four elements where a segment has many records: 22.7 to 26.0 us at 32 records of 32 rows, but 114 to 104 at 8
    // of 256
    if (J.join && J.nwg > 12 * (int)(heads.y * heads.z)) k_attn_join<D, BF, QF, 8><<<dim3((rows_wg * (D / 4) + 31) / 32, heads.y, heads.z), 256, 0, st>>>(J, rows_wg);
    else if (J.join) k_attn_join<D, BF, QF, 1><<<dim3((rows_wg * (D / 4) + 255) / 256, heads.y, heads.z), 256, 0, st>>>(J, rows_wg);
    return hip_check(hipGetLastError(), "p8x_attn_tree launch");
}

template <int D, bool BF, bool QF>
static int attn_form(const AttnJob &J, const AttnPlan &p, hipStream_t st) {
    constexpr int SHARED = D == 256 ? 4 : 8;
    if constexpr (D < 256 && !QF) {
        if (p.nt == 2) return p.share ? attn_run<D, BF, QF, 2, SHARED>(J, p.rows_wg, st) : attn_run<D, BF, QF, 2, 0>(J, p.rows_wg, st);
    }
    return p.share ? attn_run<D, BF, QF, 1, SHARED>(J, p.rows_wg, st) : attn_run<D, BF, QF, 1, 0>(J, p.rows_wg, st);
}

template <int D>
static int attn_types(const AttnJob &J, const AttnPlan &p, hipStream_t st) {
    if (J.d.q_f32) return J.c.bf16 ? attn_form<D, true, true>(J, p, st) : attn_form<D, false, true>(J, p, st);
    return J.c.bf16 ? attn_form<D, true, false>(J, p, st) : attn_form<D, false, false>(J, p, st);
}

int launch_attn_tree(const KvDev &c, const DraftDev &d, int D, void *out, size_t ldo, size_t hso, float *lse, void *ws, size_t ws_bytes,
                     hipStream_t st) {
    const AttnPlan p = attn_plan(c, d, D);
    const size_t most = p.segs * ((size_t)(c.max_len + 31) / 32 + 2);   // tiles
    if (most >= (1u << 29)) return set_error(P8X_ERR_UNSUPPORTED, "p8x_attn_tree: %zu tiles of 32 slots (fewer than 2^29)", most);
    if (c.slot_stride >= (1u << 26)) return set_error(P8X_ERR_UNSUPPORTED, "p8x_attn_tree: slot_stride %zu (below 2^26)", c.slot_stride);
    AttnJob J{c, d, out, ldo, hso, lse, (unsigned *)ws, (float *)((char *)ws + p.head_bytes), (int2 *)((char *)ws + 4 * kCounters), p.rw, p.rt, attn_waves(D, p.share) / p.rw, 1, 0, 0};
    const size_t room = ws_bytes > p.head_bytes ? (ws_bytes - p.head_bytes) / (2 * p.rec_bytes) : 0;   // workgroups with records
    int nwg = (int)std::min<size_t>(num_cus(), room);
    if (nwg < 16 || p.segs / p.rt > 65535 || p.rt > 65535) {   // whole segments then
        nwg = (int)std::min<size_t>(num_cus(), p.segs);
        J.split = 0, J.least = 1;
    }
    if (nwg >= 8) nwg = nwg / 8 * 8;
    J.nwg = nwg;
    // records of a segment, about, that one workgroup would join
    const size_t rows = std::min((size_t)d.max_tokens * d.G, (size_t)p.rows_wg), each = J.split ? nwg / p.segs * rows * (D + 2) * 4 : 0;
    J.join = J.split && (p.share || each > kJoinBytes || p.segs > kCounters);
    return D == 64 ? attn_types<64>(J, p, st) : D == 128 ? attn_types<128>(J, p, st) : attn_types<256>(J, p, st);
}

}  // namespace p8x
