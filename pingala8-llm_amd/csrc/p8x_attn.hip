// p8x_attn.hip -- attention of drafted tokens over the cache and each other (p8x_attn_tree), and the attention weight
// that accepted tokens gave (p8x_kv_score).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "p8x_kv.h"

namespace p8x {

__device__ __forceinline__ uint64_t token_mask(const DraftDev &d, int tok, int i) {
    return d.mask ? d.mask[tok] : i == 63 ? ~0ull : (2ull << i) - 1;
}

// ---- attention ----------------------------------------------------------------------------------------------
// Rows: the (token, head of the group) pairs of a sequence and key/value head, token-major; they share K and V. A wave
// multiplies tiles of 32 slots with its 16 NT rows on v_mfma_f32_16x16x32, transposed throughout so that nothing passes
// through LDS between the two products:
//   S^T [slot][row] = K Q^T: A = K (lane m = slot, 8 elements of the row at 8 (lane / 16)), B = Q, kept in registers;
//   its result has, in lane (row, g), slots 4 g + i of each 16: the weights p in that place are, as they are, the B operand
//   of O^T [element][row] = V^T P^T when the operand's k index 8 g + j stands for slot 4 g + j (j < 4) or 16 + 4 g + j - 4.
//   A = V^T: lane (m, g) loads D / 16 elements of its group's 8 slots and transposes them in registers (one v_perm a
//   dword); output tile t's row m then is element (D / 16) m + t.
// Softmax: the running maximum m of a row only moves when a score exceeds it by 2^8 in the weight, seen by each lane for
// itself, so that the usual tile needs no exchange between lanes and no rescaling; sums l stay in their lanes until the
// end. Weights stand relative to m, times 2^kBias for fp16 (subnormals).
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));

template <bool BF>
__device__ __forceinline__ float4v mfma(uint4v a, uint4v b, float4v c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (BF) return (uint32_t)to_bf16(x) | (uint32_t)to_bf16(y) << 16;
    else return (uint32_t)to_f16(x) | (uint32_t)to_f16(y) << 16;
}
template <bool BF>
__device__ __forceinline__ float part_lo(uint32_t w) { return BF ? __builtin_bit_cast(float, w << 16) : from_f16((uint16_t)w); }
template <bool BF>
__device__ __forceinline__ float part_hi(uint32_t w) { return BF ? __builtin_bit_cast(float, w & 0xFFFF0000u) : from_f16((uint16_t)(w >> 16)); }

// 8 f32 as N operands of 16 bits that sum to them: N x 11 (fp16) or N x 8 (bf16) bits
template <bool BF, int N>
__device__ __forceinline__ void split8(const float *f, uint4v *o) {
    float r[8];
    for (int e = 0; e < 8; ++e) r[e] = f[e];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = pack2<BF>(r[2 * e], r[2 * e + 1]);
            o[n][e] = w;
            if (n + 1 < N) {
                r[2 * e] -= part_lo<BF>(w);
                r[2 * e + 1] -= part_hi<BF>(w);
            }
        }
}

// waves of a workgroup, one of which a compute unit holds: 256 registers a lane, or 512 for rows of 256 elements
__host__ __device__ constexpr int attn_waves(int D) { return D == 256 ? 4 : 8; }
// A lane's pieces of an f32 query row, 8 elements at 32 k, for splitting: fp16 parts need the row scaled to 2^13 (the lanes
// 16 apart hold the rest of the row). Returns the factor of a product, f with that power taken back out.
template <int C, bool BF>
__device__ __forceinline__ float load_split(const float *q, bool on, float f, float (&x)[C][8]) {
    float mx = 0.0f;
#pragma unroll
    for (int k = 0; k < C; ++k) {
        const float4v lo = on ? *(const float4v *)(q + 32 * k) : float4v{0, 0, 0, 0}, hi = on ? *(const float4v *)(q + 32 * k + 4) : float4v{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[k][e] = lo[e];
            x[k][e + 4] = hi[e];
            mx = fmaxf(mx, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
        }
    }
    if constexpr (!BF) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const int ex = mx > 0.0f && mx < INFINITY ? 13 - (int)((__builtin_bit_cast(uint32_t, mx) >> 23) - 127) : 0;
        const int e1 = min(ex, 100);   // in two steps: 2^ex may be beyond f32
        const float s1 = ldexpf(1.0f, e1), s2 = ldexpf(1.0f, ex - e1);
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[k][e] = x[k][e] * s1 * s2;
        f = ldexpf(f, -ex);
    }
    return f;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLazy = 8.0f;   // log2 of how far a weight may exceed 1 before its row's maximum moves

struct AttnJob {
    KvDev c;
    DraftDev d;
    void *out; size_t ldo, hso;
    float *lse;
    unsigned *count;   // arrivals of a segment's workgroups, 0 between calls
    float *part;       // two records a workgroup: rows x D sums, then rows m, rows l
    int rw, rt, least; // row waves of a workgroup; row tiles of a sequence at most; units a workgroup takes at least
    int split;         // unit: a tile; 0: a whole segment (no records)
    int join;          // records are joined by a launch of their own
    int nwg;
};

// the units (32-slot tiles) of sequence s: tokens, slots, row tiles, tiles
struct SeqUnits { int nt, n, first, rts, tiles, per_seg; };
__device__ __forceinline__ SeqUnits seq_units(const AttnJob &J, int s, int rows_wg) {
    SeqUnits u;
    u.nt = seq_tokens(J.d, s, u.first);
    u.n = seq_len(J.c, s);
    u.rts = (u.nt * J.d.G + rows_wg - 1) / rows_wg;
    u.tiles = u.nt ? (u.n + 31) / 32 + (u.nt + 31) / 32 : 0;
    u.per_seg = J.split ? u.tiles : u.nt ? 1 : 0;
    return u;
}

template <int D, bool BF, bool QF, int NT>
struct Wave {
    static constexpr int C = D / 32, DV = D / 16, VW = DV / 2;       // K operands a row; elements and dwords of V a lane and slot
    static constexpr int QP = QF ? (BF ? 3 : 2) : 1, PP = QF && BF ? 3 : 2;   // 16-bit parts of a query and of a weight
    static constexpr float kBias = BF ? 0.0f : 7.0f;
    uint4v q[NT][QP][C];
    float4v o[NT][DV];
    float m[NT], l[NT], c2[NT];
    uint4v kf[2][C];
    uint32_t vf[8][VW];

    // the lane's rows' queries; f32 ones scaled to 2^13 (fp16 parts), the power put into c2
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
                c2[a] = load_split<C, BF>((const float *)d.q + at, on, d.scale < 0 ? -sc : sc, f);
                if (d.scale < 0) {
                    c2[a] = -c2[a];
#pragma unroll
                    for (int k = 0; k < C; ++k)
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[k][e] = -f[k][e];
                }
#pragma unroll
                for (int k = 0; k < C; ++k) {
                    uint4v p[QP];
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

    __device__ __forceinline__ void qk(float (&x)[NT][8]) {
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float4v s = {0, 0, 0, 0};
#pragma unroll
                for (int n = QP - 1; n >= 0; --n)   // small parts first
#pragma unroll
                    for (int c = 0; c < C; ++c) s = mfma<BF>(kf[t][c], q[a][n][c], s);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[a][4 * t + i] = s[i];
            }
    }

    // scores to weights: x[a][j] of slot j of the lane's eight (-inf: hidden)
    __device__ __forceinline__ void softmax(float (&x)[NT][8]) {
        float mx[NT];
        bool move = false;
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            mx[a] = fmaxf(fmaxf(fmaxf(x[a][0], x[a][1]), fmaxf(x[a][2], x[a][3])), fmaxf(fmaxf(x[a][4], x[a][5]), fmaxf(x[a][6], x[a][7]))) * c2[a];
            move |= mx[a] > m[a] + kLazy;
        }
        if (__any(move)) {
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                float v = fmaxf(mx[a], __shfl_xor(mx[a], 16));
                v = fmaxf(v, __shfl_xor(v, 32));
                v = fmaxf(v, m[a]);
                const float al = v == -INFINITY || m[a] == v ? 1.0f : exp2f(m[a] - v);
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

    __device__ __forceinline__ void pv(const float (&x)[NT][8]) {
        uint4v p[NT][PP];
#pragma unroll
        for (int a = 0; a < NT; ++a) split8<BF, PP>(x[a], p[a]);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
            uint4v e0, e1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                e0[j] = __builtin_amdgcn_perm(vf[2 * j + 1][w], vf[2 * j][w], 0x05040100u);
                e1[j] = __builtin_amdgcn_perm(vf[2 * j + 1][w], vf[2 * j][w], 0x07060302u);
            }
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
                for (int n = PP - 1; n >= 0; --n) {
                    o[a][2 * w] = mfma<BF>(e0, p[a][n], o[a][2 * w]);
                    o[a][2 * w + 1] = mfma<BF>(e1, p[a][n], o[a][2 * w + 1]);
                }
        }
    }
};

// 8 elements of a draft row as the cache holds them
__device__ __forceinline__ uint4v draft8(const void *p, size_t at, int f32, int bf16) {
    if (!f32) return *(const uint4v *)((const uint16_t *)p + at);
    const float4v lo = *(const float4v *)((const float *)p + at), hi = *(const float4v *)((const float *)p + at + 4);
    uint4v o;
    for (int e = 0; e < 2; ++e) {
        o[e] = to16(lo[2 * e], bf16) | (uint32_t)to16(lo[2 * e + 1], bf16) << 16;
        o[e + 2] = to16(hi[2 * e], bf16) | (uint32_t)to16(hi[2 * e + 1], bf16) << 16;
    }
    return o;
}

__device__ __forceinline__ float2 load2_agent(const float *p) {
    const uint64_t v = __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__builtin_bit_cast(float, (uint32_t)v), __builtin_bit_cast(float, (uint32_t)(v >> 32)));
}
__device__ __forceinline__ void store2_agent(float *p, float a, float b) {
    __hip_atomic_store((uint64_t *)p, (uint64_t)__builtin_bit_cast(uint32_t, b) << 32 | __builtin_bit_cast(uint32_t, a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A record: [row][D] sums, then [row] (m, l). Elements e .. e + 3 of row r over the np records of a segment, in order, eight
// loads in flight at a time; AGENT: written in this launch by other workgroups.
template <int D, bool AGENT>
__device__ __forceinline__ void join_records(const float *part, size_t rec, int rows_wg, int p0, int np, int r, int e, float4v &v, float &m, float &l) {
    m = -INFINITY, l = 0.0f, v = float4v{0, 0, 0, 0};
    for (int b = 0; b < np; b += 8) {
        float2 ml[8];
        float4v x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int p = min(b + k, np - 1);
            const float *q = part + (2 * (size_t)(p0 + p) + (p == 0 ? 1 : 0)) * rec;
            if constexpr (AGENT) {
                ml[k] = load2_agent(q + (size_t)rows_wg * D + 2 * r);
                const float2 a = load2_agent(q + (size_t)r * D + e), c = load2_agent(q + (size_t)r * D + e + 2);
                x[k] = float4v{a.x, a.y, c.x, c.y};
            } else {
                ml[k] = *(const float2 *)(q + (size_t)rows_wg * D + 2 * r);
                x[k] = *(const float4v *)(q + (size_t)r * D + e);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (b + k >= np) break;
            const float mn = fmaxf(m, ml[k].x), mb = mn == -INFINITY ? 0.0f : mn;
            const float f0 = exp2f(m - mb), f1 = exp2f(ml[k].x - mb);
            m = mn;
            l = l * f0 + ml[k].y * f1;
            v = v * f0 + x[k] * f1;
        }
    }
}

template <int D, bool BF, bool QF>
__device__ __forceinline__ void store_row(const AttnJob &J, int first, int h, int row, int e, float4v v, float m, float l) {
    constexpr float bias = BF ? 0.0f : 7.0f;
    v *= l == 0.0f ? 0.0f : 1.0f / l;
    const int G = J.d.G, i = row / G, head = h * G + row - i * G;
    const size_t at = (size_t)(first + i) * J.ldo + (size_t)head * J.hso + e;
    if constexpr (QF) *(float4v *)((float *)J.out + at) = v;
    else {
        const uint2v p = {pack2<BF>(v[0], v[1]), pack2<BF>(v[2], v[3])};
        *(uint2v *)((uint16_t *)J.out + at) = p;
    }
    if (e == 0 && J.lse) J.lse[(size_t)(first + i) * J.c.n_kv * G + head] = l == 0.0f ? -INFINITY : (m - bias + __log2f(l)) * kLn2;
}

// The records of split segments in a launch of their own: a thread four elements of a row.
template <int D, bool BF, bool QF>
__global__ __launch_bounds__(256) void k_attn_join(AttnJob J, int rows_wg) {
    const int lane = threadIdx.x & 63, s = blockIdx.z / J.c.n_kv, h = blockIdx.z % J.c.n_kv, rt = blockIdx.y;
    const int x4 = blockIdx.x * 256 + threadIdx.x, r = x4 / (D / 4), e = x4 % (D / 4) * 4;
    int total = 0, base = 0;
    for (int s0 = 0; s0 < J.c.n_seq; s0 += 64) {
        int v = 0;
        if (s0 + lane < J.c.n_seq) {
            const SeqUnits u = seq_units(J, s0 + lane, rows_wg);
            v = J.c.n_kv * u.rts * u.per_seg;
        }
        int b = s0 + lane < s ? v : 0;
        if (J.c.n_seq > 1)
            for (int o = 32; o; o >>= 1) {
                v += __shfl_xor(v, o);
                b += __shfl_xor(b, o);
            }
        else v = __builtin_amdgcn_readfirstlane(v);
        total += v;
        base += J.c.n_seq > 1 ? b : 0;
    }
    const int per = max(J.least, (total + J.nwg - 1) / J.nwg);
    const SeqUnits q = seq_units(J, s, rows_wg);
    if (rt >= q.rts || rt * rows_wg + r >= q.nt * J.d.G || r >= rows_wg) return;
    const int sa = base + (h * q.rts + rt) * q.tiles, sb = sa + q.tiles, p0 = sa / per, np = (sb - 1) / per - p0 + 1;
    if (np < 2) return;
    float4v v;
    float m, l;
    join_records<D, false>(J.part, (size_t)rows_wg * (D + 2), rows_wg, p0, np, r, e, v, m, l);
    store_row<D, BF, QF>(J, q.first, h, rt * rows_wg + r, e, v, m, l);
}

template <int D, bool BF, bool QF, int NT>
__global__ __launch_bounds__(64 * attn_waves(D)) void k_attn(AttnJob J) {
    constexpr int kWaves = attn_waves(D);
    typedef Wave<D, BF, QF, NT> W;
    constexpr int R16 = 16 * NT, DV = W::DV;
    extern __shared__ float sh[];   // [wave][row][D + 4] sums, then [wave][row] m, l
    __shared__ unsigned last;
    const KvDev &c = J.c;
    const DraftDev &d = J.d;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, ln = lane & 15;
    const int RW = J.rw, SW = kWaves / RW, rwi = wave % RW, swi = wave / RW, rows_wg = R16 * RW;
    // consecutive units on one XCD: workgroups go round robin over the eight
    const int nwg = gridDim.x, wg = nwg % 8 ? (int)blockIdx.x : (int)(blockIdx.x % 8) * (nwg / 8) + (int)(blockIdx.x / 8);

    // all units, and the workgroup's share [u0, u1)
    int total = 0;
    for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
        int v = 0;
        if (s0 + lane < c.n_seq) {
            const SeqUnits u = seq_units(J, s0 + lane, rows_wg);
            v = c.n_kv * u.rts * u.per_seg;
        }
        if (c.n_seq > 1)
            for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
        total += __builtin_amdgcn_readfirstlane(v);
    }
    const int per = max(J.least, (total + nwg - 1) / nwg);
    const int u0 = wg * per, u1 = min(total, u0 + per);
    if (u0 >= u1) return;
    // the sequence of unit u0
    int s = 0, base = 0;
    if (c.n_seq > 1)
        for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
            int v = 0;
            if (s0 + lane < c.n_seq) {
                const SeqUnits u = seq_units(J, s0 + lane, rows_wg);
                v = c.n_kv * u.rts * u.per_seg;
            }
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
    const uint32_t ko = (uint32_t)ln * (uint32_t)c.slot_stride + 8 * g, vo = 4 * g * (uint32_t)c.slot_stride + DV * ln;
    for (int u = u0; u < u1;) {
        SeqUnits q = seq_units(J, s, rows_wg);
        q.nt = __builtin_amdgcn_readfirstlane(q.nt), q.n = __builtin_amdgcn_readfirstlane(q.n), q.first = __builtin_amdgcn_readfirstlane(q.first);
        q.rts = __builtin_amdgcn_readfirstlane(q.rts), q.tiles = __builtin_amdgcn_readfirstlane(q.tiles);
        const int ps = J.split ? q.tiles : q.nt ? 1 : 0, units = c.n_kv * q.rts * ps;
        if (u >= base + units) {   // past this sequence (or none of its units)
            base += units;
            ++s;
            continue;
        }
        const int seg = (u - base) / ps, t0 = (u - base) - seg * ps, h = seg / q.rts, rt = seg - h * q.rts;
        const int t1 = J.split ? min(q.tiles, t0 + (u1 - u)) : q.tiles, ctx = (q.n + 31) / 32;
        const int sa = u - t0, sb = sa + ps;   // the segment's units
        u = min(u1, sb);
        const int rows = q.nt * d.G, row0 = rt * rows_wg + rwi * R16;
        w.load_q(d, q.first, h, row0, rows, lane);

        const uint16_t *kp = c.k + (size_t)h * c.head_stride, *vp = c.v + (size_t)h * c.head_stride;
        const int full = min(t1, q.n / 32);   // tiles of 32 slots in use
        float x[NT][8];
        for (int tb = t0 + swi; tb < full; tb += 32 * SW) {
            // offsets of the wave's next 64 halves, a lane each: tile tb + SW (lane / 2), half lane & 1
            int64_t off = -1;
            {
                const int t = tb + SW * (lane >> 1);
                if (t < full) off = slot_offset(c, s, 32 * t + 16 * (lane & 1));
            }
            const int lo = (int)off, hi = (int)(off >> 32), nt = min(32, (full - tb + SW - 1) / SW);
            auto half = [&](int i) { return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, i)); };
            int64_t h0 = half(0), h1 = half(1);
            w.load_k(kp, max(h0, (int64_t)0), max(h1, (int64_t)0), ko);
            w.load_v(vp, max(h0, (int64_t)0), max(h1, (int64_t)0), vo, (uint32_t)c.slot_stride);
            for (int i = 0; i < nt; ++i) {
                const int64_t n0 = half(2 * min(i + 1, nt - 1)), n1 = half(2 * min(i + 1, nt - 1) + 1);
                w.qk(x);
                if (i + 1 < nt) w.load_k(kp, max(n0, (int64_t)0), max(n1, (int64_t)0), ko);
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
                if (i + 1 < nt) w.load_v(vp, max(n0, (int64_t)0), max(n1, (int64_t)0), vo, (uint32_t)c.slot_stride);
                h0 = n0, h1 = n1;
            }
        }
        // the cache's last, partial tile and the drafted tokens: rows that are not there are zeros, scores are masked
        const int t_rest = max(t0, q.n / 32);
        for (int t = t_rest + (swi - (t_rest - t0) % SW + SW) % SW; t < t1; t += SW) {
            const bool draft = t >= ctx;
            uint64_t see[NT];
            if (draft) {
                const int j0 = 32 * (t - ctx), left = q.nt - j0;
#pragma unroll
                for (int a = 0; a < NT; ++a) {
                    const int r = row0 + 16 * a + ln, i = r / d.G;
                    see[a] = r < rows ? token_mask(d, q.first + i, i) >> j0 & (left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1) : 0;
                }
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int k = 0; k < W::C; ++k)
                        w.kf[b][k] = 16 * b + ln < left ? draft8(d.k, (size_t)(q.first + j0 + 16 * b + ln) * d.ld_kv + (size_t)h * d.hs_kv + 32 * k + 8 * g, d.kv_f32, BF)
                                                        : uint4v{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int jj = (j < 4 ? 0 : 12) + 4 * g + j;
                    const size_t at = (size_t)(q.first + j0 + jj) * d.ld_kv + (size_t)h * d.hs_kv + DV * ln;
#pragma unroll
                    for (int e = 0; e < W::VW; ++e) {
                        uint32_t v = 0;
                        if (jj < left) {
                            if (d.kv_f32) {
                                const float *p = (const float *)d.v + at + 2 * e;
                                v = to16(p[0], BF) | (uint32_t)to16(p[1], BF) << 16;
                            } else {
                                v = *(const uint32_t *)((const uint16_t *)d.v + at + 2 * e);
                            }
                        }
                        w.vf[j][e] = v;
                    }
                    }
            } else {
                const int j0 = 32 * t, left = q.n - j0;
                const int64_t h0 = slot_offset(c, s, j0), h1 = left > 16 ? slot_offset(c, s, j0 + 16) : -1;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int k = 0; k < W::C; ++k)
                        w.kf[b][k] = 16 * b + ln < left && (b ? h1 : h0) >= 0 ? *(const uint4v *)(kp + (b ? h1 : h0) + ko + 32 * k) : uint4v{0, 0, 0, 0};
                uint32_t in = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int jj = (j < 4 ? 0 : 12) + 4 * g + j;
                    const int64_t hb = j < 4 ? h0 : h1;
                    const bool on = jj < left && hb >= 0;
#pragma unroll
                    for (int e = 0; e < W::VW; ++e)
                        w.vf[j][e] = on ? *(const uint32_t *)(vp + hb + vo + (j & 3) * (uint32_t)c.slot_stride + 2 * e) : 0;
                    in |= (uint32_t)on << jj;
                }
#pragma unroll
                for (int a = 0; a < NT; ++a) see[a] = in;
            }
            w.qk(x);
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(see[a] >> ((j < 4 ? 0 : 12) + 4 * g + j) & 1)) x[a][j] = -INFINITY;
            w.softmax(x);
            if (draft) {
                // A hidden token's infinite or NaN value must not meet its zero weight in the product: rows with such values
                // are taken out of the operand and added element by element to the rows of o that see them.
                uint32_t odd = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < W::VW; ++e) {
                        constexpr uint32_t ex = BF ? 0x7F80u : 0x7C00u;
                        if ((w.vf[j][e] & ex) == ex || (w.vf[j][e] >> 16 & ex) == ex) odd |= 1u << j;
                    }
                if (__any(odd != 0)) {
                    const int j0 = 32 * (t - ctx);
                    for (int j = 0; j < 8; ++j) {
                        uint32_t gs = 0;   // groups (of 16 lanes) with such a row at j
                        for (int k = 0; k < 4; ++k)
                            if (__ballot(odd >> j & 1) >> (16 * k) & 0xFFFF) gs |= 1u << k;
                        if (gs >> g & 1)
                            for (int e = 0; e < W::VW; ++e) {
                                // (select over constant indices keeps vf in registers)
#pragma unroll
                                for (int jj = 0; jj < 8; ++jj)
                                    if (jj == j) w.vf[jj][e] = 0;
                            }
                        for (int k = 0; k < 4; ++k) {
                            if (!(gs >> k & 1)) continue;
                            const int tok = (j < 4 ? 0 : 12) + 4 * k + j;
#pragma unroll
                            for (int a = 0; a < NT; ++a) {
                                float p = 0;
#pragma unroll
                                for (int jj = 0; jj < 8; ++jj)
                                    if (jj == j) p = x[a][jj];
                                p = __shfl(p, 16 * k + ln);   // the row's weight of that token
                                const bool on = see[a] >> tok & 1;
#pragma unroll
                                for (int e = 0; e < DV; ++e)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        const size_t at = (size_t)(q.first + j0 + tok) * d.ld_kv + (size_t)h * d.hs_kv + DV * (4 * g + i) + e;
                                        const float v = d.kv_f32 ? from16(to16(((const float *)d.v)[at], BF), BF) : from16(((const uint16_t *)d.v)[at], BF);
                                        if (on) w.o[a][e][i] = fmaf(p, v, w.o[a][e][i]);
                                    }
                            }
                        }
                    }
                }
            }
            w.pv(x);
        }

        // the workgroup's waves of the same rows, then the segment's workgroups
        constexpr int LD = D + 4;
        float *po = sh + (size_t)wave * R16 * LD, *pm = sh + (size_t)kWaves * R16 * LD, *pl = pm + kWaves * R16;
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            float l = w.l[a];
            l += __shfl_xor(l, 16);
            l += __shfl_xor(l, 32);
            const int r = 16 * a + ln;
            if (row0 + r < rows) {
                if (g == 0) {
                    pm[wave * R16 + r] = w.m[a];
                    pl[wave * R16 + r] = l;
                }
                // element DV (4 g + i) + t of the row
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < DV; t += 4)
                        *(float4v *)(po + r * LD + DV * (4 * g + i) + t) = float4v{w.o[a][t][i], w.o[a][t + 1][i], w.o[a][t + 2][i], w.o[a][t + 3][i]};
            }
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == q.tiles;
        const int here = min(rows_wg, rows - rt * rows_wg);
        const int p0 = sa / per, np = (sb - 1) / per - p0 + 1;   // the segment's workgroups p0 .. p0 + np - 1
        const size_t rec = (size_t)rows_wg * (D + 2);
        float *mine = whole ? nullptr : J.part + (2 * (size_t)wg + (sa < wg * per ? 0 : 1)) * rec;
        for (int x4 = threadIdx.x; x4 < here * (D / 4); x4 += 64 * kWaves) {
            const int r = x4 / (D / 4), e = x4 % (D / 4) * 4, rg = r / R16, rr = r % R16;
            float m = -INFINITY;
            for (int k = 0; k < SW; ++k) m = fmaxf(m, pm[(k * RW + rg) * R16 + rr]);
            const float mb = m == -INFINITY ? 0.0f : m;
            float l = 0;
            float4v v = {0, 0, 0, 0};
            for (int k = 0; k < SW; ++k) {
                const int wv = k * RW + rg;
                const float f = exp2f(pm[wv * R16 + rr] - mb);
                l += f * pl[wv * R16 + rr];
                v += f * *(const float4v *)(sh + ((size_t)wv * R16 + rr) * LD + e);
            }
            if (whole) {
                store_row<D, BF, QF>(J, q.first, h, rt * rows_wg + r, e, v, m, l);
            } else if (J.join) {
                *(float4v *)(mine + (size_t)r * D + e) = v;
                if (e == 0) *(float2 *)(mine + (size_t)rows_wg * D + 2 * r) = make_float2(m, l);
            } else {
                store2_agent(mine + (size_t)r * D + e, v[0], v[1]);
                store2_agent(mine + (size_t)r * D + e + 2, v[2], v[3]);
                if (e == 0) store2_agent(mine + (size_t)rows_wg * D + 2 * r, m, l);
            }
        }
        if (!whole && !J.join) {
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
            if (last)
                for (int x4 = threadIdx.x; x4 < here * (D / 4); x4 += 64 * kWaves) {
                    const int r = x4 / (D / 4), e = x4 % (D / 4) * 4;
                    float4v v;
                    float m, l;
                    join_records<D, true>(J.part, rec, rows_wg, p0, np, r, e, v, m, l);
                    store_row<D, BF, QF>(J, q.first, h, rt * rows_wg + r, e, v, m, l);
                }
        }
        __syncthreads();   // sh and last are free again
    }
}

// Rows a wave and row waves a workgroup: 16 rows while they hold all, else 32 (16 with queries of several parts or
// wide rows, whose operands fill the registers).
constexpr size_t kJoinBytes = 64 << 10;   // records of more bytes than this are joined by a launch of their own
struct AttnPlan { int nt, rw, rows_wg, rt; size_t segs, rec_bytes, head_bytes; };
static AttnPlan attn_plan(const KvDev &c, const DraftDev &d, int D) {
    const int kWaves = attn_waves(D);
    AttnPlan p;
    const int rows = d.max_tokens * d.G;
    p.nt = rows <= 16 || d.q_f32 || D == 256 ? 1 : 2;
    p.rw = 1;
    while (p.rw < kWaves && p.rw * 16 * p.nt < rows) p.rw *= 2;
    p.rows_wg = 16 * p.nt * p.rw;
    p.rt = (rows + p.rows_wg - 1) / p.rows_wg;
    p.segs = (size_t)c.n_seq * c.n_kv * p.rt;
    p.head_bytes = (4 * p.segs + 255) / 256 * 256;
    p.rec_bytes = 4 * (size_t)p.rows_wg * (D + 2);
    return p;
}

size_t attn_workspace(const KvDev &c, const DraftDev &d, int D) {
    const AttnPlan p = attn_plan(c, d, D);
    return p.head_bytes + 2 * (size_t)num_cus() * p.rec_bytes;
}

template <int D, bool BF, bool QF, int NT>
static int attn_run(const AttnJob &J, int rows_wg, hipStream_t st) {
    constexpr int kWaves = attn_waves(D), lds = kWaves * 16 * NT * (D + 4 + 2) * 4;
    static const hipError_t e = hipFuncSetAttribute((const void *)k_attn<D, BF, QF, NT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return hip_check(e, "p8x_attn_tree LDS");
    k_attn<D, BF, QF, NT><<<J.nwg, 64 * kWaves, lds, st>>>(J);
    if (J.join) k_attn_join<D, BF, QF><<<dim3((rows_wg * (D / 4) + 255) / 256, J.rt, J.c.n_seq * J.c.n_kv), 256, 0, st>>>(J, rows_wg);
    return hip_check(hipGetLastError(), "p8x_attn_tree launch");
}

template <int D>
static int attn_types(const AttnJob &J, const AttnPlan &p, hipStream_t st) {
    const bool bf = J.c.bf16;
    if (J.d.q_f32) return bf ? attn_run<D, true, true, 1>(J, p.rows_wg, st) : attn_run<D, false, true, 1>(J, p.rows_wg, st);
    if constexpr (D < 256)
        if (p.nt == 2) return bf ? attn_run<D, true, false, 2>(J, p.rows_wg, st) : attn_run<D, false, false, 2>(J, p.rows_wg, st);
    return bf ? attn_run<D, true, false, 1>(J, p.rows_wg, st) : attn_run<D, false, false, 1>(J, p.rows_wg, st);
}

int launch_attn_tree(const KvDev &c, const DraftDev &d, int D, void *out, size_t ldo, size_t hso, float *lse, void *ws, size_t ws_bytes,
                     hipStream_t st) {
    const AttnPlan p = attn_plan(c, d, D);
    const size_t most = p.segs * ((size_t)(c.max_len + 31) / 32 + 2);   // units
    if (most >= (1u << 30)) return set_error(P8X_ERR_UNSUPPORTED, "p8x_attn_tree: %zu tiles of 32 slots (fewer than 2^30)", most);
    if (c.slot_stride >= (1u << 26)) return set_error(P8X_ERR_UNSUPPORTED, "p8x_attn_tree: slot_stride %zu (below 2^26)", c.slot_stride);
    AttnJob J{c, d, out, ldo, hso, lse, (unsigned *)ws, (float *)((char *)ws + p.head_bytes), p.rw, p.rt, attn_waves(D) / p.rw, 1, 0, 0};
    const size_t room = ws_bytes > p.head_bytes ? (ws_bytes - p.head_bytes) / (2 * p.rec_bytes) : 0;   // workgroups with records
    int nwg = (int)std::min<size_t>(num_cus(), room);
    if (nwg < 16) {   // whole segments then
        nwg = (int)std::min<size_t>(num_cus(), p.segs);
        J.split = 0, J.least = 1;
    }
    if (nwg >= 8) nwg = nwg / 8 * 8;
    J.nwg = nwg;
    // records of a segment, about, that one workgroup would join
    const size_t each = J.split ? nwg / p.segs * p.rec_bytes : 0;
    J.join = each > kJoinBytes && p.segs / p.rt <= 65535;
    return D == 64 ? attn_types<64>(J, p, st) : D == 128 ? attn_types<128>(J, p, st) : attn_types<256>(J, p, st);
}

// ---- scores -----------------------------------------------------------------------------------------------
// sum over the accepted tokens' rows of exp(scale q k - lse) per slot. S [row][slot] = Q K^T with K as the B operand (lane
// n = slot) straight from memory, each slot's keys read by one wave once, and Q as A from LDS, where the workgroup
// leaves its rows in operand order; a lane's four rows of every tile are added in place, the four lane groups at the end.
constexpr int kScoreWaves = 4;
// rows that LDS holds at a time; more of them take the slots again
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

        uint4v kf[2][C];
        // the tile's weights, summed over the rows: lane l < 32 has slot l's. hide: bit i of byte t set where row 4 g + i of
        // the row tile does not see the lane's slot of half t
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

        for (int tb = t0 + wave; tb < min(t1, ctx); tb += 32 * kScoreWaves) {
            // offsets of the wave's next 64 halves, a lane each
            int64_t off = -1;
            {
                const int t = tb + kScoreWaves * (lane >> 1), slot = 32 * t + 16 * (lane & 1);
                if (t < min(t1, ctx) && slot < n) off = slot_offset(c, s, slot);
            }
            const int lo = (int)off, hi = (int)(off >> 32), many = min(32, (min(t1, ctx) - tb + kScoreWaves - 1) / kScoreWaves);
            auto half = [&](int i) { return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, i)); };
            for (int i = 0; i < many; ++i) {
                const int slot = 32 * (tb + kScoreWaves * i);
                const int64_t h0 = half(2 * i), h1 = half(2 * i + 1);
                const bool on0 = h0 >= 0 && slot + ln < n, on1 = h1 >= 0 && slot + 16 + ln < n;
                const float before = lane < 32 && slot + lane < n && !rb ? J.score[base + slot + lane] : 0.0f;
#pragma unroll
                for (int k = 0; k < C; ++k) {
                    kf[0][k] = on0 ? *(const uint4v *)(kp + h0 + ko + 32 * k) : uint4v{0, 0, 0, 0};
                    kf[1][k] = on1 ? *(const uint4v *)(kp + h1 + ko + 32 * k) : uint4v{0, 0, 0, 0};
                }
                float w = rt > 0 ? sum_rows(false, 0, 0) : 0.0f;
                if ((lane < 16 ? h0 : h1) < 0) w = 0.0f;
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
    const int nb = (int)std::max<int64_t>(1, std::min<int64_t>((tiles + kScoreWaves - 1) / kScoreWaves, (4 * num_cus() + heads - 1) / heads));
    const dim3 grid(nb, c.n_kv, c.n_seq);
    if (D == 64) score_types<64>(J, grid, st);
    else if (D == 128) score_types<128>(J, grid, st);
    else score_types<256>(J, grid, st);
    return hip_check(hipGetLastError(), "p8x_kv_score launch");
}

}  // namespace p8x
