// attn_bwd.h -- the backward pass of softmax attention for gfx950 (fp16 MFMA, fp32 sums).
//
// With row statistics L (of the forward pass) and d_i = sum dO'_i o'_i:
//   P_ij = exp(c q_i.k_j - L_i),  dP_ij = dO_i.v_j,  dS_ij = P_ij (dP_ij - d_i)
//   dV_j = sum_i P_ij dO_i,  dK_j = c sum_i dS_ij q_i,  dQ_i = c sum_j dS_ij k_j
// and, with a gate, dO = sigma(g) dO', dg = dO' o' (1 - sigma(g)); the gate cancels in d.
//
// Three launches: the rows' statistics (attn_bwd_rows_kernel), dK and dV by key tile together with dQ by query
// tile (attn_bwd_kernel), and, where a key tile's queries were split over workgroups, the sum of
// their parts (attn_bwd_join_kernel).  S and dP are made twice, once for each kind of tile: 7 products instead of 5, and no
// T x S memory, no atomics (each sum has one order) and no fp32 dQ to be read and written for
// every key tile.
//
// fp16 range: P and dS are rounded to fp16 as MFMA operands, and with a gate dO, each small row times a power of two of
// its own (a small gradient behind a closed gate would have few of fp16's bits, or none), which is taken off its P again.
// P is multiplied by 2^15 there, whatever the gradients are, and keeps fp16's full precision down to 2^-29.  dS has a power of two for a workgroup, 2^ref, as large as keeps
// |dS| 2^ref <= 2^14 by the bound |dS_ij| <= |dO_i| |v_j| + |d_i| over its rows and keys, so gradients of any size keep
// full precision in dS down to 2^-28 of that bound.  Where dS is made of the rounded P, the difference of the two powers
// goes into dP - d in 32 bits (one power for both, in the exponential's argument alone, would save that product, 0.2 to 0.9 %
// of the long calls, and leave P no bits where dO is large: dV off by 1.6 % and dK by 1.8 at 8192 keys and dO of 8192, D = 128).
// Both roundings (half a step, 2^-11 of a value at most) are what the matrix instructions at this rate take; with
// them, and that of dO where there is a gate, a gradient's relative error is 3.6e-4 to 6.1e-4 against 64 bits,
// of which rounding it to fp16 is 2.1e-4.
//
// Bound by the matrix pipes: 8192 tokens of 32 heads, D = 128, causal, take 1750 to 1800 us from box to box, which is
// 1.07 to 1.10 PFLOP/s by the seven products, nine tenths of what a large fp16 product of a library reaches on the same
// card (1.2, where its power ends it); 4096 tokens of 24 heads over 4, D = 256, with a gate 782 to 805 us, of which the
// products are 715 to 735 (0.98 to 1.01 PFLOP/s), the rows 53 and the join 15.
#pragma once
#include <algorithm>
#include <cmath>

#include "attn_tiles.h"
#include "common.h"
#include "kernels.h"

namespace tsa {
namespace bwd {
namespace {

constexpr int kBlk = 32;  // rows and keys of a step

struct BwdArgs {
    Rows16 q, k, v, g /* dO, gated */, dq, dk, dv;
    const float* stat;     // [B][Hq][n_qb][64]: L log2(e) + power of 32 rows (inf: no such row, or it sees no key), then -d 2^power
    const float2* row_max; // [B][Hq][n_qb]: the largest |dO_i| and |d_i| of 32 rows; the second below 0: one is bad
    const float* key_max;  // [B][Hkv][n_kb]: the largest |v_j| of 32 keys; below 0: a bad k_j among them
    float* part;           // split key tiles: fp32 sums of each part
    const int *len_q, *len_k;
    int B, Hq, Hkv, Tq, Tk, n_qb, n_kb, n_kt, n_part, n_qt, n_kv, gated;  // n_kt, n_qt: tiles; n_kv: workgroups of the key tiles; gated: rows of g have powers
    float scale, c2;
};

// The arguments where the launch left them, read again after each `fresh`: held from the kernel's start for all
// its branches, they were 80 scalars more than there are, kept in vector registers that the products need.
typedef const __attribute__((address_space(4))) BwdArgs* args_t;
__device__ __forceinline__ args_t fresh(args_t a) {
    asm volatile("" : "+s"(a));
    return a;
}

__device__ __forceinline__ int count(const int* len, int b, int most) {
    return len ? min(max(len[b], 0), most) : most;
}

// Infinities and NaN reach what sees them and nothing else.  In the products themselves a pair that the
// mask hides has a weight of 0, but 0 times an infinity is NaN.  So a causal call's workgroups that
// meet a bad row (one whose dO or statistic is none, or, for dQ, whose key is none) copy their tiles through registers and
// put 0 for what is no number there; what sees the row gets its NaN from P, whose statistic is NaN
// (a bad key's queries have such statistics from the forward pass).
constexpr float kBad = 1e-30f;  // added below 0, so that a bound of 0 shows the mark too
__device__ __forceinline__ bool finite16(half_t x) { return __builtin_fabsf((float)x) < INFINITY; }

// The power of two with which a row of this norm is kept where a gate makes its dO: 2^power norm is at least
// 2^7 (its largest element 2^3, and what is 2^17 below that has fp16's full precision), larger rows stay as they are.  It
// ends at 48, for norms of 2^-41: smaller gradients are 0 in fp16.
__device__ __forceinline__ int row_power(float norm) {
    const int e = (int)(__builtin_bit_cast(unsigned, norm) >> 23 & 255) - 126;  // norm < 2^e
    return min(max(8 - e, 0), 48);
}

// ---------------------------------------------------------------------------------------
// Row statistics: a workgroup takes 32 rows of dO' and o' (8 lanes a row), or 32 keys' values.
// ---------------------------------------------------------------------------------------
struct RowsArgs {
    Rows16 g, o, gate, k, v, dgate;  // k: null without a mask
    half_t* gated;  // with a gate: dO [B][Hq][Tq][D], each row times 2^power
    const float* lse;
    float* stat;
    float2* row_max;
    float* key_max;
    const int *len_q, *len_k;
    int Hq, Hkv, Tq, Tk, n_qb, n_kb, n_rows;  // n_rows: workgroups of rows, those of keys follow
};

template <int D>
__global__ void __launch_bounds__(256, 3) attn_bwd_rows_kernel(RowsArgs a) {
    __shared__ float2 most[32];
    const int r = threadIdx.x >> 3, l8 = threadIdx.x & 7;
    int blk = blockIdx.x;
    if (blk < a.n_rows) {
        const int bh = blk / a.n_qb, qb = blk % a.n_qb, b = bh / a.Hq, h = bh % a.Hq;
        const int n = count(a.len_q, b, a.Tq), t = qb * kBlk + r;
        float d = 0.f, n2 = 0.f;
        half8_t x[D / 64], y[D / 64];
        float z[D / 8], u[D / 8];  // with a gate: dO, and o' / sigma
        if (t < n) {
            const half_t* g = a.g.data + b * a.g.b + h * a.g.h + t * a.g.t + 8 * l8;
            const half_t* o = a.o.data + b * a.o.b + h * a.o.h + t * a.o.t + 8 * l8;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                x[i] = *reinterpret_cast<const half8_t*>(g + 64 * i);
                y[i] = *reinterpret_cast<const half8_t*>(o + 64 * i);
                if (!a.gated) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        d = fmaf((float)x[i][j], (float)y[i][j], d);
                        n2 = fmaf((float)x[i][j], (float)x[i][j], n2);
                    }
                    continue;
                }
                const half8_t gt = *reinterpret_cast<const half8_t*>(a.gate.data + b * a.gate.b + h * a.gate.h + t * a.gate.t + 8 * l8 + 64 * i);
                half8_t dg;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // 1 / sigma, and 1 - sigma as sigma of the other sign (its own digits where sigma is near 1)
                    const float inv = 1.f + __expf(-(float)gt[j]), rest = __builtin_amdgcn_rcpf(1.f + __expf((float)gt[j]));
                    const float w = (float)x[i][j], o1 = (float)y[i][j];
                    dg[j] = (half_t)(w * o1 * rest);
                    z[8 * i + j] = w * __builtin_amdgcn_rcpf(inv);
                    u[8 * i + j] = o1 * inv;
                    n2 = fmaf(z[8 * i + j], z[8 * i + j], n2);
                }
                *reinterpret_cast<half8_t*>(a.dgate.data + b * a.dgate.b + h * a.dgate.h + t * a.dgate.t + 8 * l8 + 64 * i) = dg;
            }
        }
        n2 = sum8(n2);
        const float norm = sqrtf(n2);
        const int power = a.gated ? row_power(norm) : 0;
        if (a.gated && t < n) {
            const float up = __builtin_ldexpf(1.f, power);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                half8_t z16;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // (the product as a float, unseen: else one use of it gets it rounded at once and another twice, and
                    // where these differ d and dP come from different values)
                    float g32 = z[8 * i + j] * up;
                    asm volatile("" : "+v"(g32));
                    z16[j] = (half_t)g32;
                    // d_i goes with the dO that dP is made of, the rounded one: sum_j dS_ij then stays 0
                    // and the rounding weighs a fifth less in dQ and dK
                    const float r = (float)z16[j];
                    d = r != 0.f ? fmaf(r, u[8 * i + j], d) : d;  // (o' / sigma may be 0 times infinity)
                }
                *reinterpret_cast<half8_t*>(a.gated + ((size_t)bh * a.Tq + t) * D + 8 * l8 + 64 * i) = z16;
            }
        }
        d = sum8(d);
        if (l8 == 0) {
            float* st = a.stat + (size_t)blk * 64;
            const float lse = t < n ? a.lse[(size_t)bh * a.Tq + t] : -INFINITY;
            const bool bad = !(n2 < INFINITY) || !(lse < INFINITY);
            st[r] = bad ? NAN : lse == -INFINITY ? INFINITY : fmaf(lse, kLog2e, (float)power);
            st[32 + r] = -d;
            const float d1 = fabsf(__builtin_ldexpf(d, -power));
            // (a bad row, or one with no d, is left out of the bound: its results are NaN at any scale)
            most[r] = bad ? make_float2(0.f, -kBad) : make_float2(norm, d1 < INFINITY ? d1 : 0.f);
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            float2 m = most[threadIdx.x & 31];
            const bool bad = __builtin_amdgcn_ballot_w64(m.y < 0.f) != 0;
#pragma unroll
            for (int s = 16; s; s >>= 1) {
                m.x = fmaxf(m.x, __shfl_xor(m.x, s));
                m.y = fmaxf(m.y, __shfl_xor(m.y, s));
            }
            if (threadIdx.x == 0) a.row_max[blk] = make_float2(m.x, bad ? -fmaxf(m.y, 0.f) - kBad : m.y);
        }
    } else {
        blk -= a.n_rows;
        const int bh = blk / a.n_kb, kb = blk % a.n_kb, b = bh / a.Hkv, h = bh % a.Hkv;
        const int t = kb * kBlk + r;
        float n2 = 0.f, k2 = 0.f;
        if (t < count(a.len_k, b, a.Tk)) {
            const half_t* v = a.v.data + b * a.v.b + h * a.v.h + t * a.v.t;
            const half_t* k = a.k.data ? a.k.data + b * a.k.b + h * a.k.h + t * a.k.t : nullptr;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const half8_t x = *reinterpret_cast<const half8_t*>(v + 8 * l8 + 64 * i);
#pragma unroll
                for (int j = 0; j < 8; ++j) n2 = fmaf((float)x[j], (float)x[j], n2);
                if (k) {
                    const half8_t y = *reinterpret_cast<const half8_t*>(k + 8 * l8 + 64 * i);
#pragma unroll
                    for (int j = 0; j < 8; ++j) k2 = fmaf((float)y[j], (float)y[j], k2);
                }
            }
        }
        n2 = sum8(n2);
        k2 = sum8(k2);
        // (a value that is none is left out of the bound; its queries' d is none either)
        if (l8 == 0) most[r] = make_float2(n2 < INFINITY ? sqrtf(n2) : 0.f, k2 < INFINITY ? 0.f : -1.f);
        __syncthreads();
        if (threadIdx.x < 64) {
            float2 m = most[threadIdx.x & 31];
            const bool bad = __builtin_amdgcn_ballot_w64(m.y < 0.f) != 0;
#pragma unroll
            for (int s = 16; s; s >>= 1) m.x = fmaxf(m.x, __shfl_xor(m.x, s));
            if (threadIdx.x == 0) a.key_max[blk] = bad ? -m.x - kBad : m.x;
        }
    }
}

// ---------------------------------------------------------------------------------------
// What the tiles share
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp_mov<kDppXor1>(x));
    x = fmaxf(x, dpp_mov<kDppXor2>(x));
    x = fmaxf(x, dpp_mov<kDppHalfMirror>(x));
    x = fmaxf(x, dpp_mov<kDppRowMirror>(x));
    return max_xor32(max_xor16(x));
}
// 2^-ref
__device__ __forceinline__ float scale_back(float ref) { return __builtin_ldexpf(1.f, -(int)ref); }

// A value that is made here, not at its first use.
__device__ __forceinline__ float pinned(float x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A value as if unknown: what is made from it is made here, not held from an earlier use.
__device__ __forceinline__ int again(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// dS's power of two for a bound of |dS|: 2^ref bound <= 2^14 (up to 2^60: smaller gradients are 0 in fp16).
__device__ __forceinline__ float range_ref(float bound) {
    if (!(bound < 0x1p100f)) bound = 0x1p100f;
    const int bits = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, bound));  // (every lane's is the same)
    const int e = ((bits >> 23) & 255) - 126;                                        // bound < 2^e
    return (float)min(60, 14 - e);
}
// A workgroup's powers of two from the largest |dO_i|, |v_j| and |d_i| (every lane's are the same).  P's is 15 above the
// least of its rows', that of the largest |dO_i|: what a row's own power is above that, the statistic takes off its P.
struct Powers {
    float p, ds, up;  // up: 2^ds / 2^p, for dP - d
};
__device__ __forceinline__ Powers powers(args_t a, float most_g, float most_v, float most_d) {
    Powers x;
    x.p = 15.f + (a->gated ? (float)row_power(__builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, most_g)))) : 0.f);
    x.ds = range_ref(fmaf(most_g, most_v, most_d));
    x.up = scale_back(x.p - x.ds);
    return x;
}

__device__ __forceinline__ void lds_write_b128(unsigned addr, const half8_t& x) {
    typedef __attribute__((address_space(3))) half8_t* p_t;
    *(p_t)(addr) = x;
}
__device__ __forceinline__ float4_t lds_read_f4(unsigned addr) {
    typedef __attribute__((address_space(3))) const float4_t* p_t;
    return *(p_t)(addr);
}

// Copies of tiles of 32 rows of D elements by kN waves, 1 KiB an instruction.  The swizzle of a
// block's rows repeats every kPeriod blocks; a wave takes kPat neighbouring blocks and those a multiple of kPeriod
// on, so one offset a lane and tensor serves all of them, with a difference in the odd ones.
template <int D, int kN>
struct Copy {
    static constexpr int kBlocks = kBlk * D * 2 / 1024, kRows = 512 / D;  // of a tile; rows a block
    static constexpr int kPeriod = D == 64 ? 1 : 16 / kRows;
    static constexpr int kPat = kPeriod > kN ? kPeriod / kN : 1;
    static constexpr int kNext = kPeriod > kN ? kPeriod : kN;  // blocks from one of a wave's groups to its next
    static constexpr int kPer = kBlocks / (kN * kPat);         // groups a wave
    static constexpr unsigned kFlip = D == 128 ? 16 : 128;     // bytes by which a chunk moves from a block to the next, by XOR
    static_assert(kPat <= 2 && kPer * kN * kPat == kBlocks && kNext * kRows % (D == 64 ? 8 : 16) == 0, "one offset serves all groups");
    int w;  // which of the kN waves

    __device__ __forceinline__ int row(int lane) const { return kRows * kPat * w + lane / (D / 8); }
    __device__ __forceinline__ unsigned col(int lane) const { return 16u * (unsigned)((lane % (D / 8)) ^ swz<D>(row(lane))); }
    // This lane's offset from a tile's first row; stride in bytes, at most 2^25.
    __device__ __forceinline__ unsigned offset(int lane, unsigned stride) const { return (unsigned)row(lane) * stride + col(lane); }
    // p: the tile's first row; last: the last row there is, counted from it.
    __device__ __forceinline__ void operator()(const char* p, unsigned stride, unsigned off, int last, int lane, unsigned lds,
                                               bool clean = false) const {
        lds += 1024u * (unsigned)(kPat * w);
        int l = lane;  // (what is made of it is not held from copy to copy)
        asm volatile("" : "+v"(l));
        if (clean) {  // through registers, with 0 for what is no number
            const int r = row(l);
            const unsigned c = col(l);
#pragma unroll 1
            for (int k = 0; k < kPer * kPat; ++k) {
                const int blk = kNext * (k / kPat) + k % kPat;
                half8_t x = *reinterpret_cast<const half8_t*>(p + (size_t)stride * (unsigned)min(r + kRows * blk, last) + (k % kPat ? c ^ kFlip : c));
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = finite16(x[e]) ? x[e] : (half_t)0.f;
                lds_write_b128(lds + 1024u * (unsigned)blk + 16u * (unsigned)l, x);
            }
        } else if (last >= kBlk - 1) {
            const unsigned delta = (col(l) ^ kFlip) - col(l);
#pragma unroll
            for (int j = 0; j < kPer; ++j)
#pragma unroll
                for (int i = 0; i < kPat; ++i) {
                    const int blk = kNext * j + i;
                    dma_issue_any(p + (size_t)stride * (unsigned)(kRows * blk), off + (i ? delta : 0), lds + 1024u * (unsigned)blk);
                }
        } else {  // rows past the last are that one again
            const int r = row(l);
            const unsigned c = col(l);
#pragma unroll
            for (int j = 0; j < kPer; ++j)
#pragma unroll
                for (int i = 0; i < kPat; ++i) {
                    const int blk = kNext * j + i;
                    dma_issue_any(p, (unsigned)min(r + kRows * blk, last) * stride + (i ? c ^ kFlip : c), lds + 1024u * (unsigned)blk);
                }
        }
    }
};

// A operand of rows: A[row l % 32][16 kk + 8 (l / 32) + s] (addr: row l % 32's chunk l / 32).
__device__ __forceinline__ half8_t rows_op(unsigned addr, int kk) { return lds_read_b128(addr ^ (32u * kk)); }
// A operand of columns: A[d = 32 db + l % 32][k slot (l / 32, s)], slot s of k-step ks being row
// 16 ks + 8 (s / 4) + 4 (l / 32) + s % 4: the order in which a 32 x 32 result holds its rows.
template <int D>
__device__ __forceinline__ half8_t cols_op(unsigned a, int ks, int db) {
    // eight rows on, the swizzle has its bit 1 the other way at D >= 128, and is the same at D = 64
    constexpr unsigned kUp = D == 64 ? 0u : 32u;
    const half4_t lo = lds_read_tr16_at((a ^ (64u * db)) + (unsigned)(32 * D * ks));
    const half4_t up = lds_read_tr16_at((a ^ (64u * db + kUp)) + (unsigned)(32 * D * ks + 16 * D));
    return half8_t{lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
}

// kN operands read kPre steps in front of their use, pinned there: left alone, the compiler reads
// them all at once and spills.
template <int kN, int kPre, class Read, class Use>
__device__ __forceinline__ void ahead(const Read& read, const Use& use) {
    half8_t op[kN];
#pragma unroll
    for (int i = 0; i < kPre; ++i) op[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        if (i + kPre < kN) op[i + kPre] = read(i + kPre);
        __builtin_amdgcn_sched_barrier(0);
        use(i, op[i]);
        __builtin_amdgcn_sched_barrier(0);
    }
}
// The products of a 32-row tile at byte `tile`: its rows with kRB operands a k-step into s, and its
// columns (from block db0 on) with kRB operands of 16 rows into acc.  Addresses are one XOR next to their read; the empty
// asm keeps them from being held.
constexpr int kPreRows = 4, kPreCols = 3;  // over the operands that share a read
template <int D, int kRB>
__device__ __forceinline__ void mul_rows(unsigned rows, unsigned tile, const half8_t (&frag)[kRB][D / 16], float16_t (&s)[kRB]) {
    unsigned a = rows + tile;
    asm volatile("" : "+v"(a));
    ahead<D / 16, kPreRows / kRB>([&](int kk) { return rows_op(a, kk); },
                            [&](int kk, const half8_t& x) {
#pragma unroll
                                for (int i = 0; i < kRB; ++i) {
                                    s[i] = mfma32(x, frag[i][kk], s[i]);
                                    asm volatile("" : "+v"(s[i]));  // not moved to the result's first use, behind all reads
                                }
                            });
}
template <int D, int kRB, int kDB>
__device__ __forceinline__ void mul_cols(unsigned cols, unsigned tile, int db0, const half8_t (&op)[kRB][2], float16_t (&acc)[kRB * kDB]) {
    unsigned a = (cols + tile) ^ (64u * db0);
    asm volatile("" : "+v"(a));
    // a column block's two k-steps one after the other: their addresses are the same but for a constant
    ahead<2 * kDB, kRB == 2 ? 2 : kPreCols>([&](int i) { return cols_op<D>(a, i & 1, i >> 1); },
                             [&](int i, const half8_t& x) {
#pragma unroll
                                 for (int r = 0; r < kRB; ++r) acc[r * kDB + (i >> 1)] = mfma32(x, op[r][i & 1], acc[r * kDB + (i >> 1)]);
                             });
}

// The same with other work, a share of it behind each operand's products: while the matrix pipe has
// them, the wave goes on.  op(ks): the kRB operands of 16 rows; work(i): share i of 2 kDB.
template <int D, int kRB, int kDB, class Op, class Work>
__device__ __forceinline__ void mul_cols_beside(unsigned cols, unsigned tile, int db0, const Op& op, float16_t (&acc)[kRB * kDB], const Work& work) {
    const unsigned base = (cols + tile) ^ (64u * db0);
    constexpr int kPre = kRB == 2 ? 1 : kPreCols;
    half8_t x[2 * kDB], y[2][kRB];
    unsigned a = base;
    asm volatile("" : "+v"(a));
    op(0, y[0]);
#pragma unroll
    for (int i = 0; i < kPre; ++i) x[i] = cols_op<D>(a, i / kDB, i % kDB);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2 * kDB; ++i) {
        const int n = i + kPre;
        if (n == kDB) {  // the second k-step's addresses are made again
            a = base;
            asm volatile("" : "+v"(a));
        }
        if (n < 2 * kDB) x[n] = cols_op<D>(a, n / kDB, n % kDB);
        if (i == kDB - 1) op(1, y[1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < kRB; ++r) {
            acc[r * kDB + i % kDB] = mfma32(x[i], y[i / kDB][r], acc[r * kDB + i % kDB]);
            asm volatile("" : "+v"(acc[r * kDB + i % kDB]));
        }
        __builtin_amdgcn_sched_barrier(0);
        work(i);
        __builtin_amdgcn_sched_barrier(0);
    }
}

typedef float float8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ half8_t pack8(const float16_t& x, int half) {
    const float8_t y = half ? float8_t{x[8], x[9], x[10], x[11], x[12], x[13], x[14], x[15]}
                            : float8_t{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
    return __builtin_convertvector(y, half8_t);
}

// Half `half` of x up times the fp16 values p, rounded to fp16 (a product is v_fma_mixlo_f16: no conversions).
__device__ __forceinline__ half8_t times(const half8_t& p, const float16_t& x, int half, float up) {
    half8_t y;
#pragma unroll
    for (int r = 0; r < 8; ++r) y[r] = (half_t)fmaf((float)p[r], x[8 * half + r] * up, 0.f);
    return y;
}

// Lane-constant LDS addresses of operand reads in a tile at byte 0.
template <int D>
struct OpAddr {
    unsigned rows, cols;
    __device__ __forceinline__ OpAddr(int lane, unsigned base) {
        const int r = lane & 31, hi = lane >> 5;
        rows = base + (unsigned)r * (2 * D) + 16u * (unsigned)chunk_pos<D>(r, hi);
        const int i16 = lane & 15, vm = i16 & 3, t = 4 * hi + (i16 >> 2), chunk = 2 * ((lane >> 4) & 1) + (vm >> 1);
        cols = base + (unsigned)t * (2 * D) + 16u * (unsigned)chunk_pos<D>(t, chunk) + 8u * (vm & 1);
    }
};

// ---------------------------------------------------------------------------------------
// dK and dV of a key tile.  Waves work in pairs that own the same 32 kKB keys: the first (role P)
// makes S and P and sums dV, the second (role S) makes dP, takes P from LDS, and sums dK.  A wave so
// holds one operand (K or V) and one result in registers, which is what lets it own 64 keys (32 at
// D = 256) at two waves a SIMD: every Q and dO operand read from LDS feeds two products, where 32
// keys a wave would need all of LDS's 128 bytes a cycle to keep the MFMA pipes busy.
// Results are transposed (lane = key), so P and dS leave the first products in the second's operand
// layout.  Per step of 32 queries one barrier: P of the step, the tiles of the next one and the end of
// the last one's reads.
// ---------------------------------------------------------------------------------------
template <int D>
struct KvTile {
    static constexpr int kKB = D == 256 ? 1 : 2;    // 32-key blocks a pair
    static constexpr int kPairs = D == 256 ? 4 : 2;
    static constexpr int kW = 2 * kPairs;
    static constexpr int kKeys = 32 * kKB * kPairs;
    static constexpr int kTileB = kBlk * D * 2;     // bytes of a Q or dO tile
    static constexpr int kStage = 2 * kTileB;
    static constexpr int kStages = 3;
    static constexpr int kStatB = 256;
    static constexpr int kPB = kKB * 2048;          // bytes of a pair's P
    static constexpr int kStatAt = kStages * kStage, kPAt = kStatAt + kStages * kStatB;
    static constexpr int kLds = kPAt + 2 * kPairs * kPB;
    static constexpr int kAcc = kKB * (D / 32);     // 32 x 32 results a wave
};

// Writes kRB blocks of 32 rows by 32 kDB elements (lane = row, 4 consecutive elements a register group)
// times f.  They go through LDS (the wave's own at `lds`, 64 kRB 32 kDB bytes; no wave reads tiles any more): from the
// registers, an instruction's 64 lanes would write 16 bytes of each of 32 rows, and the address unit was
// 3.5 us of a call of 256 tokens, 4 heads, D = 128 (22 to 18).
template <int kRB, int kDB>
__device__ __forceinline__ void store_rows(const float16_t (&acc)[kRB * kDB], half_t* out, long long stride, int row0, int n_rows,
                                           int lane, float f, unsigned lds) {
    typedef __attribute__((address_space(3))) half4_t* p4_t;
    constexpr int kC = 4 * kDB;  // 16-byte chunks a row, chunk c of row r at c ^ (r % kC)
    const int r = lane & 31;
#pragma unroll
    for (int kb = 0; kb < kRB; ++kb)
#pragma unroll
        for (int db = 0; db < kDB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float16_t& x = acc[kb * kDB + db];
                *(p4_t)(lds + 16u * (unsigned)((32 * kb + r) * kC + ((4 * db + g) ^ (r % kC))) + 8u * (unsigned)(lane >> 5)) =
                    half4_t{(half_t)(x[4 * g] * f), (half_t)(x[4 * g + 1] * f), (half_t)(x[4 * g + 2] * f), (half_t)(x[4 * g + 3] * f)};
            }
#pragma unroll
    for (int i = 0; i < kRB * 32 * kC / 64; ++i) {
        const int u = 64 * i + lane, row = u / kC, c = (u % kC) ^ (row % kC);
        const half8_t x = lds_read_b128(lds + 16u * (unsigned)u);
        if (row0 + row < n_rows) *reinterpret_cast<half8_t*>(out + (row0 + row) * stride + 8 * c) = x;
    }
}

// The steps of a key tile: 32-query blocks first .. n - 1 of each query head of the group.
struct KvPlan {
    int n_q, n_k, last0, first, per, steps;
};
template <int D, bool kCausal>
__device__ __forceinline__ KvPlan kv_plan(args_t a, int b, int kt) {
    KvPlan p;
    p.n_q = count(a->len_q, b, a->Tq);
    p.n_k = count(a->len_k, b, a->Tk);
    p.last0 = p.n_k - p.n_q;  // query i sees keys up to i + last0
    const int k0 = kt * KvTile<D>::kKeys;
    p.first = kCausal ? max(0, k0 - p.last0) / kBlk : 0;
    p.per = max(0, (p.n_q + kBlk - 1) / kBlk - p.first);
    p.steps = k0 < p.n_k ? p.per * (a->Hq / a->Hkv) : 0;
    return p;
}

template <int D, bool kCausal, bool role_p>
__device__ __forceinline__ void kv_tile(args_t a, half_t* lds, int wg) {
    using T = KvTile<D>;
    constexpr int kDB = D / 32, kKK = D / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5;
    const int pair = wave % T::kPairs;
    const int n_bh = a->B * a->Hkv;
    // Workgroups go round the 256 CUs (an XCD after the other); each round begins one CU further on, so that
    // a long sequence's tiles, a power of two apart in a padded batch, do not share CUs (lengths 2048, 273, 546, 819 of
    // 32/8 heads, D = 128: 322 -> 215 us with the split in two).
    if (wg / 256 < a->n_kv / 256) wg = wg / 256 * 256 + (wg + wg / 256 * 8) % 256;
    const int bh = wg % n_bh, rest = wg / n_bh, part = rest % a->n_part, kt = rest / a->n_part;
    const int b = bh / a->Hkv, hk = bh % a->Hkv, G = a->Hq / a->Hkv;
    const KvPlan pl = kv_plan<D, kCausal>(a, b, kt);
    const int k0 = kt * T::kKeys + pair * 32 * T::kKB;
    if (kt * T::kKeys >= pl.n_k) return;
    const int u0 = (int)((long long)pl.steps * part / a->n_part), u1 = (int)((long long)pl.steps * (part + 1) / a->n_part);

    float16_t acc[T::kAcc];
#pragma unroll
    for (int i = 0; i < T::kAcc; ++i) acc[i] = float16_t{};

    const unsigned lds0 = (unsigned)(uintptr_t)(lds_void_t)(void*)lds;
    const OpAddr<D> op(lane, lds0);
    const unsigned p_at = lds0 + T::kPAt + (unsigned)pair * T::kPB + 16u * lane;

    // The steps of this part: 32-query blocks of one head after the other's, taken by running pointers
    // (products of strides held for the loop were more scalars than there are registers).
    const int n = u1 - u0, end = pl.first + pl.per, last = pl.n_q - 1;
    const int h0 = hk * G + u0 / max(1, pl.per);
    int qb = pl.first + u0 % max(1, pl.per), to_copy = qb;  // the current step's block, and the next copies'
    const unsigned q_row = 2u * (unsigned)a->q.t, g_row = 2u * (unsigned)a->g.t;  // bytes
    const char* qp = reinterpret_cast<const char*>(a->q.data + b * a->q.b + h0 * a->q.h) + (size_t)q_row * kBlk * qb;
    const char* gp = reinterpret_cast<const char*>(a->g.data + b * a->g.b + h0 * a->g.h) + (size_t)g_row * kBlk * qb;
    const float* sp = a->stat + ((size_t)(b * a->Hq + h0) * a->n_qb + qb) * 64;
    const long long q_jump = 2 * a->q.h - (long long)q_row * kBlk * pl.per, g_jump = 2 * a->g.h - (long long)g_row * kBlk * pl.per;
    const int s_jump = 64 * (a->n_qb - pl.per);
    unsigned ring = 0, ring2 = 0;  // stages of the current step and of the next copies
    // the scale of dS is the workgroup's bound
    float most_g = 0.f, most_d = 0.f, most_v = 0.f;
    bool some_bad = false;
    auto row_most = [&](int u) {
        const float2 m = a->row_max[(size_t)(b * a->Hq + hk * G + u / pl.per) * a->n_qb + pl.first + u % pl.per];
        most_g = fmaxf(most_g, m.x);
        most_d = fmaxf(most_d, fabsf(m.y));
        if (m.y < 0.f) some_bad = true;
    };
    for (int u = u0 + lane; u < u1; u += 64) row_most(u);
    {
        const int kb = kt * (T::kKeys / kBlk) + lane;
        if (lane < T::kKeys / kBlk && kb < a->n_kb) most_v = fabsf(a->key_max[(size_t)bh * a->n_kb + kb]);
    }
    const bool bad = kCausal && __builtin_amdgcn_ballot_w64(some_bad) != 0;
    // (by the second role: the first has the exponentials to do)
    const Copy<D, T::kPairs> copier = {pair};
    const unsigned q_off = copier.offset(lane, q_row), g_off = copier.offset(lane, g_row);
    auto copy = [&] {  // tiles and statistics of a step
        const unsigned st = lds0 + ring2 * T::kStage;
        copier(qp, q_row, q_off, last - to_copy * kBlk, lane, st, kCausal && bad);
        copier(gp, g_row, g_off, last - to_copy * kBlk, lane, st + T::kTileB, kCausal && bad);
        if (pair == 0) dma_issue_any4(sp, 4u * lane, lds0 + T::kStatAt + ring2 * T::kStatB);
        qp += (size_t)q_row * kBlk, gp += (size_t)g_row * kBlk, sp += 64;
        if (++to_copy == end) to_copy = pl.first, qp += q_jump, gp += g_jump, sp += s_jump;
        ring2 = ring2 + 1 == T::kStages ? 0 : ring2 + 1;
    };
    // a pair's keys are hidden from a step's queries while the last of those lies in front of the first of them
    auto hidden = [&](int x) { return kCausal && x * kBlk + kBlk - 1 + pl.last0 < k0; };

    if (!role_p && n > 0) copy();
    // K or V of the pair's keys, as B operands: slot s of k-step kk is row[16 kk + 8 hi + s]
    half8_t frag[T::kKB][kKK];
    {
        const auto& src = role_p ? a->k : a->v;
        const half_t* base = src.data + b * src.b + hk * src.h;
#pragma unroll
        for (int kb = 0; kb < T::kKB; ++kb) {
            // (past the last key its row again: what comes of it stays in lanes that store nothing)
            const half_t* row = base + min(k0 + 32 * kb + (lane & 31), pl.n_k - 1) * src.t + 8 * hi;
#pragma unroll
            for (int kk = 0; kk < kKK; ++kk) frag[kb][kk] = *reinterpret_cast<const half8_t*>(row + 16 * kk);
        }
    }
    const Powers pw = powers(a, wave_max(most_g), wave_max(most_v), wave_max(most_d));

    // register r of a result is query 4 hi + 8 (r / 4) + r % 4 of the step: hidden below this
    auto limit = [&](int x, int kb) {
        const int l = again(lane);
        return k0 + 32 * kb + (l & 31) - pl.last0 - x * kBlk - 4 * (l >> 5);
    };
    auto partly = [&](int x, int kb) { return kCausal && k0 + 32 * kb + 31 > x * kBlk + pl.last0; };
    if constexpr (role_p) {
        // round i: S of step i, then its P beside dV of step i - 1, while step i + 1 is copied.  P goes to LDS, for the
        // other role and for this one's next round
        const float c2 = a->c2;
        float16_t s[T::kKB];
        float4_t l;
        unsigned sa = 0, p_new = 0, p_old = 0;
        auto soft = [&](int x) {  // value x of S to P, 16 a key block
            const int kb = x >> 4, r = x & 15;
            s[kb][r] = pinned(fast_exp2(fmaf(s[kb][r], c2, pw.p - l[r & 3])));
            if ((r & 3) == 3 && x + 1 < 16 * T::kKB) l = lds_read_f4(sa + 32u * (((r >> 2) + 1) & 3));
            if ((r & 7) == 7) lds_write_b128(p_new + (unsigned)(kb * 2 + (r >> 3)) * 1024u, pack8(s[kb], r >> 3));
        };
        auto p_op = [&](int ks, half8_t (&y)[T::kKB]) {
#pragma unroll
            for (int kb = 0; kb < T::kKB; ++kb) y[kb] = lds_read_b128(p_old + (unsigned)(kb * 2 + ks) * 1024u);
        };
        constexpr int kShare = 16 * T::kKB / (2 * kDB);
#pragma clang loop unroll(disable)
        for (int i = 0, was = 0; i <= n; ++i) {
            asm volatile("" : "+s"(i));  // (a first round taken out of the loop spills)
            dma_wait_barrier();
            const unsigned done = ring;  // step i - 1's stage
            if (i > 0) ring = ring + 1 == T::kStages ? 0 : ring + 1;
            const bool sums = i > 0 && !hidden(was), scores = i < n && !hidden(qb);
            p_new = p_at + (unsigned)(i & 1) * (T::kPairs * T::kPB);
            p_old = p_at + (unsigned)(~i & 1) * (T::kPairs * T::kPB);
            sa = lds0 + T::kStatAt + ring * T::kStatB + 16u * hi;
            l = lds_read_f4(sa);
            if (scores) {
#pragma unroll
                for (int kb = 0; kb < T::kKB; ++kb) s[kb] = float16_t{};
                mul_rows<D, T::kKB>(op.rows, ring * T::kStage, frag, s);
#pragma unroll
                for (int kb = 0; kb < T::kKB; ++kb)
                    if (partly(qb, kb)) {
                        const int lim = limit(qb, kb);
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (8 * (r >> 2) + (r & 3) < lim) s[kb][r] = -INFINITY;
                    }
            } else {  // (what S was is not kept through this branch)
#pragma unroll
                for (int kb = 0; kb < T::kKB; ++kb) asm volatile("" : "=v"(s[kb]));
            }
            // one place that adds to dV (with more, the compiler moves the sums between registers): where there is no step i
            // its P is made of anything, and read by no one
            if (sums) {
                mul_cols_beside<D, T::kKB, kDB>(op.cols, done * T::kStage + T::kTileB, 0, p_op, acc, [&](int x) {
#pragma unroll
                    for (int j = 0; j < kShare; ++j) soft(x * kShare + j);
                });
            } else if (scores) {
#pragma unroll
                for (int x = 0; x < 16 * T::kKB; ++x) soft(x);
            }
            if (kCausal && bad && scores)  // a bad row's P is NaN where it is hidden too
#pragma unroll 1
                for (int x = 0; x < 2 * T::kKB; ++x)
                    if (partly(qb, x >> 1)) {
                        const int lim = limit(qb, x >> 1) - 16 * (x & 1);
                        half8_t y = lds_read_b128(p_new + (unsigned)x * 1024u);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (8 * (e >> 2) + (e & 3) < lim) y[e] = (half_t)0.f;
                        lds_write_b128(p_new + (unsigned)x * 1024u, y);
                    }
            was = qb;
            qb = qb + 1 == end ? pl.first : qb + 1;
        }
    } else {
        float16_t s[T::kKB];
        auto products = [&](unsigned stage) {  // dP - d of a step
            const unsigned st = stage * T::kStage, sa = lds0 + T::kStatAt + stage * T::kStatB + 128u + 16u * hi;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4_t d = lds_read_f4(sa + 32u * g);
#pragma unroll
                for (int kb = 0; kb < T::kKB; ++kb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kb][4 * g + e] = d[e];
            }
            mul_rows<D, T::kKB>(op.rows, st + T::kTileB, frag, s);
        };
        // round i: dS and dK of step i - 1, dP of step i
#pragma clang loop unroll(disable)
        for (int i = 0, was = 0; i <= n; ++i) {
            asm volatile("" : "+s"(i));  // (a first round taken out of the loop spills)
            dma_wait_barrier();
            if (i + 1 < n) copy();
            if (i > 0 && !hidden(was)) {
                const unsigned at = p_at + (unsigned)((i - 1) & 1) * (T::kPairs * T::kPB);
                half8_t ds[T::kKB][2];
                ahead<2 * T::kKB, 1>([&](int x) { return lds_read_b128(at + (unsigned)x * 1024u); },
                                     [&](int x, const half8_t& y) { ds[x >> 1][x & 1] = times(y, s[x >> 1], x & 1, pw.up); });
#pragma unroll
                for (int kb = 0; kb < T::kKB; ++kb)
                    if (partly(was, kb)) {  // 0 whatever dP is there
                        const int lim = limit(was, kb);
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (8 * (r >> 2) + (r & 3) < lim) ds[kb][r >> 3][r & 7] = (half_t)0.f;
                    }
                mul_cols<D, T::kKB, kDB>(op.cols, ring * T::kStage, 0, ds, acc);
            }
            if (i > 0) ring = ring + 1 == T::kStages ? 0 : ring + 1;
            if (i < n && !hidden(qb)) {
                products(ring);
            } else {
#pragma unroll
                for (int kb = 0; kb < T::kKB; ++kb) asm volatile("" : "=v"(s[kb]));
            }
            was = qb;
            qb = qb + 1 == end ? pl.first : qb + 1;
        }
    }

    lds_barrier();  // the tiles' LDS becomes the outputs'
    a = fresh(a);
    const float f = role_p ? scale_back(pw.p) : scale_back(pw.ds) * a->scale;
    if (a->n_part == 1) {
        const auto& out = role_p ? a->dv : a->dk;
        store_rows<T::kKB, kDB>(acc, out.data + b * out.b + hk * out.h, out.t, k0, pl.n_k, again(lane), f,
                                lds0 + (unsigned)wave * (64u * T::kKB * 32 * kDB));
    } else {  // [key tile][part][wave][16-byte group][lane]
        float4_t* w = reinterpret_cast<float4_t*>(a->part) + ((((size_t)bh * a->n_kt + kt) * a->n_part + part) * T::kW + wave) * (T::kAcc * 256) + lane;
#pragma unroll
        for (int i = 0; i < T::kAcc; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                w[(4 * i + g) * 64] = float4_t{acc[i][4 * g] * f, acc[i][4 * g + 1] * f, acc[i][4 * g + 2] * f, acc[i][4 * g + 3] * f};
    }
}

// ---------------------------------------------------------------------------------------
// dQ of a query tile, D = 64 and 128: a wave owns 32 kMB queries, with Q, dO and dQ in registers, and
// walks over the keys it sees.  S and dP are transposed (lane = query), so dS leaves them as the B
// operand of dQ^T += K^T dS^T, and L and d are one register each.
// ---------------------------------------------------------------------------------------
template <int D>
struct QTile {
    static constexpr bool kRoles = D == 256;  // waves in pairs, as for the key tiles
    static constexpr int kMB = D == 64 ? 2 : 1;
    static constexpr int kW = KvTile<D>::kW;
    static constexpr int kQueries = kRoles ? 32 * kW / 2 : 32 * kMB * kW;
    static constexpr int kTileB = kBlk * D * 2;
    static constexpr int kKRing = kRoles ? 4 : 3, kVRing = kRoles ? 2 : 3;
    static constexpr int kVAt = kKRing * kTileB, kXAt = kVAt + kVRing * kTileB;
    static constexpr int kLds = kXAt + (kRoles ? 4 * kW / 2 * 2048 : 0);
};

template <int D>
__device__ __forceinline__ Powers q_tile_powers(args_t a, int bh, int q0, int q_blocks, float most_v, int lane) {
    float n = 0.f, d = 0.f;
    const int qb = q0 / kBlk + lane;
    if (lane < q_blocks && qb < a->n_qb) {
        const float2 m = a->row_max[(size_t)bh * a->n_qb + qb];
        n = m.x;
        d = fabsf(m.y);
    }
    return powers(a, wave_max(n), wave_max(most_v), wave_max(d));
}
// The largest |v_j| of the key blocks of this lane, and whether some lane's holds a bad key.
__device__ __forceinline__ float key_most(args_t a, int bhk, int k_blocks, int lane, bool& bad) {
    float v = 0.f;
    bool some = false;
    for (int i = lane; i < k_blocks; i += 64) {
        const float x = a->key_max[(size_t)bhk * a->n_kb + i];
        v = fmaxf(v, fabsf(x));
        if (x < 0.f) some = true;
    }
    bad = __builtin_amdgcn_ballot_w64(some) != 0;
    return v;
}

template <int D, bool kCausal>
__device__ __forceinline__ void q_tile(args_t a, half_t* lds, int wg) {
    using T = QTile<D>;
    constexpr int kDB = D / 32, kKK = D / 16, kMB = T::kMB;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5;
    const int n_bh = a->B * a->Hq;
    const int bh = wg % n_bh, qt = kCausal ? a->n_qt - 1 - wg / n_bh : wg / n_bh;
    const int b = bh / a->Hq, h = bh % a->Hq, hk = h / (a->Hq / a->Hkv), bhk = b * a->Hkv + hk;
    const int n_q = count(a->len_q, b, a->Tq), n_k = count(a->len_k, b, a->Tk), last0 = n_k - n_q;
    const int tile0 = qt * T::kQueries;
    if (tile0 >= n_q) return;
    const int q0 = tile0 + wave * 32 * kMB;
    const int k_end = kCausal ? min(n_k, min(tile0 + T::kQueries, n_q) + last0) : n_k;
    const int n = max(0, (k_end + kBlk - 1) / kBlk);
    const int my_end = kCausal ? min(n_k, q0 + 32 * kMB + last0) : n_k;  // the wave's own

    half8_t qf[kMB][kKK], gf[kMB][kKK];
    float l2[kMB], nd[kMB];
#pragma unroll
    for (int m = 0; m < kMB; ++m) {
        const int q = min(q0 + 32 * m + (lane & 31), n_q - 1);  // (past the last query its row again, as for the keys)
        const half_t* qr = a->q.data + b * a->q.b + h * a->q.h + q * a->q.t + 8 * hi;
        const half_t* gr = a->g.data + b * a->g.b + h * a->g.h + q * a->g.t + 8 * hi;
        const float* st = a->stat + ((size_t)bh * a->n_qb + q / kBlk) * 64 + q % kBlk;
        l2[m] = st[0];
        nd[m] = st[32];
#pragma unroll
        for (int kk = 0; kk < kKK; ++kk) {
            qf[m][kk] = *reinterpret_cast<const half8_t*>(qr + 16 * kk);
            gf[m][kk] = *reinterpret_cast<const half8_t*>(gr + 16 * kk);
        }
    }
    float16_t acc[kMB * kDB];
#pragma unroll
    for (int i = 0; i < kMB * kDB; ++i) acc[i] = float16_t{};

    const unsigned lds0 = (unsigned)(uintptr_t)(lds_void_t)(void*)lds;
    const OpAddr<D> op(lane, lds0);
    const char *kp = reinterpret_cast<const char*>(a->k.data + b * a->k.b + hk * a->k.h), *vp = reinterpret_cast<const char*>(a->v.data + b * a->v.b + hk * a->v.h);
    const unsigned k_row = 2u * (unsigned)a->k.t, v_row = 2u * (unsigned)a->v.t;
    const float c2 = a->c2;
    unsigned ring = 2, ring2 = 0;  // stages of the current step and of the next copies
    bool bad;
    const float most_v = key_most(a, bhk, n, lane, bad);
    int left = n_k - 1;            // the last key, counted from the next copies' first
    const Copy<D, T::kW> copier = {wave};
    const unsigned k_off = copier.offset(lane, k_row), v_off = copier.offset(lane, v_row);
    auto copy = [&] {
        const unsigned st = lds0 + ring2 * T::kTileB;
        copier(kp, k_row, k_off, left, lane, st, kCausal && bad);
        copier(vp, v_row, v_off, left, lane, st + T::kVAt);
        kp += (size_t)k_row * kBlk, vp += (size_t)v_row * kBlk, left -= kBlk;
        ring2 = ring2 == 2 ? 0 : ring2 + 1;
    };
    if (n > 0) copy();
    if (n > 1) copy();
    const Powers pw = q_tile_powers<D>(a, bh, tile0, T::kQueries / kBlk, most_v, lane);
#pragma unroll
    for (int m = 0; m < kMB; ++m) l2[m] -= pw.ds;
#pragma clang loop unroll(disable)
    for (int j = 0; j < n; ++j) {
        dma_wait_barrier();
        if (j + 2 < n) copy();
        ring = ring == 2 ? 0 : ring + 1;
        if (j * kBlk >= my_end) continue;
        const unsigned st = ring * T::kTileB;
        float16_t s[kMB], w[kMB];
#pragma unroll
        for (int m = 0; m < kMB; ++m) {
            s[m] = float16_t{};
#pragma unroll
            for (int r = 0; r < 16; ++r) w[m][r] = nd[m];
        }
        mul_rows<D, kMB>(op.rows, st, qf, s);
        mul_rows<D, kMB>(op.rows, T::kVAt + st, gf, w);
        half8_t ds[kMB][2];
#pragma unroll
        for (int m = 0; m < kMB; ++m) {
#pragma unroll
            for (int r = 0; r < 16; ++r) w[m][r] *= fast_exp2(fmaf(s[m][r], c2, -l2[m]));
            if ((kCausal && j * kBlk + 31 > q0 + 32 * m + last0) || (j + 1) * kBlk > n_k) {
                // register r is key 32 j + 4 hi + 8 (r / 4) + r % 4
                const int lim = min(kCausal ? q0 + 32 * m + (lane & 31) + last0 : n_k, n_k - 1) - j * kBlk - 4 * hi;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (8 * (r >> 2) + (r & 3) > lim) w[m][r] = 0.f;
            }
            ds[m][0] = pack8(w[m], 0);
            ds[m][1] = pack8(w[m], 1);
        }
        mul_cols<D, kMB, kDB>(op.cols, st, 0, ds, acc);
    }
    lds_barrier();  // the tiles' LDS becomes the outputs'
    a = fresh(a);
    store_rows<kMB, kDB>(acc, a->dq.data + b * a->dq.b + h * a->dq.h, a->dq.t, q0, n_q, again(lane), scale_back(pw.ds) * a->scale,
                         lds0 + (unsigned)wave * (64u * kMB * 32 * kDB));
}

// The same at D = 256, by pairs of waves that own 32 queries: the first makes S and P, the second dP
// and dS, and each sums half of dQ's columns (the first a step later, when dS has come through LDS).  Q or dO and half of dQ are 128 registers a wave; all of them
// would not fit in one.
template <int D, bool kCausal, bool role_p>
__device__ __forceinline__ void q_tile_roles(args_t a, half_t* lds, int wg) {
    using T = QTile<D>;
    constexpr int kDB = D / 64, kKK = D / 16, kPairs = T::kW / 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5;
    const int pair = wave % kPairs;
    const int n_bh = a->B * a->Hq;
    const int bh = wg % n_bh, qt = kCausal ? a->n_qt - 1 - wg / n_bh : wg / n_bh;
    const int b = bh / a->Hq, h = bh % a->Hq, hk = h / (a->Hq / a->Hkv), bhk = b * a->Hkv + hk;
    const int n_q = count(a->len_q, b, a->Tq), n_k = count(a->len_k, b, a->Tk), last0 = n_k - n_q;
    const int tile0 = qt * T::kQueries;
    if (tile0 >= n_q) return;
    const int q0 = tile0 + pair * 32, my_q = q0 + (lane & 31);
    const int k_end = kCausal ? min(n_k, min(tile0 + T::kQueries, n_q) + last0) : n_k;
    const int n = max(0, (k_end + kBlk - 1) / kBlk);
    const int my_n = max(0, ((kCausal ? min(n_k, q0 + 32 + last0) : n_k) + kBlk - 1) / kBlk);  // steps of the pair's own

    half8_t frag[1][kKK];
    float stat;
    {
        const auto& src = role_p ? a->q : a->g;
        const int q = min(my_q, n_q - 1);
        const half_t* row = src.data + b * src.b + h * src.h + q * src.t + 8 * hi;
#pragma unroll
        for (int kk = 0; kk < kKK; ++kk) frag[0][kk] = *reinterpret_cast<const half8_t*>(row + 16 * kk);
        stat = a->stat[((size_t)bh * a->n_qb + q / kBlk) * 64 + q % kBlk + (role_p ? 0 : 32)];
    }
    float16_t acc[kDB];
#pragma unroll
    for (int i = 0; i < kDB; ++i) acc[i] = float16_t{};

    const unsigned lds0 = (unsigned)(uintptr_t)(lds_void_t)(void*)lds;
    const OpAddr<D> op(lane, lds0);
    const unsigned p_at = lds0 + T::kXAt + (unsigned)pair * 2048u + 16u * lane, ds_at = p_at + 2 * kPairs * 2048u;
    const char *kp = reinterpret_cast<const char*>(a->k.data + b * a->k.b + hk * a->k.h), *vp = reinterpret_cast<const char*>(a->v.data + b * a->v.b + hk * a->v.h);
    const unsigned k_row = 2u * (unsigned)a->k.t, v_row = 2u * (unsigned)a->v.t;
    bool bad;
    const float most_v = key_most(a, bhk, n, lane, bad);
    int left = n_k - 1;  // the last key, counted from the next copies' first
    const Copy<D, kPairs> copier = {pair};  // (by the second role: the first has the exponentials to do)
    const unsigned k_off = copier.offset(lane, k_row), v_off = copier.offset(lane, v_row);
    auto copy = [&](int j) {
        copier(kp, k_row, k_off, left, lane, lds0 + (unsigned)(j & 3) * T::kTileB, kCausal && bad);
        copier(vp, v_row, v_off, left, lane, lds0 + T::kVAt + (unsigned)(j & 1) * T::kTileB);
        kp += (size_t)k_row * kBlk, vp += (size_t)v_row * kBlk, left -= kBlk;
    };
    const int db0 = role_p ? 0 : kDB;  // dQ^T += K^T dS^T, this role's columns
    // register r is key 32 j + 4 hi + 8 (r / 4) + r % 4; the last that this lane's query sees
    auto limit = [&](int j) { return min(kCausal ? my_q + last0 : n_k, n_k - 1) - j * kBlk - 4 * hi; };
    auto ragged = [&](int j) { return (kCausal && j * kBlk + 31 > q0 + last0) || (j + 1) * kBlk > n_k; };
    if (!role_p && n > 0) copy(0);
    const Powers pw = q_tile_powers<D>(a, bh, tile0, T::kQueries / kBlk, most_v, lane);
    if constexpr (role_p) {
        // round j: S of step j, then its P beside dQ of step j - 2
        float16_t x1[1], &s = x1[0];
        const float l = pw.p - stat, c2 = a->c2;
        unsigned p_new = 0, ds_old = 0;
        auto soft = [&](int x) {
            s[x] = pinned(fast_exp2(fmaf(s[x], c2, l)));
            if ((x & 7) == 7) lds_write_b128(p_new + (unsigned)(x >> 3) * 1024u, pack8(s, x >> 3));
        };
        auto ds_op = [&](int ks, half8_t (&y)[1]) { y[0] = lds_read_b128(ds_old + (unsigned)ks * 1024u); };
#pragma clang loop unroll(disable)
        for (int j = 0; j < n + 2; ++j) {
            asm volatile("" : "+s"(j));
            dma_wait_barrier();
            const bool sums = j > 1 && j - 2 < my_n, scores = j < my_n;
            p_new = p_at + (unsigned)((j & 1) * kPairs * 2048);
            ds_old = ds_at + (unsigned)((j & 1) * kPairs * 2048);
            const unsigned done = (unsigned)((j - 2) & 3) * T::kTileB;
            if (scores) {
                s = float16_t{};
                mul_rows<D, 1>(op.rows, (unsigned)(j & 3) * T::kTileB, frag, x1);
                if (ragged(j)) {
                    const int lim = limit(j);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (8 * (r >> 2) + (r & 3) > lim) s[r] = -INFINITY;
                }
            } else {
                asm volatile("" : "=v"(s));
            }
            if (sums) {  // (as for the key tiles)
                mul_cols_beside<D, 1, kDB>(op.cols, done, db0, ds_op, acc, [&](int x) {
#pragma unroll
                    for (int i = 0; i < 8 / kDB; ++i) soft(x * (8 / kDB) + i);
                });
            } else if (scores) {
#pragma unroll
                for (int x = 0; x < 16; ++x) soft(x);
            }
        }
    } else {
        float16_t x1[1], &s = x1[0];
        auto products = [&](int j) {
            const unsigned st = (unsigned)(j & 1) * T::kTileB;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = stat;
            mul_rows<D, 1>(op.rows, T::kVAt + st, frag, x1);
        };
        // round j + 1: dS and dQ of step j, dP of step j + 1
#pragma clang loop unroll(disable)
        for (int j = -1; j < n + 1; ++j) {
            asm volatile("" : "+s"(j));
            dma_wait_barrier();
            if (j + 2 < n) copy(j + 2);
            if (j >= 0 && j < my_n) {
                half8_t ds1[1][2];
                half8_t(&ds)[2] = ds1[0];
#pragma unroll
                for (int x = 0; x < 2; ++x) ds[x] = times(lds_read_b128(p_at + (unsigned)((j & 1) * kPairs * 2048 + x * 1024)), s, x, pw.up);
                if (ragged(j)) {
                    const int lim = limit(j);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (8 * (r >> 2) + (r & 3) > lim) ds[r >> 3][r & 7] = (half_t)0.f;
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) lds_write_b128(ds_at + (unsigned)((j & 1) * kPairs * 2048 + x * 1024), ds[x]);
                mul_cols<D, 1, kDB>(op.cols, (unsigned)(j & 3) * T::kTileB, db0, ds1, acc);
            }
            if (j + 1 < my_n)
                products(j + 1);
            else  // no dP: what it was is not kept through the other branch
                asm volatile("" : "=v"(s));
        }
    }
    lds_barrier();  // the tiles' LDS becomes the outputs'
    a = fresh(a);
    store_rows<1, kDB>(acc, a->dq.data + b * a->dq.b + h * a->dq.h + (role_p ? 0 : D / 2), a->dq.t, q0, n_q, again(lane), scale_back(pw.ds) * a->scale,
                       lds0 + (unsigned)wave * (64u * 32 * kDB));
}

template <int D, bool kCausal>
__global__ void __launch_bounds__(64 * KvTile<D>::kW, 2) attn_bwd_kernel(BwdArgs args) {
    const args_t a = (args_t)__builtin_amdgcn_kernarg_segment_ptr();  // args, the only parameter
    constexpr int kLds = KvTile<D>::kLds > QTile<D>::kLds ? KvTile<D>::kLds : QTile<D>::kLds;
    __shared__ __align__(1024) half_t lds[kLds / 2];
    // the first half of a workgroup's waves makes P, the second dS
    const bool role_p = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) < KvTile<D>::kPairs;
    if ((int)blockIdx.x < args.n_kv) {
        if (role_p)
            kv_tile<D, kCausal, true>(fresh(a), lds, blockIdx.x);
        else
            kv_tile<D, kCausal, false>(fresh(a), lds, blockIdx.x);
    } else if constexpr (QTile<D>::kRoles) {
        if (role_p)
            q_tile_roles<D, kCausal, true>(fresh(a), lds, blockIdx.x - args.n_kv);
        else
            q_tile_roles<D, kCausal, false>(fresh(a), lds, blockIdx.x - args.n_kv);
    } else {
        q_tile<D, kCausal>(fresh(a), lds, blockIdx.x - args.n_kv);
    }
}

// The sum of a split key tile's parts, in their order: a thread for each 16-byte group that a lane wrote,
// all parts' loads on their way at once.
template <int D>
__global__ void __launch_bounds__(256) attn_bwd_join_kernel(BwdArgs a) {
    using T = KvTile<D>;
    constexpr int kWgs = T::kAcc;  // workgroups that a wave's 4 kAcc groups take
    const int lane = threadIdx.x & 63, n_bh = a.B * a.Hkv;
    const int i = blockIdx.x % kWgs * 4 + (threadIdx.x >> 6);
    const int wave = blockIdx.x / kWgs % T::kW, rest = blockIdx.x / (kWgs * T::kW), bh = rest % n_bh, kt = rest / n_bh;
    const int b = bh / a.Hkv, hk = bh % a.Hkv, n_k = count(a.len_k, b, a.Tk);
    const int key = kt * T::kKeys + wave % T::kPairs * 32 * T::kKB + 32 * (i / (D / 8)) + (lane & 31);
    if (key >= n_k) return;
    const float4_t* w = reinterpret_cast<const float4_t*>(a.part) + (((size_t)bh * a.n_kt + kt) * a.n_part * T::kW + wave) * (T::kAcc * 256) + i * 64 + lane;
    constexpr size_t kPart = (size_t)T::kW * (T::kAcc * 256);
    float4_t x = w[0];
    int p = 1;
    for (; p + 4 <= a.n_part; p += 4) {
        const float4_t y0 = w[p * kPart], y1 = w[(p + 1) * kPart], y2 = w[(p + 2) * kPart], y3 = w[(p + 3) * kPart];
        x = x + y0 + y1 + y2 + y3;
    }
    for (; p < a.n_part; ++p) x += w[p * kPart];
    const Rows16& out = wave < T::kPairs ? a.dv : a.dk;
    *reinterpret_cast<half4_t*>(out.data + b * out.b + hk * out.h + key * out.t + 4 * (lane >> 5) + 8 * (i % (D / 8))) =
        half4_t{(half_t)x[0], (half_t)x[1], (half_t)x[2], (half_t)x[3]};
}

// Sizes of a call, and where its workspace holds what.
struct Plan {
    int n_qb, n_kb, n_kt, n_qt, n_part;
    size_t stat, row_max, key_max, gated, part, bytes;
};
template <int D>
Plan plan(int B, int Hq, int Hkv, int Tq, int Tk, bool gated, bool causal, bool ragged) {
    Plan p;
    auto up = [](long long a, long long b) { return (int)((a + b - 1) / b); };
    p.n_qb = up(Tq, kBlk), p.n_kb = up(Tk, kBlk);
    p.n_kt = up(Tk, KvTile<D>::kKeys), p.n_qt = up(Tq, QTile<D>::kQueries);
    // A key tile's queries are split over workgroups where the longest tile would outlast the rest of the
    // device's work: in products of a step, against 1.3 times what a workgroup slot has to do on average
    // (of what a causal mask leaves, and of 0.7 of that where sequences have lengths, which only the device knows).  A part
    // costs its fp32 sums' way to memory and back (256 KiB at D = 256) and the join, so it has 16 steps at least.  us per
    // call by parts (1, 2, 3, 4, 6): 128 tiles of 768 steps (24/4 heads x 4096, D = 256) 1175 / 809 / 807 / 804 / 817;
    // 96 of 66 steps (3 x 701 over 1999, D = 256, ragged) 108 / 103 / 118 / 129 / 142 (there the query tiles, which are
    // not split, walk 63 steps of 3 products: those are the longest); 64 of 16 steps (2 x 512, D = 64) 51.5 / 55.9.  The 0.7 is
    // of batches with one full sequence and far shorter others; where lengths are passed that leave all rows, 4 x 2048 of 32/8 heads, D =
    // 128, take 571 for 524 without them, of 24/4 heads, D = 256, 856 for 809.
    const long long tiles = (long long)B * Hkv * p.n_kt, steps = (long long)(Hq / Hkv) * p.n_qb;
    const long long slots = D == 256 ? 256 : 512;
    const double seen = (causal ? 1 - 0.5 * std::min(1.0, (double)Tq / Tk) : 1) * (ragged ? 0.7 : 1);
    const double longest = 4.0 * steps, average = seen * (4.0 * tiles * steps + 3.0 * B * Hq * p.n_qt * p.n_kb) / slots;
    p.n_part = (int)std::max(1.0, std::min(std::ceil(longest / (1.3 * average)), (double)(steps / 16)));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t was = at;
        at += (bytes + 255) & ~(size_t)255;
        return was;
    };
    p.stat = take((size_t)B * Hq * p.n_qb * 64 * 4);
    p.row_max = take((size_t)B * Hq * p.n_qb * 8);
    p.key_max = take((size_t)B * Hkv * p.n_kb * 4);
    p.gated = gated ? take((size_t)B * Hq * Tq * D * 2) : 0;
    p.part = p.n_part > 1 ? take((size_t)tiles * p.n_part * KvTile<D>::kKeys * D * 2 * 4) : 0;
    p.bytes = at;
    return p;
}

template <int D>
hipError_t backward(const AttnRows& x, const Rows16& d_out, const Rows16& dq, const Rows16& dk, const Rows16& dv, const Rows16& dgate,
                    int B, int Hq, int Hkv, int Tq, float scale, int causal, void* ws, hipStream_t stream) {
    const int Tk = x.Sk;
    const bool gated = x.gate.data != nullptr;
    const Plan p = plan<D>(B, Hq, Hkv, Tq, Tk, gated, causal != 0, x.len_q || x.len_k);
    char* w = static_cast<char*>(ws);
    float* stat = reinterpret_cast<float*>(w + p.stat);
    float2* row_max = reinterpret_cast<float2*>(w + p.row_max);
    float* key_max = reinterpret_cast<float*>(w + p.key_max);
    half_t* g = reinterpret_cast<half_t*>(w + p.gated);
    RowsArgs r = {d_out, x.o, x.gate, causal ? x.k : Rows16{nullptr, 0, 0, 0}, x.v, dgate, gated ? g : nullptr, x.lse, stat, row_max, key_max, x.len_q, x.len_k, Hq, Hkv, Tq, Tk, p.n_qb,
                  p.n_kb, B * Hq * p.n_qb};
    hipLaunchKernelGGL(attn_bwd_rows_kernel<D>, dim3(r.n_rows + B * Hkv * p.n_kb), dim3(256), 0, stream, r);
    const Rows16 dO = gated ? Rows16{g, (long long)Hq * Tq * D, (long long)Tq * D, D} : d_out;
    BwdArgs a = {x.q, x.k, x.v, dO, dq, dk, dv, stat, row_max, key_max, reinterpret_cast<float*>(w + p.part), x.len_q, x.len_k,
                 B, Hq, Hkv, Tq, Tk, p.n_qb, p.n_kb, p.n_kt, p.n_part, p.n_qt, B * Hkv * p.n_kt * p.n_part, gated, scale, scale * kLog2e};
    const dim3 grid(a.n_kv + B * Hq * p.n_qt), block(64 * KvTile<D>::kW);
    if (causal)
        hipLaunchKernelGGL((attn_bwd_kernel<D, true>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((attn_bwd_kernel<D, false>), grid, block, 0, stream, a);
    if (p.n_part > 1)
        hipLaunchKernelGGL(attn_bwd_join_kernel<D>, dim3(B * Hkv * p.n_kt * KvTile<D>::kW * KvTile<D>::kAcc), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace
}  // namespace bwd

size_t attn_bwd_ws_bytes(int B, int Hq, int Hkv, int Tq, int Tk, int D, bool gated, bool causal) {
    size_t most = 0;  // with lengths or without
    for (const bool ragged : {false, true}) {
        const bwd::Plan p = D == 256   ? bwd::plan<256>(B, Hq, Hkv, Tq, Tk, gated, causal, ragged)
                            : D == 128 ? bwd::plan<128>(B, Hq, Hkv, Tq, Tk, gated, causal, ragged)
                                       : bwd::plan<64>(B, Hq, Hkv, Tq, Tk, gated, causal, ragged);
        most = std::max(most, p.bytes);
    }
    return most;
}

hipError_t attn_bwd(const AttnRows& x, const Rows16& d_out, const Rows16& dq, const Rows16& dk, const Rows16& dv, const Rows16& dgate,
                    int B, int Hq, int Hkv, int Tq, int D, float scale, int causal, void* ws, hipStream_t stream) {
    if (D == 256) return bwd::backward<256>(x, d_out, dq, dk, dv, dgate, B, Hq, Hkv, Tq, scale, causal, ws, stream);
    if (D == 128) return bwd::backward<128>(x, d_out, dq, dk, dv, dgate, B, Hq, Hkv, Tq, scale, causal, ws, stream);
    return bwd::backward<64>(x, d_out, dq, dk, dv, dgate, B, Hq, Hkv, Tq, scale, causal, ws, stream);
}

}  // namespace tsa
