// kv8_attn.h -- attention over the 8-bit K/V cache (see kv8.h for the format), over every block
// or over listed ones.
//
// o = softmax(scale q K^T) V per query row, one pass over the keys with a running maximum.  With
// codes k', v' and block scales sk, sv:
//   score  u_j = scale log2(e) sk (q . k'_j) + log2(sv)      (fp32, k' exact in fp16)
//   weight w_j = 2^(u_j - m + 12), m the running max of u    (fp16 operand of P V)
//   o = sum_j w_j v'_j / sum_j w_j / sv
// The value scale goes into the exponent, so the matrix instructions see whole numbers only and a
// weight is rounded once, whatever the blocks' scales are; 2^12 keeps weights down to 2^-36 of the
// largest in fp16's range.
#pragma once
#include "kv8.h"

namespace tsa {
namespace {

struct Kv8AttnArgs {
    Kv8 c;
    Rows16 q, gate, o;
    const int *len, *n_new, *blocks;
    float* part;  // split keys: [B][Hkv][rows][nsplit][D] sums, then as many (m, l) pairs
    int T, Hq, G, top, nsplit, causal;
    float c2;  // scale log2(e)
};

constexpr float kKvBias = 12.f;

// 8 codes (two words) as fp16: the byte under 0x64 is 1024 + code + 128.
__device__ __forceinline__ half8_t kv8_halves(unsigned w0, unsigned w1) {
    const half2_t off = {(half_t)1152.f, (half_t)1152.f};
    union { half2_t h[4]; half8_t v; } r;
    const unsigned hi = 0x64646464u;
    r.h[0] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(hi, w0, 0x04010400u)) - off;
    r.h[1] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(hi, w0, 0x04030402u)) - off;
    r.h[2] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(hi, w1, 0x04010400u)) - off;
    r.h[3] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(hi, w1, 0x04030402u)) - off;
    return r.v;
}

// max / sum over the four lanes that hold a row's keys (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float kv8_max4(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return max_xor32(x);
}
__device__ __forceinline__ float kv8_sum4(float x) {
    x += __shfl_xor(x, 16);
    return sum_xor32(x);
}

// A wave's state for NT tiles of 16 query rows: lane l owns row l % 16 of each.
template <int D, int NT>
struct Kv8State {
    half8_t q[NT][D / 32];  // operand B: step (i, s) holds d = 64 i + 16 (l / 16) + 8 s + 0 .. 7
    float4_t o[NT][D / 16]; // O^T: d = 16 dt + 4 (l / 16) + r
    float m[NT], l[NT];     // l: this lane's keys only
    int limit[NT];          // last key the row sees, -1: none
};

// One block's keys: kload(a, i, s) and vload(dt, s) give the operands, f the score factor, lsv
// and isv the value scale's log2 and reciprocal, p0 the block's first key; w returns the weights.
template <int D, int NT, class KLoad, class VLoad>
__device__ __forceinline__ void kv8_block(Kv8State<D, NT>& st, int p0, float f, float lsv, float isv, KLoad kload,
                                          VLoad vload, float4_t (&w)[NT][4]) {
    const int lane = threadIdx.x & 63, g4 = lane >> 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int a = 0; a < 4; ++a) w[nt][a] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const half8_t kf = kload(a, i, s);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) w[nt][a] = mfma16(kf, st.q[nt][2 * i + s], w[nt][a]);
            }
    half8_t p[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float big = -INFINITY;
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float u = w[nt][a][r] * f + lsv;
                w[nt][a][r] = p0 + 16 * a + 4 * g4 + r <= st.limit[nt] ? u : -INFINITY;
                big = fmaxf(big, w[nt][a][r]);
            }
        big = kv8_max4(big);
        const float m_new = fmaxf(st.m[nt], big);
        if (__any(m_new != st.m[nt])) {
            const float alpha = m_new == st.m[nt] ? 1.f : fast_exp2(st.m[nt] - m_new);
            st.m[nt] = m_new;
            st.l[nt] *= alpha;
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) st.o[nt][dt] *= alpha;
        }
        const float ref = m_new == -INFINITY ? 0.f : m_new - kKvBias;
        float sum = 0.f;
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                w[nt][a][r] = fast_exp2(w[nt][a][r] - ref);
                sum += w[nt][a][r];
                p[nt][a >> 1][4 * (a & 1) + r] = (half_t)w[nt][a][r];
            }
        // a block of scale NaN adds nothing where every key is masked
        st.l[nt] += sum == 0.f ? 0.f : sum * isv;
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const half8_t vf = vload(dt, s);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) st.o[nt][dt] = mfma16(vf, p[nt][s], st.o[nt][dt]);
        }
}

__device__ __forceinline__ bool kv8_bad(half_t x) {
    return (__builtin_bit_cast(unsigned short, x) & 0x7c00) == 0x7c00;
}

// A full block from its page.
template <int D, int NT>
__device__ __forceinline__ void kv8_page_block(Kv8State<D, NT>& st, const Kv8& c, int page, int h, int blk, float c2) {
    const int lane = threadIdx.x & 63;
    const size_t head = (size_t)page * c.Hkv + h;
    const uint4* kp = reinterpret_cast<const uint4*>(c.k + head * (kKvBlock * D)) + lane;
    const uint4* vp = reinterpret_cast<const uint4*>(c.v + head * (kKvBlock * D)) + lane;
    const float sk = c.k_scale[head], sv = c.v_scale[head];
    uint4 kr[4][D / 64], vr[D / 16];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int i = 0; i < D / 64; ++i) kr[a][i] = kp[(a * (D / 64) + i) * 64];
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) vr[dt] = vp[dt * 64];
    float4_t w[NT][4];
    kv8_block<D, NT>(
        st, blk * kKvBlock, c2 * sk, __builtin_amdgcn_logf(sv), 1.f / sv,
        [&](int a, int i, int s) { return s ? kv8_halves(kr[a][i].z, kr[a][i].w) : kv8_halves(kr[a][i].x, kr[a][i].y); },
        [&](int dt, int s) { return s ? kv8_halves(vr[dt].z, vr[dt].w) : kv8_halves(vr[dt].x, vr[dt].y); }, w);
}

// The open block from the ring.  Values that are not finite are left out of the matrix products,
// where a masked key's weight 0 would turn them into NaN for every query, and added for the
// queries that see them.  Elements of rows behind the sequence are whatever the ring held.
template <int D, int NT>
__device__ __forceinline__ void kv8_open_block(Kv8State<D, NT>& st, const Kv8& c, int b, int h, int blk, int len, float c2) {
    const int lane = threadIdx.x & 63, g4 = lane >> 4;
    const size_t at = kv8_open_at<D>(c, b, h, blk);
    const half_t* kp = c.k_open + at + lane * 16;
    const half_t* vp = c.v_open + at + lane * 16;
    const int p0 = blk * kKvBlock;
    bool bad = false;
    float4_t w[NT][4];
    kv8_block<D, NT>(
        st, p0, c2, 0.f, 1.f,
        [&](int a, int i, int s) { return *reinterpret_cast<const half8_t*>(kp + (a * (D / 64) + i) * 1024 + 8 * s); },
        [&](int dt, int s) {
            half8_t v = *reinterpret_cast<const half8_t*>(vp + dt * 1024 + 8 * s);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = p0 + 32 * s + 16 * (j >> 2) + 4 * g4 + (j & 3);
                const bool x = kv8_bad(v[j]);
                bad |= x && key < len;
                if (x || key >= len) v[j] = (half_t)0.f;
            }
            return v;
        },
        w);
    if (!__any(bad)) return;
    const half_t* vo = c.v_open + at;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll 1
        for (int x = 0; x < kKvBlock; ++x) {
            const int j = x >> 2, g = x & 3, key = 16 * (j >> 2) + 4 * g + (j & 3);
            float wj = 0.f;
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) wj = j == 4 * a + r ? w[nt][a][r] : wj;
            wj = __shfl(wj, 16 * g + (lane & 15));
            if (p0 + key > st.limit[nt]) continue;
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const half_t y = vo[kv8_v_at<D>(key, 16 * dt + 4 * g4 + e)];
                    if (kv8_bad(y)) st.o[nt][dt][e] += wj * (float)y;
                }
        }
}

// Workgroup (tile, b Hkv + h, split): 16 NT query rows of one K/V head's group over the split's
// share of their blocks, the blocks dealt to the four waves in turn.
// kList: a tile is one query's heads (16 NT at a time) over its listed blocks; otherwise rows are
// t G + g over all the sequence's blocks.
template <int D, int NT, bool kList>
__global__ void __launch_bounds__(256)
kv8_attn_kernel(Kv8AttnArgs p) {
    constexpr int kRows = 16 * NT;
    __shared__ float acc[kRows][D + 4];
    __shared__ float ml[4][2][kRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g4 = lane >> 4, n = lane & 15;
    const Kv8& c = p.c;
    const int b = blockIdx.y / c.Hkv, h = blockIdx.y % c.Hkv, split = blockIdx.z;
    const Kv8Seq sq = kv8_seq(c, p.len, p.n_new, b, p.T);
    int row0, row_end;
    if constexpr (kList) {
        const int per = (p.G + kRows - 1) / kRows;
        const int t = blockIdx.x / per;
        row0 = t * p.G + blockIdx.x % per * kRows;
        row_end = (t + 1) * p.G;
    } else {
        row0 = blockIdx.x * kRows;
        row_end = p.T * p.G;
    }
    row_end = min(row_end, (sq.n + sq.t0) * p.G);
    if (row0 >= row_end) return;

    Kv8State<D, NT> st;
    int see = -1;  // the last key that any row sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + 16 * nt + n;
        const int t = row / p.G, g = row % p.G;
        const bool is = row < row_end;
        const int pos = sq.len - (sq.n + sq.t0) + t;  // below 0: in front of the sequence
        st.limit[nt] = !is ? -1 : p.causal ? min(pos, sq.len - 1) : sq.len - 1;
        see = max(see, st.limit[nt]);
        const half_t* qr = p.q.data + b * p.q.b + (long long)(h * p.G + g) * p.q.h + t * p.q.t;
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s)
                st.q[nt][2 * i + s] = is ? *reinterpret_cast<const half8_t*>(qr + 64 * i + 16 * g4 + 8 * s) : half8_t{};
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) st.o[nt][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
        st.m[nt] = -INFINITY;
        st.l[nt] = 0.f;
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) see = max(see, __shfl_xor(see, x));
    see = __builtin_amdgcn_readfirstlane(see);

    const int nb = see / kKvBlock + (see >= 0 ? 1 : 0);  // blocks that any row sees
    const int items = kList ? p.top : nb;
    const int per = (items + p.nsplit - 1) / p.nsplit;
    const int end = min(items, (split + 1) * per);
    const int* list = kList ? p.blocks + (((size_t)b * c.Hkv + h) * p.T + row0 / p.G) * p.top : nullptr;
    const int n_full = sq.len / kKvBlock;
    int open = 0;  // how often the open block is among this wave's
    for (int i = split * per + wave; i < end; i += 4) {
        const int blk = kList ? list[i] : i;
        if (blk < 0 || blk >= nb) continue;
        if (blk >= n_full) {
            ++open;
            continue;
        }
        const int page = kv8_page(c, b, blk);
        if (page >= 0) kv8_page_block<D, NT>(st, c, page, h, blk, p.c2);
    }
    for (; open > 0; --open) kv8_open_block<D, NT>(st, c, b, h, n_full, sq.len, p.c2);

    // the four waves' sums, relative to their common maximum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        st.l[nt] = kv8_sum4(st.l[nt]);
        if (g4 == 0) {
            ml[wave][0][16 * nt + n] = st.m[nt];
            ml[wave][1][16 * nt + n] = st.l[nt];
        }
    }
    for (int w = 0; w < 4; ++w) {
        __syncthreads();
        if (wave != w) continue;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = 16 * nt + n;
            const float m = fmaxf(fmaxf(ml[0][0][r], ml[1][0][r]), fmaxf(ml[2][0][r], ml[3][0][r]));
            const float f = st.m[nt] == m ? 1.f : fast_exp2(st.m[nt] - m);
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) {
                float4_t* at = reinterpret_cast<float4_t*>(&acc[r][16 * dt + 4 * g4]);
                *at = w ? *at + st.o[nt][dt] * f : st.o[nt][dt] * f;
            }
        }
    }
    __syncthreads();
    const size_t rows_all = (size_t)p.T * p.G;
    for (int i = threadIdx.x; i < min(kRows, row_end - row0) * D; i += 256) {
        const int r = i / D, d = i % D, row = row0 + r;
        float m = -INFINITY, l = 0.f;
        for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w][0][r]);
        for (int w = 0; w < 4; ++w) l += ml[w][0][r] == m ? ml[w][1][r] : ml[w][1][r] * fast_exp2(ml[w][0][r] - m);
        if (p.nsplit > 1) {
            const size_t at = ((size_t)blockIdx.y * rows_all + row) * p.nsplit + split;
            p.part[at * D + d] = acc[r][d];
            if (d == 0) {
                float* pair = p.part + (size_t)gridDim.y * rows_all * p.nsplit * D + 2 * at;
                pair[0] = m;
                pair[1] = l;
            }
        } else {
            const int t = row / p.G, hq = h * p.G + row % p.G;
            float y = l == 0.f ? 0.f : acc[r][d] / l;
            if (p.gate.data) y /= 1.f + __expf(-(float)p.gate.data[b * p.gate.b + hq * p.gate.h + t * p.gate.t + d]);
            p.o.data[b * p.o.b + hq * p.o.h + t * p.o.t + d] = (half_t)y;
        }
    }
}

// Joins the splits of one row: workgroup (row, b Hkv + h), thread d.
template <int D>
__global__ void __launch_bounds__(D)
kv8_join_kernel(Kv8AttnArgs p) {
    const Kv8& c = p.c;
    const int b = blockIdx.y / c.Hkv, h = blockIdx.y % c.Hkv, row = blockIdx.x, d = threadIdx.x;
    const Kv8Seq sq = kv8_seq(c, p.len, p.n_new, b, p.T);
    const int t = row / p.G, hq = h * p.G + row % p.G;
    if (t >= sq.n + sq.t0) return;
    const size_t rows_all = (size_t)p.T * p.G;
    const size_t at = ((size_t)blockIdx.y * rows_all + row) * p.nsplit;
    const float* pair = p.part + (size_t)gridDim.y * rows_all * p.nsplit * D + 2 * at;
    float m = -INFINITY, l = 0.f, y = 0.f;
    for (int s = 0; s < p.nsplit; ++s) m = fmaxf(m, pair[2 * s]);
    for (int s = 0; s < p.nsplit; ++s) {
        if (pair[2 * s + 1] == 0.f) continue;
        const float f = pair[2 * s] == m ? 1.f : fast_exp2(pair[2 * s] - m);
        l += f * pair[2 * s + 1];
        y += f * p.part[(at + s) * D + d];
    }
    y = l == 0.f ? 0.f : y / l;
    if (p.gate.data) y /= 1.f + __expf(-(float)p.gate.data[b * p.gate.b + hq * p.gate.h + t * p.gate.t + d]);
    p.o.data[b * p.o.b + hq * p.o.h + t * p.o.t + d] = (half_t)y;
}

// Key splits of one tile: as many workgroups as the chip takes twice, not fewer than 4 blocks each.
inline int kv8_splits(long long tiles, int items) {
    const long long want = (1024 + tiles - 1) / tiles;
    const long long most = (items + 3) / 4;
    return (int)(want < most ? want : most);
}
inline long long kv8_tiles(int B, int T, int Hq, int Hkv, bool list) {
    const long long G = Hq / Hkv;
    return (long long)B * Hkv * (list ? (long long)T * ((G + 15) / 16) : (T * G + 15) / 16);
}
inline size_t kv8_part_bytes(int B, int T, int Hq, int Hkv, int D, int nsplit) {
    return nsplit > 1 ? (size_t)B * T * Hq * nsplit * (D + 2) * 4 : 0;
}

template <int D, bool kList>
hipError_t kv8_attn_d(Kv8AttnArgs p, hipStream_t stream) {
    const long long tiles = kv8_tiles(1, p.T, p.G, 1, kList);
    const dim3 grid((unsigned)tiles, (unsigned)(p.c.B * p.c.Hkv), (unsigned)p.nsplit);
    hipLaunchKernelGGL((kv8_attn_kernel<D, 1, kList>), grid, dim3(256), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.nsplit == 1) return e;
    const dim3 rows((unsigned)(p.T * p.G), (unsigned)(p.c.B * p.c.Hkv));
    hipLaunchKernelGGL(kv8_join_kernel<D>, rows, dim3(D), 0, stream, p);
    return hipGetLastError();
}
template <bool kList>
hipError_t kv8_attn_any(const Kv8AttnArgs& p, hipStream_t stream) {
    if (p.c.D == 64) return kv8_attn_d<64, kList>(p, stream);
    if (p.c.D == 128) return kv8_attn_d<128, kList>(p, stream);
    return kv8_attn_d<256, kList>(p, stream);
}

}  // namespace

hipError_t kv8_attn(const Kv8& c, const Rows16& q, const Rows16& gate, const Rows16& o, const int* len, const int* n_new,
                    int T, int Hq, int nb_hint, float scale, int causal, void* ws, hipStream_t stream) {
    const int nsplit = kv8_splits(kv8_tiles(c.B, T, Hq, c.Hkv, false), nb_hint);
    return kv8_attn_any<false>({c, q, gate, o, len, n_new, nullptr, (float*)ws, T, Hq, Hq / c.Hkv, 0, nsplit, causal, scale * kLog2e}, stream);
}

hipError_t kv8_attn_blocks(const Kv8& c, const Rows16& q, const Rows16& gate, const Rows16& o, const int* len,
                           const int* n_new, int T, int Hq, const int* blocks, int top, float scale, void* ws,
                           hipStream_t stream) {
    const int nsplit = kv8_splits(kv8_tiles(c.B, T, Hq, c.Hkv, true), top);
    return kv8_attn_any<true>({c, q, gate, o, len, n_new, blocks, (float*)ws, T, Hq, Hq / c.Hkv, top, nsplit, 1, scale * kLog2e}, stream);
}

}  // namespace tsa
