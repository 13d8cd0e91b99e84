// kv8_attn.h -- attention over the 8-bit K/V cache (see kv8.h for the format), over every block
// or over listed ones.
//
// o = softmax(scale q K^T) V per query row, one pass over the keys with a running maximum.  With
// codes k', v' and block scales sk, sv:
//   score  u_j = scale log2(e) sk (q . k'_j) + log2(sv)      (fp32, k' exact in fp16)
//   weight w_j = 2^(u_j - m + 12), m a running max of u      (fp16 operand of P V)
//   o = sum_j w_j v'_j / sum_j w_j / sv
// The value scale goes into the exponent, so the matrix instructions see whole numbers only and a
// weight is rounded once, whatever the blocks' scales are.  m is raised only when a score passes it
// by more than 3, so most blocks rescale nothing; weights reach up to 2^15 and keep fp16's whole
// range below (2^-24 is 2^-36 of the largest's at least: with m raised past 8 and weights of 2^7
// at m, small values next to a dominant key lost their last bits).
#pragma once
#include <climits>

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

constexpr float kKvBias = 12.f;  // a weight at the running maximum is 2^12,
constexpr float kKvSlack = 3.f;  // and up to 2^15 before the maximum is raised

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
__device__ __forceinline__ bool kv8_bad(half_t x) {
    return (__builtin_bit_cast(unsigned short, x) & 0x7c00) == 0x7c00;
}

// A wave's state for a tile of 16 query rows: lane l owns row l % 16.
template <int D>
struct Kv8Rows {
    half8_t q[D / 32];   // operand B: step (i, s) holds d = 64 i + 16 (l / 16) + 8 s + 0 .. 7
    float4_t o[D / 16];  // O^T: d = 16 dt + 4 (l / 16) + r
    float m, l;          // l: this lane's keys only
    int limit;           // last key the row sees, -1: none
};

// A block's scales as the softmax takes them: the score's factor (scale log2(e) sk), log2(sv) and
// 1 / sv.
struct Kv8Scale {
    float f, lsv, isv;
};

// The full blocks of a wave's work, in turn.  Each lane looks one of the next 64 items up (an entry
// of the list, or the item itself; its page; its scales), so that a block's are lane reads and no
// load waits for another once in 64 blocks.
template <bool kList>
struct Kv8Walk {
    int item, end, step;   // the next 64 are item + step * lane, below end
    int nb, n_full;        // blocks that are seen, and the full ones of them
    int open;              // how often the open block came up
    unsigned long long todo;
    int blks, pages;       // of this lane's item
    Kv8Scale scales;

    __device__ __forceinline__ void look(const Kv8& c, int b, int h, const int* list, float c2) {
        const int i = item + step * (int)(threadIdx.x & 63);
        blks = i < end ? (kList ? list[i] : i) : -1;
        if (kList || n_full < nb) open += __popcll(__ballot(blks >= n_full && blks < nb));
        const bool is = blks >= 0 && blks < n_full;
        pages = is ? kv8_page(c, b, blks) : -1;
        const size_t head = (size_t)max(pages, 0) * c.Hkv + h;
        const float sk = c.k_scale[head], sv = c.v_scale[head];
        scales = {c2 * sk, __builtin_amdgcn_logf(sv), __builtin_amdgcn_rcpf(sv)};
        todo = __ballot(pages >= 0);
        item += 64 * step;
    }
    // The next block; false when there is none.
    __device__ __forceinline__ bool next(const Kv8& c, int b, int h, const int* list, float c2, int& blk, int& page, Kv8Scale& sc) {
        while (todo == 0) {
            if (item >= end) return false;
            look(c, b, h, list, c2);
        }
        const int l = __builtin_ctzll(todo);
        todo &= todo - 1;
        auto read = [&](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l)); };
        blk = __builtin_amdgcn_readlane(blks, l);
        page = __builtin_amdgcn_readlane(pages, l);
        sc = {read(scales.f), read(scales.lsv), read(scales.isv)};
        return true;
    }
};

// Scores (w: raw q . k') to weights for 16 KA keys from p0 on: raises the running maximum where a
// score passes it by more than the slack, rescaling what there is, and adds to the row sums.
// `masked` (the same on all lanes): some row may not see all of the keys.
template <int D, int KA>
__device__ __forceinline__ void kv8_softmax(Kv8Rows<D>& st, float4_t (&w)[KA], int p0, const Kv8Scale& sc, bool masked) {
    const int left = st.limit - p0 - 4 * (int)((threadIdx.x & 63) >> 4);  // key 16 a + r is seen up to this
    if (masked) {
#pragma unroll
        for (int a = 0; a < KA; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) w[a][r] = 16 * a + r <= left ? w[a][r] : -INFINITY;
    }
    float big = -INFINITY;
#pragma unroll
    for (int a = 0; a < KA; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) big = fmaxf(big, w[a][r]);
    big = __builtin_fmaf(big, sc.f, sc.lsv);  // of this lane's keys
    if (__any(big > st.m + kKvSlack)) {
        const float m_new = fmaxf(st.m, max_xor32(max_xor16(big)));
        const float alpha = m_new == st.m ? 1.f : fast_exp2(st.m - m_new);
        st.m = m_new;
        st.l *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) st.o[dt] *= alpha;
    }
    const float c = sc.lsv - (st.m == -INFINITY ? 0.f : st.m - kKvBias);
    float sum = 0.f;
#pragma unroll
    for (int a = 0; a < KA; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) w[a][r] = fast_exp2(__builtin_fmaf(w[a][r], sc.f, c));
    if (masked) {  // again: of a block of scale NaN, a key that is not seen weighs 0
#pragma unroll
        for (int a = 0; a < KA; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) w[a][r] = 16 * a + r <= left ? w[a][r] : 0.f;
    }
#pragma unroll
    for (int a = 0; a < KA; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += w[a][r];
    st.l += sum == 0.f ? 0.f : sum * sc.isv;
}
// Weights of key tiles 2 s and 2 s + 1 as operand B.
template <int KA>
__device__ __forceinline__ half8_t kv8_weights(const float4_t (&w)[KA], int s) {
    return __builtin_convertvector(__builtin_shufflevector(w[2 * s], w[2 * s + 1], 0, 1, 2, 3, 4, 5, 6, 7), half8_t);
}

// 16 KA keys: kload(a, i, s) and vload(s, m, o) give the operands; between() is called where the
// keys' operands are done with.
template <int D, int NT, int KA, class KLoad, class VLoad, class Between>
__device__ __forceinline__ void kv8_keys(Kv8Rows<D> (&st)[NT], int p0, const Kv8Scale& sc, bool masked, KLoad kload,
                                         VLoad vload, Between between) {
    float4_t w[NT][KA];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int a = 0; a < KA; ++a) w[nt][a] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int a = 0; a < KA; ++a) {
                const half8_t kf = kload(a, i, s);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) w[nt][a] = mfma16(kf, st[nt].q[2 * i + s], w[nt][a]);
            }
    between();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) kv8_softmax<D, KA>(st[nt], w[nt], p0, sc, masked);
#pragma unroll
    for (int s = 0; s < KA / 2; ++s) {
        half8_t p[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) p[nt] = kv8_weights<KA>(w[nt], s);
#pragma unroll
        for (int m = 0; m < D / 32; ++m)
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                const half8_t vf = vload(s, m, o);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) st[nt].o[2 * m + o] = mfma16(vf, p[nt], st[nt].o[2 * m + o]);
            }
    }
}

// The same from operands in LDS (kb, vb: this lane's of K and V), read a few ahead of their products;
// between(e) is called among K's.  The queries' last kQl steps lie in LDS too (qb: this lane's).
template <int D, int NT, int KA, int kQl, class Between>
__device__ __forceinline__ void kv8_lds_keys(Kv8Rows<D> (&st)[NT], int p0, const Kv8Scale& sc, bool masked, const half8_t* kb,
                                             const half8_t* vb, const half8_t* qb, Between between) {
    constexpr int kOps = KA * (D / 32), kAhead = D == 256 ? 3 : 6, kQr = D / 32 - kQl;
    float4_t w[NT][KA];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int a = 0; a < KA; ++a) w[nt][a] = float4_t{0.f, 0.f, 0.f, 0.f};
    half8_t op[kOps], ql[NT];
    auto read_k = [&](int e) {  // key tile e % KA, step e / KA
        const int a = e % KA, x = e / KA;
        op[e] = kb[((a * (D / 64) + x / 2) * 2 + x % 2) * 64];
    };
#pragma unroll
    for (int e = 0; e < kAhead; ++e) read_k(e);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < kOps; ++e) {
        if (e + kAhead < kOps) read_k(e + kAhead);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            w[nt][e % KA] = mfma16(op[e], e / KA < kQr ? st[nt].q[e / KA] : ql[nt], w[nt][e % KA]);
        if (kQl && (e + 1) % KA == 0 && (e + 1) / KA >= kQr && e + 1 < kOps) {  // the next step's queries
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) ql[nt] = qb[(((e + 1) / KA - kQr) * NT + nt) * 64];
        }
        between(e);
        __builtin_amdgcn_sched_barrier(0);
    }
    auto read_v = [&](int e) { op[e] = vb[e * 64]; };  // (s, m, o) in order
#pragma unroll
    for (int e = 0; e < kAhead; ++e) read_v(e);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) kv8_softmax<D, KA>(st[nt], w[nt], p0, sc, masked);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < KA / 2; ++s) {
        half8_t p[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) p[nt] = kv8_weights<KA>(w[nt], s);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
            const int e = s * (D / 16) + dt;
            if (e + kAhead < kOps) read_v(e + kAhead);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) st[nt].o[dt] = mfma16(op[e], p[nt], st[nt].o[dt]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __builtin_amdgcn_s_setprio(0);
}

// The open block from the ring: n of its rows are the sequence's, those behind are whatever the
// ring held.  Values that are not finite are left out of the matrix products, where a masked key's
// weight 0 would turn them into NaN for every query, and added for the queries that see them.
template <int D>
__device__ __forceinline__ void kv8_open_block(Kv8Rows<D>& st, const Kv8& c, int b, int h, int blk, int n, float c2) {
    typedef unsigned uint4_v __attribute__((ext_vector_type(4)));
    typedef unsigned short ushort8_t __attribute__((ext_vector_type(8)));
    const int lane = threadIdx.x & 63, g4 = lane >> 4;
    const size_t at = kv8_open_at<D>(c, b, h, blk);
    const half8_t* kp = reinterpret_cast<const half8_t*>(c.k_open + at) + 2 * lane;
    const half8_t* vp = reinterpret_cast<const half8_t*>(c.v_open + at) + 2 * lane;
#pragma unroll 1
    for (int s = 0; 32 * s < n; ++s) {  // half a block at a time
        const int p0 = blk * kKvBlock + 32 * s;
        float4_t w[2] = {float4_t{0.f, 0.f, 0.f, 0.f}, float4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int a = 0; a < 2; ++a) w[a] = mfma16(kp[((2 * s + a) * (D / 64) + i) * 128 + x], st.q[2 * i + x], w[a]);
        kv8_softmax<D, 2>(st, w, p0, {c2, 0.f, 1.f}, true);
        const half8_t p = kv8_weights<2>(w, 0);
        uint4_v keep;  // elements of rows that there are
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int key = 32 * s + 16 * (j >> 1) + 4 * g4 + 2 * (j & 1);
            keep[j] = (key < n ? 0xffffu : 0u) | (key + 1 < n ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int m = 0; m < D / 32; m += 2) {  // 64 d at a time
            half8_t v[4];
            ushort8_t big = {};
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = vp[(s * (D / 32) + m + (x >> 1)) * 128 + (x & 1)];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                v[x] = __builtin_bit_cast(half8_t, __builtin_bit_cast(uint4_v, v[x]) & keep);
                big = __builtin_elementwise_max(big, __builtin_bit_cast(ushort8_t, v[x]) & (unsigned short)0x7fff);
            }
            int most = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) most = max(most, (int)big[j]);
            const bool bad = __any(most >= 0x7c00);
            if (bad) {
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[x][j] = kv8_bad(v[x][j]) ? (half_t)0.f : v[x][j];
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) st.o[2 * m + x] = mfma16(v[x], p, st.o[2 * m + x]);
            if (!bad) continue;
            const half_t* vo = c.v_open + at;
#pragma unroll 1
            for (int y = 0; y < 32; ++y) {
                const int j = y >> 2, g = y & 3, key = 16 * (j >> 2) + 4 * g + (j & 3);
                float wj = 0.f;
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r) wj = j == 4 * a + r ? w[a][r] : wj;
                wj = __shfl(wj, 16 * g + (lane & 15));
                if (p0 + key > st.limit) continue;
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const half_t z = vo[kv8_v_at<D>(32 * s + key, 16 * (2 * m + x) + 4 * g4 + e)];
                        if (kv8_bad(z)) st.o[2 * m + x][e] += wj * (float)z;
                    }
            }
        }
    }
}

// The queries of 16 of the T G rows t G + g of a K/V head's group, from row0 on.
template <int D>
__device__ __forceinline__ void kv8_queries(Kv8Rows<D>& st, const Kv8AttnArgs& p, int b, int h, int row0, int row_end) {
    const int lane = threadIdx.x & 63, g4 = lane >> 4, row = row0 + (lane & 15), t = row / p.G, g = row % p.G;
    const half_t* qr = p.q.data + b * p.q.b + (long long)(h * p.G + g) * p.q.h + t * p.q.t;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s)
            st.q[2 * i + s] = row < row_end ? *reinterpret_cast<const half8_t*>(qr + 64 * i + 16 * g4 + 8 * s) : half8_t{};
}
// NT tiles from row0 on with nothing summed yet, and which keys they see: the last that any row
// does (`most`) and the last that all do (`least`).
template <int D, int NT>
__device__ __forceinline__ void kv8_begin(Kv8Rows<D> (&st)[NT], const Kv8AttnArgs& p, const Kv8Seq& sq, int b, int h, int row0,
                                          int row_end, int& most, int& least) {
    most = -1;
    least = INT_MAX;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        kv8_queries<D>(st[nt], p, b, h, row0 + 16 * nt, row_end);
        const int row = row0 + 16 * nt + (int)(threadIdx.x & 15);
        const bool is = row < row_end;
        const int pos = sq.len - (sq.n + sq.t0) + row / p.G;  // below 0: in front of the sequence
        st[nt].limit = !is ? -1 : p.causal ? min(pos, sq.len - 1) : sq.len - 1;
        most = max(most, st[nt].limit);
        if (is) least = min(least, st[nt].limit);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) st[nt].o[dt] = float4_t{0.f, 0.f, 0.f, 0.f};
        st[nt].m = -INFINITY;
        st[nt].l = 0.f;
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
        most = max(most, __shfl_xor(most, x));
        least = min(least, __shfl_xor(least, x));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(least);
}

// The queries have arrived: said in front of a loop that only reads them, the loop waits for none
// of the loads that it has under way itself.
template <int D, int NT>
__device__ __forceinline__ void kv8_arrived(Kv8Rows<D> (&st)[NT]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) asm volatile("" : "+v"(st[nt].q[i]));
}

// Where a split's sums of a row lie: [row][split][D] sums, behind all of them (m, l) pairs.
template <int D>
__device__ __forceinline__ float* kv8_part(const Kv8AttnArgs& p, size_t bh, int row, int split) {
    return p.part + ((bh * p.T * p.G + row) * p.nsplit + split) * D;
}
template <int D>
__device__ __forceinline__ float* kv8_pair(const Kv8AttnArgs& p, size_t bh, int row, int split) {
    const size_t rows = (size_t)p.c.B * p.c.Hkv * p.T * p.G;
    return p.part + rows * p.nsplit * D + ((bh * p.T * p.G + row) * p.nsplit + split) * 2;
}

// 4 consecutive d of a finished row, times the gate.
__device__ __forceinline__ void kv8_store4(const Kv8AttnArgs& p, int b, int hq, int t, int d, float4_t y, float l, half4_t gate) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that saw no key is 0
    half4_t out;
    float g[4] = {inv, inv, inv, inv};
    if (p.gate.data) {
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = inv * __builtin_amdgcn_rcpf(1.f + __expf(-(float)gate[e]));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = (half_t)(y[e] * g[e]);
    *reinterpret_cast<half4_t*>(p.o.data + b * p.o.b + hq * p.o.h + t * p.o.t + d) = out;
}
__device__ __forceinline__ half4_t kv8_gate4(const Kv8AttnArgs& p, int b, int hq, int t, int d) {
    if (!p.gate.data) return half4_t{};
    return *reinterpret_cast<const half4_t*>(p.gate.data + b * p.gate.b + hq * p.gate.h + t * p.gate.t + d);
}

// Keys that a wave of the row kernel takes at a time, and their codes in registers.
template <int D>
struct Kv8Regs {
    static constexpr int kKeys = D == 256 ? 32 : 64, kN = kKeys * D / 1024;
    uint4 k[kN], v[kN];

    __device__ __forceinline__ void load_k(const Kv8& c, int page, int h, int part) {
        const size_t head = (size_t)page * c.Hkv + h;
        const uint4* kp = reinterpret_cast<const uint4*>(c.k + head * (kKvBlock * D)) + part * (kN * 64) + (threadIdx.x & 63);
#pragma unroll
        for (int i = 0; i < kN; ++i) k[i] = kp[i * 64];
    }
    __device__ __forceinline__ void load_v(const Kv8& c, int page, int h, int part) {
        const size_t head = (size_t)page * c.Hkv + h;
        const uint4* vp = reinterpret_cast<const uint4*>(c.v + head * (kKvBlock * D)) + part * (kN * 64) + (threadIdx.x & 63);
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = vp[i * 64];
    }
};

// Few rows: workgroup (tile, b Hkv + h, split), one tile of 16 query rows of a K/V head's group over
// the split's share of their blocks, the blocks dealt to the four waves in turn.  A wave's
// next keys are on their way to registers as soon as its last ones have been multiplied, its next
// values likewise.
// kList: a tile is one query's heads (16 at a time) over its listed blocks; otherwise rows are
// t G + g over all the sequence's blocks.
template <int D, bool kList>
__global__ void __launch_bounds__(256, 2)
kv8_row_kernel(Kv8AttnArgs p) {
    constexpr int kParts = kKvBlock / Kv8Regs<D>::kKeys, kRow = D + 4;
    __shared__ __align__(16) float acc[2][16][kRow];
    __shared__ float ml[4][2][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g4 = lane >> 4, n = lane & 15;
    const Kv8& c = p.c;
    const int b = blockIdx.y / c.Hkv, h = blockIdx.y % c.Hkv, split = blockIdx.z;
    const Kv8Seq sq = kv8_seq(c, p.len, p.n_new, b, p.T);
    int row0, row_end;
    if constexpr (kList) {
        const int per = (p.G + 15) / 16, t = blockIdx.x / per;
        row0 = t * p.G + blockIdx.x % per * 16;
        row_end = (t + 1) * p.G;
    } else {
        row0 = blockIdx.x * 16;
        row_end = p.T * p.G;
    }
    row_end = min(row_end, (sq.n + sq.t0) * p.G);
    if (row0 >= row_end) return;

    Kv8Rows<D> rows[1], &st = rows[0];
    int see, least;
    kv8_begin<D, 1>(rows, p, sq, b, h, row0, row_end, see, least);
    const int nb = see / kKvBlock + (see >= 0 ? 1 : 0);  // blocks that any row sees
    const int n_full = min(sq.len / kKvBlock, nb);
    const int items = kList ? p.top : nb;
    const int per = (items + p.nsplit - 1) / p.nsplit;
    const int end = min(items, (split + 1) * per);
    const int* list = kList ? p.blocks + (((size_t)b * c.Hkv + h) * p.T + row0 / p.G) * p.top : nullptr;
    Kv8Walk<kList> walk = {split * per + wave, end, 4, nb, n_full, 0, 0};
    int blk = 0, page = -1;
    Kv8Scale sc = {};
    auto next = [&]() {
        if (!walk.next(c, b, h, list, p.c2, blk, page, sc)) page = -1;
    };
    // rows of one query see whole blocks but the last; several queries' last one or two are masked
    auto masked = [&](int k) { return (k + 1) * kKvBlock - 1 > least; };
    next();
    if (page >= 0) {
        Kv8Regs<D> x;
        x.load_k(c, page, h, 0);
        x.load_v(c, page, h, 0);
        kv8_arrived<D, 1>(rows);
        while (page >= 0) {
            const int now = blk, here = page;
            const Kv8Scale scale = sc;
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                const bool last = part == kParts - 1;
                if (last) next();
                const int to = last ? page : here;
                kv8_keys<D, 1, Kv8Regs<D>::kKeys / 16>(
                    rows, now * kKvBlock + part * Kv8Regs<D>::kKeys, scale, masked(now),
                    [&](int a, int i, int s) {
                        const uint4& k = x.k[a * (D / 64) + i];
                        return s ? kv8_halves(k.z, k.w) : kv8_halves(k.x, k.y);
                    },
                    [&](int s, int m, int o) {
                        const uint4& v = x.v[s * (D / 32) + m];
                        return o ? kv8_halves(v.z, v.w) : kv8_halves(v.x, v.y);
                    },
                    [&]() {
                        if (to >= 0) x.load_k(c, to, h, last ? 0 : part + 1);
                    });
                if (to >= 0) x.load_v(c, to, h, last ? 0 : part + 1);
            }
        }
    }
    for (; walk.open > 0; --walk.open) kv8_open_block<D>(st, c, b, h, n_full, sq.len - n_full * kKvBlock, p.c2);

    // the four waves' sums, relative to their common maximum
    st.l = sum_xor32(sum_xor16(st.l));
    if (g4 == 0) {
        ml[wave][0][n] = st.m;
        ml[wave][1][n] = st.l;
    }
    __syncthreads();
    {
        const float m = fmaxf(fmaxf(ml[0][0][n], ml[1][0][n]), fmaxf(ml[2][0][n], ml[3][0][n]));
        const float f = st.m == m ? 1.f : fast_exp2(st.m - m);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) st.o[dt] *= f;
    }
    if (wave >= 2) {
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<float4_t*>(&acc[wave & 1][n][16 * dt + 4 * g4]) = st.o[dt];
    }
    __syncthreads();
    if (wave < 2) {
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
            float4_t* at = reinterpret_cast<float4_t*>(&acc[wave][n][16 * dt + 4 * g4]);
            *at += st.o[dt];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(16, row_end - row0) * (D / 4); i += 256) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w][0][r]);
#pragma unroll
        for (int w = 0; w < 4; ++w) l += ml[w][0][r] == m ? ml[w][1][r] : ml[w][1][r] * fast_exp2(ml[w][0][r] - m);
        const float4_t y = *reinterpret_cast<const float4_t*>(&acc[0][r][d]) + *reinterpret_cast<const float4_t*>(&acc[1][r][d]);
        if (p.nsplit > 1) {
            if (l != 0.f) *reinterpret_cast<float4_t*>(kv8_part<D>(p, blockIdx.y, row0 + r, split) + d) = y;
            if (d == 0) *reinterpret_cast<float2*>(kv8_pair<D>(p, blockIdx.y, row0 + r, split)) = float2{m, l};
        } else {
            const int t = (row0 + r) / p.G, hq = h * p.G + (row0 + r) % p.G;
            kv8_store4(p, b, hq, t, d, y, l, kv8_gate4(p, b, hq, t, d));
        }
    }
}

constexpr int kKvMaxSplits = 128;

// Many rows: a workgroup is kWaves waves of 16 NT query rows each over one split of their blocks.  A
// stage of kKeys keys and their values (16 KiB of codes at the most) goes from memory to registers
// two stages ahead, is turned into fp16 operands once for all waves, and lies in one of two LDS
// buffers in operand order, so every LDS access is 16 consecutive bytes a lane and a code is
// converted once per 16 NT kWaves rows.  One barrier a stage.  Two waves a SIMD: two workgroups of 4
// waves a CU, or at D = 256, NT = 2 one of 8 (a thread then holds half as many codes, without which
// the 128 sums and 64 query registers spill).
template <int D, int NT>
struct Kv8Tile {
    static constexpr int kWaves = D == 256 && NT == 2 ? 8 : 4, kThreads = 64 * kWaves;
    static constexpr int kKeys = D == 256 ? 32 : 64, kParts = kKvBlock / kKeys;
    static constexpr int kUnits = kKeys * D / 16;          // 16-code units of K (or V) a stage
    static constexpr int kN = kUnits / kThreads;           // of them a thread moves
    static constexpr int kRows = 16 * NT * kWaves;
    static constexpr int kQl = D == 256 && NT == 2 ? 3 : 0;  // steps of the queries kept in LDS, likewise
};
template <int D, int NT>
__global__ void __launch_bounds__((Kv8Tile<D, NT>::kThreads), 2)
kv8_tile_kernel(Kv8AttnArgs p, int tiles, int streams) {
    using C = Kv8Tile<D, NT>;
    __shared__ __align__(16) half8_t buf[2][4 * C::kUnits];  // K's halves, then V's
    __shared__ __align__(16) half8_t qs[C::kQl ? C::kWaves : 1][C::kQl ? C::kQl * NT : 1][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g4 = lane >> 4, n = lane & 15;
    const Kv8& c = p.c;
    // Workgroups go round the 8 XCDs.  The tiles of one (head, split) read the same keys: they go to
    // one XCD, the last (longest) tiles of its heads first, or where the heads and splits are no
    // multiple of 8, each XCD takes an eighth of all in a row.
    int stream, rank;
    const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
    if ((streams & 7) == 0) {
        const int per = streams >> 3;
        stream = xcd * per + slot % per;
        rank = slot / per;
    } else {
        const int at = xcd * (int)(gridDim.x >> 3) + slot;
        if (at >= streams * tiles) return;
        stream = at / tiles;
        rank = at % tiles;
    }
    const int tile = tiles - 1 - rank, bh = stream / p.nsplit, split = stream % p.nsplit;
    const int b = bh / c.Hkv, h = bh % c.Hkv;
    const Kv8Seq sq = kv8_seq(c, p.len, p.n_new, b, p.T);
    const int front = sq.len - (sq.n + sq.t0);  // position of row t = 0
    const int row_end = min(p.T, sq.n + sq.t0) * p.G;
    if (tile * C::kRows >= row_end) return;

    Kv8Rows<D> st[NT];
    const int row0 = tile * C::kRows + wave * 16 * NT;
    int see, least;
    kv8_begin<D, NT>(st, p, sq, b, h, row0, row_end, see, least);
    // the last key that any row of the workgroup sees
    const int all = p.causal ? min(front + (min(row_end, (tile + 1) * C::kRows) - 1) / p.G, sq.len - 1) : sq.len - 1;
    const int nb = all < 0 ? 0 : all / kKvBlock + 1;
    const int n_full = min(sq.len / kKvBlock, nb);
    const int per = (nb + p.nsplit - 1) / p.nsplit;
    const int end = min(nb, (split + 1) * per);
    const bool open = split * per <= n_full && n_full < end;
    Kv8Walk<false> walk = {split * per, min(end, n_full), 1, n_full, n_full, 0, 0};
    int blk = 0, page = -1, part = 0;
    Kv8Scale sc = {};
    auto next = [&]() {
        if (!walk.next(c, b, h, nullptr, p.c2, blk, page, sc)) page = -1;
    };

    struct Stage {
        int p0;  // first key, -1: none
        Kv8Scale sc;
    };
    uint4 rk[C::kN], rv[C::kN];
    auto load = [&]() -> Stage {  // codes of the stage at (page, part) to registers, and on to the next
        if (page < 0) return {-1, {}};
        const size_t head = (size_t)page * c.Hkv + h;
        const uint4* kp = reinterpret_cast<const uint4*>(c.k + head * (kKvBlock * D)) + part * C::kUnits + tid;
        const uint4* vp = reinterpret_cast<const uint4*>(c.v + head * (kKvBlock * D)) + part * C::kUnits + tid;
#pragma unroll
        for (int x = 0; x < C::kN; ++x) rk[x] = kp[x * C::kThreads];
#pragma unroll
        for (int x = 0; x < C::kN; ++x) rv[x] = vp[x * C::kThreads];
        const Stage s = {blk * kKvBlock + part * C::kKeys, sc};
        if (++part == C::kParts) {
            part = 0;
            next();
        }
        return s;
    };
    // Unit x of the registers (K's, then V's) to LDS as fp16.
    auto store = [&](int to, int x) {
        const bool isv = x >= C::kN;
        const uint4& r = isv ? rv[x - C::kN] : rk[x];
        half8_t* at = &buf[to][(isv ? 2 * C::kUnits : 0) + ((tid >> 6) + C::kWaves * (isv ? x - C::kN : x)) * 128 + lane];
        at[0] = kv8_halves(r.x, r.y);
        at[64] = kv8_halves(r.z, r.w);
    };
    auto store_all = [&](int to) {
#pragma unroll
        for (int x = 0; x < 2 * C::kN; ++x) store(to, x);
    };
    next();
    Stage now = load();
    if (now.p0 >= 0) store_all(0);
    Stage then = load();
    kv8_arrived<D, NT>(st);
    half8_t* ql = &qs[C::kQl ? wave : 0][0][lane];  // a wave reads its own only
#pragma unroll
    for (int x = 0; x < C::kQl; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) ql[(x * NT + nt) * 64] = st[nt].q[D / 32 - C::kQl + x];
    lds_barrier();
    for (int u = 0; now.p0 >= 0; u ^= 1) {
        const half8_t* kb = &buf[u][lane];
        const half8_t* vb = kb + 2 * C::kUnits;
        // The next stage's codes are converted among the products of K's operands, and the one after
        // that is sent for behind them.  (Behind the last stage the registers hold old codes; what
        // is written is not read.)  A wave that sees none of the stage's keys, on the diagonal, runs
        // them masked: a branch round the products would cost it a copy of all its sums.
        kv8_lds_keys<D, NT, C::kKeys / 16, C::kQl>(st, now.p0, now.sc, now.p0 + C::kKeys - 1 > least, kb, vb, ql, [&](int e) {
            constexpr int kOps = C::kKeys / 16 * (D / 32), kEvery = kOps / (4 * C::kN);
            if (e % kEvery == kEvery - 1 && e / kEvery < 2 * C::kN) store(u ^ 1, e / kEvery);
        });
        const Stage after = load();
        lds_barrier();
        now = then;
        then = after;
    }
    if (open && see >= n_full * kKvBlock) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            kv8_queries<D>(st[nt], p, b, h, row0 + 16 * nt, row_end);  // again: not held through the loop's end
            kv8_open_block<D>(st[nt], c, b, h, n_full, sq.len - n_full * kKvBlock, p.c2);
        }
    }

#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float l = sum_xor32(sum_xor16(st[nt].l));
        const int row = row0 + 16 * nt + n;
        if (row >= row_end) continue;
        if (p.nsplit > 1) {
            if (l != 0.f) {
                float* at = kv8_part<D>(p, bh, row, split) + 4 * g4;
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<float4_t*>(at + 16 * dt) = st[nt].o[dt];
            }
            if (g4 == 0) *reinterpret_cast<float2*>(kv8_pair<D>(p, bh, row, split)) = float2{st[nt].m, l};
        } else {
            const int t = row / p.G, hq = h * p.G + row % p.G;
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt)
                kv8_store4(p, b, hq, t, 16 * dt + 4 * g4, st[nt].o[dt], l, kv8_gate4(p, b, hq, t, 16 * dt + 4 * g4));
        }
    }
}

// Joins the splits of 1024 / D rows: workgroup (rows, b Hkv + h), D / 4 lanes a row.  Every address
// is known at once, so that the loads wait for memory together and not for each other: a row's
// maxima and sums, its first splits' sums (unread where they were not written), its gate.
template <int D>
__global__ void __launch_bounds__(256)
kv8_join_kernel(Kv8AttnArgs p) {
    constexpr int kLanes = D / 4, kRows = 256 / kLanes, kAhead = 16;
    __shared__ float fs[kRows][kKvMaxSplits];
    const Kv8& c = p.c;
    const int b = blockIdx.y / c.Hkv, h = blockIdx.y % c.Hkv;
    const int r = threadIdx.x / kLanes, x = threadIdx.x % kLanes, n_rows = p.T * p.G;
    const int row = min((int)blockIdx.x * kRows + r, n_rows - 1);
    const float2* pair = reinterpret_cast<const float2*>(kv8_pair<D>(p, blockIdx.y, row, 0));
    const float4_t* at = reinterpret_cast<const float4_t*>(kv8_part<D>(p, blockIdx.y, row, 0)) + x;
    float2 ml[kKvMaxSplits / kLanes];
#pragma unroll
    for (int i = 0; i < kKvMaxSplits / kLanes; ++i) ml[i] = pair[min(x + i * kLanes, p.nsplit - 1)];
    float4_t part[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) part[s] = at[(size_t)min(s, p.nsplit - 1) * (D / 4)];
    const int t = row / p.G, hq = h * p.G + row % p.G;
    const half4_t gate = kv8_gate4(p, b, hq, t, 4 * x);
    const Kv8Seq sq = kv8_seq(c, p.len, p.n_new, b, p.T);
    const bool is = (int)blockIdx.x * kRows + r < n_rows && t < sq.n + sq.t0;  // rows of padding have no sums
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kKvMaxSplits / kLanes; ++i) {
        if (x + i * kLanes >= p.nsplit) ml[i] = float2{-INFINITY, 0.f};
        m = fmaxf(m, ml[i].x);
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
#pragma unroll
    for (int i = 0; i < kKvMaxSplits / kLanes; ++i) {
        float f = ml[i].y == 0.f ? 0.f : ml[i].x == m ? 1.f : fast_exp2(ml[i].x - m);
        if (ml[i].y != ml[i].y) f = ml[i].y;  // a row of NaN, whatever its maximum
        l += ml[i].y == 0.f ? 0.f : f * ml[i].y;
        if (x + i * kLanes < p.nsplit) fs[r][x + i * kLanes] = f;
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) l += __shfl_xor(l, o);
    __syncthreads();
    if (!is) return;
    float4_t y = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](const float4_t& v, float f) {
        if (f != 0.f) y += v * f;  // sums that no key went into were not written
    };
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
        if (s < p.nsplit) add(part[s], fs[r][s]);
    for (int s0 = kAhead; s0 < p.nsplit; s0 += kAhead) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s) part[s] = at[(size_t)min(s0 + s, p.nsplit - 1) * (D / 4)];
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
            if (s0 + s < p.nsplit) add(part[s], fs[r][s0 + s]);
    }
    kv8_store4(p, b, hq, t, 4 * x, y, l, gate);
}

// How a call's rows are cut into tiles and its keys into splits.
struct Kv8Plan {
    int rows;       // of a tile
    long long tiles;  // of one K/V head
    int nsplit;
};
// One tile of 16 rows where there are no more (and for listed blocks, one query's heads), else
// workgroups of 64, or of 128 (256 at D = 256) rows.  items: blocks of the longest sequence, or of a list.
inline Kv8Plan kv8_plan(int B, int T, int Hq, int Hkv, int D, int items, bool list) {
    const long long G = Hq / Hkv, rows = T * G;
    Kv8Plan q;
    q.rows = list || rows <= 16 ? 16 : rows <= 64 ? 64 : D == 256 ? 256 : 128;
    q.tiles = list ? T * ((G + 15) / 16) : (rows + q.rows - 1) / q.rows;
    const long long all = q.tiles * B * Hkv;
    // row tiles: as many workgroups as the chip takes twice, not fewer than 4 blocks each; the others
    // as many as it takes once
    const long long want = q.rows == 16 ? (1024 + all - 1) / all : (q.rows == 256 ? 256 : 512) / all;
    const long long most = (items + 3) / 4;
    const long long n = want < most ? want : most;
    q.nsplit = (int)(n < 1 ? 1 : n < kKvMaxSplits ? n : kKvMaxSplits);
    return q;
}
inline size_t kv8_part_bytes(int B, int T, int Hq, int D, int nsplit) {
    return nsplit > 1 ? (size_t)B * T * Hq * nsplit * (D + 2) * 4 : 0;
}

template <int D, bool kList>
hipError_t kv8_attn_d(const Kv8AttnArgs& p, const Kv8Plan& q, hipStream_t stream) {
    const int BH = p.c.B * p.c.Hkv;
    if (kList || q.rows == 16) {
        const dim3 grid((unsigned)q.tiles, (unsigned)BH, (unsigned)p.nsplit);
        hipLaunchKernelGGL((kv8_row_kernel<D, kList>), grid, dim3(256), 0, stream, p);
    } else {
        const dim3 grid((unsigned)((q.tiles * BH * p.nsplit + 7) / 8 * 8));
        if (q.rows == 64)
            hipLaunchKernelGGL((kv8_tile_kernel<D, 1>), grid, dim3(Kv8Tile<D, 1>::kThreads), 0, stream, p, (int)q.tiles, BH * p.nsplit);
        else
            hipLaunchKernelGGL((kv8_tile_kernel<D, 2>), grid, dim3(Kv8Tile<D, 2>::kThreads), 0, stream, p, (int)q.tiles, BH * p.nsplit);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.nsplit == 1) return e;
    constexpr int kRows = 1024 / D;
    const dim3 rows((unsigned)((p.T * p.G + kRows - 1) / kRows), (unsigned)BH);
    hipLaunchKernelGGL(kv8_join_kernel<D>, rows, dim3(256), 0, stream, p);
    return hipGetLastError();
}
template <bool kList>
hipError_t kv8_attn_any(const Kv8AttnArgs& p, const Kv8Plan& q, hipStream_t stream) {
    if (p.c.D == 64) return kv8_attn_d<64, kList>(p, q, stream);
    if (p.c.D == 128) return kv8_attn_d<128, kList>(p, q, stream);
    return kv8_attn_d<256, kList>(p, q, stream);
}

}  // namespace

hipError_t kv8_attn(const Kv8& c, const Rows16& q, const Rows16& gate, const Rows16& o, const int* len, const int* n_new,
                    int T, int Hq, int nb_hint, float scale, int causal, void* ws, hipStream_t stream) {
    const Kv8Plan plan = kv8_plan(c.B, T, Hq, c.Hkv, c.D, nb_hint, false);
    return kv8_attn_any<false>({c, q, gate, o, len, n_new, nullptr, (float*)ws, T, Hq, Hq / c.Hkv, 0, plan.nsplit, causal, scale * kLog2e},
                               plan, stream);
}

hipError_t kv8_attn_blocks(const Kv8& c, const Rows16& q, const Rows16& gate, const Rows16& o, const int* len,
                           const int* n_new, int T, int Hq, const int* blocks, int top, float scale, void* ws,
                           hipStream_t stream) {
    const Kv8Plan plan = kv8_plan(c.B, T, Hq, c.Hkv, c.D, top, true);
    return kv8_attn_any<true>({c, q, gate, o, len, n_new, blocks, (float*)ws, T, Hq, Hq / c.Hkv, top, plan.nsplit, 1, scale * kLog2e}, plan,
                              stream);
}

}  // namespace tsa
