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
    float *part, *pair;  // split keys: D sums for each slot (see kv8_slot), and a pair (m, l)
    int T, Hq, G, top, nsplit, causal;
    int share;  // above 0: the keys of all sequences are dealt to so many workgroups a head (Kv8Deal)
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

// The full blocks of a wave's work, in turn.  Each lane looks one of the next 64 items up (part
// item % kParts of a block: an entry of the list, or item / kParts itself; its page; its scales), so
// that a block's are lane reads and no load waits for another but once in 64 items.
template <bool kList, int kParts>
struct Kv8Walk {
    int item, end, step;   // the next 64 are item + step * lane, below end
    int nb, n_full;        // blocks that are seen, and the full ones of them
    int open;              // how often the open block came up
    unsigned long long todo;
    int blks, pages;       // of this lane's item
    Kv8Scale scales;

    __device__ __forceinline__ void look(const Kv8& c, int b, int h, const int* list, float c2) {
        const int i = item + step * (int)(threadIdx.x & 63);
        blks = i < end ? (kList ? list[i / kParts] : i / kParts) : -1;
        // the open block is taken whole, with its first part
        if (kList || n_full < nb) open += __popcll(__ballot(blks >= n_full && blks < nb && i % kParts == 0));
        const bool is = blks >= 0 && blks < n_full;
        pages = is ? kv8_page(c, b, blks) : -1;
        const size_t head = (size_t)max(pages, 0) * c.Hkv + h;
        const float sk = c.k_scale[head], sv = c.v_scale[head];
        scales = {c2 * sk, __builtin_amdgcn_logf(sv), __builtin_amdgcn_rcpf(sv)};
        todo = __ballot(pages >= 0);
        item += 64 * step;
    }
    // The next block; false when there is none.
    __device__ __forceinline__ bool next(const Kv8& c, int b, int h, const int* list, float c2, int& blk, int& part, int& page,
                                         Kv8Scale& sc) {
        while (todo == 0) {
            if (item >= end) return false;
            look(c, b, h, list, c2);
        }
        const int l = __builtin_ctzll(todo);
        todo &= todo - 1;
        part = (item - 64 * step + l * step) % kParts;
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
    if (masked && !(sc.f > 0.f && sc.lsv == sc.lsv)) {  // a key that is not seen weighs 0 (-inf times NaN, or times a factor that underflowed)
        int again = left;
        asm volatile("" : "+v"(again));  // compared here, and not kept from above on every path
#pragma unroll
        for (int a = 0; a < KA; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) w[a][r] = 16 * a + r <= again ? w[a][r] : 0.f;
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

// The same in two parts from operands in LDS (kb, vb: this lane's of K and V), read kAhead before
// their products.  Scores: between(e) is called among the products.
template <int D, int NT, int KA, int kAhead, class Between>
__device__ __forceinline__ void kv8_lds_scores(const Kv8Rows<D> (&st)[NT], float4_t (&w)[NT][KA], const half8_t* kb, Between between) {
    constexpr int kOps = KA * (D / 32);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int a = 0; a < KA; ++a) w[nt][a] = float4_t{0.f, 0.f, 0.f, 0.f};
    half8_t op[kOps];
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
            w[nt][e % KA] = mfma16(op[e], st[nt].q[e / KA], w[nt][e % KA]);
        between(e);
        __builtin_amdgcn_sched_barrier(0);
    }
}
// Sums: p are the weights of key steps of 32.
template <int D, int NT, int KS, int kAhead>
__device__ __forceinline__ void kv8_lds_sums(Kv8Rows<D> (&st)[NT], const half8_t (&p)[NT][KS], const half8_t* vb) {
    constexpr int kOps = KS * (D / 16);
    half8_t op[kOps];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) op[e] = vb[e * 64];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < kOps; ++e) {  // (s, m, o) in order
        if (e + kAhead < kOps) op[e + kAhead] = vb[(e + kAhead) * 64];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) st[nt].o[e % (D / 16)] = mfma16(op[e], p[nt][e / (D / 16)], st[nt].o[e % (D / 16)]);
        __builtin_amdgcn_sched_barrier(0);
    }
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
            float4_t more[4] = {};  // (not on the sums themselves, which are to stay in place)
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
                        if (kv8_bad(z)) more[x][e] += wj * (float)z;
                    }
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) st.o[2 * m + x] += more[x];
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
// The last key that query row t G + g sees.  A row in front of position 0 sees none, causal or not.
__device__ __forceinline__ int kv8_limit(const Kv8AttnArgs& p, const Kv8Seq& sq, int row) {
    const int pos = sq.len - (sq.n + sq.t0) + row / p.G;
    return pos < 0 ? -1 : p.causal ? min(pos, sq.len - 1) : sq.len - 1;
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
        st[nt].limit = is ? kv8_limit(p, sq, row) : -1;
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

// Where a split's sums of a row lie: slot [row of all][split], or where all sequences' keys are dealt
// out [head][segment][row], workgroup w's segment of sequence b being w + b.
__device__ __forceinline__ size_t kv8_slot(const Kv8AttnArgs& p, size_t bh, int row, int split) {
    return (bh * p.T * p.G + row) * p.nsplit + split;
}
__device__ __forceinline__ size_t kv8_dealt_slot(const Kv8AttnArgs& p, int h, int seg, int row) {
    return ((size_t)h * (p.share + p.c.B) + seg) * (p.T * p.G) + row;
}
template <int D>
__device__ __forceinline__ float* kv8_part(const Kv8AttnArgs& p, size_t slot) {
    return p.part + slot * D;
}
__device__ __forceinline__ float2* kv8_pair(const Kv8AttnArgs& p, size_t slot) { return reinterpret_cast<float2*>(p.pair) + slot; }

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
template <int D, bool kOnce>
struct Kv8Regs {
    static constexpr int kKeys = D == 256 ? 32 : 64, kN = kKeys * D / 1024;
    uint4 k[kN], v[kN];

    __device__ __forceinline__ void load_k(const Kv8& c, int page, int h, int part) {
        const size_t head = (size_t)page * c.Hkv + h;
        const uint4* kp = reinterpret_cast<const uint4*>(c.k + head * (kKvBlock * D)) + part * (kN * 64) + (threadIdx.x & 63);
#pragma unroll
        for (int i = 0; i < kN; ++i) k[i] = kv8_codes<kOnce>(kp + i * 64);
    }
    __device__ __forceinline__ void load_v(const Kv8& c, int page, int h, int part) {
        const size_t head = (size_t)page * c.Hkv + h;
        const uint4* vp = reinterpret_cast<const uint4*>(c.v + head * (kKvBlock * D)) + part * (kN * 64) + (threadIdx.x & 63);
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = kv8_codes<kOnce>(vp + i * 64);
    }
};

constexpr int kKvMaxSplits = 128;

// Which tile, (sequence, head) and split a workgroup of the kernels below has.  Workgroups go round
// the 8 XCDs.  The tiles of one (head, split) read the same keys: they go to one XCD, the last
// (longest) tiles of its heads first, or where the heads and splits are no multiple of 8, each XCD
// takes an eighth of all in a row.
struct Kv8Place {
    int tile, bh, b, h, split;
    __device__ __forceinline__ bool find(const Kv8AttnArgs& p, int tiles, int streams) {
        int stream, rank;
        const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
        if ((streams & 7) == 0) {
            const int per = streams >> 3;
            stream = xcd * per + slot % per;
            rank = slot / per;
        } else {
            const int at = xcd * (int)(gridDim.x >> 3) + slot;
            if (at >= streams * tiles) return false;
            stream = at / tiles;
            rank = at % tiles;
        }
        tile = tiles - 1 - rank;
        bh = stream / p.nsplit;
        split = stream % p.nsplit;
        b = bh / p.c.Hkv;
        h = bh % p.c.Hkv;
        return true;
    }
};

// The blocks of a split of a tile of rows [first, end): those that some row sees, shared out.
struct Kv8Share {
    int n_full;   // full blocks that are seen
    bool open;    // the open block is this split's
    Kv8Walk<false, 1> walk;
    __device__ __forceinline__ void find(const Kv8AttnArgs& p, const Kv8Seq& sq, int last_row, int split) {
        const int front = sq.len - (sq.n + sq.t0);  // position of row t = 0
        const int all = p.causal ? min(front + last_row / p.G, sq.len - 1) : sq.len - 1;
        const int nb = all < 0 ? 0 : all / kKvBlock + 1;
        n_full = min(sq.len / kKvBlock, nb);
        const int per = (nb + p.nsplit - 1) / p.nsplit, end = min(nb, (split + 1) * per);
        open = split * per <= n_full && n_full < end;
        walk = {split * per, min(end, n_full), 1, n_full, n_full, 0, 0};
    }
};

// A wave's finished rows, or a split's sums of them.
template <int D, int NT>
__device__ __forceinline__ void kv8_finish(Kv8Rows<D> (&st)[NT], const Kv8AttnArgs& p, const Kv8Place& at, int row0, int row_end) {
    const int lane = threadIdx.x & 63, g4 = lane >> 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float l = sum_xor32(sum_xor16(st[nt].l));
        const int row = row0 + 16 * nt + (lane & 15);
        if (row >= row_end) continue;
        if (p.nsplit > 1) {
            if (l != 0.f) {
                float* part = kv8_part<D>(p, kv8_slot(p, at.bh, row, at.split)) + 4 * g4;
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<float4_t*>(part + 16 * dt) = st[nt].o[dt];
            }
            if (g4 == 0) *kv8_pair(p, kv8_slot(p, at.bh, row, at.split)) = float2{st[nt].m, l};
        } else {
            const int t = row / p.G, hq = at.h * p.G + row % p.G;
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt)
                kv8_store4(p, at.b, hq, t, 16 * dt + 4 * g4, st[nt].o[dt], l, kv8_gate4(p, at.b, hq, t, 16 * dt + 4 * g4));
        }
    }
}

// All sequences' keys dealt out: one head's, in the order of the sequences, are cut into as many
// workgroups' as the chip takes, so that all of them have as much to do whatever the lengths are (24/4
// heads, D = 256: 32 sequences of 16385 to 32768 keys 283 us with 8 splits each, 264 dealt out; 24 of
// 32768, 272 and 259; 32 of 24576, 250 both).  They are counted in rounds, in which each of a
// workgroup's 4 waves takes a part; a sequence has one at least, and no more than kKvMaxSplits segments.
template <int kParts>
struct Kv8Deal {
    int groups, per, odd;  // workgroups; rounds of each, the first `odd` having one more
    int total, before;     // rounds of all sequences, of those before one
    int lane_own, lane_end;  // a lane's sequence's rounds, and those up to its end

    static __device__ __forceinline__ int rounds(const Kv8AttnArgs& p, int b) {
        const int n = p.n_new ? min(max(p.n_new[b], 0), p.T) : p.T;
        const int len = min(max(p.len[b], 0), p.c.max_blocks * kKvBlock);
        return n > 0 ? max(((len + kKvBlock - 1) / kKvBlock * kParts + 3) / 4, 1) : 0;
    }
    // 64 sequences from b0 on; the rounds of all of them.
    __device__ __forceinline__ int look(const Kv8AttnArgs& p, int b0) {
        const int lane = threadIdx.x & 63;
        lane_own = b0 + lane < p.c.B ? rounds(p, b0 + lane) : 0;
        lane_end = lane_own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int z = __shfl_up(lane_end, o);
            lane_end += lane >= o ? z : 0;
        }
        return __builtin_amdgcn_readlane(lane_end, 63);
    }
    __device__ __forceinline__ void find(const Kv8AttnArgs& p) {
        int most = 0;
        total = 0;
        for (int b0 = 0; b0 < p.c.B; b0 += 64) {
            total += look(p, b0);
            most = max(most, lane_own);
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o));
        most = __builtin_amdgcn_readfirstlane(most);
        groups = max(1, min(p.share, total / max(2, (most + kKvMaxSplits - 3) / (kKvMaxSplits - 2))));
        per = total / groups;
        odd = total % groups;
    }
    // The first round of a workgroup, and the workgroup of a round.
    __device__ __forceinline__ int front(int w) const { return w * per + min(w, odd); }
    __device__ __forceinline__ int group(int x) const {
        const int y = odd * (per + 1);
        return x < y ? x / (per + 1) : odd + (x - y) / max(per, 1);
    }
    // The sequence that a round (below total) is of; `before` is its own.
    __device__ __forceinline__ int seek(const Kv8AttnArgs& p, int x) {
        before = 0;
        for (int b0 = 0;; b0 += 64) {
            const int all = p.c.B > 64 ? look(p, b0) : total;
            const unsigned long long is = __ballot(before + lane_end > x);
            if (is != 0) {
                const int l = __builtin_ctzll(is);
                before += __builtin_amdgcn_readlane(lane_end - lane_own, l);
                return b0 + l;
            }
            if (b0 + 64 >= p.c.B) return p.c.B;  // (the lengths changed under the call)
            before += all;
        }
    }
    // The rounds of sequence b; `before` is its own.
    __device__ __forceinline__ int own(const Kv8AttnArgs& p, int b) {
        before = 0;
        for (int b0 = 0;; b0 += 64) {
            const int all = p.c.B > 64 ? look(p, b0) : total;
            if (b < b0 + 64) {
                before += __builtin_amdgcn_readlane(lane_end - lane_own, b - b0);
                return __builtin_amdgcn_readlane(lane_own, b - b0);
            }
            before += all;
        }
    }
};

// Few rows: tiles of 16 query rows of a K/V head's group over one split of their blocks, a stage of
// keys (half a block at D = 256, else a block) at a time.  A wave's next keys are on their way to
// registers as soon as its last ones have been multiplied, its next values likewise.
// kWaves = 4: a workgroup is one tile and split, the stages dealt to its waves in turn and their
// sums joined; 1: a wave is a tile by itself, and nothing is joined.
// kList: a tile is one query's heads (16 at a time) over its listed blocks; otherwise rows are
// t G + g over all the sequence's blocks.  Neighbouring queries share most of their listed blocks:
// an eighth of all tiles in a row goes to each XCD (workgroups go round them), whose L2 then serves
// the blocks again (700 queries of 16 blocks, 24/4 heads, D = 256: 115 -> 109 us; a wave a tile 102).
// Bound by memory with one query a sequence (32 of 16385 to 32768 keys, D = 256: 264 us, 6.1 TB/s);
// where queries share their blocks by the vector instructions that turn codes into fp16.
// kDeal: all sequences' keys are dealt out, and a workgroup goes through its segments.
template <int D, bool kList, int kWaves, bool kDeal>
__global__ void __launch_bounds__(256, 2)
kv8_row_kernel(Kv8AttnArgs p, int tiles) {
    using Regs = Kv8Regs<D, !kList>;
    constexpr int kParts = kKvBlock / Regs::kKeys, kRow = D + 4;
    __shared__ __align__(16) float acc[kWaves == 4 ? 2 : 1][kWaves == 4 ? 16 : 1][kRow];
    __shared__ float ml[4][2][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g4 = lane >> 4, n = lane & 15;
    const Kv8& c = p.c;
    int at = blockIdx.x;
    if constexpr (kList) at = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
    if constexpr (kWaves == 1) at = 4 * at + wave;
    int tile = 0, b, h, split = 0, bh = 0;
    Kv8Deal<kParts> deal;
    int from = 0, to = 0;  // this workgroup's rounds
    if constexpr (kDeal) {
        h = at % c.Hkv;
        deal.find(p);
        // neighbours an eighth of the keys apart (next to each other 268 us for the 32 sequences, 264)
        split = at / c.Hkv;
        split = split % 8 * (p.share / 8) + split / 8;
        if (split >= deal.groups) return;
        from = deal.front(split);
        to = deal.front(split + 1);
        if (from == to) return;
        b = deal.seek(p, from);
        if (b >= c.B) return;
    } else {
        if (at >= tiles * c.B * c.Hkv * p.nsplit) return;
        tile = at % tiles, bh = at / tiles % (c.B * c.Hkv), split = at / tiles / (c.B * c.Hkv);
        b = bh / c.Hkv, h = bh % c.Hkv;
    }
    for (;;) {  // segments of a deal, else once
        const Kv8Seq sq = kv8_seq(c, p.len, p.n_new, b, p.T);
        int row0, row_end;
        if constexpr (kList) {
            const int per = (p.G + 15) / 16, t = tile / per;
            row0 = t * p.G + tile % per * 16;
            row_end = (t + 1) * p.G;
        } else {
            row0 = tile * 16;
            row_end = p.T * p.G;
        }
        row_end = min(row_end, (sq.n + sq.t0) * p.G);
        if (!kDeal && row0 >= row_end) return;

        Kv8Rows<D> rows[1], &st = rows[0];
        int see, least;
        kv8_begin<D, 1>(rows, p, sq, b, h, row0, row_end, see, least);
        const int nb = see / kKvBlock + (see >= 0 ? 1 : 0);  // blocks that any row sees
        const int n_full = min(sq.len / kKvBlock, nb);
        const int items = (kList ? p.top : nb) * kParts;
        int begin, end;
        if constexpr (kDeal) {
            begin = max(from - deal.before, 0) * 4;
            end = min((to - deal.before) * 4, items);
        } else {
            const int per = (items + p.nsplit - 1) / p.nsplit;
            begin = split * per;
            end = min(items, begin + per);
        }
        const int* list = kList ? p.blocks + (((size_t)b * c.Hkv + h) * p.T + row0 / p.G) * p.top : nullptr;
        Kv8Walk<kList, kParts> walk = {begin + (kWaves == 4 ? wave : 0), end, kWaves, nb, n_full, 0, 0};
        int blk = 0, part = 0, page = -1;
        Kv8Scale sc = {};
        auto next = [&]() {
            if (!walk.next(c, b, h, list, p.c2, blk, part, page, sc)) page = -1;
        };
        next();
        if (page >= 0) {
            Regs x;
            x.load_k(c, page, h, part);
            x.load_v(c, page, h, part);
            kv8_arrived<D, 1>(rows);
            while (page >= 0) {
                // rows of one query see whole blocks but the last; several queries' last one or two are masked
                const int p0 = blk * kKvBlock + part * Regs::kKeys;
                const Kv8Scale scale = sc;
                next();
                kv8_keys<D, 1, Regs::kKeys / 16>(
                    rows, p0, scale, p0 + Regs::kKeys - 1 > least,
                    [&](int a, int i, int s) {
                        const uint4& k = x.k[a * (D / 64) + i];
                        return s ? kv8_halves(k.z, k.w) : kv8_halves(k.x, k.y);
                    },
                    [&](int s, int m, int o) {
                        const uint4& v = x.v[s * (D / 32) + m];
                        return o ? kv8_halves(v.z, v.w) : kv8_halves(v.x, v.y);
                    },
                    [&]() {
                        if (page >= 0) x.load_k(c, page, h, part);
                    });
                if (page >= 0) x.load_v(c, page, h, part);
            }
        }
        for (; walk.open > 0; --walk.open) kv8_open_block<D>(st, c, b, h, n_full, sq.len - n_full * kKvBlock, p.c2);

        if constexpr (kWaves == 1) {
            kv8_finish<D, 1>(rows, p, {tile, bh, b, h, split}, row0, row_end);
            return;
        }
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
            if (kDeal || p.nsplit > 1) {
                const size_t slot = kDeal ? kv8_dealt_slot(p, h, split + b, row0 + r) : kv8_slot(p, bh, row0 + r, split);
                if (l != 0.f) *reinterpret_cast<float4_t*>(kv8_part<D>(p, slot) + d) = y;
                if (d == 0) *kv8_pair(p, slot) = float2{m, l};
            } else {
                const int t = (row0 + r) / p.G, hq = h * p.G + (row0 + r) % p.G;
                kv8_store4(p, b, hq, t, d, y, l, kv8_gate4(p, b, hq, t, d));
            }
        }
        if constexpr (!kDeal) return;
        do {  // the next sequence, if any of its rounds are this workgroup's
            deal.before += Kv8Deal<kParts>::rounds(p, b);
            if (deal.before >= to) return;
            if (++b >= c.B) return;
        } while (Kv8Deal<kParts>::rounds(p, b) == 0);
        __syncthreads();
    }
}

// A stage of keys on its way from memory to LDS.
struct Kv8Stage {
    int p0 = -1;  // first key, -1: none
    int page = 0, part = 0;
    Kv8Scale sc = {};
};
// The next stage of a walk in parts of kParts a block.
template <int kParts, class Walk>
__device__ __forceinline__ void kv8_step(Kv8Stage& s, Walk& walk, const Kv8& c, int b, int h, float c2) {
    if (s.p0 >= 0 && s.part + 1 < kParts) {
        s.p0 += kKvBlock / kParts;
        ++s.part;
        return;
    }
    int blk, part;
    s.p0 = walk.next(c, b, h, nullptr, c2, blk, part, s.page, s.sc) ? blk * kKvBlock : -1;
    s.part = 0;
}

// More rows than a tile: a workgroup is 4 waves of 16 NT query rows each over one split of their
// blocks.  A stage of kKeys keys and their values (16 KiB of codes at the most) goes from memory to
// registers, is turned into fp16 operands once for all waves, and lies in one of two LDS buffers in
// operand order, so every LDS access is 16 consecutive bytes a lane and a code is converted once
// per 64 NT rows.  One barrier a stage.  Two sets of registers are filled in turn, three stages
// ahead of their use: 18 rows over 8 sequences of 16384, 24/4 heads, D = 256, need the bandwidth
// (one set 68 us, two, past the caches, 65).
template <int D, int NT>
struct Kv8Tile {
    static constexpr int kKeys = D == 256 ? 32 : 64, kParts = kKvBlock / kKeys;
    static constexpr int kUnits = kKeys * D / 16;  // 16-code units of K (or V) a stage
    static constexpr int kN = kUnits / 256;        // of them a thread moves
    static constexpr int kRows = 64 * NT;
};
// kOnce: a (sequence, head) is one tile.
template <int D, int NT, bool kOnce>
__global__ void __launch_bounds__(256, 2)
kv8_tile_kernel(Kv8AttnArgs p, int tiles, int streams) {
    using C = Kv8Tile<D, NT>;
    constexpr int KA = C::kKeys / 16, kAhead = D == 256 ? 3 : 6;
    __shared__ __align__(16) half8_t buf[2][4 * C::kUnits];  // K's halves, then V's
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Kv8& c = p.c;
    Kv8Place at;
    if (!at.find(p, tiles, streams)) return;
    const Kv8Seq sq = kv8_seq(c, p.len, p.n_new, at.b, p.T);
    const int row_end = min(p.T, sq.n + sq.t0) * p.G;
    if (at.tile * C::kRows >= row_end) return;

    Kv8Rows<D> st[NT];
    const int row0 = at.tile * C::kRows + wave * 16 * NT;
    int see, least;
    kv8_begin<D, NT>(st, p, sq, at.b, at.h, row0, row_end, see, least);
    Kv8Share share;
    share.find(p, sq, min(row_end, (at.tile + 1) * C::kRows) - 1, at.split);

    struct Set {
        uint4 k[C::kN], v[C::kN];
    } r[2];
    auto load = [&](Set& x, const Kv8Stage& s) {
        if (s.p0 < 0) return;
        const size_t head = (size_t)s.page * c.Hkv + at.h;
        const uint4* kp = reinterpret_cast<const uint4*>(c.k + head * (kKvBlock * D)) + s.part * C::kUnits + tid;
        const uint4* vp = reinterpret_cast<const uint4*>(c.v + head * (kKvBlock * D)) + s.part * C::kUnits + tid;
#pragma unroll
        for (int i = 0; i < C::kN; ++i) x.k[i] = kv8_codes<kOnce>(kp + i * 256);
#pragma unroll
        for (int i = 0; i < C::kN; ++i) x.v[i] = kv8_codes<kOnce>(vp + i * 256);
    };
    // Unit i of a set (K's, then V's) to LDS as fp16.
    auto store = [&](int to, const Set& x, int i) {
        const bool isv = i >= C::kN;
        const uint4& y = isv ? x.v[i - C::kN] : x.k[i];
        half8_t* u = &buf[to][(isv ? 2 * C::kUnits : 0) + ((tid >> 6) + 4 * (isv ? i - C::kN : i)) * 128 + lane];
        u[0] = kv8_halves(y.x, y.y);
        u[64] = kv8_halves(y.z, y.w);
    };
    // The stages, `now` in buffer 0 and the next two in the sets.  One behind the last keeps its
    // scales and has no key that a row sees.
    constexpr int kNone = INT_MAX / 2;
    Kv8Stage now, next[2];
    auto step = [&](Kv8Stage& s) { kv8_step<C::kParts>(s, share.walk, c, at.b, at.h, p.c2); };
    step(now);
    if (now.p0 >= 0) {
        load(r[0], now);
#pragma unroll
        for (int i = 0; i < 2 * C::kN; ++i) store(0, r[0], i);
        next[0] = now;
        step(next[0]);
        load(r[0], next[0]);
        next[1] = next[0];
        if (next[0].p0 >= 0) step(next[1]);
        load(r[1], next[1]);
        kv8_arrived<D, NT>(st);
        lds_barrier();
        do {
#pragma unroll
            for (int u = 0; u < 2; ++u) {  // the stage in buffer u
                const half8_t* kb = &buf[u][lane];
                float4_t w[NT][KA];
                // The next stage's codes are converted among the products of K's operands, and its
                // set is filled again behind them.  (Behind the last stage the registers hold old
                // codes; what is written is not seen.)  A wave that sees none of the stage's keys, on
                // the diagonal, runs them masked: a branch round the products, or a way out of the
                // loop between its halves, would cost it a copy of all its sums.
                kv8_lds_scores<D, NT, KA, kAhead>(st, w, kb, [&](int e) {
                    constexpr int kEvery = KA * (D / 32) / (4 * C::kN);
                    if (e % kEvery == kEvery - 1 && e / kEvery < 2 * C::kN) store(u ^ 1, r[u], e / kEvery);
                });
                Kv8Stage after = next[u ^ 1];
                if (after.p0 >= 0) step(after);
                load(r[u], after);
                const int p0 = now.p0 < 0 ? kNone : now.p0;
                half8_t wp[NT][KA / 2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    kv8_softmax<D, KA>(st[nt], w[nt], p0, now.sc, p0 + C::kKeys - 1 > least);
#pragma unroll
                    for (int s = 0; s < KA / 2; ++s) wp[nt][s] = kv8_weights<KA>(w[nt], s);
                }
                kv8_lds_sums<D, NT, KA / 2, kAhead>(st, wp, kb + 2 * C::kUnits);
                lds_barrier();
                now = next[u];
                next[u] = after;
            }
        } while (now.p0 >= 0);
    }
    if (share.open && see >= share.n_full * kKvBlock) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            kv8_queries<D>(st[nt], p, at.b, at.h, row0 + 16 * nt, row_end);  // again: not held through the loop's end
            kv8_open_block<D>(st[nt], c, at.b, at.h, share.n_full, sq.len - share.n_full * kKvBlock, p.c2);
        }
    }
    kv8_finish<D, NT>(st, p, at, row0, row_end);
}

// ---- Many rows at D = 128 and 256 ----
// v_mfma_f32_32x32x16_f16 in place of the 16-row one: half the instructions for the same products,
// and its sums stay where they are over the branch that rescales them (two tiles of 16 rows moved
// all sums in every stage).  Lane l owns query row l % 32 and half h = l / 32 of the keys.  Register
// 4 a + e of a score tile of 32 keys holds key kv8_key32(a) + 4 h + e: K's rows are put in that
// order in LDS, so that the weights of registers 8 x .. 8 x + 7 are the keys of the 8 consecutive
// codes g4 = 2 x + h of a V unit.
__device__ __forceinline__ constexpr int kv8_key32(int a) { return 16 * (a & 1) + 4 * (a & 2); }

template <int D>
struct Kv8Rows32 {
    half8_t q[D / 16];    // operand B: step u holds d = 16 u + 8 h + 0 .. 7
    float16_t o[D / 32];  // O^T: d = 32 m + 8 (r / 4) + 4 h + r % 4 in register r
    float m, l;           // l: this lane's keys only
    int limit;            // last key the row sees, -1: none
};

// kv8_softmax for 32 KT keys.
template <int D, int KT>
__device__ __forceinline__ void kv8_softmax32(Kv8Rows32<D>& st, float16_t (&w)[KT], int p0, const Kv8Scale& sc, bool masked) {
    const int left = st.limit - p0 - 4 * (int)((threadIdx.x & 63) >> 5);
    if (masked) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) w[t][r] = 32 * t + kv8_key32(r >> 2) + (r & 3) <= left ? w[t][r] : -INFINITY;
    }
    float big = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) big = fmaxf(big, w[t][r]);
    big = __builtin_fmaf(big, sc.f, sc.lsv);  // of this lane's keys
    if (__any(big > st.m + kKvSlack)) {
        const float m_new = fmaxf(st.m, max_xor32(big));
        const float alpha = m_new == st.m ? 1.f : fast_exp2(st.m - m_new);
        st.m = m_new;
        st.l *= alpha;
#pragma unroll
        for (int m = 0; m < D / 32; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[m][r] *= alpha;
    }
    const float c = sc.lsv - (st.m == -INFINITY ? 0.f : st.m - kKvBias);
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) w[t][r] = fast_exp2(__builtin_fmaf(w[t][r], sc.f, c));
    if (masked && !(sc.f > 0.f && sc.lsv == sc.lsv)) {  // a key that is not seen weighs 0 (-inf times NaN, or times a factor that underflowed)
        int again = left;
        asm volatile("" : "+v"(again));  // compared here, and not kept from above on every path
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) w[t][r] = 32 * t + kv8_key32(r >> 2) + (r & 3) <= again ? w[t][r] : 0.f;
    }
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += w[t][r];
    st.l += sum == 0.f ? 0.f : sum * sc.isv;
}
// Weights of registers 8 x .. 8 x + 7 of a score tile as operand B.
__device__ __forceinline__ half8_t kv8_weights32(const float16_t& w, int x) {
    typedef float float8_v __attribute__((ext_vector_type(8)));
    const float8_v y = x ? __builtin_shufflevector(w, w, 8, 9, 10, 11, 12, 13, 14, 15) : __builtin_shufflevector(w, w, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_convertvector(y, half8_t);
}

// Where a lane's row of queries starts (its half of each step of 16 d).
__device__ __forceinline__ const half_t* kv8_query32(const Kv8AttnArgs& p, int b, int h, int row) {
    const int t = row / p.G, g = row % p.G;
    return p.q.data + b * p.q.b + (long long)(h * p.G + g) * p.q.h + t * p.q.t + 8 * ((threadIdx.x & 63) >> 5);
}

// kv8_open_block for 32 rows, whose queries are read from qr (is_row: the lane's row is one): held in
// registers with the sums they would spill at D = 256.
template <int D>
__device__ __forceinline__ void kv8_open_block32(Kv8Rows32<D>& st, const half_t* qr, bool is_row, const Kv8& c, int b, int h, int blk,
                                                 int n, float c2) {
    const int lane = threadIdx.x & 63, hi = lane >> 5, x32 = lane & 31;
    const size_t at = kv8_open_at<D>(c, b, h, blk);
    const half_t* ko = c.k_open + at;
    const half_t* vo = c.v_open + at;
    const int row = kv8_key32(x32 >> 3) + 4 * ((x32 >> 2) & 1) + (x32 & 3);  // this lane's key as operand A
#pragma unroll 1
    for (int s = 0; 32 * s < n; ++s) {  // half a block at a time
        const int p0 = blk * kKvBlock + 32 * s;
        float16_t w[1] = {};
#pragma unroll
        for (int u = 0; u < D / 16; ++u) {
            const half8_t q = is_row ? *reinterpret_cast<const half8_t*>(qr + 16 * u) : half8_t{};
            w[0] = mfma32(*reinterpret_cast<const half8_t*>(ko + kv8_k_at<D>(32 * s + row, 16 * u + 8 * hi)), q, w[0]);
            if (u % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // some loads at a time
        }
        kv8_softmax32<D, 1>(st, w, p0, {c2, 0.f, 1.f}, true);
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // 16 keys at a time
            const half8_t p = kv8_weights32(w[0], x);
            const int g4 = 2 * x + hi;  // keys 16 i + 4 g4 + e
            half8_t v[D / 32];
#pragma unroll
            for (int m = 0; m < D / 32; ++m) v[m] = *reinterpret_cast<const half8_t*>(vo + kv8_v_at<D>(32 * s + 4 * g4, 32 * m + x32));
            __builtin_amdgcn_sched_barrier(0);  // the loads wait for memory together (39 open rows at D = 256: 20 us, 7)
#pragma unroll
            for (int m = 0; m < D / 32; ++m) {
                bool bad = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool is = 32 * s + 16 * (j >> 2) + 4 * g4 + (j & 3) < n;
                    const bool off = kv8_bad(v[m][j]);
                    bad |= is && off;
                    if (!is || off) v[m][j] = (half_t)0.f;
                }
                st.o[m] = mfma32(v[m], p, st.o[m]);
                if (!__any(bad)) continue;
                float16_t more = {};  // (not on the sums themselves, which are to stay in place)
#pragma unroll 1
                for (int y = 0; y < 16; ++y) {  // a key: register 8 x + j of half g
                    const int j = y >> 1, g = y & 1, key = 16 * (j >> 2) + 4 * (2 * x + g) + (j & 3);
                    float wj = 0.f;
#pragma unroll
                    for (int r = 0; r < 8; ++r) wj = j == r ? w[0][8 * x + r] : wj;
                    wj = __shfl(wj, 32 * g + x32);
                    if (p0 + key > st.limit) continue;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const half_t z = vo[kv8_v_at<D>(32 * s + key, 32 * m + 8 * (r >> 2) + 4 * hi + (r & 3))];
                        if (kv8_bad(z)) more[r] += wj * (float)z;
                    }
                }
                st.o[m] += more;
            }
        }
    }
}

// A workgroup is 8 waves of 32 rows over one split of their blocks.  A stage of kKeys keys goes from
// memory to registers two stages ahead (a unit of K and one of V a thread), is turned into fp16
// operands once for all waves, and lies in one of two LDS buffers in operand order.  One barrier a
// stage.
// Bound by the card's power at D = 128 (prompt of 8192, 32 heads: 0.56 ms, 0.98 PFLOP/s, 1.8 GHz; the
// fp16 kernel of attn_fwd.hip, 0.53-0.55 ms at 1.6 GHz): two groups of waves taking turns at matrix
// and vector instructions needed 13 % fewer cycles and the same time.  At D = 256 (512 tokens over
// 16384, 24/4 heads: 0.21 ms, 0.95 PFLOP/s) by LDS, which the operands of 32 rows keep busy for as
// long as the matrix units; the two groups' second barrier a stage cost it 8 %.
template <int D>
struct Kv8Wide {
    static constexpr int kRows = 32 * 8;
    static constexpr int kKeys = D == 256 ? 32 : 64, kParts = kKvBlock / kKeys, KT = kKeys / 32;
    static constexpr int kUnits = kKeys * D / 16;  // 512: of K and of V, one a thread
    static constexpr int kAhead = D == 256 ? 3 : 4;  // operands read ahead of their products
    // At D = 256 128 sums and 64 registers of queries leave too few for the rest: the queries' last
    // steps are kept in LDS and read as operands with K's.
    static constexpr int kQl = D == 256 ? 6 : 0, kQr = D / 16 - kQl;
    static_assert(kUnits == 512, "a thread moves one unit of K and one of V a stage");
};
template <int D>
__global__ void __launch_bounds__(512, 2)
kv8_wide_kernel(Kv8AttnArgs p, int tiles, int streams) {
    using C = Kv8Wide<D>;
    constexpr int KT = C::KT;
    __shared__ __align__(16) half8_t kbuf[2][2 * C::kUnits];
    __shared__ __align__(16) half8_t vbuf[2][2 * C::kUnits];
    __shared__ __align__(16) half8_t qbuf[C::kQl ? 8 : 1][C::kQl ? C::kQl : 1][64];
    const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Kv8& c = p.c;
    Kv8Place at;
    if (!at.find(p, tiles, streams)) return;
    const Kv8Seq sq = kv8_seq(c, p.len, p.n_new, at.b, p.T);
    const int row_end = min(p.T, sq.n + sq.t0) * p.G;
    if (at.tile * C::kRows >= row_end) return;

    Kv8Rows32<D> st;
    int row = at.tile * C::kRows + wave * 32 + (lane & 31);
    const half_t* qr = kv8_query32(p, at.b, at.h, row);
#pragma unroll
    for (int u = 0; u < D / 16; ++u) st.q[u] = row < row_end ? *reinterpret_cast<const half8_t*>(qr + 16 * u) : half8_t{};
    st.limit = row < row_end ? kv8_limit(p, sq, row) : -1;
    int see = st.limit, least = row < row_end ? st.limit : INT_MAX;  // the last key that any, that every row sees
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        see = max(see, __shfl_xor(see, x));
        least = min(least, __shfl_xor(least, x));
    }
    see = __builtin_amdgcn_readfirstlane(see);
    least = __builtin_amdgcn_readfirstlane(least);
#pragma unroll
    for (int m = 0; m < D / 32; ++m) st.o[m] = float16_t{};
    st.m = -INFINITY;
    st.l = 0.f;
    Kv8Share share;
    share.find(p, sq, min(row_end, (at.tile + 1) * C::kRows) - 1, at.split);

    uint4 rk, rv;
    auto load = [&](const Kv8Stage& s) {
        if (s.p0 < 0) return;
        const size_t head = ((size_t)s.page * c.Hkv + at.h) * (kKvBlock * D);
        rk = reinterpret_cast<const uint4*>(c.k + head)[s.part * C::kUnits + tid];
        rv = reinterpret_cast<const uint4*>(c.v + head)[s.part * C::kUnits + tid];
    };
    // Where this thread's unit goes.  K: key 16 a + rr (a = tile / (D / 64)) of score tile a / 2, d =
    // 16 u + 0 .. 15: step u, halves 0 and 1, the key's row.  V: d = 32 m + dd and + 16, codes g4 of
    // half block s: step x = g4 / 2, half g4 % 2.
    const int g4 = (lane >> 4) & 3, rr = lane & 15, tile = tid >> 6;
    const int ka = tile / (D / 64), ku = tile % (D / 64) * 4 + g4, quad = rr >> 2;
    // score row of a key: register groups 0, 1, 2, 3 hold quads h, 4 + h, 2 + h, 6 + h
    const int krow = 8 * (2 * (quad >> 1) + (ka & 1)) + 4 * (quad & 1) + (rr & 3);
    const int kto = (ka / 2 * (D / 16) + ku) * 64 + krow;
    const int vto = (tile * 2 + (g4 >> 1)) * 64 + (g4 & 1) * 32 + rr;
    auto store_k = [&](int u) {
        kbuf[u][kto] = kv8_halves(rk.x, rk.y);
        kbuf[u][kto + 32] = kv8_halves(rk.z, rk.w);
    };
    auto store_v = [&](int u) {
        vbuf[u][vto] = kv8_halves(rv.x, rv.y);
        vbuf[u][vto + 16] = kv8_halves(rv.z, rv.w);
    };
    Kv8Stage now, then, after;
    auto step = [&](Kv8Stage& s) { kv8_step<C::kParts>(s, share.walk, c, at.b, at.h, p.c2); };
    step(then);
    if (then.p0 >= 0) {
        constexpr int kOps = KT * (D / 16);
        half8_t op[kOps], wp[2 * KT] = {};
        float16_t w[KT];
        half8_t* ql = &qbuf[C::kQl ? wave : 0][0][lane];  // a wave reads its own only
        // A stage's scores, with the next one's codes converted and written among the products.
        // (Behind the last stage the registers hold old codes; what is written is not read.)
        auto scores = [&](int u) {
            const half8_t* kb = &kbuf[u][lane];
            half8_t qop[D / 16];
            auto read_k = [&](int e) {  // tile e % KT, step e / KT
                op[e] = kb[(e % KT * (D / 16) + e / KT) * 64];
                if (e % KT == 0 && e / KT >= C::kQr) qop[e / KT] = ql[(e / KT - C::kQr) * 64];
            };
#pragma unroll
            for (int t = 0; t < KT; ++t) w[t] = float16_t{};
#pragma unroll
            for (int e = 0; e < C::kAhead; ++e) read_k(e);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < kOps; ++e) {
                if (e + C::kAhead < kOps) read_k(e + C::kAhead);
                w[e % KT] = mfma32(op[e], e / KT < C::kQr ? st.q[e / KT] : qop[e / KT], w[e % KT]);
                if (e == kOps / 4) store_k(u ^ 1);
                if (e == kOps / 2) store_v(u ^ 1);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto softmax = [&]() {
            kv8_softmax32<D, KT>(st, w, now.p0, now.sc, now.p0 + C::kKeys - 1 > least);
#pragma unroll
            for (int x = 0; x < 2 * KT; ++x) wp[x] = kv8_weights32(w[x / 2], x % 2);
        };
        // A stage's sums.  Product e: half block e / (D / 16), d block m, key step x (in LDS: half, m, x).
        auto sums = [&](int u) {
            const half8_t* vb = &vbuf[u][lane];
#pragma unroll
            for (int e = 0; e < C::kAhead; ++e) op[e] = vb[e * 64];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < kOps; ++e) {
                if (e + C::kAhead < kOps) op[e + C::kAhead] = vb[(e + C::kAhead) * 64];
                const int s = e / (D / 16), m = e % (D / 16) / 2, x = e % 2;
                st.o[m] = mfma32(op[e], wp[2 * s + x], st.o[m]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        load(then);
        store_k(0);
        store_v(0);
        after = then;
        step(after);
        load(after);
#pragma unroll
        for (int u = 0; u < D / 16; ++u) asm volatile("" : "+v"(st.q[u]));  // arrived (see kv8_arrived)
#pragma unroll
        for (int x = 0; x < C::kQl; ++x) ql[x * 64] = st.q[C::kQr + x];
        lds_barrier();
        int u = 0;
        do {  // (its end behind the barrier: left among the products, the sums were moved in every stage)
            now = then;
            then = after;
            scores(u);
            if (then.p0 >= 0) step(after);
            load(after);
            softmax();
            __builtin_amdgcn_s_setprio(1);
            sums(u);
            __builtin_amdgcn_s_setprio(0);
            lds_barrier();
            u ^= 1;
        } while (then.p0 >= 0);
    }
    asm volatile("" : "+v"(row));  // what follows from it below is computed again, not held through the loop
    if (share.open && see >= share.n_full * kKvBlock) {
        kv8_open_block32<D>(st, kv8_query32(p, at.b, at.h, row), row < row_end, c, at.b, at.h, share.n_full, sq.len - share.n_full * kKvBlock, p.c2);
    }
    const float l = sum_xor32(st.l);
    if (row >= row_end) return;
    if (p.nsplit > 1) {
        if (l != 0.f) {
            float* part = kv8_part<D>(p, kv8_slot(p, at.bh, row, at.split)) + 4 * hi;
#pragma unroll
            for (int m = 0; m < D / 32; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    *reinterpret_cast<float4_t*>(part + 32 * m + 8 * r) =
                        float4_t{st.o[m][4 * r], st.o[m][4 * r + 1], st.o[m][4 * r + 2], st.o[m][4 * r + 3]};
        }
        if (hi == 0) *kv8_pair(p, kv8_slot(p, at.bh, row, at.split)) = float2{st.m, l};
    } else {
        const int t = row / p.G, hq = at.h * p.G + row % p.G;
#pragma unroll
        for (int m = 0; m < D / 32; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 32 * m + 8 * r + 4 * hi;
                kv8_store4(p, at.b, hq, t, d, float4_t{st.o[m][4 * r], st.o[m][4 * r + 1], st.o[m][4 * r + 2], st.o[m][4 * r + 3]}, l,
                           kv8_gate4(p, at.b, hq, t, d));
            }
    }
}

// Joins the splits of 1024 / D rows: workgroup (rows, b Hkv + h), D / 4 lanes a row.  Every address
// is known at once, so that the loads wait for memory together and not for each other: a row's
// maxima and sums, its first splits' sums (unread where they were not written), its gate.
template <int D, bool kDeal>
__global__ void __launch_bounds__(256)
kv8_join_kernel(Kv8AttnArgs p) {
    constexpr int kLanes = D / 4, kRows = 256 / kLanes, kAhead = 16;
    __shared__ float fs[kRows][kKvMaxSplits];
    const Kv8& c = p.c;
    const int b = blockIdx.y / c.Hkv, h = blockIdx.y % c.Hkv;
    const int r = threadIdx.x / kLanes, x = threadIdx.x % kLanes, n_rows = p.T * p.G;
    const int row = min((int)blockIdx.x * kRows + r, n_rows - 1);
    int n = p.nsplit;
    size_t slot = kv8_slot(p, blockIdx.y, row, 0), step = 1;
    if constexpr (kDeal) {
        using Deal = Kv8Deal<kKvBlock / Kv8Regs<D, true>::kKeys>;
        Deal deal;
        deal.find(p);
        const int own = deal.own(p, b), first = deal.group(deal.before);
        n = own ? min(deal.group(deal.before + own - 1) - first + 1, kKvMaxSplits) : 1;
        slot = kv8_dealt_slot(p, h, first + b, row);
        step = n_rows;
    }
    const float2* pair = kv8_pair(p, slot);
    const float4_t* at = reinterpret_cast<const float4_t*>(kv8_part<D>(p, slot)) + x;
    float2 ml[kKvMaxSplits / kLanes];
#pragma unroll
    for (int i = 0; i < kKvMaxSplits / kLanes; ++i) ml[i] = pair[min(x + i * kLanes, n - 1) * step];
    float4_t part[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) part[s] = at[min(s, n - 1) * step * (D / 4)];
    const int t = row / p.G, hq = h * p.G + row % p.G;
    const half4_t gate = kv8_gate4(p, b, hq, t, 4 * x);
    const Kv8Seq sq = kv8_seq(c, p.len, p.n_new, b, p.T);
    const bool is = (int)blockIdx.x * kRows + r < n_rows && t < sq.n + sq.t0;  // rows of padding have no sums
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kKvMaxSplits / kLanes; ++i) {
        if (x + i * kLanes >= n) ml[i] = float2{-INFINITY, 0.f};
        m = fmaxf(m, ml[i].x);
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
#pragma unroll
    for (int i = 0; i < kKvMaxSplits / kLanes; ++i) {
        float f = ml[i].y == 0.f ? 0.f : ml[i].x == m ? 1.f : fast_exp2(ml[i].x - m);
        if (ml[i].y != ml[i].y) f = ml[i].y;  // a row of NaN, whatever its maximum
        l += ml[i].y == 0.f ? 0.f : f * ml[i].y;
        if (x + i * kLanes < n) fs[r][x + i * kLanes] = f;
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
        if (s < n) add(part[s], fs[r][s]);
    for (int s0 = kAhead; s0 < n; s0 += kAhead) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s) part[s] = at[min(s0 + s, n - 1) * step * (D / 4)];
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
            if (s0 + s < n) add(part[s], fs[r][s0 + s]);
    }
    kv8_store4(p, b, hq, t, 4 * x, y, l, gate);
}

// Listed tiles from which on a wave takes one by itself: as many as the chip has room for waves of
// the kernel (fewer leave SIMDs empty, and a tile's four waves are joined instead).
constexpr int kKvWaveTiles = 2048;

// How a call's rows are cut into tiles and its keys into splits.
struct Kv8Plan {
    int rows;       // of a tile
    long long tiles;  // of one K/V head
    int nsplit;
    int share;      // above 0: keys are dealt to so many workgroups a head
    int splits;     // no call with fewer items has more
};
// At D = 64 65 to 128 rows are two tiles of 64 where the call has at most this many blocks (a
// sequence's by the K/V heads), and one of 128 above.  Up to 16 blocks a CU the call waits more than it
// computes, and twice the workgroups wait less (96 rows, 8 x 2777 keys, 2 heads: 20.2 us with 128 rows, 16.0
// with 64; 1 x 32000, 4 heads: 36.0, 26.9; at 4096 blocks 25.5 to 38.6, 26.7 to 33.2); with more, two tiles
// convert every code twice (32 x 8000, 2 heads: 38.7, 42.1).
constexpr long long kKvSmallTileBlocks = 4096;

// One tile of 16 rows where there are no more (and for listed blocks, one query's heads), else
// workgroups of 64 rows, or more at D = 64 of 128 and at D = 128 and 256 of 256.  items: blocks of the
// longest sequence, or of a list.
inline Kv8Plan kv8_plan(const Kv8& c, int T, int Hq, int items, bool list) {
    const long long G = Hq / c.Hkv, rows = T * G;
    Kv8Plan q;
    const bool small = rows <= 64 || (rows <= 128 && (c.D != 64 || (long long)c.B * c.Hkv * items <= kKvSmallTileBlocks));
    q.rows = list || rows <= 16 ? 16 : small ? 64 : c.D == 64 ? 128 : 256;
    q.tiles = list ? T * ((G + 15) / 16) : (rows + q.rows - 1) / q.rows;
    const long long all = q.tiles * c.B * c.Hkv;
    // row tiles: as many workgroups as the chip takes twice, but two stages of keys a wave at the
    // least; the others as many as it takes once, but 2 blocks at the least (500 tokens of one head,
    // D = 256: 4 blocks 40 us, 2 31; 300 tokens over 2300, 4 heads, D = 128: 26, 24), or 4 of 64 rows (8
    // sequences of 2777, 5 tokens, 16/2 heads, D = 64: 4 blocks 12.5 us, 2 14.3)
    const bool few = q.rows == 16;
    const int parts = c.D == 256 ? 2 : 1;
    const long long want = few ? (1024 + all - 1) / all : (q.rows == 256 ? 256 : 512) / all;
    const long long most = few ? ((long long)items * parts + 7) / 8 : q.rows == 64 ? (items + 3) / 4 : (items + 1) / 2;
    long long n = want < most ? want : most;
    n = n < 1 ? 1 : n < kKvMaxSplits ? n : kKvMaxSplits;
    q.splits = (int)n;
    // The sums of splits of 256 rows that fill the chip take as long to write and join as 8 blocks to
    // multiply (7 x 640 tokens, 6/2 heads, D = 256: 56 us in 2 splits, 51 in one).
    if (q.rows == 256 && n > 1 && items * (n - 1) * 256 <= 8 * all * n * n) n = 1;
    q.nsplit = (int)n;
    // Several sequences whose keys fill the chip: dealt out (parts are counted in ints).  Where two
    // stages a wave are the bound, most workgroups would have two short segments one after the other.
    q.share = few && !list && c.B > 1 && want > 1 && want < most && c.B * ((long long)c.max_blocks * parts + 4) < INT_MAX
                  ? 1024 / c.Hkv & ~7 : 0;
    return q;
}
inline size_t kv8_slots(const Kv8& c, int T, int Hq, const Kv8Plan& q) {
    return (q.share ? q.share + c.B : q.nsplit > 1 ? (size_t)c.B * q.nsplit : 0) * T * Hq;
}
// Enough for every call with no more items too.
inline size_t kv8_part_bytes(const Kv8& c, int T, int Hq, const Kv8Plan& q) {
    const size_t own = kv8_slots(c, T, Hq, q), fewer = q.splits > 1 ? (size_t)c.B * q.splits * T * Hq : 0;
    return (own > fewer ? own : fewer) * (c.D + 2) * 4;
}

template <int D, bool kList>
hipError_t kv8_attn_d(const Kv8AttnArgs& p, const Kv8Plan& q, hipStream_t stream) {
    const int BH = p.c.B * p.c.Hkv;
    if (kList || q.rows == 16) {
        const long long n = q.tiles * BH * p.nsplit;
        bool done = false;
        if constexpr (kList) {
            if ((done = n >= kKvWaveTiles)) {
                const dim3 grid((unsigned)((n + 31) / 32 * 8));
                hipLaunchKernelGGL((kv8_row_kernel<D, true, 1, false>), grid, dim3(256), 0, stream, p, (int)q.tiles);
            }
        }
        if constexpr (!kList) {
            if ((done = p.share > 0))
                hipLaunchKernelGGL((kv8_row_kernel<D, false, 4, true>), dim3((unsigned)(p.share * p.c.Hkv)), dim3(256), 0, stream, p, 1);
        }
        if (!done) {
            const dim3 grid((unsigned)((n + 7) / 8 * 8));
            hipLaunchKernelGGL((kv8_row_kernel<D, kList, 4, false>), grid, dim3(256), 0, stream, p, (int)q.tiles);
        }
    } else {
        const dim3 grid((unsigned)((q.tiles * BH * p.nsplit + 7) / 8 * 8));
        const int streams = BH * p.nsplit;
        if (q.rows == 64 && q.tiles == 1)
            hipLaunchKernelGGL((kv8_tile_kernel<D, 1, true>), grid, dim3(256), 0, stream, p, (int)q.tiles, streams);
        else if (q.rows == 64)
            hipLaunchKernelGGL((kv8_tile_kernel<D, 1, false>), grid, dim3(256), 0, stream, p, (int)q.tiles, streams);
        else if constexpr (D == 64)
            hipLaunchKernelGGL((kv8_tile_kernel<D, 2, false>), grid, dim3(256), 0, stream, p, (int)q.tiles, streams);
        else
            hipLaunchKernelGGL(kv8_wide_kernel<D>, grid, dim3(512), 0, stream, p, (int)q.tiles, streams);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || (p.nsplit == 1 && !p.share)) return e;
    constexpr int kRows = 1024 / D;
    const dim3 rows((unsigned)((p.T * p.G + kRows - 1) / kRows), (unsigned)BH);
    if constexpr (!kList) {
        if (p.share) {
            hipLaunchKernelGGL((kv8_join_kernel<D, true>), rows, dim3(256), 0, stream, p);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL((kv8_join_kernel<D, false>), rows, dim3(256), 0, stream, p);
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
    const Kv8Plan plan = kv8_plan(c, T, Hq, nb_hint, false);
    float* part = (float*)ws;
    return kv8_attn_any<false>({c, q, gate, o, len, n_new, nullptr, part, part ? part + kv8_slots(c, T, Hq, plan) * c.D : nullptr, T, Hq,
                                Hq / c.Hkv, 0, plan.nsplit, causal, plan.share, scale * kLog2e}, plan, stream);
}

hipError_t kv8_attn_blocks(const Kv8& c, const Rows16& q, const Rows16& gate, const Rows16& o, const int* len,
                           const int* n_new, int T, int Hq, const int* blocks, int top, float scale, void* ws,
                           hipStream_t stream) {
    const Kv8Plan plan = kv8_plan(c, T, Hq, top, true);
    float* part = (float*)ws;
    return kv8_attn_any<true>({c, q, gate, o, len, n_new, blocks, part, part ? part + kv8_slots(c, T, Hq, plan) * c.D : nullptr, T, Hq,
                               Hq / c.Hkv, top, plan.nsplit, 1, plan.share, scale * kLog2e}, plan, stream);
}

}  // namespace tsa
