// rope.h -- rotary positions of queries and keys, and their gradient (the rotation back).
//
// Pair i of a row at position p turns by p f_i: (a, b) <- m (a cos - b sin, a sin + b cos).  The
// frequencies come as whole turns per position in 2^-64 (the host makes them in 80-bit floats), so
// p f_i mod 1 is one 64-bit product that wraps by itself: exact to 2^-65 p turns at every position,
// where a 32-bit product of position and frequency is off by a hundredth of a turn at p = 131072.  The fraction's
// distance from the nearest quarter turn, at most an eighth, then becomes a float, and sine and
// cosine are their power series to x^9 and x^10 (rest below 2.5e-9 at pi / 4).
//
// Bound by memory: every element is read and written once.  A workgroup takes some tokens of all heads (or a
// share of them): it makes the sines and cosines of their pairs once, one a thread, while the first rows are on their way
// (3 x 2001 fp32 rows of 18 heads: 14.7 us without that, 13.4 with), and leaves them in
// LDS; then a thread turns kVec pairs of a head at a time (two loads of 16 bytes where rot allows).  Neighbouring
// threads go over a row, then over what lies next to it in memory, tokens or heads.  8192 tokens of 64 heads,
// D = 128: 54 us in fresh memory, 4970 GB/s of 268 MB, where a large copy has 5080.  One token of 28 heads: 3.1 us
// on the device, 7.5 a call.
#pragma once
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace tsa {
namespace {

constexpr float kTurn = 6.2831853071795865f;

// Sine and cosine of ph 2^-64 turns.
__device__ __forceinline__ void sincos_turns(unsigned long long ph, float& s, float& c) {
    const unsigned quarter = (unsigned)((ph + (1ull << 61)) >> 62);
    const long long rest = (long long)(ph - ((unsigned long long)quarter << 62));
    // rest 2^-64 turns in radians: the halves converted apart, one rounding in the sum
    const float hi = (float)(int)(rest >> 32) * (kTurn * 0x1p-32f);
    const float x = fmaf((float)(unsigned)rest, kTurn * 0x1p-64f, hi);
    const float y = x * x;
    const float sx = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
    const float cx = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    s = quarter & 1 ? cx : sx;
    c = quarter & 1 ? sx : cx;
    if (quarter & 2) s = -s;
    if ((quarter + 1) & 2) c = -c;
}

template <typename T, int kN>
struct __align__(kN * sizeof(T) >= 16 ? 16 : kN * sizeof(T)) Pack {
    T x[kN];
};

struct RopeTensor {
    const void* in;
    void* out;
    long long in_b, in_h, in_t, out_b, out_h, out_t;
};
struct RopeArgs {
    RopeTensor q, k;
    const unsigned long long* freq;
    const int *pos, *len, *n_new;
    float amp;
    // H: heads of q and k; units a row; tokens, and items (units of all their rows), a workgroup column;
    // share: items a workgroup; flip: turn back; heads_next: a token's heads lie side by side
    int Hq, H, B, T, rot, units, tokens, items, share, flip, heads_next;
};

// kVec pairs: interleaved in x then y, or their first elements in x and their second in y.
template <typename T, bool kInter, int kVec>
__device__ __forceinline__ void rotate(T (&x)[kVec], T (&y)[kVec], const float (&s)[kVec], const float (&c)[kVec]) {
    T e[2 * kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) e[kInter ? i : 2 * i] = x[i], e[kInter ? kVec + i : 2 * i + 1] = y[i];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const float p = (float)e[2 * i], q = (float)e[2 * i + 1];
        e[2 * i] = (T)fmaf(p, c[i], -(q * s[i]));
        e[2 * i + 1] = (T)fmaf(q, c[i], p * s[i]);
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) x[i] = e[kInter ? i : 2 * i], y[i] = e[kInter ? kVec + i : 2 * i + 1];
}

constexpr int kThreads = 256, kAtOnce = 4, kAngles = 256;  // angles a workgroup makes at most: tokens rot / 2
constexpr int kColumns = 1 << 23;  // columns of tokens in a grid's x (whose threads are fewer than 2^32); the next ones are in its z

// Unit u of a row: pairs u kVec .. + kVec - 1 while those are below rot / 2, then the elements behind
// the rotated ones, 2 kVec at a time (only where they have to be copied: out of place).
template <typename T, bool kInter, int kVec>
__global__ void __launch_bounds__(kThreads) rope_kernel(RopeArgs a) {
    __shared__ __align__(16) float sines[kAngles], cosines[kAngles];
    const int tid = threadIdx.x, half = a.rot / 2;
    const long long row0 = ((long long)blockIdx.z * kColumns + blockIdx.x) * a.tokens, rows = (long long)a.B * a.T;
    // Row r of the column, if it is a token (not padding, nor past the last).
    auto token = [&](int r, int& b, int& t, int& n) {
        const long long row = row0 + r;
        if (row >= rows) return false;
        b = (int)((unsigned)row / (unsigned)a.T);  // (rows of all sequences fit an int)
        t = (int)((unsigned)row % (unsigned)a.T);
        n = a.n_new ? min(max(a.n_new[b], 0), a.T) : a.T;
        return t < n;
    };
    // A thread's angle (there are no more than threads), whose numbers are on their way in front of the rows.
    bool mine = false;
    unsigned long long phase = 0;
    if (tid < a.tokens * half) {
        const int r = (int)((unsigned)tid / (unsigned)half), pair = tid - r * half;
        int b, t, n;
        if (token(r, b, t, n)) {
            mine = true;
            const long long p = a.pos ? (long long)a.pos[row0 + r] : (a.len ? (long long)a.len[b] - n : 0) + t;
            phase = (unsigned long long)p * a.freq[pair];
        }
    }
    // kAtOnce units' loads on their way together, the first of them while the angles are made
    using P = Pack<T, kVec>;
    const int end = min(a.items, (int)(blockIdx.y + 1) * a.share);
    P v[kAtOnce][2];
    T *lo[kAtOnce], *up[kAtOnce];
    int angle[kAtOnce];  // of the unit's first pair; -1: copied, -2: nothing there
    auto load = [&](int i0) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const int i = i0 + j * kThreads;
            angle[j] = -2;
            if (i >= end) continue;
            const int x = (int)((unsigned)i / (unsigned)a.units), u = i - x * a.units;
            int h, r;
            if (a.heads_next)
                r = (int)((unsigned)x / (unsigned)a.H), h = x - r * a.H;
            else
                h = (int)((unsigned)x / (unsigned)a.tokens), r = x - h * a.tokens;
            int b, t, n;
            if (!token(r, b, t, n)) continue;
            const bool turn = u * 2 * kVec < a.rot, is_q = h < a.Hq;
            const RopeTensor& y = is_q ? a.q : a.k;
            const int hh = is_q ? h : h - a.Hq;
            // the unit's elements: kVec at e0, kVec at e1
            const int e0 = kInter || !turn ? u * 2 * kVec : u * kVec, e1 = kInter || !turn ? e0 + kVec : e0 + half;
            const T* src = static_cast<const T*>(y.in) + b * y.in_b + hh * y.in_h + t * y.in_t;
            T* dst = static_cast<T*>(y.out) + b * y.out_b + hh * y.out_h + t * y.out_t;
            v[j][0] = *reinterpret_cast<const P*>(src + e0);
            v[j][1] = *reinterpret_cast<const P*>(src + e1);
            lo[j] = dst + e0, up[j] = dst + e1;
            angle[j] = turn ? r * half + u * kVec : -1;
        }
    };
    int i0 = blockIdx.y * a.share + tid;
    load(i0);
    if (mine) {
        float s, c;
        sincos_turns(phase, s, c);
        sines[tid] = s * (a.flip ? -a.amp : a.amp);
        cosines[tid] = c * a.amp;
    }
    lds_barrier();
    while (i0 < end) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            if (angle[j] == -2) continue;
            if (angle[j] >= 0) {
                float s[kVec], c[kVec];
#pragma unroll
                for (int e = 0; e < kVec; ++e) s[e] = sines[angle[j] + e], c[e] = cosines[angle[j] + e];
                rotate<T, kInter, kVec>(v[j][0].x, v[j][1].x, s, c);
            }
            *reinterpret_cast<P*>(lo[j]) = v[j][0];
            *reinterpret_cast<P*>(up[j]) = v[j][1];
        }
        i0 += kThreads * kAtOnce;
        load(i0);
    }
}

template <typename T, bool kInter>
hipError_t launch_rope(const RopeArgs& a, const dim3& grid, int vec, hipStream_t stream) {
    if constexpr (sizeof(T) == 2)
        if (vec == 8) {
            hipLaunchKernelGGL((rope_kernel<T, kInter, 8>), grid, dim3(kThreads), 0, stream, a);
            return hipGetLastError();
        }
    if (vec == 4)
        hipLaunchKernelGGL((rope_kernel<T, kInter, 4>), grid, dim3(kThreads), 0, stream, a);
    else if (vec == 2)
        hipLaunchKernelGGL((rope_kernel<T, kInter, 2>), grid, dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((rope_kernel<T, kInter, 1>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

RopeTensor tensor(const RopeRows& in, const RopeRows& out) {
    return {in.data, out.data, in.b, in.h, in.t, out.b, out.h, out.t};
}

}  // namespace

hipError_t rope(const unsigned long long* freq, float amp, int rot, int interleaved, int f32, const RopeRows& q,
                const RopeRows& q_out, int Hq, const RopeRows& k, const RopeRows& k_out, int Hk, const int* pos,
                const int* len, const int* n_new, int B, int T, int D, int back, hipStream_t stream) {
    // the widest loads that the rotated part's halves allow, up to 16 bytes (two of them a unit; with 8 fp32 pairs, which
    // is four, 3 x 2001 rows of 18 heads by halves take 13.4 us for 11.0; interleaved fp16 with 4 pairs, which is
    // one, 8192 x 64 heads of D = 128 take 56.1 for 54.6)
    const int most_vec = f32 ? 4 : 8, vec = std::min(most_vec, rot % 16 == 0 ? 8 : rot % 8 == 0 ? 4 : rot % 4 == 0 ? 2 : 1);
    // elements that do not turn are copied unless every tensor is rotated in place
    const bool copy = rot < D && (q.data != q_out.data || (Hk && k.data != k_out.data));
    RopeArgs a = {tensor(q, q_out), tensor(k, k_out), freq, pos, len, n_new, amp, Hq, Hq + Hk, B, T, rot, (copy ? D : rot) / (2 * vec)};
    const long long rows = (long long)B * T;
    // tokens of a workgroup: two units a thread, at most 256 angles, and 512 workgroups where there are the rows
    a.tokens = (int)std::max<long long>(1, std::min<long long>({512 / (a.H * a.units), 512 / rot, rows / 512}));
    a.items = a.tokens * a.H * a.units;
    a.flip = back;
    a.heads_next = q.h < q.t && T > 1;
    // one workgroup a column of tokens where there are enough of them; else its items are dealt out, a unit a thread at least
    const long long columns = (rows + a.tokens - 1) / a.tokens, most = (a.items + kThreads - 1) / kThreads;
    const long long deal = std::max(1LL, std::min({most, 1024 / columns, 65535LL}));
    a.share = (int)((most + deal - 1) / deal) * kThreads;
    const dim3 grid((unsigned)std::min<long long>(columns, kColumns), (unsigned)((a.items + a.share - 1) / a.share),
                    (unsigned)((columns + kColumns - 1) / kColumns));
    if (f32)
        return interleaved ? launch_rope<float, true>(a, grid, vec, stream) : launch_rope<float, false>(a, grid, vec, stream);
    return interleaved ? launch_rope<half_t, true>(a, grid, vec, stream) : launch_rope<half_t, false>(a, grid, vec, stream);
}

}  // namespace tsa
