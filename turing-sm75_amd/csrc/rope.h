// rope.h -- rotary positions of queries and keys, and their gradient (the rotation back).
//
// Pair i of a row at position p turns by p f_i: (a, b) <- m (a cos - b sin, a sin + b cos).  The
// frequencies come as whole turns per position in 2^-64 (the host makes them in 80-bit floats), so
// p f_i mod 1 is one 64-bit product that wraps by itself: exact to 2^-65 p turns at every position,
// where a 32-bit product of position and frequency is off by a hundredth of a turn at p = 131072.  The fraction's
// distance from the nearest quarter turn, at most an eighth, then becomes a float, and sine and
// cosine are their power series to x^9 and x^10 (rest below 2.5e-9 at pi / 4).
//
// Bound by memory: every element is read and written once.  A thread keeps the sines and cosines of
// kVec pairs of one token and walks over some of its heads, so they cost a fraction of a head's
// loads and stores (kVec = 8: two 16-byte loads of fp16).
#pragma once
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
    int Hq, H, B, T, rot, units, per, flip;  // H: heads of q and k; units a row; heads a thread; flip: turn back
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

// Unit u of a row: pairs u kVec .. + kVec - 1 while those are below rot / 2, then the elements behind
// the rotated ones, 2 kVec at a time (only where they have to be copied: out of place).
constexpr int kAtOnce = 4;
template <typename T, bool kInter, int kVec>
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs a) {
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const int u = (int)(at % a.units);
    const long long row = at / a.units;  // (sequence, token)
    if (row >= (long long)a.B * a.T) return;
    const int b = (int)(row / a.T), t = (int)(row % a.T);
    const int n = a.n_new ? min(max(a.n_new[b], 0), a.T) : a.T;
    if (t >= n) return;
    const bool turn = u * 2 * kVec < a.rot;
    float s[kVec], c[kVec];
    if (turn) {
        const long long p = a.pos ? (long long)a.pos[row] : (a.len ? (long long)a.len[b] - n : 0) + t;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            sincos_turns((unsigned long long)p * a.freq[u * kVec + i], s[i], c[i]);
            s[i] *= a.flip ? -a.amp : a.amp;
            c[i] *= a.amp;
        }
    }
    const int lo = kInter || !turn ? u * 2 * kVec : u * kVec;  // the unit's elements: kVec at lo, kVec at up
    const int up = kInter || !turn ? lo + kVec : lo + a.rot / 2;
    const int h0 = blockIdx.y * a.per, h1 = min(h0 + a.per, a.H);
    using P = Pack<T, kVec>;
    auto rows = [&](int h, const T*& src, T*& dst) {
        const bool is_q = h < a.Hq;
        const RopeTensor& x = is_q ? a.q : a.k;
        const int hh = is_q ? h : h - a.Hq;
        src = static_cast<const T*>(x.in) + b * x.in_b + hh * x.in_h + t * x.in_t;
        dst = static_cast<T*>(x.out) + b * x.out_b + hh * x.out_h + t * x.out_t;
    };
    // kAtOnce heads' loads on their way together
    for (int h = h0; h < h1; h += kAtOnce) {
        P v[kAtOnce][2];
        T* dst[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (h + i < h1) {
                const T* src;
                rows(h + i, src, dst[i]);
                v[i][0] = *reinterpret_cast<const P*>(src + lo);
                v[i][1] = *reinterpret_cast<const P*>(src + up);
            }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (h + i < h1) {
                if (turn) rotate<T, kInter, kVec>(v[i][0].x, v[i][1].x, s, c);
                *reinterpret_cast<P*>(dst[i] + lo) = v[i][0];
                *reinterpret_cast<P*>(dst[i] + up) = v[i][1];
            }
    }
}

template <typename T, bool kInter>
hipError_t launch_rope(RopeArgs& a, const dim3& grid, bool wide, hipStream_t stream) {
    if (wide)
        hipLaunchKernelGGL((rope_kernel<T, kInter, 8>), grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((rope_kernel<T, kInter, 1>), grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

RopeTensor tensor(const RopeRows& in, const RopeRows& out) {
    return {in.data, out.data, in.b, in.h, in.t, out.b, out.h, out.t};
}

}  // namespace

hipError_t rope(const unsigned long long* freq, float amp, int rot, int interleaved, int f32, const RopeRows& q,
                const RopeRows& q_out, int Hq, const RopeRows& k, const RopeRows& k_out, int Hk, const int* pos,
                const int* len, const int* n_new, int B, int T, int D, int back, hipStream_t stream) {
    // 16-byte loads need rows whose pairs come in eights
    const bool wide = rot % 16 == 0;
    // elements that do not turn are copied unless every tensor is rotated in place
    const bool copy = rot < D && (q.data != q_out.data || (Hk && k.data != k_out.data));
    const int H = Hq + Hk, units = (copy ? D : rot) / (wide ? 16 : 2);
    const long long threads = (long long)B * T * units;
    // heads a thread: one where that does not fill the device, else 8 to share the sines
    const long long groups = (threads + 255) / 256;
    const int per = groups * H <= 2048 ? 1 : groups * H <= 8192 ? 4 : 8;
    const dim3 grid((unsigned)groups, (unsigned)((H + per - 1) / per));
    RopeArgs a = {tensor(q, q_out), tensor(k, k_out), freq, pos, len, n_new, amp, Hq, H, B, T, rot, units, per, back};
    if (f32)
        return interleaved ? launch_rope<float, true>(a, grid, wide, stream) : launch_rope<float, false>(a, grid, wide, stream);
    return interleaved ? launch_rope<half_t, true>(a, grid, wide, stream) : launch_rope<half_t, false>(a, grid, wide, stream);
}

}  // namespace tsa
