// kv8_select.h -- the blocks of an 8-bit K/V cache that each query attends to, by a cheap score.
//
// With A the largest |q| of the group's heads, qc = rint(127 q / A), and a block's summary m
// (8 bits, step m_scale; see kv8_cache.h), the score is max_g sum_d qc[g][d] m[d], a whole number
// below 2^24, times m_scale: one fp32 product, so every order of summing gives the same score and
// the same choice.  A group's queries share their blocks (A does not change the order).
#pragma once
#include <climits>

#include "kv8.h"

namespace tsa {
namespace {

struct Kv8SelectArgs {
    Kv8 c;
    Rows16 q;
    const int *len, *n_new;
    signed char* qc;   // [B][Hkv][T][G][D]
    float* score;      // [B][Hkv][T][nb]
    int* blocks;       // [B][Hkv][T][top]
    int T, Hq, G, top, first, recent, nb;
};

// Workgroup (t, b Hkv + h): the group's query codes.
template <int D>
__global__ void __launch_bounds__(256)
kv8_qcode_kernel(Kv8SelectArgs p) {
    __shared__ int red;
    const int b = blockIdx.y / p.c.Hkv, h = blockIdx.y % p.c.Hkv, t = blockIdx.x;
    const Kv8Seq sq = kv8_seq(p.c, p.len, p.n_new, b, p.T);
    if (t >= sq.n + sq.t0) return;
    const half_t* q = p.q.data + b * p.q.b + (long long)h * p.G * p.q.h + t * p.q.t;
    if (threadIdx.x == 0) red = 1;
    __syncthreads();
    int most = 0;
    for (int i = threadIdx.x; i < p.G * D; i += 256)
        most = max(most, (int)(__builtin_bit_cast(unsigned short, q[i / D * p.q.h + i % D]) & 0x7fff));
    atomicMax(&red, most);
    __syncthreads();
    most = red;
    const float a = (float)__builtin_bit_cast(half_t, (unsigned short)most);
    signed char* qc = p.qc + ((size_t)blockIdx.y * p.T + t) * p.G * D;
    // a group with an infinity or NaN has no order: all its codes are 0
    for (int i = threadIdx.x; i < p.G * D; i += 256)
        qc[i] = most < 0x7c00 ? (signed char)(int)rintf(127.f * (float)q[i / D * p.q.h + i % D] / a) : (signed char)0;
}

// Workgroup (t and 256 blocks, b Hkv + h): a block a thread.
template <int D>
__global__ void __launch_bounds__(256)
kv8_score_kernel(Kv8SelectArgs p) {
    extern __shared__ int qs[];
    const int parts = (p.nb + 255) / 256, i0 = (int)(blockIdx.x % parts) * 256;
    const int b = blockIdx.y / p.c.Hkv, h = blockIdx.y % p.c.Hkv, t = blockIdx.x / parts;
    const Kv8Seq sq = kv8_seq(p.c, p.len, p.n_new, b, p.T);
    const int pos = sq.len - (sq.n + sq.t0) + t;
    if (t >= sq.n + sq.t0 || pos < 0) return;
    const int own = min(pos / kKvBlock, p.nb);
    if (i0 >= own) return;  // the own block has no score
    const size_t row = (size_t)blockIdx.y * p.T + t;
    const int* qc = reinterpret_cast<const int*>(p.qc + row * p.G * D);
    for (int i = threadIdx.x; i < p.G * D / 4; i += 256) qs[i] = qc[i];
    __syncthreads();
    const int blk = i0 + threadIdx.x;
    if (blk >= own) return;
    const int page = kv8_page(p.c, b, blk);
    float score = -INFINITY;
    if (page >= 0) {
        const size_t head = (size_t)page * p.c.Hkv + h;
        const int* m = reinterpret_cast<const int*>(p.c.k_sum + head * D);
        int best = INT_MIN;
        for (int g = 0; g < p.G; ++g) {
            int s = 0;
            for (int i = 0; i < D / 4; ++i) s = __builtin_amdgcn_sdot4(m[i], qs[g * (D / 4) + i], s, false);
            best = max(best, s);
        }
        const float x = (float)best * p.c.k_sum_scale[head];
        score = x == x ? x : -INFINITY;  // a block that holds an infinity or NaN
    }
    p.score[row * p.nb + blk] = score;
}

// A score as a whole number of the same order; 0 is below every score.
__device__ __forceinline__ unsigned kv8_order(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);  // -0 ties with 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Workgroup (t, b Hkv + h): the `top` best of the row's blocks, the lowest index first among
// equals, listed ascending.  Four rounds over the scores' bytes find the last value that is kept.
__global__ void __launch_bounds__(256)
kv8_pick_kernel(Kv8SelectArgs p) {
    __shared__ int hist[256];
    __shared__ int found[2];  // the round's byte, and how many of it are still to be kept
    __shared__ int sums[2][4];
    const int b = blockIdx.y / p.c.Hkv, t = blockIdx.x, tid = threadIdx.x;
    const Kv8Seq sq = kv8_seq(p.c, p.len, p.n_new, b, p.T);
    if (t >= sq.n + sq.t0) return;
    const int pos = sq.len - (sq.n + sq.t0) + t;
    const size_t row = (size_t)blockIdx.y * p.T + t;
    int* out = p.blocks + row * p.top;
    const int n = pos < 0 ? 0 : pos / kKvBlock + 1;
    const int kept = min(n, p.top);
    for (int i = kept + tid; i < p.top; i += 256) out[i] = -1;
    if (n <= p.top) {
        for (int i = tid; i < n; i += 256) out[i] = i;
        return;
    }
    const float* score = p.score + row * p.nb;
    auto order = [&](int i) {
        return i < p.first || i >= n - 1 - p.recent ? 0xffffffffu : i < p.nb ? kv8_order(score[i]) : 0u;
    };
    unsigned value = 0;
    int left = p.top;  // of the values that share the bytes found so far, how many are kept
    for (int shift = 24; shift >= 0; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += 256) {
            const unsigned u = order(i);
            if (shift == 24 || u >> (shift + 8) == value >> (shift + 8)) atomicAdd(&hist[u >> shift & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int i = 255;
            while (hist[i] < left) left -= hist[i--];
            found[0] = i;
            found[1] = left;
        }
        __syncthreads();
        value |= (unsigned)found[0] << shift;
        left = found[1];
        __syncthreads();
    }
    // those above `value`, and the first `left` equal to it, in order
    int done = 0, equal = 0;
    for (int i0 = 0; i0 < n; i0 += 256) {
        const int i = i0 + tid;
        const unsigned u = i < n ? order(i) : 0;
        const bool eq = i < n && u == value;
        const unsigned long long eqs = __ballot(eq), below = (1ull << (tid & 63)) - 1;
        if ((tid & 63) == 0) sums[0][tid >> 6] = __popcll(eqs);
        __syncthreads();
        int before = equal + __popcll(eqs & below);
        for (int w = 0; w < tid >> 6; ++w) before += sums[0][w];
        const bool take = i < n && (u > value || (eq && before < left));
        const unsigned long long takes = __ballot(take);
        if ((tid & 63) == 0) sums[1][tid >> 6] = __popcll(takes);
        __syncthreads();
        int at = done + __popcll(takes & below);
        for (int w = 0; w < tid >> 6; ++w) at += sums[1][w];
        if (take) out[at] = i;
        for (int w = 0; w < 4; ++w) {
            equal += sums[0][w];
            done += sums[1][w];
        }
        __syncthreads();
    }
}

inline size_t kv8_select_qc_bytes(int B, int T, int Hq, int D) { return ((size_t)B * T * Hq * D + 255) / 256 * 256; }
inline size_t kv8_select_bytes(int B, int T, int Hq, int Hkv, int D, int nb) {
    return kv8_select_qc_bytes(B, T, Hq, D) + (size_t)B * Hkv * T * nb * 4;
}

template <int D>
hipError_t kv8_select_d(const Kv8SelectArgs& p, hipStream_t stream) {
    const dim3 rows((unsigned)p.T, (unsigned)(p.c.B * p.c.Hkv));
    hipLaunchKernelGGL(kv8_qcode_kernel<D>, rows, dim3(256), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)((p.nb + 255) / 256 * p.T), (unsigned)(p.c.B * p.c.Hkv));
    hipLaunchKernelGGL(kv8_score_kernel<D>, grid, dim3(256), p.G * D, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kv8_pick_kernel, rows, dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace

hipError_t kv8_select(const Kv8& c, const Rows16& q, const int* len, const int* n_new, int T, int Hq, int top, int first,
                      int recent, int* blocks, int nb, void* ws, hipStream_t stream) {
    const Kv8SelectArgs p{c, q, len, n_new, (signed char*)ws, (float*)((char*)ws + kv8_select_qc_bytes(c.B, T, Hq, c.D)),
                          blocks, T, Hq, Hq / c.Hkv, top, first, recent, nb};
    if (c.D == 64) return kv8_select_d<64>(p, stream);
    if (c.D == 128) return kv8_select_d<128>(p, stream);
    return kv8_select_d<256>(p, stream);
}

size_t kv8_ws_bytes(int B, int T, int Hq, int Hkv, int D, int nb, int top) {
    const bool list = top > 0;
    const size_t part = kv8_part_bytes(B, T, Hq, Hkv, D, kv8_splits(kv8_tiles(B, T, Hq, Hkv, list), list ? top : nb));
    const size_t sel = list ? kv8_select_bytes(B, T, Hq, Hkv, D, nb) : 0;
    return part > sel ? part : sel;
}

}  // namespace tsa
