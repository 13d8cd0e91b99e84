// kv8_cache.h -- writing the 8-bit K/V cache and reading it back (see kv8.h for the format).
//
//   write  a = max|x| over a full block of one head, scale = a / 127, code = rint(127 x / a).
//          127 x has at most 18 bits, so the fp32 quotient rounds to the code of the real numbers
//          (a quotient that is not halfway between two codes is at least 2^-19 of its value away
//          from there, an fp32 rounding at most 2^-24): codes do not depend on how a prompt is cut
//          into calls.  A block with an infinity or NaN gets the scale NaN and codes 0.
//          The keys' summary is the sum of a block's codes, whole numbers, in 8 bits of its own.
//   read   value = code * scale rounded to fp16; rows of the open block as they were given.
#pragma once
#include "kv8.h"

namespace tsa {
namespace {

// A thread moves patches of 4 keys x 8 d: a row's 8 d are 16 bytes, and 4 keys of one d are one
// word of V's codes.  2 D patches a block, 256 threads (128 at D = 64).
template <int D>
constexpr int kv8_threads() {
    return D == 64 ? 128 : 256;
}
// The codes go through LDS on their way from patches to 16-byte units in the page's order.  Unit u
// lies at u ^ (the bits of u that the lanes of a write differ in), so that they use all banks.
__device__ __forceinline__ int kv8_swz(bool isv, int u) { return u ^ ((isv ? u >> 6 : u >> 4) & 15); }

template <int D>
struct Kv8WriteLds {
    uint4 units[4 * D];
    int sum[D];
    int red[2];
};

// One block of K or V of one (sequence, head): the new rows into the ring where they may still be
// needed, and a full block's codes, scale and summary into its page.
template <int D, bool kV>
__device__ __forceinline__ void kv8_write_block(const Kv8& c, const half_t* __restrict__ rows, long long st,
                                                const Kv8Seq& sq, int b, int h, int blk, int last,
                                                Kv8WriteLds<D>& lds) {
    constexpr int kThreads = kv8_threads<D>(), kN = 2 * D / kThreads;
    const int tid = threadIdx.x;
    const int start = sq.len - sq.n;
    const int p0 = blk * kKvBlock;
    const int r0 = max(start - p0, 0);           // rows before it are in the ring
    const int r1 = min(sq.len - p0, kKvBlock);   // rows behind it are not there yet
    const int page = r1 == kKvBlock ? kv8_uniform_page(c, b, blk) : -1;
    half_t* ring = (kV ? c.v_open : c.k_open) + kv8_open_at<D>(c, b, h, blk);
    const half_t* in = rows + (long long)(sq.t0 + p0 - start) * st;  // row r at in + r * st
    half8_t x[kN][4];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        const int i = tid + n * kThreads, r = i / (D / 8) * 4, d = i % (D / 8) * 8;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[n][e] = half8_t{};
            if (r + e >= r0 && r + e < r1) x[n][e] = *reinterpret_cast<const half8_t*>(in + (long long)(r + e) * st + d);
        }
        if (blk >= last - 1) {
            if (!kV) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r + e >= r0 && r + e < r1) *reinterpret_cast<half8_t*>(ring + kv8_k_at<D>(r + e, d)) = x[n][e];
            } else if (r >= r0 && r + 4 <= r1) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    *reinterpret_cast<half4_t*>(ring + kv8_v_at<D>(r, d + j)) = half4_t{x[n][0][j], x[n][1][j], x[n][2][j], x[n][3][j]};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r + e >= r0 && r + e < r1)
#pragma unroll
                        for (int j = 0; j < 8; ++j) ring[kv8_v_at<D>(r + e, d + j)] = x[n][e][j];
            }
        }
        if (page >= 0 && r < r0) {  // the block's older rows
            if (!kV) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r + e < r0) x[n][e] = *reinterpret_cast<const half8_t*>(ring + kv8_k_at<D>(r + e, d));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const half4_t y = *reinterpret_cast<const half4_t*>(ring + kv8_v_at<D>(r, d + j));
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (r + e < r0) x[n][e][j] = y[e];
                }
            }
        }
    }
    if (page < 0) return;

    // max |x| as the bits of its fp16: infinities and NaN are at least 0x7c00
    typedef unsigned short ushort8_t __attribute__((ext_vector_type(8)));
    ushort8_t m8 = {};
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            m8 = __builtin_elementwise_max(m8, __builtin_bit_cast(ushort8_t, x[n][e]) & (unsigned short)0x7fff);
    int most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, (int)m8[j]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o));
    if (tid < 2) lds.red[tid] = tid;  // the largest |x|'s bits, and the largest |sum|, at least 1
    if (!kV && tid < D) lds.sum[tid] = 0;
    __syncthreads();
    if ((tid & 63) == 0) atomicMax(&lds.red[0], most);
    __syncthreads();
    most = lds.red[0];
    const bool finite = most < 0x7c00;
    const float a = finite ? (float)__builtin_bit_cast(half_t, (unsigned short)max(most, 1)) : 1.f;
    const float scale = finite ? a / 127.f : __builtin_nanf("");
    const float r = 1.f / a;
    const size_t head = (size_t)page * c.Hkv + h;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        const int i = tid + n * kThreads, row = i / (D / 8) * 4, d = i % (D / 8) * 8;
        unsigned q[4][8];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < 8; ++j) q[e][j] = kv8_code(finite ? (float)x[n][e][j] : 0.f, a, r);
        if (kV) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = kv8_v_at<D>(row, d + j);
                reinterpret_cast<unsigned*>(&lds.units[kv8_swz(true, at >> 4)])[(at & 15) >> 2] = kv8_pack(q[0][j], q[1][j], q[2][j], q[3][j]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = kv8_k_at<D>(row + e, d);
                reinterpret_cast<uint2*>(&lds.units[kv8_swz(false, at >> 4)])[(at & 15) >> 3] =
                    uint2{kv8_pack(q[e][0], q[e][1], q[e][2], q[e][3]), kv8_pack(q[e][4], q[e][5], q[e][6], q[e][7])};
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                atomicAdd(&lds.sum[d + j], (int)(q[0][j] + q[1][j] + q[2][j] + q[3][j] - 4u * __builtin_bit_cast(unsigned, kKvMagic)));
        }
    }
    __syncthreads();
    uint4* codes = reinterpret_cast<uint4*>((kV ? c.v : c.k) + head * (kKvBlock * D));
    for (int u = tid; u < 4 * D; u += kThreads) codes[u] = lds.units[kv8_swz(kV, u)];
    if (tid == 0) (kV ? c.v_scale : c.k_scale)[head] = scale;
    if (!kV) {
        const int sum = tid < D ? lds.sum[tid] : 0;
        most = abs(sum);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o));
        if ((tid & 63) == 0) atomicMax(&lds.red[1], most);
        __syncthreads();
        const float big = (float)lds.red[1];
        if (tid < D) c.k_sum[head * D + tid] = (signed char)(int)rintf(127.f * (float)sum / big);
        if (tid == 0) c.k_sum_scale[head] = (scale * big) * (1.f / (kKvBlock * 127));
    }
}

// Workgroup (w, 2 h + isv, b): block w of those that the new tokens touch.  The first block's
// older rows are read from the ring slot that the last block but one or the last may overwrite:
// the first block's workgroup does that one too, afterwards.
template <int D>
__global__ void __launch_bounds__(kv8_threads<D>())
kv8_write_kernel(Kv8 c, Rows16 k, Rows16 v, const int* __restrict__ len, const int* __restrict__ n_new, int T) {
    __shared__ Kv8WriteLds<D> lds;
    const int w = blockIdx.x, h = blockIdx.y >> 1, b = blockIdx.z;
    const Kv8Seq sq = kv8_seq(c, len, n_new, b, T);
    if (sq.n == 0) return;
    const int first = (sq.len - sq.n) / kKvBlock, last = (sq.len - 1) / kKvBlock;
    int blk = first + w;
    // the block, other than the first, that writes the first's ring slot
    const int twin = last - ((last - first) & 1);
    if (blk > last || (w > 0 && blk == twin)) return;
    for (;;) {
        if (blockIdx.y & 1)
            kv8_write_block<D, true>(c, v.data + b * v.b + h * v.h, v.t, sq, b, h, blk, last, lds);
        else
            kv8_write_block<D, false>(c, k.data + b * k.b + h * k.h, k.t, sq, b, h, blk, last, lds);
        if (w > 0 || twin == blk) break;
        blk = twin;
        __syncthreads();
    }
}

// Workgroup (w, 2 h + isv, b): block w of those that rows start .. start + S - 1 touch.  Units of
// 16 codes in, rows through LDS (a pad of 16 bytes a row), 16 bytes of a row out, both past the
// caches (131072 tokens, 4 heads, D = 256: 155 -> 142 us, 5.7 TB/s).
template <int D>
__global__ void __launch_bounds__(kv8_threads<D>())
kv8_read_kernel(Kv8 c, const int* __restrict__ len, const int* __restrict__ start, int S, Rows16 k, Rows16 v) {
    constexpr int kThreads = kv8_threads<D>(), kN = 4 * D / kThreads, kRow = D + 8;
    __shared__ __align__(16) half_t tile[kKvBlock * kRow];
    const int h = blockIdx.y >> 1, b = blockIdx.z, tid = threadIdx.x;
    const bool isv = blockIdx.y & 1;
    const Rows16& x = isv ? v : k;
    if (!x.data) return;
    const int n = min(max(kv8_uniform(len + b), 0), c.max_blocks * kKvBlock);
    const int first = start ? max(kv8_uniform(start + b), 0) : 0;
    if (first >= n) return;
    const int blk = first / kKvBlock + blockIdx.x;
    if (blk >= c.max_blocks) return;
    const int p0 = blk * kKvBlock;
    const long long end = min((long long)n, (long long)first + S);
    const int r0 = max(first - p0, 0), r1 = (int)min(end - p0, (long long)kKvBlock);
    if (r1 <= r0) return;
    half8_t y[kN][2];
    if (p0 + kKvBlock > n) {
        const half8_t* ring = reinterpret_cast<const half8_t*>((isv ? c.v_open : c.k_open) + kv8_open_at<D>(c, b, h, blk));
#pragma unroll
        for (int i = 0; i < kN; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) y[i][j] = ring[2 * (tid + i * kThreads) + j];
    } else {
        const int page = kv8_uniform_page(c, b, blk);
        if (page < 0) return;
        const size_t head = (size_t)page * c.Hkv + h;
        const uint4* codes = reinterpret_cast<const uint4*>((isv ? c.v : c.k) + head * (kKvBlock * D));
        uint4 w[kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) w[i] = kv8_codes<true>(codes + tid + i * kThreads);
        const float scale = (isv ? c.v_scale : c.k_scale)[head], off = -128.f * scale;
        // (code + 128) scale - 128 scale: one rounding, of code * scale
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const unsigned u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int j = 0; j < 16; ++j)
                y[i][j >> 3][j & 7] = (half_t)__builtin_fmaf((float)(u[j >> 2] >> (8 * (j & 3)) & 255u), scale, off);
        }
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        const int u = tid + i * kThreads;
        if (isv) {
            const int t = u >> 6, d = t % (D / 32) * 32 + (u & 15), r = t / (D / 32) * 32 + ((u >> 4) & 3) * 4;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                tile[(r + ((j >> 2) & 1) * 16 + (j & 3)) * kRow + d + (j >> 3) * 16] = y[i][j >> 3][j & 7];
        } else {
            const int t = u >> 6, r = t / (D / 64) * 16 + (u & 15), d = t % (D / 64) * 64 + ((u >> 4) & 3) * 16;
#pragma unroll
            for (int j = 0; j < 2; ++j) *reinterpret_cast<half8_t*>(&tile[r * kRow + d + 8 * j]) = y[i][j];
        }
    }
    __syncthreads();
    half_t* rows = x.data + b * x.b + h * x.h + (long long)(p0 - first) * x.t;
    for (int i = tid + r0 * (D / 8); i < r1 * (D / 8); i += kThreads) {
        const int r = i / (D / 8), d = i % (D / 8) * 8;
        __builtin_nontemporal_store(*reinterpret_cast<const half8_t*>(&tile[r * kRow + d]), reinterpret_cast<half8_t*>(rows + r * x.t + d));
    }
}

}  // namespace

hipError_t kv8_write(const Kv8& c, const Rows16& k, const Rows16& v, const int* len, const int* n_new, int T,
                     hipStream_t stream) {
    // T rows in a row touch at most this many blocks
    const dim3 grid((unsigned)((T + 62) / kKvBlock + 1), (unsigned)(2 * c.Hkv), (unsigned)c.B);
    if (c.D == 64)
        hipLaunchKernelGGL(kv8_write_kernel<64>, grid, dim3(kv8_threads<64>()), 0, stream, c, k, v, len, n_new, T);
    else if (c.D == 128)
        hipLaunchKernelGGL(kv8_write_kernel<128>, grid, dim3(kv8_threads<128>()), 0, stream, c, k, v, len, n_new, T);
    else
        hipLaunchKernelGGL(kv8_write_kernel<256>, grid, dim3(kv8_threads<256>()), 0, stream, c, k, v, len, n_new, T);
    return hipGetLastError();
}

hipError_t kv8_read(const Kv8& c, const int* len, const int* start, int S, const Rows16& k, const Rows16& v,
                    hipStream_t stream) {
    const dim3 grid((unsigned)(start ? (S + 62) / kKvBlock + 1 : (S - 1) / kKvBlock + 1), (unsigned)(2 * c.Hkv), (unsigned)c.B);
    if (c.D == 64)
        hipLaunchKernelGGL(kv8_read_kernel<64>, grid, dim3(kv8_threads<64>()), 0, stream, c, len, start, S, k, v);
    else if (c.D == 128)
        hipLaunchKernelGGL(kv8_read_kernel<128>, grid, dim3(kv8_threads<128>()), 0, stream, c, len, start, S, k, v);
    else
        hipLaunchKernelGGL(kv8_read_kernel<256>, grid, dim3(kv8_threads<256>()), 0, stream, c, len, start, S, k, v);
    return hipGetLastError();
}

}  // namespace tsa
