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

constexpr int kKvThreads = 256;

// One block of K or V of one (sequence, head): the new rows into the ring where they may still be
// needed, and a full block's codes, scale and summary into its page.
template <int D>
__device__ void kv8_write_block(const Kv8& c, bool isv, const half_t* __restrict__ rows, long long st, const Kv8Seq& sq,
                                int b, int h, int blk, int last, half_t* tile, int* red) {
    const int tid = threadIdx.x;
    const int start = sq.len - sq.n;
    const int p0 = blk * kKvBlock;
    const int r0 = max(start - p0, 0);                    // rows before it are in the ring
    const int r1 = min(sq.len - p0, kKvBlock);            // rows behind it are not there yet
    const bool full = r1 == kKvBlock;
    half_t* ring = (isv ? c.v_open : c.k_open) + kv8_open_at<D>(c, b, h, blk);
    if (blk >= last - 1) {
        for (int i = tid; i < (r1 - r0) * D; i += kKvThreads) {
            const int r = r0 + i / D, d = i % D;
            ring[kv8_at<D>(isv, r, d)] = rows[(long long)(sq.t0 + p0 + r - start) * st + d];
        }
    }
    if (!full) return;
    const int page = kv8_page(c, b, blk);
    if (page < 0) return;
    int most = 0;  // max |x| as the bits of its fp16: infinities and NaN are at least 0x7c00
    for (int i = tid; i < kKvBlock * D; i += kKvThreads) {
        const int r = i / D, d = i % D;
        const half_t x = r < r0 ? ring[kv8_at<D>(isv, r, d)] : rows[(long long)(sq.t0 + p0 + r - start) * st + d];
        tile[i] = x;
        most = max(most, (int)(__builtin_bit_cast(unsigned short, x) & 0x7fff));
    }
    if (tid == 0) red[0] = 0;
    __syncthreads();
    atomicMax(&red[0], most);
    __syncthreads();
    most = red[0];
    const bool finite = most < 0x7c00;
    const float a = (float)__builtin_bit_cast(half_t, (unsigned short)max(most, 1));
    const float scale = finite ? a / 127.f : __builtin_nanf("");
    const size_t head = (size_t)page * c.Hkv + h;
    unsigned char* codes = (isv ? c.v : c.k) + head * (kKvBlock * D);
    auto code = [&](int r, int d) { return finite ? (int)rintf(127.f * (float)tile[r * D + d] / a) : 0; };
    for (int i = tid; i < kKvBlock * D; i += kKvThreads) {
        const int r = i / D, d = i % D;
        codes[kv8_at<D>(isv, r, d)] = (unsigned char)(code(r, d) + 128);
    }
    if (tid == 0) (isv ? c.v_scale : c.k_scale)[head] = scale;
    if (!isv) {
        int sum = 0;
        if (tid < D)
            for (int r = 0; r < kKvBlock; ++r) sum += code(r, tid);
        if (tid == 0) red[1] = 1;
        __syncthreads();
        if (tid < D) atomicMax(&red[1], abs(sum));
        __syncthreads();
        const float big = (float)red[1];
        if (tid < D) c.k_sum[head * D + tid] = (signed char)(int)rintf(127.f * (float)sum / big);
        if (tid == 0) c.k_sum_scale[head] = (scale * big) * (1.f / (kKvBlock * 127));
    }
}

// Workgroup (w, 2 h + isv, b): block w of those that the new tokens touch.  The first block's
// older rows are read from the ring slot that the last block but one or the last may overwrite:
// the first block's workgroup does that one too, afterwards.
template <int D>
__global__ void __launch_bounds__(kKvThreads)
kv8_write_kernel(Kv8 c, Rows16 k, Rows16 v, const int* __restrict__ len, const int* __restrict__ n_new, int T) {
    __shared__ half_t tile[kKvBlock * D];
    __shared__ int red[2];
    const int w = blockIdx.x, h = blockIdx.y >> 1, b = blockIdx.z;
    const bool isv = blockIdx.y & 1;
    const Kv8Seq sq = kv8_seq(c, len, n_new, b, T);
    if (sq.n == 0) return;
    const int first = (sq.len - sq.n) / kKvBlock, last = (sq.len - 1) / kKvBlock;
    const int blk = first + w;
    if (blk > last) return;
    // the block, other than the first, that writes the first's ring slot
    const int twin = last - ((last - first) & 1);
    if (w > 0 && blk == twin) return;
    const Rows16& x = isv ? v : k;
    const half_t* rows = x.data + b * x.b + h * x.h;
    kv8_write_block<D>(c, isv, rows, x.t, sq, b, h, blk, last, tile, red);
    if (w == 0 && twin > first) {
        __syncthreads();
        kv8_write_block<D>(c, isv, rows, x.t, sq, b, h, twin, last, tile, red);
    }
}

// Workgroup (w, 2 h + isv, b): block w of those that rows start .. start + S - 1 touch.
template <int D>
__global__ void __launch_bounds__(kKvThreads)
kv8_read_kernel(Kv8 c, const int* __restrict__ len, const int* __restrict__ start, int S, Rows16 k, Rows16 v) {
    __shared__ half_t tile[kKvBlock * D];
    const int h = blockIdx.y >> 1, b = blockIdx.z, tid = threadIdx.x;
    const bool isv = blockIdx.y & 1;
    const int n = min(max(len[b], 0), c.max_blocks * kKvBlock);
    const int first = start ? max(start[b], 0) : 0;
    if (first >= n) return;
    const int blk = first / kKvBlock + blockIdx.x;
    if (blk >= c.max_blocks) return;
    const int p0 = blk * kKvBlock;
    const long long end = min((long long)n, (long long)first + S);
    const int r0 = max(first - p0, 0), r1 = (int)min(end - p0, (long long)kKvBlock);
    if (r1 <= r0) return;
    const bool open = p0 + kKvBlock > n;
    if (open) {
        const half_t* ring = (isv ? c.v_open : c.k_open) + kv8_open_at<D>(c, b, h, blk);
        for (int i = tid; i < kKvBlock * D; i += kKvThreads) tile[i] = ring[kv8_at<D>(isv, i / D, i % D)];
    } else {
        const int page = kv8_page(c, b, blk);
        if (page < 0) return;
        const size_t head = (size_t)page * c.Hkv + h;
        const unsigned char* codes = (isv ? c.v : c.k) + head * (kKvBlock * D);
        const float scale = (isv ? c.v_scale : c.k_scale)[head];
        for (int i = tid; i < kKvBlock * D; i += kKvThreads)
            tile[i] = (half_t)((float)((int)codes[kv8_at<D>(isv, i / D, i % D)] - 128) * scale);
    }
    __syncthreads();
    const Rows16& x = isv ? v : k;
    if (!x.data) return;
    half_t* rows = x.data + b * x.b + h * x.h;
    for (int i = tid + r0 * D; i < r1 * D; i += kKvThreads)
        rows[(long long)(p0 + i / D - first) * x.t + i % D] = tile[i];
}

}  // namespace

hipError_t kv8_write(const Kv8& c, const Rows16& k, const Rows16& v, const int* len, const int* n_new, int T,
                     hipStream_t stream) {
    const dim3 grid((unsigned)((T - 1) / kKvBlock + 2), (unsigned)(2 * c.Hkv), (unsigned)c.B);
    if (c.D == 64)
        hipLaunchKernelGGL(kv8_write_kernel<64>, grid, dim3(kKvThreads), 0, stream, c, k, v, len, n_new, T);
    else if (c.D == 128)
        hipLaunchKernelGGL(kv8_write_kernel<128>, grid, dim3(kKvThreads), 0, stream, c, k, v, len, n_new, T);
    else
        hipLaunchKernelGGL(kv8_write_kernel<256>, grid, dim3(kKvThreads), 0, stream, c, k, v, len, n_new, T);
    return hipGetLastError();
}

hipError_t kv8_read(const Kv8& c, const int* len, const int* start, int S, const Rows16& k, const Rows16& v,
                    hipStream_t stream) {
    // rows that start inside a block touch one block more
    const dim3 grid((unsigned)((S - 1) / kKvBlock + (start ? 2 : 1)), (unsigned)(2 * c.Hkv), (unsigned)c.B);
    if (c.D == 64)
        hipLaunchKernelGGL(kv8_read_kernel<64>, grid, dim3(kKvThreads), 0, stream, c, len, start, S, k, v);
    else if (c.D == 128)
        hipLaunchKernelGGL(kv8_read_kernel<128>, grid, dim3(kKvThreads), 0, stream, c, len, start, S, k, v);
    else
        hipLaunchKernelGGL(kv8_read_kernel<256>, grid, dim3(kKvThreads), 0, stream, c, len, start, S, k, v);
    return hipGetLastError();
}

}  // namespace tsa
