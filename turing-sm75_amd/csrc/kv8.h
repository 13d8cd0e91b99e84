// kv8.h -- the 8-bit K/V cache: where its elements lie, shared by the kernels that write it
// (kv8_cache.h), attend to it (kv8_attn.h) and select blocks of it (kv8_select.h).
//
// A block is 64 tokens of one sequence.  A full block of one K/V head is 64 x D codes, a byte
// each (code + 128, code = rint(127 x / max|x|) in -127 .. 127), with one fp32 scale max|x| / 127.
// The tokens behind the last full block are fp16 rows in a ring of two blocks per sequence, block i
// in slot i % 2.  A write keeps its rows of the last block that it touches and of the one before, so
// a sequence may be cut back to any length in the two blocks at its longest length's end, as far as
// it wrote them itself; further back only to whole blocks, which need no row of the ring.  (After
// 129 tokens, a cut to 65 and one more, block 0 is still not in the ring: slot 0 is block 2's.)
//
// Both are laid out as the operands of v_mfma_f32_16x16x32_f16 (lane l holds row l % 16 and 8
// consecutive k at 8 * (l / 16)), so that a wave reads 1 KiB of consecutive codes per load, 16
// bytes a lane, and no transpose is left for the attention:
//   K, operand A of S^T = K Q^T: the 16 bytes of lane l in tile (a, i) are key 16 a + l % 16,
//      d = 64 i + 16 (l / 16) + 0 .. 15: the first 8 are one k-step, the last 8 another (k is
//      any order of d that Q follows too);
//   V, operand A of O^T = V^T P^T: the 16 bytes of lane l in tile (s, m) are keys 32 s + 16 i +
//      4 (l / 16) + e of d = 32 m + 16 o + l % 16 for byte 8 o + 4 i + e: the keys whose P the lane
//      holds after S^T, so P needs no exchange.  The first 8 bytes are tile 2 m of O^T, the others
//      2 m + 1.
// Both halves of a block (32 keys) are consecutive.  The ring holds its fp16 elements in the same
// order.
#pragma once
#include <stdint.h>

#include "common.h"
#include "kernels.h"

namespace tsa {
namespace {

constexpr int kKvBlock = 64;

// Element offset of (key r, d) within a block of one head.
template <int D>
__device__ __forceinline__ int kv8_k_at(int r, int d) {
    return ((((r >> 4) * (D / 64) + (d >> 6)) * 4 + ((d >> 4) & 3)) * 16 + (r & 15)) * 16 + (d & 15);
}
template <int D>
__device__ __forceinline__ int kv8_v_at(int r, int d) {
    return ((((r >> 5) * (D / 32) + (d >> 5)) * 4 + ((r >> 2) & 3)) * 16 + (d & 15)) * 16 + ((d >> 4) & 1) * 8 +
           ((r >> 4) & 1) * 4 + (r & 3);
}

// 127 x / a as a division would round it (with r = 1 / a rounded, one correction of y r by its exact
// remainder gives the correctly rounded quotient), then to a whole number, ties to even: the sum
// with 1.5 2^23 + 128 leaves rint(127 x / a) + 128 in its low byte.
constexpr float kKvMagic = 12582912.f + 128.f;
__device__ __forceinline__ unsigned kv8_code(float x, float a, float r) {
    const float y = 127.f * x, q = y * r;
    return __builtin_bit_cast(unsigned, __builtin_fmaf(__builtin_fmaf(-q, a, y), r, q) + kKvMagic);
}
// The low bytes of four words.
__device__ __forceinline__ unsigned kv8_pack(unsigned b0, unsigned b1, unsigned b2, unsigned b3) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b3, b2, 0x0c0c0400u), __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u), 0x05040100u);
}

// A value at an address that is the same on all lanes and that the kernel does not write: a scalar
// load (the compiler takes a vector load where it cannot see that).
template <typename T>
__device__ __forceinline__ T kv8_uniform(const T* p) {
    return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// 16 codes.  kOnce: no other workgroup of the call reads them, unless sequences share their pages, and
// they pass the caches by (attention of one token each for 32 sequences of up to 32768, D = 256: 308 ->
// 283 us; where queries share their blocks, 115 -> 184 us).  Sequences that share pages pay for it: the
// host does not see their tables, and pages of a sequence's own are taken for the common case (32 x
// 32768, 24/4 heads, D = 256: own pages 378 us past the caches and 403 through them, all pages shared
// 194 and 132).
template <bool kOnce>
__device__ __forceinline__ uint4 kv8_codes(const uint4* p) {
    typedef unsigned uint4_v __attribute__((ext_vector_type(4)));
    const uint4_v* q = reinterpret_cast<const uint4_v*>(p);
    return __builtin_bit_cast(uint4, kOnce ? __builtin_nontemporal_load(q) : *q);
}

// A sequence's tokens: `len` of them, the last `n` new; rows of a call's T start at new row `t0`
// (rows before it would lie in front of the sequence).  Every count is clamped to what the cache
// and the call hold, so that no value of the device arrays leads out of bounds.
struct Kv8Seq {
    int len, n, t0;
};
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8& c, const int* __restrict__ len, const int* __restrict__ n_new,
                                          int b, int T) {
    Kv8Seq s;
    s.len = min(max(kv8_uniform(len + b), 0), c.max_blocks * kKvBlock);
    const int n = n_new ? min(max(kv8_uniform(n_new + b), 0), T) : T;
    s.n = min(n, s.len);
    s.t0 = n - s.n;
    return s;
}

// The page of block `blk` of sequence b, -1 where the table names none.
__device__ __forceinline__ int kv8_page(const Kv8& c, int b, int blk) {
    const int p = c.table[(size_t)b * c.max_blocks + blk];
    return p >= 0 && p < c.n_pages ? p : -1;
}

// The same, sequence and block being the same on all lanes.
__device__ __forceinline__ int kv8_uniform_page(const Kv8& c, int b, int blk) {
    const int p = kv8_uniform(c.table + (size_t)b * c.max_blocks + blk);
    return p >= 0 && p < c.n_pages ? p : -1;
}

// The ring's fp16 block of (sequence, head) that block blk uses, as an element offset.
template <int D>
__device__ __forceinline__ size_t kv8_open_at(const Kv8& c, int b, int h, int blk) {
    return ((size_t)(b * 2 + (blk & 1)) * c.Hkv + h) * (kKvBlock * D);
}

}  // namespace
}  // namespace tsa
