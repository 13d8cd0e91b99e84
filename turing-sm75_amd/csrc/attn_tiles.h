// attn_tiles.h -- tiles of rows in LDS, as the attention kernels share them: the bank swizzle, the
// operand reads and the copies from global memory.
#pragma once
#include "common.h"

namespace tsa {

// 16-byte chunk swizzle of an LDS tile row: chunk c of row r lives at c ^ swz<D>(r).
// LDS has 64 banks of 4 bytes; a 256-byte D = 128 row spans all of them, so a chunk's
// banks depend on its position only.  The K operand reads (ds_read_b128, 16 lanes per
// cycle) take 16 consecutive rows at one chunk: swz is a permutation of r % 16.  The
// transposing V reads (ds_read_b64_tr_b16, 32 lanes per cycle) take 4 aligned rows x 4
// chunks of one aligned chunk block: swz moves the 4 rows to 4 different chunk blocks.
// At D = 64 two rows share the 64 banks and the other formula keeps both read patterns
// conflict free.
template <int D>
__device__ __forceinline__ int swz(int r) {
    if (D >= 128) return 4 * (r & 3) + ((r >> 2) & 3);  // D = 256: a row is two bank periods
    return (2 * (r & 3) + ((r >> 2) & 1)) & 7;
}

template <int D>
__device__ __forceinline__ int chunk_pos(int r, int c) {
    return c ^ swz<D>(r);
}

typedef __attribute__((address_space(3))) void* lds_void_t;

// LDS reads at a byte address held as an integer (so that address arithmetic can be an
// XOR with an immediate plus an offset folded into the instruction).
__device__ __forceinline__ half8_t lds_read_b128(unsigned addr) {
    typedef __attribute__((address_space(3))) const half8_t* p_t;
    return *(p_t)(addr);
}
__device__ __forceinline__ half4_t lds_read_tr16_at(unsigned addr) {
    typedef __attribute__((address_space(3))) fp16x4_t* p_t;
    return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((p_t)(addr)));
}

// src = base + off (64-bit base in SGPRs, 32-bit VGPR offset).  Inline asm on purpose:
// the compiler does not track LDS written by DMA per buffer and would wait for every
// copy in flight before the first LDS read of the other buffer; the kernel orders the
// copies itself (vmcnt(0) and a barrier at the end of each tile).
__device__ __forceinline__ void dma_issue(const void* base, unsigned off, unsigned lds_addr) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "{m0}"(lds_addr)
                 : "memory");
}
// The same for kernels with many scalar values, whose base may have come back from a vector register
// (v_readlane) just before: the compiler does not see that the asm reads it as an address, which takes
// five wait states after such a write, and gives none.  A scalar move waits for it by itself, and
// nothing has to wait for the move.
__device__ __forceinline__ void dma_issue_any(const void* base, unsigned off, unsigned lds_addr) {
    const void* at;
    asm volatile("s_mov_b64 %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0"
                 : "=&s"(at) : "v"(off), "s"(base), "{m0}"(lds_addr) : "memory");
}
// One dword a lane (256 bytes).
__device__ __forceinline__ void dma_issue_any4(const void* base, unsigned off, unsigned lds_addr) {
    const void* at;
    asm volatile("s_mov_b64 %0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, %0"
                 : "=&s"(at) : "v"(off), "s"(base), "{m0}"(lds_addr) : "memory");
}
__device__ __forceinline__ void dma_wait_barrier() {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's copies have landed
    lds_barrier();
}

}  // namespace tsa
