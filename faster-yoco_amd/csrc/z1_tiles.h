// Device helpers shared by the kernels that multiply tiles by matrix instructions (8-bit products, matrices' updates); not part
// of the C ABI.
#pragma once

#include "z1_block.h"

namespace z1blk {

typedef int i8 __attribute__((ext_vector_type(8)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f16 __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

#define Z1B_LDS __attribute__((address_space(3)))

// The 32 x 32 result of a matrix instruction gives lane l column l % 32 and rows 8 (i/4) + 4 (l/32) + i%4, i = 0..15.
// Reading its first operand's rows in this order makes those 16 consecutive: 16 (l/32) + i.
__device__ __forceinline__ int spread(int row) { return 16 * ((row >> 2) & 1) + 4 * (row >> 3) + (row & 3); }

// All waves of the workgroup are here, their reads from LDS are done, and of their loads all but the LATER last ones have
// arrived, direct loads into LDS among them.
template <int LATER = 0>
__device__ __forceinline__ void meet() {
    static_assert(LATER < 64, "the counter's range");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LATER) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A raw buffer of `bytes` (none where negative) from p: loads whose lane offset lies past it give zeros (word 3: the raw
// 32-bit data format).  The scalar offset of a load need not count in that check: it only moves within a row's own bytes.
// Without a branch: a loop around it keeps its loads on their way.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int64_t bytes) {
    const uint32_t low = (uint32_t)bytes, high = (uint32_t)(bytes >> 32);
    const uint32_t n = (low | (uint32_t)-(int)(high != 0)) & ~(uint32_t)((int)high >> 31);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)n, 0x00020000);
}
// 16 bytes a lane, straight into LDS at `to` + 16 * lane.
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t from, void* to, int lane_at, int at) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Z1B_LDS void*)to, 16, lane_at, at, 0, 0);
}

// Staging keeps rows of 128 bytes (one block of K).  A lane of a direct load writes 16 bytes at its own place in a run of
// 1024, so the order of a row's eight 16-byte pieces is changed at the source: piece p of a row lies at p ^ key(row).  LDS
// has 64 banks of 4 bytes, two rows: the 16 rows that neighbouring lanes read together are eight of either parity, with
// eight different keys.
__device__ __forceinline__ int key_plain(int row) { return row >> 1 & 7; }
__device__ __forceinline__ int key_spread(int row) { return (row >> 1 & 3) | (row >> 4 & 1) << 2; }

}  // namespace z1blk
