// Copies from memory into LDS by the memory pipeline, and transposed reads from there (token operators).
#pragma once
#include "common.h"

namespace sengine {

// One LDS copy: 64 lanes x 16 bytes from rsrc at each lane's offset to LDS bytes dst..dst + 1023; lanes out of
// the buffer's range write zeros.  Written as asm so that later LDS reads do not wait for it: the caller waits
// (vmcnt) and, where other waves copied too, meets them at a barrier.  It returns nothing in registers.
// A memory instruction reads an SGPR that a VALU instruction wrote only five wait states later, and the descriptor
// comes from one (v_readfirstlane, or v_readlane where it was spilled): the compiler, which does not see the load,
// cannot put them, so the move and the s_nop are those five.  m0 is named as written, so that no use of the compiler's
// own is moved across; that it is not saved, which the compiler then warns of, is as it should be.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void lds_copy(u32x4_t rsrc, uint32_t dst, int voff) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 3\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(dst), "v"(voff), "s"(rsrc)
      : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ __forceinline__ uint32_t scalar(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// Buffer of `bytes` bytes from base (both the same in all lanes).
__device__ __forceinline__ u32x4_t row_buffer(const uint8_t* base, int bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)base;
  return u32x4_t{scalar((uint32_t)a), scalar((uint32_t)(a >> 32) & 0xffffu), scalar((uint32_t)bytes),
                 (uint32_t)kBufferDword3};
}

__device__ __forceinline__ uint32_t lds_offset(const uint8_t* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
}

// Two transposed reads of 16-bit values.  Sixteen lanes name 4 rows of 16 values, lane a the values
// 4 (a % 4).. of row a / 4; lane a then has the four rows' value a.  The first read is the low half.
__device__ __forceinline__ u32x4_t read_transposed(const uint8_t* lo, const uint8_t* hi) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4* ptr_t;
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr_t)lo));
  const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr_t)hi));
  return u32x4_t{a[0], a[1], b[0], b[1]};
}

// Workgroup id -> place in an order of which each of the eight XCDs, to which workgroups go in turn, takes one
// contiguous range.
__device__ __forceinline__ int xcd_order(int id, int total) {
  const int per = total >> 3, rest = total & 7, xcd = id & 7;
  return xcd * per + (xcd < rest ? xcd : rest) + (id >> 3);
}

}  // namespace sengine
