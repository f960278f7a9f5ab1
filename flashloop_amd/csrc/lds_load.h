// Transfers from memory to LDS without registers in between (mx_matmul.hip, paged_attention.hip).
#pragma once

#include "fl_common.h"

namespace fl {
namespace {

typedef int32_t lds_buffer_t __attribute__((ext_vector_type(4)));  // a buffer resource, wave-uniform
typedef __attribute__((address_space(3))) uint8_t lds_u8;

// A raw buffer over `bytes` bytes at p (wave-uniform): what a load finds past the end is zero.  Word 3
// is the gfx9 raw-buffer format.
__device__ __forceinline__ lds_buffer_t raw_buffer(const void* p, int64_t bytes) {
  const uint64_t u = reinterpret_cast<uintptr_t>(p);
  return lds_buffer_t{__builtin_amdgcn_readfirstlane(static_cast<int>(u)), __builtin_amdgcn_readfirstlane(static_cast<int>(u >> 32)),
                    __builtin_amdgcn_readfirstlane(static_cast<int>(min(bytes, static_cast<int64_t>(0x7FFFFFFF)))), 0x00020000};
}

// Memory to LDS: lane l's 16 (or 4) bytes of buffer r at voff + soff go to lds + 16 (4) l.  The compiler counts
// no LDS write for these, so the kernel waits for them itself (vmcnt, ahead of the step's barrier).  m0 is
// on the clobber list for what else a compiler sets it for; its warning says that no one saves it here.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int BYTES>
__device__ __forceinline__ void to_lds(lds_buffer_t r, uint32_t voff, uint32_t soff, uint32_t lds) {
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(r), "s"(soff)
                 : "m0", "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(r), "s"(soff)
                 : "m0", "memory");
}
#pragma clang diagnostic pop

}  // namespace
}  // namespace fl
