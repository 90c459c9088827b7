// Loads from memory to LDS that skip registers.
#pragma once

#include <cstdint>

namespace vmhip {

// Sixteen bytes a lane from memory (a uniform address and a lane's offset) to
// LDS, lane by lane behind `to` (uniform).  Written as a statement of its own
// because the compiler would have every LDS read wait for it, also reads of
// another buffer; wait_loads() waits.  What the compiler sees to for its own
// instructions is done here.  m0, which says where to, is an operand, so that the
// compiler writes it and knows.  A load may follow one wait state behind m0's write,
// five behind a vector instruction that wrote its address (v_readfirstlane, v_readlane
// of a register kept elsewhere), and at once behind a scalar one, which waits for the
// vector instruction by itself: the address is moved onto itself (five states
// instead: 32 heads of 128, f16, 500 tokens behind 30000 298 us for 295).
__device__ __forceinline__ void lds_load16(const char* from, uint32_t offset, char* to) {
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(to)));
    asm volatile("s_mov_b64 %2, %2\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "{m0}"(__builtin_amdgcn_readfirstlane(at)), "v"(offset), "s"(from)
                 : "memory");
}

__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }

}  // namespace vmhip
