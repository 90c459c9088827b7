// Checks of the paged cache that its entry points share (kv_paged.hip,
// attention_paged.hip).
#pragma once

#include <cstdint>

#include "vm_hip.h"

namespace vmhip {

// VM_HIP_EINVAL with a message that names `who`, or 0.
int check_kv_paged(const vm_hip_kv_paged* c, const char* who);
int check_page_size(int64_t page_size, const char* who);

inline int log2_of(int64_t power) {
    int s = 0;
    while ((int64_t{1} << s) < power) ++s;
    return s;
}

}  // namespace vmhip
