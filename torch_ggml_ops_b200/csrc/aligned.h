// Whether pointers that a C entry was given are multiples of n bytes (null is): a kernel that reads at another address faults.
#pragma once

#include <cstdint>

namespace tgo {

template <typename... P>
bool aligned_to(uintptr_t n, P... p) {
    return ((reinterpret_cast<uintptr_t>(p) % n == 0) && ...);
}
constexpr const char* kMisaligned = "pointers must be aligned to their types";

}  // namespace tgo
