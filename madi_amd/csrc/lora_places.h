// lora_places.h -- where the adapters' kernels (lora.hip) read a row of x.  Plain C++: a test goes through it on the host.
#pragma once

#include <stdint.h>

namespace madi {

// The element of a row of k (a multiple of 64) at which a load of four starts that is to take `at`, a multiple of 4:
// past the row's end the row's last four elements, so that no load is behind a branch and none outside the row.
constexpr uint32_t lora_x_place(uint32_t at, uint32_t k) { return at < k ? at : k - 4; }

}  // namespace madi
