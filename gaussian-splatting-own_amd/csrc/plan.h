// What the launchers of the many-tensor operators decide by arithmetic alone.  No GPU header is needed, so that the tests
// compile this file by itself and drive the code that the library runs.
#pragma once

#include <cstddef>
#include <cstdint>

#include "../../include/gsr.h"

namespace gsr {

// What of the gradients the norm pass leaves in the last-level cache, for those that come to them next.
constexpr uint64_t kLastLevelBytes = 256ull << 20;

inline size_t size_of(uint64_t type) { return type == GSR_F32 ? 4 : 2; }

// Whether the gradients of a list take more than that: in bytes, for a long list of short tensors has many chunks and
// little in them.
inline bool past_last_level(int count, const GsrGrad* h_grads) {
  uint64_t bytes = 0;
  for (int k = 0; k < count; k++) bytes += h_grads[k].n * size_of(h_grads[k].type);
  return bytes > kLastLevelBytes;
}

}  // namespace gsr
