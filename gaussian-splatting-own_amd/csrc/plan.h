// What the launchers of the many-tensor operators decide by arithmetic alone.  No GPU header is needed, so that the tests
// compile this file by itself and drive the code that the library runs.
#pragma once

#include <cstddef>
#include <cstdint>

#include "../../include/gsr.h"

#if defined(__HIPCC__)
#define GSR_BOTH_SIDES __host__ __device__ __forceinline__
#else
#define GSR_BOTH_SIDES inline
#endif

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

// n / d for every 32-bit n by a multiplication (Granlund and Montgomery 1994, the round-up method): with
// l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1, q = (t + ((n - t) >> 1)) >> (l - 1), t = mulhi(m, n); d > 1.
struct Divisor {
  uint32_t d, m, shift;
  GSR_BOTH_SIDES uint32_t quotient(uint32_t n) const {
    if (d == 1) return n;
    const uint32_t t = (uint32_t)(((uint64_t)m * n) >> 32);
    return (t + ((n - t) >> 1)) >> shift;
  }
};

inline Divisor divisor(uint32_t d) {
  Divisor v = {d, 0, 0};
  if (d > 1) {
    uint32_t l = 0;
    while ((1ull << l) < d) l++;
    v.m = (uint32_t)(((((uint64_t)1 << l) - d) << 32) / d + 1);
    v.shift = l - 1;
  }
  return v;
}

// Whether a vector, which begins at a multiple of K units of the output, never reaches into a third row: column and
// length together stay below two rows.  All rows of 15 bytes and more, and those that divide a vector in half.
inline bool lies_in_two_rows(uint32_t units, uint32_t unit) {
  const uint32_t k = 16 / unit;
  return units + k - 2 < 2 * units || 2 * units == k;
}

}  // namespace gsr
