// Norm over many gradient tensors: what its launcher hands to the kernels that clip by it (gradnorm.hip, optim.hip).
#pragma once

#include "gsr_common.h"
#include "plan.h"

namespace gsr {

// Workgroups of a launch of the norm pass at most, and so its partial results.
constexpr int kNormBlocks = 512;
// Partial results that every clipping wave joins by itself; more of them (over 480 tensors) are joined by a kernel of
// their own first, which costs a launch (4 us) but not their reading by every wave.
constexpr int kMostJoined = 4 * kNormBlocks;
// Descriptors of a launch: 24 bytes each, 2.9 KB of kernel arguments, which every launch copies.  A choice, not a limit
// that was found: more of them a launch have not been measured.
constexpr int kGradsPerLaunch = 120;

// Writes the partial results of all gradients to `partials` (norm_partials_most(count) doubles) and their number to
// *used (0 when there is no element, at most kMostJoined).  Arguments have been checked.
int norm_partials(int count, const GsrGrad* h_grads, int norm_type, double* partials, int* used, hipStream_t stream);
inline size_t norm_partials_most(int count) { return kNormBlocks * ((size_t)count / kGradsPerLaunch + 1); }
// GSR_OK if the list, the norm's type and the scratch are usable; the message names `what`.
int check_norm(const char* what, int count, const GsrGrad* h_grads, int norm_type, const float* norm, const void* scratch,
               size_t scratch_bytes);

// Joins two partial results.  A maximum keeps a NaN once it has met one, as the sums do by themselves.
template <int NORM>
__device__ __forceinline__ double norm_join(double a, double b) {
  if (NORM == GSR_NORM_MAX) return b > a || b != b ? b : a;
  return a + b;
}

// Joins the 64 lanes' results; every lane gets the same bits (each step adds the same two numbers in both lanes).
template <int NORM>
__device__ __forceinline__ double norm_join_wave(double v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = norm_join<NORM>(v, __shfl_xor(v, d));
  return v;
}

// The norm from the partial results, by each wave for itself: no barrier, and the same order in every wave of a
// launch, so that all of them clip by the same bits.  Eight requests of a lane are under way at once (the results come
// from the other XCDs' workgroups, past the L2: one after the other 512 of them take 4.7 us).
template <int NORM>
__device__ __forceinline__ double norm_of_partials(const double* __restrict__ partials, int used) {
  double v = 0.0;
  for (int first = threadIdx.x & 63; first < used; first += 8 * 64) {
    double p[8];
#pragma unroll
    for (int k = 0; k < 8; k++) p[k] = first + 64 * k < used ? partials[first + 64 * k] : 0.0;   // zeros add nothing
#pragma unroll
    for (int k = 0; k < 8; k++) v = norm_join<NORM>(v, p[k]);
  }
  v = norm_join_wave<NORM>(v);
  return NORM == GSR_NORM_2 ? sqrt(v) : v;
}

// min(1, max_norm / (norm + 1e-6)), the rule of torch.nn.utils.clip_grad_norm_: a NaN norm gives NaN, an infinite one 0.
// An infinite bound never clips.
__device__ __forceinline__ float clip_coefficient(double norm, double max_norm) {
  if (max_norm == __builtin_inf()) return 1.0f;
  const double c = max_norm / (norm + 1e-6);
  return c < 1.0 || c != c ? (float)c : 1.0f;
}

}  // namespace gsr
