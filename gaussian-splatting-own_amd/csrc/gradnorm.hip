// Global norm over many gradient tensors, and clipping by it, on gfx950.
//
//     N = (sum_t sum_i |g_ti|^p)^(1/p)   p = 1, 2;   N = max |g_ti| for the maximum
//     g <- g min(1, max_norm / (N + 1e-6))
//
// What bounds both is HBM: the norm reads every gradient once (1.4 GB of fp32: 229 us, 6.2 TB/s; a copy of that size
// reaches 4.9), clipping reads it once more and writes it only where the coefficient is below 1 (236 MB: 136 us with two
// sets of gradients in turn, 102 on the same one again, part of which the caches still hold).  One
// launch walks the tensors of a list (their descriptors are kernel arguments: nothing is copied to the device, so a call
// can be captured into a graph); every workgroup leaves one partial result, and the kernel that clips joins those by
// itself instead of waiting for a kernel that would.
//
// The sums are held in 64 bits: squares of the whole fp32 range neither overflow nor vanish, and the result does not
// depend on how many workgroups shared the work beyond its last bits.  They are not what bounds it: 240 MB in 61 tensors
// take 46.5 us as bf16, 46.1 as fp16 and 46.2 as fp32, which has half the elements.  Behind a clip that has written the
// tensors it is 64 us: the written lines are still on their way out.
#include "gradnorm.h"

#include <algorithm>
#include <new>

namespace {

using gsr::global_at;
using gsr::kGradsPerLaunch;
using gsr::kNormBlocks;
using gsr::size_of;

// 1.4 GB and 236 MB of fp32, norm alone: 230 and 37.6 us with 512 workgroups (kNormBlocks) of 512 threads and four
// accesses in flight; 1024 workgroups 237 / 40, 256 of them 265 / 37.5; 1024 workgroups of 256 threads 233 / 40, 256 of
// 1024 235 / 37; two accesses 227 / 38 (but the clip 842 us instead of 795), eight 236 / 38.
constexpr int kBlock = 512;
constexpr int kRounds = 4;                                   // 16-byte accesses of a thread in flight
constexpr uint32_t kChunk = kBlock * kRounds * 16;           // bytes
constexpr uint32_t kClipBlocks = 1024;                       // workgroups of a clipping launch at most

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Tensors are cut into chunks at 16-byte boundaries of the address, so that every access inside is aligned whatever
// the tensor's own alignment; its first and last vectors may be cut and go element by element.
struct GradChunk {
  uintptr_t begin, end;
  uint32_t first;                                            // number of its first chunk
  uint32_t type;
};
// MOST: a short list is handed over in a short structure (every launch copies its arguments: 3 KB of them cost the
// host half a microsecond and the kernel's first loads more).
template <int MOST>
struct GradChunks {
  uint32_t chunks;
  int count;
  GradChunk t[MOST];
};
constexpr int kFewGrads = 8;

__device__ __forceinline__ float bf16_to_f32(uint32_t b) { return __uint_as_float(b << 16); }
__device__ __forceinline__ float f16_to_f32(uint32_t h) {
  return (float)__builtin_bit_cast(_Float16, (unsigned short)h);
}
// Rounded to nearest, ties to even; a NaN stays one.
__device__ __forceinline__ uint32_t f32_to_bf16(float f) {
  const uint32_t u = __float_as_uint(f);
  if (f != f) return (u >> 16) | 0x40u;
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ uint32_t f32_to_f16(float f) {
  return (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)f);
}

template <int TYPE>
struct Elem;
template <>
struct Elem<GSR_F32> {
  static constexpr int kSize = 4;
  __device__ static __forceinline__ float load(uintptr_t a) { return *global_at<const float>(a); }
  __device__ static __forceinline__ void store(uintptr_t a, float v) { *global_at<float>(a) = v; }
};
template <>
struct Elem<GSR_F16> {
  static constexpr int kSize = 2;
  __device__ static __forceinline__ float load(uintptr_t a) { return f16_to_f32(*global_at<const uint16_t>(a)); }
  __device__ static __forceinline__ void store(uintptr_t a, float v) { *global_at<uint16_t>(a) = (uint16_t)f32_to_f16(v); }
};
template <>
struct Elem<GSR_BF16> {
  static constexpr int kSize = 2;
  __device__ static __forceinline__ float load(uintptr_t a) { return bf16_to_f32(*global_at<const uint16_t>(a)); }
  __device__ static __forceinline__ void store(uintptr_t a, float v) { *global_at<uint16_t>(a) = (uint16_t)f32_to_bf16(v); }
};

template <int NORM>
__device__ __forceinline__ double add(double acc, float x) {
  const double d = (double)x;
  if (NORM == GSR_NORM_2) return __builtin_fma(d, d, acc);
  if (NORM == GSR_NORM_1) return acc + __builtin_fabs(d);
  return gsr::norm_join<NORM>(acc, __builtin_fabs(d));
}

template <int NORM, int TYPE>
__device__ __forceinline__ double add_word(double acc, uint32_t w) {
  if (TYPE == GSR_F32) return add<NORM>(acc, __uint_as_float(w));
  if (TYPE == GSR_F16) return add<NORM>(add<NORM>(acc, f16_to_f32(w & 0xffffu)), f16_to_f32(w >> 16));
  return add<NORM>(add<NORM>(acc, __uint_as_float(w << 16)), __uint_as_float(w & 0xffff0000u));
}

template <int NORM, int TYPE>
__device__ __forceinline__ double add_vector(double acc, u4 v) {
  acc = add_word<NORM, TYPE>(acc, v.x);
  acc = add_word<NORM, TYPE>(acc, v.y);
  acc = add_word<NORM, TYPE>(acc, v.z);
  return add_word<NORM, TYPE>(acc, v.w);
}

// A thread's vectors of the chunk at `base`: all that lie wholly inside the tensor are requested before the first is
// used; the one or two of a tensor that its ends cut go element by element behind them.
template <int NORM, int TYPE>
__device__ __forceinline__ double add_chunk(double acc, uintptr_t base, uintptr_t begin, uintptr_t end) {
  const uintptr_t mine = base + threadIdx.x * 16u;
  u4 v[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    const uintptr_t a = mine + (uintptr_t)r * kBlock * 16;
    v[r] = a >= begin && a + 16 <= end ? *global_at<const u4>(a) : (u4){0, 0, 0, 0};     // zeros add nothing
  }
#pragma unroll
  for (int r = 0; r < kRounds; r++) acc = add_vector<NORM, TYPE>(acc, v[r]);
  if (base >= begin && base + kChunk <= end) return acc;
  for (int r = 0; r < kRounds; r++) {
    const uintptr_t a = mine + (uintptr_t)r * kBlock * 16;
    if (a < end && (a < begin || a + 16 > end))
      for (uintptr_t e = a < begin ? begin : a; e < a + 16 && e < end; e += Elem<TYPE>::kSize)
        acc = add<NORM>(acc, Elem<TYPE>::load(e));
  }
  return acc;
}

// The product of an fp16 element, rounded to fp32 before it is rounded to fp16, as torch's is: left to itself the compiler
// makes both one mixed-precision instruction that rounds once, which differs where the fp32 product is a tie.
__device__ __forceinline__ float product_16(float g, float c) {
  float p = g * c;
  asm("" : "+v"(p));
  return p;
}

template <int TYPE>
__device__ __forceinline__ uint32_t scale_word(uint32_t w, float c) {
  if (TYPE == GSR_F32) return __float_as_uint(__uint_as_float(w) * c);
  if (TYPE == GSR_F16) return f32_to_f16(product_16(f16_to_f32(w & 0xffffu), c)) | f32_to_f16(product_16(f16_to_f32(w >> 16), c)) << 16;
  return f32_to_bf16(__uint_as_float(w << 16) * c) | f32_to_bf16(__uint_as_float(w & 0xffff0000u) * c) << 16;
}

template <int TYPE>
__device__ __forceinline__ u4 scale_vector(u4 v, float c) {
  const u4 o = {scale_word<TYPE>(v.x, c), scale_word<TYPE>(v.y, c), scale_word<TYPE>(v.z, c), scale_word<TYPE>(v.w, c)};
  return o;
}

// STREAM: past the caches.
template <int TYPE, bool STREAM>
__device__ __forceinline__ void scale_chunk(float c, uintptr_t base, uintptr_t begin, uintptr_t end) {
  const uintptr_t mine = base + threadIdx.x * 16u;
  u4 v[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    const uintptr_t a = mine + (uintptr_t)r * kBlock * 16;
    v[r] = (u4){0, 0, 0, 0};
    if (a >= begin && a + 16 <= end) v[r] = STREAM ? __builtin_nontemporal_load(global_at<const u4>(a)) : *global_at<const u4>(a);
  }
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    const uintptr_t a = mine + (uintptr_t)r * kBlock * 16;
    if (a < begin || a + 16 > end) continue;
    if (STREAM) __builtin_nontemporal_store(scale_vector<TYPE>(v[r], c), global_at<u4>(a));
    else *global_at<u4>(a) = scale_vector<TYPE>(v[r], c);
  }
  if (base >= begin && base + kChunk <= end) return;
  for (int r = 0; r < kRounds; r++) {
    const uintptr_t a = mine + (uintptr_t)r * kBlock * 16;
    if (a < end && (a < begin || a + 16 > end))
      for (uintptr_t e = a < begin ? begin : a; e < a + 16 && e < end; e += Elem<TYPE>::kSize)
        Elem<TYPE>::store(e, TYPE == GSR_F16 ? product_16(Elem<TYPE>::load(e), c) : Elem<TYPE>::load(e) * c);
  }
}

// The descriptors, in LDS: kernel arguments lie in host memory, and a search that walks them there pays its round trip
// at every step.  All of them come in one (301 tensors in three launches, with the cut vectors moved behind the loads:
// 55 -> 45 us).
template <int MOST>
__device__ __forceinline__ const GradChunk* stage(const GradChunks<MOST>& a, GradChunk* s_t) {
  static_assert(sizeof(GradChunk) == 24 && MOST * 3 <= kBlock, "three words a descriptor, a word a thread");
  if ((int)threadIdx.x < 3 * a.count) ((uint64_t*)s_t)[threadIdx.x] = ((const uint64_t*)a.t)[threadIdx.x];
  __syncthreads();
  return s_t;
}

// The tensor that chunk c lies in (the last whose first chunk is not behind it).
__device__ __forceinline__ int tensor_of(const GradChunk* t, int count, uint32_t c) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t[mid].first <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Joins the workgroup's results into *out.
template <int NORM>
__device__ __forceinline__ void join_block(double acc, double* out) {
  __shared__ double s_wave[kBlock / 64];
  acc = gsr::norm_join_wave<NORM>(acc);
  if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kBlock / 64; w++) acc = gsr::norm_join<NORM>(acc, s_wave[w]);
    *out = acc;
  }
}

template <int NORM, int MOST>
__global__ void __launch_bounds__(kBlock) norm_kernel(GradChunks<MOST> a, double* __restrict__ partials) {
  __shared__ GradChunk s_t[MOST];
  const GradChunk* t = stage(a, s_t);
  double acc = 0.0;
  int k = tensor_of(t, a.count, blockIdx.x);
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    while (k + 1 < a.count && t[k + 1].first <= c) k++;
    const uintptr_t begin = t[k].begin, end = t[k].end;
    const uintptr_t base = (begin & ~(uintptr_t)15) + (uintptr_t)(c - t[k].first) * kChunk;
    switch (t[k].type) {
      case GSR_F32: acc = add_chunk<NORM, GSR_F32>(acc, base, begin, end); break;
      case GSR_F16: acc = add_chunk<NORM, GSR_F16>(acc, base, begin, end); break;
      default: acc = add_chunk<NORM, GSR_BF16>(acc, base, begin, end); break;
    }
  }
  join_block<NORM>(acc, partials + blockIdx.x);
}

// The partial results of very many launches, joined to one in front of the kernels that take them.
template <int NORM>
__global__ void __launch_bounds__(kBlock) norm_join_kernel(double* __restrict__ partials, int used) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < used; i += kBlock) acc = gsr::norm_join<NORM>(acc, partials[i]);
  join_block<NORM>(acc, partials);                           // behind a barrier: every thread has read its share
}

template <int NORM>
__global__ void __launch_bounds__(64) norm_final_kernel(const double* __restrict__ partials, int used, float* __restrict__ norm) {
  const double n = gsr::norm_of_partials<NORM>(partials, used);
  if (threadIdx.x == 0) *norm = (float)n;
}

// The same factor for 16-bit elements, in fp32 as torch forms `max_norm / (norm + 1e-6)`: the reciprocal of the sum,
// times the bound, each rounded.  bf16 has 128 significands, fp16 1024, and a factor like 0.37 puts whole classes of them
// on rounding ties (175 * 0.37 = 64.75), so that one last bit of it moves every element of a class the same way and the
// next norm with them; with torch's bits the results are torch's, bit for bit.  fp32 elements have no such classes: they
// take the factor rounded once from 64 bits, as the clipped step does.  A norm beyond fp32 has that one only.
__device__ __forceinline__ float clip_coefficient_16(double norm, double max_norm) {
  const float n = (float)norm;
  if (n == __builtin_inff() || max_norm == __builtin_inf()) return gsr::clip_coefficient(norm, max_norm);
  const float c = 1.0f / (n + 1e-6f) * (float)max_norm;
  return c < 1.0f || c != c ? c : 1.0f;
}

// Walks the chunks backwards, eight by eight: what the norm pass read last is still in the last-level cache, and
// chunk c falls to a workgroup of number c mod 8 in both passes, the same XCD, whose L2 may hold it.  With the norm pass,
// 1.4 GB / 236 MB / 24 MB: 814 / 107 / 13.9 us forwards, 795 / 106 / 17.2 backwards one by one, 782 / 102 / 13.9 so.
template <int NORM, int MOST>
__global__ void __launch_bounds__(kBlock) clip_kernel(GradChunks<MOST> a, const double* __restrict__ partials, int used,
                                                      double max_norm, float* __restrict__ norm, int stream) {
  const double n = gsr::norm_of_partials<NORM>(partials, used);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const float c32 = gsr::clip_coefficient(n, max_norm), c16 = clip_coefficient_16(n, max_norm);
  if (c32 == 1.0f && c16 == 1.0f) return;                    // x * 1 is x: nothing to write
  __shared__ GradChunk s_t[MOST];
  const GradChunk* t = stage(a, s_t);
  const uint32_t eights = (a.chunks + 7) / 8;
  int k = a.count - 1;
  for (uint32_t i = blockIdx.x; i < eights * 8; i += gridDim.x) {
    const uint32_t c = (eights - 1 - i / 8) * 8 + i % 8;
    if (c >= a.chunks) continue;
    if (t[k].first > c) k = tensor_of(t, k, c);              // one of those before
    const float coefficient = t[k].type == GSR_F32 ? c32 : c16;
    if (coefficient == 1.0f) continue;
    const uintptr_t begin = t[k].begin, end = t[k].end;
    const uintptr_t base = (begin & ~(uintptr_t)15) + (uintptr_t)(c - t[k].first) * kChunk;
    switch (t[k].type + (stream ? 4u : 0u)) {
      case GSR_F32: scale_chunk<GSR_F32, false>(coefficient, base, begin, end); break;
      case GSR_F16: scale_chunk<GSR_F16, false>(coefficient, base, begin, end); break;
      case GSR_BF16: scale_chunk<GSR_BF16, false>(coefficient, base, begin, end); break;
      case GSR_F32 + 4: scale_chunk<GSR_F32, true>(coefficient, base, begin, end); break;
      case GSR_F16 + 4: scale_chunk<GSR_F16, true>(coefficient, base, begin, end); break;
      default: scale_chunk<GSR_BF16, true>(coefficient, base, begin, end); break;
    }
  }
}

inline uint64_t chunks_of(const GsrGrad& g) {
  if (!g.n) return 0;
  const uintptr_t begin = (uintptr_t)g.grad;
  return ((begin & 15) + g.n * size_of(g.type) + kChunk - 1) / kChunk;
}

// Descriptors of the next launch from h_grads[*at ..), empty tensors left out; advances *at.
template <int MOST>
inline void fill(GradChunks<MOST>& a, int count, const GsrGrad* h_grads, int* at) {
  a.count = 0;
  a.chunks = 0;
  for (; *at < count && a.count < MOST; ++*at) {
    const GsrGrad& g = h_grads[*at];
    const uint64_t chunks = chunks_of(g);
    if (!chunks) continue;
    const uintptr_t begin = (uintptr_t)g.grad;
    a.t[a.count++] = {begin, begin + g.n * size_of(g.type), a.chunks, (uint32_t)g.type};
    a.chunks += (uint32_t)chunks;
  }
}

template <int MOST>
int launch_norm(int count, const GsrGrad* h_grads, int norm_type, double* partials, int* used, hipStream_t stream) {
  GradChunks<MOST> a;
  for (int at = 0; at < count;) {
    fill(a, count, h_grads, &at);
    if (!a.chunks) continue;
    double* out = partials + *used;
    const dim3 grid(std::min<uint32_t>(a.chunks, kNormBlocks)), block(kBlock);
    if (norm_type == GSR_NORM_2) hipLaunchKernelGGL((norm_kernel<GSR_NORM_2, MOST>), grid, block, 0, stream, a, out);
    else if (norm_type == GSR_NORM_1) hipLaunchKernelGGL((norm_kernel<GSR_NORM_1, MOST>), grid, block, 0, stream, a, out);
    else hipLaunchKernelGGL((norm_kernel<GSR_NORM_MAX, MOST>), grid, block, 0, stream, a, out);
    const int rc = gsr::check_launch("grad_norm");
    if (rc != GSR_OK) return rc;
    *used += (int)grid.x;
  }
  return GSR_OK;
}

template <int MOST>
int launch_clip(int count, const GsrGrad* h_grads, int norm_type, const double* partials, int used, double max_norm,
                float* norm, hipStream_t stream) {
  // Gradients beyond the size of the last-level cache are scaled past it: with the norm pass, 472 MB of fp32 take 236 us
  // so and 262 through it, 1.4 GB 768 and 821; 165 MB the other way round 80 and 73, 236 MB 111 and 103.  Smaller ones
  // go through it although buffers that take turns would rather not (118 MB 55 us past it, 64 through it): what reads
  // them next, as the step does, finds them there (236 MB, clip and step together 391 us past it, 370 through it).
  const bool stream_past = gsr::past_last_level(count, h_grads);
  GradChunks<MOST> a;
  for (int at = 0; at < count;) {
    fill(a, count, h_grads, &at);
    if (!a.chunks) continue;
    const dim3 grid(std::min<uint32_t>((a.chunks + 7) / 8 * 8, kClipBlocks)), block(kBlock);
    if (norm_type == GSR_NORM_2)
      hipLaunchKernelGGL((clip_kernel<GSR_NORM_2, MOST>), grid, block, 0, stream, a, partials, used, max_norm, norm, (int)stream_past);
    else if (norm_type == GSR_NORM_1)
      hipLaunchKernelGGL((clip_kernel<GSR_NORM_1, MOST>), grid, block, 0, stream, a, partials, used, max_norm, norm, (int)stream_past);
    else
      hipLaunchKernelGGL((clip_kernel<GSR_NORM_MAX, MOST>), grid, block, 0, stream, a, partials, used, max_norm, norm, (int)stream_past);
    const int rc = gsr::check_launch("clip_grads");
    if (rc != GSR_OK) return rc;
    norm = nullptr;                                          // the first launch has written it
  }
  return GSR_OK;
}

}  // namespace

namespace gsr {

int check_norm(const char* what, int count, const GsrGrad* h_grads, int norm_type, const float* norm, const void* scratch,
               size_t scratch_bytes) {
  GSR_REQUIRE(count >= 0, "%s: %d tensors", what, count);
  GSR_REQUIRE(count == 0 || h_grads, "%s: null tensor list", what);
  GSR_REQUIRE(norm_type == GSR_NORM_MAX || norm_type == GSR_NORM_1 || norm_type == GSR_NORM_2, "%s: norm type %d", what,
              norm_type);
  GSR_REQUIRE(norm, "%s: null pointer for the norm", what);
  uint64_t chunks = 0;
  for (int k = 0; k < count; k++) {
    const GsrGrad& g = h_grads[k];
    GSR_REQUIRE(g.type == GSR_F32 || g.type == GSR_F16 || g.type == GSR_BF16, "%s: tensor %d has unknown type %llu", what, k,
                (unsigned long long)g.type);
    if (!g.n) continue;
    GSR_REQUIRE(g.grad, "%s: null pointer in tensor %d", what, k);
    GSR_REQUIRE((uintptr_t)g.grad % size_of(g.type) == 0, "%s: tensor %d is not aligned to its elements", what, k);
    GSR_REQUIRE(g.n <= ((size_t)1 << 44), "%s: tensor %d has %zu elements", what, k, g.n);
    chunks += chunks_of(g);
  }
  GSR_REQUIRE(chunks < ((uint64_t)1 << 31), "%s: %llu chunks of gradients", what, (unsigned long long)chunks);
  if (scratch_bytes < gsr_grad_norm_bytes(count))
    return fail(GSR_E_SCRATCH, "%s: scratch too small: %zu of %zu bytes", what, scratch_bytes, gsr_grad_norm_bytes(count));
  if (!scratch || ((uintptr_t)scratch & 255)) return fail(GSR_E_SCRATCH, "%s: scratch must be 256-byte aligned", what);
  return GSR_OK;
}

int norm_partials(int count, const GsrGrad* h_grads, int norm_type, double* partials, int* used, hipStream_t stream) {
  *used = 0;
  const int rc = count <= kFewGrads ? launch_norm<kFewGrads>(count, h_grads, norm_type, partials, used, stream)
                                    : launch_norm<kGradsPerLaunch>(count, h_grads, norm_type, partials, used, stream);
  if (rc != GSR_OK || *used <= kMostJoined) return rc;
  if (norm_type == GSR_NORM_2) hipLaunchKernelGGL(norm_join_kernel<GSR_NORM_2>, dim3(1), dim3(kBlock), 0, stream, partials, *used);
  else if (norm_type == GSR_NORM_1) hipLaunchKernelGGL(norm_join_kernel<GSR_NORM_1>, dim3(1), dim3(kBlock), 0, stream, partials, *used);
  else hipLaunchKernelGGL(norm_join_kernel<GSR_NORM_MAX>, dim3(1), dim3(kBlock), 0, stream, partials, *used);
  *used = 1;
  return check_launch("grad_norm");
}

}  // namespace gsr

namespace {

int write_norm(const double* partials, int used, int norm_type, float* norm, hipStream_t stream) {
  if (norm_type == GSR_NORM_2) hipLaunchKernelGGL(norm_final_kernel<GSR_NORM_2>, dim3(1), dim3(64), 0, stream, partials, used, norm);
  else if (norm_type == GSR_NORM_1) hipLaunchKernelGGL(norm_final_kernel<GSR_NORM_1>, dim3(1), dim3(64), 0, stream, partials, used, norm);
  else hipLaunchKernelGGL(norm_final_kernel<GSR_NORM_MAX>, dim3(1), dim3(64), 0, stream, partials, used, norm);
  return gsr::check_launch("grad_norm");
}

// Whether two tensors of the list share memory (each would be scaled by its own workgroups, in any order).
// -1 without the memory to find out.
int any_overlap(int count, const GsrGrad* h_grads) {
  struct Span { uintptr_t begin, end; };
  Span few[64];
  Span* spans = count <= 64 ? few : new (std::nothrow) Span[count];
  if (!spans) return -1;
  int n = 0;
  for (int k = 0; k < count; k++) {
    const uintptr_t begin = (uintptr_t)h_grads[k].grad;
    if (h_grads[k].n) spans[n++] = {begin, begin + h_grads[k].n * size_of(h_grads[k].type)};
  }
  std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  int found = 0;
  for (int k = 1; k < n; k++) found |= spans[k].begin < spans[k - 1].end;
  if (spans != few) delete[] spans;
  return found;
}

}  // namespace

extern "C" size_t gsr_grad_norm_bytes(int count) {
  return gsr::align_up((size_t)gsr::norm_partials_most(count > 0 ? count : 0) * sizeof(double), 256);
}

extern "C" int gsr_grad_norm(int count, const GsrGrad* h_grads, int norm_type, float* norm, void* scratch,
                             size_t scratch_bytes, void* stream) {
  int rc = gsr::check_norm("grad_norm", count, h_grads, norm_type, norm, scratch, scratch_bytes);
  if (rc != GSR_OK) return rc;
  int used = 0;
  rc = gsr::norm_partials(count, h_grads, norm_type, (double*)scratch, &used, (hipStream_t)stream);
  if (rc != GSR_OK) return rc;
  return write_norm((const double*)scratch, used, norm_type, norm, (hipStream_t)stream);
}

extern "C" int gsr_clip_grads(int count, const GsrGrad* h_grads, int norm_type, double max_norm, float* norm, void* scratch,
                              size_t scratch_bytes, void* stream) {
  int rc = gsr::check_norm("clip_grads", count, h_grads, norm_type, norm, scratch, scratch_bytes);
  if (rc != GSR_OK) return rc;
  GSR_REQUIRE(max_norm >= 0.0, "clip_grads: bound %g", max_norm);
  const int overlap = any_overlap(count, h_grads);
  GSR_REQUIRE(overlap >= 0, "clip_grads: no memory to compare %d tensors", count);
  GSR_REQUIRE(!overlap, "clip_grads: two tensors of the list share memory");
  double* partials = (double*)scratch;
  int used = 0;
  rc = gsr::norm_partials(count, h_grads, norm_type, partials, &used, (hipStream_t)stream);
  if (rc != GSR_OK) return rc;
  if (used == 0) return write_norm(partials, 0, norm_type, norm, (hipStream_t)stream);
  if (count <= kFewGrads)
    return launch_clip<kFewGrads>(count, h_grads, norm_type, partials, used, max_norm, norm, (hipStream_t)stream);
  return launch_clip<kGradsPerLaunch>(count, h_grads, norm_type, partials, used, max_norm, norm, (hipStream_t)stream);
}
