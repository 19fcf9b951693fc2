// Fused Adam step for the Gaussian model's parameter tensors on gfx950.
//
// The reference optimises six tensors with torch.optim.Adam(lr per group,
// eps = 1e-15, betas (0.9, 0.999), no weight decay, no amsgrad)
// (scene/gaussian_model.py:154-163, train.py:126-128).  PyTorch runs that as a
// chain of elementwise passes per tensor; here one launch updates all tensors:
// every element is read once (parameter, gradient, both moments: 16 B) and
// written once (12 B), which is the HBM minimum of 28 B per element.
//
// Arithmetic follows torch.optim.Adam's single-tensor path operation by
// operation:
//     m <- m + (1 - b1) (g - m)                      (lerp)
//     v <- b2 v + (1 - b2) g g                       (mul, addcmul)
//     p <- p - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// with the bias corrections and the weights 1 - b1, 1 - b2 formed on the host in double, as
// Python does (the hyper-parameters cross the ABI as doubles for that reason).
// `grad_scale` multiplies the gradient first (1/world_size after a summing
// all-reduce; 1 otherwise).
//
// gsr_adam_step_clipped is the same update with the gradients' norm and the bound on it in front: a norm pass
// (gradnorm.hip) and ONE update launch whose waves join its partial results while their own loads are under way, so
// that the clipped gradients are never written and no kernel of a single workgroup stands between the two.  It reads
// each gradient twice: 4 B (2 B for a 16-bit one) on top of the 28 B an element.  6M Gaussians: 1880 us, 227 of them
// the norm pass (11.3 GB, 6.0 TB/s); 1M 274, with bf16 gradients 259.  Gradients up to the size of the last-level cache
// are read through it (1M: 274 us, nontemporally 281; 6M: 1930 and 1880).  Walking the tensors backwards, as the clip
// does, changes nothing here: the parameters and moments pass by in between.
#include "gradnorm.h"

namespace {

constexpr int kBlock = 256;
constexpr int kPerThread = 4;                    // one 16-byte access per array
// 16-byte accesses per array and thread, a block's width apart, all of a thread's loads ahead of its arithmetic; and
// every access nontemporal: each element is touched once per step, so nothing is gained by keeping it in the L2.
// 1M Gaussians (59M elements): one round with ordinary accesses 332 us, nontemporal 317, two rounds 304, three 299,
// four 302.
constexpr int kRounds = 3;
constexpr int kPerBlock = kBlock * kPerThread * kRounds;
#define GSR_LD(p) __builtin_nontemporal_load(p)
#define GSR_ST(p, v) __builtin_nontemporal_store(v, p)

struct AdamTensors {
  GsrAdamTensor t[GSR_ADAM_MAX_TENSORS];
  uint32_t first_block[GSR_ADAM_MAX_TENSORS + 1];
  int count;
};

// w1 = 1 - b1 and w2 = 1 - b2 are formed on the host in double and rounded once, as Python forms them
__device__ __forceinline__ void adam_update(float& p, float g, float& m, float& v, float w1, float b2, float w2,
                                            float step_size, float inv_bc2_sqrt, float eps, float grad_scale) {
  g = g * grad_scale;
  m = m + w1 * (g - m);
  v = v * b2 + w2 * g * g;
  const float denom = sqrtf(v) * inv_bc2_sqrt + eps;
  p = p - step_size * (m / denom);
}

__global__ void __launch_bounds__(kBlock) adam_kernel(AdamTensors a, float w1, float b2, float w2, float eps, float bc1,
                                                      float inv_bc2_sqrt, float grad_scale) {
  // which tensor this block works on: at most GSR_ADAM_MAX_TENSORS, linear search in scalar registers
  int k = 0;
  while (k + 1 < a.count && blockIdx.x >= a.first_block[k + 1]) k++;
  const GsrAdamTensor t = a.t[k];
  const size_t block_base = (size_t)(blockIdx.x - a.first_block[k]) * kPerBlock + (size_t)threadIdx.x * kPerThread;
  const float step_size = t.lr / bc1;
  if (t.vec4 && block_base - (size_t)threadIdx.x * kPerThread + kPerBlock <= t.n) {
    // a whole block of vector accesses: all loads of the thread's rounds first
    typedef float f4 __attribute__((ext_vector_type(4)));
    f4 p[kRounds], g[kRounds], m[kRounds], v[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
      const size_t base = block_base + (size_t)r * kBlock * kPerThread;
      p[r] = GSR_LD(reinterpret_cast<f4*>(t.param + base));
      g[r] = GSR_LD(reinterpret_cast<const f4*>(t.grad + base));
      m[r] = GSR_LD(reinterpret_cast<f4*>(t.exp_avg + base));
      v[r] = GSR_LD(reinterpret_cast<f4*>(t.exp_avg_sq + base));
    }
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
      const size_t base = block_base + (size_t)r * kBlock * kPerThread;
      float px = p[r].x, py = p[r].y, pz = p[r].z, pw = p[r].w, mx = m[r].x, my = m[r].y, mz = m[r].z, mw = m[r].w;
      float vx = v[r].x, vy = v[r].y, vz = v[r].z, vw = v[r].w;
      adam_update(px, g[r].x, mx, vx, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      adam_update(py, g[r].y, my, vy, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      adam_update(pz, g[r].z, mz, vz, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      adam_update(pw, g[r].w, mw, vw, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      const f4 po = {px, py, pz, pw}, mo = {mx, my, mz, mw}, vo = {vx, vy, vz, vw};
      GSR_ST(reinterpret_cast<f4*>(t.param + base), po);
      GSR_ST(reinterpret_cast<f4*>(t.exp_avg + base), mo);
      GSR_ST(reinterpret_cast<f4*>(t.exp_avg_sq + base), vo);
    }
    return;
  }
  for (int r = 0; r < kRounds; r++) {
    const size_t base = block_base + (size_t)r * kBlock * kPerThread;
    for (size_t i = base; i < base + kPerThread && i < t.n; i++) {
      float p = t.param[i], m = t.exp_avg[i], v = t.exp_avg_sq[i];
      adam_update(p, t.grad[i], m, v, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      t.param[i] = p; t.exp_avg[i] = m; t.exp_avg_sq[i] = v;
    }
  }
}

struct ClipArgs {
  const double* partials;   // of the norm pass
  int used;
  int skip_nonfinite;
  double max_norm;
  float* norm;
};

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef unsigned short us4 __attribute__((ext_vector_type(4)));

// Four gradients from element `i` (aligned to four of them), and one, as fp32; the conversions are exact.
template <int TYPE, bool CACHED>
__device__ __forceinline__ f4 grads_at(const void* grad, size_t i) {
  if (TYPE == GSR_F32) {
    const f4* at = (const f4*)((const float*)grad + i);
    return CACHED ? *at : GSR_LD(at);
  }
  if (TYPE == GSR_F16) {
    const h4* at = (const h4*)((const _Float16*)grad + i);
    const h4 h = CACHED ? *at : GSR_LD(at);
    return (f4){(float)h.x, (float)h.y, (float)h.z, (float)h.w};
  }
  const us4* at = (const us4*)((const unsigned short*)grad + i);
  const us4 h = CACHED ? *at : GSR_LD(at);
  return (f4){__uint_as_float((uint32_t)h.x << 16), __uint_as_float((uint32_t)h.y << 16),
              __uint_as_float((uint32_t)h.z << 16), __uint_as_float((uint32_t)h.w << 16)};
}
template <int TYPE>
__device__ __forceinline__ float grad_at(const void* grad, size_t i) {
  if (TYPE == GSR_F32) return ((const float*)grad)[i];
  if (TYPE == GSR_F16) return (float)((const _Float16*)grad)[i];
  return __uint_as_float((uint32_t)((const unsigned short*)grad)[i] << 16);
}

// One workgroup's elements of tensor `t`, whose gradient is of type TYPE.  The factor on the gradients comes after the
// loads are issued: joining the partial results hides behind them.
// CACHED: the norm pass has left the gradients in the last-level cache, they are read through it.
template <int NORM, int TYPE, bool CACHED>
__device__ __forceinline__ void clipped_block(const GsrAdamTensor& t, size_t first, const ClipArgs& clip, float w1, float b2,
                                              float w2, float eps, float step_size, float inv_bc2_sqrt, float grad_scale) {
  const size_t block_base = first + (size_t)threadIdx.x * kPerThread;
  const bool whole = t.vec4 && first + kPerBlock <= t.n;
  f4 p[kRounds], g[kRounds], m[kRounds], v[kRounds];
  if (whole) {
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
      const size_t base = block_base + (size_t)r * kBlock * kPerThread;
      p[r] = GSR_LD(reinterpret_cast<f4*>(t.param + base));
      g[r] = grads_at<TYPE, CACHED>(t.grad, base);
      m[r] = GSR_LD(reinterpret_cast<f4*>(t.exp_avg + base));
      v[r] = GSR_LD(reinterpret_cast<f4*>(t.exp_avg_sq + base));
    }
  }
  const double norm = fabs((double)grad_scale) * gsr::norm_of_partials<NORM>(clip.partials, clip.used);
  if (clip.norm && blockIdx.x == 0 && threadIdx.x == 0) *clip.norm = (float)norm;
  if (clip.skip_nonfinite && !(norm < __builtin_inf())) return;
  grad_scale *= gsr::clip_coefficient(norm, clip.max_norm);
  if (whole) {
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
      const size_t base = block_base + (size_t)r * kBlock * kPerThread;
      float px = p[r].x, py = p[r].y, pz = p[r].z, pw = p[r].w, mx = m[r].x, my = m[r].y, mz = m[r].z, mw = m[r].w;
      float vx = v[r].x, vy = v[r].y, vz = v[r].z, vw = v[r].w;
      adam_update(px, g[r].x, mx, vx, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      adam_update(py, g[r].y, my, vy, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      adam_update(pz, g[r].z, mz, vz, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      adam_update(pw, g[r].w, mw, vw, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      const f4 po = {px, py, pz, pw}, mo = {mx, my, mz, mw}, vo = {vx, vy, vz, vw};
      GSR_ST(reinterpret_cast<f4*>(t.param + base), po);
      GSR_ST(reinterpret_cast<f4*>(t.exp_avg + base), mo);
      GSR_ST(reinterpret_cast<f4*>(t.exp_avg_sq + base), vo);
    }
    return;
  }
  for (int r = 0; r < kRounds; r++) {
    const size_t base = block_base + (size_t)r * kBlock * kPerThread;
    for (size_t i = base; i < base + kPerThread && i < t.n; i++) {
      float px = t.param[i], mx = t.exp_avg[i], vx = t.exp_avg_sq[i];
      adam_update(px, grad_at<TYPE>(t.grad, i), mx, vx, w1, b2, w2, step_size, inv_bc2_sqrt, eps, grad_scale);
      t.param[i] = px; t.exp_avg[i] = mx; t.exp_avg_sq[i] = vx;
    }
  }
}

struct GradTypes {
  uint8_t of[GSR_ADAM_MAX_TENSORS];
};

template <int NORM, bool CACHED>
__global__ void __launch_bounds__(kBlock) adam_clipped_kernel(AdamTensors a, GradTypes types, ClipArgs clip, float w1, float b2,
                                                              float w2, float eps, float bc1, float inv_bc2_sqrt,
                                                              float grad_scale) {
  int k = 0;
  while (k + 1 < a.count && blockIdx.x >= a.first_block[k + 1]) k++;
  const GsrAdamTensor t = a.t[k];
  const size_t first = (size_t)(blockIdx.x - a.first_block[k]) * kPerBlock;
  const float step_size = t.lr / bc1;
  switch (types.of[k]) {
    case GSR_F32:
      clipped_block<NORM, GSR_F32, CACHED>(t, first, clip, w1, b2, w2, eps, step_size, inv_bc2_sqrt, grad_scale);
      break;
    case GSR_F16:
      clipped_block<NORM, GSR_F16, CACHED>(t, first, clip, w1, b2, w2, eps, step_size, inv_bc2_sqrt, grad_scale);
      break;
    default:
      clipped_block<NORM, GSR_BF16, CACHED>(t, first, clip, w1, b2, w2, eps, step_size, inv_bc2_sqrt, grad_scale);
      break;
  }
}

}  // namespace

extern "C" int gsr_adam_step(int count, const GsrAdamTensor* h_tensors, double beta1, double beta2, double eps, int step,
                             float grad_scale, void* stream) {
  GSR_REQUIRE(count >= 0 && count <= GSR_ADAM_MAX_TENSORS, "adam_step: %d tensors (at most %d)", count,
              GSR_ADAM_MAX_TENSORS);
  GSR_REQUIRE(step >= 1, "adam_step: step counts from 1, got %d", step);
  GSR_REQUIRE(count == 0 || h_tensors, "adam_step: null tensor list");
  AdamTensors a{};
  a.count = 0;
  uint32_t blocks = 0;
  for (int k = 0; k < count; k++) {
    const GsrAdamTensor& t = h_tensors[k];
    if (t.n == 0) continue;
    GSR_REQUIRE(t.param && t.grad && t.exp_avg && t.exp_avg_sq, "adam_step: null pointer in tensor %d", k);
    GsrAdamTensor u = t;
    u.vec4 = (((uintptr_t)t.param | (uintptr_t)t.grad | (uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & 15) == 0;
    a.t[a.count] = u;
    a.first_block[a.count] = blocks;
    blocks += (uint32_t)((t.n + kPerBlock - 1) / kPerBlock);
    a.count++;
  }
  a.first_block[a.count] = blocks;
  if (blocks == 0) return GSR_OK;
  // bias corrections as Python forms them (double), then rounded once
  const double bc1 = 1.0 - pow(beta1, (double)step);
  const double bc2_sqrt = sqrt(1.0 - pow(beta2, (double)step));
  hipLaunchKernelGGL(adam_kernel, dim3(blocks), dim3(kBlock), 0, (hipStream_t)stream, a, (float)(1.0 - beta1),
                     (float)beta2, (float)(1.0 - beta2), (float)eps, (float)bc1, (float)(1.0 / bc2_sqrt), grad_scale);
  return gsr::check_launch("adam_step");
}

extern "C" int gsr_adam_step_clipped(int count, const GsrAdamTensor* h_tensors, const int* h_grad_types, double beta1,
                                     double beta2, double eps, int step, float grad_scale, int norm_type, double max_norm,
                                     int skip_nonfinite, float* norm, void* scratch, size_t scratch_bytes, void* stream) {
  GSR_REQUIRE(count >= 0 && count <= GSR_ADAM_MAX_TENSORS, "adam_step_clipped: %d tensors (at most %d)", count,
              GSR_ADAM_MAX_TENSORS);
  GSR_REQUIRE(step >= 1, "adam_step_clipped: step counts from 1, got %d", step);
  GSR_REQUIRE(count == 0 || h_tensors, "adam_step_clipped: null tensor list");
  GSR_REQUIRE(max_norm >= 0.0, "adam_step_clipped: bound %g", max_norm);
  GsrGrad grads[GSR_ADAM_MAX_TENSORS];
  for (int k = 0; k < count; k++) {
    const int type = h_grad_types ? h_grad_types[k] : GSR_F32;
    grads[k] = {const_cast<float*>(h_tensors[k].grad), h_tensors[k].n, (uint64_t)type};
    if (h_tensors[k].n)
      GSR_REQUIRE(h_tensors[k].param && h_tensors[k].exp_avg && h_tensors[k].exp_avg_sq,
                  "adam_step_clipped: null pointer in tensor %d", k);
  }
  int rc = gsr::check_norm("adam_step_clipped", count, grads, norm_type, norm, scratch, scratch_bytes);
  if (rc != GSR_OK) return rc;
  AdamTensors a{};
  GradTypes types{};
  uint64_t blocks = 0;
  for (int k = 0; k < count; k++) {
    const GsrAdamTensor& t = h_tensors[k];
    if (t.n == 0) continue;
    GsrAdamTensor u = t;
    const uintptr_t grad_align = grads[k].type == GSR_F32 ? 15 : 7;
    u.vec4 = (((uintptr_t)t.param | (uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & 15) == 0 && ((uintptr_t)t.grad & grad_align) == 0;
    types.of[a.count] = (uint8_t)grads[k].type;
    a.t[a.count] = u;
    a.first_block[a.count] = (uint32_t)blocks;
    blocks += (t.n + kPerBlock - 1) / kPerBlock;
    a.count++;
  }
  GSR_REQUIRE(blocks < ((uint64_t)1 << 24), "adam_step_clipped: too many elements");     // fewer than 2^32 threads
  a.first_block[a.count] = (uint32_t)blocks;
  if (blocks == 0) return gsr_grad_norm(0, nullptr, norm_type, norm, scratch, scratch_bytes, stream);   // writes 0
  ClipArgs clip = {(const double*)scratch, 0, skip_nonfinite, max_norm, norm};
  rc = gsr::norm_partials(count, grads, norm_type, (double*)scratch, &clip.used, (hipStream_t)stream);
  if (rc != GSR_OK) return rc;
  const double bc1 = 1.0 - pow(beta1, (double)step);
  const double bc2_sqrt = sqrt(1.0 - pow(beta2, (double)step));
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(kBlock), 0, (hipStream_t)stream, a, types, clip, (float)(1.0 - beta1),
                       (float)beta2, (float)(1.0 - beta2), (float)eps, (float)bc1, (float)(1.0 / bc2_sqrt), grad_scale);
  };
  const bool cached = !gsr::past_last_level(count, grads);
  if (norm_type == GSR_NORM_2) launch(cached ? adam_clipped_kernel<GSR_NORM_2, true> : adam_clipped_kernel<GSR_NORM_2, false>);
  else if (norm_type == GSR_NORM_1) launch(cached ? adam_clipped_kernel<GSR_NORM_1, true> : adam_clipped_kernel<GSR_NORM_1, false>);
  else launch(cached ? adam_clipped_kernel<GSR_NORM_MAX, true> : adam_clipped_kernel<GSR_NORM_MAX, false>);
  return gsr::check_launch("adam_step_clipped");
}
