// Rows of many tensors at once on gfx950: the positions of the kept ones, and copies by position.
//
// A model's parameters and both moments of its optimiser are tensors that share their first dimension: one row of each
// belongs to one Gaussian.  Refinement forks rows (copies and children), frees others and closes the gaps.  Here that is
//     index = positions of the non-zero bytes of keep, ascending           (gsr_keep_rows)
//     out_t[j] = concat(rows_t, appended_t or zeros)[index[j]]             (gsr_select_rows)
// with the concatenation never built and every tensor moved by one launch.
//
// Both are bound by HBM.  The copy works on the OUTPUT: a thread fills 16 contiguous bytes of it, wherever its rows
// begin, and finds row and column by one multiplication (division by the row's length); with short rows (3, 12, 16, 180
// bytes) that keeps every store full and the loads of a wave in few cache lines, which one wave a row would not.
#include <algorithm>

#include "gsr_common.h"

namespace {

constexpr int kBlock = 256;
constexpr int kRounds = 4;                         // vectors of a thread, a block's width apart
constexpr int kPerBlock = kBlock * kRounds;        // vectors of 16 bytes
constexpr int kRowsPerLaunch = 48;                 // descriptors that fit the kernel arguments

// n / d for every 32-bit n by a multiplication (Granlund and Montgomery 1994, the round-up method): with
// l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1, q = (t + ((n - t) >> 1)) >> (l - 1), t = mulhi(m, n); d > 1.
struct Divisor {
  uint32_t d, m, shift;
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    if (d == 1) return n;
    const uint32_t t = __umulhi(m, n);
    return (t + ((n - t) >> 1)) >> shift;
  }
};

struct Moves {
  struct One {
    const char* rows;
    const char* appended;                          // null: rows behind the last are zeros
    char* out;
    uint64_t row_bytes;
    Divisor units;                                 // units of a row
    uint32_t unit;                                 // bytes of a unit: what rows, their length and the pointers are multiples of
    uint32_t first_block;
  } t[kRowsPerLaunch];
  int count;
  uint32_t n_rows, n_appended, n_out;
  const void* index;
};

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// 16 bytes at any address that is a multiple of the unit: the hardware's wide accesses ask for 4
typedef uint32_t u4_4 __attribute__((ext_vector_type(4), aligned(4)));

template <int U> struct Unit;
template <> struct Unit<16> { typedef u4_4 type; };
template <> struct Unit<8> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(4))); };
template <> struct Unit<4> { typedef uint32_t type; };
template <> struct Unit<2> { typedef uint16_t type; };
template <> struct Unit<1> { typedef uint8_t type; };

// Where row `i` of the concatenation lies; null for a row of zeros.  An index that is negative or behind the last
// row is one.
template <typename I>
__device__ __forceinline__ const char* row_at(const Moves::One& t, I i, uint32_t n_rows, uint32_t n_appended) {
  const uint64_t u = (uint64_t)(int64_t)i;
  if (u < n_rows) return t.rows + u * t.row_bytes;
  if (t.appended && u - n_rows < n_appended) return t.appended + (u - n_rows) * t.row_bytes;
  return nullptr;
}

// One workgroup's vectors of tensor `t`; K = 16 / U units a vector.
template <int U, typename I>
__device__ __forceinline__ void move_block(const Moves& a, const Moves::One& t, uint32_t block) {
  typedef typename Unit<U>::type T;
  constexpr int K = 16 / U;
  const I* index = (const I*)a.index;
  const uint64_t total = (uint64_t)a.n_out * t.units.d;                  // units of the output
  const uint64_t first = (uint64_t)block * kPerBlock * K;
  const uint32_t row0 = (uint32_t)(first / t.units.d), col0 = (uint32_t)(first % t.units.d);
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    const uint32_t at = (uint32_t)(r * kBlock + threadIdx.x) * K;
    if (first + at >= total) return;
    const uint32_t over = t.units.quotient(col0 + at);
    uint32_t row = row0 + over, col = col0 + at - over * t.units.d;
    T v[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
      v[k] = T{};
      if (row < a.n_out) {
        const char* from = row_at(t, index[row], a.n_rows, a.n_appended);
        if (from) v[k] = *(const T*)(from + (uint64_t)col * U);
      }
      if (++col == t.units.d) { col = 0; row++; }
    }
    T* to = (T*)t.out + first + at;
#pragma unroll
    for (int k = 0; k < K; k++)
      if (first + at + k < total) to[k] = v[k];
  }
}

template <typename I>
__global__ void __launch_bounds__(kBlock) move_kernel(Moves a) {
  int k = 0;
  while (k + 1 < a.count && blockIdx.x >= a.t[k + 1].first_block) k++;
  const Moves::One t = a.t[k];
  const uint32_t block = blockIdx.x - t.first_block;
  switch (t.unit) {
    case 16: move_block<16, I>(a, t, block); break;
    case 8: move_block<8, I>(a, t, block); break;
    case 4: move_block<4, I>(a, t, block); break;
    case 2: move_block<2, I>(a, t, block); break;
    default: move_block<1, I>(a, t, block); break;
  }
}

// ---- positions of the kept rows ----

constexpr int kTile = kBlock * 16;                 // flags a workgroup takes at a time
constexpr uint32_t kMostBlocks = 1024;             // every workgroup adds up the counts of those before it

struct Flags {
  uintptr_t base;                                  // keep, rounded down to 16 bytes
  uint32_t skip;                                   // bytes of that which are not flags
  uint32_t end;                                    // skip + n
  uint32_t tiles, tiles_per_block;
};

// The flags of thread's vector in tile `tile`, a bit each.
__device__ __forceinline__ uint32_t flags_of(const Flags& f, uint32_t tile) {
  const uint32_t at = tile * kTile + threadIdx.x * 16;
  if (at >= f.end) return 0;
  uint32_t bits = 0;
  if (at >= f.skip && at + 16 <= f.end) {
    const u4 v = *(const u4*)(f.base + at);
#pragma unroll
    for (int b = 0; b < 16; b++) bits |= ((v[b >> 2] >> (8 * (b & 3))) & 0xffu ? 1u : 0u) << b;
  } else {
    for (int b = 0; b < 16; b++)
      if (at + b >= f.skip && at + b < f.end && *(const uint8_t*)(f.base + at + b)) bits |= 1u << b;
  }
  return bits;
}

__global__ void __launch_bounds__(kBlock) keep_count_kernel(Flags f, uint32_t* __restrict__ counts) {
  const uint32_t last = min(f.tiles, (blockIdx.x + 1) * f.tiles_per_block);
  uint32_t mine = 0;
  for (uint32_t tile = blockIdx.x * f.tiles_per_block; tile < last; tile++) mine += __popc(flags_of(f, tile));
  __shared__ uint32_t s_wave[kBlock / 64];
  mine = gsr::wave_sum(mine);
  if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = mine;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
}

__global__ void __launch_bounds__(kBlock) keep_write_kernel(Flags f, const uint32_t* __restrict__ counts,
                                                            int32_t* __restrict__ index, uint32_t* __restrict__ count) {
  __shared__ uint32_t s_wave[kBlock / 64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  uint32_t before = 0;
  for (uint32_t b = threadIdx.x; b < blockIdx.x; b += kBlock) before += counts[b];
  before = gsr::wave_sum(before);
  if (lane == 0) s_wave[wave] = before;
  __syncthreads();
  uint32_t at = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
  const uint32_t last = min(f.tiles, (blockIdx.x + 1) * f.tiles_per_block);
  for (uint32_t tile = blockIdx.x * f.tiles_per_block; tile < last; tile++) {
    uint32_t bits = flags_of(f, tile);
    const uint32_t mine = __popc(bits);
    const uint32_t upto = gsr::wave_inclusive_sum(mine);
    __syncthreads();                               // s_wave has been read
    if (lane == 63) s_wave[wave] = upto;
    __syncthreads();
    uint32_t to = at + upto - mine;
    for (int w = 0; w < wave; w++) to += s_wave[w];
    const uint32_t position = tile * kTile + threadIdx.x * 16 - f.skip;
    while (bits) {
      const int b = __ffs(bits) - 1;
      index[to++] = (int32_t)(position + b);
      bits &= bits - 1;
    }
    at += s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *count = at;
}

constexpr uint64_t kMostRows = 0x7fff0000ull;      // row numbers are 32-bit signed, with room to round up

Divisor divisor(uint32_t d) {
  Divisor v = {d, 0, 0};
  if (d > 1) {
    uint32_t l = 0;
    while ((1ull << l) < d) l++;
    v.m = (uint32_t)(((((uint64_t)1 << l) - d) << 32) / d + 1);
    v.shift = l - 1;
  }
  return v;
}

}  // namespace

extern "C" size_t gsr_keep_rows_bytes(void) { return kMostBlocks * sizeof(uint32_t); }

extern "C" int gsr_keep_rows(uint64_t n, const uint8_t* keep, int32_t* index, uint32_t* count, void* scratch,
                             size_t scratch_bytes, void* stream) {
  GSR_REQUIRE(n <= kMostRows, "keep_rows: %llu rows", (unsigned long long)n);
  GSR_REQUIRE(count && (n == 0 || (keep && index)), "keep_rows: null pointer");
  if (!scratch || ((uintptr_t)scratch & 255)) return gsr::fail(GSR_E_SCRATCH, "keep_rows: scratch must be 256-byte aligned");
  if (scratch_bytes < gsr_keep_rows_bytes())
    return gsr::fail(GSR_E_SCRATCH, "keep_rows: scratch too small: %zu of %zu bytes", scratch_bytes, gsr_keep_rows_bytes());
  Flags f;
  f.base = (uintptr_t)keep & ~(uintptr_t)15;
  f.skip = (uint32_t)((uintptr_t)keep & 15);
  f.end = f.skip + (uint32_t)n;
  f.tiles = (f.end + kTile - 1) / kTile;
  if (n == 0) f.tiles = 0;
  f.tiles_per_block = std::max(1u, (f.tiles + kMostBlocks - 1) / kMostBlocks);
  const uint32_t blocks = std::max(1u, (f.tiles + f.tiles_per_block - 1) / f.tiles_per_block);
  uint32_t* counts = (uint32_t*)scratch;
  if (blocks > 1) {                                // one workgroup has nothing before it
    hipLaunchKernelGGL(keep_count_kernel, dim3(blocks), dim3(kBlock), 0, (hipStream_t)stream, f, counts);
    const int rc = gsr::check_launch("keep_rows");
    if (rc != GSR_OK) return rc;
  }
  hipLaunchKernelGGL(keep_write_kernel, dim3(blocks), dim3(kBlock), 0, (hipStream_t)stream, f, counts, index, count);
  return gsr::check_launch("keep_rows");
}

extern "C" int gsr_select_rows(int count, const GsrRows* h_tensors, uint64_t n_rows, uint64_t n_appended, uint64_t n_out,
                               const void* index, int index_bytes, void* stream) {
  GSR_REQUIRE(count >= 0 && (count == 0 || h_tensors), "select_rows: %d tensors, list %p", count, (const void*)h_tensors);
  GSR_REQUIRE(n_rows + n_appended <= kMostRows && n_rows <= kMostRows && n_out <= kMostRows,
              "select_rows: %llu of %llu + %llu rows", (unsigned long long)n_out, (unsigned long long)n_rows,
              (unsigned long long)n_appended);
  GSR_REQUIRE(index_bytes == 4 || index_bytes == 8, "select_rows: an index of %d bytes", index_bytes);
  GSR_REQUIRE(n_out == 0 || (index && (uintptr_t)index % index_bytes == 0), "select_rows: null or misaligned index");
  for (int k = 0; k < count; k++) {
    const GsrRows& t = h_tensors[k];
    if (t.row_bytes == 0 || n_out == 0) continue;
    GSR_REQUIRE(t.row_bytes < (1ull << 31), "select_rows: tensor %d has rows of %zu bytes", k, t.row_bytes);
    GSR_REQUIRE(t.out && (t.rows || n_rows == 0), "select_rows: null pointer in tensor %d", k);
  }
  Moves a;
  a.n_rows = (uint32_t)n_rows;
  a.n_appended = (uint32_t)n_appended;
  a.n_out = (uint32_t)n_out;
  a.index = index;
  for (int at = 0; at < count && n_out;) {
    a.count = 0;
    uint64_t blocks = 0;
    for (; at < count && a.count < kRowsPerLaunch; at++) {
      const GsrRows& t = h_tensors[at];
      if (t.row_bytes == 0) continue;
      const uint64_t all = (n_out * t.row_bytes + 16ull * kPerBlock - 1) / (16ull * kPerBlock);
      if (blocks && blocks + all > 0x7fffffffull) break;
      GSR_REQUIRE(all <= 0x7fffffffull, "select_rows: tensor %d is too large", at);
      Moves::One& u = a.t[a.count++];
      u.rows = (const char*)t.rows;
      u.appended = n_appended ? (const char*)t.appended : nullptr;
      u.out = (char*)t.out;
      u.row_bytes = t.row_bytes;
      const uintptr_t align = (uintptr_t)u.rows | (uintptr_t)u.appended | (uintptr_t)u.out;
      // 8- and 16-byte units are read and written through 4-byte aligned wide accesses: only the row's length counts
      u.unit = (align & 3) ? 1 : 16;
      if ((align & 3) == 2) u.unit = 2;
      while (t.row_bytes % u.unit) u.unit >>= 1;
      u.units = divisor((uint32_t)(t.row_bytes / u.unit));
      u.first_block = (uint32_t)blocks;
      blocks += all;
    }
    if (!a.count) break;
    if (index_bytes == 4) hipLaunchKernelGGL(move_kernel<int32_t>, dim3((uint32_t)blocks), dim3(kBlock), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(move_kernel<int64_t>, dim3((uint32_t)blocks), dim3(kBlock), 0, (hipStream_t)stream, a);
    const int rc = gsr::check_launch("select_rows");
    if (rc != GSR_OK) return rc;
  }
  return GSR_OK;
}
