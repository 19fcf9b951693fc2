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
// 18 tensors of 6.3M rows, 90 % kept, 7.9 GB: 1423 us, 5.6 TB/s.  One row in ten of a million, six tensors: 21 us for
// 48 MB of rows, which are 96 MB of the 128-byte lines that they lie in.
#include <algorithm>

#include "gsr_common.h"
#include "plan.h"

namespace {

using gsr::Divisor;
using gsr::divisor;
using gsr::lies_in_two_rows;

constexpr int kBlock = 256;
// Vectors of a thread, a block's width apart.  Everything is read and written once, so the accesses are nontemporal.
// 6.3M rows of 18 tensors, 90 % kept (7.9 GB): 1504 us; ordinary loads 1508, ordinary stores 1564, both 1580; four
// rounds 1515, eight 1616.
constexpr int kRounds = 2;
constexpr int kPerBlock = kBlock * kRounds;        // vectors of 16 bytes
constexpr int kRowsPerLaunch = 48;                 // descriptors of a launch, 2.7 KB of kernel arguments; more not measured

struct Moves {
  struct One {
    const char* rows;
    const char* appended;                          // null: rows behind the last are zeros
    char* out;
    uint64_t row_bytes;
    Divisor units;                                 // units of a row
    uint16_t unit;                                 // bytes of a unit: what rows, their length and the pointers are multiples of
    uint16_t wide;                                 // lies_in_two_rows
    uint32_t first_block;
  } t[kRowsPerLaunch];
  int count;
  uint32_t n_rows, n_appended, n_out;
  const void* index;
};

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// A unit, and 16 bytes at any multiple of one: global memory takes wide accesses at every byte.
template <int U> struct Unit;
template <> struct Unit<4> { typedef uint32_t type; typedef uint32_t wide __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Unit<2> { typedef uint16_t type; typedef uint32_t wide __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Unit<1> { typedef uint8_t type; typedef uint32_t wide __attribute__((ext_vector_type(4), aligned(1))); };

template <int U>
__device__ __forceinline__ u4 load_wide(const char* at) {
  return __builtin_nontemporal_load((const typename Unit<U>::wide*)at);
}
template <int U>
__device__ __forceinline__ void store_wide(char* at, u4 v) {
  __builtin_nontemporal_store((typename Unit<U>::wide)v, (typename Unit<U>::wide*)at);
}

// Where a row of the concatenation lies, and its number within its own buffer of `of` rows; `at` is null for a row of
// zeros, which an index that is negative or behind the last row stands for.
struct Place {
  const char* at;
  uint32_t row, of;
};

template <typename I>
__device__ __forceinline__ Place place_of(const Moves& a, const Moves::One& t, I i) {
  const uint64_t u = (uint64_t)(int64_t)i;
  if (u < a.n_rows) return {t.rows + u * t.row_bytes, (uint32_t)u, a.n_rows};
  if (t.appended && u - a.n_rows < a.n_appended)
    return {t.appended + (u - a.n_rows) * t.row_bytes, (uint32_t)(u - a.n_rows), a.n_appended};
  return {nullptr, 0, 0};
}

// Unit by unit: the 16 bytes from unit `col` of row `row` on.
template <int U, typename I>
__device__ __forceinline__ void move_units(const Moves& a, const Moves::One& t, uint64_t unit, uint64_t total, uint32_t row,
                                           uint32_t col) {
  typedef typename Unit<U>::type T;
  constexpr int K = 16 / U;
  T v[K];
#pragma unroll
  for (int k = 0; k < K; k++) {
    v[k] = 0;
    if (row < a.n_out) {
      const Place p = place_of(a, t, ((const I*)a.index)[row]);
      if (p.at) v[k] = *(const T*)(p.at + (uint64_t)col * U);
    }
    if (++col == t.units.d) { col = 0; row++; }
  }
  if (unit + K <= total) {
    u4 all;
    __builtin_memcpy(&all, v, 16);
    store_wide<U>(t.out + unit * U, all);
  } else {
#pragma unroll
    for (int k = 0; k < K; k++)
      if (unit + k < total) ((T*)t.out)[unit + k] = v[k];
  }
}

// One workgroup's vectors of tensor `t`: rows so short that a vector may lie in three or more of them.
template <int U, typename I>
__device__ __forceinline__ void move_block(const Moves& a, const Moves::One& t, uint32_t block) {
  constexpr int K = 16 / U;                                              // units of a vector
  const uint64_t total = (uint64_t)a.n_out * t.units.d;                  // units of the output
  const uint64_t first = (uint64_t)block * kPerBlock * K;
  const uint32_t row0 = (uint32_t)(first / t.units.d), col0 = (uint32_t)(first % t.units.d);
  for (int r = 0; r < kRounds; r++) {
    const uint32_t at = (uint32_t)(r * kBlock + threadIdx.x) * K;
    if (first + at >= total) return;
    const uint32_t over = t.units.quotient(col0 + at);
    move_units<U, I>(a, t, first + at, total, row0 + over, col0 + at - over * t.units.d);
  }
}

// The same for rows that lies_in_two_rows holds for, the ordinary case.  One wide load from where the vector begins,
// past the end of its row if it is split, and where the second row does not happen to follow the first in memory
// another, from as far before that.  The loads of all rounds go out before the first store.
template <int U, typename I>
__device__ __forceinline__ void move_block_wide(const Moves& a, const Moves::One& t, uint32_t block) {
  constexpr uint32_t K = 16 / U;
  const I* index = (const I*)a.index;
  const uint32_t w = t.units.d;
  const uint64_t total = (uint64_t)a.n_out * w;
  const uint64_t first = (uint64_t)block * kPerBlock * K;
  const uint32_t row0 = (uint32_t)(first / w), col0 = (uint32_t)(first % w);
  uint32_t row[kRounds], col[kRounds];
  I i0[kRounds], i1[kRounds];
  u4 v[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    const uint32_t at = (uint32_t)(r * kBlock + threadIdx.x) * K;
    const uint32_t over = t.units.quotient(col0 + at);
    row[r] = row0 + over;
    col[r] = col0 + at - over * w;
    i0[r] = index[min(row[r], a.n_out - 1)];
    i1[r] = index[min(row[r] + 1, a.n_out - 1)];
  }
  bool whole[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    const uint64_t unit = first + (uint32_t)(r * kBlock + threadIdx.x) * K;
    const uint32_t here = w - col[r];                                    // units of the vector in its first row, if below K
    const Place p = place_of(a, t, i0[r]), q = place_of(a, t, i1[r]);
    const bool split = here < K, follows = p.at && q.at == p.at + t.row_bytes;
    // a wide load must not leave its buffer: behind the last row, or before the first
    whole[r] = unit + K <= total && !(split && ((p.at && p.row + 1 == p.of) || (q.at && !follows && q.row == 0)));
    u4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    if (whole[r] && p.at) x = load_wide<U>(p.at + (uint64_t)col[r] * U);
    if (whole[r] && split && !follows && q.at) y = load_wide<U>(q.at - (uint64_t)here * U);
    const int from_first = follows || !split ? 16 : (int)here * U;       // bytes
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int n = from_first - 4 * k;                                  // of them in word k
      const uint32_t mask = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
      v[r][k] = (x[k] & mask) | (y[k] & ~mask);
    }
  }
#pragma unroll
  for (int r = 0; r < kRounds; r++) {
    const uint64_t unit = first + (uint32_t)(r * kBlock + threadIdx.x) * K;
    if (whole[r]) store_wide<U>(t.out + unit * U, v[r]);
    else if (unit < total) move_units<U, I>(a, t, unit, total, row[r], col[r]);
  }
}

template <int U, typename I>
__device__ __forceinline__ void move(const Moves& a, const Moves::One& t, uint32_t block) {
  if (t.wide) move_block_wide<U, I>(a, t, block);
  else move_block<U, I>(a, t, block);
}

template <typename I>
__global__ void __launch_bounds__(kBlock) move_kernel(Moves a) {
  int k = 0;
  while (k + 1 < a.count && blockIdx.x >= a.t[k + 1].first_block) k++;
  const Moves::One t = a.t[k];
  const uint32_t block = blockIdx.x - t.first_block;
  if (t.unit == 4) move<4, I>(a, t, block);
  else if (t.unit == 2) move<2, I>(a, t, block);
  else move<1, I>(a, t, block);
}

// ---- positions of the kept rows ----

constexpr int kTile = kBlock * 16;                 // flags a workgroup takes at a time
constexpr uint32_t kMostBlocks = 1024;             // every workgroup adds up the counts of those before it

// Up to here one workgroup takes all tiles and no counts are needed: a launch (3.5 us for the host) against 0.6 us a tile.
constexpr uint32_t kFewTiles = 4;

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
    const u4 v = *gsr::global_at<const u4>(f.base + at);
#pragma unroll
    for (int b = 0; b < 16; b++) bits |= ((v[b >> 2] >> (8 * (b & 3))) & 0xffu ? 1u : 0u) << b;
  } else {
    for (int b = 0; b < 16; b++)
      if (at + b >= f.skip && at + b < f.end && *gsr::global_at<const uint8_t>(f.base + at + b)) bits |= 1u << b;
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

// A tile's positions meet in LDS and leave it as full lines (6.3M flags, 90 % kept: 14 us); written by the threads that
// find them they are single words all over a tile's stretch (31 us).
__global__ void __launch_bounds__(kBlock) keep_write_kernel(Flags f, const uint32_t* __restrict__ counts,
                                                            int32_t* __restrict__ index, uint64_t* landing, uint32_t ticket) {
  __shared__ uint32_t s_wave[kBlock / 64];
  __shared__ int32_t s_index[kTile];
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
    __syncthreads();                               // s_wave and s_index have been read
    if (lane == 63) s_wave[wave] = upto;
    __syncthreads();
    uint32_t to = upto - mine;
    for (int w = 0; w < wave; w++) to += s_wave[w];
    const uint32_t position = tile * kTile + threadIdx.x * 16 - f.skip;
    while (bits) {
      const int b = __ffs(bits) - 1;
      s_index[to++] = (int32_t)(position + b);
      bits &= bits - 1;
    }
    const uint32_t found = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < found; i += kBlock) index[at + i] = s_index[i];
    at += found;
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0)
    __hip_atomic_store(landing, (uint64_t)ticket << 32 | at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

constexpr uint64_t kMostRows = 0x7fff0000ull;      // row numbers are 32-bit signed, with room to round up

constexpr uint64_t kMostMoveBlocks = 0xffffffull;  // a launch has fewer than 2^32 threads: 137 GB of rows

}  // namespace

extern "C" size_t gsr_keep_rows_bytes(void) { return kMostBlocks * sizeof(uint32_t); }

extern "C" int gsr_keep_rows(uint64_t n, const uint8_t* keep, int32_t* index, uint64_t* landing, uint32_t ticket, void* scratch,
                             size_t scratch_bytes, void* stream) {
  GSR_REQUIRE(n <= kMostRows, "keep_rows: %llu rows", (unsigned long long)n);
  GSR_REQUIRE(landing && (n == 0 || (keep && index)), "keep_rows: null pointer");
  GSR_REQUIRE((uintptr_t)landing % 8 == 0, "keep_rows: the landing word is not aligned");
  if (!scratch || ((uintptr_t)scratch & 255)) return gsr::fail(GSR_E_SCRATCH, "keep_rows: scratch must be 256-byte aligned");
  if (scratch_bytes < gsr_keep_rows_bytes())
    return gsr::fail(GSR_E_SCRATCH, "keep_rows: scratch too small: %zu of %zu bytes", scratch_bytes, gsr_keep_rows_bytes());
  Flags f;
  f.base = (uintptr_t)keep & ~(uintptr_t)15;
  f.skip = (uint32_t)((uintptr_t)keep & 15);
  f.end = f.skip + (uint32_t)n;
  f.tiles = (f.end + kTile - 1) / kTile;
  if (n == 0) f.tiles = 0;
  f.tiles_per_block = f.tiles <= kFewTiles ? std::max(1u, f.tiles) : (f.tiles + kMostBlocks - 1) / kMostBlocks;
  const uint32_t blocks = std::max(1u, (f.tiles + f.tiles_per_block - 1) / f.tiles_per_block);
  uint32_t* counts = (uint32_t*)scratch;
  if (blocks > 1) {                                // one workgroup has nothing before it
    hipLaunchKernelGGL(keep_count_kernel, dim3(blocks), dim3(kBlock), 0, (hipStream_t)stream, f, counts);
    const int rc = gsr::check_launch("keep_rows");
    if (rc != GSR_OK) return rc;
  }
  hipLaunchKernelGGL(keep_write_kernel, dim3(blocks), dim3(kBlock), 0, (hipStream_t)stream, f, counts, index, landing, ticket);
  return gsr::check_launch("keep_rows");
}

extern "C" int gsr_select_rows(int count, const GsrRows* h_tensors, uint64_t n_rows, uint64_t n_appended, uint64_t n_out,
                               const void* index, int index_bytes, void* stream) {
  GSR_REQUIRE(count >= 0 && (count == 0 || h_tensors), "select_rows: %d tensors, list %p", count, (const void*)h_tensors);
  GSR_REQUIRE(n_rows <= kMostRows && n_appended <= kMostRows && n_rows + n_appended <= kMostRows && n_out <= kMostRows,
              "select_rows: %llu of %llu + %llu rows", (unsigned long long)n_out, (unsigned long long)n_rows,
              (unsigned long long)n_appended);
  GSR_REQUIRE(index_bytes == 4 || index_bytes == 8, "select_rows: an index of %d bytes", index_bytes);
  GSR_REQUIRE(n_out == 0 || (index && (uintptr_t)index % index_bytes == 0), "select_rows: null or misaligned index");
  for (int k = 0; k < count; k++) {
    const GsrRows& t = h_tensors[k];
    if (t.row_bytes == 0 || n_out == 0) continue;
    GSR_REQUIRE(t.row_bytes < (1ull << 31), "select_rows: tensor %d has rows of %zu bytes", k, t.row_bytes);
    GSR_REQUIRE(t.out && (t.rows || n_rows == 0), "select_rows: null pointer in tensor %d", k);
    GSR_REQUIRE(n_out * t.row_bytes <= kMostMoveBlocks * 16ull * kPerBlock, "select_rows: tensor %d is too large", k);
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
      if (blocks && blocks + all > kMostMoveBlocks) break;
      Moves::One& u = a.t[a.count++];
      u.rows = (const char*)t.rows;
      u.appended = n_appended ? (const char*)t.appended : nullptr;
      u.out = (char*)t.out;
      u.row_bytes = t.row_bytes;
      const uintptr_t align = (uintptr_t)u.rows | (uintptr_t)u.appended | (uintptr_t)u.out;
      u.unit = 4;
      while ((align | t.row_bytes) % u.unit) u.unit >>= 1;
      u.units = divisor((uint32_t)(t.row_bytes / u.unit));
      u.wide = lies_in_two_rows(u.units.d, u.unit);
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
