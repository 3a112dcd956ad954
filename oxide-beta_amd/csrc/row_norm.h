// row_norm.h -- what the norms over the last dimension share (internal to the library): how many
// threads and accesses a row takes, sums over a row's threads, and the sum of the blocks' shares of
// a parameter's gradient.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "common.h"
#include "storage.h"

namespace oxh {
namespace row_norm {

// The sums of Count values over a row's Lanes threads (whole waves) in one fixed order, in every
// thread.  `slot` is a buffer of 16 floats for each value; consecutive calls alternate between two.
template <int Lanes, int Count>
__device__ __forceinline__ void row_sums(float (&v)[Count], float (*slot)[16]) {
  wave_sums_rows(v);
  if constexpr (Lanes == 64) return;
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int c = 0; c < Count; ++c) slot[c][wave] = v[c];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < Count; ++c) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < Lanes / 64; ++i) total += slot[c][i];
    v[c] = total;
  }
}
template <int Lanes>
__device__ __forceinline__ float row_sum(float v, float *slot) {
  float one[1] = {v};
  row_sums<Lanes>(one, reinterpret_cast<float(*)[16]>(slot));
  return one[0];
}

// out[c] = sum over the partial rows for the columns below `split`, out2[c - split] from there on
// (either may be null): 16 columns per block (from `first` on), 64 strands of rows each, a strand's
// rows in order and the strands by halves.
static __global__ __launch_bounds__(1024) void column_sums_kernel(const float *partial, float *out,
                                                                  float *out2, uint32_t split,
                                                                  uint32_t rows, uint32_t columns,
                                                                  uint32_t first) {
  __shared__ float part[64][17];
  const uint32_t c = threadIdx.x & 15, strand = threadIdx.x >> 4;
  const uint32_t column = first + blockIdx.x * 16 + c;
  float sum = 0.0f;
  if (column < columns) {
#pragma unroll 8
    for (uint32_t r = strand; r < rows; r += 64)
      sum += partial[static_cast<uint64_t>(r) * columns + column];
  }
  part[strand][c] = sum;
  __syncthreads();
#pragma unroll
  for (uint32_t half = 32; half != 0; half /= 2) {
    if (strand < half) part[strand][c] += part[strand + half][c];
    __syncthreads();
  }
  if (strand != 0 || column >= columns) return;
  if (column < split) {
    if (out != nullptr) out[column] = part[0][c];
  } else if (out2 != nullptr) {
    out2[column - split] = part[0][c];
  }
}

template <int Lanes, int Chunks>
struct Shape {
  static constexpr int lanes = Lanes, chunks = Chunks;
};

// Calls run(Shape<lanes, chunks>) with the fewest threads per row that keep it within 8 accesses,
// and where that is one wave within 32 values, each.  Limit: columns never exceed it.
template <int N, uint64_t Limit, typename Run>
void with_shape(uint64_t columns, Run run) {
  const uint64_t packs = (columns + N - 1) / N;
  if constexpr (N == 1) {  // rows of fewer values than an access
    run(Shape<64, 1>());
  } else {
    if (packs <= 64) return run(Shape<64, 1>());
    if (packs <= 128) return run(Shape<64, 2>());
    if (packs <= 256) return run(Shape<64, 4>());
    if (packs <= 512) return run(std::conditional_t<N <= 4, Shape<64, 8>, Shape<256, 2>>());
    if (packs <= 1024) return run(Shape<256, 4>());
    if (Limit / N <= 2048 || packs <= 2048) return run(Shape<256, 8>());
    if constexpr (Limit / N > 2048)
      if (Limit / N <= 4096 || packs <= 4096) return run(Shape<1024, 4>());
    if constexpr (Limit / N > 4096) run(Shape<1024, 8>());
  }
}

// Calls run(pack, ragged) for rows of these columns: 16 bytes per access, or one value where a row
// has fewer.
template <typename T, typename Run>
void with_pack(uint64_t columns, Run run) {
  constexpr int kPack = 16 / sizeof(T);
  typedef std::integral_constant<int, kPack> Packed;
  if (columns % kPack == 0) run(Packed(), std::false_type());
  else if (columns > kPack) run(Packed(), std::true_type());
  else run(std::integral_constant<int, 1>(), std::false_type());
}

// Blocks that a parameter's gradient is summed over (rows of `partial`, which stays within 8 MB up
// to 8192 columns).
inline uint64_t block_limit(uint64_t columns) {
  return std::min<uint64_t>(2048, std::max<uint64_t>(256, (1ull << 21) / columns));
}

// Rows that one block takes by itself, whose share is the parameter's gradient: a second launch is
// about as long as three more rows of a wave, or one of a block (RMS norm, bfloat16 16 x 1024: 7.2
// us a call, 10.1 with two launches; 32 x 1024: 8.3 and 10.1, but 9.3 and 6.0 on the device;
// float32 2 x 4096: 7.4 and 10.1; 8 x 4096: 13.7 and 10.2).
constexpr uint64_t rows_alone(int groups) { return groups > 1 ? 4 * groups : 2; }

// Blocks of so many threads that one launch takes: it numbers its threads with 32 bits.
constexpr uint64_t most_blocks(uint64_t threads) { return (1ull << 31) / threads; }

// Runs column_sums_kernel over all columns of `partial` [rows, columns].
inline void launch_column_sums(hipStream_t stream, const float *partial, float *out, float *out2,
                               uint32_t split, uint32_t rows, uint32_t columns) {
  constexpr uint32_t most = static_cast<uint32_t>(most_blocks(1024)) * 16;
  for (uint32_t first = 0; first < columns; first += most)
    launch(column_sums_kernel, dim3((std::min(columns - first, most) + 15) / 16), dim3(1024), 0,
           stream, partial, out, out2, split, rows, columns, first);
}

inline bool aligned_to(const void *p, uint64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

inline oxh_status check_rows(const char *what, int dtype, uint64_t rows, uint64_t columns) {
  OXH_REQUIRE(storage::valid(dtype), OXH_INVALID_SHAPE,
              std::string(what) + ": dtype is neither OXH_F32 nor OXH_BF16");
  OXH_REQUIRE(columns >= 1 && columns < (1ull << 31), OXH_INVALID_SHAPE,
              std::string(what) + ": columns out of range");
  OXH_REQUIRE(rows < (1ull << 31), OXH_INVALID_SHAPE, std::string(what) + ": too many rows");
  OXH_REQUIRE(rows <= (1ull << 60) / columns, OXH_INVALID_SHAPE,
              std::string(what) + ": element count overflow");
  return ok();
}

}  // namespace row_norm
}  // namespace oxh
