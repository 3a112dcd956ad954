// rms_norm.hip -- root-mean-square norm over the last dimension, of a residual sum where there is
// one, and its gradients.
//
//   s = x + r;  q = 1 / sqrt(mean(s^2) + epsilon);  y = s q w
//   d = dy w;   dx = dr = ds + q (d - s q mean(s q d));   dw = sum over rows of dy s q
//
// Rows are float32 or bfloat16; the sum, the statistics, both dot products and the weight
// gradient are float32, and each output is rounded once (y from the unrounded s).  No counterpart
// in the reference, whose only norm is BatchNorm2d.
//
// The bound is memory, so a row is read once and kept in registers: forward of a bfloat16 sum of
// 16384 x 4096 moves 537 MB in 97 us (5.5 TB/s, a large copy's rate); backward of float32 3584 x
// 1280 moves 73 MB in 15 us (4.8 TB/s) and sums the weight gradient's shares in 4 us more.  Small
// calls are launches: one row of 1024 takes 2.4 us, backward of bfloat16 1021 x 1537 9.2 and 2.8.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "common.h"
#include "storage.h"

namespace {

using oxh::storage::bf16;
using oxh::storage::load_places;
using oxh::storage::Places;
using oxh::storage::places_at;
using oxh::storage::store_places;

// The sum over a row's Lanes threads (whole waves) in one fixed order, in every thread.  `slot`
// is a buffer of 16 floats; consecutive calls alternate between two.
template <int Lanes>
__device__ __forceinline__ float row_sum(float v, float *slot) {
  float one[1] = {v};
  oxh::wave_sums_rows(one);
  if constexpr (Lanes == 64) return one[0];
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) slot[wave] = one[0];
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < Lanes / 64; ++i) total += slot[i];
  return total;
}

template <typename T>
struct Forward {
  const T *x, *r;
  const float *w;
  T *s, *y;
  float *q;
  uint64_t rows;
  uint32_t columns;
  float inverse_columns, epsilon;
};

// One row per Lanes threads, kept in registers between its two uses: Chunks accesses of N values
// per thread cover it.
template <typename T, int N, int Lanes, int Chunks, bool Ragged>
__global__ __launch_bounds__(Lanes < 256 ? 256 : Lanes) void rms_norm_forward_kernel(
    Forward<T> a) {
  __shared__ float slot[16];
  constexpr int kRows = Lanes < 256 ? 256 / Lanes : 1;
  const uint32_t lane = threadIdx.x % Lanes;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kRows + threadIdx.x / Lanes;
  if (row >= a.rows) return;  // whole waves: Lanes == 64 when a block holds several rows
  const uint64_t base = row * a.columns;
  float v[Chunks][N];
  float squares = 0.0f;
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
    if (at < a.columns) {
      const Places here = places_at<N, Ragged>(at, a.columns);
      load_places<T, N, Ragged>(a.x + base, here, v[c]);
      if (a.r != nullptr) {
        float r[N];
        load_places<T, N, Ragged>(a.r + base, here, r);
#pragma unroll
        for (int i = 0; i < N; ++i) v[c][i] += r[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[c][i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) squares = fmaf(v[c][i], v[c][i], squares);
  }
  const float q =
      1.0f / sqrtf(row_sum<Lanes>(squares, slot) * a.inverse_columns + a.epsilon);
  if (lane == 0 && a.q != nullptr) a.q[row] = q;
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
    if (at >= a.columns) continue;
    const Places here = places_at<N, Ragged>(at, a.columns);
    if (a.s != nullptr) store_places<T, N, Ragged>(a.s + base, here, v[c]);
    float w[N];
    load_places<float, N, Ragged>(a.w, here, w);
#pragma unroll
    for (int i = 0; i < N; ++i) v[c][i] = v[c][i] * q * w[i];
    store_places<T, N, Ragged>(a.y + base, here, v[c]);
  }
}

// Rows longer than the registers of a block: two passes over the operands.  The second forms the
// sum again (from x and r, not from the rounded one); a thread reads its elements before it writes
// them, so s may be x or r here too.
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_forward_long_kernel(Forward<T> a) {
  __shared__ float slot[16];
  const uint64_t base = static_cast<uint64_t>(blockIdx.x) * a.columns;
  float squares = 0.0f;
  for (uint32_t at = threadIdx.x; at < a.columns; at += 1024) {
    float v = oxh::storage::widen(a.x[base + at]);
    if (a.r != nullptr) v += oxh::storage::widen(a.r[base + at]);
    squares = fmaf(v, v, squares);
  }
  const float q = 1.0f / sqrtf(row_sum<1024>(squares, slot) * a.inverse_columns + a.epsilon);
  if (threadIdx.x == 0 && a.q != nullptr) a.q[blockIdx.x] = q;
  for (uint32_t at = threadIdx.x; at < a.columns; at += 1024) {
    float v = oxh::storage::widen(a.x[base + at]);
    if (a.r != nullptr) v += oxh::storage::widen(a.r[base + at]);
    if (a.s != nullptr) a.s[base + at] = static_cast<T>(v);
    a.y[base + at] = static_cast<T>(v * q * a.w[at]);
  }
}

template <typename T>
struct Backward {
  const T *g, *sg, *s;
  const float *w, *q;
  T *dx;
  float *partial;
  uint64_t rows;
  uint32_t columns;
  float inverse_columns;
};

// Each group of Lanes threads takes every groups-th row and keeps its share of the weight
// gradient in registers; a block's groups add theirs in shared memory, in order, and each block's
// sum goes to its row of `partial`.
template <typename T, int N, int Lanes, int Chunks, bool Ragged>
__global__ __launch_bounds__(Lanes < 256 ? 256 : Lanes) void rms_norm_backward_kernel(
    Backward<T> a) {
  __shared__ float slot[2][16];
  constexpr int kGroups = Lanes < 256 ? 256 / Lanes : 1;  // of a block
  const uint32_t lane = threadIdx.x % Lanes, own = threadIdx.x / Lanes;
  const uint64_t groups = static_cast<uint64_t>(gridDim.x) * kGroups;
  float dw[Chunks][N], w[Chunks][N];
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
#pragma unroll
    for (int i = 0; i < N; ++i) dw[c][i] = w[c][i] = 0.0f;
    if (at < a.columns)
      load_places<float, N, Ragged>(a.w, places_at<N, Ragged>(at, a.columns), w[c]);
  }
  int turn = 0;
  for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * kGroups + own; row < a.rows;
       row += groups) {
    const uint64_t base = row * a.columns;
    const float q = a.q[row];
    float unit[Chunks][N], d[Chunks][N];
    // the stream's gradient, loaded with the rest where the registers allow it
    constexpr bool kEarly = Chunks * N <= 32 && Lanes < 1024;
    typename oxh::storage::Pack<T, N>::type stream[kEarly ? Chunks : 1];
    float dot = 0.0f;
#pragma unroll
    for (int c = 0; c < Chunks; ++c) {
      const uint32_t at = (c * Lanes + lane) * N;
#pragma unroll
      for (int i = 0; i < N; ++i) unit[c][i] = d[c][i] = 0.0f;
      if (at >= a.columns) continue;
      const Places here = places_at<N, Ragged>(at, a.columns);
      load_places<T, N, Ragged>(a.s + base, here, unit[c]);
      load_places<T, N, Ragged>(a.g + base, here, d[c]);
      if (kEarly && a.sg != nullptr)
        stream[kEarly ? c : 0] = oxh::storage::raw<T, N>(a.sg + base + here.start);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        unit[c][i] *= q;
        dw[c][i] = fmaf(d[c][i], unit[c][i], dw[c][i]);
        d[c][i] *= w[c][i];
        dot = fmaf(unit[c][i], d[c][i], dot);
      }
    }
    const float mean = row_sum<Lanes>(dot, slot[turn]) * a.inverse_columns;
    turn ^= 1;
#pragma unroll
    for (int c = 0; c < Chunks; ++c) {
      const uint32_t at = (c * Lanes + lane) * N;
      if (at >= a.columns) continue;
      const Places here = places_at<N, Ragged>(at, a.columns);
      float out[N];
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = q * (d[c][i] - unit[c][i] * mean);
      if (a.sg != nullptr) {
        float sg[N];
        if constexpr (kEarly) oxh::storage::widen_all<T, N>(stream[c], sg);
        else oxh::storage::load<T, N>(a.sg + base + here.start, sg);
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] += sg[i];  // skipped ones are not stored
      }
      store_places<T, N, Ragged>(a.dx + base, here, out);
    }
  }
  if (a.partial == nullptr) return;
  float *to = a.partial + static_cast<uint64_t>(blockIdx.x) * a.columns;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int c = 0; c < Chunks; ++c) {
      const uint32_t at = (c * Lanes + lane) * N;
      if (at >= a.columns) continue;
      store_places<float, N, Ragged>(to, places_at<N, Ragged>(at, a.columns), dw[c]);
    }
  } else {
    __shared__ float shares[kGroups][Lanes * Chunks * N];
#pragma unroll
    for (int c = 0; c < Chunks; ++c) {
      const uint32_t at = (c * Lanes + lane) * N;
      if (at >= a.columns) continue;
      store_places<float, N, Ragged>(shares[own], places_at<N, Ragged>(at, a.columns), dw[c]);
    }
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < a.columns; at += 256) {
      float sum = shares[0][at];
#pragma unroll
      for (int i = 1; i < kGroups; ++i) sum += shares[i][at];
      to[at] = sum;
    }
  }
}

// Rows longer than the registers of a block: two passes over a row, and the weight gradient's
// share kept in `partial` itself.
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_backward_long_kernel(Backward<T> a) {
  __shared__ float slot[2][16];
  int turn = 0;
  float *dw = a.partial == nullptr
                  ? nullptr
                  : a.partial + static_cast<uint64_t>(blockIdx.x) * a.columns;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const uint64_t base = row * a.columns;
    const float q = a.q[row];
    float dot = 0.0f;
    for (uint32_t at = threadIdx.x; at < a.columns; at += 1024) {
      const float g = oxh::storage::widen(a.g[base + at]);
      const float unit = oxh::storage::widen(a.s[base + at]) * q;
      dot = fmaf(unit, g * a.w[at], dot);
    }
    const float mean = row_sum<1024>(dot, slot[turn]) * a.inverse_columns;
    turn ^= 1;
    for (uint32_t at = threadIdx.x; at < a.columns; at += 1024) {
      const float g = oxh::storage::widen(a.g[base + at]);
      const float unit = oxh::storage::widen(a.s[base + at]) * q;
      float out = q * (g * a.w[at] - unit * mean);
      if (a.sg != nullptr) out += oxh::storage::widen(a.sg[base + at]);
      a.dx[base + at] = static_cast<T>(out);
      if (dw != nullptr) dw[at] = row == blockIdx.x ? g * unit : fmaf(g, unit, dw[at]);
    }
  }
}

// out[c] = sum over the partial rows: 16 columns per block (from `first` on), 64 strands of rows
// each, a strand's rows in order and the strands by halves.
__global__ __launch_bounds__(1024) void rms_norm_weight_kernel(const float *partial, float *out,
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
  if (strand == 0 && column < columns) out[column] = part[0][c];
}

// Values of a row that a block's registers hold.  The backward keeps five per value of its row and
// its masks need more: past these limits the registers spill, and two passes are faster (bfloat16
// 1024 x 32769: 146 us, 441 in registers; float32 512 x 20001: 53 and 105; within the limits
// bfloat16 1024 x 16383: 46 us, 74 in two passes; float32 1024 x 16384: 40 and 79).
template <typename T>
constexpr uint64_t forward_limit() {
  return 1024 * 8 * (16 / sizeof(T));
}
constexpr uint64_t backward_limit(bool ragged) { return ragged ? 16384 : 32768; }

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

// Blocks that the backward's weight gradient is summed over (rows of `partial`, which stays within
// 8 MB up to 8192 columns).
uint64_t block_limit(uint64_t columns) {
  return std::min<uint64_t>(2048, std::max<uint64_t>(256, (1ull << 21) / columns));
}

oxh_status check_rows(const char *what, int dtype, uint64_t rows, uint64_t columns) {
  OXH_REQUIRE(oxh::storage::valid(dtype), OXH_INVALID_SHAPE,
              std::string(what) + ": dtype is neither OXH_F32 nor OXH_BF16");
  OXH_REQUIRE(columns >= 1 && columns < (1ull << 31), OXH_INVALID_SHAPE,
              std::string(what) + ": columns out of range");
  OXH_REQUIRE(rows < (1ull << 31), OXH_INVALID_SHAPE, std::string(what) + ": too many rows");
  OXH_REQUIRE(rows <= (1ull << 60) / columns, OXH_INVALID_SHAPE,
              std::string(what) + ": element count overflow");
  return oxh::ok();
}

bool aligned_to(const void *p, uint64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// Blocks of so many threads that one launch takes: it numbers its threads with 32 bits.
constexpr uint64_t most_blocks(uint64_t threads) { return (1ull << 31) / threads; }

// The rows in as many launches as that asks for (two from 2^25 rows of a wave each), `per` rows a
// block: run(blocks, rows' arguments).
template <typename T, typename Run>
void by_launches(Forward<T> a, uint64_t threads, uint64_t per, Run run) {
  const uint64_t most = most_blocks(threads) * per;
  for (uint64_t left = a.rows; left != 0; left -= a.rows) {
    a.rows = std::min(left, most);
    run(dim3(static_cast<uint32_t>((a.rows + per - 1) / per)), a);
    const uint64_t on = a.rows * a.columns;
    a.x += on;
    a.y += on;
    if (a.r != nullptr) a.r += on;
    if (a.s != nullptr) a.s += on;
    if (a.q != nullptr) a.q += a.rows;
  }
}

template <typename T>
oxh_status forward(hipStream_t stream, const Forward<T> &a) {
  if (a.columns > forward_limit<T>()) {
    by_launches(a, 1024, 1, [&](dim3 blocks, const Forward<T> &part) {
      oxh::launch(rms_norm_forward_long_kernel<T>, blocks, dim3(1024), 0, stream, part);
    });
    return oxh::launched("rms_norm_forward");
  }
  with_pack<T>(a.columns, [&](auto pack, auto ragged) {
    constexpr int N = decltype(pack)::value;
    with_shape<N, forward_limit<T>()>(a.columns, [&](auto shape) {
      using S = decltype(shape);
      constexpr int threads = S::lanes < 256 ? 256 : S::lanes, per = threads / S::lanes;
      by_launches(a, threads, per, [&](dim3 blocks, const Forward<T> &part) {
        oxh::launch(rms_norm_forward_kernel<T, N, S::lanes, S::chunks, decltype(ragged)::value>,
                    blocks, dim3(threads), 0, stream, part);
      });
    });
  });
  return oxh::launched("rms_norm_forward");
}

// Rows that one block takes by itself, whose share is the weight gradient: a second launch is about
// as long as three more rows of a wave, or one of a block (bfloat16 16 x 1024: 7.2 us a call, 10.1
// with two launches; 32 x 1024: 8.3 and 10.1, but 9.3 and 6.0 on the device; float32 2 x 4096: 7.4
// and 10.1; 8 x 4096: 13.7 and 10.2).
constexpr uint64_t rows_alone(int groups) { return groups > 1 ? 4 * groups : 2; }

template <typename T>
oxh_status backward(hipStream_t stream, Backward<T> a, float *weight_gradient) {
  uint64_t blocks = std::min<uint64_t>(a.rows, block_limit(a.columns));
  // a single block's share is the weight gradient
  auto choose = [&](uint64_t count) {
    blocks = count;
    if (blocks == 1 && weight_gradient != nullptr) a.partial = weight_gradient;
  };
  if (a.columns > backward_limit(a.columns % (16 / sizeof(T)) != 0)) {
    choose(blocks);
    oxh::launch(rms_norm_backward_long_kernel<T>, dim3(static_cast<uint32_t>(blocks)),
                dim3(1024), 0, stream, a);
  } else {
    with_pack<T>(a.columns, [&](auto pack, auto ragged) {
      constexpr int N = decltype(pack)::value;
      with_shape<N, backward_limit(decltype(ragged)::value)>(a.columns, [&](auto shape) {
        using S = decltype(shape);
        constexpr int threads = S::lanes < 256 ? 256 : S::lanes, per = threads / S::lanes;
        // two blocks per compute unit (float32 3584 x 1280: 16.8 us, 20.5 with one, 19.3 with
        // four), and every group the same number of rows, but for the last ones
        const uint64_t most = std::min<uint64_t>(block_limit(a.columns), 512),
                       rounds = (a.rows + most * per - 1) / (most * per);
        choose(a.rows <= rows_alone(per) ? 1 : (a.rows + rounds * per - 1) / (rounds * per));
        oxh::launch(rms_norm_backward_kernel<T, N, S::lanes, S::chunks, decltype(ragged)::value>,
                    dim3(static_cast<uint32_t>(blocks)), dim3(threads), 0, stream, a);
      });
    });
  }
  oxh_status st = oxh::launched("rms_norm_backward");
  if (st != OXH_OK || weight_gradient == nullptr || blocks == 1) return st;
  constexpr uint32_t most = static_cast<uint32_t>(most_blocks(1024)) * 16;
  for (uint32_t first = 0; first < a.columns; first += most)
    oxh::launch(rms_norm_weight_kernel, dim3((std::min(a.columns - first, most) + 15) / 16),
                dim3(1024), 0, stream, static_cast<const float *>(a.partial), weight_gradient,
                static_cast<uint32_t>(blocks), a.columns, first);
  return oxh::launched("rms_norm_weight_gradient");
}

}  // namespace

extern "C" {

oxh_status oxh_rms_norm_forward(oxh_stream stream, int dtype, uint64_t rows, uint64_t columns,
                                float epsilon, const void *input, const void *residual,
                                const float *weight, void *sum, void *output,
                                float *inverse_rms) {
  oxh_status st = check_rows("rms norm", dtype, rows, columns);
  if (st != OXH_OK) return st;
  OXH_REQUIRE(std::isfinite(epsilon) && epsilon >= 0.0f, OXH_EXECUTION,
              "rms norm epsilon must be non-negative and finite");
  if (rows == 0) return oxh::ok();
  OXH_REQUIRE(input != nullptr && weight != nullptr && output != nullptr, OXH_INVALID_SHAPE,
              "rms norm: null pointer");
  const uint64_t bytes = rows * columns * oxh::storage::bytes_of(dtype);
  const uint64_t element = oxh::storage::bytes_of(dtype);
  OXH_REQUIRE(aligned_to(input, element) && aligned_to(residual, element) &&
                  aligned_to(sum, element) && aligned_to(output, element) &&
                  aligned_to(weight, 4) && aligned_to(inverse_rms, 4),
              OXH_INVALID_SHAPE, "rms norm: a pointer is not aligned to its elements");
  // the sum may be written over an operand, nothing else may overlap
  auto apart = [&](const void *a, uint64_t an, const void *b, uint64_t bn) {
    return a == nullptr || b == nullptr || !oxh::any_overlap(a, an, b, bn);
  };
  OXH_REQUIRE(apart(output, bytes, input, bytes) && apart(output, bytes, residual, bytes) &&
                  apart(output, bytes, sum, bytes) && apart(output, bytes, weight, columns * 4) &&
                  apart(sum, bytes, weight, columns * 4) &&
                  apart(inverse_rms, rows * 4, output, bytes) &&
                  apart(inverse_rms, rows * 4, sum, bytes) &&
                  apart(inverse_rms, rows * 4, input, bytes) &&
                  apart(inverse_rms, rows * 4, residual, bytes) &&
                  apart(inverse_rms, rows * 4, weight, columns * 4),
              OXH_INVALID_SHAPE, "rms norm: an output overlaps an operand or another output");
  OXH_REQUIRE(sum == nullptr || (!oxh::partial_overlap(sum, input, bytes) &&
                                 (residual == nullptr ||
                                  !oxh::partial_overlap(sum, residual, bytes))),
              OXH_INVALID_SHAPE, "rms norm: the sum partially overlaps an operand");
  const uint32_t cols = static_cast<uint32_t>(columns);
  const float inverse = 1.0f / static_cast<float>(columns);
  if (dtype == OXH_F32)
    return forward<float>(oxh::as_stream(stream),
                          {static_cast<const float *>(input), static_cast<const float *>(residual),
                           weight, static_cast<float *>(sum), static_cast<float *>(output),
                           inverse_rms, rows, cols, inverse, epsilon});
  return forward<bf16>(oxh::as_stream(stream),
                       {static_cast<const bf16 *>(input), static_cast<const bf16 *>(residual),
                        weight, static_cast<bf16 *>(sum), static_cast<bf16 *>(output),
                        inverse_rms, rows, cols, inverse, epsilon});
}

oxh_status oxh_rms_norm_backward_workspace_size(uint64_t rows, uint64_t columns,
                                                uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  oxh_status st = check_rows("rms norm", OXH_F32, rows, columns);
  if (st != OXH_OK) return st;
  *bytes = (std::min(rows, block_limit(columns)) * columns * 4 + 255) / 256 * 256;
  return oxh::ok();
}

oxh_status oxh_rms_norm_backward(oxh_stream stream, int dtype, uint64_t rows, uint64_t columns,
                                 const void *gradient, const void *sum_gradient,
                                 const void *sum, const float *weight, const float *inverse_rms,
                                 void *input_gradient, float *weight_gradient, void *workspace,
                                 uint64_t workspace_bytes) {
  oxh_status st = check_rows("rms norm backward", dtype, rows, columns);
  if (st != OXH_OK) return st;
  if (rows == 0) {
    if (weight_gradient == nullptr) return oxh::ok();
    return oxh_memset0_async(weight_gradient, columns * 4, stream);
  }
  OXH_REQUIRE(gradient != nullptr && sum != nullptr && weight != nullptr &&
                  inverse_rms != nullptr && input_gradient != nullptr,
              OXH_INVALID_SHAPE, "rms norm backward: null pointer");
  const uint64_t element = oxh::storage::bytes_of(dtype), bytes = rows * columns * element;
  OXH_REQUIRE(aligned_to(gradient, element) && aligned_to(sum_gradient, element) &&
                  aligned_to(sum, element) && aligned_to(input_gradient, element) &&
                  aligned_to(weight, 4) && aligned_to(inverse_rms, 4) &&
                  aligned_to(weight_gradient, 4),
              OXH_INVALID_SHAPE, "rms norm backward: a pointer is not aligned to its elements");
  uint64_t needed = 0;
  if (weight_gradient != nullptr) {
    st = oxh_rms_norm_backward_workspace_size(rows, columns, &needed);
    if (st != OXH_OK) return st;
    OXH_REQUIRE(workspace != nullptr && workspace_bytes >= needed && oxh::aligned16(workspace),
                OXH_INVALID_SHAPE, "rms norm backward: workspace too small or misaligned");
  }
  struct Span {
    const void *p;
    uint64_t n;
  };
  const Span in[] = {{gradient, bytes}, {sum, bytes},           {weight, columns * 4},
                     {inverse_rms, rows * 4}, {sum_gradient, bytes}};
  const Span out[] = {{input_gradient, bytes}, {weight_gradient, columns * 4},
                      {needed != 0 ? workspace : nullptr, needed}};
  for (int o = 0; o < 3; ++o) {
    if (out[o].p == nullptr) continue;
    for (int i = 0; i < 5; ++i) {
      if (in[i].p == nullptr || (o == 0 && i == 4 && in[i].p == out[o].p)) continue;
      OXH_REQUIRE(!oxh::any_overlap(out[o].p, out[o].n, in[i].p, in[i].n), OXH_INVALID_SHAPE,
                  "rms norm backward: an output or the workspace overlaps an operand");
    }
    for (int k = 0; k < o; ++k)
      OXH_REQUIRE(out[k].p == nullptr ||
                      !oxh::any_overlap(out[o].p, out[o].n, out[k].p, out[k].n),
                  OXH_INVALID_SHAPE, "rms norm backward: two outputs overlap");
  }
  const uint32_t cols = static_cast<uint32_t>(columns);
  const float inverse = 1.0f / static_cast<float>(columns);
  float *partial = weight_gradient != nullptr ? static_cast<float *>(workspace) : nullptr;
  if (dtype == OXH_F32)
    return backward<float>(
        oxh::as_stream(stream),
        {static_cast<const float *>(gradient), static_cast<const float *>(sum_gradient),
         static_cast<const float *>(sum), weight, inverse_rms,
         static_cast<float *>(input_gradient), partial, rows, cols, inverse},
        weight_gradient);
  return backward<bf16>(
      oxh::as_stream(stream),
      {static_cast<const bf16 *>(gradient), static_cast<const bf16 *>(sum_gradient),
       static_cast<const bf16 *>(sum), weight, inverse_rms, static_cast<bf16 *>(input_gradient),
       partial, rows, cols, inverse},
      weight_gradient);
}

}  // extern "C"
