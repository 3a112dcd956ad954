// layer_norm.hip -- layer norm over the last dimension, of a residual sum where there is one, and
// its gradients.
//
//   s = x + r;  m = mean(s);  q = 1 / sqrt(mean((s - m)^2) + epsilon);  y = (s - m) q w + b
//   u = (s - m) q;  d = dy w;  dx = dr = ds + q (d - mean(d) - u mean(u d))
//   dw = sum over rows of dy u;  db = sum over rows of dy
//
// Rows are float32 or bfloat16; the sum, the statistics, the dot products and the parameters'
// gradients are float32, and each output is rounded once (y from the unrounded s).  The variance
// is the mean of squared deviations from the row's own mean, not a difference of moments, so a row
// far from zero keeps its digits.
//
// The bound is memory, so a row is read once and kept in registers over both of its statistics:
// bfloat16 16384 x 4096 forward with the sum 97 to 103 us (537 MB, 5.2 to 5.5 TB/s), backward with the
// parameters' gradients 105 us a call (537 MB, 5.1 TB/s; its kernels 99 to 103 and 7 for the blocks'
// shares).  Small ones are launches and a row's load, sum and store: 1 x 2048 3 us of 6.5 a call,
// backward float32 1021 x 1537 16.7 a call, its kernels 14 and 4 in a trace (its rows begin anywhere:
// 1021 x 1536 takes 10 and 4 there).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "common.h"
#include "row_norm.h"
#include "storage.h"

namespace {

using namespace oxh::row_norm;
using oxh::storage::bf16;
using oxh::storage::load_places;
using oxh::storage::Places;
using oxh::storage::places_at;
using oxh::storage::store_places;
using oxh::storage::widen;

// The place of an access at `at`, which past the row's end is the row's last one again: so no load is
// behind a branch, and all are on their way before the first is used.
template <int N>
__device__ __forceinline__ uint32_t inside(uint32_t at, uint32_t columns) {
  return min(at, columns - N);
}
// Its values, those skipped or past the row's end 0.
template <typename T, int N>
__device__ __forceinline__ void counted(const typename oxh::storage::Pack<T, N>::type &x,
                                        uint32_t at, uint32_t columns, float (&v)[N]) {
  oxh::storage::widen_all<T, N>(x, v);
  const uint32_t skip = at - inside<N>(at, columns);
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) v[i] = i < skip ? 0.0f : v[i];
}

// Stores access c of a row's lane.  A ragged row's last one goes value by value, in the one chunk that
// holds it: the others have no such path to pass (float32 1021 x 1537 backward: 16.7 us a call, 17.5
// with a path in each).
template <typename T, int N, int Lanes, bool Ragged>
__device__ __forceinline__ void store_chunk(T *row, int c, uint32_t lane, uint32_t columns,
                                            const float (&v)[N]) {
  const uint32_t at = (c * Lanes + lane) * N;
  if (at + N <= columns) {
    oxh::storage::store<T, N>(row + at, v);
  } else if constexpr (Ragged) {
    if (static_cast<uint32_t>(c) != (columns - 1) / (Lanes * N) || at >= columns) return;
    store_places<T, N, true>(row, places_at<N, true>(at, columns), v);
  }
}

template <typename T>
struct Forward {
  const T *x, *r;
  const float *w, *b;
  T *s, *y;
  float *m, *q;
  uint64_t rows;
  uint32_t columns;
  float inverse_columns, epsilon;
};

// One row per Lanes threads, kept in registers: Chunks accesses of N values per thread cover it.
template <typename T, int N, int Lanes, int Chunks, bool Ragged>
__global__ __launch_bounds__(Lanes < 256 ? 256 : Lanes) void layer_norm_forward_kernel(
    Forward<T> a) {
  __shared__ float slot[2][16];
  constexpr int kRows = Lanes < 256 ? 256 / Lanes : 1;
  const uint32_t lane = threadIdx.x % Lanes;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kRows + threadIdx.x / Lanes;
  if (row >= a.rows) return;  // whole waves: Lanes == 64 when a block holds several rows
  const uint64_t base = row * a.columns;
  using Pack = typename oxh::storage::Pack<T, N>::type;
  Pack x[Chunks], r[Chunks];
#pragma unroll
  for (int c = 0; c < Chunks; ++c)
    x[c] = oxh::storage::raw<T, N>(a.x + base + inside<N>((c * Lanes + lane) * N, a.columns));
  if (a.r != nullptr)
#pragma unroll
    for (int c = 0; c < Chunks; ++c)
      r[c] = oxh::storage::raw<T, N>(a.r + base + inside<N>((c * Lanes + lane) * N, a.columns));
  float v[Chunks][N];
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
    counted<T, N>(x[c], at, a.columns, v[c]);
    if (a.r != nullptr) {
      float more[N];
      counted<T, N>(r[c], at, a.columns, more);
#pragma unroll
      for (int i = 0; i < N; ++i) v[c][i] += more[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) sum += v[c][i];
  }
  const float mean = row_sum<Lanes>(sum, slot[0]) * a.inverse_columns;
  float squares = 0.0f;
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
    if (at >= a.columns) continue;
    const Places here = places_at<N, Ragged>(at, a.columns);
    if (a.s != nullptr) store_chunk<T, N, Lanes, Ragged>(a.s + base, c, lane, a.columns, v[c]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[c][i] -= mean;
      const float counted = Ragged && static_cast<uint32_t>(i) < here.skip ? 0.0f : v[c][i];
      squares = fmaf(counted, counted, squares);
    }
  }
  const float q = 1.0f / sqrtf(row_sum<Lanes>(squares, slot[1]) * a.inverse_columns + a.epsilon);
  if (lane == 0) {
    if (a.m != nullptr) a.m[row] = mean;
    if (a.q != nullptr) a.q[row] = q;
  }
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
    if (at >= a.columns) continue;
    const Places here = places_at<N, Ragged>(at, a.columns);
    float w[N], b[N];
    load_places<float, N, Ragged>(a.w, here, w);
    if (a.b != nullptr) load_places<float, N, Ragged>(a.b, here, b);
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[c][i] = fmaf(v[c][i] * q, w[i], a.b != nullptr ? b[i] : 0.0f);
    store_chunk<T, N, Lanes, Ragged>(a.y + base, c, lane, a.columns, v[c]);
  }
}

// Rows longer than the registers of a block: three passes over the operands, each of which forms
// the sum again (from x and r, not from the rounded one); a thread reads an element for the last
// time before it writes it, so s may be x or r here too.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_forward_long_kernel(Forward<T> a) {
  __shared__ float slot[2][16];
  const uint64_t base = static_cast<uint64_t>(blockIdx.x) * a.columns;
  auto value = [&](uint32_t at) {
    float v = widen(a.x[base + at]);
    if (a.r != nullptr) v += widen(a.r[base + at]);
    return v;
  };
  float sum = 0.0f;
  for (uint32_t at = threadIdx.x; at < a.columns; at += 1024) sum += value(at);
  const float mean = row_sum<1024>(sum, slot[0]) * a.inverse_columns;
  float squares = 0.0f;
  for (uint32_t at = threadIdx.x; at < a.columns; at += 1024) {
    const float v = value(at) - mean;
    squares = fmaf(v, v, squares);
  }
  const float q = 1.0f / sqrtf(row_sum<1024>(squares, slot[1]) * a.inverse_columns + a.epsilon);
  if (threadIdx.x == 0) {
    if (a.m != nullptr) a.m[blockIdx.x] = mean;
    if (a.q != nullptr) a.q[blockIdx.x] = q;
  }
  for (uint32_t at = threadIdx.x; at < a.columns; at += 1024) {
    const float v = value(at);
    if (a.s != nullptr) a.s[base + at] = static_cast<T>(v);
    a.y[base + at] =
        static_cast<T>(fmaf((v - mean) * q, a.w[at], a.b != nullptr ? a.b[at] : 0.0f));
  }
}

// The blocks' shares of dw and db: rows `stride` apart (both null where neither is asked for; a
// single block's are the gradients, of which one may be null).
template <typename T>
struct Backward {
  const T *g, *sg, *s;
  const float *w, *m, *q;
  T *dx;
  float *dw, *db;
  uint64_t rows, stride;
  uint32_t columns;
  float inverse_columns;
};

// Each group of Lanes threads takes every groups-th row and keeps its shares of dw and db in
// registers; a block's groups add theirs in shared memory, in order, and each block's sums go to
// its row of the shares.
template <typename T, int N, int Lanes, int Chunks, bool Ragged>
__global__ __launch_bounds__(Lanes < 256 ? 256 : Lanes) void layer_norm_backward_kernel(
    Backward<T> a) {
  __shared__ float slot[2][2][16];
  constexpr int kGroups = Lanes < 256 ? 256 / Lanes : 1;  // of a block
  const uint32_t lane = threadIdx.x % Lanes, own = threadIdx.x / Lanes;
  const uint64_t groups = static_cast<uint64_t>(gridDim.x) * kGroups;
  float dw[Chunks][N], db[Chunks][N], w[Chunks][N];
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
#pragma unroll
    for (int i = 0; i < N; ++i) dw[c][i] = db[c][i] = w[c][i] = 0.0f;
    if (at < a.columns)
      load_places<float, N, Ragged>(a.w, places_at<N, Ragged>(at, a.columns), w[c]);
  }
  int turn = 0;
  for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * kGroups + own; row < a.rows;
       row += groups) {
    const uint64_t base = row * a.columns;
    const float q = a.q[row], m = a.m[row];
    float unit[Chunks][N], d[Chunks][N];
    // the stream's gradient, loaded with the rest where the registers allow it
    constexpr bool kEarly = Chunks * N <= 32 && Lanes < 1024;
    typename oxh::storage::Pack<T, N>::type stream[kEarly ? Chunks : 1];
    float dots[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < Chunks; ++c) {
      const uint32_t at = (c * Lanes + lane) * N;
#pragma unroll
      for (int i = 0; i < N; ++i) unit[c][i] = d[c][i] = 0.0f;
      if (at >= a.columns) continue;
      const Places here = places_at<N, Ragged>(at, a.columns);
      load_places<T, N, Ragged>(a.s + base, here, unit[c]);
      load_places<T, N, Ragged>(a.g + base, here, d[c]);  // skipped ones are 0: so are their sums
      if (kEarly && a.sg != nullptr)
        stream[kEarly ? c : 0] = oxh::storage::raw<T, N>(a.sg + base + here.start);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        unit[c][i] = (unit[c][i] - m) * q;
        dw[c][i] = fmaf(d[c][i], unit[c][i], dw[c][i]);
        db[c][i] += d[c][i];
        d[c][i] *= w[c][i];
        dots[0] += d[c][i];
        dots[1] = fmaf(unit[c][i], d[c][i], dots[1]);
      }
    }
    row_sums<Lanes>(dots, slot[turn]);
    turn ^= 1;
    const float mean = dots[0] * a.inverse_columns, along = dots[1] * a.inverse_columns;
#pragma unroll
    for (int c = 0; c < Chunks; ++c) {
      const uint32_t at = (c * Lanes + lane) * N;
      if (at >= a.columns) continue;
      const Places here = places_at<N, Ragged>(at, a.columns);
      float out[N];
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = q * (d[c][i] - mean - unit[c][i] * along);
      if (a.sg != nullptr) {
        float sg[N];
        if constexpr (kEarly) oxh::storage::widen_all<T, N>(stream[c], sg);
        else oxh::storage::load<T, N>(a.sg + base + here.start, sg);
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] += sg[i];  // skipped ones are not stored
      }
      store_chunk<T, N, Lanes, Ragged>(a.dx + base, c, lane, a.columns, out);
    }
  }
  // Skipped values of a ragged access belong to another thread's: their shares are 0 there and are
  // not stored.
  auto share = [&](const float (&v)[Chunks][N], float *to) {
    if constexpr (kGroups == 1) {
      if (to == nullptr) return;
#pragma unroll
      for (int c = 0; c < Chunks; ++c)
        store_chunk<float, N, Lanes, Ragged>(to, c, lane, a.columns, v[c]);
    } else {
      __shared__ float shares[kGroups][Lanes * Chunks * N];
      if (to == nullptr) return;  // the same for the whole block
      __syncthreads();
#pragma unroll
      for (int c = 0; c < Chunks; ++c)
        store_chunk<float, N, Lanes, Ragged>(shares[own], c, lane, a.columns, v[c]);
      __syncthreads();
      for (uint32_t at = threadIdx.x; at < a.columns; at += 256) {
        float sum = shares[0][at];
#pragma unroll
        for (int i = 1; i < kGroups; ++i) sum += shares[i][at];
        to[at] = sum;
      }
    }
  };
  const uint64_t row = blockIdx.x * a.stride;
  share(dw, a.dw == nullptr ? nullptr : a.dw + row);
  share(db, a.db == nullptr ? nullptr : a.db + row);
}

// Rows longer than the registers of a block: two passes over a row, and the shares of dw and db
// kept in memory.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_backward_long_kernel(Backward<T> a) {
  __shared__ float slot[2][2][16];
  int turn = 0;
  float *dw = a.dw == nullptr ? nullptr : a.dw + blockIdx.x * a.stride;
  float *db = a.db == nullptr ? nullptr : a.db + blockIdx.x * a.stride;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const uint64_t base = row * a.columns;
    const float q = a.q[row], m = a.m[row];
    float dots[2] = {0.0f, 0.0f};
    for (uint32_t at = threadIdx.x; at < a.columns; at += 1024) {
      const float d = widen(a.g[base + at]) * a.w[at];
      dots[0] += d;
      dots[1] = fmaf((widen(a.s[base + at]) - m) * q, d, dots[1]);
    }
    row_sums<1024>(dots, slot[turn]);
    turn ^= 1;
    const float mean = dots[0] * a.inverse_columns, along = dots[1] * a.inverse_columns;
    const bool first = row == blockIdx.x;
    for (uint32_t at = threadIdx.x; at < a.columns; at += 1024) {
      const float g = widen(a.g[base + at]), unit = (widen(a.s[base + at]) - m) * q;
      float out = q * (g * a.w[at] - mean - unit * along);
      if (a.sg != nullptr) out += widen(a.sg[base + at]);
      a.dx[base + at] = static_cast<T>(out);
      if (dw != nullptr) dw[at] = first ? g * unit : fmaf(g, unit, dw[at]);
      if (db != nullptr) db[at] = first ? g : db[at] + g;
    }
  }
}

// Values of a row that a block's registers hold, the backward's with seven for each (float32 1024 x
// 16384 backward: 49 us, 104 in two passes over the row; bfloat16 4096 x 10240 86 and 248).
template <typename T>
constexpr uint64_t forward_limit() {
  return 1024 * 8 * (16 / sizeof(T));
}
constexpr uint64_t kBackwardLimit = 16384;

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
    if (a.m != nullptr) a.m += a.rows;
    if (a.q != nullptr) a.q += a.rows;
  }
}

template <typename T>
oxh_status forward(hipStream_t stream, const Forward<T> &a) {
  if (a.columns > forward_limit<T>()) {
    by_launches(a, 1024, 1, [&](dim3 blocks, const Forward<T> &part) {
      oxh::launch(layer_norm_forward_long_kernel<T>, blocks, dim3(1024), 0, stream, part);
    });
    return oxh::launched("layer_norm_forward");
  }
  with_pack<T>(a.columns, [&](auto pack, auto ragged) {
    constexpr int N = decltype(pack)::value;
    with_shape<N, forward_limit<T>()>(a.columns, [&](auto shape) {
      using S = decltype(shape);
      constexpr int threads = S::lanes < 256 ? 256 : S::lanes, per = threads / S::lanes;
      by_launches(a, threads, per, [&](dim3 blocks, const Forward<T> &part) {
        oxh::launch(layer_norm_forward_kernel<T, N, S::lanes, S::chunks, decltype(ragged)::value>,
                    blocks, dim3(threads), 0, stream, part);
      });
    });
  });
  return oxh::launched("layer_norm_forward");
}

// partial: the blocks' shares, [blocks][dw | db], null where neither gradient is asked for.
template <typename T>
oxh_status backward(hipStream_t stream, Backward<T> a, float *partial, float *weight_gradient,
                    float *bias_gradient) {
  uint64_t blocks = std::min<uint64_t>(a.rows, block_limit(a.columns));
  a.stride = 2ull * a.columns;
  auto choose = [&](uint64_t count) {
    blocks = count;
    const bool alone = blocks == 1;  // its shares are the gradients
    a.dw = alone ? weight_gradient : partial;
    a.db = alone ? bias_gradient : partial == nullptr ? nullptr : partial + a.columns;
  };
  if (a.columns > kBackwardLimit) {
    choose(blocks);
    oxh::launch(layer_norm_backward_long_kernel<T>, dim3(static_cast<uint32_t>(blocks)),
                dim3(1024), 0, stream, a);
  } else {
    with_pack<T>(a.columns, [&](auto pack, auto ragged) {
      constexpr int N = decltype(pack)::value;
      with_shape<N, kBackwardLimit>(a.columns, [&](auto shape) {
        using S = decltype(shape);
        constexpr int threads = S::lanes < 256 ? 256 : S::lanes, per = threads / S::lanes;
        // two blocks per compute unit, every group the same number of rows but for the last ones
        const uint64_t most = std::min<uint64_t>(block_limit(a.columns), 512),
                       rounds = (a.rows + most * per - 1) / (most * per);
        choose(a.rows <= rows_alone(per) ? 1 : (a.rows + rounds * per - 1) / (rounds * per));
        oxh::launch(
            layer_norm_backward_kernel<T, N, S::lanes, S::chunks, decltype(ragged)::value>,
            dim3(static_cast<uint32_t>(blocks)), dim3(threads), 0, stream, a);
      });
    });
  }
  oxh_status st = oxh::launched("layer_norm_backward");
  if (st != OXH_OK || partial == nullptr || blocks == 1) return st;
  launch_column_sums(stream, partial, weight_gradient, bias_gradient, a.columns,
                     static_cast<uint32_t>(blocks), 2 * a.columns);
  return oxh::launched("layer_norm_parameter_gradients");
}

}  // namespace

extern "C" {

oxh_status oxh_layer_norm_forward(oxh_stream stream, int dtype, uint64_t rows, uint64_t columns,
                                  float epsilon, const void *input, const void *residual,
                                  const float *weight, const float *bias, void *sum, void *output,
                                  float *mean, float *inverse_deviation) {
  oxh_status st = check_rows("layer norm", dtype, rows, columns);
  if (st != OXH_OK) return st;
  OXH_REQUIRE(std::isfinite(epsilon) && epsilon >= 0.0f, OXH_EXECUTION,
              "layer norm epsilon must be non-negative and finite");
  if (rows == 0) return oxh::ok();
  OXH_REQUIRE(input != nullptr && weight != nullptr && output != nullptr, OXH_INVALID_SHAPE,
              "layer norm: null pointer");
  const uint64_t element = oxh::storage::bytes_of(dtype), bytes = rows * columns * element;
  OXH_REQUIRE(aligned_to(input, element) && aligned_to(residual, element) &&
                  aligned_to(sum, element) && aligned_to(output, element) &&
                  aligned_to(weight, 4) && aligned_to(bias, 4) && aligned_to(mean, 4) &&
                  aligned_to(inverse_deviation, 4),
              OXH_INVALID_SHAPE, "layer norm: a pointer is not aligned to its elements");
  // the sum may be written over an operand, nothing else may overlap
  struct Span {
    const void *p;
    uint64_t n;
  };
  const Span in[] = {{input, bytes}, {residual, bytes}, {weight, columns * 4}, {bias, columns * 4}};
  const Span out[] = {{sum, bytes}, {output, bytes}, {mean, rows * 4}, {inverse_deviation, rows * 4}};
  for (int o = 0; o < 4; ++o) {
    if (out[o].p == nullptr) continue;
    for (int i = 0; i < 4; ++i) {
      if (in[i].p == nullptr || (o == 0 && i < 2 && in[i].p == out[o].p)) continue;
      OXH_REQUIRE(!oxh::any_overlap(out[o].p, out[o].n, in[i].p, in[i].n), OXH_INVALID_SHAPE,
                  "layer norm: an output overlaps an operand");
    }
    for (int k = 0; k < o; ++k)
      OXH_REQUIRE(out[k].p == nullptr ||
                      !oxh::any_overlap(out[o].p, out[o].n, out[k].p, out[k].n),
                  OXH_INVALID_SHAPE, "layer norm: two outputs overlap");
  }
  const uint32_t cols = static_cast<uint32_t>(columns);
  const float inverse = 1.0f / static_cast<float>(columns);
  if (dtype == OXH_F32)
    return forward<float>(oxh::as_stream(stream),
                          {static_cast<const float *>(input), static_cast<const float *>(residual),
                           weight, bias, static_cast<float *>(sum), static_cast<float *>(output),
                           mean, inverse_deviation, rows, cols, inverse, epsilon});
  return forward<bf16>(oxh::as_stream(stream),
                       {static_cast<const bf16 *>(input), static_cast<const bf16 *>(residual),
                        weight, bias, static_cast<bf16 *>(sum), static_cast<bf16 *>(output), mean,
                        inverse_deviation, rows, cols, inverse, epsilon});
}

oxh_status oxh_layer_norm_backward_workspace_size(uint64_t rows, uint64_t columns,
                                                  uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  oxh_status st = check_rows("layer norm", OXH_F32, rows, columns);
  if (st != OXH_OK) return st;
  *bytes = (std::min(rows, block_limit(columns)) * columns * 8 + 255) / 256 * 256;
  return oxh::ok();
}

oxh_status oxh_layer_norm_backward(oxh_stream stream, int dtype, uint64_t rows, uint64_t columns,
                                   const void *gradient, const void *sum_gradient,
                                   const void *sum, const float *weight, const float *mean,
                                   const float *inverse_deviation, void *input_gradient,
                                   float *weight_gradient, float *bias_gradient, void *workspace,
                                   uint64_t workspace_bytes) {
  oxh_status st = check_rows("layer norm backward", dtype, rows, columns);
  if (st != OXH_OK) return st;
  const bool parameters = weight_gradient != nullptr || bias_gradient != nullptr;
  OXH_REQUIRE(!parameters || columns < (1ull << 30), OXH_INVALID_SHAPE,
              "layer norm backward: columns out of range");
  if (rows == 0) {
    if (weight_gradient != nullptr) st = oxh_memset0_async(weight_gradient, columns * 4, stream);
    if (st != OXH_OK || bias_gradient == nullptr) return st;
    return oxh_memset0_async(bias_gradient, columns * 4, stream);
  }
  OXH_REQUIRE(gradient != nullptr && sum != nullptr && weight != nullptr && mean != nullptr &&
                  inverse_deviation != nullptr && input_gradient != nullptr,
              OXH_INVALID_SHAPE, "layer norm backward: null pointer");
  const uint64_t element = oxh::storage::bytes_of(dtype), bytes = rows * columns * element;
  OXH_REQUIRE(aligned_to(gradient, element) && aligned_to(sum_gradient, element) &&
                  aligned_to(sum, element) && aligned_to(input_gradient, element) &&
                  aligned_to(weight, 4) && aligned_to(mean, 4) &&
                  aligned_to(inverse_deviation, 4) && aligned_to(weight_gradient, 4) &&
                  aligned_to(bias_gradient, 4),
              OXH_INVALID_SHAPE, "layer norm backward: a pointer is not aligned to its elements");
  uint64_t needed = 0;
  if (parameters) {
    st = oxh_layer_norm_backward_workspace_size(rows, columns, &needed);
    if (st != OXH_OK) return st;
    OXH_REQUIRE(workspace != nullptr && workspace_bytes >= needed && oxh::aligned16(workspace),
                OXH_INVALID_SHAPE, "layer norm backward: workspace too small or misaligned");
  }
  struct Span {
    const void *p;
    uint64_t n;
  };
  const Span in[] = {{gradient, bytes}, {sum, bytes}, {weight, columns * 4}, {mean, rows * 4},
                     {inverse_deviation, rows * 4}, {sum_gradient, bytes}};
  const Span out[] = {{input_gradient, bytes}, {weight_gradient, columns * 4},
                      {bias_gradient, columns * 4}, {needed != 0 ? workspace : nullptr, needed}};
  for (int o = 0; o < 4; ++o) {
    if (out[o].p == nullptr) continue;
    for (int i = 0; i < 6; ++i) {
      if (in[i].p == nullptr || (o == 0 && i == 5 && in[i].p == out[o].p)) continue;
      OXH_REQUIRE(!oxh::any_overlap(out[o].p, out[o].n, in[i].p, in[i].n), OXH_INVALID_SHAPE,
                  "layer norm backward: an output or the workspace overlaps an operand");
    }
    for (int k = 0; k < o; ++k)
      OXH_REQUIRE(out[k].p == nullptr ||
                      !oxh::any_overlap(out[o].p, out[o].n, out[k].p, out[k].n),
                  OXH_INVALID_SHAPE, "layer norm backward: two outputs overlap");
  }
  const uint32_t cols = static_cast<uint32_t>(columns);
  const float inverse = 1.0f / static_cast<float>(columns);
  float *partial = parameters ? static_cast<float *>(workspace) : nullptr;
  if (dtype == OXH_F32)
    return backward<float>(
        oxh::as_stream(stream),
        {static_cast<const float *>(gradient), static_cast<const float *>(sum_gradient),
         static_cast<const float *>(sum), weight, mean, inverse_deviation,
         static_cast<float *>(input_gradient), nullptr, nullptr, rows, 0, cols, inverse},
        partial, weight_gradient, bias_gradient);
  return backward<bf16>(
      oxh::as_stream(stream),
      {static_cast<const bf16 *>(gradient), static_cast<const bf16 *>(sum_gradient),
       static_cast<const bf16 *>(sum), weight, mean, inverse_deviation,
       static_cast<bf16 *>(input_gradient), nullptr, nullptr, rows, 0, cols, inverse},
      partial, weight_gradient, bias_gradient);
}

}  // extern "C"
