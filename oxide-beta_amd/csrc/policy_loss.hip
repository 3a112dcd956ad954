// policy_loss.hip -- the clipped policy loss with a KL term of rows of logits, and its gradient
// with respect to the logits.
//
//   p = softmax(x);  l = log p[action];  r = exp(l - old);  d = reference - l
//   loss of a row = -min(r A, clip(r, 1 - low, 1 + high) A) + kl (exp(d) - d - 1)
//   loss = sum of w * row's;  dx = outer w c (onehot - p),  c = -[r free] r A + kl (1 - exp(d))
//
// r is free where the minimum takes r A: below 1 + high for A >= 0, above 1 - low for A < 0 (the
// borders among it).  A row of weight 0 is not read: its gradient and its log probability are 0.
//
// Logits are float32 or bfloat16.  Exponentials are float32, their sum over the threads, the
// logarithm and everything a row comes to float64 (a ratio next to the clip's border, a loss whose
// rows cancel), by one wave of the row's threads; a gradient is rounded once.
//
// The bound is memory: a row is read once, kept in registers, and its gradient written from them
// (bfloat16 8192 x 32768: 218 us a call, 1.07 GB at 4.9 TB/s, 96 % of a large copy's rate; a trace has
// 218 to 223 and 5 for the sum of the rows' losses, 236 to 243 for a program's first calls).  Few rows
// are launches: float32 509 x 1003 10.7 us a call, its kernels 5.5 and 1.7.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "common.h"
#include "row_norm.h"
#include "softmax.h"
#include "storage.h"

namespace {

using oxh::softmax::exp_nonpos;
using oxh::softmax::target_index;
using oxh::storage::bf16;
using oxh::storage::load;
using oxh::storage::Pack;
using oxh::storage::Places;
using oxh::storage::places_at;
using oxh::storage::raw;
using oxh::storage::store_places;
using oxh::storage::widen;
using oxh::storage::widen_all;

template <typename T>
struct Args {
  const T *logits;
  const float *actions, *old, *advantages, *reference, *weights, *outer;
  T *gradient;
  float *log_probs, *loss;
  uint32_t *error_flag;
  double *row_loss;
  uint64_t rows, classes;
  float low, high, kl;
};

// What a row comes to: its share of the loss, the slope of it along the log probability, and that.
struct Row {
  double loss, slope, log_prob;
};
template <typename T>
__device__ __forceinline__ Row row_value(const Args<T> &a, uint64_t row, double weight,
                                         double log_prob) {
  const double advantage = a.advantages[row];
  const double ratio = exp(log_prob - static_cast<double>(a.old[row]));
  const double low = 1.0 - static_cast<double>(a.low), high = 1.0 + static_cast<double>(a.high);
  const double held = ratio < low ? low : ratio > high ? high : ratio;  // NaN stays
  const double gain = ratio * advantage, bound = held * advantage;
  const bool free = !(gain > bound);
  Row r{free ? -gain : -bound, free ? -gain : 0.0, log_prob};
  if (a.reference != nullptr) {
    const double d = static_cast<double>(a.reference[row]) - log_prob, e = expm1(d);
    r.loss += static_cast<double>(a.kl) * (e - d);
    r.slope -= static_cast<double>(a.kl) * e;
  }
  r.loss *= weight;
  r.slope *= weight;
  return r;
}

template <typename T>
__device__ __forceinline__ double weight_of(const Args<T> &a, uint64_t row) {
  return a.weights != nullptr ? static_cast<double>(a.weights[row])
                              : 1.0 / static_cast<double>(a.rows);
}

template <typename T>
__device__ __forceinline__ float exp_of(float x, float maximum) {
  if constexpr (sizeof(T) == 2) {
    // Of bfloat16 logits: the product is rounded, and its constant, to 1.3 |d| of 2^-24.  In the sum
    // that counts as p |d|, in all no more than the entropy of p, below ln(classes): the logarithm,
    // which the float32 log probability and loss take, is off by less than 2^-19 from this.
    return __builtin_amdgcn_exp2f((x - maximum) * 1.44269502162933349609375f);
  } else {
    return exp_nonpos(x - maximum);
  }
}

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, oxh::dpp_move<0xB1>(v));
  v = fmaxf(v, oxh::dpp_move<0x4E>(v));
  v = fmaxf(v, oxh::dpp_move<0x141>(v));
  v = fmaxf(v, oxh::dpp_move<0x140>(v));
  return fmaxf(fmaxf(oxh::read_lane(v, 0), oxh::read_lane(v, 16)),
               fmaxf(oxh::read_lane(v, 32), oxh::read_lane(v, 48)));
}

// One row per Lanes threads, kept in registers: Chunks accesses of N values per thread cover it.
template <typename T, int N, int Lanes, int Chunks, bool Ragged>
__global__ __launch_bounds__(Lanes < 256 ? 256 : Lanes) void policy_loss_kernel(Args<T> a) {
  constexpr int kRows = Lanes < 256 ? 256 / Lanes : 1, kWaves = Lanes / 64;
  __shared__ float most[kWaves];
  __shared__ double sums[kWaves];
  __shared__ float scale[2];
  const uint32_t lane = threadIdx.x % Lanes, columns = static_cast<uint32_t>(a.classes);
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kRows + threadIdx.x / Lanes;
  if (row >= a.rows) return;  // whole waves: Lanes == 64 when a block holds several rows
  const uint64_t base = row * a.classes;
  const double weight = weight_of(a, row);
  const bool leader = lane < 64;  // of the wave that forms what the row comes to
  if (weight == 0.0) {            // the same for all of the row's threads
    if (lane == 0) {
      if (a.log_probs != nullptr) a.log_probs[row] = 0.0f;
      if (a.loss != nullptr) a.row_loss[row] = 0.0;
    }
    if (a.gradient == nullptr) return;
    float zero[N] = {};
#pragma unroll
    for (int c = 0; c < Chunks; ++c) {
      const uint32_t at = (c * Lanes + lane) * N;
      if (at < columns)
        store_places<T, N, Ragged>(a.gradient + base, places_at<N, Ragged>(at, columns), zero);
    }
    return;
  }
  typename Pack<T, N>::type x[Chunks];
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
    if (at < columns) x[c] = raw<T, N>(a.logits + base + places_at<N, Ragged>(at, columns).start);
  }
  uint64_t action = 0;
  const bool valid = target_index(a.actions[row], a.classes, action);
  const float chosen = widen(a.logits[base + action]);
  float m = -INFINITY;
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
    if (at >= columns) continue;
    float v[N];
    widen_all<T, N>(x[c], v);  // a ragged access repeats values of the row: the same maximum
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);
  }
  m = wave_max(m);
  if constexpr (kWaves > 1) {
    if (threadIdx.x % 64 == 0) most[threadIdx.x / 64] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) m = fmaxf(m, most[i]);
  }
  float part = 0.0f;
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
    if (at >= columns) continue;
    const Places here = places_at<N, Ragged>(at, columns);
    float v[N];
    widen_all<T, N>(x[c], v);
    float own = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = exp_of<T>(v[i], m);
      own += Ragged && static_cast<uint32_t>(i) < here.skip ? 0.0f : v[i];
    }
    part += own;
    if constexpr (sizeof(T) == 4) {  // kept for the gradient
      if constexpr (N == 1) {
        x[c] = v[0];
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[c][i] = v[i];
      }
    }
  }
  double total[1] = {static_cast<double>(part)};
  oxh::wave_sums_rows(total);
  if constexpr (kWaves > 1) {
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = total[0];
    __syncthreads();
  }
  float off = 0.0f, at_action = 0.0f;  // the gradient is e * off, but for the action's
  if (leader) {
    if constexpr (kWaves > 1) {
      total[0] = 0.0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) total[0] += sums[i];
    }
    const double away = static_cast<double>(chosen) - static_cast<double>(m);
    Row r = row_value(a, row, weight, away - log(total[0]));
    if (!valid) r = {NAN, NAN, NAN};
    if (lane == 0) {
      if (!valid && a.error_flag != nullptr) *a.error_flag = 1u;
      if (a.log_probs != nullptr) a.log_probs[row] = static_cast<float>(r.log_prob);
      if (a.loss != nullptr) a.row_loss[row] = r.loss;
    }
    if (a.gradient != nullptr) {
      const double slope = r.slope * static_cast<double>(*a.outer);
      off = static_cast<float>(-slope / total[0]);
      // 1 - p of the others' exponentials
      const double own = static_cast<double>(exp_of<T>(chosen, m));
      at_action = static_cast<float>(slope * ((total[0] - own) / total[0]));
      if (kWaves > 1 && lane == 0) {
        scale[0] = off;
        scale[1] = at_action;
      }
    }
  }
  if (a.gradient == nullptr) return;
  if constexpr (kWaves > 1) {
    __syncthreads();
    off = scale[0];
    at_action = scale[1];
  }
#pragma unroll
  for (int c = 0; c < Chunks; ++c) {
    const uint32_t at = (c * Lanes + lane) * N;
    if (at >= columns) continue;
    const Places here = places_at<N, Ragged>(at, columns);
    float v[N];
    widen_all<T, N>(x[c], v);
    const uint64_t place = action - here.start;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = exp_of<T>(v[i], m);
      v[i] = place == static_cast<uint64_t>(i) ? at_action : v[i] * off;
    }
    store_places<T, N, Ragged>(a.gradient + base, here, v);
  }
}

// Rows longer than the registers of a block: a pass for the maximum and the sum below it, rescaled
// where the maximum grows, and one for the gradient.
template <typename T>
__global__ __launch_bounds__(1024) void policy_loss_long_kernel(Args<T> a) {
  __shared__ float most[16];
  __shared__ double sums[16];
  __shared__ float scale[2];
  const uint64_t row = blockIdx.x, base = row * a.classes;
  const double weight = weight_of(a, row);
  if (weight == 0.0) {
    if (threadIdx.x == 0) {
      if (a.log_probs != nullptr) a.log_probs[row] = 0.0f;
      if (a.loss != nullptr) a.row_loss[row] = 0.0;
    }
    if (a.gradient != nullptr)
      for (uint64_t i = threadIdx.x; i < a.classes; i += 1024)
        a.gradient[base + i] = static_cast<T>(0.0f);
    return;
  }
  uint64_t action = 0;
  const bool valid = target_index(a.actions[row], a.classes, action);
  const float chosen = widen(a.logits[base + action]);
  float m = -INFINITY;
  double part = 0.0;
  for (uint64_t i = threadIdx.x; i < a.classes; i += 1024) {
    const float x = widen(a.logits[base + i]);
    if (x > m) {
      part *= m == -INFINITY ? 0.0 : static_cast<double>(exp_of<T>(m, x));
      m = x;
    }
    if (!(x == -INFINITY)) part += static_cast<double>(exp_of<T>(x, m));  // NaN is added
  }
  const float own = m;
  m = wave_max(m);
  if (threadIdx.x % 64 == 0) most[threadIdx.x / 64] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) m = fmaxf(m, most[i]);
  // a thread without a finite value has a sum of 0, or of NaN
  if (own != -INFINITY) part *= static_cast<double>(exp_of<T>(own, m));
  double total[1] = {m == -INFINITY ? static_cast<double>(NAN) : part};
  oxh::wave_sums_rows(total);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = total[0];
  __syncthreads();
  if (threadIdx.x < 64) {
    total[0] = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) total[0] += sums[i];
    const double away = static_cast<double>(chosen) - static_cast<double>(m);
    Row r = row_value(a, row, weight, away - log(total[0]));
    if (!valid) r = {NAN, NAN, NAN};
    if (threadIdx.x == 0) {
      if (!valid && a.error_flag != nullptr) *a.error_flag = 1u;
      if (a.log_probs != nullptr) a.log_probs[row] = static_cast<float>(r.log_prob);
      if (a.loss != nullptr) a.row_loss[row] = r.loss;
      if (a.gradient != nullptr) {
        const double slope = r.slope * static_cast<double>(*a.outer);
        scale[0] = static_cast<float>(-slope / total[0]);
        const double e = static_cast<double>(exp_of<T>(chosen, m));
        scale[1] = static_cast<float>(slope * ((total[0] - e) / total[0]));
      }
    }
  }
  if (a.gradient == nullptr) return;
  __syncthreads();
  const float off = scale[0], at_action = scale[1];
  for (uint64_t i = threadIdx.x; i < a.classes; i += 1024) {
    const float e = exp_of<T>(widen(a.logits[base + i]), m);
    a.gradient[base + i] = static_cast<T>(i == action ? at_action : e * off);
  }
}

// The sum of the rows' losses: thread t adds rows t, t + 1024, ... in order, then a fixed tree.
constexpr int kSumBlock = 1024, kSumLoads = 8;
__device__ __forceinline__ void sum_rows(double s, double *lds, uint32_t waves, float *loss) {
  double w[1] = {s};
  oxh::wave_sums_rows(w);
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = w[0];
  __syncthreads();
  if (threadIdx.x != 0) return;
  double total = 0.0;
  for (uint32_t i = 0; i < waves; ++i) total += lds[i];
  *loss = static_cast<float>(total);
}
__global__ __launch_bounds__(kSumBlock) void policy_loss_sum_kernel(const double *row_loss,
                                                                    uint64_t rows, float *loss) {
  __shared__ double lds[kSumBlock / 64];
  double s = 0.0;
  for (uint64_t base = 0; base < rows; base += kSumBlock * kSumLoads) {
    double v[kSumLoads];
#pragma unroll
    for (int i = 0; i < kSumLoads; ++i) {
      const uint64_t r = base + threadIdx.x + static_cast<uint64_t>(i) * kSumBlock;
      v[i] = r < rows ? row_loss[r] : 0.0;
    }
#pragma unroll
    for (int i = 0; i < kSumLoads; ++i) s += v[i];
  }
  sum_rows(s, lds, kSumBlock / 64, loss);
}

// Few short rows (a batch of a classifier's logits): one block, a thread per row, and the loss in
// the same launch (a quarter of the rows above 16 classes).  Float32 128 x 10: 7.9 us a call, 10.4 in
// two launches; 1024 x 10 8.8 and 10.4; 128 x 32 7.8 and 10.5, 256 x 32 10.3 and 10.5.
constexpr uint64_t kSmallRows = 1024, kSmallClasses = 32;
template <typename T, int C>
__global__ __launch_bounds__(1024) void policy_loss_small_kernel(Args<T> a) {
  __shared__ double lds[kSmallRows / 64];
  const uint64_t row = threadIdx.x;
  double row_loss = 0.0;
  if (row < a.rows) {
    const double weight = weight_of(a, row);
    const uint32_t classes = static_cast<uint32_t>(a.classes);
    const T *x = a.logits + row * a.classes;
    T *g = a.gradient == nullptr ? nullptr : a.gradient + row * a.classes;
    if (weight == 0.0) {
      if (a.log_probs != nullptr) a.log_probs[row] = 0.0f;
      if (g != nullptr)
        for (uint32_t i = 0; i < classes; ++i) g[i] = static_cast<T>(0.0f);
    } else {
      float v[C];
#pragma unroll
      for (int i = 0; i < C; ++i)
        v[i] = widen(x[static_cast<uint32_t>(i) < classes ? i : classes - 1]);
      uint64_t action = 0;
      const bool valid = target_index(a.actions[row], a.classes, action);
      const float chosen = widen(x[action]);
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < C; ++i) m = fmaxf(m, v[i]);
      double total = 0.0;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        v[i] = exp_of<T>(v[i], m);
        if (static_cast<uint32_t>(i) < classes) total += static_cast<double>(v[i]);
      }
      const double away = static_cast<double>(chosen) - static_cast<double>(m);
      Row r = row_value(a, row, weight, away - log(total));
      if (!valid) r = {NAN, NAN, NAN};
      if (!valid && a.error_flag != nullptr) *a.error_flag = 1u;
      if (a.log_probs != nullptr) a.log_probs[row] = static_cast<float>(r.log_prob);
      row_loss = r.loss;
      if (g != nullptr) {
        const double slope = r.slope * static_cast<double>(*a.outer);
        const float off = static_cast<float>(-slope / total);
        const double own = static_cast<double>(exp_of<T>(chosen, m));
        const float at_action = static_cast<float>(slope * ((total - own) / total));
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (static_cast<uint32_t>(i) < classes)
            g[i] = static_cast<T>(static_cast<uint64_t>(i) == action ? at_action : v[i] * off);
      }
    }
  }
  if (a.loss != nullptr) sum_rows(row_loss, lds, blockDim.x / 64, a.loss);
}

// 16-byte accesses of a row that a block's registers hold (1024 threads with 16 each).
constexpr uint64_t kMostPacks = 16384;

template <int Lanes, int Chunks>
struct Shape {
  static constexpr int lanes = Lanes, chunks = Chunks;
};
// Calls run(Shape<lanes, chunks>): a wave per row up to four accesses, blocks of eight waves from
// 1024 accesses on so that two share a compute unit and one's loads cover the other's sums (bfloat16
// 8192 x 32768: 223 us a call, with sixteen waves 231; float32 8192 x 16384 196 and 199, 2048 x 8192
// with four waves 25.6 for 26.3).
template <int N, typename Run>
void with_shape(uint64_t columns, Run run) {
  const uint64_t packs = (columns + N - 1) / N;
  if constexpr (N == 1) {  // rows of fewer values than an access
    run(Shape<64, 1>());
  } else {
    if (packs <= 64) return run(Shape<64, 1>());
    if (packs <= 128) return run(Shape<64, 2>());
    if (packs <= 256) return run(Shape<64, 4>());
    if (packs <= 512) return run(Shape<256, 2>());
    if (packs <= 1024) return run(Shape<256, 4>());
    if (packs <= 2048) return run(Shape<512, 4>());
    if (packs <= 4096) return run(Shape<512, 8>());
    if (packs <= 8192) return run(Shape<1024, 8>());
    run(Shape<1024, 16>());
  }
}

template <typename T>
oxh_status policy_loss(hipStream_t stream, Args<T> a) {
  if (a.classes <= kSmallClasses && a.rows <= (a.classes <= 16 ? kSmallRows : kSmallRows / 4)) {
    const dim3 block(static_cast<uint32_t>((a.rows + 63) / 64 * 64));
    if (a.classes <= 16)
      oxh::launch(policy_loss_small_kernel<T, 16>, dim3(1), block, 0, stream, a);
    else
      oxh::launch(policy_loss_small_kernel<T, 32>, dim3(1), block, 0, stream, a);
    return oxh::launched("policy_loss");
  }
  constexpr int kPack = 16 / sizeof(T);
  if (a.classes > kMostPacks * kPack) {
    oxh::launch(policy_loss_long_kernel<T>, dim3(static_cast<uint32_t>(a.rows)), dim3(1024), 0,
                stream, a);
  } else {
    oxh::row_norm::with_pack<T>(a.classes, [&](auto pack, auto ragged) {
      constexpr int N = decltype(pack)::value;
      with_shape<N>(a.classes, [&](auto shape) {
        using S = decltype(shape);
        constexpr int threads = S::lanes < 256 ? 256 : S::lanes, per = threads / S::lanes;
        oxh::launch(policy_loss_kernel<T, N, S::lanes, S::chunks, decltype(ragged)::value>,
                    dim3(static_cast<uint32_t>((a.rows + per - 1) / per)), dim3(threads), 0,
                    stream, a);
      });
    });
  }
  oxh_status st = oxh::launched("policy_loss");
  if (st != OXH_OK || a.loss == nullptr) return st;
  oxh::launch(policy_loss_sum_kernel, dim3(1), dim3(kSumBlock), 0, stream,
              static_cast<const double *>(a.row_loss), a.rows, a.loss);
  return oxh::launched("policy_loss_sum");
}

uint64_t workspace_bytes_of(uint64_t rows) { return (rows * 8 + 255) / 256 * 256; }

oxh_status check_logits(uint64_t rows, uint64_t classes) {
  OXH_REQUIRE(rows > 0 && classes > 0, OXH_INVALID_SHAPE, "policy loss: empty logits");
  // one launch numbers its threads with 32 bits
  OXH_REQUIRE(rows <= oxh::row_norm::most_blocks(1024) && classes < (1ull << 31) - 65536,
              OXH_INVALID_SHAPE, "policy loss: logits too large");
  return oxh::ok();
}

}  // namespace

extern "C" {

oxh_status oxh_policy_loss_workspace_size(uint64_t rows, uint64_t classes, uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  oxh_status st = check_logits(rows, classes);
  if (st != OXH_OK) return st;
  *bytes = workspace_bytes_of(rows);
  return oxh::ok();
}

oxh_status oxh_policy_loss(oxh_stream stream, int dtype, uint64_t rows, uint64_t classes,
                           float clip_low, float clip_high, float kl, const void *logits,
                           const float *actions, const float *old_log_probs,
                           const float *advantages, const float *reference_log_probs,
                           const float *weights, const float *outer_gradient, float *loss,
                           float *log_probs, void *gradient, uint32_t *error_flag,
                           void *workspace, uint64_t workspace_bytes) {
  using oxh::row_norm::aligned_to;
  OXH_REQUIRE(oxh::storage::valid(dtype), OXH_INVALID_SHAPE,
              "policy loss: dtype is neither OXH_F32 nor OXH_BF16");
  oxh_status st = check_logits(rows, classes);
  if (st != OXH_OK) return st;
  OXH_REQUIRE(std::isfinite(clip_low) && clip_low >= 0.0f && clip_low <= 1.0f &&
                  std::isfinite(clip_high) && clip_high >= 0.0f,
              OXH_EXECUTION, "policy loss: the clip must be finite and non-negative, its lower "
                             "part at most 1");
  OXH_REQUIRE(std::isfinite(kl) && kl >= 0.0f, OXH_EXECUTION,
              "policy loss: the KL coefficient must be non-negative and finite");
  OXH_REQUIRE(kl == 0.0f || reference_log_probs != nullptr, OXH_INVALID_SHAPE,
              "policy loss: the KL term needs the reference's log probabilities");
  OXH_REQUIRE(logits != nullptr && actions != nullptr && old_log_probs != nullptr &&
                  advantages != nullptr,
              OXH_INVALID_SHAPE, "policy loss: null pointer");
  OXH_REQUIRE(gradient == nullptr || outer_gradient != nullptr, OXH_INVALID_SHAPE,
              "policy loss: the gradient needs the upstream gradient scalar");
  const uint64_t element = oxh::storage::bytes_of(dtype), bytes = rows * classes * element;
  OXH_REQUIRE(aligned_to(logits, element) && aligned_to(gradient, element) &&
                  aligned_to(actions, 4) && aligned_to(old_log_probs, 4) &&
                  aligned_to(advantages, 4) && aligned_to(reference_log_probs, 4) &&
                  aligned_to(weights, 4) && aligned_to(outer_gradient, 4) &&
                  aligned_to(loss, 4) && aligned_to(log_probs, 4) && aligned_to(error_flag, 4),
              OXH_INVALID_SHAPE, "policy loss: a pointer is not aligned to its elements");
  uint64_t needed = 0;
  if (loss != nullptr) {
    needed = workspace_bytes_of(rows);
    OXH_REQUIRE(workspace != nullptr && workspace_bytes >= needed && oxh::aligned16(workspace),
                OXH_INVALID_SHAPE, "policy loss: workspace too small or misaligned");
  }
  struct Span {
    const void *p;
    uint64_t n;
  };
  const Span in[] = {{logits, bytes}, {actions, rows * 4}, {old_log_probs, rows * 4},
                     {advantages, rows * 4}, {reference_log_probs, rows * 4}, {weights, rows * 4},
                     {outer_gradient, 4}};
  const Span out[] = {{loss, 4}, {log_probs, rows * 4}, {gradient, bytes}, {error_flag, 4},
                      {needed != 0 ? workspace : nullptr, needed}};
  for (int o = 0; o < 5; ++o) {
    if (out[o].p == nullptr) continue;
    for (const Span &i : in)
      OXH_REQUIRE(i.p == nullptr || !oxh::any_overlap(out[o].p, out[o].n, i.p, i.n),
                  OXH_INVALID_SHAPE, "policy loss: an output or the workspace overlaps an operand");
    for (int k = 0; k < o; ++k)
      OXH_REQUIRE(out[k].p == nullptr ||
                      !oxh::any_overlap(out[o].p, out[o].n, out[k].p, out[k].n),
                  OXH_INVALID_SHAPE, "policy loss: two outputs overlap");
  }
  const float *reference = kl == 0.0f ? nullptr : reference_log_probs;
  auto args = [&](auto type) {
    using T = decltype(type);
    return Args<T>{static_cast<const T *>(logits), actions, old_log_probs, advantages, reference,
                   weights, outer_gradient, static_cast<T *>(gradient), log_probs, loss,
                   error_flag, static_cast<double *>(workspace), rows, classes, clip_low,
                   clip_high, kl};
  };
  if (dtype == OXH_F32) return policy_loss(oxh::as_stream(stream), args(float()));
  return policy_loss(oxh::as_stream(stream), args(bf16()));
}

}  // extern "C"
