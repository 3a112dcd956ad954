// delta_rule.hip -- the gated delta rule: a state S [keys, values] for each head, whose answer to a
// key each step moves towards a value.
//
//   a_t = sigmoid(gate_t);  b_t = sigmoid(write_t)
//   P = a_t S_{t-1};  S_t = P + b_t k_t (v_t - P' k_t)';  o_t = scale S_t' q_t
//
// Few steps are taken one by one, the state in a wave's registers (delta_step_kernel).  More go by
// chunks of 64.  With g_t the sum of log a from the chunk's start, G_ti = exp(g_t - g_i) and S0 the
// state before it, the errors e_t = v_t - P' k_t solve a triangular system,
//
//   A_ti = G_ti k_t.k_i (i < t);  y_t = v_t - exp(g_t) S0' k_t;  e + A (b e) = y
//   e = y - N (b y)   with   N + A b N = A
//   o = scale (exp(g) q S0 + (G o q k') (b e));  S = exp(g_64) S0 + k' (exp(g_64 - g) b e)
//
// N and G o q k' depend on no state: delta_prepare_kernel forms them for all chunks at once.
// delta_scan_kernel goes from chunk to chunk, a wave for each 16 columns of values, which never
// meet: the state stays in its registers in the layout of the matrix cores' results, which is that
// of their next operand, so that a chunk is products alone.  b is never divided by: it may be 0.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "common.h"
#include "delta_rule.h"
#include "row_norm.h"
#include "storage.h"

namespace {

using namespace oxh::delta;
using oxh::storage::widen;

template <typename T>
struct PrepareArgs {
  Dims d;
  const T *query, *key, *gate, *write;
  char *heads;  // Chunk<T> of (batch, head, chunk)
  char *keys;   // transposed keys of (batch, key head, chunk)
};

// A block per chunk and value head.
template <typename T, int KT, bool Whole>
__global__ __launch_bounds__(256) void delta_prepare_kernel(PrepareArgs<T> a) {
  using Op = operand<T>;
  __shared__ System<T, KT> m;
  const Dims &d = a.d;
  const Place at(d, blockIdx.x, blockIdx.y, blockIdx.z);
  if (at.rows == 0) return;
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T *query = a.query + at.key_row * d.keys;
  const uint64_t stride = static_cast<uint64_t>(d.key_heads) * d.keys;
  char *out = a.heads + at.head_chunk(d) * Chunk<T>::bytes;
  solve<T, KT, Whole>(
      m, d, at, a.key, a.gate, a.write, reinterpret_cast<Gates *>(out + Chunk<T>::gates), [&] {
        // G o q k', as the operand of a product from the left: a lane its step t, keys' steps i
        const uint32_t first = wave == 1 ? 0 : wave, last = wave == 1 ? 1 : wave;
        for (uint32_t ti = first; ti <= last; ++ti) {
          const uint32_t t = index_of(ti, n);
          Op q[KT];
#pragma unroll
          for (int s = 0; s < KT; ++s)
            q[s] = load_row<T, Whole>(query + min(t, at.rows - 1) * stride, 32 * s + 8 * g, d.keys);
          for (int step = 0; step <= static_cast<int>(ti >> 1); ++step) {
            f32x4 half[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              f32x4 acc = {};
#pragma unroll
              for (int s = 0; s < KT; ++s)
                acc = product(m.key_row(index_of(2 * step + e, n), s, g), q[s], acc);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const uint32_t i = 32 * step + 8 * g + 4 * e + r;
                half[e][r] = i <= t ? acc[r] * m.between(t, i) * d.scale : 0.0f;
              }
            }
            Op *to = reinterpret_cast<Op *>(out + Chunk<T>::within);
            to[lower_place(ti, step) * 64 + lane] = rounded<T>(join(half[0], half[1]));
          }
        }
      });
  for (int p = wave; p < kTriangle; p += 4) {
    const int ti = p < 2 ? p : 2 + (p - 2) / 2, step = p < 2 ? 0 : (p - 2) % 2;
    const float *row = &m.mat[index_of(ti, n)][32 * step + 8 * g];
    f32x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = row[i];
    const Split<T, Chunk<T>::kParts> parts(v);
    Op *to = reinterpret_cast<Op *>(out + Chunk<T>::system);
#pragma unroll
    for (int q = 0; q < Chunk<T>::kParts; ++q)
      to[(p * Chunk<T>::kParts + q) * 64 + lane] = parts.part[q];
  }
  if (at.head % d.group == 0)
    store_transposed<T, KT>(m.tile, reinterpret_cast<Op *>(a.keys) + at.key_chunk(d) * (4 * KT * 64));
}

template <typename T>
struct ScanArgs {
  Dims d;
  const T *query, *key, *value;
  const char *heads, *keys;
  const float *from;  // states before the first chunk, null: 0
  float *to;          // and after the last, may be null
  T *out;
  char *saved;        // what the backward reads, may be null
  uint32_t all;       // chunks of the whole sequence
};

// A wave per 16 columns of a head's values.
template <typename T, int KT, bool Whole>
__global__ __launch_bounds__(256) void delta_scan_kernel(ScanArgs<T> a) {
  using Op = operand<T>;
  constexpr int P = Chunk<T>::kParts;
  const Dims &d = a.d;
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t slab = blockIdx.x * (blockDim.x >> 6) +
                        __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (slab >= d.slabs) return;
  const uint32_t h = blockIdx.y, b = blockIdx.z, kh = h / d.group;
  const uint32_t column = 16 * slab + n;
  const bool in = column < d.values;
  const uint32_t col = in ? column : d.values - 1;
  const uint32_t length = length_of(d, b);
  const uint64_t head = static_cast<uint64_t>(b) * d.heads + h;
  const uint64_t stride = static_cast<uint64_t>(d.key_heads) * d.keys;
  const uint64_t value_stride = static_cast<uint64_t>(d.heads) * d.values;

  f32x4 state[2 * KT];
  const uint64_t state_at = head * d.keys * d.values + col;
#pragma unroll
  for (int i = 0; i < 2 * KT; ++i) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t k = index_of(i, 4 * g + r);
      state[i][r] = a.from != nullptr && (Whole || k < d.keys)
                        ? a.from[state_at + static_cast<uint64_t>(k) * d.values]
                        : 0.0f;
    }
  }

  for (uint32_t chunk = 0; chunk < d.chunks; ++chunk) {
    const uint32_t begin = (d.first + chunk) * kChunk;
    const uint64_t row0 = static_cast<uint64_t>(b) * d.time + begin;
    T *out = a.out + row0 * value_stride + static_cast<uint64_t>(h) * d.values + col;
    const uint32_t held = min(d.time - begin, static_cast<uint32_t>(kChunk));
    if (begin >= length) {
      if (in)
        for (uint32_t t = g; t < held; t += 4) out[t * value_stride] = static_cast<T>(0.0f);
      continue;
    }
    const uint32_t rows = min(length - begin, static_cast<uint32_t>(kChunk));
    const T *key = a.key + row0 * stride + static_cast<uint64_t>(kh) * d.keys;
    const T *query = a.query + row0 * stride + static_cast<uint64_t>(kh) * d.keys;
    const T *value = a.value + row0 * value_stride + static_cast<uint64_t>(h) * d.values + col;
    const char *operands = a.heads + (head * d.chunks + chunk) * Chunk<T>::bytes;
    const Gates *gates = reinterpret_cast<const Gates *>(operands + Chunk<T>::gates);
    const Op *system = reinterpret_cast<const Op *>(operands + Chunk<T>::system) + lane;
    const Op *within = reinterpret_cast<const Op *>(operands + Chunk<T>::within) + lane;
    const Op *keys = reinterpret_cast<const Op *>(a.keys) + lane +
                     ((static_cast<uint64_t>(b) * d.key_heads + kh) * d.chunks + chunk) *
                         (4 * KT * 64);
    auto vec = [&](const float *v, int tile) {
      return *reinterpret_cast<const f32x4 *>(v + 32 * (tile >> 1) + 8 * g + 4 * (tile & 1));
    };

    f32x4 y[4], q[4];
    Op state_high[KT];
    {
      // the state as an operand, and its products with keys and queries
      f32x4 held_by[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = f32x4{};
#pragma unroll
      for (int s = 0; s < KT; ++s) {
        const Split<T, P> st(join(state[2 * s], state[2 * s + 1]));
        state_high[s] = st.part[0];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint64_t row = min(index_of(i, n), rows - 1) * stride;
          held_by[i] =
              product<T, P>(load_row<T, Whole>(key + row, 32 * s + 8 * g, d.keys), st, held_by[i]);
          q[i] = product(load_row<T, Whole>(query + row, 32 * s + 8 * g, d.keys), st.part[0], q[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 since = vec(gates->since, i);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t t = min(index_of(i, 4 * g + r), rows - 1);
          y[i][r] = widen(value[t * value_stride]) - since[r] * held_by[i][r];
        }
        q[i] *= since * d.scale;
      }
    }
    if (a.saved != nullptr) {
      Op *to = reinterpret_cast<Op *>(a.saved) +
               ((head * a.all + d.first + chunk) * d.slabs + slab) * ((KT + 2) * 64) + lane;
#pragma unroll
      for (int s = 0; s < KT; ++s) to[s * 64] = state_high[s];
    }
    // e = y - N (b y)
    f32x4 e[4];
    {
      f32x4 weighted[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        weighted[i] = -vec(gates->write, i) * y[i];
        e[i] = y[i];
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Split<T, P> w(join(weighted[2 * s], weighted[2 * s + 1]));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((i >> 1) < s) continue;
          const Op *from = system + lower_place(i, s) * P * 64;
          if constexpr (P == 2) e[i] = product(from[64], w.part[0], e[i]);
          e[i] = product<T, P>(from[0], w, e[i]);
        }
      }
    }
    if (a.saved != nullptr) {
      Op *to = reinterpret_cast<Op *>(a.saved) +
               ((head * a.all + d.first + chunk) * d.slabs + slab) * ((KT + 2) * 64) + lane;
#pragma unroll
      for (int s = 0; s < 2; ++s) to[(KT + s) * 64] = rounded<T>(join(e[2 * s], e[2 * s + 1]));
    }
    // o = exp(g) q S0 + (G o q k') (b e);  S = exp(g_64) S0 + k' (exp(g_64 - g) b e)
    const float whole = gates->since[kChunk - 1];
#pragma unroll
    for (int i = 0; i < 2 * KT; ++i) state[i] *= whole;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x4 u[2], left[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u[i] = vec(gates->write, 2 * s + i) * e[2 * s + i];
        left[i] = vec(gates->until, 2 * s + i) * u[i];
      }
      const Split<T, P> wrote(join(u[0], u[1]));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((i >> 1) >= s) q[i] = product<T, P>(within[lower_place(i, s) * 64], wrote, q[i]);
      const Split<T, P> l(join(left[0], left[1]));
#pragma unroll
      for (int i = 0; i < 2 * KT; ++i)
        state[i] = product<T, P>(keys[(2 * i + s) * 64], l, state[i]);
    }
    if (in) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t t = index_of(i, 4 * g + r);
          if (t < held) out[t * value_stride] = static_cast<T>(t < rows ? q[i][r] : 0.0f);
        }
      }
    }
  }
  if (a.to == nullptr || !in) return;
#pragma unroll
  for (int i = 0; i < 2 * KT; ++i) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t k = index_of(i, 4 * g + r);
      if (Whole || k < d.keys) a.to[state_at + static_cast<uint64_t>(k) * d.values] = state[i][r];
    }
  }
}

template <typename T>
struct StepArgs {
  Dims d;
  const T *query, *key, *value, *gate, *write;
  const float *from;
  float *to;
  T *out;
};

// A wave per 32 columns of a head's values: a lane R consecutive keys of 4 columns, kept in
// registers from step to step.
template <typename T, int R, bool Whole>
__global__ __launch_bounds__(256) void delta_step_kernel(StepArgs<T> a) {
  const Dims &d = a.d;
  const uint32_t lane = threadIdx.x & 63, part = lane >> 3;
  const uint32_t tiles = (d.values + 31) / 32;
  const uint64_t id = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const uint32_t tile = static_cast<uint32_t>(id % tiles);
  const uint64_t head = id / tiles;
  if (head >= static_cast<uint64_t>(d.batch) * d.heads) return;
  const uint32_t b = static_cast<uint32_t>(head / d.heads), h = static_cast<uint32_t>(head % d.heads);
  const uint32_t kh = h / d.group, column = tile * 32 + (lane & 7) * 4;
  const uint32_t length = length_of(d, b);
  const uint32_t first = part * R;  // its keys
  float s[R][4];
  const uint64_t state_at = head * d.keys * d.values + column;
  // a lane's columns: all four of them, or those below the values' end
  const bool four = column + 4 <= d.values;
#pragma unroll
  for (int j = 0; j < R; ++j) {
#pragma unroll
    for (int c = 0; c < 4; ++c) s[j][c] = 0.0f;
    if (a.from == nullptr || !(Whole || first + j < d.keys)) continue;
    const float *p = a.from + state_at + static_cast<uint64_t>(first + j) * d.values;
    if (four) {
      oxh::storage::load<float, 4>(p, s[j]);
    } else {
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c)
        if (column + c < d.values) s[j][c] = p[c];
    }
  }
  for (uint32_t t = 0; t < d.time; ++t) {
    const uint64_t row = static_cast<uint64_t>(b) * d.time + t;
    T *out = a.out + (row * d.heads + h) * d.values + column;
    if (t >= length) {
      if (part == 0)
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c)
          if (column + c < d.values) out[c] = static_cast<T>(0.0f);
      continue;
    }
    const uint64_t key_at = (row * d.key_heads + kh) * d.keys + first;
    float k[R], q[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool held = Whole || first + j < d.keys;
      k[j] = held ? widen(a.key[key_at + j]) : 0.0f;
      q[j] = held ? widen(a.query[key_at + j]) : 0.0f;
    }
    const float decay = sigmoid(widen(a.gate[row * d.heads + h]));
    const float beta = sigmoid(widen(a.write[row * d.heads + h]));
    const T *value = a.value + (row * d.heads + h) * d.values + column;
    float v[4], dot[4];
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c) {
      v[c] = column + c < d.values ? widen(value[c]) : 0.0f;
      dot[c] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[j][c] *= decay;
        dot[c] = fmaf(k[j], s[j][c], dot[c]);
      }
#pragma unroll
    for (int m = 8; m < 64; m *= 2)
#pragma unroll
      for (int c = 0; c < 4; ++c) dot[c] += __shfl_xor(dot[c], m);
    float o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v[c] = beta * (v[c] - dot[c]);
      o[c] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[j][c] = fmaf(k[j], v[c], s[j][c]);
        o[c] = fmaf(q[j], s[j][c], o[c]);
      }
#pragma unroll
    for (int m = 8; m < 64; m *= 2)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] += __shfl_xor(o[c], m);
    if (part == 0) {
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c)
        if (column + c < d.values) out[c] = static_cast<T>(o[c] * d.scale);
    }
  }
  if (a.to == nullptr) return;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    if (!(Whole || first + j < d.keys)) continue;
    float *p = a.to + state_at + static_cast<uint64_t>(first + j) * d.values;
    if (four) {
      oxh::storage::store<float, 4>(p, s[j]);
    } else {
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c)
        if (column + c < d.values) p[c] = s[j][c];
    }
  }
}

// ------------------------------------------------------------------------------------ host side

// Steps taken one by one where no backward is to follow.
constexpr uint64_t kStepLimit = 16;

template <typename T>
struct ForwardPlan {
  Plan p;
  uint64_t head_bytes, key_bytes, state_bytes;  // of the workspace
  uint64_t bytes() const { return head_bytes + key_bytes + state_bytes; }
  ForwardPlan(const oxh_delta_shape &s, float scale, const int32_t *lengths)
      : p(s, scale, lengths) {
    const uint64_t head = s.batch * s.heads * Chunk<T>::bytes;
    const uint64_t key = s.batch * s.key_heads * p.steps * 4 * Chunk<T>::operand_bytes;
    p.segment = std::min(p.all, std::max<uint64_t>(1, kPrepared / std::max<uint64_t>(1, head + key)));
    head_bytes = round_up(p.segment * head, 256);
    key_bytes = round_up(p.segment * key, 256);
    state_bytes = p.segment < p.all ? round_up(p.state_elements(s) * 4, 256) : 0;
  }
};

template <typename T>
oxh_status by_steps(hipStream_t stream, const StepArgs<T> &a) {
  const uint64_t waves = static_cast<uint64_t>(a.d.batch) * a.d.heads * ((a.d.values + 31) / 32);
  const dim3 blocks(static_cast<uint32_t>((waves + 3) / 4));
  auto rows = [&](auto r) {
    constexpr int R = decltype(r)::value;
    if (a.d.keys == 8 * R)
      oxh::launch(delta_step_kernel<T, R, true>, blocks, dim3(256), 0, stream, a);
    else
      oxh::launch(delta_step_kernel<T, R, false>, blocks, dim3(256), 0, stream, a);
  };
  if (a.d.keys <= 32) rows(std::integral_constant<int, 4>());
  else if (a.d.keys <= 64) rows(std::integral_constant<int, 8>());
  else rows(std::integral_constant<int, 16>());
  return oxh::launched("gated_delta_rule_steps");
}

template <typename T>
oxh_status by_chunks(hipStream_t stream, const ForwardPlan<T> &plan, const T *query, const T *key, const T *value,
                     const T *gate, const T *write, const float *initial, T *out, float *final,
                     char *saved, char *workspace) {
  const Plan &p = plan.p;
  char *heads = workspace, *keys = heads + plan.head_bytes;
  float *between = reinterpret_cast<float *>(keys + plan.key_bytes);
  for (uint64_t first = 0; first < p.all; first += p.segment) {
    Dims d = p.d;
    d.first = static_cast<uint32_t>(first);
    d.chunks = static_cast<uint32_t>(std::min(p.segment, p.all - first));
    const bool last = first + p.segment >= p.all;
    const PrepareArgs<T> prepare{d, query, key, gate, write, heads, keys};
    const ScanArgs<T> scan{d, query, key, value, heads, keys, first == 0 ? initial : between,
                           last ? final : between, out, saved, static_cast<uint32_t>(p.all)};
    with_keys(d.keys, [&](auto steps, auto whole) {
      constexpr int KT = decltype(steps)::value;
      constexpr bool W = decltype(whole)::value;
      oxh::launch(delta_prepare_kernel<T, KT, W>, dim3(d.chunks, d.heads, d.batch), dim3(256), 0,
                  stream, prepare);
      oxh::launch(delta_scan_kernel<T, KT, W>, dim3(d.slabs, d.heads, d.batch), dim3(64), 0,
                  stream, scan);
    });
    oxh_status st = oxh::launched("gated_delta_rule");
    if (st != OXH_OK) return st;
  }
  return oxh::ok();
}

bool by_steps_alone(const oxh_delta_shape &s, bool saves) {
  return s.time == 0 || (!saves && s.time <= kStepLimit);
}

template <typename T>
uint64_t saved_bytes(const oxh_delta_shape &s) {
  const uint64_t steps = round_up(s.key_dim, 32) / 32;
  return s.batch * s.heads * ((s.time + kChunk - 1) / kChunk) * ((s.value_dim + 15) / 16) *
         (steps + 2) * Chunk<T>::operand_bytes;
}

}  // namespace

extern "C" {

oxh_status oxh_gated_delta_rule_saved_size(int dtype, const oxh_delta_shape *shape,
                                           uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  oxh_status st = check_shape(dtype, shape);
  if (st != OXH_OK) return st;
  *bytes = dtype == OXH_F32 ? saved_bytes<float>(*shape) : saved_bytes<bf16>(*shape);
  return oxh::ok();
}

oxh_status oxh_gated_delta_rule_workspace_size(int dtype, const oxh_delta_shape *shape, int saves,
                                               uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  oxh_status st = check_shape(dtype, shape);
  if (st != OXH_OK) return st;
  *bytes = 0;
  if (by_steps_alone(*shape, saves != 0)) return oxh::ok();
  *bytes = dtype == OXH_F32 ? ForwardPlan<float>(*shape, 1.0f, nullptr).bytes()
                            : ForwardPlan<bf16>(*shape, 1.0f, nullptr).bytes();
  return oxh::ok();
}

oxh_status oxh_gated_delta_rule_forward(oxh_stream stream, int dtype, const oxh_delta_shape *shape,
                                        float scale, const void *query, const void *key,
                                        const void *value, const void *gate, const void *write,
                                        const float *initial_state, const int32_t *lengths,
                                        void *output, float *final_state, void *saved,
                                        uint64_t saved_size, void *workspace,
                                        uint64_t workspace_bytes) {
  oxh_status st = check_shape(dtype, shape);
  if (st != OXH_OK) return st;
  const oxh_delta_shape &s = *shape;
  OXH_REQUIRE(std::isfinite(scale), OXH_EXECUTION, "gated delta rule: scale must be finite");
  if (s.batch == 0) return oxh::ok();
  const Sizes z(dtype, s);
  std::vector<Span> in = {{query, z.query, z.element}, {key, z.query, z.element},
                          {value, z.value, z.element}, {gate, z.gate, z.element},
                          {write, z.gate, z.element}};
  std::vector<Span> out = {{output, z.value, z.element}};
  for (const auto *list : {&in, &out})
    for (const Span &x : *list)
      OXH_REQUIRE(x.p != nullptr || x.bytes == 0, OXH_INVALID_SHAPE,
                  "gated delta rule: null pointer");
  in.push_back({lengths, s.batch * 4, 4});
  out.push_back({final_state, z.state, 4});
  const bool steps = by_steps_alone(s, saved != nullptr);
  uint64_t needed = 0;
  if (!steps) {
    st = oxh_gated_delta_rule_workspace_size(dtype, shape, saved != nullptr, &needed);
    if (st != OXH_OK) return st;
    OXH_REQUIRE(workspace != nullptr && workspace_bytes >= needed && oxh::aligned16(workspace),
                OXH_INVALID_SHAPE, "gated delta rule: workspace too small or misaligned");
    out.push_back({workspace, needed, 16});
    if (saved != nullptr) {
      uint64_t kept = 0;
      st = oxh_gated_delta_rule_saved_size(dtype, shape, &kept);
      if (st != OXH_OK) return st;
      OXH_REQUIRE(saved_size >= kept && oxh::aligned16(saved), OXH_INVALID_SHAPE,
                  "gated delta rule: saved is too small or misaligned");
      out.push_back({saved, kept, 16});
    }
  }
  st = check_apart(in, out);
  if (st != OXH_OK) return st;
  // the final state may be written over the initial one
  if (initial_state != nullptr) {
    const Span initial{initial_state, z.state, 4};
    OXH_REQUIRE(oxh::row_norm::aligned_to(initial_state, 4), OXH_INVALID_SHAPE,
                "gated delta rule: a pointer is not aligned to its elements");
    for (const Span &o : out)
      OXH_REQUIRE(o.p == nullptr || (o.p == final_state && initial.p == o.p) ||
                      !oxh::any_overlap(o.p, o.bytes, initial.p, initial.bytes),
                  OXH_INVALID_SHAPE, "gated delta rule: an output overlaps an operand");
  }
  auto run = [&](auto type) {
    using T = decltype(type);
    hipStream_t on = oxh::as_stream(stream);
    const ForwardPlan<T> plan(s, scale, lengths);
    if (steps) {
      const StepArgs<T> a{plan.p.d, static_cast<const T *>(query), static_cast<const T *>(key),
                          static_cast<const T *>(value), static_cast<const T *>(gate),
                          static_cast<const T *>(write), initial_state, final_state,
                          static_cast<T *>(output)};
      return by_steps(on, a);
    }
    return by_chunks<T>(on, plan, static_cast<const T *>(query), static_cast<const T *>(key),
                        static_cast<const T *>(value), static_cast<const T *>(gate),
                        static_cast<const T *>(write), initial_state, static_cast<T *>(output),
                        final_state, static_cast<char *>(saved), static_cast<char *>(workspace));
  };
  return dtype == OXH_F32 ? run(float()) : run(bf16());
}

}  // extern "C"
