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
#include <cstddef>
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
  char *keys;   // operands of keys, queries and transposed keys of (batch, key head, chunk)
};

// A block per chunk and value head.
template <typename T, int P, int KT, bool Whole>
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
  char *out = a.heads + at.head_chunk(d) * Chunk<T, P>::bytes;
  const bool first_head = at.head % d.group == 0;  // brings what its key head's others share
  Op *keys = reinterpret_cast<Op *>(a.keys) + at.key_chunk(d) * (12 * KT * 64) + lane;
  Op *queries = keys + 4 * KT * 64, *across = queries + 4 * KT * 64;
  solve<T, KT, Whole>(
      m, d, at, a.key, a.gate, a.write, reinterpret_cast<Gates *>(out + Chunk<T, P>::gates), [&] {
        // G o q k', as the operand of a product from the left: a lane its step t, keys' steps i
        const uint32_t first = wave == 1 ? 0 : wave, last = wave == 1 ? 1 : wave;
        for (uint32_t ti = first; ti <= last; ++ti) {
          const uint32_t t = index_of(ti, n);
          Op q[KT];
#pragma unroll
          for (int s = 0; s < KT; ++s)
            q[s] = load_row<T, Whole>(query + min(t, at.rows - 1) * stride, 32 * s + 8 * g, d.keys);
          if (first_head)
#pragma unroll
            for (int s = 0; s < KT; ++s) queries[(ti * KT + s) * 64] = q[s];
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
            Op *to = reinterpret_cast<Op *>(out + Chunk<T, P>::within);
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
    const Split<T, P> parts(v);
    Op *to = reinterpret_cast<Op *>(out + Chunk<T, P>::system);
#pragma unroll
    for (int q = 0; q < P; ++q)
      to[(p * P + q) * 64 + lane] = parts.part[q];
  }
  if (!first_head) return;
#pragma unroll
  for (int s = 0; s < KT; ++s)
    keys[(wave * KT + s) * 64] = m.key_row(index_of(wave, n), s, g);
  store_transposed<T, KT>(m.tile, across - lane);
}

template <typename T>
struct ScanArgs {
  Dims d;
  const T *value;
  const char *heads, *keys;
  const float *from;  // states before the first chunk, null: 0
  float *to;          // and after the last, may be null
  T *out;
  char *saved;        // what the backward reads, may be null
  uint32_t all;       // chunks of the whole sequence
};

// What the block's waves hand each other, as operands: the state, b y, b e, exp(g_64 - g) b e, and e
// for the backward.
template <typename T, int P, int KT, int C>
struct Exchange {
  operand<T> state[KT][C][P][64], weighted[2][C][P][64], wrote[2][C][P][64], left[2][C][P][64],
      error[2][C][64];
};

// A block of four waves per C slabs of 16 columns of a head's values.  A wave takes 16 of a chunk's
// steps and 32 of the keys: whatever stands on the left of a product (keys, queries, the chunk's
// matrices) is one wave's alone and goes from memory to its registers, a chunk ahead, as soon as the
// present chunk's is used; what stands on the right goes through shared memory, three times a
// chunk.
template <typename T, int P, int KT, int C>
__global__ __launch_bounds__(256) void delta_scan_kernel(ScanArgs<T> a) {
  using Op = operand<T>;
  using Kept = Chunk<T, P>;
  __shared__ Exchange<T, P, KT, C> m;
  const Dims &d = a.d;
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = w & 1;
  const int pair = w >> 1;  // of tiles of 16 steps: an operand of 32
  // blocks of a head share what they read: on one XCD
  const oxh::BlockTile block = oxh::xcd_block();
  const uint32_t h = block.y, b = block.z, kh = h / d.group;
  const uint32_t length = length_of(d, b), start = d.first * kChunk;
  const uint32_t live =
      length <= start ? 0 : min((length - start + kChunk - 1) / kChunk, d.chunks);
  const uint64_t head = static_cast<uint64_t>(b) * d.heads + h;
  const uint64_t value_stride = static_cast<uint64_t>(d.heads) * d.values;
  const uint64_t row0 = static_cast<uint64_t>(b) * d.time + start;
  const T *values = a.value + row0 * value_stride + static_cast<uint64_t>(h) * d.values;
  T *outs = a.out + row0 * value_stride + static_cast<uint64_t>(h) * d.values;
  const char *chunks = a.heads + head * d.chunks * Kept::bytes;
  constexpr uint32_t kOperand = 64 * sizeof(Op), kKeys = 4 * KT * kOperand;
  const char *keys =
      a.keys + (static_cast<uint64_t>(b) * d.key_heads + kh) * d.chunks * (3 * kKeys);
  uint32_t cols[C];  // this lane's; those past the last are the last again, and not stored
  bool in[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t column = 16 * (block.x * C + c) + n;
    in[c] = column < d.values;
    cols[c] = in[c] ? column : d.values - 1;
  }
  auto rows_of = [&](uint32_t chunk) -> uint32_t {
    return min(length - start - chunk * kChunk, static_cast<uint32_t>(kChunk));
  };
  const bool holds = w < KT;  // keys 32 w on
  const uint64_t state_at = head * d.keys * d.values;
  auto key_at = [&](int tile, int r) { return 32 * w + index_of(tile, 4 * g + r); };
  f32x4 state[2][C];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      state[i][c] = f32x4{};
      if (a.from == nullptr || !holds) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t k = key_at(i, r), there = min(k, d.keys - 1);
        const float v = a.from[state_at + static_cast<uint64_t>(there) * d.values + cols[c]];
        state[i][c][r] = k < d.keys ? v : 0.0f;
      }
    }

  // The left operands of a chunk's four products and its values, each loaded where the chunk before
  // has used its own (not before: their registers are the same).  No load or store of the loop is behind a branch, so that each use waits for
  // its own loads alone: the last chunk loads itself again, and stores that are not to be go past
  // their buffer's end.
  Op key[KT], query[KT], solve[2][P], scores[2], back[2][2];
  T value[C][4];
  f32x4 since, until, write;
  float whole = 0.0f;
  const uint32_t value_bytes = static_cast<uint32_t>(value_stride * sizeof(T));
  const uint32_t lane_at = lane * sizeof(Op);
  auto load_keys = [&](uint32_t chunk) {
    const char *from = keys + (chunk * uint64_t{3 * kKeys} + w * (KT * kOperand));
#pragma unroll
    for (int s = 0; s < KT; ++s) key[s] = load_at<Op>(from + s * kOperand, lane_at);
#pragma unroll
    for (int s = 0; s < KT; ++s) query[s] = load_at<Op>(from + kKeys + s * kOperand, lane_at);
  };
  auto load_values = [&](uint32_t chunk) {
    const uint32_t last = rows_of(chunk) - 1;
    const char *from = reinterpret_cast<const char *>(values + chunk * kChunk * value_stride);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t row = min(index_of(w, 4 * g + r), last) * value_bytes;
#pragma unroll
      for (int c = 0; c < C; ++c)
        value[c][r] = load_at<T>(from, row + cols[c] * static_cast<uint32_t>(sizeof(T)));
    }
  };
  auto operands_of = [&](uint32_t chunk, uint64_t part) {
    return chunks + (chunk * Kept::bytes + part);
  };
  auto load_system = [&](uint32_t chunk) {
    const char *from = operands_of(chunk, Kept::system);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int p = 0; p < P; ++p)
        solve[s][p] =
            load_at<Op>(from + (lower_place(w, min(s, pair)) * P + p) * kOperand, lane_at);
  };
  auto load_rest = [&](uint32_t chunk) {
    whole = load_at<float>(operands_of(chunk, Kept::gates) + offsetof(Gates, since),
                           (kChunk - 1) * 4);
    const char *from = operands_of(chunk, Kept::within);
#pragma unroll
    for (int s = 0; s < 2; ++s)
      scores[s] = load_at<Op>(from + lower_place(w, min(s, pair)) * kOperand, lane_at);
    const char *k = keys + (chunk * uint64_t{3 * kKeys} + 2 * kKeys + 4 * min(w, KT - 1u) * kOperand);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        back[i][s] = load_at<Op>(k + (2 * i + s) * kOperand, lane_at);
  };
  auto load_gates = [&](uint32_t chunk) {
    const char *gates = operands_of(chunk, Kept::gates);
    const uint32_t at = index_of(w, 4 * g) * 4;
    since = load_at<f32x4>(gates + offsetof(Gates, since), at);
    until = load_at<f32x4>(gates + offsetof(Gates, until), at);
    write = load_at<f32x4>(gates + offsetof(Gates, write), at);
  };
  typedef T quarter __attribute__((ext_vector_type(4)));
  // a wave's half of an operand that two waves form, and the state's, which is its own
  auto hand = [&](Op(&to)[P][64], f32x4 v) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const quarter q = __builtin_convertvector(v, quarter);
      reinterpret_cast<quarter *>(&to[p][lane])[half] = q;
      if (p + 1 < P) v -= __builtin_convertvector(q, f32x4);
    }
  };
  // what the backward reads of a chunk; a block of one slab brings its half of the pair's lanes
  const uint32_t kept = (d.slabs + 1) / 2 * (2 * KT + 4) * kOperand;
  auto saved_of = [&](uint32_t chunk) {
    return buffer_of(a.saved + ((head * a.all + d.first + chunk) * kept), a.saved == nullptr ? 0 : kept);
  };
  const bool brings = C == 2 || (g >> 1) == (block.x & 1);
  auto saved_at = [&](int place) {
    return brings ? (block.x * C / 2 * (2 * KT + 4) + place) * kOperand + lane_at : kNowhere;
  };
  auto hand_state = [&](uint32_t chunk) {
    if (KT < 4 && !holds) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const Split<T, P> st(join(state[0][c], state[1][c]));
#pragma unroll
      for (int p = 0; p < P; ++p) m.state[w][c][p][lane] = st.part[p];
    }
    if (a.saved == nullptr) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      store_to(saved_of(chunk), saved_at(2 * w + i),
               turned(&m.state[w][0][0][0], C == 2 ? P * 64 : 0, i, n, g));
  };
  // right operands of 64 steps, all of them on their way before the first is used
  auto read_pairs = [&](Op(&to)[2][C][P], const Op(&from)[2][C][P][64]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int p = 0; p < P; ++p) to[s][c][p] = from[s][c][p][lane];
    __builtin_amdgcn_sched_barrier(0);
  };
  if (live != 0) {
    load_keys(0);
    load_values(0);
    load_gates(0);
    load_system(0);
    load_rest(0);
    hand_state(0);
  }
  for (uint32_t chunk = 0; chunk < live; ++chunk) {
    const uint32_t next = min(chunk + 1, live - 1);
    lds_barrier();
    f32x4 y[C] = {}, o[C] = {};
    {
      Op right[KT][C][P];
#pragma unroll
      for (int s = 0; s < KT; ++s)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int p = 0; p < P; ++p) right[s][c][p] = m.state[s][c][p][lane];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < KT; ++s) {
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int c = 0; c < C; ++c) y[c] = product(key[s], right[s][c][p], y[c]);
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = product(query[s], right[s][c][0], o[c]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_keys(next);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = widen(value[c][r]);
      y[c] = v - since * y[c];
      o[c] *= since * d.scale;
      hand(m.weighted[pair][c], -write * y[c]);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_values(next);
    lds_barrier();
    // e = y - N (b y)
    {
      Op right[2][C][P];
      read_pairs(right, m.weighted);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (s > pair) continue;
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int q = P - 1 - p; q >= 0; --q)
#pragma unroll
            for (int c = 0; c < C; ++c) y[c] = product(solve[s][p], right[s][c][q], y[c]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_system(next);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (a.saved != nullptr)
        reinterpret_cast<quarter *>(&m.error[pair][c][lane])[half] =
            __builtin_convertvector(y[c], quarter);
      y[c] *= write;
      hand(m.wrote[pair][c], y[c]);
      hand(m.left[pair][c], until * y[c]);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_gates(next);
    lds_barrier();
    // o = exp(g) q S0 + (G o q k') (b e);  S = exp(g_64) S0 + k' (exp(g_64 - g) b e)
    Op left[2][C][P], wrote[2][C][P];
    read_pairs(left, m.left);
    read_pairs(wrote, m.wrote);
    if (KT == 4 || holds) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) state[i][c] *= whole;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) state[i][c] = product(back[i][s], left[s][c][p], state[i][c]);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s > pair) continue;
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = product(scores[s], wrote[s][c][p], o[c]);
    }
    if (a.saved != nullptr)
      store_to(saved_of(chunk), saved_at(2 * KT + w),
               turned(&m.error[pair][0][0], C == 2 ? 64 : 0, half, n, g));
    __builtin_amdgcn_sched_barrier(0);
    load_rest(next);
    const uint32_t rows = rows_of(chunk);
    const auto to = buffer_of(outs + chunk * kChunk * value_stride, kChunk * value_bytes);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t t = index_of(w, 4 * g + r);
#pragma unroll
      for (int c = 0; c < C; ++c)
        store_to(to, t < rows && in[c]
                         ? t * value_bytes + cols[c] * static_cast<uint32_t>(sizeof(T))
                         : kNowhere,
                 static_cast<T>(o[c][r]));
    }
    if (chunk + 1 < live) hand_state(chunk + 1);
  }
  // steps past the row's end
  const uint32_t end = min(d.time - start, d.chunks * kChunk);
  for (uint32_t t = (length <= start ? 0 : length - start) + 4 * w + g; t < end; t += 16) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (in[c]) outs[t * value_stride + cols[c]] = static_cast<T>(0.0f);
  }
  if (a.to == nullptr || !holds) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t k = key_at(i, r);
      if (k >= d.keys) continue;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (in[c]) a.to[state_at + static_cast<uint64_t>(k) * d.values + cols[c]] = state[i][c][r];
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

template <typename T, int P>
struct ForwardPlan {
  Plan p;
  uint64_t head_bytes, key_bytes, state_bytes;  // of the workspace
  uint64_t bytes() const { return head_bytes + key_bytes + state_bytes; }
  ForwardPlan(const oxh_delta_shape &s, float scale, const int32_t *lengths)
      : p(s, scale, lengths) {
    const uint64_t head = s.batch * s.heads * Chunk<T, P>::bytes;
    const uint64_t key = s.batch * s.key_heads * p.steps * 12 * kOperandBytes<T>;
    p.divide(head + key);
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

template <typename T, int P>
oxh_status by_chunks(hipStream_t stream, const ForwardPlan<T, P> &plan, const T *query, const T *key, const T *value,
                     const T *gate, const T *write, const float *initial, T *out, float *final,
                     char *saved, char *workspace) {
  const Plan &p = plan.p;
  char *heads = workspace, *keys = heads + plan.head_bytes;
  float *between = reinterpret_cast<float *>(keys + plan.key_bytes);
  // slabs of a block: as many as leave a block for each compute unit
  const uint64_t all_heads = static_cast<uint64_t>(p.d.batch) * p.d.heads;
  const uint32_t pairs = (p.d.slabs + 1) / 2;
  const bool two = all_heads * pairs >= oxh::kComputeUnits;
  for (uint64_t first = 0; first < p.all; first += p.segment) {
    Dims d = p.d;
    d.first = static_cast<uint32_t>(first);
    d.chunks = static_cast<uint32_t>(std::min(p.segment, p.all - first));
    const bool last = first + p.segment >= p.all;
    const PrepareArgs<T> prepare{d, query, key, gate, write, heads, keys};
    const ScanArgs<T> scan{d, value, heads, keys, first == 0 ? initial : between,
                           last ? final : between, out, saved, static_cast<uint32_t>(p.all)};
    with_keys(d.keys, d.keys % 32 == 0, [&](auto steps, auto whole) {
      constexpr int KT = decltype(steps)::value;
      constexpr bool W = decltype(whole)::value;
      oxh::launch(delta_prepare_kernel<T, P, KT, W>, dim3(d.chunks, d.heads, d.batch), dim3(256), 0,
                  stream, prepare);
      if (two)
        oxh::launch(delta_scan_kernel<T, P, KT, 2>, dim3(pairs, d.heads, d.batch), dim3(256), 0,
                    stream, scan);
      else
        oxh::launch(delta_scan_kernel<T, P, KT, 1>, dim3(2 * pairs, d.heads, d.batch), dim3(256), 0,
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
  return s.batch * s.heads * ((s.time + kChunk - 1) / kChunk) * pairs_of(s.value_dim) *
         (2 * steps + 4) * kOperandBytes<T>;
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
  *bytes = dtype == OXH_F32 ? ForwardPlan<float, 1>(*shape, 1.0f, nullptr).bytes()
                            : ForwardPlan<bf16, 2>(*shape, 1.0f, nullptr).bytes();
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
    if (steps) {
      const StepArgs<T> a{Plan(s, scale, lengths).d, static_cast<const T *>(query),
                          static_cast<const T *>(key), static_cast<const T *>(value),
                          static_cast<const T *>(gate), static_cast<const T *>(write),
                          initial_state, final_state, static_cast<T *>(output)};
      return by_steps(on, a);
    }
    auto chunks = [&](auto parts) {
      constexpr int P = decltype(parts)::value;
      return by_chunks<T, P>(
          on, ForwardPlan<T, P>(s, scale, lengths), static_cast<const T *>(query),
          static_cast<const T *>(key), static_cast<const T *>(value), static_cast<const T *>(gate),
          static_cast<const T *>(write), initial_state, static_cast<T *>(output), final_state,
          static_cast<char *>(saved), static_cast<char *>(workspace));
    };
    // a state that is handed on keeps 16 bits of what is formed on its way, one that serves these
    // outputs alone as many as they do
    if constexpr (sizeof(T) == 2)
      if (final_state != nullptr) return chunks(std::integral_constant<int, 2>());
    return chunks(std::integral_constant<int, 1>());
  };
  return dtype == OXH_F32 ? run(float()) : run(bf16());
}

}  // extern "C"
