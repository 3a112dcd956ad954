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
// delta_scan_kernel goes from chunk to chunk; columns of values never meet, so a block takes 16 or 32
// of them, its waves the state in the layout of the matrix cores' results, which is that of their next
// operand.  b is never divided by: it may be 0.
//
// What is rounded.  float32 operands: nothing, the matrix cores take float32.  bfloat16 ones: q, k and
// v as they are; the state, N, G o q k', b y and b e as operands of products, 8 bits each, their sums
// and the state itself float32: outputs are 2.4e-3 to 4.3e-3 off in the mean square, the more the longer
// a state lasts and the narrower it is, 1.7e-3 being their own rounding.  A state that is handed on is
// formed from pairs of such operands that add up to 16 bits (2^-17; 2e-6 to 6e-6 in the mean square):
// rounding it to 8 at each of many chunks is no error of one output but of all later calls.
//
// Measured, bfloat16, heads of 128 keys and 128 values: 8 x 2048 x 16 heads with what the backward reads
// 60 us to prepare (183 MB, 3.1 TB/s) and 144 to scan (511 MB, 3.5 TB/s): memory.  1 x 32768 x 16 heads
// with a final state 3 x 64 and 3 x 220 us, 1.3 us a chunk: the way of a chunk through one block (its
// three exchanges, about 300 instructions of a wave and 96 KB from the caches at 64 bytes a cycle),
// on half of the compute units.  Loading the same two chunks again and again took as long.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <string>

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
  char *keys;   // operands of keys, queries and transposed keys of (batch, key head, chunk), or null
};

// A block per chunk and value head.  Its own work is 64 x 64 products; what it reads and writes bounds
// it, or for one chunk of few heads the inversion's 16 dependent steps and three more barriers
// (float32 128 x 28 x 4 heads of 32: 15 to 18 us).
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
  // the first of a key head's value heads brings what they share
  const bool copies = a.keys != nullptr && at.head % d.group == 0;
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
          if (copies)
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
  if (!copies) return;
#pragma unroll
  for (int s = 0; s < KT; ++s)
    keys[(wave * KT + s) * 64] = m.key_row(index_of(wave, n), s, g);
  store_transposed<T, KT>(m.tile, across - lane);
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

// What the block's waves hand each other, as operands: the state, b y, b e, exp(g_64 - g) b e, and e
// for the backward; and a chunk's keys, queries and gates.
template <typename T, int P, int KT, int C>
struct Exchange {
  operand<T> state[KT][C][P][64], weighted[2][C][P][64], wrote[2][C][P][64], left[2][C][P][64],
      error[2][C][64];
  Gates gates[2];                             // of the chunks with even and with odd numbers
  RowTile<T, C == 2 ? KT : 0> keys[2], queries;  // where they are staged
};

// A block of eight waves per C slabs of 16 columns of a head's values.  Each holds 16 of the keys;
// the first four follow the errors of 16 of a chunk's steps each, the others form those steps'
// outputs beside them, a stage behind (four waves with all of it: 250 us a launch where this takes
// 220).  What they form of each other's products goes through shared memory, three times a chunk; what
// stands on the left of a product, or here of its transpose, is one wave's alone, and is loaded a chunk
// ahead, as soon as the present chunk's is used.  The chunk's matrices go straight to registers.  So do
// keys and queries with one slab, as operands that were prepared: few blocks are as fast as a chunk's
// way through one, and shared memory takes longer (1 x 32768 x 16 heads: 654 us of scans, 807 with
// rows staged).  Blocks of two slabs stage their rows in shared memory, where the sums over the keys
// and those over the steps both find their operands: of many blocks the bytes count, a third less
// without the copies (8 x 2048 x 16 heads: 204 us prepared and scanned, 270 with copies).
template <typename T, int P, int KT, int C, bool Packed>
__global__ __launch_bounds__(512, Packed && sizeof(T) == 2 && C == 2 && P == 1 ? 4 : 2) void
delta_scan_kernel(ScanArgs<T> a) {
  using Op = operand<T>;
  using Kept = Chunk<T, P>;
  __shared__ Exchange<T, P, KT, C> m;
  const Dims &d = a.d;
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const bool errs = wave < 4;
  const int pair = w >> 1, half = w & 1;  // of tiles of 16 steps: an operand of 32
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
  constexpr bool kStaged = C == 2;
  const char *copies =
      a.keys + (static_cast<uint64_t>(b) * d.key_heads + kh) * d.chunks * (3 * kKeys);
  const uint32_t value_bytes = static_cast<uint32_t>(value_stride * sizeof(T));
  // A lane's columns: of two slabs those that make its 4 rows of two results 8 in sequence.
  auto column_of = [&](int c, uint32_t n) {
    return C == 2 ? 32 * block.x + index_of(c, n) : 16 * block.x + n;
  };
  constexpr uint32_t kValue = sizeof(T);
  auto rows_of = [&](uint32_t chunk) -> uint32_t {
    return min(length - start - chunk * kChunk, static_cast<uint32_t>(kChunk));
  };
  const uint32_t tile = wave ^ 4;  // of 16 keys: half an operand
  const bool holds = tile < 2 * KT;
  const uint64_t state_at = head * d.keys * d.values;
  auto key_at = [&](int r) { return index_of(tile, 4 * g + r); };
  f32x4 state[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    state[c] = f32x4{};
    if (a.from == nullptr || !holds) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t k = key_at(r), there = min(k, d.keys - 1);
      const float v = a.from[state_at + static_cast<uint64_t>(there) * d.values +
                             min(column_of(c, n), d.values - 1)];
      state[c][r] = k < d.keys && column_of(c, n) < d.values ? v : 0.0f;
    }
  }

  // No load or store of the loop is behind a branch, so that each use waits for its own loads alone:
  // the last chunk loads itself again, and stores that are not to be go past their buffer's end.
  const uint32_t lane_at = lane * sizeof(Op);
  Op back[2];
  auto load_copies = [&](uint32_t chunk, uint32_t part, auto &to, uint32_t first) {
    const auto from = buffer_of(copies + (chunk * uint64_t{3 * kKeys} + part * kKeys), kKeys);
#pragma unroll
    for (uint32_t s = 0; s < sizeof(to) / sizeof(Op); ++s)
      to[s] = load_from<Op>(from, lane_at, (first + s) * kOperand);
  };
  auto load_back = [&](uint32_t chunk) { load_copies(chunk, 2, back, 2 * min(tile, 2 * KT - 1u)); };
  auto operands_of = [&](uint32_t chunk, uint64_t part) {
    return buffer_of(chunks + (chunk * Kept::bytes + part),
                     static_cast<uint32_t>(Kept::bytes - part));
  };
  typedef T quarter __attribute__((ext_vector_type(4)));
  // a wave's half of an operand that two waves form
  auto hand = [&](Op(&to)[P][64], f32x4 v, uint32_t half) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const quarter q = __builtin_convertvector(v, quarter);
      reinterpret_cast<quarter *>(&to[p][lane])[half] = q;
      if (p + 1 < P) v -= widened(q);
    }
  };
  auto hand_state = [&] {
    if (KT < 4 && !holds) return;
#pragma unroll
    for (int c = 0; c < C; ++c) hand(m.state[tile >> 1][c], state[c], tile & 1);
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
  // S = exp(g_64) S0 + k' (exp(g_64 - g) b e)
  auto advance = [&](uint32_t chunk) {
    if (KT == 4 || holds) {
      Op left[2][C][P];
      const float whole = m.gates[chunk & 1].since[kChunk - 1];
      if constexpr (kStaged)
#pragma unroll
        for (int s = 0; s < 2; ++s) back[s] = m.keys[chunk & 1].across(tile, s, n, g);
      read_pairs(left, m.left);
#pragma unroll
      for (int c = 0; c < C; ++c) state[c] *= whole;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int c = 0; c < C; ++c) state[c] = product(back[s], left[s][c][p], state[c]);
    }
    if constexpr (!kStaged) {
      __builtin_amdgcn_sched_barrier(0);
      load_back(min(chunk + 1, live - 1));
    }
    hand_state();
  };
  // a lane's 4 steps
  auto gates_of = [&](uint32_t chunk, float(Gates::*which)[kChunk]) {
    return *reinterpret_cast<const f32x4 *>(&(m.gates[chunk & 1].*which)[index_of(w, 4 * g)]);
  };
  if (live != 0) {
    if constexpr (!kStaged) load_back(0);
    hand_state();
  }
  if (errs) {
    Op key[KT], solve[2][P];
    // the values: a lane its columns of 4 steps, or in a row's order 8 columns of a step, which a
    // product with columns of the identity brings there
    constexpr bool kRows = Packed && sizeof(T) == 2 && kStaged;
    T value[C][4];
    Op row, unit[C];
    uint32_t at[C][4], row_at = kNowhere;
    if constexpr (kRows) {
      const uint32_t first = 32 * (C == 2 ? block.x : block.x >> 1) + 8 * g;
      if (first < d.values) row_at = index_of(w, n) * value_bytes + first * kValue;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          unit[c][i] = static_cast<T>(first + i == column_of(c, n) ? 1.0f : 0.0f);
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          at[c][r] = column_of(c, n) < d.values
                         ? index_of(w, 4 * g + r) * value_bytes + column_of(c, n) * kValue
                         : kNowhere;
    }
    auto read_keys = [&](uint32_t chunk) {
      if constexpr (kStaged) {
#pragma unroll
        for (int s = 0; s < KT; ++s) key[s] = m.keys[chunk & 1].along(index_of(w, n), s, g);
      } else {
        load_copies(chunk, 0, key, w * KT);
      }
    };
    auto load_values = [&](uint32_t chunk) {
      const auto from = buffer_of(values + chunk * kChunk * value_stride,
                                  rows_of(chunk) * value_bytes);
      if constexpr (kRows) {
        row = load_from<Op>(from, row_at, 0);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < C; ++c) value[c][r] = load_from<T>(from, at[c][r], 0);
      }
    };
    auto load_system = [&](uint32_t chunk) {
      const auto from = operands_of(chunk, Kept::system);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int p = 0; p < P; ++p)
          solve[s][p] =
              load_from<Op>(from, lane_at, (lower_place(w, min(s, pair)) * P + p) * kOperand);
    };
    if (live != 0) {
      load_values(0);
      load_system(0);
      if constexpr (kStaged) lds_barrier();
      read_keys(0);
    }
    for (uint32_t chunk = 0; chunk < live; ++chunk) {
      const uint32_t next = min(chunk + 1, live - 1);
      lds_barrier();
      f32x4 y[C] = {}, v[C] = {};
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
        for (int s = 0; s < KT; ++s)
#pragma unroll
          for (int p = P - 1; p >= 0; --p)
#pragma unroll
            for (int c = 0; c < C; ++c) y[c] = product(key[s], right[s][c][p], y[c]);
        if constexpr (kRows)
#pragma unroll
          for (int c = 0; c < C; ++c) v[c] = product(row, unit[c], v[c]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (!kStaged) read_keys(next);
      const f32x4 since = gates_of(chunk, &Gates::since), write = gates_of(chunk, &Gates::write);
      const f32x4 until = gates_of(chunk, &Gates::until);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if constexpr (!kRows)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[c][r] = widen(value[c][r]);
        y[c] = v[c] - since * y[c];
        hand(m.weighted[pair][c], -write * y[c], half);
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
        hand(m.left[pair][c], until * y[c], half);
        hand(m.wrote[pair][c], y[c], half);
      }
      lds_barrier();
      if constexpr (kStaged) read_keys(next);
      advance(chunk);
    }
  } else {
    Op scores[2], query[KT];
    f32x4 o[C] = {}, gates;  // and 4 of a chunk's gates, a lane
    const uint32_t row_bytes = d.key_heads * d.keys * kValue;
    using Part = RowPart<T, kStaged ? KT : 0, Packed>;
    const Part part(threadIdx.x - 256, row_bytes, d.keys);
    typename Part::Values key_part, query_part;
    const uint64_t key_row0 = (row0 * d.key_heads + kh) * d.keys;
    auto load_rows = [&](typename Part::Values &to, const T *from, uint32_t chunk) {
      const uint64_t first = chunk * kChunk * static_cast<uint64_t>(d.key_heads) * d.keys;
      part.load(to, buffer_of(from + key_row0 + first, rows_of(chunk) * row_bytes), d.keys);
    };
    auto load_scores = [&](uint32_t chunk) {
      const auto from = operands_of(chunk, Kept::within);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        scores[s] = load_from<Op>(from, lane_at, lower_place(w, min(s, pair)) * kOperand);
    };
    // The outputs are formed transposed: a lane a step, its columns in sequence.
    const uint32_t step = index_of(w, n), first = column_of(0, 4 * g);
    // what the backward reads of a chunk; a block of one slab brings its half of the pair's lanes
    const uint32_t kept = (d.slabs + 1) / 2 * (2 * KT + 4) * kOperand;
    const bool brings = C == 2 || (g >> 1) == (block.x & 1);
    auto saved_of = [&](uint32_t chunk, bool there) {
      return buffer_of(a.saved + ((head * a.all + d.first + chunk) * kept), there ? kept : 0);
    };
    auto saved_at = [&](int place) {
      return brings ? (block.x * C / 2 * (2 * KT + 4) + place) * kOperand + lane_at : kNowhere;
    };
    // o = exp(g) q S0 + (G o q k') (b e) of a chunk, the first part there
    Op wrote[2][C][P];
    auto finish = [&](uint32_t chunk, bool there) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (s > pair) continue;
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int c = 0; c < C; ++c) o[c] = product(wrote[s][c][p], scores[s], o[c]);
      }
      const auto to = buffer_of(outs + chunk * kChunk * value_stride,
                                there ? rows_of(chunk) * value_bytes : 0);
      const uint32_t at = step * value_bytes + first * kValue;
      // 16 bytes at a time end with a row's values: 8 of bfloat16, 4 of float32
      if constexpr (Packed && C == 2 && sizeof(T) == 2) {
        store_to(to, first < d.values ? at : kNowhere, rounded<T>(join(o[0], o[1])));
      } else {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          if constexpr (Packed) {
            store_to(to, first + 4 * c < d.values ? at + 4 * c * kValue : kNowhere,
                     __builtin_convertvector(o[c], quarter));
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              store_to(to, first + 4 * c + r < d.values ? at + (4 * c + r) * kValue : kNowhere,
                       static_cast<T>(o[c][r]));
          }
        }
      }
    };
    auto load_gates = [&](uint32_t chunk) {
      gates = load_from<f32x4>(buffer_of(chunks + (chunk * Kept::bytes + Kept::gates), sizeof(Gates)),
                               lane * 16, 0);
    };
    auto hand_gates = [&](uint32_t chunk) {
      if (w == 0 && lane < sizeof(Gates) / 16)
        reinterpret_cast<f32x4 *>(&m.gates[chunk & 1])[lane] = gates;
      __builtin_amdgcn_sched_barrier(0);
      load_gates(min(chunk + 1, live - 1));
    };
    // the errors of a chunk for the backward
    auto save_errors = [&](uint32_t chunk, bool there) {
      if (a.saved != nullptr)
        store_to(saved_of(chunk, there), saved_at(2 * KT + w),
                 turned<C == 2>(&m.error[pair][0][0], C == 2 ? 64 : 0, half, n, g));
    };
    if (live != 0) {
      load_scores(0);
      load_gates(0);
      if constexpr (kStaged) {
        load_rows(key_part, a.key, 0);
        part.store(m.keys[0], key_part);
        __builtin_amdgcn_sched_barrier(0);
        load_rows(key_part, a.key, min(1u, live - 1));
        load_rows(query_part, a.query, 0);
      } else {
        load_copies(0, 1, query, w * KT);
      }
      hand_gates(0);
      if constexpr (kStaged) lds_barrier();
    }
    for (uint32_t chunk = 0; chunk < live; ++chunk) {
      lds_barrier();
      // the chunk before's outputs, while the others form this one's errors; before the first one
      // nothing is there
      const uint32_t before = max(chunk, 1u) - 1, next = min(chunk + 1, live - 1);
      read_pairs(wrote, m.wrote);
      if constexpr (kStaged) {
        part.store(m.queries, query_part);
        part.store(m.keys[(chunk + 1) & 1], key_part);
        __builtin_amdgcn_sched_barrier(0);
        load_rows(query_part, a.query, next);
        load_rows(key_part, a.key, min(chunk + 2, live - 1));
      } else {
        finish(before, chunk != 0);
        __builtin_amdgcn_sched_barrier(0);
        load_scores(chunk);
      }
      save_errors(before, chunk != 0);
      if (a.saved != nullptr && w < KT) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          store_to(saved_of(chunk, true), saved_at(2 * w + i),
                   turned<C == 2>(&m.state[w][0][0][0], C == 2 ? P * 64 : 0, i, n, g));
      }
      lds_barrier();
      if constexpr (kStaged) {
        finish(before, chunk != 0);
        __builtin_amdgcn_sched_barrier(0);
        load_scores(chunk);
      }
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = f32x4{};
      constexpr int kAtOnce = kStaged && KT == 4 ? 2 : KT;  // more would leave registers for one block alone
#pragma unroll
      for (int from = 0; from < KT; from += kAtOnce) {
        Op right[kAtOnce][C];
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s) {
          if constexpr (kStaged) query[from + s] = m.queries.along(step, from + s, g);
#pragma unroll
          for (int c = 0; c < C; ++c) right[s][c] = m.state[from + s][c][0][lane];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s)
#pragma unroll
          for (int c = 0; c < C; ++c) o[c] = product(right[s][c], query[from + s], o[c]);
        __builtin_amdgcn_sched_barrier(0);
      }
      const float since = m.gates[chunk & 1].since[step] * d.scale;
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] *= since;
      if constexpr (!kStaged) {
        __builtin_amdgcn_sched_barrier(0);
        load_copies(next, 1, query, w * KT);
      }
      lds_barrier();
      advance(chunk);
      hand_gates(chunk + 1);
    }
    if (live != 0) {
      read_pairs(wrote, m.wrote);
      save_errors(live - 1, true);
      finish(live - 1, true);
    }
  }
  // steps past the row's end
  const uint32_t end = min(d.time - start, d.chunks * kChunk);
  for (uint32_t t = (length <= start ? 0 : length - start) + 4 * wave + g; t < end; t += 32) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (column_of(c, n) < d.values)
        outs[t * value_stride + column_of(c, n)] = static_cast<T>(0.0f);
  }
  if (a.to == nullptr || !holds) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint32_t k = key_at(r);
    if (k >= d.keys) continue;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (column_of(c, n) < d.values)
        a.to[state_at + static_cast<uint64_t>(k) * d.values + column_of(c, n)] = state[c][r];
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
// registers from step to step.  One step reads and writes the state once, in 16 bytes a lane of a row
// of 128: 64 rows of 32 heads of 128 x 128 in 57 us a call, 4.7 TB/s, which bounds it (48 us and 5.6
// TB/s in a trace of two sets of states in turn, of which the caches keep a part).
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

// Steps taken one by one where no backward is to follow: they cost about 1.5 us each, or with many
// heads their products on the vector units; a chunk costs as much for one step as for 64.  (16 steps
// of 16 heads: 28 us one by one, 16 by a chunk in bfloat16, and 25 and 23 in float32; of 512 heads 44
// and 53, 38 and 96; 8 steps of 16 heads: 16 and 15, 14 and 23.)  float32 chunks are four times as
// dear on the matrix cores, so many heads take more steps (48 of 512 heads: 88 us and 98).
uint64_t step_limit(const oxh_delta_shape &s, bool f32) {
  const uint64_t waves = s.batch * s.heads * ((s.value_dim + 31) / 32);
  return f32 && waves >= 8 * oxh::kComputeUnits ? 48 : 16;
}

template <typename T, int P>
struct ForwardPlan {
  Plan p;
  bool two;                                     // slabs of a block of the scan
  uint64_t head_bytes, key_bytes, state_bytes;  // of the workspace
  uint64_t bytes() const { return head_bytes + key_bytes + state_bytes; }
  ForwardPlan(const oxh_delta_shape &s, float scale, const int32_t *lengths)
      : p(s, scale, lengths) {
    const uint64_t head = s.batch * s.heads * Chunk<T, P>::bytes;
    // Two where that leaves a block for each compute unit (a head of 128 values has 4 such blocks.
    // Of 1024 steps, one and two slabs: bfloat16 128 blocks 41 and 48 us, 256 blocks 57 and 52, 512
    // blocks 128 and 94; float32 73 and 111, 137 and 131, 305 and 263).
    two = s.batch * s.heads * ((p.d.slabs + 1) / 2) >= oxh::kComputeUnits;
    const uint64_t key = two ? 0 : s.batch * s.key_heads * p.steps * 12 * kOperandBytes<T>;
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
oxh_status by_chunks(hipStream_t stream, const ForwardPlan<T, P> &plan, const T *query,
                     const T *key, const T *value, const T *gate, const T *write,
                     const float *initial, T *out, float *final, char *saved, char *workspace) {
  const Plan &p = plan.p;
  char *heads = workspace, *keys = plan.two ? nullptr : heads + plan.head_bytes;
  float *between = reinterpret_cast<float *>(heads + plan.head_bytes + plan.key_bytes);
  const uint32_t pairs = (p.d.slabs + 1) / 2;
  // whether 16 bytes of a row are loaded and stored at once
  const bool packed = p.d.values % (16 / sizeof(T)) == 0 && p.d.keys % (16 / sizeof(T)) == 0 &&
                      oxh::aligned16(query) && oxh::aligned16(key) && oxh::aligned16(value) &&
                      oxh::aligned16(out);
  for (uint64_t first = 0; first < p.all; first += p.segment) {
    Dims d = p.d;
    d.first = static_cast<uint32_t>(first);
    d.chunks = static_cast<uint32_t>(std::min(p.segment, p.all - first));
    const bool last = first + p.segment >= p.all;
    const PrepareArgs<T> prepare{d, query, key, gate, write, heads, keys};
    const ScanArgs<T> scan{d, query, key, value, heads, keys, first == 0 ? initial : between,
                           last ? final : between, out, saved, static_cast<uint32_t>(p.all)};
    with_keys(d.keys, d.keys % 32 == 0, [&](auto steps, auto whole) {
      constexpr int KT = decltype(steps)::value;
      constexpr bool W = decltype(whole)::value;
      oxh::launch(delta_prepare_kernel<T, P, KT, W>, dim3(d.chunks, d.heads, d.batch), dim3(256), 0,
                  stream, prepare);
      auto go = [&](auto columns, auto packs) {
        constexpr int C = decltype(columns)::value;
        oxh::launch(delta_scan_kernel<T, P, KT, C, decltype(packs)::value>,
                    dim3(2 / C * pairs, d.heads, d.batch), dim3(512), 0, stream, scan);
      };
      auto slabs = [&](auto packs) {
        if (plan.two) go(std::integral_constant<int, 2>(), packs);
        else go(std::integral_constant<int, 1>(), packs);
      };
      if (packed) slabs(std::true_type());
      else slabs(std::false_type());
    });
    oxh_status st = oxh::launched("gated_delta_rule");
    if (st != OXH_OK) return st;
  }
  return oxh::ok();
}

// Bytes of the workspace of every form that a call by chunks may take (P: it hands a state on or not).
// The one of two operands' parts has the larger chunks, so it may prepare fewer of them at a time and
// need less in all (8 x 6144 x 16 heads of 128: 126 MB, the other 160).
template <typename T>
uint64_t chunks_bytes(const oxh_delta_shape &s) {
  const uint64_t one = ForwardPlan<T, 1>(s, 1.0f, nullptr).bytes();
  return sizeof(T) == 4 ? one : std::max(one, ForwardPlan<T, 2>(s, 1.0f, nullptr).bytes());
}

bool by_steps_alone(int dtype, const oxh_delta_shape &s, bool saves) {
  return s.time == 0 || (!saves && s.time <= step_limit(s, dtype == OXH_F32));
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
  if (by_steps_alone(dtype, *shape, saves != 0)) return oxh::ok();
  *bytes = dtype == OXH_F32 ? chunks_bytes<float>(*shape) : chunks_bytes<bf16>(*shape);
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
  Spans in = {{query, z.query, z.element}, {key, z.query, z.element},
              {value, z.value, z.element}, {gate, z.gate, z.element},
              {write, z.gate, z.element}};
  Spans out = {{output, z.value, z.element}};
  for (const auto *list : {&in, &out})
    for (const Span &x : *list)
      OXH_REQUIRE(x.p != nullptr || x.bytes == 0, OXH_INVALID_SHAPE,
                  "gated delta rule: null pointer");
  in.push_back({lengths, s.batch * 4, 4});
  out.push_back({final_state, z.state, 4});
  const bool steps = by_steps_alone(dtype, s, saved != nullptr);
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
