// delta_rule_backward.hip -- gradients of the gated delta rule (delta_rule.hip), by its chunks.
//
// With the notation there, u = b e, and the gradients do of the outputs and dS of the state behind
// the chunk:
//
//   du = scale (G o q k')' do + exp(g_64 - g) k dS;  x = du - N' (b du);  dv = b x
//   dS0 = exp(g_64) dS + scale q' (exp(g) do) - k' (exp(g) dv)
//   M1 = scale G o (do u') (i <= t);  M2 = -G o (dv u') (i < t)
//   dq = scale exp(g) do S0' + M1 k
//   dk = -exp(g) dv S0' + exp(g_64 - g) u dS' + M1' q + (M2 + M2') k
//   dwrite = (e . x) b (1 - b)
//   dgate_s = (1 - a_s) (sum over t >= s of (q.dq - dk.k from S0) + over i < s of (k.dk from dS)
//             + <dS, exp(g_64) S0> + over i < s <= t of H_ti),  H = G o (scale (do u') o q k'
//             - (dv u') o k k')
//
// The last sum is that of (H's rows - its columns) over t >= s: the pairs that do not span s take
// themselves away to the last bit, whatever their operands were rounded to.
//
// Three kernels: what depends on no state, for all chunks at once; the state's gradient from the
// last chunk to the first, a block for 16 or 32 columns of values; and the products over the values,
// a block per chunk and key head.  S0 and e are the forward's.
//
// Rounded as the forward's: of bfloat16 operands u, x, dS, S0, e, M1, M2 and the matrices keep 8 bits
// where they are operands, sums and dS itself float32; gradients are 2.3e-3 to 4.3e-3 off in the
// mean square, those of gates, whose terms cancel, up to 6.5e-3.  The gates' sums are float32 throughout
// but for those operands.
//
// Measured, bfloat16, 8 x 2048 x 16 heads of 128 keys and values, in two parts: 2 x 37 us to prepare, 2 x
// 82 to scan (509 MB in both, 3.1 TB/s) and 2 x 99 for the products (721 MB, 3.6 TB/s; their matrix
// work is 30 us): memory, with two blocks a compute unit.  float32 128 x 28 x 4 heads of 32, one chunk:
// 15, 12 and 20 us, the chain of a block's stages.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <string>

#include "common.h"
#include "delta_rule.h"
#include "storage.h"

namespace {

using namespace oxh::delta;
using oxh::storage::widen;

// What a chunk's kernels leave each other, per value head; then per pair of slabs dS (tiles of 16
// keys) and x (tiles of 16 steps) as operands of sums over the values.
template <typename T>
struct Back {
  static constexpr uint64_t gates = 0, system = sizeof(Gates),
                            within = system + kTriangle * kOperandBytes<T>,
                            pairs = within + kTriangle * kOperandBytes<T>;
  static __host__ __device__ constexpr uint64_t pair(uint64_t steps) {
    return (2 * steps + 4) * kOperandBytes<T>;
  }
  static __host__ __device__ constexpr uint64_t bytes(uint64_t steps, uint64_t count) {
    return pairs + count * pair(steps);
  }
};

template <typename T>
struct Args {
  Dims d;
  const T *query, *key, *gate, *write, *gradient;
  const char *saved;
  char *heads, *keys;   // Back<T> of (batch, head, chunk); keys, their transpose, queries' transpose,
                        // or null
  const float *from;    // gradients of the states behind the launch's chunks, null: 0
  float *to;            // and before them, may be null
  T *dquery, *dkey, *dvalue, *dgate, *dwrite;
  uint32_t all, pairs;  // chunks of the whole sequence; pairs of slabs
};

template <typename T, int KT, bool Whole>
__global__ __launch_bounds__(256) void delta_backward_prepare_kernel(Args<T> a) {
  using Op = operand<T>;
  __shared__ System<T, KT> m;
  const Dims &d = a.d;
  const Place at(d, blockIdx.x, blockIdx.y, blockIdx.z);
  if (at.rows == 0) return;
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T *query = a.query + at.key_row * d.keys;
  const uint64_t stride = static_cast<uint64_t>(d.key_heads) * d.keys;
  char *out = a.heads + at.head_chunk(d) * Back<T>::bytes(KT, a.pairs);
  solve<T, KT, Whole>(
      m, d, at, a.key, a.gate, a.write, reinterpret_cast<Gates *>(out + Back<T>::gates), [&] {
        // (G o q k')', a lane its key's step i, queries' steps t
        const uint32_t first = wave == 1 ? 2 : wave - 2, last = wave == 1 ? 3 : wave - 2;
        for (uint32_t ki = first; ki <= last; ++ki) {
          const uint32_t i = index_of(ki, n);
          for (int step = ki >> 1; step < 2; ++step) {
            f32x4 half[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              f32x4 acc = {};
              const T *row = query + min(index_of(2 * step + e, n), at.rows - 1) * stride;
#pragma unroll
              for (int s = 0; s < KT; ++s)
                acc = product(load_row<T, Whole>(row, 32 * s + 8 * g, d.keys), m.key_row(i, s, g),
                              acc);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const uint32_t t = 32 * step + 8 * g + 4 * e + r;
                half[e][r] = i <= t ? acc[r] * m.between(t, i) * d.scale : 0.0f;
              }
            }
            Op *to = reinterpret_cast<Op *>(out + Back<T>::within);
            to[upper_place(ki, step) * 64 + lane] = rounded<T>(join(half[0], half[1]));
          }
        }
      });
  for (int p = wave; p < kTriangle; p += 4) {
    const int ki = p < 4 ? p / 2 : p - 2, step = p < 4 ? p % 2 : 1;
    const uint32_t i = index_of(ki, n);
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = m.mat[32 * step + 8 * g + j][i];
    reinterpret_cast<Op *>(out + Back<T>::system)[p * 64 + lane] = rounded<T>(v);
  }
  if (a.keys == nullptr || at.head % d.group != 0) return;
  Op *to = reinterpret_cast<Op *>(a.keys) + at.key_chunk(d) * (12 * KT * 64);
#pragma unroll
  for (int s = 0; s < KT; ++s)
    to[(wave * KT + s) * 64 + lane] = m.key_row(index_of(wave, n), s, g);
  store_transposed<T, KT>(m.tile, to + 4 * KT * 64);
  __syncthreads();
  load_tile<T, KT, Whole>(m.tile, d, at, a.query);
  __syncthreads();
  store_transposed<T, KT>(m.tile, to + 8 * KT * 64);
}

// The sums over the 16 lanes of a group.
__device__ __forceinline__ float row_total(float v) {
  v += oxh::dpp_move<0xB1>(v);
  v += oxh::dpp_move<0x4E>(v);
  v += oxh::dpp_move<0x141>(v);
  v += oxh::dpp_move<0x140>(v);
  return v;
}

// What the block's waves hand each other, as operands: dS, do, scale exp(g) do, -b du, -exp(g) dv, x
// for the products and dv; and a chunk's keys (of those with even and with odd numbers) and queries
// where they are staged.
template <typename T, int KT, int C>
struct Exchange {
  operand<T> state[KT][C][64], out[2][C][64], decayed[2][C][64], weighted[2][C][64],
      taken[2][C][64], x[2][C][64], dv[2][C][64];
  RowTile<T, C == 2 ? KT : 0> keys[2], queries;
};

// A block of eight waves per C slabs of 16 columns of a head's values, from the last chunk to the
// first.  They share a chunk as the forward's do: each holds 16 of the keys, the first four follow x,
// the others bring the rows and do, and store what a chunk leaves a stage behind.
template <typename T, int KT, int C, bool Packed>
__global__ __launch_bounds__(512, Packed && sizeof(T) == 2 && C == 2 ? 4 : 2) void
delta_backward_scan_kernel(Args<T> a) {
  using Op = operand<T>;
  using Kept = Back<T>;
  __shared__ Exchange<T, KT, C> m;
  const Dims &d = a.d;
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const int pair = w >> 1, half = w & 1;
  const oxh::BlockTile block = oxh::xcd_block();
  const uint32_t h = block.y, b = block.z, kh = h / d.group;
  const uint32_t length = length_of(d, b), start = d.first * kChunk;
  const uint32_t live =
      length <= start ? 0 : min((length - start + kChunk - 1) / kChunk, d.chunks);
  const uint64_t head = static_cast<uint64_t>(b) * d.heads + h;
  const uint64_t value_stride = static_cast<uint64_t>(d.heads) * d.values;
  const uint64_t row0 = static_cast<uint64_t>(b) * d.time + start;
  const uint64_t value0 = row0 * value_stride + static_cast<uint64_t>(h) * d.values;
  const T *gradients = a.gradient + value0;
  T *dvalues = a.dvalue + value0;
  const uint64_t block_bytes = Kept::bytes(KT, a.pairs);
  char *chunks = a.heads + head * d.chunks * block_bytes;
  constexpr uint32_t kOperand = 64 * sizeof(Op), kKeys = 4 * KT * kOperand, kValue = sizeof(T);
  constexpr bool kStaged = C == 2;
  const char *copies =
      a.keys + (static_cast<uint64_t>(b) * d.key_heads + kh) * d.chunks * (3 * kKeys);
  const uint32_t value_bytes = static_cast<uint32_t>(value_stride * sizeof(T));
  auto column_of = [&](int c) { return 16 * (block.x * C + c) + n; };
  auto rows_of = [&](uint32_t chunk) -> uint32_t {
    return min(length - start - chunk * kChunk, static_cast<uint32_t>(kChunk));
  };
  const uint32_t tile = wave ^ 4;  // of 16 keys: half an operand
  const bool holds = tile < 2 * KT;
  const uint64_t state_at = head * d.keys * d.values;
  auto key_at = [&](int r) { return index_of(tile, 4 * g + r); };
  f32x4 ds[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    ds[c] = f32x4{};
    if (a.from == nullptr || !holds) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t k = key_at(r), there = min(k, d.keys - 1);
      const float v = a.from[state_at + static_cast<uint64_t>(there) * d.values +
                             min(column_of(c), d.values - 1)];
      ds[c][r] = k < d.keys && column_of(c) < d.values ? v : 0.0f;
    }
  }

  // Loaded and stored as the forward's.
  typedef T quarter __attribute__((ext_vector_type(4)));
  Op back[2], forth[2];
  float whole = 0.0f;
  const uint32_t lane_at = lane * sizeof(Op);
  auto operands_of = [&](uint32_t chunk, uint64_t part) {
    return buffer_of(chunks + (chunk * block_bytes + part),
                     static_cast<uint32_t>(Kept::pairs - part));
  };
  auto load_copies = [&](uint32_t chunk, uint32_t part, auto &to, uint32_t first) {
    const auto from = buffer_of(copies + (chunk * uint64_t{3 * kKeys} + part * kKeys), kKeys);
#pragma unroll
    for (uint32_t s = 0; s < sizeof(to) / sizeof(Op); ++s)
      to[s] = load_from<Op>(from, lane_at, (first + s) * kOperand);
  };
  auto load_rest = [&](uint32_t chunk) {
    whole = load_from<float>(operands_of(chunk, Kept::gates),
                             offsetof(Gates, since) + (kChunk - 1) * 4, 0);
    if constexpr (!kStaged) {
      load_copies(chunk, 1, back, 2 * min(tile, 2 * KT - 1u));
      load_copies(chunk, 2, forth, 2 * min(tile, 2 * KT - 1u));
    }
  };
  auto hand = [&](Op(&to)[64], f32x4 v, uint32_t half) {
    reinterpret_cast<quarter *>(&to[lane])[half] = __builtin_convertvector(v, quarter);
  };
  auto hand_state = [&] {
    if (KT < 4 && !holds) return;
#pragma unroll
    for (int c = 0; c < C; ++c) hand(m.state[tile >> 1][c], ds[c], tile & 1);
  };
  auto read_pairs = [&](Op(&to)[2][C], const Op(&from)[2][C][64]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int c = 0; c < C; ++c) to[s][c] = from[s][c][lane];
  };
  // dS0 = exp(g_64) dS + scale q' (exp(g) do) - k' (exp(g) dv)
  auto advance = [&](uint32_t chunk, uint32_t next) {
    if (KT == 4 || holds) {
#pragma unroll
      for (int c = 0; c < C; ++c) ds[c] *= whole;
      // one sum after the other: both sums' operands would take registers of a second block
      {
        Op right[2][C];
        if constexpr (kStaged)
#pragma unroll
          for (int s = 0; s < 2; ++s) forth[s] = m.queries.across(tile, s, n, g);
        read_pairs(right, m.decayed);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int c = 0; c < C; ++c) ds[c] = product(forth[s], right[s][c], ds[c]);
      }
      __builtin_amdgcn_sched_barrier(0);
      {
        Op right[2][C];
        if constexpr (kStaged)
#pragma unroll
          for (int s = 0; s < 2; ++s) back[s] = m.keys[chunk & 1].across(tile, s, n, g);
        read_pairs(right, m.taken);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int c = 0; c < C; ++c) ds[c] = product(back[s], right[s][c], ds[c]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_rest(next);
    if (chunk != 0) hand_state();
  };
  if (live != 0) {
    load_rest(live - 1);
    hand_state();
  }
  if (wave < 4) {
    Op key[KT], scores[2], solve[2];
    f32x4 since, until, write;
    auto read_keys = [&](uint32_t chunk) {
      if constexpr (kStaged) {
#pragma unroll
        for (int s = 0; s < KT; ++s) key[s] = m.keys[chunk & 1].along(index_of(w, n), s, g);
      } else {
        load_copies(chunk, 0, key, w * KT);
      }
    };
    auto load_triangle = [&](uint32_t chunk, uint64_t part, Op(&to)[2]) {
      const auto from = operands_of(chunk, part);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        to[s] = load_from<Op>(from, lane_at, upper_place(w, max(s, pair)) * kOperand);
    };
    auto load_gates = [&](uint32_t chunk) {
      const auto from = operands_of(chunk, Kept::gates);
      const uint32_t at = index_of(w, 4 * g) * 4;
      since = load_from<f32x4>(from, at, offsetof(Gates, since));
      until = load_from<f32x4>(from, at, offsetof(Gates, until));
      write = load_from<f32x4>(from, at, offsetof(Gates, write));
    };
    if (live != 0) {
      const uint32_t last = live - 1;
      load_triangle(last, Kept::within, scores);
      load_gates(last);
      load_triangle(last, Kept::system, solve);
      if constexpr (kStaged) lds_barrier();
      read_keys(last);
    }
    for (uint32_t chunk = live; chunk-- != 0;) {
      const uint32_t next = chunk == 0 ? 0 : chunk - 1;
      lds_barrier();
      // du = scale (G o q k')' do + exp(g_64 - g) k dS
      f32x4 x[C] = {};
      {
        Op right[KT][C];
#pragma unroll
        for (int s = 0; s < KT; ++s)
#pragma unroll
          for (int c = 0; c < C; ++c) right[s][c] = m.state[s][c][lane];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < KT; ++s)
#pragma unroll
          for (int c = 0; c < C; ++c) x[c] = product(key[s], right[s][c], x[c]);
      }
      __builtin_amdgcn_sched_barrier(0);
      {
        Op out[2][C];
        read_pairs(out, m.out);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < C; ++c) x[c] *= until;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (s < pair) continue;
#pragma unroll
          for (int c = 0; c < C; ++c) x[c] = product(scores[s], out[s][c], x[c]);
        }
      }
#pragma unroll
      for (int c = 0; c < C; ++c) hand(m.weighted[pair][c], -write * x[c], half);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (!kStaged) read_keys(next);
      load_triangle(next, Kept::within, scores);
      lds_barrier();
      // x = du - N' (b du);  dv = b x
      {
        Op right[2][C];
        read_pairs(right, m.weighted);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (s < pair) continue;
#pragma unroll
          for (int c = 0; c < C; ++c) x[c] = product(solve[s], right[s][c], x[c]);
        }
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        hand(m.x[pair][c], x[c], half);
        x[c] *= write;
        hand(m.taken[pair][c], -since * x[c], half);
        hand(m.dv[pair][c], x[c], half);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_triangle(next, Kept::system, solve);
      load_gates(next);
      lds_barrier();
      advance(chunk, next);
      if constexpr (kStaged) read_keys(next);
    }
  } else {
    // do, as the forward has its values
    constexpr bool kRows = Packed && sizeof(T) == 2 && kStaged;
    T gradient[C][4];
    Op row, unit[C];
    uint32_t at[C][4], row_at = kNowhere;
    if constexpr (kRows) {
      const uint32_t first = 32 * block.x + 8 * g;
      if (first < d.values) row_at = index_of(w, n) * value_bytes + first * kValue;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          unit[c][i] = static_cast<T>(first + i == column_of(c) ? 1.0f : 0.0f);
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          at[c][r] = column_of(c) < d.values
                         ? index_of(w, 4 * g + r) * value_bytes + column_of(c) * kValue
                         : kNowhere;
    }
    f32x4 since, v[C] = {};
    auto load_gradients = [&](uint32_t chunk) {
      const auto from = buffer_of(gradients + chunk * kChunk * value_stride,
                                  rows_of(chunk) * value_bytes);
      if constexpr (kRows) {
        row = load_from<Op>(from, row_at, 0);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < C; ++c) gradient[c][r] = load_from<T>(from, at[c][r], 0);
      }
      since = load_from<f32x4>(operands_of(chunk, Kept::gates), index_of(w, 4 * g) * 4,
                               offsetof(Gates, since));
    };
    auto hand_out = [&] {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        v[c] = f32x4{};
        if constexpr (kRows) {
          v[c] = product(row, unit[c], v[c]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) v[c][r] = widen(gradient[c][r]);
        }
        hand(m.out[pair][c], v[c], half);
        v[c] *= since * d.scale;
      }
    };
    const uint32_t row_bytes = d.key_heads * d.keys * kValue;
    using Part = RowPart<T, kStaged ? KT : 0, Packed>;
    const Part part(threadIdx.x - 256, row_bytes, d.keys);
    typename Part::Values key_part, query_part;
    const uint64_t key_row0 = (row0 * d.key_heads + kh) * d.keys;
    auto load_rows = [&](typename Part::Values &to, const T *from, uint32_t chunk) {
      const uint64_t first = chunk * kChunk * static_cast<uint64_t>(d.key_heads) * d.keys;
      part.load(to, buffer_of(from + key_row0 + first, rows_of(chunk) * row_bytes), d.keys);
    };
    // what the products read of a chunk; a block of one slab brings its half of the pair's lanes
    const uint32_t kept = a.pairs * static_cast<uint32_t>(Kept::pair(KT));
    auto pairs_at = [&](uint32_t chunk, bool there) {
      return buffer_of(chunks + (chunk * block_bytes + Kept::pairs), there ? kept : 0);
    };
    const bool brings = C == 2 || (g >> 1) == (block.x & 1);
    auto pair_at = [&](int place) {
      return brings ? (block.x * C / 2 * (2 * KT + 4) + place) * kOperand + lane_at : kNowhere;
    };
    // x and dv of a chunk: a lane its step's 8 columns
    auto finish = [&](uint32_t chunk, bool there) {
      constexpr uint32_t kApart = C == 2 ? 64 : 0;
      store_to(pairs_at(chunk, there), pair_at(2 * KT + w),
               turned<false>(&m.x[pair][0][0], kApart, half, n, g));
      const Op dv = turned<false>(&m.dv[pair][0][0], kApart, half, n, g);
      const auto to = buffer_of(dvalues + chunk * kChunk * value_stride,
                                there ? rows_of(chunk) * value_bytes : 0);
      const uint32_t first = 32 * (C == 2 ? block.x : block.x >> 1) + 8 * g;
      const uint32_t from = index_of(w, n) * value_bytes + first * kValue;
      if constexpr (Packed) {
        if constexpr (sizeof(T) == 2) {
          store_to(to, brings && first < d.values ? from : kNowhere, dv);
        } else {
#pragma unroll
          for (uint32_t i = 0; i < 8; i += 4)
            store_to(to, brings && first + i < d.values ? from + i * kValue : kNowhere,
                     f32x4{dv[i], dv[i + 1], dv[i + 2], dv[i + 3]});
        }
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          store_to(to, brings && first + i < d.values ? from + i * kValue : kNowhere,
                   static_cast<T>(dv[i]));
      }
    };
    if (live != 0) {
      const uint32_t last = live - 1, next = last == 0 ? 0 : last - 1;
      load_gradients(last);
      if constexpr (kStaged) {
        load_rows(key_part, a.key, last);
        part.store(m.keys[last & 1], key_part);
        __builtin_amdgcn_sched_barrier(0);
        load_rows(key_part, a.key, next);
        load_rows(query_part, a.query, last);
      }
      hand_out();
      __builtin_amdgcn_sched_barrier(0);
      load_gradients(next);
      if constexpr (kStaged) lds_barrier();
    }
    for (uint32_t chunk = live; chunk-- != 0;) {
      const uint32_t next = chunk == 0 ? 0 : chunk - 1, after = next == 0 ? 0 : next - 1;
      lds_barrier();
      // the chunk before's (it is the one behind this), while the others form this one's du; at the
      // last chunk nothing is there
      finish(min(chunk + 1, live - 1), chunk + 1 != live);
#pragma unroll
      for (int c = 0; c < C; ++c) hand(m.decayed[pair][c], v[c], half);
      if constexpr (kStaged) {
        part.store(m.queries, query_part);
        part.store(m.keys[(chunk + 1) & 1], key_part);
        __builtin_amdgcn_sched_barrier(0);
        load_rows(query_part, a.query, next);
        load_rows(key_part, a.key, after);
      }
      if (w < KT) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          store_to(pairs_at(chunk, true), pair_at(2 * w + i),
                   turned<false>(&m.state[w][0][0], C == 2 ? 64 : 0, i, n, g));
      }
      lds_barrier();
      hand_out();
      __builtin_amdgcn_sched_barrier(0);
      load_gradients(after);
      lds_barrier();
      advance(chunk, next);
    }
    if (live != 0) finish(0, true);
  }
  // steps past the row's end
  const uint32_t end = min(d.time - start, d.chunks * kChunk);
  for (uint32_t t = (length <= start ? 0 : length - start) + 4 * wave + g; t < end; t += 32) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (column_of(c) < d.values) dvalues[t * value_stride + column_of(c)] = static_cast<T>(0.0f);
  }
  if (a.to == nullptr || !holds) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint32_t k = key_at(r);
    if (k >= d.keys) continue;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (column_of(c) < d.values)
        a.to[state_at + static_cast<uint64_t>(k) * d.values + column_of(c)] = ds[c][r];
  }
}

constexpr int kColumns = 32;  // of values that the products take at a time: a pair of slabs

template <typename T, int KT>
struct Products {
  // of a pair of slabs the forward's state and errors, the state's gradient and x, as they were
  // stored: tiles of 16 keys, then of 16 steps
  struct Pair {
    operand<T> kept[2 * KT + 4][64], back[2 * KT + 4][64];
  };
  union {
    Pair pairs[2];
    // then the chunk's keys and queries and the matrices over them; past a row's 64 columns what is
    // not to be written
    struct {
      RowTile<T, KT> keys, queries;
      alignas(32) T one[kChunk][kChunk + 8], one_t[kChunk][kChunk + 8], two[kChunk][kChunk + 8];
    };
    // and the results' rows
    alignas(16) float rows[kChunk][32 * KT + 4];
  };
  double sums[kChunk];
  float rows_at[kChunk], columns_at[4][kChunk], before[kChunk], errors[kChunk], across[4];
};

// A block per chunk and key head, its value heads in turn (Shared: more than one, whose sums take 64
// registers more); a wave 16 of the steps.  Rows and columns
// are numbered by index_of, so that a wave's values of keys and queries beside its results are those
// of the operands that it multiplies them with.
template <typename T, int KT, bool Whole, bool WholeValues, bool Shared>
__global__ __launch_bounds__(256, sizeof(T) == 2 && !Shared ? 2 : 1) void delta_backward_products_kernel(
    Args<T> a) {
  using Op = operand<T>;
  using Pair = typename Products<T, KT>::Pair;
  __shared__ Products<T, KT> m;
  const Dims &d = a.d;
  const oxh::BlockTile tile = oxh::xcd_block();
  const uint32_t chunk = tile.x, kh = tile.y, b = tile.z;
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = w >> 1;
  const uint32_t row = threadIdx.x >> 2, part = threadIdx.x & 3;  // of the results' rows
  const uint64_t stride = static_cast<uint64_t>(d.key_heads) * d.keys;
  const uint64_t value_stride = static_cast<uint64_t>(d.heads) * d.values;
  f32x8 sums_q[Shared ? KT : 1] = {}, sums_k[Shared ? KT : 1] = {};
  const Place first(d, chunk, kh * d.group, b);
  const uint32_t held = min(d.time - first.begin, static_cast<uint32_t>(kChunk)), rows = first.rows;
  const RowPart<T, KT, Whole> brings(threadIdx.x, static_cast<uint32_t>(stride * sizeof(T)), d.keys);
  const uint32_t t_row = index_of(w, n), t_read = rows == 0 ? 0 : min(t_row, rows - 1);
  const uint64_t to_keys = first.key_row * d.keys + row * stride;
  for (uint32_t turn = 0; turn < (Shared ? d.group : 1); ++turn) {
    const uint32_t h = kh * d.group + turn;
    const Place at(d, chunk, h, b);
    if (rows == 0) {
      if (threadIdx.x < held) {
        const uint64_t to = at.value_row + static_cast<uint64_t>(threadIdx.x) * d.heads;
        a.dgate[to] = a.dwrite[to] = static_cast<T>(0.0f);
      }
      continue;
    }
    const char *block = a.heads + at.head_chunk(d) * Back<T>::bytes(KT, a.pairs);
    const char *gates = block + Back<T>::gates;
    const uint64_t value_at = at.value_row * d.values + t_read * value_stride;
    const char *saved = a.saved + ((static_cast<uint64_t>(b) * d.heads + h) * a.all + d.first + chunk) *
                                      a.pairs * Back<T>::pair(KT);
    f32x4 one[4] = {}, two[4] = {}, q1[2 * KT] = {}, k1[2 * KT] = {}, k2[2 * KT] = {};
    float across = 0.0f, errors = 0.0f;  // <dS, S0>, and of this lane's row e x
    Op out_next;
    auto fetch = [&](uint32_t i, Pair &to) {
      const char *kept = saved + i * Back<T>::pair(KT);
      const char *back = block + Back<T>::pairs + i * Back<T>::pair(KT);
      constexpr int kPieces = Back<T>::pair(KT) / 1024;
#pragma unroll
      for (int q = 0; q < (kPieces + 3) / 4; ++q) {
        const uint32_t p = 4 * q + w;
        if (kPieces % 4 != 0 && p >= kPieces) continue;
        copy_16(kept + p * 1024 + 16 * lane, reinterpret_cast<char *>(&to.kept[0][0]) + p * 1024);
        copy_16(back + p * 1024 + 16 * lane, reinterpret_cast<char *>(&to.back[0][0]) + p * 1024);
      }
      out_next = load_row<T, WholeValues>(a.gradient + value_at, kColumns * i + 8 * g, d.values);
    };
    lds_barrier();  // the rows of the head before are read
    fetch(0, m.pairs[0]);
    if (threadIdx.x < kChunk) {
      // the sums of the decay again, as the first kernel formed them
      const uint64_t from = at.value_row + static_cast<uint64_t>(min(lane, rows - 1)) * d.heads;
      double sum = lane < rows ? log_sigmoid(widen(a.gate[from])) : 0.0f;
#pragma unroll
      for (int i = 1; i < 64; i *= 2) {
        const double before = __shfl_up(sum, i);
        if (lane >= static_cast<uint32_t>(i)) sum += before;
      }
      m.sums[lane] = sum;
    }
    for (uint32_t i = 0; i < a.pairs; ++i) {
      arrived();
      const Op out = t_row < rows ? out_next : Op{};
      if (i + 1 < a.pairs) fetch(i + 1, m.pairs[(i + 1) & 1]);
      const Pair &s = m.pairs[i & 1];
      const Op e = s.kept[2 * KT + w][lane], x = s.back[2 * KT + w][lane];
      Op others[4];
#pragma unroll
      for (int it = 0; it < 4; ++it) others[it] = s.kept[2 * KT + it][lane];
#pragma unroll
      for (int j = 0; j < 8; ++j) errors = fmaf(widen(e[j]), widen(x[j]), errors);
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        if ((it >> 1) > pair) continue;
        one[it] = product(out, others[it], one[it]);
        two[it] = product(x, others[it], two[it]);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        Op state[KT], gradient[KT];
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          state[k] = s.kept[half * KT + k][lane];
          gradient[k] = s.back[half * KT + k][lane];
        }
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const int to = half * KT + k;
          q1[to] = product(out, state[k], q1[to]);
          k1[to] = product(x, state[k], k1[to]);
          k2[to] = product(e, gradient[k], k2[to]);
        }
        // a quarter of the tiles each wave
#pragma unroll
        for (int k = 0; k < KT; ++k)
          if (static_cast<uint32_t>(half * KT + k) % 4 == w)
#pragma unroll
            for (int j = 0; j < 8; ++j) across = fmaf(widen(state[k][j]), widen(gradient[k][j]), across);
      }
    }
    // the chunk's keys and queries where the pairs were
    {
      typename RowPart<T, KT, Whole>::Values keys, queries;
      const uint32_t bytes = rows * static_cast<uint32_t>(stride * sizeof(T));
      brings.load(keys, buffer_of(a.key + at.key_row * d.keys, bytes), d.keys);
      brings.load(queries, buffer_of(a.query + at.key_row * d.keys, bytes), d.keys);
      lds_barrier();
      brings.store(m.keys, keys);
      brings.store(m.queries, queries);
      lds_barrier();
    }
    // q k' and k k' again, for what their pairs' decays are worth
    f32x4 qk[4] = {}, kk[4] = {};
#pragma unroll
    for (int s = 0; s < KT; ++s) {
      const Op q = m.queries.along(t_row, s, g), k = m.keys.along(t_row, s, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if ((i >> 1) > pair) continue;
        const Op other = m.keys.along(index_of(i, n), s, g);
        qk[i] = product(q, other, qk[i]);
        kk[i] = product(k, other, kk[i]);
      }
    }
    const uint32_t t0 = index_of(w, 4 * g);  // this lane's first row of the results
    const f32x4 since = load_at<f32x4>(gates + offsetof(Gates, since), t0 * 4);
    const f32x4 until = load_at<f32x4>(gates + offsetof(Gates, until), t0 * 4);
    const f32x4 write = load_at<f32x4>(gates + offsetof(Gates, write), t0 * 4);
    float beta[4];
#pragma unroll
    for (int it = 0; it < 4; ++it)
      beta[it] = load_at<float>(gates + offsetof(Gates, write), index_of(it, n) * 4);
    errors += __shfl_xor(errors, 16);
    errors += __shfl_xor(errors, 32);
    if (g == 0) m.errors[t_row] = errors;
    {
      float total[1] = {across};
      oxh::wave_sums_rows(total);
      if (lane == 0) m.across[w] = total[0];
    }
    f32x4 after = {}, before = {};  // H's rows first
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const uint32_t i = index_of(it, n);
      float down = 0.0f;  // and columns
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t t = t0 + r;
        // no decay between a step and a later one is asked for
        const float between = beta[it] * expf(static_cast<float>(i <= t ? m.sums[t] - m.sums[i] : 0.0));
        const float x = i <= t ? one[it][r] * between * d.scale : 0.0f;
        const float y = i < t ? -two[it][r] * write[r] * between : 0.0f;
        const float worth = (i < t ? x * qk[it][r] : 0.0f) + y * kk[it][r];
        m.one[t][i] = static_cast<T>(x);
        m.one_t[i][t] = static_cast<T>(x);
        // the pairs the other way round are another lane's
        m.two[t][i <= t ? i : kChunk] = static_cast<T>(y);
        m.two[i][i <= t ? t : kChunk] = static_cast<T>(y);
        after[r] += worth;
        down += worth;
      }
      down += __shfl_xor(down, 16);
      down += __shfl_xor(down, 32);
      if (g == 0) m.columns_at[w][i] = down;
    }
    lds_barrier();
    // the rows of this wave of both matrices and of the first one's transpose
    Op x[2], xt[2], y[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      x[s] = *reinterpret_cast<const Op *>(&m.one[t_row][32 * s + 8 * g]);
      xt[s] = *reinterpret_cast<const Op *>(&m.one_t[t_row][32 * s + 8 * g]);
      y[s] = *reinterpret_cast<const Op *>(&m.two[t_row][32 * s + 8 * g]);
    }
#pragma unroll
    for (int i = 0; i < 2 * KT; ++i) {
      q1[i] *= since * d.scale;
      k1[i] *= -since * write;
      k2[i] *= until * write;
      Op k[2], q[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        k[s] = m.keys.across(i, s, n, g);
        q[s] = m.queries.across(i, s, n, g);
      }
      // of the wave's own steps: a lane's four are half of its 8
      const Op own = pair == 0 ? k[0] : k[1], asked = pair == 0 ? q[0] : q[1];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float kr = widen(w & 1 ? own[4 + r] : own[r]), qr = widen(w & 1 ? asked[4 + r] : asked[r]);
        after[r] = fmaf(qr, q1[i][r], fmaf(kr, k1[i][r], after[r]));
        before[r] = fmaf(kr, k2[i][r], before[r]);
      }
      k1[i] += k2[i];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        q1[i] = product(x[s], k[s], q1[i]);
        k1[i] = product(y[s], k[s], k1[i]);
        k1[i] = product(xt[s], q[s], k1[i]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      after[r] = row_total(after[r]);
      before[r] = row_total(before[r]);
    }
    if (n == 0) {
      *reinterpret_cast<f32x4 *>(&m.rows_at[t0]) = after;
      *reinterpret_cast<f32x4 *>(&m.before[t0]) = before;
    }
    // the rows whole: each thread 8 keys at a time of its row, stored with the last head's
    auto rows_of = [&](const f32x4(&v)[2 * KT], f32x8(&sums)[Shared ? KT : 1], T *to) {
      lds_barrier();
#pragma unroll
      for (int i = 0; i < 2 * KT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) m.rows[t0 + r][index_of(i, n)] = v[i][r];
      lds_barrier();
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const uint32_t k = (part + 4 * i) * 8;
        const float *p = &m.rows[row][k];
        f32x8 own = join(*reinterpret_cast<const f32x4 *>(p), *reinterpret_cast<const f32x4 *>(p + 4));
        if constexpr (Shared) {
          sums[i] += own;
          if (turn + 1 < d.group) continue;
          own = sums[i];
        }
        if (row < held)
          store_row<T, Whole>(to + to_keys, k, d.keys, rounded<T>(row < rows ? own : f32x8{}));
      }
    };
    rows_of(q1, sums_q, a.dquery);
    rows_of(k1, sums_k, a.dkey);
    if (threadIdx.x < kChunk) {
      float later = m.rows_at[lane], earlier = m.before[lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) later -= m.columns_at[i][lane];
      const float own = earlier;
#pragma unroll
      for (int i = 1; i < 64; i *= 2) {
        const float x = __shfl_down(later, i), y = __shfl_up(earlier, i);
        if (lane + i < 64) later += x;
        if (lane >= static_cast<uint32_t>(i)) earlier += y;
      }
      if (lane < held) {
        const uint64_t to = at.value_row + static_cast<uint64_t>(lane) * d.heads;
        const bool live = lane < rows;
        const float beta = load_at<float>(gates + offsetof(Gates, write), lane * 4);
        const float whole = load_at<float>(gates + offsetof(Gates, since), (kChunk - 1) * 4);
        const float constant =
            whole * ((m.across[0] + m.across[1]) + (m.across[2] + m.across[3]));
        const float decay = later + (earlier - own) + constant;
        a.dgate[to] = static_cast<T>(live ? decay * sigmoid(-widen(a.gate[to])) : 0.0f);
        a.dwrite[to] =
            static_cast<T>(live ? m.errors[lane] * beta * sigmoid(-widen(a.write[to])) : 0.0f);
      }
    }
  }
  if (rows != 0 || row >= held) return;
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    store_row<T, Whole>(a.dquery + to_keys, (part + 4 * i) * 8, d.keys, Op{});
    store_row<T, Whole>(a.dkey + to_keys, (part + 4 * i) * 8, d.keys, Op{});
  }
}

template <typename T>
struct BackPlan {
  Plan p;
  bool two;  // slabs of a block of the scan, as the forward's
  uint64_t head_bytes, key_bytes, state_bytes;
  uint64_t bytes() const { return head_bytes + key_bytes + state_bytes; }
  explicit BackPlan(const oxh_delta_shape &s, float scale, const int32_t *lengths)
      : p(s, scale, lengths) {
    const uint64_t head = s.batch * s.heads * Back<T>::bytes(p.steps, pairs_of(s.value_dim));
    two = s.batch * s.heads * pairs_of(s.value_dim) >= oxh::kComputeUnits;
    const uint64_t key = two ? 0 : s.batch * s.key_heads * p.steps * 12 * kOperandBytes<T>;
    p.divide(head + key);
    head_bytes = round_up(p.segment * head, 256);
    key_bytes = round_up(p.segment * key, 256);
    state_bytes = p.segment < p.all ? round_up(p.state_elements(s) * 4, 256) : 0;
  }
};

template <typename T>
oxh_status backward(hipStream_t stream, const BackPlan<T> &plan, Args<T> a, const float *final,
                    float *initial, char *workspace) {
  a.heads = workspace;
  a.keys = plan.two ? nullptr : a.heads + plan.head_bytes;
  float *between = reinterpret_cast<float *>(a.heads + plan.head_bytes + plan.key_bytes);
  const Plan &p = plan.p;
  a.all = static_cast<uint32_t>(p.all);
  const uint64_t launches = (p.all + p.segment - 1) / p.segment;
  a.pairs = (p.d.slabs + 1) / 2;
  constexpr uint64_t kPack = 16 / sizeof(T);
  const bool keys16 = oxh::aligned16(a.query) && oxh::aligned16(a.key);
  const bool packed = p.d.values % kPack == 0 && p.d.keys % kPack == 0 && keys16 &&
                      oxh::aligned16(a.gradient) && oxh::aligned16(a.dvalue);
  for (uint64_t i = launches; i-- != 0;) {
    const uint64_t first = i * p.segment;
    a.d = p.d;
    a.d.first = static_cast<uint32_t>(first);
    a.d.chunks = static_cast<uint32_t>(std::min(p.segment, p.all - first));
    a.from = i + 1 == launches ? final : between;
    a.to = i == 0 ? initial : between;
    const Dims &d = a.d;
    with_keys(d.keys, d.keys % 32 == 0 && keys16, [&](auto steps, auto whole) {
      constexpr int KT = decltype(steps)::value;
      constexpr bool W = decltype(whole)::value;
      oxh::launch(delta_backward_prepare_kernel<T, KT, W>, dim3(d.chunks, d.heads, d.batch),
                  dim3(256), 0, stream, a);
      auto go = [&](auto columns, auto packs) {
        constexpr int C = decltype(columns)::value;
        oxh::launch(delta_backward_scan_kernel<T, KT, C, decltype(packs)::value>,
                    dim3(2 / C * a.pairs, d.heads, d.batch), dim3(512), 0, stream, a);
      };
      auto slabs = [&](auto packs) {
        if (plan.two) go(std::integral_constant<int, 2>(), packs);
        else go(std::integral_constant<int, 1>(), packs);
      };
      if (packed) slabs(std::true_type());
      else slabs(std::false_type());
      const dim3 grid(d.chunks, d.key_heads, d.batch);
      auto products = [&](auto values, auto shared) {
        oxh::launch(delta_backward_products_kernel<T, KT, W, decltype(values)::value,
                                                   decltype(shared)::value>,
                    grid, dim3(256), 0, stream, a);
      };
      auto by_group = [&](auto values) {
        if (d.group > 1) products(values, std::true_type());
        else products(values, std::false_type());
      };
      if (d.values % kColumns == 0) by_group(std::true_type());
      else by_group(std::false_type());
    });
    oxh_status st = oxh::launched("gated_delta_rule_backward");
    if (st != OXH_OK) return st;
  }
  return oxh::ok();
}

}  // namespace

extern "C" {

oxh_status oxh_gated_delta_rule_backward_workspace_size(int dtype, const oxh_delta_shape *shape,
                                                        uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  oxh_status st = check_shape(dtype, shape);
  if (st != OXH_OK) return st;
  *bytes = dtype == OXH_F32 ? BackPlan<float>(*shape, 1.0f, nullptr).bytes()
                            : BackPlan<bf16>(*shape, 1.0f, nullptr).bytes();
  return oxh::ok();
}

oxh_status oxh_gated_delta_rule_backward(
    oxh_stream stream, int dtype, const oxh_delta_shape *shape, float scale, const void *gradient,
    const void *query, const void *key, const void *value, const void *gate, const void *write,
    const void *saved, uint64_t saved_size, const float *final_state_gradient,
    const int32_t *lengths, void *query_gradient, void *key_gradient, void *value_gradient,
    void *gate_gradient, void *write_gradient, float *initial_state_gradient, void *workspace,
    uint64_t workspace_bytes) {
  oxh_status st = check_shape(dtype, shape);
  if (st != OXH_OK) return st;
  const oxh_delta_shape &s = *shape;
  OXH_REQUIRE(std::isfinite(scale), OXH_EXECUTION, "gated delta rule: scale must be finite");
  if (s.batch == 0) return oxh::ok();
  const Sizes z(dtype, s);
  uint64_t kept = 0, needed = 0;
  st = oxh_gated_delta_rule_saved_size(dtype, shape, &kept);
  if (st == OXH_OK) st = oxh_gated_delta_rule_backward_workspace_size(dtype, shape, &needed);
  if (st != OXH_OK) return st;
  Spans in = {{gradient, z.value, z.element}, {query, z.query, z.element},
              {key, z.query, z.element},      {value, z.value, z.element},
              {gate, z.gate, z.element},      {write, z.gate, z.element},
              {saved, kept, 16}};
  Spans out = {{query_gradient, z.query, z.element}, {key_gradient, z.query, z.element},
               {value_gradient, z.value, z.element}, {gate_gradient, z.gate, z.element},
               {write_gradient, z.gate, z.element},  {workspace, needed, 16}};
  for (const auto *list : {&in, &out})
    for (const Span &x : *list)
      OXH_REQUIRE(x.p != nullptr || x.bytes == 0, OXH_INVALID_SHAPE,
                  "gated delta rule backward: null pointer");
  OXH_REQUIRE(saved_size >= kept, OXH_INVALID_SHAPE,
              "gated delta rule backward: saved is too small");
  OXH_REQUIRE(workspace_bytes >= needed, OXH_INVALID_SHAPE,
              "gated delta rule backward: workspace too small");
  in.push_back({lengths, s.batch * 4, 4});
  // the initial state's gradient may be written over the final one's
  out.push_back({initial_state_gradient, z.state, 4});
  if (final_state_gradient != initial_state_gradient) in.push_back({final_state_gradient, z.state, 4});
  st = check_apart(in, out);
  if (st != OXH_OK) return st;
  hipStream_t on = oxh::as_stream(stream);
  if (s.time == 0) {
    if (initial_state_gradient == nullptr || initial_state_gradient == final_state_gradient)
      return oxh::ok();
    if (final_state_gradient == nullptr)
      return oxh_memset0_async(initial_state_gradient, z.state, stream);
    return oxh_memcpy_d2d_async(initial_state_gradient, final_state_gradient, z.state, stream);
  }
  auto run = [&](auto type) {
    using T = decltype(type);
    Args<T> a{};
    a.query = static_cast<const T *>(query);
    a.key = static_cast<const T *>(key);
    a.gate = static_cast<const T *>(gate);
    a.write = static_cast<const T *>(write);
    a.gradient = static_cast<const T *>(gradient);
    a.saved = static_cast<const char *>(saved);
    a.dquery = static_cast<T *>(query_gradient);
    a.dkey = static_cast<T *>(key_gradient);
    a.dvalue = static_cast<T *>(value_gradient);
    a.dgate = static_cast<T *>(gate_gradient);
    a.dwrite = static_cast<T *>(write_gradient);
    return backward<T>(on, BackPlan<T>(s, scale, lengths), a, final_state_gradient,
                       initial_state_gradient, static_cast<char *>(workspace));
  };
  return dtype == OXH_F32 ? run(float()) : run(bf16());
}

}  // extern "C"
