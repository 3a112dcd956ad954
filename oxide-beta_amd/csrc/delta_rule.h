// delta_rule.h -- the gated delta rule's tiles (internal to the library): shapes, operands of the
// matrix cores and where a call keeps them between its kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "common.h"
#include "row_norm.h"
#include "storage.h"

namespace oxh {
namespace delta {

using storage::bf16;

constexpr int kChunk = 64;  // steps of a chunk

struct Dims {
  uint32_t batch, time, key_heads, heads, keys, values;
  uint32_t group, slabs;       // value heads of a key head; slabs of 16 value columns
  uint32_t first, chunks;      // the chunks of this launch: [first, first + chunks)
  const int32_t *lengths;      // may be null
  float scale;
};

// Steps of batch row b.
__device__ __forceinline__ uint32_t length_of(const Dims &d, uint32_t b) {
  if (d.lengths == nullptr) return d.time;
  const int32_t n = d.lengths[b];
  return n <= 0 ? 0u : min(static_cast<uint32_t>(n), d.time);
}

// The matrix cores' 16 x 16 products take A as (row = lane % 16) and B as (column = lane % 16), both
// with 8 values of the summed axis per lane, and leave C as (column = lane % 16, rows = 4 per lane
// group of 16).  Which index of the summed axis a lane's values stand for is free as long as A and
// B agree, and which index a row of a tile stands for is free altogether.  With rows numbered as
// below, the C tiles 2 m and 2 m + 1 of a lane are its 8 consecutive indexes 32 m + 8 group + 0..7:
// the result of one product is the B operand of the next as it stands, in the same registers.
__device__ __forceinline__ uint32_t index_of(uint32_t tile, uint32_t row) {
  return 32 * (tile >> 1) + ((row >> 2) << 3) + ((tile & 1) << 2) + (row & 3);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

// 8 values of a lane.
template <typename T>
struct Operand;
template <>
struct Operand<bf16> {
  typedef bf16x8 type;
};
template <>
struct Operand<float> {
  typedef f32x8 type;
};
template <typename T>
using operand = typename Operand<T>::type;

// c + a b over 32 indexes.
__device__ __forceinline__ f32x4 product(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 product(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

template <typename T>
__device__ __forceinline__ operand<T> rounded(f32x8 v) {
  return __builtin_convertvector(v, operand<T>);
}
__device__ __forceinline__ f32x8 widened(bf16x8 v) { return __builtin_convertvector(v, f32x8); }
__device__ __forceinline__ f32x8 widened(f32x8 v) { return v; }
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 widened(bf16x4 v) { return __builtin_convertvector(v, f32x4); }
__device__ __forceinline__ f32x4 widened(f32x4 v) { return v; }

// A float32 operand as bfloat16 ones that add up to it: to 2^-17 of each value with two.
template <typename T, int Parts>
struct Split {
  operand<T> part[Parts];
  __device__ __forceinline__ explicit Split(f32x8 v) {
#pragma unroll
    for (int p = 0; p < Parts; ++p) {
      part[p] = rounded<T>(v);
      if (p + 1 < Parts) v -= widened(part[p]);
    }
  }
};
__device__ __forceinline__ f32x8 join(f32x4 low, f32x4 high) {
  return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A lane's load from `at` bytes behind an address that is the same for the wave (of memory, said so:
// a load that might be of shared memory would have to wait for all others).
template <typename V, int Align = alignof(V)>
__device__ __forceinline__ V load_at(const void *base, uint32_t at) {
  typedef V __attribute__((aligned(Align))) type;
  typedef __attribute__((address_space(1))) const type *pointer;
  return *(pointer)(reinterpret_cast<const char *>(base) + at);
}

// 8 consecutive values of a row of `count`, from place `at` on; those past its end are 0.
template <typename T, bool Whole>
__device__ __forceinline__ operand<T> load_row(const T *row, uint32_t at, uint32_t count) {
  if (Whole || at + 8 <= count) {
    operand<T> v;
    if constexpr (sizeof(T) == 2) {
      v = storage::raw<T, 8>(row + at);
    } else {
      const auto low = storage::raw<T, 4>(row + at), high = storage::raw<T, 4>(row + at + 4);
      v = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return v;
  }
  operand<T> v = {};
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i)
    if (at + i < count) v[i] = row[at + i];
  return v;
}

template <typename T, bool Whole>
__device__ __forceinline__ void store_row(T *row, uint32_t at, uint32_t count, operand<T> v) {
  if (Whole || at + 8 <= count) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<typename storage::Pack<T, 8>::type *>(row + at) = v;
    } else {
      typedef typename storage::Pack<T, 4>::type half;
      *reinterpret_cast<half *>(row + at) = __builtin_shufflevector(v, v, 0, 1, 2, 3);
      *reinterpret_cast<half *>(row + at + 4) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
    }
    return;
  }
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i)
    if (at + i < count) row[at + i] = v[i];
}

// Where the operands of a chunk lie, in units of a wave's operand (64 lanes, each its 8 values in
// one piece).  Triangles of 64 x 64 are six operands: (tile, step) = (0,0) (1,0) (2,0) (2,1) (3,0)
// (3,1) for the lower one, (0,0) (0,1) (1,0) (1,1) (2,1) (3,1) for its transpose.
constexpr int kTriangle = 6;
__device__ __forceinline__ int lower_place(int tile, int step) {
  return tile < 2 ? tile : 2 * tile - 2 + step;
}
__device__ __forceinline__ int upper_place(int tile, int step) {
  return tile < 2 ? 2 * tile + step : tile + 2;
}

// Operands of two slabs of 16 columns in shared memory, the first one's from `first` on, the other's
// `apart` behind: each lane a column, 8 rows.  From there the operand of their transpose, for sums
// over the columns: a lane one of the 16 rows that index_of numbers for tile `half`, 8 of the 32
// columns.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
// Mixed: the slabs' lanes are the pair's columns in the order of index_of.
template <bool Mixed>
__device__ __forceinline__ bf16x8 turned(const bf16x8 *first, uint32_t apart, int half, uint32_t n,
                                         uint32_t g) {
  // 16 lanes read four columns' 16 rows, four of them each, and get a row of it
  s16x4 v[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t at = Mixed ? e * apart + 4 * g : (g >> 1) * apart + 8 * (g & 1) + 4 * e;
    v[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(
        reinterpret_cast<const s16x4 *>(first + at + (n & 3) * 16 + (n >> 2)) + half));
  }
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
}
template <bool Mixed>
__device__ __forceinline__ f32x8 turned(const f32x8 *first, uint32_t apart, int half, uint32_t n,
                                        uint32_t g) {
  f32x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t at = Mixed ? (i >> 2) * apart + 4 * g + (i & 3)
                              : (g >> 1) * apart + 8 * (g & 1) + i;
    v[i] = reinterpret_cast<const float *>(first + at + (n >> 2) * 16)[4 * half + (n & 3)];
  }
  return v;
}

// 16 bytes of each lane from memory to `to` + 16 * lane in shared memory, without a stop in
// registers; they are there behind arrived().
__device__ __forceinline__ void copy_16(const void *from, void *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
__device__ __forceinline__ void arrived() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Where the block's waves see each other's shared memory; loads from memory stay on their way.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Stores to places of a buffer that begins anywhere (the same for the wave); those past its bytes,
// kNowhere among them, do not happen.
constexpr uint32_t kNowhere = 0xFFFFFFF0u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void *p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, static_cast<int>(bytes), 0x00020000);
}
// A lane's load from place `at` of a buffer, `further` (the same for the wave) behind it; 0 past the
// buffer's end.
template <typename V>
__device__ __forceinline__ V load_from(__amdgpu_buffer_rsrc_t from, uint32_t at, uint32_t further) {
  if constexpr (sizeof(V) == 2) {
    return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b16(from, at, further, 0));
  } else if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b32(from, at, further, 0));
  } else if constexpr (sizeof(V) == 16) {
    return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(from, at, further, 0));
  } else {
    struct Halves {
      f32x4 low, high;
    };
    const Halves x = {load_from<f32x4>(from, at, further), load_from<f32x4>(from, at + 16, further)};
    return __builtin_bit_cast(V, x);
  }
}
template <typename V>
__device__ __forceinline__ void store_to(__amdgpu_buffer_rsrc_t to, uint32_t at, V v) {
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  if constexpr (sizeof(V) == 2) {
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), to, at, 0, 0);
  } else if constexpr (sizeof(V) == 4) {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), to, at, 0, 0);
  } else if constexpr (sizeof(V) == 8) {
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), to, at, 0, 0);
  } else if constexpr (sizeof(V) == 16) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to, at, 0, 0);
  } else {
    struct Halves {
      u32x4 low, high;
    };
    const Halves x = __builtin_bit_cast(Halves, v);
    __builtin_amdgcn_raw_buffer_store_b128(x.low, to, at, 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(x.high, to, at == kNowhere ? at : at + 16, 0, 0);
  }
}

// 64 rows of a head's keys or queries in shared memory, as they lie in memory: pieces of 16 bytes,
// those of a row in an order by the row that lets 16 rows' same pieces come from different banks.
// KT 0: none.
template <typename T, int KT>
struct RowTile {
  static constexpr uint32_t per = 16 / sizeof(T), pieces = 32 * (KT == 0 ? 1 : KT) / per,
                            span = KT == 3 ? 4 * pieces / 3 : pieces;
  f32x4 piece[KT == 0 ? 1 : kChunk * span];
  static __device__ __forceinline__ uint32_t place(uint32_t row, uint32_t piece) {
    const uint32_t order = (row & 3) | ((row >> 1) & 12);
    return row * span + (piece ^ (order * (sizeof(T) / 2) & (span - 1)));
  }
  // The operand of a sum over the keys: a lane its row, 8 keys of step s.
  __device__ __forceinline__ operand<T> along(uint32_t row, int s, uint32_t g) const {
    return *reinterpret_cast<const operand<T> *>(&piece[place(row, (4 * s + g) * 8 / per)]);
  }
  // The operand of a sum over the rows: a lane its key of a tile of 16, 8 rows of step s.
  __device__ __forceinline__ operand<T> across(uint32_t tile, int s, uint32_t n, uint32_t g) const {
    if constexpr (sizeof(T) == 2) {
      s16x4 v[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x4 *at = &piece[place(32 * s + 8 * g + 4 * e + (n >> 2), 4 * (tile >> 1) + (n & 3))];
        v[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4 *)(reinterpret_cast<const s16x4 *>(at) + (tile & 1)));
      }
      return __builtin_bit_cast(
          operand<T>, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      operand<T> v;
      const uint32_t key = index_of(tile, n);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = piece[place(32 * s + 8 * g + i, key >> 2)][key & 3];
      return v;
    }
  }
};

// The part of such a tile that one of 256 threads brings: by way of its registers, a load ahead.
// Packed: 16 bytes at a time, else its elements. Rows past a chunk's and keys past the last are 0.
template <typename T, int KT, bool Packed>
struct RowPart {
  using Tile = RowTile<T, KT>;
  static constexpr int count = KT == 0 ? 1 : kChunk * Tile::pieces / 256;
  struct Values {
    f32x4 v[count];
  };
  uint32_t at[count], to[count];
  __device__ __forceinline__ RowPart(uint32_t thread, uint32_t row_bytes, uint32_t keys) {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const uint32_t id = 256 * i + thread, row = id / Tile::pieces, piece = id % Tile::pieces;
      at[i] = piece * Tile::per < keys ? row * row_bytes + piece * 16 : kNowhere;
      to[i] = Tile::place(row, piece);
    }
  }
  __device__ __forceinline__ void load(Values &x, __amdgpu_buffer_rsrc_t from,
                                       uint32_t keys) const {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      if constexpr (Packed) {
        x.v[i] = load_from<f32x4>(from, at[i], 0);
      } else {
        typedef T part __attribute__((ext_vector_type(Tile::per)));
        const uint32_t piece = (256 * i + threadIdx.x % 256) % Tile::pieces;
        part y;
#pragma unroll
        for (uint32_t e = 0; e < Tile::per; ++e)
          y[e] = load_from<T>(from, piece * Tile::per + e < keys ? at[i] + e * sizeof(T) : kNowhere,
                              0);
        x.v[i] = __builtin_bit_cast(f32x4, y);
      }
    }
  }
  __device__ __forceinline__ void store(Tile &tile, const Values &x) const {
#pragma unroll
    for (int i = 0; i < count; ++i) tile.piece[to[i]] = x.v[i];
  }
};

// exp of the decay's sums of a chunk: from its start (`since`), to its end (`until`), and b.
struct Gates {
  float since[kChunk], until[kChunk], write[kChunk];
};

template <typename T>
constexpr uint64_t kOperandBytes = 64 * 8 * sizeof(T);

template <typename T, int P>
struct Chunk {  // per value head
  static constexpr uint64_t gates = 0, system = sizeof(Gates),
                            within = system + kTriangle * P * kOperandBytes<T>,
                            bytes = within + kTriangle * kOperandBytes<T>;
};

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }
// log sigmoid(x), not below -100: exp of it is 0 beside any other decay, and sums of it stay sums.
__device__ __forceinline__ float log_sigmoid(float x) {
  const float v = fminf(x, 0.0f) - log1pf(expf(-fabsf(x)));
  return v < -100.0f ? -100.0f : x != x ? x : v;
}

// A chunk of a head: its rows, and where it lies among the rows' heads and the launch's chunks.
struct Place {
  uint32_t chunk, head, batch, key_head, begin, rows;
  uint64_t row0, key_row, value_row;
  __device__ __forceinline__ Place(const Dims &d, uint32_t chunk_, uint32_t head_, uint32_t batch_)
      : chunk(chunk_), head(head_), batch(batch_), key_head(head_ / d.group) {
    begin = (d.first + chunk) * kChunk;
    const uint32_t length = length_of(d, batch);
    rows = begin < length ? min(length - begin, static_cast<uint32_t>(kChunk)) : 0;
    row0 = static_cast<uint64_t>(batch) * d.time + begin;
    key_row = row0 * d.key_heads + key_head;  // times keys: the first row of its key head
    value_row = row0 * d.heads + head;        // times values
  }
  __device__ __forceinline__ uint64_t head_chunk(const Dims &d) const {
    return (static_cast<uint64_t>(batch) * d.heads + head) * d.chunks + chunk;
  }
  __device__ __forceinline__ uint64_t key_chunk(const Dims &d) const {
    return (static_cast<uint64_t>(batch) * d.key_heads + key_head) * d.chunks + chunk;
  }
};

template <typename T, int KT>
struct System {
  float mat[kChunk][68];  // A, then N
  float inverse[4][16][20];
  double sums[kChunk];
  float betas[kChunk];
  alignas(32) T tile[kChunk][32 * KT + 8];
  __device__ __forceinline__ float between(uint32_t t, uint32_t i) const {
    return expf(static_cast<float>(sums[t] - sums[i]));
  }
  __device__ __forceinline__ operand<T> key_row(uint32_t row, int step, uint32_t g) const {
    return *reinterpret_cast<const operand<T> *>(&tile[row][32 * step + 8 * g]);
  }
};

// The chunk's rows of a head of keys (or queries).  Steps past the row's length repeat its last one
// with a decay of 1 and b = 0: nothing of them reaches a step of the row or the state.
template <typename T, int KT, bool Whole>
__device__ __forceinline__ void load_tile(T (&tile)[kChunk][32 * KT + 8], const Dims &d,
                                          const Place &at, const T *from) {
  const uint32_t r = threadIdx.x >> 2, part = threadIdx.x & 3;
  const T *row = from + (at.key_row + static_cast<uint64_t>(min(r, at.rows - 1)) * d.key_heads) * d.keys;
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    const uint32_t k = (part + 4 * i) * 8;
    *reinterpret_cast<operand<T> *>(&tile[r][k]) = load_row<T, Whole>(row, k, d.keys);
  }
}

// Its transpose as operands: a lane its key index, 8 steps.
template <typename T, int KT>
__device__ __forceinline__ void store_transposed(const T (&tile)[kChunk][32 * KT + 8],
                                                 operand<T> *to) {
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  for (int p = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); p < 4 * KT; p += 4) {
    const uint32_t at = index_of(p >> 1, n), from = 32 * (p & 1) + 8 * g;
    operand<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = tile[from + i][at];
    to[p * 64 + lane] = v;
  }
}

// Leaves N of a chunk in m.mat (rows and columns in order), its keys in m.tile and its gates in
// memory.  The last three of the block's four waves run `meanwhile` beside the first one's
// inversions (keys and sums of the decay are there by then).
template <typename T, int KT, bool Whole, typename Meanwhile>
__device__ __forceinline__ void solve(System<T, KT> &m, const Dims &d, const Place &at,
                                      const T *key, const T *gate, const T *write, Gates *gates,
                                      Meanwhile meanwhile) {
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  load_tile<T, KT, Whole>(m.tile, d, at, key);
  if (wave == 0) {
    const uint64_t row = at.value_row + static_cast<uint64_t>(min(lane, at.rows - 1)) * d.heads;
    const bool own = lane < at.rows;
    const float decay = own ? log_sigmoid(storage::widen(gate[row])) : 0.0f;
    const float beta = own ? sigmoid(storage::widen(write[row])) : 0.0f;
    double sum = decay;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
      const double before = __shfl_up(sum, i);
      if (lane >= static_cast<uint32_t>(i)) sum += before;
    }
    const double last = __shfl(sum, 63);
    m.sums[lane] = sum;
    m.betas[lane] = beta;
    gates->since[lane] = expf(static_cast<float>(sum));
    gates->until[lane] = expf(static_cast<float>(last - sum));
    gates->write[lane] = beta;
  }
  __syncthreads();

  // A: this wave's 16 steps against those of the tiles up to the end of their half
  for (uint32_t it = 0; it <= (wave | 1); ++it) {
    f32x4 acc = {};
    if (it <= wave) {
#pragma unroll
      for (int s = 0; s < KT; ++s)
        acc = product(m.key_row(16 * wave + n, s, g), m.key_row(16 * it + n, s, g), acc);
    }
    const uint32_t i = 16 * it + n;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t t = 16 * wave + 4 * g + r;
      m.mat[t][i] = i < t ? acc[r] * m.between(t, i) : 0.0f;
    }
  }
  __syncthreads();

  if (wave == 0) {
    // (1 + A b) of each diagonal block of 16, inverted: a lane its column n of block g
    float x[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      x[t] = static_cast<uint32_t>(t) == n ? 1.0f : 0.0f;
#pragma unroll
      for (int i = 0; i < t; ++i)
        x[t] = fmaf(-m.mat[16 * g + t][16 * g + i] * m.betas[16 * g + i], x[i], x[t]);
      m.inverse[g][t][n] = x[t];
    }
  } else {
    meanwhile();
  }
  __syncthreads();

  // N by block rows, a wave its 16 columns: N_j = (1 + A b)_jj^-1 (A_j - sum over i < j of
  // (A b)_ji N_i), the blocks above as they left the matrix cores
  f32x4 solved[4];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    if (j < wave) continue;
    f32x4 acc;
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] = m.mat[16 * j + 4 * g + r][16 * wave + n];
#pragma unroll
    for (uint32_t i = 0; i < j; ++i) {
      if (i < wave) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t k = 16 * i + 4 * g + r;
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(-m.mat[16 * j + n][k] * m.betas[k],
                                                   solved[i][r], acc, 0, 0, 0);
      }
    }
    solved[j] = f32x4{};
#pragma unroll
    for (int r = 0; r < 4; ++r)
      solved[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(m.inverse[j][n][4 * g + r], acc[r],
                                                       solved[j], 0, 0, 0);
  }
  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    if (j < wave) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) m.mat[16 * j + 4 * g + r][16 * wave + n] = solved[j][r];
  }
  __syncthreads();
}

// ------------------------------------------------------------------------------------ host side

constexpr uint64_t kMostKeys = 128;
// Bytes of operands that a call prepares before it scans their chunks: what the last-level cache
// holds beside the tensors (1 x 32768 x 16 heads: 861 us, 844 with 64 MiB, 954 with 400; 8 x 2048 x 16
// heads with gradients 654, 647 and 636).
constexpr uint64_t kPrepared = 192ull << 20;

inline uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// What the forward leaves the backward of a chunk and a pair of slabs: its state (tiles of 16 keys)
// and its errors (tiles of 16 steps) as operands of sums over the values.
inline uint64_t pairs_of(uint64_t values) { return (values + 31) / 32; }

struct Plan {
  Dims d;
  uint64_t all, segment, steps;  // chunks; those prepared at a time; 32 keys each
  Plan(const oxh_delta_shape &s, float scale, const int32_t *lengths)
      : d{static_cast<uint32_t>(s.batch), static_cast<uint32_t>(s.time),
          static_cast<uint32_t>(s.key_heads), static_cast<uint32_t>(s.heads),
          static_cast<uint32_t>(s.key_dim), static_cast<uint32_t>(s.value_dim),
          static_cast<uint32_t>(s.heads / s.key_heads),
          static_cast<uint32_t>((s.value_dim + 15) / 16), 0, 0, lengths, scale},
        all((s.time + kChunk - 1) / kChunk), segment(0), steps(round_up(s.key_dim, 32) / 32) {}
  // Takes as many chunks at a time as `bytes` each allow, in equal parts.
  void divide(uint64_t bytes) {
    const uint64_t most = std::max<uint64_t>(1, kPrepared / std::max<uint64_t>(1, bytes));
    const uint64_t parts = (all + most - 1) / most;
    segment = parts == 0 ? 0 : (all + parts - 1) / parts;
  }
  uint64_t state_elements(const oxh_delta_shape &s) const {
    return s.batch * s.heads * s.key_dim * s.value_dim;
  }
};

// Calls run(32 keys each, whether rows are loaded without a look at their end).
template <typename Run>
void with_keys(uint64_t keys, bool packed, Run run) {
  auto whole = [&](auto steps) {
    if (packed) run(steps, std::true_type());
    else run(steps, std::false_type());
  };
  if (keys <= 32) whole(std::integral_constant<int, 1>());
  else if (keys <= 64) whole(std::integral_constant<int, 2>());
  else if (keys <= 96) whole(std::integral_constant<int, 3>());
  else whole(std::integral_constant<int, 4>());
}

inline oxh_status check_shape(int dtype, const oxh_delta_shape *s) {
  OXH_REQUIRE(s != nullptr, OXH_INVALID_SHAPE, "gated delta rule: shape is null");
  OXH_REQUIRE(storage::valid(dtype), OXH_INVALID_SHAPE,
              "gated delta rule: dtype is neither OXH_F32 nor OXH_BF16");
  OXH_REQUIRE(s->key_dim >= 1 && s->key_dim <= kMostKeys, OXH_INVALID_SHAPE,
              "gated delta rule: key_dim must be 1..128");
  OXH_REQUIRE(s->value_dim >= 1 && s->value_dim <= 4096, OXH_INVALID_SHAPE,
              "gated delta rule: value_dim must be 1..4096");
  OXH_REQUIRE(s->key_heads >= 1 && s->heads >= 1 && s->heads % s->key_heads == 0 &&
                  s->heads <= 65535,
              OXH_INVALID_SHAPE, "gated delta rule: heads must be a multiple of key_heads, at "
                                 "most 65535");
  OXH_REQUIRE(s->batch <= 65535, OXH_INVALID_SHAPE, "gated delta rule: batch above 65535");
  OXH_REQUIRE(s->time < (1ull << 31) - kChunk, OXH_INVALID_SHAPE,
              "gated delta rule: too many steps");
  // a chunk's rows lie within 32 bits of each other
  OXH_REQUIRE(s->heads * s->value_dim < (1ull << 24), OXH_INVALID_SHAPE,
              "gated delta rule: heads * value_dim must be below 2^24");
  // one launch numbers its threads with 32 bits
  const uint64_t heads = s->batch * s->heads;
  OXH_REQUIRE(heads * std::max<uint64_t>((s->time + kChunk - 1) / kChunk, 1) <= (1ull << 23) &&
                  heads * ((s->value_dim + 15) / 16) <= (1ull << 24),
              OXH_INVALID_SHAPE, "gated delta rule: more heads and steps than one call takes");
  return ok();
}

// Bytes of a call's tensors.
struct Sizes {
  uint64_t element, query, value, gate, state;
  Sizes(int dtype, const oxh_delta_shape &s)
      : element(storage::bytes_of(dtype)),
        query(s.batch * s.time * s.key_heads * s.key_dim * element),
        value(s.batch * s.time * s.heads * s.value_dim * element),
        gate(s.batch * s.time * s.heads * element),
        state(s.batch * s.heads * s.key_dim * s.value_dim * 4) {}
};

struct Span {
  const void *p;
  uint64_t bytes, align;
};
// A call's operands or outputs: no more than this many, and no memory that could be refused.
struct Spans {
  Span span[12];
  int count = 0;
  Spans(std::initializer_list<Span> from) {
    for (const Span &x : from) push_back(x);
  }
  void push_back(const Span &x) { span[count++] = x; }
  const Span *begin() const { return span; }
  const Span *end() const { return span + count; }
};
// Aligned to their elements; no output over an operand or another output.
inline oxh_status check_apart(const Spans &in, const Spans &out) {
  for (const auto *list : {&in, &out})
    for (const Span &x : *list)
      OXH_REQUIRE(row_norm::aligned_to(x.p, x.align), OXH_INVALID_SHAPE,
                  "gated delta rule: a pointer is not aligned to its elements");
  for (const Span &o : out) {
    if (o.p == nullptr) continue;
    for (const Span &i : in)
      OXH_REQUIRE(i.p == nullptr || !any_overlap(o.p, o.bytes, i.p, i.bytes),
                  OXH_INVALID_SHAPE,
                  "gated delta rule: an output, saved or the workspace overlaps an operand");
    for (const Span *k = out.begin(); k != &o; ++k)
      OXH_REQUIRE(k->p == nullptr || !any_overlap(o.p, o.bytes, k->p, k->bytes),
                  OXH_INVALID_SHAPE, "gated delta rule: two outputs overlap");
  }
  return ok();
}

}  // namespace delta
}  // namespace oxh
