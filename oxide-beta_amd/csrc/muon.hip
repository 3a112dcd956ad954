// muon.hip -- orthogonalisation of matrices by Newton-Schulz products, and the optimizer step that
// moves each weight matrix by its orthogonalised momentum.
//
//   M = mu M + G;  V = G + mu M (Nesterov) or M;  X = V / (|V|_F + epsilon)
//   rounds times:  A = X X';  B = b A + c A A;  X = a X + B X,   (a, b, c) = (3.4445, -4.775, 2.0315)
//   W = W - lr (wd W + sqrt(max(1, rows / columns)) X)
//
// with X transposed where rows > columns, so A is the smaller Gram matrix.  Every singular value s
// of X goes to a s + b s^3 + c s^5 per round, which takes (0, 1] into about [0.7, 1.21] within five
// rounds (K. Jordan's quintic, 2024).  No counterpart in the reference, whose one optimizer is
// AdamW.
//
// Products.  An operand value v is held as two float16 numbers, hi = f16(S v) and lo =
// f16(S v - hi) with S = 2^14, which together keep 22 bits of it; a product is summed as hi hi' +
// hi lo' + lo hi' in float32 on the matrix cores (the omitted lo lo' is below 2^-22 of the
// product).  No entry overflows: |X| and |A| stay below 1.5 and |B| below 2.9 for |X|_F <= 1.  The
// term a X is taken from a float32 copy of X: the error of X itself is what grows from round to
// round (by up to a = 3.4445 in the directions of small singular values), that of the products
// stays relative to B X.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "common.h"

namespace {

typedef _Float16 f16;
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kScale = 16384.0f, kUnscale = 1.0f / (16384.0f * 16384.0f);

// A matrix of a launch group.  Short = min(rows, columns) and Long are the sides of X; ps and pl
// the same rounded up to the tile, the padding zero throughout.  `scratch` holds, in order:
//   x [ps][pl] float32; xs: X in halves; xt0, xt1: X' in halves (one is read while the other is
//   written); ga [ps][ps] float32: A; gs, bs: A and B in halves; the norm's partial sums.
// Halves of a matrix with k columns: per row, blocks of 32 columns, 32 hi then 32 lo.
struct Matrix {
  const float *gradient;
  float *momentum;  // null: orthogonalize
  float *target;    // the parameter, or the output
  char *scratch;
  uint32_t rows, columns, ps, pl;
  uint32_t first_block;  // of this launch
  float scale;
};
constexpr int kGroup = 32;
struct Group {
  Matrix m[kGroup];
  uint32_t count, blocks;
  float momentum, lr, decay, epsilon;
  int nesterov;
};

constexpr uint32_t kNormParts = 256;

struct Layout {
  uint64_t x, xs, xt0, xt1, ga, gs, bs, parts, total;
};
__host__ __device__ inline Layout layout_of(uint64_t ps, uint64_t pl) {
  const uint64_t wide = ps * pl * 4, square = ps * ps * 4;
  Layout l;
  l.x = 0;
  l.xs = wide;
  l.xt0 = 2 * wide;
  l.xt1 = 3 * wide;
  l.ga = 4 * wide;
  l.gs = l.ga + square;
  l.bs = l.gs + square;
  l.parts = l.bs + square;
  l.total = l.parts + kNormParts * 4;
  return l;
}

__device__ __forceinline__ const Matrix &matrix_of(const Group &g, uint32_t block) {
  uint32_t j = 0;
  while (j + 1 < g.count && g.m[j + 1].first_block <= block) ++j;  // block-uniform
  return g.m[j];
}

// V of one element; M (already updated) where there is a momentum.
__device__ __forceinline__ float direction(const Group &g, const Matrix &m, uint64_t i) {
  const float grad = m.gradient[i];
  if (m.momentum == nullptr) return grad;
  const float mom = m.momentum[i];
  return g.nesterov ? grad + g.momentum * mom : mom;
}

// M = mu M + G, and the partial sums of V^2: block p of a matrix's kNormParts (or fewer, the
// others then 0) takes every parts-th run of 256 elements.
__global__ __launch_bounds__(256) void muon_norm_kernel(Group g) {
  __shared__ float wave[4];
  const Matrix &m = matrix_of(g, blockIdx.x);
  const uint32_t part = blockIdx.x - m.first_block;
  const uint64_t n = static_cast<uint64_t>(m.rows) * m.columns;
  float sum = 0.0f;
  for (uint64_t i = part * 256ull + threadIdx.x; i < n; i += kNormParts * 256ull) {
    if (m.momentum != nullptr) m.momentum[i] = g.momentum * m.momentum[i] + m.gradient[i];
    const float v = direction(g, m, i);
    sum = fmaf(v, v, sum);
  }
  float one[1] = {sum};
  oxh::wave_sums_rows(one);
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = one[0];
  __syncthreads();
  if (threadIdx.x == 0) {
    float *parts = reinterpret_cast<float *>(m.scratch + layout_of(m.ps, m.pl).parts);
    parts[part] = (wave[0] + wave[1]) + (wave[2] + wave[3]);
  }
}

__device__ __forceinline__ void halves_of(float v, f16 &hi, f16 &lo) {
  const float s = v * kScale;
  hi = static_cast<f16>(s);
  lo = static_cast<f16>(s - static_cast<float>(hi));
}
// Offset of (row, column) in halves of k columns; lo is 32 further.
__device__ __forceinline__ uint64_t halves_at(uint32_t row, uint32_t column, uint32_t k) {
  return (static_cast<uint64_t>(row) * k + (column & ~31u)) * 2 + (column & 31u);
}

// X = V / (|V| + epsilon) in its three forms, a 32 x 32 tile per block.
__global__ __launch_bounds__(256) void muon_start_kernel(Group g) {
  __shared__ float tile[32][33];
  __shared__ float wave[4];
  const Matrix &m = matrix_of(g, blockIdx.x);
  const Layout l = layout_of(m.ps, m.pl);
  const float *parts = reinterpret_cast<const float *>(m.scratch + l.parts);
  float one[1] = {parts[threadIdx.x]};
  oxh::wave_sums_rows(one);
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = one[0];
  __syncthreads();
  const float norm = sqrtf((wave[0] + wave[1]) + (wave[2] + wave[3])) + g.epsilon;
  const uint32_t tiles = m.pl / 32, b = blockIdx.x - m.first_block;
  const uint32_t i0 = b / tiles * 32, j0 = b % tiles * 32;
  const bool tall = m.rows > m.columns;
  const uint32_t s = tall ? m.columns : m.rows, n = tall ? m.rows : m.columns;
  const uint32_t tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  // read along the rows of V
  for (uint32_t k = ty; k < 32; k += 8) {
    const uint32_t i = tall ? i0 + tx : i0 + k, j = tall ? j0 + k : j0 + tx;
    float v = 0.0f;
    if (i < s && j < n)
      v = direction(g, m, tall ? static_cast<uint64_t>(j) * m.columns + i
                               : static_cast<uint64_t>(i) * m.columns + j) / norm;
    if (tall) tile[tx][k] = v;
    else tile[k][tx] = v;
  }
  __syncthreads();
  float *x = reinterpret_cast<float *>(m.scratch + l.x);
  f16 *xs = reinterpret_cast<f16 *>(m.scratch + l.xs);
  f16 *xt = reinterpret_cast<f16 *>(m.scratch + l.xt0);
  for (uint32_t k = ty; k < 32; k += 8) {
    f16 hi, lo;
    const float v = tile[k][tx], t = tile[tx][k];
    x[static_cast<uint64_t>(i0 + k) * m.pl + j0 + tx] = v;
    halves_of(v, hi, lo);
    f16 *p = xs + halves_at(i0 + k, j0 + tx, m.pl);
    p[0] = hi;
    p[32] = lo;
    halves_of(t, hi, lo);
    f16 *q = xt + halves_at(j0 + k, i0 + tx, m.ps);
    q[0] = hi;
    q[32] = lo;
  }
}

enum class Step { Gram, Poly, Apply, Last };

// One of a round's three products, a tile of 2 x 2 waves by T x T blocks of 32 x 32 per block of
// threads.  Both operands are halves with the summed index along the rows.  A and B are
// symmetric: only tiles on and below the diagonal are summed, the others are their mirrors.
template <Step S, int T>
__global__ __launch_bounds__(256) void muon_product_kernel(Group g, int odd) {
  constexpr int kTile = 64 * T;
  // per operand row: 32 summed values, 8 pieces of 16 bytes (hi 0..3, lo 4..7), each at its place
  // exclusive-or the row's low bits, so that 8 rows' same piece lie in 8 different bank groups
  __shared__ __attribute__((aligned(16))) char stage[2][kTile * 128];
  const Matrix &m = matrix_of(g, blockIdx.x);
  const Layout l = layout_of(m.ps, m.pl);
  const uint32_t b = blockIdx.x - m.first_block;
  uint32_t ti, tj;
  if constexpr (S == Step::Gram || S == Step::Poly) {
    ti = static_cast<uint32_t>((sqrtf(8.0f * b + 1.0f) - 1.0f) * 0.5f);
    while (ti * (ti + 1) / 2 > b) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= b) ++ti;
    tj = b - ti * (ti + 1) / 2;
  } else {
    const uint32_t across = m.pl / kTile;
    ti = b / across;
    tj = b % across;
  }
  const uint32_t k_total = S == Step::Gram ? m.pl : m.ps;
  const f16 *pa, *pb;
  f16 *gs = reinterpret_cast<f16 *>(m.scratch + l.gs), *bs = reinterpret_cast<f16 *>(m.scratch + l.bs);
  f16 *xs = reinterpret_cast<f16 *>(m.scratch + l.xs);
  f16 *from = reinterpret_cast<f16 *>(m.scratch + (odd ? l.xt1 : l.xt0));
  f16 *to = reinterpret_cast<f16 *>(m.scratch + (odd ? l.xt0 : l.xt1));
  if constexpr (S == Step::Gram) pa = pb = xs;
  else if constexpr (S == Step::Poly) pa = pb = gs;
  else pa = bs, pb = from;
  const char *sa = reinterpret_cast<const char *>(pa) + static_cast<uint64_t>(ti) * kTile * k_total * 4;
  const char *sb = reinterpret_cast<const char *>(pb) + static_cast<uint64_t>(tj) * kTile * k_total * 4;

  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t wi = wave >> 1, wj = wave & 1;
  constexpr int kLoads = kTile * 8 / 256;  // 16-byte pieces per thread per operand
  uint4 ra[kLoads], rb[kLoads];
  auto fetch = [&](uint32_t k) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t piece = i * 256 + threadIdx.x, row = piece >> 3, c = piece & 7;
      const uint64_t at = static_cast<uint64_t>(row) * k_total * 4 + k * 4 + c * 16;
      ra[i] = *reinterpret_cast<const uint4 *>(sa + at);
      rb[i] = *reinterpret_cast<const uint4 *>(sb + at);
    }
  };
  f32x16 acc[T][T];
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  fetch(0);
  for (uint32_t k = 0; k < k_total; k += 32) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t piece = i * 256 + threadIdx.x, row = piece >> 3, c = piece & 7;
      *reinterpret_cast<uint4 *>(stage[0] + row * 128 + ((c ^ (row & 7)) * 16)) = ra[i];
      *reinterpret_cast<uint4 *>(stage[1] + row * 128 + ((c ^ (row & 7)) * 16)) = rb[i];
    }
    __syncthreads();
    if (k + 32 < k_total) fetch(k + 32);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      f16x8 ah[T], al[T], bh[T], bl[T];
      const uint32_t c = half * 2 + (lane >> 5);
#pragma unroll
      for (int i = 0; i < T; ++i) {
        const uint32_t row = (wi * T + i) * 32 + (lane & 31);
        ah[i] = *reinterpret_cast<f16x8 *>(stage[0] + row * 128 + ((c ^ (row & 7)) * 16));
        al[i] = *reinterpret_cast<f16x8 *>(stage[0] + row * 128 + (((c + 4) ^ (row & 7)) * 16));
      }
#pragma unroll
      for (int j = 0; j < T; ++j) {
        const uint32_t row = (wj * T + j) * 32 + (lane & 31);
        bh[j] = *reinterpret_cast<f16x8 *>(stage[1] + row * 128 + ((c ^ (row & 7)) * 16));
        bl[j] = *reinterpret_cast<f16x8 *>(stage[1] + row * 128 + (((c + 4) ^ (row & 7)) * 16));
      }
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < T; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], acc[i][j], 0, 0, 0);
        }
    }
  }

  // Lane l holds column l % 32 and, in register r, row 8 (r / 4) + 4 (l / 32) + r % 4 of each
  // 32 x 32 block: four consecutive rows per register quad.
  float *x = reinterpret_cast<float *>(m.scratch + l.x), *ga = reinterpret_cast<float *>(m.scratch + l.ga);
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const uint32_t column = tj * kTile + (wj * T + j) * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t row = ti * kTile + (wi * T + i) * 32 + 8 * q + 4 * (lane >> 5);
        float v[4];
        f16x4 hi, lo;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = acc[i][j][4 * q + r] * kUnscale;
          if constexpr (S == Step::Poly)
            v[r] = kB * ga[static_cast<uint64_t>(row + r) * m.ps + column] + kC * v[r];
          if constexpr (S == Step::Apply || S == Step::Last)
            v[r] += kA * x[static_cast<uint64_t>(row + r) * m.pl + column];
          f16 h, w;
          halves_of(v[r], h, w);
          hi[r] = h;
          lo[r] = w;
        }
        if constexpr (S == Step::Last) {
          const bool tall = m.rows > m.columns;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t wr = tall ? column : row + r, wc = tall ? row + r : column;
            if (wr >= m.rows || wc >= m.columns) continue;
            float *t = m.target + static_cast<uint64_t>(wr) * m.columns + wc;
            *t = m.momentum == nullptr ? v[r] : *t - g.lr * (g.decay * *t + m.scale * v[r]);
          }
        } else {
          // along the rows, and the transposed entry, four of a row at once
          f16 *straight = S == Step::Gram ? gs : S == Step::Poly ? bs : xs;
          f16 *mirror = S == Step::Apply ? to : straight;
          const uint32_t k_straight = S == Step::Apply ? m.pl : m.ps;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f16 *p = straight + halves_at(row + r, column, k_straight);
            p[0] = hi[r];
            p[32] = lo[r];
            if constexpr (S == Step::Apply)
              x[static_cast<uint64_t>(row + r) * m.pl + column] = v[r];
            if constexpr (S == Step::Gram)
              ga[static_cast<uint64_t>(row + r) * m.ps + column] = v[r];
          }
          if (S == Step::Apply || ti != tj) {
            f16 *p = mirror + halves_at(column, row, m.ps);
            *reinterpret_cast<f16x4 *>(p) = hi;
            *reinterpret_cast<f16x4 *>(p + 32) = lo;
            if constexpr (S == Step::Gram)
              *reinterpret_cast<float4 *>(ga + static_cast<uint64_t>(column) * m.ps + row) =
                  make_float4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    }
}

// ---------------------------------------------------------------- host

struct Item {
  const float *gradient;
  float *momentum, *target;
  uint64_t rows, columns;
};

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// Tile side for a launch group: 128 where its products then still have a tile for every compute
// unit, else 64.
uint32_t tile_of(const Item *items, size_t count) {
  uint64_t tiles = 0;
  for (size_t i = 0; i < count; ++i) {
    const uint64_t s = round_up(std::min(items[i].rows, items[i].columns), 128) / 128;
    tiles += s * (s + 1) / 2;
  }
  return tiles >= oxh::kComputeUnits ? 128 : 64;
}

uint64_t scratch_of(const Item *items, size_t count) {
  const uint32_t tile = tile_of(items, count);
  uint64_t total = 0;
  for (size_t i = 0; i < count; ++i)
    total += round_up(layout_of(round_up(std::min(items[i].rows, items[i].columns), tile),
                                round_up(std::max(items[i].rows, items[i].columns), tile))
                          .total,
                      256);
  return total;
}

uint64_t scratch_of_all(const std::vector<Item> &items) {
  uint64_t most = 256;
  for (size_t at = 0; at < items.size(); at += kGroup)
    most = std::max(most, scratch_of(&items[at], std::min<size_t>(kGroup, items.size() - at)));
  return most;
}

template <Step S>
oxh_status product(hipStream_t stream, Group &g, uint32_t tile, int odd, const char *what) {
  g.blocks = 0;
  for (uint32_t i = 0; i < g.count; ++i) {
    const uint32_t s = g.m[i].ps / tile, l = g.m[i].pl / tile;
    g.m[i].first_block = g.blocks;
    g.blocks += S == Step::Gram || S == Step::Poly ? s * (s + 1) / 2 : s * l;
  }
  if (tile == 128)
    oxh::launch(muon_product_kernel<S, 2>, dim3(g.blocks), dim3(256), 0, stream, g, odd);
  else
    oxh::launch(muon_product_kernel<S, 1>, dim3(g.blocks), dim3(256), 0, stream, g, odd);
  return oxh::launched(what);
}

oxh_status run_group(hipStream_t stream, Group &g, uint32_t tile, uint32_t rounds) {
  g.blocks = 0;
  for (uint32_t i = 0; i < g.count; ++i) g.m[i].first_block = g.blocks, g.blocks += kNormParts;
  oxh::launch(muon_norm_kernel, dim3(g.blocks), dim3(256), 0, stream, g);
  oxh_status st = oxh::launched("muon_norm");
  if (st != OXH_OK) return st;
  g.blocks = 0;
  for (uint32_t i = 0; i < g.count; ++i) {
    g.m[i].first_block = g.blocks;
    g.blocks += (g.m[i].ps / 32) * (g.m[i].pl / 32);
  }
  oxh::launch(muon_start_kernel, dim3(g.blocks), dim3(256), 0, stream, g);
  st = oxh::launched("muon_start");
  for (uint32_t r = 0; r < rounds && st == OXH_OK; ++r) {
    st = product<Step::Gram>(stream, g, tile, r & 1, "muon_gram");
    if (st == OXH_OK) st = product<Step::Poly>(stream, g, tile, r & 1, "muon_poly");
    if (st != OXH_OK) return st;
    st = r + 1 < rounds ? product<Step::Apply>(stream, g, tile, r & 1, "muon_apply")
                        : product<Step::Last>(stream, g, tile, r & 1, "muon_last");
  }
  return st;
}

struct Hyper {
  float lr, decay, momentum, epsilon;
  bool nesterov;
};

oxh_status run_all(hipStream_t stream, const std::vector<Item> &items, const Hyper &h,
                   uint32_t rounds, char *workspace) {
  for (size_t at = 0; at < items.size(); at += kGroup) {
    const size_t count = std::min<size_t>(kGroup, items.size() - at);
    const uint32_t tile = tile_of(&items[at], count);
    Group g{};
    g.count = static_cast<uint32_t>(count);
    g.momentum = h.momentum;
    g.lr = h.lr;
    g.decay = h.decay;
    g.epsilon = h.epsilon;
    g.nesterov = h.nesterov ? 1 : 0;
    uint64_t offset = 0;
    for (size_t i = 0; i < count; ++i) {
      const Item &it = items[at + i];
      Matrix &m = g.m[i];
      m.gradient = it.gradient;
      m.momentum = it.momentum;
      m.target = it.target;
      m.scratch = workspace + offset;
      m.rows = static_cast<uint32_t>(it.rows);
      m.columns = static_cast<uint32_t>(it.columns);
      m.ps = static_cast<uint32_t>(round_up(std::min(it.rows, it.columns), tile));
      m.pl = static_cast<uint32_t>(round_up(std::max(it.rows, it.columns), tile));
      m.scale = std::sqrt(std::max(1.0f, static_cast<float>(it.rows) /
                                             static_cast<float>(it.columns)));
      offset += round_up(layout_of(m.ps, m.pl).total, 256);
    }
    oxh_status st = run_group(stream, g, tile, rounds);
    if (st != OXH_OK) return st;
  }
  return oxh::ok();
}

// Sides whose tiles and block counts fit 32 bits.
oxh_status check_sides(uint64_t rows, uint64_t columns) {
  OXH_REQUIRE(rows >= 1 && columns >= 1, OXH_INVALID_SHAPE, "muon: an empty matrix");
  OXH_REQUIRE(std::min(rows, columns) <= (1u << 16) && std::max(rows, columns) <= (1u << 20) &&
                  columns * rows <= (1ull << 32),
              OXH_INVALID_SHAPE, "muon: a matrix side or size is too large");
  return oxh::ok();
}

oxh_status items_of(const oxh_muon_tensor *tensors, uint32_t count, std::vector<Item> &items) {
  OXH_REQUIRE(tensors != nullptr || count == 0, OXH_INVALID_SHAPE, "muon: null table");
  for (uint32_t i = 0; i < count; ++i) {
    const oxh_muon_tensor &t = tensors[i];
    oxh_status st = check_sides(t.rows, t.columns);
    if (st != OXH_OK) return st;
    items.push_back({t.gradient, t.momentum, t.parameter, t.rows, t.columns});
  }
  return oxh::ok();
}

bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

oxh_status check_workspace(uint64_t needed, const void *workspace, uint64_t bytes) {
  OXH_REQUIRE(workspace != nullptr && bytes >= needed && oxh::aligned16(workspace),
              OXH_INVALID_SHAPE, "muon: workspace too small or misaligned");
  return oxh::ok();
}

}  // namespace

extern "C" {

oxh_status oxh_orthogonalize_workspace_size(uint64_t count, uint64_t rows, uint64_t columns,
                                            uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  *bytes = 256;
  if (count == 0) return oxh::ok();
  oxh_status st = check_sides(rows, columns);
  if (st != OXH_OK) return st;
  OXH_REQUIRE(count <= 65536, OXH_INVALID_SHAPE, "orthogonalize: too many matrices");
  *bytes = scratch_of_all(std::vector<Item>(count, Item{nullptr, nullptr, nullptr, rows, columns}));
  return oxh::ok();
}

oxh_status oxh_orthogonalize(oxh_stream stream, uint64_t count, uint64_t rows, uint64_t columns,
                             uint32_t rounds, float epsilon, const float *input, float *output,
                             void *workspace, uint64_t workspace_bytes) {
  uint64_t needed = 0;
  oxh_status st = oxh_orthogonalize_workspace_size(count, rows, columns, &needed);
  if (st != OXH_OK) return st;
  OXH_REQUIRE(rounds >= 1 && rounds <= 64, OXH_INVALID_SHAPE,
              "orthogonalize: rounds outside 1..64");
  OXH_REQUIRE(std::isfinite(epsilon) && epsilon > 0.0f, OXH_EXECUTION,
              "orthogonalize: epsilon must be positive and finite");
  if (count == 0) return oxh::ok();
  OXH_REQUIRE(input != nullptr && output != nullptr && aligned4(input) && aligned4(output),
              OXH_INVALID_SHAPE, "orthogonalize: null or misaligned pointer");
  st = check_workspace(needed, workspace, workspace_bytes);
  if (st != OXH_OK) return st;
  const uint64_t bytes = count * rows * columns * 4;
  OXH_REQUIRE(!oxh::any_overlap(input, bytes, output, bytes) &&
                  !oxh::any_overlap(workspace, needed, input, bytes) &&
                  !oxh::any_overlap(workspace, needed, output, bytes),
              OXH_INVALID_SHAPE, "orthogonalize: buffers overlap");
  std::vector<Item> items;
  for (uint64_t i = 0; i < count; ++i)
    items.push_back({input + i * rows * columns, nullptr, output + i * rows * columns, rows,
                     columns});
  return run_all(oxh::as_stream(stream), items, {0.0f, 0.0f, 0.0f, epsilon, false}, rounds,
                 static_cast<char *>(workspace));
}

oxh_status oxh_muon_workspace_size(const oxh_muon_tensor *tensors, uint32_t count,
                                   uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  std::vector<Item> items;
  oxh_status st = items_of(tensors, count, items);
  if (st != OXH_OK) return st;
  *bytes = scratch_of_all(items);
  return oxh::ok();
}

oxh_status oxh_muon_multi_tensor(oxh_stream stream, float learning_rate, float weight_decay,
                                 float momentum, int nesterov, float epsilon, uint32_t rounds,
                                 const oxh_muon_tensor *tensors, uint32_t count, void *workspace,
                                 uint64_t workspace_bytes) {
  OXH_REQUIRE(std::isfinite(learning_rate) && std::isfinite(weight_decay) &&
                  std::isfinite(momentum),
              OXH_INVALID_SHAPE, "muon: hyper-parameters must be finite");
  OXH_REQUIRE(rounds >= 1 && rounds <= 64, OXH_INVALID_SHAPE, "muon: rounds outside 1..64");
  OXH_REQUIRE(std::isfinite(epsilon) && epsilon > 0.0f, OXH_EXECUTION,
              "muon: epsilon must be positive and finite");
  std::vector<Item> items;
  oxh_status st = items_of(tensors, count, items);
  if (st != OXH_OK) return st;
  if (count == 0) return oxh::ok();
  const uint64_t needed = scratch_of_all(items);
  st = check_workspace(needed, workspace, workspace_bytes);
  if (st != OXH_OK) return st;
  // every written range against every other range: sorted by address, neighbours may not meet
  // unless both are read only
  struct Range {
    uintptr_t begin, end;
    bool written;
  };
  std::vector<Range> ranges;
  auto add = [&](const void *p, uint64_t bytes, bool written) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    ranges.push_back({at, at + bytes, written});
  };
  add(workspace, needed, true);
  for (const Item &it : items) {
    OXH_REQUIRE(it.gradient != nullptr && it.momentum != nullptr && it.target != nullptr &&
                    aligned4(it.gradient) && aligned4(it.momentum) && aligned4(it.target),
                OXH_INVALID_SHAPE, "muon: null or misaligned pointer");
    const uint64_t bytes = it.rows * it.columns * 4;
    add(it.gradient, bytes, false);
    add(it.momentum, bytes, true);
    add(it.target, bytes, true);
  }
  std::sort(ranges.begin(), ranges.end(),
            [](const Range &a, const Range &b) { return a.begin < b.begin; });
  uintptr_t end_any = 0, end_written = 0;
  for (const Range &r : ranges) {
    OXH_REQUIRE(r.begin >= end_written && (!r.written || r.begin >= end_any), OXH_INVALID_SHAPE,
                "muon: a buffer that is written overlaps another");
    end_any = std::max(end_any, r.end);
    if (r.written) end_written = std::max(end_written, r.end);
  }
  return run_all(oxh::as_stream(stream), items,
                 {learning_rate, weight_decay, momentum, epsilon, nesterov != 0}, rounds,
                 static_cast<char *>(workspace));
}

}  // extern "C"
