// muon.hip -- orthogonalisation of matrices by Newton-Schulz products, and the optimizer step that
// moves each weight matrix by its orthogonalised momentum.
//
//   M = mu M + G;  V = G + mu M (Nesterov) or M;  X = V / (|V|_F + epsilon)
//   rounds times:  A = X X';  B = b A + c A A;  X = a X + B X
//   (a, b, c) = (3.4445, -4.775, 2.0315)
//   W = W - lr (wd W + sqrt(max(1, rows / columns)) X)
//
// with X transposed where rows > columns, so A is the smaller Gram matrix.  Every singular value s
// of X goes to a s + b s^3 + c s^5 per round, which takes (0, 1] into about [0.7, 1.21] within five
// rounds (K. Jordan's quintic, 2024).  No counterpart in the reference, whose one optimizer is
// AdamW.
//
// Products.  An operand value v is held as two float16 numbers, hi = f16(S v) and lo =
// f16(S v - hi) with S = 2^14, which together keep 22 bits of it from |v| = 2^-17 on, and below an
// absolute 2^-39; a product is summed as hi hi' + hi lo' + lo hi' in float32 on the matrix cores
// (the omitted lo lo' is below 2^-22 of the product).  No entry overflows: |X| and |A| stay below
// 1.5 and |B| below 2.9 for |X|_F <= 1.
//
// The absolute part is of the largest rows' scale, not a small row's own: in a matrix of 1000 x 1280
// in which some rows are 1e-6 of the others, entries start near 2^-30, and those rows of the result
// are 1.2e-3 of themselves off (1.3e-6 of the whole result, as any).  A scale for each row would not
// do: A A and B X sum over rows.
//
// X itself is kept as halves too, and a X and b A are added to the summed products from them.  The
// error of X grows from round to round (by up to a = 3.4445 in the directions of small singular
// values): with 22 bits in place of float32's 24 the result of five rounds on 1000 x 1280 matrices
// of rank 125 is 9.5e-6 of its norm off, with a float32 copy beside the halves 8.6e-6, and the
// copies made B X of 12 x 512 x 2048 move 250 MB in place of 100.  B + a I as the factor would
// save the addition, but then a X has the error of a factor's halves: 3.0e-5.
//
// Bound.  Three matrix instructions for each of the plain product's, half of A and of A A: 5 (s^2 n
// + s^3 + 2 s^2 n) multiply-adds for X of s x n.  Large matrices come near the matrix cores' rate:
// 4096 x 4096 in 4.1 ms, 335 TFLOP/s or 1005 of float16 (a library's largest float16 products reach
// 1092 here); 12 x 512 x 2048 in 602 us (three launches a round, which leave the cores a part of
// the time), and 1000 x 1280 in 223 us, where each of 15 products takes 12 to 18 us: 136 tiles on
// 256 compute units, each a chain of loads.  Short sides of up to 128 take fewer launches: one for
// a matrix that a compute unit holds, seven in slabs of its columns.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <string>
#include <type_traits>
#include <vector>

#include "common.h"

namespace {

typedef _Float16 f16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kScale = 16384.0f, kUnscale = 1.0f / (16384.0f * 16384.0f);
// A small X keeps its bits down to |V|_F = 2^-32 epsilon; 8^30 and S^2 stay within float32.
constexpr int kMostShift = 30;

// A matrix of a launch group.  Short = min(rows, columns) and Long are the sides of X; ps and pl
// the same rounded up to the tile, the padding zero throughout.  `scratch` holds, in order:
//   xt0, xt1 [pl][ps]: X' in halves (one is read while the other is written); gs, bs [ps][ps]: A
//   and B in halves; the norm's partial sums; |X|_F before the first round.
// Halves of a matrix with k columns: per row, blocks of 32 columns, 32 hi then 32 lo.
struct Matrix {
  const float *gradient;
  float *momentum;  // null: orthogonalize
  float *target;    // the parameter, or the output
  char *scratch;
  uint64_t parts;  // offset of the norm's partial sums
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
  uint64_t xt0, xt1, gs, bs, parts, length, total;
};
__host__ __device__ inline Layout layout_of(uint64_t ps, uint64_t pl) {
  const uint64_t wide = ps * pl * 4, square = ps * ps * 4;
  Layout l;
  l.xt0 = 0;
  l.xt1 = wide;
  l.gs = 2 * wide;
  l.bs = l.gs + square;
  l.parts = l.bs + square;
  l.length = l.parts + kNormParts * 4;
  l.total = l.length + 4;
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

// M = mu M + G, and the partial sums of V^2: block p of a matrix's kNormParts takes every parts-th
// run of a block's elements, four per thread where `packed` (the pointers are 16-byte aligned; the
// last n % 4 elements are the first block's).
constexpr int kNormThreads = 1024;
__global__ __launch_bounds__(kNormThreads) void muon_norm_kernel(Group g) {
  __shared__ float wave[kNormThreads / 64];
  const Matrix &m = matrix_of(g, blockIdx.x);
  const uint32_t part = blockIdx.x - m.first_block;
  const uint64_t n = static_cast<uint64_t>(m.rows) * m.columns;
  const bool packed = ((reinterpret_cast<uintptr_t>(m.gradient) |
                        reinterpret_cast<uintptr_t>(m.momentum)) & 15u) == 0;
  float sum = 0.0f;
  auto take = [&](float grad, float &mom) {
    float v = grad;
    if (m.momentum != nullptr) {
      mom = g.momentum * mom + grad;
      v = g.nesterov ? grad + g.momentum * mom : mom;
    }
    sum = fmaf(v, v, sum);
  };
  const uint64_t packs = packed ? n / 4 : 0;
  const f32x4 *gradient = reinterpret_cast<const f32x4 *>(m.gradient);
  f32x4 *momentum = reinterpret_cast<f32x4 *>(m.momentum);
#pragma unroll 4
  for (uint64_t i = part * static_cast<uint64_t>(kNormThreads) + threadIdx.x; i < packs;
       i += static_cast<uint64_t>(kNormParts) * kNormThreads) {
    f32x4 mom{0.0f, 0.0f, 0.0f, 0.0f};
    const f32x4 grad = gradient[i];
    if (momentum != nullptr) mom = momentum[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float one = mom[e];
      take(grad[e], one);
      mom[e] = one;
    }
    if (momentum != nullptr) momentum[i] = mom;
  }
  for (uint64_t i = packs * 4 + part * static_cast<uint64_t>(kNormThreads) + threadIdx.x; i < n;
       i += static_cast<uint64_t>(kNormParts) * kNormThreads) {
    float mom = m.momentum != nullptr ? m.momentum[i] : 0.0f;
    take(m.gradient[i], mom);
    if (m.momentum != nullptr) m.momentum[i] = mom;
  }
  float one[1] = {sum};
  oxh::wave_sums_rows(one);
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = one[0];
  __syncthreads();
  if (threadIdx.x == 0) {
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kNormThreads / 64; ++w) total += wave[w];
    reinterpret_cast<float *>(m.scratch + m.parts)[part] = total;
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

// Both halves in one word, hi below.
__device__ __forceinline__ uint32_t halves_word(float v) {
  f16 hi, lo;
  halves_of(v, hi, lo);
  return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, hi)) |
         static_cast<uint32_t>(__builtin_bit_cast(uint16_t, lo)) << 16;
}
// 16 consecutive such words to their place in halves.
__device__ __forceinline__ void store_line(const uint32_t *words, f16 *to) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const u32x4 w0 = *reinterpret_cast<const u32x4 *>(words + 8 * e);
    const u32x4 w1 = *reinterpret_cast<const u32x4 *>(words + 8 * e + 4);
    u32x4 hi, lo;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      hi[k] = (w0[2 * k] & 0xFFFFu) | w0[2 * k + 1] << 16;
      lo[k] = w0[2 * k] >> 16 | (w0[2 * k + 1] & 0xFFFF0000u);
      hi[2 + k] = (w1[2 * k] & 0xFFFFu) | w1[2 * k + 1] << 16;
      lo[2 + k] = w1[2 * k] >> 16 | (w1[2 * k + 1] & 0xFFFF0000u);
    }
    *reinterpret_cast<u32x4 *>(to + 8 * e) = hi;
    *reinterpret_cast<u32x4 *>(to + 8 * e + 32) = lo;
  }
}

// A small X is kept as 2^k X, and A and B as 4^k A and 4^k B, so that their entries do not fall below
// the halves' range: k is 0 unless |X|_F = |V|_F / (|V|_F + epsilon) is below 1/4, and then leaves
// `length`, which bounds X, between 1/4 and 1/2 (4^k B below 1.3).  A round takes a singular value of
// up to 1.5 to at most 3.4445 times itself, so before round r the length is |X|_F 3.4445^r.
__device__ __forceinline__ int shift_of(float length) {
  return min(max(-1 - __builtin_amdgcn_frexp_expf(length), 0), kMostShift);
}

// X' = (V / (|V| + epsilon))' in halves, a 32 x 32 tile per block.
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
  const float size = sqrtf((wave[0] + wave[1]) + (wave[2] + wave[3]));
  const float norm = size + g.epsilon, length = size / norm;
  const float scale = ldexpf(1.0f, shift_of(length));
  if (blockIdx.x == m.first_block && threadIdx.x == 0)
    *reinterpret_cast<float *>(m.scratch + l.length) = length;
  const uint32_t tiles = m.pl / 32, b = blockIdx.x - m.first_block;
  const uint32_t i0 = b / tiles * 32, j0 = b % tiles * 32;
  const bool tall = m.rows > m.columns;
  const uint32_t s = tall ? m.columns : m.rows, n = tall ? m.rows : m.columns;
  const uint32_t tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  // read along the rows of V
#pragma unroll
  for (uint32_t k = ty; k < 32; k += 8) {
    const uint32_t i = tall ? i0 + tx : i0 + k, j = tall ? j0 + k : j0 + tx;
    float v = 0.0f;
    if (i < s && j < n)
      v = direction(g, m, tall ? static_cast<uint64_t>(j) * m.columns + i
                               : static_cast<uint64_t>(i) * m.columns + j) / norm * scale;
    if (tall) tile[tx][k] = v;
    else tile[k][tx] = v;
  }
  __syncthreads();
  // 16 bytes of a row per thread: eight hi or lo
  f16 *xt = reinterpret_cast<f16 *>(m.scratch + l.xt0);
  const uint32_t row = threadIdx.x >> 3, piece = threadIdx.x & 7, first = (piece & 3) * 8;
  f16x8 turned;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f16 hi, lo;
    halves_of(tile[first + e][row], hi, lo);
    turned[e] = piece < 4 ? hi : lo;
  }
  *reinterpret_cast<f16x8 *>(xt + halves_at(j0 + row, i0, m.ps) + piece * 8) = turned;
}

__device__ __forceinline__ f16x8 join(s16x4 a, s16x4 b) {
  return __builtin_bit_cast(f16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

enum class Step { Gram, Poly, Apply, Last };

// The block shapes of the products: Groups times WM x WN waves of TM x TN blocks of 32 x 32, and
// K blocks of 32 summed values per stage, of whose 2 K halves each group takes every Groups-th.
// Direct loads (from memory straight to shared memory, one stage ahead) need fewer registers than
// loads through registers (two stages ahead), so that two blocks share a compute unit where there
// are two: 12 x 512 x 2048, of 128 and 64, 604 us and 687.  One block alone waits longer for them:
// 4096 x 4096, of 192, 4.63 ms and 4.02; 1000 x 1280, of 64, 270 us and 230, and 222 with four
// groups; 1091 x 87, of 32, 108 us and 98.
template <int WM_, int WN_, int TM_, int TN_, int K_, int Groups_, bool Direct_>
struct Shape {
  static constexpr bool Direct = Direct_;
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, K = K_, Groups = Groups_;
  static constexpr int threads = WM * WN * Groups * 64, tile = WM * TM * 32;
  static_assert(WM * TM == WN * TN && 2 * K % Groups == 0, "square tiles, whole halves");
};
using Wide = Shape<2, 2, 3, 3, 1, 2, false>;    // 192 x 192
using Medium = Shape<2, 2, 2, 2, 1, 2, true>;   // 128 x 128
using Small = Shape<2, 2, 1, 1, 2, 2, true>;    // 64 x 64
using Few = Shape<2, 2, 1, 1, 2, 4, false>;     // 64 x 64, where no compute unit has two
using Tiny = Shape<1, 1, 1, 1, 4, 8, false>;    // 32 x 32

// The tile of index b among rows x columns tiles, or (Symmetric) among those on and below the
// diagonal of rows x rows: bands of four tile rows, each taken column by column, so that the run
// of tiles that one XCD computes shares few operand rows in its L2.
struct Tile {
  uint32_t row, column;
};
template <bool Symmetric>
__device__ __forceinline__ Tile tile_at(uint32_t b, uint32_t rows, uint32_t columns) {
  uint32_t band, at;
  if constexpr (Symmetric) {
    // a band's full columns and its triangle: 16 band + 10 tiles, 8 band^2 + 2 band before it
    band = static_cast<uint32_t>((sqrtf(8.0f * b + 1.0f) - 1.0f) * 0.125f);
    while (8 * band * band + 2 * band > b) --band;
    while (8 * (band + 1) * (band + 1) + 2 * (band + 1) <= b) ++band;
    at = b - (8 * band * band + 2 * band);
  } else {
    band = b / (4 * columns);
    at = b - band * 4 * columns;
  }
  const uint32_t height = min(4u, rows - 4 * band);
  const uint32_t full = Symmetric ? height * (4 * band + 1) : ~0u;
  if (at < full) return {4 * band + at % height, at / height};
  at -= full;  // the triangle's columns right of its first: height - 1, height - 2, ... tiles
  uint32_t column = 1;
  while (at >= height - column) at -= height - column, ++column;
  return {4 * band + column + at, 4 * band + column};
}

// The lane's four consecutive rows, in each quad q (rows 8 q + 4 (lane / 32) ..), of a column whose
// 32 values lie at `line` as halves: each lane loads 16-byte pieces 2 h and 2 h + 1 of hi and lo, h
// = lane / 32, and exchanges with lane ^ 32 the half of each that the other's rows are.
__device__ __forceinline__ void column_of(const f16 *line, uint32_t lane, f32x4 (&value)[4]) {
  u32x4 hi[2], lo[2];
  const f16 *p = line + (lane >> 5) * 16;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    hi[e] = *reinterpret_cast<const u32x4 *>(p + 8 * e);
    lo[e] = *reinterpret_cast<const u32x4 *>(p + 32 + 8 * e);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const auto h = __builtin_amdgcn_permlane32_swap(hi[e][k], hi[e][k + 2], false, false);
      const auto l = __builtin_amdgcn_permlane32_swap(lo[e][k], lo[e][k + 2], false, false);
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        // hi + lo has at most 23 bits
        const uint32_t hw = h[o], lw = l[o];
        auto half = [](uint32_t word) {
          return static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(word)));
        };
        value[2 * o + e][2 * k] = half(hw) + half(lw);
        value[2 * o + e][2 * k + 1] = half(hw >> 16) + half(lw >> 16);
      }
    }
}

// One of a round's three products, a square tile per block of threads.  A A and B X sum along the
// rows of their operands, which pass through shared memory as they lie; A = X X' sums along the
// columns of X', which transposed reads of the shared memory turn.  A and B are symmetric: only
// tiles on and below the diagonal are summed, the others are their mirrors.  growth: 3.4445 to the
// number of rounds before.
template <Step S, class Sh>
__global__ __launch_bounds__(Sh::threads) void muon_product_kernel(Group g, int odd, float growth) {
  constexpr int kTile = Sh::tile, TM = Sh::TM, TN = Sh::TN, K = Sh::K;
  // per operand row and K block: 32 summed values, 8 pieces of 16 bytes (hi 0..3, lo 4..7), each
  // at its place exclusive-or bits 1 to 3 of the row: the 16 rows that one pass of a fragment's
  // reads takes lie in different banks (with bits 0 to 2, two and two share them: 1.05 times the
  // time)
  constexpr int kStage = kTile * 128 * K;
  __shared__ __attribute__((aligned(16))) char stage[2 * 2 * kStage];  // [turn][a, b][K][row][128]
  const uint32_t id = oxh::xcd_contiguous(blockIdx.x, gridDim.x);
  const Matrix &m = matrix_of(g, id);
  const Layout l = layout_of(m.ps, m.pl);
  constexpr bool kSymmetric = S == Step::Gram || S == Step::Poly;
  const Tile t = tile_at<kSymmetric>(id - m.first_block, m.ps / kTile, m.pl / kTile);
  const uint32_t ti = t.row, tj = t.column;
  const uint32_t k_total = S == Step::Gram ? m.pl : m.ps;
  const f16 *pa, *pb;
  f16 *gs = reinterpret_cast<f16 *>(m.scratch + l.gs);
  f16 *bs = reinterpret_cast<f16 *>(m.scratch + l.bs);
  f16 *from = reinterpret_cast<f16 *>(m.scratch + (odd ? l.xt1 : l.xt0));
  f16 *to = reinterpret_cast<f16 *>(m.scratch + (odd ? l.xt0 : l.xt1));
  if constexpr (S == Step::Gram) pa = pb = from;
  else if constexpr (S == Step::Poly) pa = pb = gs;
  else pa = bs, pb = from;
  // of the operands' rows ti kTile .., or (Gram) columns
  const uint64_t tile_bytes = kTile * 4 * (S == Step::Gram ? uint64_t{1} : k_total);
  const char *sa = reinterpret_cast<const char *>(pa) + ti * tile_bytes;
  const char *sb = reinterpret_cast<const char *>(pb) + tj * tile_bytes;

  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t group = wave / (Sh::WM * Sh::WN), place = wave % (Sh::WM * Sh::WN);
  const uint32_t wi = place / Sh::WN, wj = place % Sh::WN;
  // Gram: lines of 256 bytes, which are 64 columns of a row, or 32 of two rows where a tile has no
  // more.  A line's 32-byte pieces lie at their places exclusive-or a number of the line
  // (`turn_of`), so that the pieces of four rows that 32 lanes read together, or of eight rows, lie
  // in different banks.
  constexpr int kLineRows = kTile == 32 ? 2 : 1, kAcross = kTile >= 64 ? kTile / 64 : 1;
  auto turn_of = [](uint32_t line) {
    return kLineRows == 2 ? (line & 1) << 1 | (line >> 1 & 1) : (line & 3) << 1 | (line >> 2 & 1);
  };
  // Direct: operands pass from memory to shared memory without a stop in registers.  Each load of
  // a wave fills 1024 bytes there in the order of its lanes, so a lane loads the piece that belongs
  // at its place (both ways do).
  constexpr int kLoads = 2 * K * kTile * 8 / Sh::threads, kRows = Sh::threads / 8;
  static_assert(kLoads % 2 == 0 && (kRows == 64 || (kRows == 128 && kTile == 64 && K == 2)),
                "passes of rows, or of lines");
  u32x4 held[kLoads];
  const uint32_t blocks = k_total / 32;  // a multiple of the tile's
  constexpr bool kTail = kTile < 32 * K;
  const uint32_t r0 = threadIdx.x >> 3, c0 = (threadIdx.x & 7) ^ (r0 >> 1 & 7);
  const uint32_t line0 = threadIdx.x >> 4,
                 piece0 = ((threadIdx.x >> 1 & 7) ^ turn_of(line0)) << 1 | (threadIdx.x & 1);
  auto fetch = [&](uint32_t block, char *to_stage) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t pass = i % (kLoads / 2);
      const char *p = i < kLoads / 2 ? sa : sb;
      // a block of 32 summed values, the same for the wave; past the last one (whose products are
      // left out) the last is read again
      auto source = [&](uint32_t ahead) {
        return static_cast<uint64_t>(kTail ? min(block + ahead, blocks - 1) : block + ahead) * 128;
      };
      if constexpr (S == Step::Gram) {
        // passes of lines: for each 32 rows the tile's columns 64 by 64
        const uint32_t line = pass * (kRows / 2) + line0, lines = line / 32;
        const uint32_t row = line % 32 * kLineRows + piece0 / (16 / kLineRows);
        p += source((pass * (kRows / 2) + wave * 4) / 32 / kAcross * kLineRows +
                    wave * 4 % 32 * kLineRows / 32) * m.ps;
        p += row % 32 * m.ps * 4 + lines % kAcross * 256 + piece0 % (16 / kLineRows) * 16;
      } else {
        const uint32_t row = kTile % kRows == 0 ? pass * kRows % kTile + r0
                                                : (pass * kRows + r0) % kTile;
        p += source((pass * kRows + wave * 8) / kTile);
        p += row * k_total * 4 + c0 * 16;
      }
      if constexpr (Sh::Direct) {
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void *)p,
            (__attribute__((address_space(3))) void *)(to_stage +
                                                       (i * Sh::threads + wave * 64) * 16),
            16, 0, 0);
      } else {
        held[i] = *reinterpret_cast<const u32x4 *>(p);
      }
    }
  };
  auto put = [&](char *to_stage) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      *reinterpret_cast<u32x4 *>(to_stage + (i * Sh::threads + threadIdx.x) * 16) = held[i];
  };
  // Ends with every thread's operands there.
  auto arrive = [] {
    if constexpr (Sh::Direct) {
      __builtin_amdgcn_sched_barrier(0);  // behind the products
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
  };
  // hi and lo of rows (Gram: columns) 32 t .. of an operand's stage, 16 summed values
  auto operand = [&](const char *in, uint32_t t, uint32_t half, f16x8 &hi, f16x8 &lo) {
    if constexpr (S == Step::Gram) {
      const uint32_t row = half * 16 + (lane >> 5) * 4 + (lane >> 2 & 3);
      const uint32_t line = row / kLineRows % 32;
      const uint32_t pass = kLineRows == 2 ? row / 64 : row / 32 * (kTile / 64) + t / 2;
      const uint32_t part = (kLineRows == 2 ? row & 1 : t & 1) * 4 + (lane >> 4 & 1);
      const char *p = in + (pass * 32 + line) * 256 + (lane & 3) * 8;
      constexpr int kEight = 8 / kLineRows * 256;  // eight rows further: the same turn
      auto read = [&](uint32_t at) {
        const char *q = p + ((at ^ turn_of(line)) << 5);
        return join(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)q),
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(q + kEight)));
      };
      hi = read(part);
      lo = read(part + 2);
    } else {
      const uint32_t row = t * 32 + (lane & 31), c = (half & 1) * 2 + (lane >> 5);
      const char *p = in + (half >> 1) * kTile * 128 + row * 128;
      hi = *reinterpret_cast<const f16x8 *>(p + ((c ^ (row >> 1 & 7)) * 16));
      lo = *reinterpret_cast<const f16x8 *>(p + (((c + 4) ^ (row >> 1 & 7)) * 16));
    }
  };
  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  // Direct: a stage is loaded while the one before is multiplied, from behind its last fragments'
  // reads into the buffer whose readers passed the barrier.  Through registers: loaded two stages
  // ahead, and written to that buffer behind the first fragments' reads.  Loading further ahead, or
  // more per stage, changed nothing.
  fetch(0, stage);
  if constexpr (!Sh::Direct) {
    put(stage);
    if (K < blocks) fetch(K, stage);
  }
  arrive();
  int turn = 0;
  for (uint32_t block = 0; block < blocks; block += K) {
    const char *now = stage + turn * 2 * kStage;
    turn ^= 1;
    constexpr int kParts = 2 * K / Sh::Groups;
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      f16x8 ah[TM], al[TM], bh[TN], bl[TN];
      const uint32_t half = part * Sh::Groups + group;
      const bool within = !kTail || block + half / 2 < blocks;
      if (within) {
#pragma unroll
        for (int i = 0; i < TM; ++i) operand(now, wi * TM + i, half, ah[i], al[i]);
#pragma unroll
        for (int j = 0; j < TN; ++j) operand(now + kStage, wj * TN + j, half, bh[j], bl[j]);
      }
      if constexpr (Sh::Direct) {
        if (part == kParts - 1 && block + K < blocks) fetch(block + K, stage + turn * 2 * kStage);
      } else if (part == 0 && block + K < blocks) {
        put(stage + turn * 2 * kStage);
        if (block + 2 * K < blocks) fetch(block + 2 * K, stage);
      }
      if (!within) continue;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], acc[i][j], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], acc[i][j], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], acc[i][j], 0, 0, 0);
    }
    arrive();
  }

  // The groups' sums meet: block t of a wave's TM x TN is finished by group t % Groups, which adds
  // the groups' in their order; one block per group and turn goes through the shared memory.
  if constexpr (Sh::Groups > 1) {
    constexpr int kGroups = Sh::Groups, kBlocks = TM * TN;
    constexpr int kTurn = kBlocks < kGroups ? kBlocks : kGroups;
    static_assert(Sh::WM * Sh::WN * kTurn * kGroups * 4096 <= 4 * kStage, "exchange space");
    float *space = reinterpret_cast<float *>(stage);
#pragma unroll
    for (int t0 = 0; t0 < kBlocks; t0 += kGroups) {
#pragma unroll
      for (int o = 0; o < kGroups; ++o) {
        if (t0 + o >= kBlocks) continue;
        float *slot = space + ((place * kTurn + o) * kGroups + group) * 1024 + lane * 4;
        const f32x16 &sums = acc[(t0 + o) / TN][(t0 + o) % TN];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4 *>(slot + q * 256) =
              f32x4{sums[4 * q], sums[4 * q + 1], sums[4 * q + 2], sums[4 * q + 3]};
      }
      __syncthreads();
#pragma unroll
      for (int o = 0; o < kGroups; ++o) {
        if (t0 + o >= kBlocks || o != static_cast<int>(group)) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int other = 0; other < kGroups; ++other)
            sum += *reinterpret_cast<const f32x4 *>(
                space + ((place * kTurn + o) * kGroups + other) * 1024 + lane * 4 + q * 256);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[(t0 + o) / TN][(t0 + o) % TN][4 * q + r] = sum[r];
        }
      }
      __syncthreads();
    }
  }

  // Lane l holds column l % 32 and, in register r, row 8 (r / 4) + 4 (l / 32) + r % 4 of each
  // 32 x 32 block: four consecutive rows per register quad.  The halves go through the wave's own
  // part of the shared memory (whose operands have been read: a barrier ended the sums), by columns
  // and (A and B off the diagonal) by rows, and leave as whole lines: 32 hi and 32 lo of a row.
  constexpr uint32_t kPitch = 36;  // words per line of the wave's 32 x 32 words
  constexpr int kFinishing = TM * TN < Sh::Groups ? TM * TN : Sh::Groups;  // groups with a block
  static_assert(Sh::WM * Sh::WN * kFinishing * 32 * kPitch * 4 <= 4 * kStage, "turning space");
  uint32_t *turned = reinterpret_cast<uint32_t *>(stage) + wave * 32 * kPitch;
  // `again` takes 4^k out of the product of operands kept larger, `next` turns 2^k X into 2^k' X, as
  // the next round has it, or X
  float again = 1.0f, next = 1.0f;
  if constexpr (S != Step::Gram) {
    const float length = *reinterpret_cast<const float *>(m.scratch + l.length) * growth;
    const int k = shift_of(length);
    again = ldexpf(1.0f, -2 * k);
    next = ldexpf(1.0f, (S == Step::Apply ? shift_of(length * kA) : 0) - k);
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      if (Sh::Groups > 1 && (i * TN + j) % Sh::Groups != static_cast<int>(group)) continue;
      const uint32_t row0 = ti * kTile + (wi * TM + i) * 32;
      const uint32_t column0 = tj * kTile + (wj * TN + j) * 32;
      const uint32_t column = column0 + (lane & 31);
      // X or A at this place: among the operand rows just read
      f32x4 addend[4];
      if constexpr (S != Step::Gram) column_of(pb + halves_at(column, row0, m.ps), lane, addend);
      u32x4 words[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t at = 8 * q + 4 * (lane >> 5), row = row0 + at;
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = acc[i][j][4 * q + r] * (kUnscale * again);
        if constexpr (S == Step::Poly) v = kB / kScale * addend[q] + kC * v;
        if constexpr (S == Step::Apply || S == Step::Last)
          v = (v + kA / kScale * addend[q]) * next;
        if constexpr (S == Step::Last) {
          const bool tall = m.rows > m.columns;
          const uint32_t wr0 = tall ? column : row, wc0 = tall ? row : column;
          float *t = m.target + static_cast<uint64_t>(wr0) * m.columns + wc0;
          const uint64_t next = tall ? 1 : m.columns;
          // entries past the sides are read from the last ones, and not written
          const uint32_t left = tall ? (wr0 < m.rows && wc0 < m.columns ? m.columns - wc0 : 0u)
                                     : (wc0 < m.columns && wr0 < m.rows ? m.rows - wr0 : 0u);
          if (left != 0) {
            if (m.momentum != nullptr) {
              f32x4 w;
#pragma unroll
              for (uint32_t r = 0; r < 4; ++r) w[r] = t[min(r, left - 1) * next];
#pragma unroll
              for (int r = 0; r < 4; ++r) v[r] = w[r] - g.lr * (g.decay * w[r] + m.scale * v[r]);
            }
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
              if (r < left) t[r * next] = v[r];
          }
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) words[q][r] = halves_word(v[r]);
          *reinterpret_cast<u32x4 *>(turned + (lane & 31) * kPitch + at) = words[q];
        }
      }
      if constexpr (S != Step::Last) {
        f16 *result = S == Step::Gram ? gs : S == Step::Poly ? bs : to;
        const uint32_t *line = turned + (lane >> 1) * kPitch + (lane & 1) * 16;
        __builtin_amdgcn_wave_barrier();
        store_line(line, result + halves_at(column0 + (lane >> 1), row0 + (lane & 1) * 16, m.ps));
        __builtin_amdgcn_wave_barrier();
        if (kSymmetric && ti != tj) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              turned[(8 * q + 4 * (lane >> 5) + r) * kPitch + (lane & 31)] = words[q][r];
          __builtin_amdgcn_wave_barrier();
          store_line(line, result + halves_at(row0 + (lane >> 1), column0 + (lane & 1) * 16, m.ps));
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
}

// ---------------------------------------------------------------- one block per matrix
//
// A matrix whose X' in halves fits the shared memory of a compute unit is stepped from start to end
// by one block of 12 waves, X staying in registers.  Each wave owns blocks of 16 columns of X
// (along its long side), as 16 x 16 results of the matrix cores: lane l holds column l % 16 and, of
// row block r, rows 16 r + 4 (l / 16) .. + 3.  Summed indexes are taken 32 at a time in the order
// 16 r + 4 (l / 16) + i that this gives: a pair of row blocks is then an operand of B X as it lies,
// and transposed reads of the shared memory (16 lanes fetch 4 rows of 16 float16 and each gets a
// column of 4) give the same order for X X'.
//
// The bound is one compute unit's shared memory and its barriers: of the 88000 cycles that 96 x
// 192 takes (40 us), a round is 14500: X X' 3000 (its operands are 2250 of the shared memory's), A
// and A A 4600 with their halves, shared among the waves that summed a tile, B X 4700 (3400), X' in
// halves 2000.  The way in is 14000: twelve loads at a time, 7000 where eight took 9300.

constexpr int kWhole = 163840;  // bytes of shared memory, the last for the norm's parts
constexpr int kWholeWaves = 12;
// X': bytes of a row of PS values in halves (hi, then lo), an odd number of 32-byte steps, so that
// eight rows lie in different banks; every other eight rows have the 16-byte halves of each step
// exchanged, so that sixteen rows' stores do too.
constexpr int whole_pitch(int ps) { return ps * 4 + 32; }
// A and B: for each lane quad the rows' pieces of 16 bytes that it reads (per 32 summed values, hi
// and lo), an odd number of them to a row.
constexpr int square_pitch(int ps) { return (ps / 16 + 1) * 16; }
constexpr int square_bytes(int ps) { return 4 * ps * square_pitch(ps); }

// Four values as hi and lo.
__device__ __forceinline__ void halves_of(const f32x4 &v, s16x4 &hi, s16x4 &lo) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    f16 h, w;
    halves_of(v[r], h, w);
    hi[r] = __builtin_bit_cast(short, h);
    lo[r] = __builtin_bit_cast(short, w);
  }
}

// acc += a b' in halves.
__device__ __forceinline__ void multiply(const f16x8 (&a)[2], const f16x8 (&b)[2], f32x4 &acc) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[1], b[0], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[0], acc, 0, 0, 0);
}

//
// Slab: the same for a matrix of too many columns, in slabs of 12 x 16 of them, a block each, and a
// launch for each round: it adds the slabs' shares of A in order, takes its columns of X through B,
// and leaves its share of the next A.  Launch 0 makes X, launch `rounds` the result.
constexpr uint32_t kSlabColumns = 16 * kWholeWaves;
struct SlabLayout {
  uint64_t shares, parts, total;  // X lies first
};
__host__ __device__ inline SlabLayout slab_layout(uint64_t ps, uint64_t slabs) {
  const uint64_t side = ps / 32, tiles = side * (side + 1) / 2;
  SlabLayout l;
  l.shares = slabs * ps * kSlabColumns * 4;
  l.parts = l.shares + 2 * slabs * tiles * 4096;
  l.total = l.parts + kNormParts * 4;
  return l;
}

template <int PS, int Blocks, bool Slab>
__global__ __launch_bounds__(64 * kWholeWaves) void muon_whole_kernel(Group g, uint32_t rounds,
                                                                      uint32_t round) {
  __shared__ __attribute__((aligned(16))) char shared[kWhole];
  float *const parts = reinterpret_cast<float *>(shared + kWhole - 4 * kWholeWaves);
  constexpr int kRowBlocks = PS / 16, kPitch = whole_pitch(PS), kSquare = square_pitch(PS);
  constexpr int kSide = PS / 32, kTiles = kSide * (kSide + 1) / 2;  // of 32 x 32, lower ones of A
  constexpr int kSplits = kWholeWaves / kTiles;                     // of the sums of A
  // the waves that finish a tile's four 16 x 16 blocks, and how many each
  constexpr int kShare = kSplits >= 4 ? 4 : kSplits >= 2 ? 2 : 1, kOwn = 4 / kShare;
  constexpr int kOwnRows = kShare == 1 ? 2 : 1, kOwnColumns = kOwn / kOwnRows;
  // X' first; then, over it, the sums to be joined, A and B
  constexpr int kSums = kSplits > 1 ? kTiles * 4 * kSplits * 1024 : 0;
  char *const sums = shared, *const sa = shared + kSums, *const sb = sa + square_bytes(PS);
  static_assert(kSums + 2 * square_bytes(PS) <= kWhole, "shared memory");
  const Matrix &m = Slab ? matrix_of(g, blockIdx.x) : g.m[blockIdx.x];
  const bool tall = m.rows > m.columns;
  const uint32_t s = tall ? m.columns : m.rows, n_all = tall ? m.rows : m.columns;
  const uint32_t slab = Slab ? blockIdx.x - m.first_block : 0, column0 = slab * kSlabColumns;
  const uint32_t n = Slab ? min(n_all - column0, kSlabColumns) : n_all;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t col = lane & 15, quad = lane >> 4;
  const uint32_t column_blocks = (n + 31) / 32 * 2;
  f32x4 x[Blocks][kRowBlocks];
  // Slab: X as the threads hold it; the shares of A, of even and of odd launches
  const uint32_t slabs = (n_all + kSlabColumns - 1) / kSlabColumns;
  const SlabLayout sl = slab_layout(PS, slabs);
  f32x4 *const kept_x = reinterpret_cast<f32x4 *>(m.scratch) +
                        slab * kRowBlocks * 64 * kWholeWaves + threadIdx.x;
  auto shares = [&](uint32_t launch, uint32_t of) {
    return reinterpret_cast<f32x4 *>(m.scratch + sl.shares) +
           ((launch & 1) * slabs + of) * kTiles * 4 * 64 + lane;
  };
  // offset of (i, j) of X in the matrix
  auto place = [&](uint32_t i, uint32_t j) {
    return tall ? static_cast<uint64_t>(column0 + j) * m.columns + i
                : static_cast<uint64_t>(i) * m.columns + column0 + j;
  };
  // The matrix lies in the shared memory as in memory, its rows an odd number of words apart, on
  // the way in and out.  A thread moves kBatch of its elements at a time: load(b, offset in memory)
  // for each, then use(b, offset there, offset in memory).
  float *const words = reinterpret_cast<float *>(shared);
  const uint32_t pitch = m.columns | 1;
  constexpr int kBatch = 12;
  auto each = [&](auto load, auto use) {
    constexpr uint32_t kThreads = 64 * kWholeWaves;
    const uint32_t rows_on = kThreads / m.columns, columns_on = kThreads % m.columns;
    const uint32_t all = m.rows * m.columns;
    uint32_t row = threadIdx.x / m.columns, column = threadIdx.x % m.columns;
    auto batch = [&](uint32_t at, auto whole) {
      constexpr bool kWholeBatch = decltype(whole)::value;
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (kWholeBatch || at + b * kThreads < all) load(b, at + b * kThreads);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (kWholeBatch || at + b * kThreads < all)
          use(b, row * pitch + column, at + b * kThreads);
        row += rows_on;
        column += columns_on;
        if (column >= m.columns) column -= m.columns, ++row;
      }
    };
    uint32_t at = threadIdx.x;
    for (; at + (kBatch - 1) * kThreads < all; at += kBatch * kThreads)
      batch(at, std::true_type());
    if (at < all) batch(at, std::false_type());
  };
  const uint32_t step_i = tall ? 1 : pitch, step_j = tall ? pitch : 1;

  if constexpr (Slab) {
    if (round != 0) {
#pragma unroll
      for (int r = 0; r < kRowBlocks; ++r) x[0][r] = kept_x[r * 64 * kWholeWaves];
    } else {
      const float *norms = reinterpret_cast<const float *>(m.scratch + sl.parts);
      float one[1] = {threadIdx.x < kNormParts ? norms[threadIdx.x] : 0.0f};
      oxh::wave_sums_rows(one);
      if (lane == 0) parts[wave] = one[0];
      __syncthreads();
      float total = 0.0f;
#pragma unroll
      for (int w = 0; w < kWholeWaves; ++w) total += parts[w];
      const float inverse = 1.0f / (sqrtf(total) + g.epsilon);
      const uint32_t j = wave * 16 + col;
#pragma unroll
      for (int r = 0; r < kRowBlocks; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t i = 16 * r + 4 * quad + e;
          x[0][r][e] = i < s && j < n ? direction(g, m, place(i, j)) * inverse : 0.0f;
        }
    }
  } else {
  float squares = 0.0f, grad[kBatch], mom[kBatch];
  each([&](int b, uint32_t at) {
    grad[b] = m.gradient[at];
    if (m.momentum != nullptr) mom[b] = m.momentum[at];
  }, [&](int b, uint32_t to, uint32_t at) {
    float v = grad[b];
    if (m.momentum != nullptr) {
      const float now = g.momentum * mom[b] + v;
      m.momentum[at] = now;
      v = g.nesterov ? v + g.momentum * now : now;
    }
    words[to] = v;
    squares = fmaf(v, v, squares);
  });
  float one[1] = {squares};
  oxh::wave_sums_rows(one);
  if (lane == 0) parts[wave] = one[0];
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int w = 0; w < kWholeWaves; ++w) total += parts[w];
  const float inverse = 1.0f / (sqrtf(total) + g.epsilon);
#pragma unroll
  for (int c = 0; c < Blocks; ++c) {
    const uint32_t j = (c * kWholeWaves + wave) * 16 + col;
#pragma unroll
    for (int r = 0; r < kRowBlocks; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t i = 16 * r + 4 * quad + e;
        x[c][r][e] = i < s && j < n ? words[i * step_i + j * step_j] * inverse : 0.0f;
      }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  }

  // this wave's tile of A and its share of the sum
  const uint32_t tile = wave % kTiles, split = wave / kTiles;
  uint32_t ti = 0;
  while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
  const uint32_t tj = tile - ti * (ti + 1) / 2;

  // this wave's blocks of A, and the first one's place in the tile
  f32x4 own[kOwnRows][kOwnColumns];
  const uint32_t i0 = kShare == 1 ? 0 : kShare == 2 ? split : split >> 1;
  const uint32_t j0 = kShare == 4 ? split & 1 : 0;
  // own = the products of X's columns here
  auto gram = [&]() {
#pragma unroll
    for (int c = 0; c < Blocks; ++c) {
      const uint32_t block = c * kWholeWaves + wave;
      if (block >= column_blocks) continue;
      char *row = shared + (block * 16 + col) * kPitch + ((quad * 8) ^ ((col & 8) * 2));
#pragma unroll
      for (int r = 0; r < kRowBlocks; ++r) {
        s16x4 hi, lo;
        halves_of(x[c][r], hi, lo);
        *reinterpret_cast<s16x4 *>(row + 32 * r) = hi;
        *reinterpret_cast<s16x4 *>(row + 2 * PS + 32 * r) = lo;
      }
    }
    __syncthreads();

    f32x4 acc[2][2] = {};
    if (split < kSplits) {
      // rows 32 t + 16 b of X as an operand: column 16 b + .. of the rows of X' in shared memory
      auto operand = [&](uint32_t k, uint32_t t, int b, f16x8(&out)[2]) {
        const char *p = shared + (k * 32 + quad * 4 + (col >> 2)) * kPitch + (t * 32 + b * 16) * 2 +
                        (((col & 3) * 8) ^ ((quad & 2) * 8));
#pragma unroll
        for (int h = 0; h < 2; ++h)
          out[h] = join(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_s16x4 *)(p + h * 2 * PS)),
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_s16x4 *)(p + h * 2 * PS + 16 * kPitch)));
      };
      for (uint32_t k = split; k < column_blocks / 2; k += kSplits) {
        f16x8 a[2][2], b[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) operand(k, ti, i, a[i]);
#pragma unroll
        for (int j = 0; j < 2; ++j) operand(k, tj, j, b[j]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) multiply(a[i], b[j], acc[i][j]);
      }
    }
    __syncthreads();
    if constexpr (kSplits > 1) {
      f32x4 *slot = reinterpret_cast<f32x4 *>(sums) + tile * 4 * kSplits * 64 + lane;
      if (split < kSplits) {
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q)
          if (q / kOwn != split) slot[(q * kSplits + split) * 64] = acc[q >> 1][q & 1];
      }
      __syncthreads();
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) {
        if (q / kOwn != split) continue;
        f32x4 sum = {};
#pragma unroll
        for (uint32_t p = 0; p < kSplits; ++p)
          sum += p == split ? acc[q >> 1][q & 1] : slot[(q * kSplits + p) * 64];
        own[q % kOwn / kOwnColumns][q % kOwn % kOwnColumns] = sum;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) own[q >> 1][q & 1] = acc[q >> 1][q & 1];
    }
  };
  // X = a X + (b A + c A A) X
  auto apply = [&]() {
    // block (i, j) of this wave's tile of A or B to the columns' rows of `to` and, off the
    // diagonal, to the rows' rows: there two lanes with neighbouring columns share their four rows'
    // words
    auto keep = [&](char *to, const f32x4 &v, uint32_t i, uint32_t j) {
      s16x4 hi, lo;
      halves_of(v, hi, lo);
      char *p = to + (quad * PS + tj * 32 + j * 16 + col) * kSquare + ti * 32 + i * 8;
      *reinterpret_cast<s16x4 *>(p) = hi;
      *reinterpret_cast<s16x4 *>(p + 16) = lo;
      if (ti == tj) return;  // both lie in this tile
      const u32x2 mine[2] = {__builtin_bit_cast(u32x2, hi), __builtin_bit_cast(u32x2, lo)};
      const bool odd = col & 1;
      char *q = to + ((col >> 2) * PS + ti * 32 + i * 16 + quad * 4 + (odd ? 2 : 0)) * kSquare +
                tj * 32 + j * 8 + (col & 2) * 2;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // the pair of rows this lane stores, of its own column and the neighbour's
        const uint32_t kept = odd ? mine[h][1] : mine[h][0], sent = odd ? mine[h][0] : mine[h][1];
        const uint32_t got = static_cast<uint32_t>(
            __builtin_amdgcn_update_dpp(0, static_cast<int>(sent), 0xB1, 0xF, 0xF, false));
        const uint32_t first = odd ? got : kept, second = odd ? kept : got;
        *reinterpret_cast<uint32_t *>(q + h * 16) = (first & 0xFFFFu) | second << 16;
        *reinterpret_cast<uint32_t *>(q + h * 16 + kSquare) = first >> 16 | (second & 0xFFFF0000u);
      }
    };
    // 16 rows of A or B as an operand
    auto rows_of = [&](const char *from, uint32_t row, int k, f16x8(&out)[2]) {
      const char *p = from + (quad * PS + row + col) * kSquare + k * 32;
      out[0] = *reinterpret_cast<const f16x8 *>(p);
      out[1] = *reinterpret_cast<const f16x8 *>(p + 16);
    };
    if (split < kShare) {
#pragma unroll
      for (int i = 0; i < kOwnRows; ++i)
#pragma unroll
        for (int j = 0; j < kOwnColumns; ++j) {
          own[i][j] *= kUnscale;
          keep(sa, own[i][j], i0 + i, j0 + j);
        }
    }
    __syncthreads();
    if (split < kShare) {
      f32x4 square[kOwnRows][kOwnColumns] = {};
#pragma unroll
      for (int k = 0; k < kSide; ++k) {
        f16x8 a[kOwnRows][2], b[kOwnColumns][2];
#pragma unroll
        for (int i = 0; i < kOwnRows; ++i) rows_of(sa, ti * 32 + (i0 + i) * 16, k, a[i]);
#pragma unroll
        for (int j = 0; j < kOwnColumns; ++j) rows_of(sa, tj * 32 + (j0 + j) * 16, k, b[j]);
#pragma unroll
        for (int i = 0; i < kOwnRows; ++i)
#pragma unroll
          for (int j = 0; j < kOwnColumns; ++j) multiply(a[i], b[j], square[i][j]);
      }
#pragma unroll
      for (int i = 0; i < kOwnRows; ++i)
#pragma unroll
        for (int j = 0; j < kOwnColumns; ++j)
          keep(sb, kB * own[i][j] + kC * (square[i][j] * kUnscale), i0 + i, j0 + j);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < Blocks; ++c) {
      if (static_cast<uint32_t>(c * kWholeWaves) + wave >= column_blocks) continue;
      f16x8 b[kSide][2];
#pragma unroll
      for (int k = 0; k < kSide; ++k) {
        s16x4 h0, l0, h1, l1;
        halves_of(x[c][2 * k], h0, l0);
        halves_of(x[c][2 * k + 1], h1, l1);
        b[k][0] = join(h0, h1);
        b[k][1] = join(l0, l1);
      }
#pragma unroll
      for (int r = 0; r < kRowBlocks; ++r) {
        f32x4 sum = {};
#pragma unroll
        for (int k = 0; k < kSide; ++k) {
          f16x8 a[2];
          rows_of(sb, r * 16, k, a);
          multiply(a, b[k], sum);
        }
        x[c][r] = kA * x[c][r] + sum * kUnscale;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
  };
  if constexpr (Slab) {
    auto each_own = [&](auto use) {
      if (split >= kShare) return;
#pragma unroll
      for (int i = 0; i < kOwnRows; ++i)
#pragma unroll
        for (int j = 0; j < kOwnColumns; ++j)
          use(own[i][j], (tile * 4 + (i0 + i) * 2 + j0 + j) * 64);
    };
    if (round != 0) {
      each_own([&](f32x4 &sum, uint32_t at) {
        sum = shares(round + 1, 0)[at];
#pragma unroll 8
        for (uint32_t p = 1; p < slabs; ++p) sum += shares(round + 1, p)[at];
      });
      apply();
    }
    if (round != rounds) {
#pragma unroll
      for (int r = 0; r < kRowBlocks; ++r) kept_x[r * 64 * kWholeWaves] = x[0][r];
      gram();
      each_own([&](f32x4 &share, uint32_t at) { shares(round, slab)[at] = share; });
    } else {
      const uint32_t j = wave * 16 + col;
#pragma unroll
      for (int r = 0; r < kRowBlocks; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t i = 16 * r + 4 * quad + e;
          if (i >= s || j >= n) continue;
          float *to = m.target + place(i, j);
          *to = m.momentum == nullptr ? x[0][r][e]
                                      : *to - g.lr * (g.decay * *to + m.scale * x[0][r][e]);
        }
    }
    return;
  }
  for (uint32_t turn = 0; turn < rounds; ++turn) {
    gram();
    apply();
  }
  uint32_t again = col;  // so that no offset is kept from the way in
  asm volatile("" : "+v"(again));
#pragma unroll
  for (int c = 0; c < Blocks; ++c) {
    const uint32_t j = (c * kWholeWaves + wave) * 16 + again;
#pragma unroll
    for (int r = 0; r < kRowBlocks; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t i = 16 * r + 4 * quad + e;
        if (i < s && j < n) words[i * step_i + j * step_j] = x[c][r][e];
      }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  float w[kBatch];
  each([&](int b, uint32_t at) {
    if (m.momentum != nullptr) w[b] = m.target[at];
  }, [&](int b, uint32_t from, uint32_t at) {
    const float v = words[from];
    m.target[at] =
        m.momentum == nullptr ? v : w[b] - g.lr * (g.decay * w[b] + m.scale * v);
  });
}

// ---------------------------------------------------------------- host

struct Item {
  const float *gradient;
  float *momentum, *target;
  uint64_t rows, columns;
};

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// Whether one block steps the whole matrix: the rows of the shared memory that hold X', and at most
// this many column blocks per wave (one matrix of 96 x 192 40 us, 72 in tiles; of 64 x 384 45, 47
// in slabs; of 128 x 192 58, 73 in tiles; of 96 x 384 and 128 x 256, whose two column blocks spill,
// 92 and 116, and 60 in slabs and 74 in tiles).
constexpr int whole_blocks(int ps) { return ps == 32 ? 6 : ps == 64 ? 3 : 1; }
bool whole(const Item &it) {
  const uint64_t s = std::min(it.rows, it.columns), n = std::max(it.rows, it.columns);
  if (s > 128) return false;
  const int ps = static_cast<int>(round_up(s, 32));
  return round_up(n, 32) * whole_pitch(ps) <= kWhole - 4 * kWholeWaves &&
         round_up(n, 32) <= 16ull * kWholeWaves * whole_blocks(ps);
}

// Whether a matrix goes in slabs: 7 launches in place of the tiles' 17, but the least work per
// launch is a slab's round, and every block adds all slabs' shares (64 x 1000: 50 us, 84 in tiles;
// 20 x 10000: 48 and 247; four of 69 x 2045: 85 and 128; 128 x 512: 92 and 80; 128 x 2000: 107 and
// 108; 128 x 19000: 280 and 434).
constexpr uint64_t kMostSlabs = 100;
bool slabbed(const Item &it) {
  const uint64_t s = std::min(it.rows, it.columns), n = std::max(it.rows, it.columns);
  return (s <= 96 || (s <= 128 && n >= 2048)) && n <= kMostSlabs * kSlabColumns;
}

// Tile sides of a launch group: `square` of A and B, of which the tiles on and below the diagonal
// are summed, and `apply` of B X.
struct Tiles {
  uint32_t square, apply;
  uint32_t pad() const { return std::max(square, apply); }
};

// Small tiles spread a product over more compute units, large ones load less per product.  Each
// product takes
//   32 where its tiles of 32 are at most one per compute unit (512 x 512: 101 us, 135 with 64;
//     1024 x 1024: 282 and 201; 512 x 2048, whose B X has 1024 such tiles: 166 with 32 for both
//     products, 145 with 32 and 64, 190 with 64);
//   128 where there is one for every other compute unit (B X of 1000 x 4000, 256 tiles: 422 us, 443
//     with 64; of 1536 x 1536, 144 tiles: 524 both; of 1000 x 1280, 80 tiles: 302 and 230; all of
//     2560 x 2560, 210 and 400 tiles: 1367 and 1608) and padding to 128 adds at most a tenth (32
//     matrices of 300 x 1200, padded 1.26 times: 739 and 618);
//   64 otherwise (`Few` up to a block per compute unit: 1024 x 1024, 136 and 256 tiles, 201 us and
//     254 without; everywhere, 12 x 512 x 2048 takes 716 and 657 without);
// and both take 192 where the square products just fill one round of a block per compute unit, with
// the same limit on padding (4096 x 4096, 253 tiles: 4.06 ms, 4.80 with 128; 2560 x 2560, 105
// tiles: 1641 and 1367 us; 12 x 1024 x 1024, 252 tiles padded 1.27 times: 1330 and 1079).  That is
// one matrix of a short side of 3841 to 4224; more rounds than one were not measured with 192, and a
// list of such matrices is slower than they are one by one (two of 4096 x 4096 8.8 ms and 8.1, three
// 13.0 and 12.1).
Tiles tiles_of(const Item *items, size_t count) {
  struct Count {
    uint64_t square = 0, apply = 0, area = 0;
  };
  auto of = [&](uint64_t tile) {
    Count c;
    for (size_t i = 0; i < count; ++i) {
      const uint64_t s = round_up(std::min(items[i].rows, items[i].columns), tile) / tile,
                     n = round_up(std::max(items[i].rows, items[i].columns), tile) / tile;
      c.square += s * (s + 1) / 2;
      c.apply += s * n;
      c.area += s * n * tile * tile;
    }
    return c;
  };
  const uint64_t units = oxh::kComputeUnits;
  const Count tiny = of(Tiny::tile), small = of(Small::tile), medium = of(Medium::tile),
              wide = of(Wide::tile);
  auto fits = [&](const Count &c) { return c.area * 10 <= small.area * 11; };
  if (wide.square <= units && wide.square * 8 >= units * 7 && fits(wide))
    return {Wide::tile, Wide::tile};
  auto pick = [&](uint64_t in_tiny, uint64_t in_medium) -> uint32_t {
    if (in_tiny <= units) return Tiny::tile;
    return fits(medium) && in_medium * 2 >= units ? Medium::tile : Small::tile;
  };
  return {pick(tiny.square, medium.square), pick(tiny.apply, medium.apply)};
}

uint64_t scratch_of(const Item *items, size_t count) {
  const uint32_t pad = tiles_of(items, count).pad();
  uint64_t total = 0;
  for (size_t i = 0; i < count; ++i)
    total += round_up(layout_of(round_up(std::min(items[i].rows, items[i].columns), pad),
                                round_up(std::max(items[i].rows, items[i].columns), pad))
                          .total,
                      256);
  return total;
}

// The matrices that one block takes, those that go in slabs, and the others.
struct Parted {
  std::vector<Item> large, slabs, small;
};
Parted part(const std::vector<Item> &items) {
  Parted p;
  for (const Item &it : items)
    (whole(it) ? p.small : slabbed(it) ? p.slabs : p.large).push_back(it);
  return p;
}

uint64_t side_of(const Item &it) { return round_up(std::min(it.rows, it.columns), 32); }
uint64_t slabs_of(const Item &it) {
  return (std::max(it.rows, it.columns) + kSlabColumns - 1) / kSlabColumns;
}
// Calls run(group) with the slabbed matrices of this side, a launch group at a time.
template <typename Run>
oxh_status slab_groups(const std::vector<Item> &slabs, uint64_t side, Run run) {
  std::vector<Item> group;
  auto flush = [&]() {
    if (group.empty()) return oxh::ok();
    const oxh_status st = run(group);
    group.clear();
    return st;
  };
  for (const Item &it : slabs) {
    if (side_of(it) != side) continue;
    group.push_back(it);
    if (group.size() < kGroup) continue;
    oxh_status st = flush();
    if (st != OXH_OK) return st;
  }
  return flush();
}

uint64_t scratch_of_all(const Parted &items) {
  uint64_t most = 0;
  const std::vector<Item> &large = items.large;
  for (size_t at = 0; at < large.size(); at += kGroup)
    most = std::max(most, scratch_of(&large[at], std::min<size_t>(kGroup, large.size() - at)));
  for (uint64_t side = 32; side <= 128; side += 32)
    slab_groups(items.slabs, side, [&](const std::vector<Item> &group) {
      uint64_t total = 0;
      for (const Item &it : group) total += round_up(slab_layout(side, slabs_of(it)).total, 256);
      most = std::max(most, total);
      return oxh::ok();
    });
  return most;
}

template <Step S>
oxh_status product(hipStream_t stream, Group &g, uint32_t tile, int odd, float growth,
                   const char *what) {
  g.blocks = 0;
  for (uint32_t i = 0; i < g.count; ++i) {
    const uint32_t s = g.m[i].ps / tile, l = g.m[i].pl / tile;
    g.m[i].first_block = g.blocks;
    g.blocks += S == Step::Gram || S == Step::Poly ? s * (s + 1) / 2 : s * l;
  }
  auto start = [&](auto shape) {
    using Sh = decltype(shape);
    oxh::launch(muon_product_kernel<S, Sh>, dim3(g.blocks), dim3(Sh::threads), 0, stream,
                g, odd, growth);
  };
  if (tile == Wide::tile) start(Wide());
  else if (tile == Medium::tile) start(Medium());
  else if (tile == Small::tile && g.blocks <= oxh::kComputeUnits) start(Few());
  else if (tile == Small::tile) start(Small());
  else start(Tiny());
  return oxh::launched(what);
}

oxh_status run_norm(hipStream_t stream, Group &g) {
  g.blocks = 0;
  for (uint32_t i = 0; i < g.count; ++i) g.m[i].first_block = g.blocks, g.blocks += kNormParts;
  oxh::launch(muon_norm_kernel, dim3(g.blocks), dim3(kNormThreads), 0, stream, g);
  return oxh::launched("muon_norm");
}

oxh_status run_group(hipStream_t stream, Group &g, const Tiles &tiles, uint32_t rounds) {
  oxh_status st = run_norm(stream, g);
  if (st != OXH_OK) return st;
  g.blocks = 0;
  for (uint32_t i = 0; i < g.count; ++i) {
    g.m[i].first_block = g.blocks;
    g.blocks += (g.m[i].ps / 32) * (g.m[i].pl / 32);
  }
  oxh::launch(muon_start_kernel, dim3(g.blocks), dim3(256), 0, stream, g);
  st = oxh::launched("muon_start");
  float growth = 1.0f;
  for (uint32_t r = 0; r < rounds && st == OXH_OK; ++r) {
    const uint32_t square = tiles.square, apply = tiles.apply;
    st = product<Step::Gram>(stream, g, square, r & 1, growth, "muon_gram");
    if (st == OXH_OK) st = product<Step::Poly>(stream, g, square, r & 1, growth, "muon_poly");
    if (st != OXH_OK) return st;
    st = r + 1 < rounds ? product<Step::Apply>(stream, g, apply, r & 1, growth, "muon_apply")
                        : product<Step::Last>(stream, g, apply, r & 1, growth, "muon_last");
    growth *= kA;
  }
  return st;
}

struct Hyper {
  float lr, decay, momentum, epsilon;
  bool nesterov;
};

void describe(const Item &it, Matrix &m) {
  m.gradient = it.gradient;
  m.momentum = it.momentum;
  m.target = it.target;
  m.rows = static_cast<uint32_t>(it.rows);
  m.columns = static_cast<uint32_t>(it.columns);
  m.scale =
      std::sqrt(std::max(1.0f, static_cast<float>(it.rows) / static_cast<float>(it.columns)));
}

// Launches the small matrices with sides in this class, a group at a time.
template <int PS, int Blocks>
oxh_status run_whole(hipStream_t stream, const std::vector<Item> &small, Group g,
                     uint32_t rounds) {
  g.count = 0;
  auto flush = [&]() {
    if (g.count == 0) return oxh::ok();
    oxh::launch(muon_whole_kernel<PS, Blocks, false>, dim3(g.count), dim3(64 * kWholeWaves), 0,
                stream, g, rounds, 0u);
    g.count = 0;
    return oxh::launched("muon_whole");
  };
  for (const Item &it : small) {
    const uint64_t s = std::min(it.rows, it.columns), n = std::max(it.rows, it.columns);
    const bool few = round_up(n, 32) <= 16ull * kWholeWaves;
    if (round_up(s, 32) != PS || few != (Blocks == 1)) continue;
    describe(it, g.m[g.count++]);
    if (g.count == kGroup) {
      oxh_status st = flush();
      if (st != OXH_OK) return st;
    }
  }
  return flush();
}

// The slabbed matrices of this side.
template <int PS>
oxh_status run_slabs(hipStream_t stream, const std::vector<Item> &slabs, Group g, uint32_t rounds,
                     char *workspace) {
  return slab_groups(slabs, PS, [&](const std::vector<Item> &group) {
    g.count = static_cast<uint32_t>(group.size());
    uint64_t offset = 0;
    for (uint32_t i = 0; i < g.count; ++i) {
      const SlabLayout l = slab_layout(PS, slabs_of(group[i]));
      describe(group[i], g.m[i]);
      g.m[i].scratch = workspace + offset;
      g.m[i].parts = l.parts;
      offset += round_up(l.total, 256);
    }
    oxh_status st = run_norm(stream, g);
    uint32_t blocks = 0;
    for (uint32_t i = 0; i < g.count; ++i) {
      g.m[i].first_block = blocks;
      blocks += static_cast<uint32_t>(slabs_of(group[i]));
    }
    for (uint32_t round = 0; round <= rounds && st == OXH_OK; ++round) {
      oxh::launch(muon_whole_kernel<PS, 1, true>, dim3(blocks), dim3(64 * kWholeWaves), 0, stream,
                  g, rounds, round);
      st = oxh::launched("muon_slab");
    }
    return st;
  });
}

oxh_status run_all(hipStream_t stream, const Parted &items, const Hyper &h, uint32_t rounds,
                   char *workspace) {
  Group g{};
  g.momentum = h.momentum;
  g.lr = h.lr;
  g.decay = h.decay;
  g.epsilon = h.epsilon;
  g.nesterov = h.nesterov ? 1 : 0;
  oxh_status st = oxh::ok();
  const std::vector<Item> &small = items.small, &large = items.large;
  if (!small.empty()) {
    st = run_whole<32, 1>(stream, small, g, rounds);
    if (st == OXH_OK) st = run_whole<32, whole_blocks(32)>(stream, small, g, rounds);
    if (st == OXH_OK) st = run_whole<64, 1>(stream, small, g, rounds);
    if (st == OXH_OK) st = run_whole<64, whole_blocks(64)>(stream, small, g, rounds);
    if (st == OXH_OK) st = run_whole<96, 1>(stream, small, g, rounds);
    if (st == OXH_OK) st = run_whole<128, 1>(stream, small, g, rounds);
  }
  if (!items.slabs.empty()) {
    if (st == OXH_OK) st = run_slabs<32>(stream, items.slabs, g, rounds, workspace);
    if (st == OXH_OK) st = run_slabs<64>(stream, items.slabs, g, rounds, workspace);
    if (st == OXH_OK) st = run_slabs<96>(stream, items.slabs, g, rounds, workspace);
    if (st == OXH_OK) st = run_slabs<128>(stream, items.slabs, g, rounds, workspace);
  }
  for (size_t at = 0; at < large.size() && st == OXH_OK; at += kGroup) {
    const size_t count = std::min<size_t>(kGroup, large.size() - at);
    const Tiles tiles = tiles_of(&large[at], count);
    const uint32_t pad = tiles.pad();
    g.count = static_cast<uint32_t>(count);
    uint64_t offset = 0;
    for (size_t i = 0; i < count; ++i) {
      const Item &it = large[at + i];
      Matrix &m = g.m[i];
      describe(it, m);
      m.scratch = workspace + offset;
      m.ps = static_cast<uint32_t>(round_up(std::min(it.rows, it.columns), pad));
      m.pl = static_cast<uint32_t>(round_up(std::max(it.rows, it.columns), pad));
      m.parts = layout_of(m.ps, m.pl).parts;
      offset += round_up(layout_of(m.ps, m.pl).total, 256);
    }
    st = run_group(stream, g, tiles, rounds);
  }
  return st;
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

// Runs a C entry's body; what its containers may throw becomes a status.
template <typename Body>
oxh_status guarded(Body body) {
  try {
    return body();
  } catch (const std::exception &e) {
    return oxh::fail(OXH_EXECUTION, e.what());
  }
}

oxh_status check_workspace(uint64_t needed, const void *workspace, uint64_t bytes) {
  OXH_REQUIRE(needed == 0 || (workspace != nullptr && bytes >= needed &&
                              oxh::aligned16(workspace)),
              OXH_INVALID_SHAPE, "muon: workspace too small or misaligned");
  return oxh::ok();
}

}  // namespace

extern "C" {

oxh_status oxh_orthogonalize_workspace_size(uint64_t count, uint64_t rows, uint64_t columns,
                                            uint64_t *bytes) {
  return guarded([&]() -> oxh_status {
    OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
    *bytes = 0;
    if (count == 0) return oxh::ok();
    oxh_status st = check_sides(rows, columns);
    if (st != OXH_OK) return st;
    OXH_REQUIRE(count <= 65536, OXH_INVALID_SHAPE, "orthogonalize: too many matrices");
    *bytes = scratch_of_all(
        part(std::vector<Item>(count, Item{nullptr, nullptr, nullptr, rows, columns})));
    return oxh::ok();
  });
}

oxh_status oxh_orthogonalize(oxh_stream stream, uint64_t count, uint64_t rows, uint64_t columns,
                             uint32_t rounds, float epsilon, const float *input, float *output,
                             void *workspace, uint64_t workspace_bytes) {
  return guarded([&]() -> oxh_status {
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
                    (needed == 0 || (!oxh::any_overlap(workspace, needed, input, bytes) &&
                                     !oxh::any_overlap(workspace, needed, output, bytes))),
                OXH_INVALID_SHAPE, "orthogonalize: buffers overlap");
    std::vector<Item> items;
    for (uint64_t i = 0; i < count; ++i)
      items.push_back({input + i * rows * columns, nullptr, output + i * rows * columns, rows,
                       columns});
    return run_all(oxh::as_stream(stream), part(items), {0.0f, 0.0f, 0.0f, epsilon, false}, rounds,
                   static_cast<char *>(workspace));
  });
}

oxh_status oxh_muon_workspace_size(const oxh_muon_tensor *tensors, uint32_t count,
                                   uint64_t *bytes) {
  return guarded([&]() -> oxh_status {
    OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
    std::vector<Item> items;
    oxh_status st = items_of(tensors, count, items);
    if (st != OXH_OK) return st;
    *bytes = scratch_of_all(part(items));
    return oxh::ok();
  });
}

oxh_status oxh_muon_multi_tensor(oxh_stream stream, float learning_rate, float weight_decay,
                                 float momentum, int nesterov, float epsilon, uint32_t rounds,
                                 const oxh_muon_tensor *tensors, uint32_t count, void *workspace,
                                 uint64_t workspace_bytes) {
  return guarded([&]() -> oxh_status {
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
    const Parted parted = part(items);
    const uint64_t needed = scratch_of_all(parted);
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
    if (needed != 0) add(workspace, needed, true);
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
    return run_all(oxh::as_stream(stream), parted,
                   {learning_rate, weight_decay, momentum, epsilon, nesterov != 0}, rounds,
                   static_cast<char *>(workspace));
  });
}

}  // extern "C"
