// recurrence.hip -- the gated linear recurrence along the time axis of [batch, time, channels], and
// its gradients.
//
//   a_t = sigmoid(g_t);  h_t = a_t h_{t-1} + (1 - a_t) u_t          per batch row and channel
//   l_t = dh_t + a_{t+1} l_{t+1};  du_t = (1 - a_t) l_t;
//   dg_t = a_t (1 - a_t) (h_{t-1} - u_t) l_t;  dh_0 = a_1 l_1
//
// A row's steps at or past its length give 0, take no gradient and leave the state.  No
// counterpart in the reference, which has no layer along a sequence.
//
// Composing two steps' maps h -> a h + b is associative, so time is cut into tiles that a block
// scans, and into segments where rows and channels alone leave compute units idle.  The bound is
// memory: forward 8 x 2048 x 2048 float32 takes 80 us (5.0 TB/s), backward 153 us (5.3 TB/s).
// Split, the operands are read twice: forward 1 x 131072 x 512 bfloat16 takes 56 us for the
// segments' maps and 68 us for the states, 671 MB at 5.4 TB/s (one pass over its 403 MB would need
// the segments' states handed on inside one launch).  A single step of 64 x 2048 takes 3.4 us, a
// launch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "common.h"
#include "storage.h"

namespace {

using oxh::storage::bf16;
using oxh::storage::widen;

// sigmoid(g) and 1 - sigmoid(g): with e = exp(-g) they are r = 1 / (1 + e) and e r, the latter as
// 1 - r (exact enough above 1/2) where g < 0, since e may overflow there.  With u = 2^-24 the larger
// one is within 4 u; the smaller within (8 + 1.25 |g|) u, as exp2 takes g log2(e) rounded (measured
// 64 u at |g| = 86), and 0 beyond |g| = 88, where it would be denormal.  That rounding carried along
// (three operations a gate) leaves 3 u at any gate and costs what the caches or few waves do not
// hide: backward bfloat16 8 x 2048 x 2048 115 us and 110, 6 x 11621 x 112 27.8 and 25.1, forward 1 x
// 131072 x 512 125 and 120, float32 55 x 39 x 2907 19.6 and 18.3.
struct Gate {
  float keep, take;
};
__device__ __forceinline__ Gate gate_of(float g) {
  const float e = __builtin_amdgcn_exp2f(g * -1.44269504f);
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  return {r, g < 0.0f ? 1.0f - r : e * r};
}

struct Layout {
  uint32_t time, channels, groups;  // groups: blocks across the channels
  uint32_t segments, steps;         // steps per segment
  bool lines;                       // every group's channels of a step are whole lines of memory
};
// Both directions run h -> keep h + add over their steps in the order taken (backwards in time
// for the gradients, where h is a_{t+1} l_{t+1}, the gradient that reaches step t from later ones,
// and add = a_t dh_t).
template <typename T>
struct Args : Layout {
  const T *u, *g, *h, *dh;  // forward: u, g
  T *out, *dg;              // h, or du and dg
  const float *first;       // the state before the first step taken, or null
  const float *origin;      // backward: h before step 0, or null
  float *last;              // the one after the last, or null
  const int32_t *lengths;
  float *parts;  // per batch row: entry 0 the first state, entry s + 1 segment s's (keep, add)
};

__device__ __forceinline__ uint32_t length_of(const int32_t *lengths, uint32_t row,
                                              uint32_t time) {
  if (lengths == nullptr) return time;
  const int32_t n = lengths[row];
  return n < 0 ? 0u : min(static_cast<uint32_t>(n), time);
}

template <typename T, int V>
using Raw = typename oxh::storage::Pack<T, V>::type;

template <typename T, int V, bool Once = false>
__device__ __forceinline__ Raw<T, V> raw_load(const T *p) {
  if constexpr (Once) return __builtin_nontemporal_load(reinterpret_cast<const Raw<T, V> *>(p));
  else return *reinterpret_cast<const Raw<T, V> *>(p);
}
template <typename T, int V>
__device__ __forceinline__ float part_of(const Raw<T, V> &x, int v) {
  if constexpr (V == 1) return widen(x);
  else return widen(x[v]);
}

// A map h -> a h + b of V channels.
template <int V>
struct Map {
  float a[V], b[V];
  __device__ __forceinline__ void identity() {
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = 1.0f, b[v] = 0.0f;
  }
  // this map after `before`
  __device__ __forceinline__ void after(const Map &before) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      b[v] = fmaf(a[v], before.b[v], b[v]);
      a[v] *= before.a[v];
    }
  }
};

// The maps of all threads that share channels composed in time order.  A block is W waves of
// 64 / Lanes time groups of Lanes threads; `mine` becomes the composition of the groups before
// this thread's, and the whole block's is returned.  `shared` [W][2][Lanes * V]; two buffers in
// turn need one barrier per call.
template <int V, int Lanes, int W>
__device__ __forceinline__ Map<V> scan_groups(Map<V> &mine, float *shared) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % Lanes;
  Map<V> upto = mine;
#pragma unroll
  for (int d = Lanes; d < 64; d *= 2) {
    Map<V> before;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      before.a[v] = __shfl_up(upto.a[v], d);
      before.b[v] = __shfl_up(upto.b[v], d);
    }
    if (lane >= static_cast<uint32_t>(d)) upto.after(before);
  }
  if constexpr (W > 1) {
    if (lane >= 64 - Lanes) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        shared[(wave * 2) * Lanes * V + c * V + v] = upto.a[v];
        shared[(wave * 2 + 1) * Lanes * V + c * V + v] = upto.b[v];
      }
    }
  }
  // exclusive within the wave
#pragma unroll
  for (int v = 0; v < V; ++v) {
    mine.a[v] = Lanes < 64 ? __shfl_up(upto.a[v], Lanes & 63) : 1.0f;
    mine.b[v] = Lanes < 64 ? __shfl_up(upto.b[v], Lanes & 63) : 0.0f;
  }
  if (lane < Lanes) mine.identity();
  if constexpr (W == 1) {
    Map<V> all;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      all.a[v] = Lanes < 64 ? __shfl(upto.a[v], 64 - Lanes + c) : upto.a[v];
      all.b[v] = Lanes < 64 ? __shfl(upto.b[v], 64 - Lanes + c) : upto.b[v];
    }
    return all;
  } else {
    __syncthreads();
    Map<V> all;
    all.identity();
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w == static_cast<int>(wave)) mine.after(all);
      Map<V> next;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        next.a[v] = shared[(w * 2) * Lanes * V + c * V + v];
        next.b[v] = shared[(w * 2 + 1) * Lanes * V + c * V + v];
      }
      next.after(all);
      all = next;
    }
    return all;
  }
}

struct Place {
  uint32_t row, segment, channel;
  bool in;        // the thread's channels exist
  uint32_t skip;  // the first ones that are another thread's
};
template <int V, int Lanes, bool Ragged>
__device__ __forceinline__ Place place_of(const Layout &l) {
  const uint32_t id = l.lines ? blockIdx.x : oxh::xcd_contiguous(blockIdx.x, gridDim.x);
  const uint32_t group = id % l.groups, rest = id / l.groups, channels = l.channels;
  Place p;
  p.segment = rest % l.segments;
  p.row = rest / l.segments;
  p.channel = group * Lanes * V + (threadIdx.x % Lanes) * V;
  p.in = p.channel < channels;
  p.skip = 0;
  if (Ragged && p.in) {
    const oxh::storage::Places at = oxh::storage::places_at<V, Ragged>(p.channel, channels);
    p.channel = at.start;
    p.skip = at.skip;
  }
  return p;
}

// The steps below the row's length, a range of the steps in the order taken.
struct Live {
  uint32_t begin, end;
};
template <bool Back, typename T>
__device__ __forceinline__ Live live_of(const Args<T> &a, uint32_t row) {
  const uint32_t n = length_of(a.lengths, row, a.time);
  return Back ? Live{a.time - n, a.time} : Live{0, n};
}

// Offset of the thread's channels at time 0 (of channel 0 for threads without, whose loads then
// stay in bounds and whose results go nowhere), and of the k-th step taken behind it.
template <int V, typename T>
__device__ __forceinline__ uint64_t row_start(const Args<T> &a, const Place &p) {
  return static_cast<uint64_t>(p.row) * a.time * a.channels + (p.in ? p.channel : 0);
}
template <bool Back, typename T>
__device__ __forceinline__ uint64_t row_of(const Args<T> &a, uint32_t k) {
  return static_cast<uint64_t>(Back ? a.time - 1 - k : k) * a.channels;
}

template <int V>
__device__ __forceinline__ void load_state(const float *p, float (&h)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = p[v];
}
template <int V>
__device__ __forceinline__ void store_state(float *p, uint32_t skip, const float (&h)[V]) {
#pragma unroll
  for (uint32_t v = 0; v < V; ++v)
    if (v >= skip) p[v] = h[v];
}

// Where the time axis is split: segment s's map to entry s + 1 of `parts`, and the first state to
// entry 0.  Each time group takes a run of the segment's steps of its own.
template <typename T, int V, int Lanes, int W, int S, bool Back, bool Ragged>
__global__ __launch_bounds__(64 * W) void recurrence_parts_kernel(Args<T> a) {
  __shared__ float shared[W * 2 * Lanes * V];
  constexpr uint32_t kGroups = 64 / Lanes * W;
  const Place p = place_of<V, Lanes, Ragged>(a);
  const Live live = live_of<Back>(a, p.row);
  const uint32_t share = (a.steps + kGroups - 1) / kGroups;
  const uint32_t first = p.segment * a.steps + threadIdx.x / Lanes * share;
  const uint32_t begin = max(first, live.begin);
  const uint32_t end = min(min(first + share, (p.segment + 1) * a.steps), live.end);
  const T *add = (Back ? a.dh : a.u) + row_start<V>(a, p), *gates = a.g + row_start<V>(a, p);
  Map<V> map;
  map.identity();
  auto step = [&](const Raw<T, V> &x, const Raw<T, V> &g) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Gate gate = gate_of(part_of<T, V>(g, v));
      const float b = (Back ? gate.keep : gate.take) * part_of<T, V>(x, v);
      map.b[v] = fmaf(gate.keep, map.b[v], b);
      map.a[v] *= gate.keep;
    }
  };
  uint32_t k = begin;
  for (; k + S <= end; k += S) {
    Raw<T, V> x[S], g[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const uint64_t at = row_of<Back>(a, k + s);
      x[s] = raw_load<T, V>(add + at);
      g[s] = raw_load<T, V>(gates + at);
    }
#pragma unroll
    for (int s = 0; s < S; ++s) step(x[s], g[s]);
  }
  for (; k < end; ++k) {
    const uint64_t at = row_of<Back>(a, k);
    step(raw_load<T, V>(add + at), raw_load<T, V>(gates + at));
  }
  const Map<V> all = scan_groups<V, Lanes, W>(map, shared);
  if (!p.in || threadIdx.x >= Lanes) return;
  float *entry = a.parts + (static_cast<uint64_t>(p.row) * (a.segments + 1) + p.segment + 1) * 2 *
                               a.channels + p.channel;
  store_state<V>(entry, p.skip, all.a);
  store_state<V>(entry + a.channels, p.skip, all.b);
  if (p.segment == 0) {
    float h[V] = {};
    if (a.first != nullptr)
      load_state<V>(a.first + static_cast<uint64_t>(p.row) * a.channels + p.channel, h);
    store_state<V>(entry - a.channels, p.skip, h);
  }
}

// The recurrence over one segment (the whole time axis where it is not split), in tiles of
// kGroups * S steps: each thread composes its S steps, the block scans the compositions, and each
// thread runs its steps again from the state that reaches them.  The next tile's operands are
// loaded before the present one's work.
// Once: what it moves is far more than the caches hold, and bypasses them.
template <typename T, int V, int Lanes, int W, int S, bool Back, bool Ragged, bool Once = false>
__global__ __launch_bounds__(64 * W) void recurrence_kernel(Args<T> a) {
  __shared__ float shared[2][W * 2 * Lanes * V];
  constexpr uint32_t kGroups = 64 / Lanes * W, kTile = kGroups * S;
  Place p = place_of<V, Lanes, Ragged>(a);
  const Live live = live_of<Back>(a, p.row);
  const uint32_t group = threadIdx.x / Lanes;
  const uint64_t row = row_start<V>(a, p);
  const uint64_t state = static_cast<uint64_t>(p.row) * a.channels + (p.in ? p.channel : 0);
  float h[V] = {};  // before the tile
  int turn = 0;
  if (a.segments > 1) {
    // the entries before this segment, shared out among the time groups
    const float *entry = a.parts + (p.in ? p.channel : 0) +
                         static_cast<uint64_t>(p.row) * (a.segments + 1) * 2 * a.channels;
    const uint32_t share = (p.segment + kGroups - 1) / kGroups;
    const uint32_t begin = group * share, end = min(begin + share, p.segment);
    Map<V> map;
    map.identity();
    for (uint32_t s = begin; s < end; ++s) {
      const float *e = entry + static_cast<uint64_t>(s + 1) * 2 * a.channels;
      Map<V> next;
      load_state<V>(e, next.a);
      load_state<V>(e + a.channels, next.b);
      next.after(map);
      map = next;
    }
    load_state<V>(entry + a.channels, h);
    const Map<V> all = scan_groups<V, Lanes, W>(map, shared[turn]);
    turn ^= 1;
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = fmaf(all.a[v], h[v], all.b[v]);
  } else if (a.first != nullptr) {
    load_state<V>(a.first + state, h);
  }

  const uint32_t begin = p.segment * a.steps, end = min(begin + a.steps, a.time);
  const uint32_t live_end = min(end, live.end);
  constexpr int kOperands = Back ? 4 : 2;
  Raw<T, V> next[kOperands][S];
  auto load_step = [&](int s, uint32_t k) {
    const uint64_t at = row + row_of<Back>(a, k);
    next[0][s] = raw_load<T, V, Once>((Back ? a.dh : a.u) + at);
    next[1][s] = raw_load<T, V, Once>(a.g + at);
    if constexpr (Back) {
      next[2][s] = raw_load<T, V, Once>(a.u + at);
      if (k + 1 != a.time) next[3][s] = raw_load<T, V, Once>(a.h + at - a.channels);
    }
  };
  // whether every step of a tile is live (and, backwards, has a step before it)
  auto whole = [&](uint32_t tile) {
    return tile >= live.begin && tile + kTile <= live_end &&
           (!Back || tile + kTile < a.time);
  };
  auto fetch = [&](uint32_t tile) {
    const uint32_t k = tile + group * S;
    if (whole(tile)) {
#pragma unroll
      for (int s = 0; s < S; ++s) load_step(s, k + s);
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (k + s >= live.begin && k + s < live_end) load_step(s, k + s);
    }
  };
  float keep[S][V], add[S][V], take[S][V], slope[S][V];
  Map<V> map;
  auto compose = [&](uint32_t tile, auto all_live) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const uint32_t k = tile + group * S + s;
      const bool on = decltype(all_live)::value ||
                      (k >= live.begin && k < live_end);
      const bool oldest = !decltype(all_live)::value && Back && k + 1 == a.time;
      float before[V] = {};
      if (oldest && a.origin != nullptr) load_state<V>(a.origin + state, before);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gate gate = gate_of(part_of<T, V>(next[1][s], v));
        const float x = part_of<T, V>(next[0][s], v);
        keep[s][v] = on ? gate.keep : 1.0f;
        if constexpr (Back) {
          const float prev = oldest ? before[v] : part_of<T, V>(next[3][s], v);
          add[s][v] = on ? x : 0.0f;  // dh
          take[s][v] = on ? gate.take : 0.0f;
          slope[s][v] = on ? prev - part_of<T, V>(next[2][s], v) : 0.0f;
          map.b[v] = keep[s][v] * (map.b[v] + add[s][v]);
        } else {
          add[s][v] = on ? gate.take * x : 0.0f;
          map.b[v] = fmaf(keep[s][v], map.b[v], add[s][v]);
        }
        map.a[v] *= keep[s][v];
      }
    }
  };
  // x: the state before this thread's steps
  auto finish = [&](uint32_t tile, float (&x)[V], auto all_live) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const uint32_t k = tile + group * S + s;
      const bool on = decltype(all_live)::value || (k >= live.begin && k < live_end);
      if (!decltype(all_live)::value && k >= end) continue;
      const uint64_t at = row + row_of<Back>(a, k);
      float y[V], z[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if constexpr (Back) {  // beyond the length take and slope are 0, but l need not be finite
          const float l = x[v] + add[s][v];
          y[v] = on ? take[s][v] * l : 0.0f;
          z[v] = keep[s][v] * y[v] * slope[s][v];
          x[v] = keep[s][v] * l;
        } else {
          x[v] = fmaf(keep[s][v], x[v], add[s][v]);
          y[v] = on ? x[v] : 0.0f;
        }
      }
      const oxh::storage::Places here{0, p.skip};
      oxh::storage::store_places<T, V, Ragged, Once>(a.out + at, here, y);
      if constexpr (Back) oxh::storage::store_places<T, V, Ragged, Once>(a.dg + at, here, z);
    }
  };
  if (begin < end) fetch(begin);
  for (uint32_t tile = begin; tile < end; tile += kTile) {
    const bool all_live = whole(tile);
    map.identity();
    if (all_live) compose(tile, std::true_type());
    else compose(tile, std::false_type());
    if (tile + kTile < end) fetch(tile + kTile);
    const Map<V> all = scan_groups<V, Lanes, W>(map, shared[turn]);
    turn ^= 1;
    float x[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      x[v] = fmaf(map.a[v], h[v], map.b[v]);
      h[v] = fmaf(all.a[v], h[v], all.b[v]);
    }
    if (!p.in) continue;
    // whole tiles without their lengths' questions; backward over segments, of few tiles each, one
    // form is faster (5 x 1537 x 333 bfloat16 14.1 us and 14.4; 8 x 2048 x 2048 whole 112.0 and 110.7)
    if (!(Back && W == 4) && all_live) finish(tile, x, std::true_type());
    else finish(tile, x, std::false_type());
  }
  // every thread has read the first state, which may lie where the last one goes
  __syncthreads();
  if (a.last != nullptr && p.in && p.segment + 1 == a.segments && group == 0)
    store_state<V>(a.last + state, p.skip, h);
}

std::string message(const char *what, const char *problem) {
  return std::string(what) + problem;
}

struct Span {
  const void *p;
  uint64_t n;
};

// Outputs distinct from the operands and from each other; `same` names pairs that may be the same
// buffer (not overlap partly).
oxh_status check_apart(const char *what, const Span *in, int ins, const Span *out,
                       int outs, int same_in, int same_out) {
  for (int o = 0; o < outs; ++o) {
    if (out[o].p == nullptr || out[o].n == 0) continue;
    for (int i = 0; i < ins; ++i) {
      if (in[i].p == nullptr || in[i].n == 0) continue;
      if (i == same_in && o == same_out && in[i].p == out[o].p) continue;
      OXH_REQUIRE(!oxh::any_overlap(out[o].p, out[o].n, in[i].p, in[i].n), OXH_INVALID_SHAPE,
                  message(what, ": an output overlaps an operand"));
    }
    for (int k = 0; k < o; ++k)
      OXH_REQUIRE(out[k].p == nullptr || out[k].n == 0 ||
                      !oxh::any_overlap(out[o].p, out[o].n, out[k].p, out[k].n),
                  OXH_INVALID_SHAPE, message(what, ": two outputs overlap"));
  }
  return oxh::ok();
}

bool aligned_to(const void *p, uint64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

oxh_status check_shape(const char *what, int dtype, uint64_t batch, uint64_t time,
                       uint64_t channels) {
  OXH_REQUIRE(oxh::storage::valid(dtype), OXH_INVALID_SHAPE,
              message(what, ": dtype is neither OXH_F32 nor OXH_BF16"));
  OXH_REQUIRE(batch <= 65535, OXH_INVALID_SHAPE, message(what, ": batch above 65535"));
  OXH_REQUIRE(time < (1ull << 31) && channels < (1ull << 31), OXH_INVALID_SHAPE,
              message(what, ": time or channels too large"));
  OXH_REQUIRE(channels == 0 || batch * time <= (1ull << 58) / channels, OXH_INVALID_SHAPE,
              message(what, ": element count overflow"));
  return oxh::ok();
}

// How a call is laid out: the channels per thread and per block, the steps per thread and tile,
// and the segments of the time axis.
struct Plan {
  int values, lanes;
  bool brief;
  uint32_t groups, segments, steps;
};

// Waves per block, and steps per thread and tile.  Eight waves of four steps (backward: two) hold
// the bytes in flight of four waves of eight in half the registers each, and more of them hide more
// (forward 8 x 2048 x 2048 float32 87 us, 94 with four; 10 x 356 x 855 12.6 and 15.7; over segments
// 5 x 1537 x 333 bfloat16 14.2 and 14.6; backward 8 x 2048 x 2048 float32 167 and 171).  Backward
// over segments takes four waves of two and twice the blocks, whose waits overlap freely (5 x 1537
// x 333 15.6 us, 18.3 with eight waves; 1 x 5824 x 955 23.1 and 24.2; 1 x 131072 x 512 198 and
// 200).
constexpr int kWaves = 8;
constexpr int waves_of(int values, bool back, bool split) {
  return back && split && values != 1 ? 4 : kWaves;
}
constexpr int steps_of(int values, bool back) { return (values == 1 ? 8 : 4) / (back ? 2 : 1); }

// A tile takes about as long as 9 MB moved (3 us), a second launch as two tiles, and it reads half
// the operands again.  So the time axis is taken whole where blocks across rows and channels give
// every compute unit one, or where its tiles are at most two and one more for each 3 MB of a tensor
// (8 x 2048 x 512 float32, 8 tiles: 24.6 us whole, 28.7 split; 2 x 512 x 1024, 2 tiles: 7.6 and 12;
// 5 x 1537 x 333 bfloat16, 7 tiles: 23.7 and 14.2; 1 x 4096 x 2048 float32, 16 tiles: 41 and 30);
// there 32 channels per block where 64 leave more than half of the units without (8 x 2048 x 512,
// 64 blocks: 24.6 and 39; 10 x 356 x 855, 140 blocks: 15.4 and 12.6).  Otherwise it is split for
// two blocks of eight waves per unit, or four of four, a tile at least per segment (3 x 700 x 130:
// 10.5 us with one, 16.3 with two).
Plan plan_of(uint64_t batch, uint64_t time, uint64_t channels, uint64_t element, bool back) {
  Plan p;
  p.values = channels < 4 ? 1 : 4;
  auto across = [&](int lanes) {
    p.lanes = lanes;
    p.groups = static_cast<uint32_t>((channels + lanes * p.values - 1) / (lanes * p.values));
    return batch * p.groups;
  };
  auto tiles = [&](bool split, uint64_t &tile) {
    tile = 64 / p.lanes * waves_of(p.values, back, split) * steps_of(p.values, back);
    return (time + tile - 1) / tile;
  };
  p.segments = 1;
  p.steps = static_cast<uint32_t>(time);
  // 32 channels per block where there are no more (1 x 65536 x 32 bfloat16: 11.2 us, 16.8 with 64
  // per block) or up to 64 in few rows (1 x 65536 x 64: 14.0 and 16.2; 1000 x 33 x 64: 16.8 and
  // 10.1)
  const uint64_t units = oxh::kComputeUnits;
  const int lanes = p.values == 1 ? 32 : channels <= (batch < units ? 64 : 32) ? 8 : 16;
  const uint64_t blocks = across(lanes);
  // Few steps: one wave steps 256 channels one after the other, 4 loads ahead, at about 0.3 us a
  // step (64 x 4 x 2048 float32: 3.8 us, 16 in tiles; 4 x 16 x 1024 bfloat16: 6.2 and 5.0), while a
  // tile of idle steps takes as long as a full one (256 x 32 x 4096: 110 us, 33 by waves).
  p.brief = time <= std::min<uint64_t>(64, std::max<uint64_t>(8, blocks / 64));
  if (p.brief) across(64);
  if (p.brief || blocks >= units) return p;
  uint64_t tile;
  if (p.values == 4 && blocks * 2 < units) across(8);
  if (tiles(false, tile) <= 2 + batch * time * channels * element / (3u << 20)) return p;
  across(lanes);
  const uint64_t all = tiles(true, tile);
  // at most 256 segments, whose maps a block goes through (backward 1 x 30000 x 100 float32: 24 us,
  // 28 with 469)
  const uint64_t per_unit = 16 / waves_of(p.values, back, true);
  const uint64_t wanted =
      std::min({(per_unit * units + blocks - 1) / blocks, all, uint64_t{256}});
  if (wanted < 2) return p;
  const uint64_t per = (all + wanted - 1) / wanted;
  p.steps = static_cast<uint32_t>(per * tile);
  p.segments = static_cast<uint32_t>((all + per - 1) / per);
  return p;
}

uint64_t parts_bytes(const Plan &p, uint64_t batch, uint64_t channels) {
  return p.segments == 1 ? 0 : batch * (p.segments + 1) * 2 * channels * 4;
}

template <typename T, int V, int Lanes, bool Back, bool Ragged, int W>
oxh_status run_tiles(hipStream_t stream, uint64_t batch, Args<T> a, const char *what) {
  constexpr int S = steps_of(V, Back);
  const uint64_t blocks = batch * a.groups * a.segments;
  if (a.segments > 1) {
    oxh::launch(recurrence_parts_kernel<T, V, Lanes, W, S, Back, Ragged>,
                dim3(static_cast<uint32_t>(blocks)), dim3(64 * W), 0, stream, a);
    oxh_status st = oxh::launched(what);
    if (st != OXH_OK) return st;
  }
  // What passes beyond the 256 MB last-level cache is not kept there, where blocks write whole
  // lines (backward 8 x 2048 x 2048 float32, 805 MB: 160 us, 172 with the default policy; forward
  // 1 x 131072 x 512 bfloat16, 403 MB: 128 and 152; off lines it costs: backward 8 x 2048 x 2048
  // bfloat16 161 us, 118 with the default); smaller calls leave their results to the next one.
  constexpr uint64_t kCached = 256ull << 20;
  const uint64_t moved = batch * a.time * a.channels * sizeof(T) * (Back ? 6 : 3);
  if constexpr (V == 4 && Lanes == 16) {
    if (moved > kCached && a.lines) {
      oxh::launch(recurrence_kernel<T, V, Lanes, W, S, Back, Ragged, true>,
                  dim3(static_cast<uint32_t>(blocks)), dim3(64 * W), 0, stream, a);
      return oxh::launched(what);
    }
  }
  oxh::launch(recurrence_kernel<T, V, Lanes, W, S, Back, Ragged>,
              dim3(static_cast<uint32_t>(blocks)), dim3(64 * W), 0, stream, a);
  return oxh::launched(what);
}

template <typename T, int V, int Lanes, bool Back, bool Ragged>
oxh_status run_split(hipStream_t stream, uint64_t batch, const Args<T> &a, const char *what) {
  constexpr int kWhole = waves_of(V, Back, false), kSplit = waves_of(V, Back, true);
  if (kSplit != kWhole && a.segments > 1)
    return run_tiles<T, V, Lanes, Back, Ragged, kSplit>(stream, batch, a, what);
  return run_tiles<T, V, Lanes, Back, Ragged, kWhole>(stream, batch, a, what);
}

template <typename T, bool Back, int V, bool Ragged>
oxh_status run_plan(hipStream_t stream, uint64_t batch, const Args<T> &a, const Plan &p,
                    const char *what) {
  if (p.brief) {
    const dim3 grid(static_cast<uint32_t>(batch * p.groups));
    oxh::launch(recurrence_kernel<T, V, 64, 1, 4, Back, Ragged>, grid, dim3(64), 0, stream, a);
    return oxh::launched(what);
  }
  if constexpr (V == 1) {
    return run_split<T, 1, 32, Back, Ragged>(stream, batch, a, what);
  } else {
    return p.lanes == 8 ? run_split<T, 4, 8, Back, Ragged>(stream, batch, a, what)
                        : run_split<T, 4, 16, Back, Ragged>(stream, batch, a, what);
  }
}

template <typename T, bool Back>
oxh_status run(hipStream_t stream, uint64_t batch, Args<T> a, const char *what) {
  const Plan p = plan_of(batch, a.time, a.channels, sizeof(T), Back);
  a.groups = p.groups;
  a.segments = p.segments;
  a.steps = p.steps;
  // Lines that two groups share stay in one L2 if neighbouring blocks are on one XCD (forward 8 x
  // 2048 x 2048 bfloat16 16 bytes off a line: 42 us, 60 without; backward 1 x 5824 x 955 24 and
  // 34); those of their own are better spread over the XCDs (forward 16 x 1024 x 4096 bfloat16: 83
  // us, 104 together).
  constexpr uint64_t kLine = 128;
  a.lines = a.channels * sizeof(T) % kLine == 0 &&
            p.lanes * p.values * sizeof(T) % kLine == 0;
  for (const void *x : {static_cast<const void *>(a.u), static_cast<const void *>(a.g),
                        static_cast<const void *>(a.h), static_cast<const void *>(a.dh),
                        static_cast<const void *>(a.out), static_cast<const void *>(a.dg)})
    a.lines = a.lines && aligned_to(x, kLine);
  // a launch numbers its threads with 32 bits
  const uint64_t waves = p.brief ? 1 : waves_of(p.values, Back, p.segments > 1);
  OXH_REQUIRE(batch * p.groups * p.segments * 64 * waves < (1ull << 32), OXH_INVALID_SHAPE,
              std::string(what) + ": too many rows and channels for one launch");
  if (p.values == 1) return run_plan<T, Back, 1, false>(stream, batch, a, p, what);
  return a.channels % 4 == 0 ? run_plan<T, Back, 4, false>(stream, batch, a, p, what)
                             : run_plan<T, Back, 4, true>(stream, batch, a, p, what);
}

template <typename T>
oxh_status forward(hipStream_t stream, uint64_t batch, const void *input, const void *gate,
                   const float *initial_state, const int32_t *lengths, void *output,
                   float *final_state, void *workspace, uint32_t time, uint32_t channels) {
  Args<T> a{};
  a.u = static_cast<const T *>(input);
  a.g = static_cast<const T *>(gate);
  a.out = static_cast<T *>(output);
  a.first = initial_state;
  a.last = final_state;
  a.lengths = lengths;
  a.parts = static_cast<float *>(workspace);
  a.time = time;
  a.channels = channels;
  return run<T, false>(stream, batch, a, "gated_recurrence_forward");
}

template <typename T>
oxh_status backward(hipStream_t stream, uint64_t batch, const void *gradient, const void *input,
                    const void *gate, const void *output, const float *initial_state,
                    const float *final_state_gradient, const int32_t *lengths,
                    void *input_gradient, void *gate_gradient, float *initial_state_gradient,
                    void *workspace, uint32_t time, uint32_t channels) {
  Args<T> a{};
  a.dh = static_cast<const T *>(gradient);
  a.u = static_cast<const T *>(input);
  a.g = static_cast<const T *>(gate);
  a.h = static_cast<const T *>(output);
  a.out = static_cast<T *>(input_gradient);
  a.dg = static_cast<T *>(gate_gradient);
  a.first = final_state_gradient;
  a.origin = initial_state;
  a.last = initial_state_gradient;
  a.lengths = lengths;
  a.parts = static_cast<float *>(workspace);
  a.time = time;
  a.channels = channels;
  return run<T, true>(stream, batch, a, "gated_recurrence_backward");
}

}  // namespace

extern "C" {

oxh_status oxh_gated_recurrence_workspace_size(uint64_t batch, uint64_t time, uint64_t channels,
                                               uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  oxh_status st = check_shape("gated recurrence", OXH_F32, batch, time, channels);
  if (st != OXH_OK) return st;
  *bytes = 0;
  if (batch == 0 || channels == 0) return oxh::ok();
  for (const uint64_t element : {2, 4})
    for (const bool back : {false, true})
      *bytes = std::max(*bytes, parts_bytes(plan_of(batch, time, channels, element, back), batch,
                                            channels));
  *bytes = (*bytes + 255) / 256 * 256;
  return oxh::ok();
}

oxh_status oxh_gated_recurrence_forward(oxh_stream stream, int dtype, uint64_t batch,
                                        uint64_t time, uint64_t channels, const void *input,
                                        const void *gate, const float *initial_state,
                                        const int32_t *lengths, void *output,
                                        float *final_state, void *workspace,
                                        uint64_t workspace_bytes) {
  const char *const what = "gated recurrence";
  oxh_status st = check_shape(what, dtype, batch, time, channels);
  if (st != OXH_OK) return st;
  if (batch == 0 || channels == 0) return oxh::ok();
  const uint64_t element = oxh::storage::bytes_of(dtype),
                 bytes = batch * time * channels * element, states = batch * channels * 4;
  OXH_REQUIRE(time == 0 || (input != nullptr && gate != nullptr && output != nullptr),
              OXH_INVALID_SHAPE, message(what, ": null pointer"));
  OXH_REQUIRE(aligned_to(input, element) && aligned_to(gate, element) &&
                  aligned_to(output, element) && aligned_to(initial_state, 4) &&
                  aligned_to(final_state, 4) && aligned_to(lengths, 4),
              OXH_INVALID_SHAPE, message(what, ": a pointer is not aligned to its elements"));
  uint64_t needed = 0;
  st = oxh_gated_recurrence_workspace_size(batch, time, channels, &needed);
  if (st != OXH_OK) return st;
  OXH_REQUIRE(needed == 0 || (workspace != nullptr && workspace_bytes >= needed &&
                              oxh::aligned16(workspace)),
              OXH_INVALID_SHAPE, message(what, ": workspace too small or misaligned"));
  const Span in[] = {{input, bytes}, {gate, bytes}, {initial_state, states}, {lengths, batch * 4}};
  const Span out[] = {{output, bytes}, {final_state, states}, {workspace, needed}};
  st = check_apart(what, in, 4, out, 3, 2, 1);
  if (st != OXH_OK) return st;
  const uint32_t t = static_cast<uint32_t>(time), c = static_cast<uint32_t>(channels);
  const auto run_typed = dtype == OXH_F32 ? forward<float> : forward<bf16>;
  return run_typed(oxh::as_stream(stream), batch, input, gate, initial_state, lengths, output,
                   final_state, workspace, t, c);
}

oxh_status oxh_gated_recurrence_backward(
    oxh_stream stream, int dtype, uint64_t batch, uint64_t time, uint64_t channels,
    const void *gradient, const void *input, const void *gate, const void *output,
    const float *initial_state, const float *final_state_gradient, const int32_t *lengths,
    void *input_gradient, void *gate_gradient, float *initial_state_gradient, void *workspace,
    uint64_t workspace_bytes) {
  const char *const what = "gated recurrence backward";
  oxh_status st = check_shape(what, dtype, batch, time, channels);
  if (st != OXH_OK) return st;
  if (batch == 0 || channels == 0) return oxh::ok();
  const uint64_t element = oxh::storage::bytes_of(dtype),
                 bytes = batch * time * channels * element, states = batch * channels * 4;
  OXH_REQUIRE(time == 0 || (gradient != nullptr && input != nullptr && gate != nullptr &&
                            output != nullptr && input_gradient != nullptr &&
                            gate_gradient != nullptr),
              OXH_INVALID_SHAPE, message(what, ": null pointer"));
  OXH_REQUIRE(aligned_to(gradient, element) && aligned_to(input, element) &&
                  aligned_to(gate, element) && aligned_to(output, element) &&
                  aligned_to(input_gradient, element) && aligned_to(gate_gradient, element) &&
                  aligned_to(initial_state, 4) && aligned_to(final_state_gradient, 4) &&
                  aligned_to(initial_state_gradient, 4) && aligned_to(lengths, 4),
              OXH_INVALID_SHAPE, message(what, ": a pointer is not aligned to its elements"));
  uint64_t needed = 0;
  st = oxh_gated_recurrence_workspace_size(batch, time, channels, &needed);
  if (st != OXH_OK) return st;
  OXH_REQUIRE(needed == 0 || (workspace != nullptr && workspace_bytes >= needed &&
                              oxh::aligned16(workspace)),
              OXH_INVALID_SHAPE, message(what, ": workspace too small or misaligned"));
  const Span in[] = {{gradient, bytes},       {input, bytes},
                     {gate, bytes},           {output, bytes},
                     {initial_state, states}, {final_state_gradient, states},
                     {lengths, batch * 4}};
  const Span out[] = {{input_gradient, bytes},
                      {gate_gradient, bytes},
                      {initial_state_gradient, states},
                      {workspace, needed}};
  st = check_apart(what, in, 7, out, 4, 5, 2);
  if (st != OXH_OK) return st;
  const uint32_t t = static_cast<uint32_t>(time), c = static_cast<uint32_t>(channels);
  const auto run_typed = dtype == OXH_F32 ? backward<float> : backward<bf16>;
  return run_typed(oxh::as_stream(stream), batch, gradient, input, gate, output, initial_state,
                   final_state_gradient, lengths, input_gradient, gate_gradient,
                   initial_state_gradient, workspace, t, c);
}

}  // extern "C"
