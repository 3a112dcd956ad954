// recurrence.hip -- the gated linear recurrence along the time axis of [batch, time, channels], and
// its gradients.
//
//   a_t = sigmoid(g_t);  h_t = a_t h_{t-1} + (1 - a_t) u_t          per batch row and channel
//   l_t = dh_t + a_{t+1} l_{t+1};  du_t = (1 - a_t) l_t;
//   dg_t = a_t (1 - a_t) (h_{t-1} - u_t) l_t;  dh_0 = a_1 l_1
//
// A row's steps at or past its length give 0, take no gradient and leave the state.  No
// counterpart in the reference, which has no layer along a sequence.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "common.h"
#include "storage.h"

namespace {

using oxh::storage::bf16;
using oxh::storage::widen;

// sigmoid(g) and 1 - sigmoid(g), each to a few roundings however small: with e = exp(-|g|), they
// are 1 / (1 + e) and e / (1 + e), the larger one for the sign of g first.
struct Gate {
  float keep, take;
};
__device__ __forceinline__ Gate gate_of(float g) {
  const float e = __expf(-fabsf(g));
  const float large = __builtin_amdgcn_rcpf(1.0f + e), small = e * large;
  return g >= 0.0f ? Gate{large, small} : Gate{small, large};
}

template <typename T>
struct Forward {
  const T *u, *g;
  const float *state;
  T *h;
  float *final;
  const int32_t *lengths;
  uint32_t time, channels;
};

__device__ __forceinline__ uint32_t length_of(const int32_t *lengths, uint32_t row,
                                              uint32_t time) {
  if (lengths == nullptr) return time;
  const int32_t n = lengths[row];
  return n < 0 ? 0u : min(static_cast<uint32_t>(n), time);
}

template <typename T>
__global__ __launch_bounds__(64) void recurrence_forward_kernel(Forward<T> a) {
  const uint32_t c = blockIdx.x * 64 + threadIdx.x, row = blockIdx.y;
  if (c >= a.channels) return;
  const uint32_t n = length_of(a.lengths, row, a.time);
  const uint64_t at = static_cast<uint64_t>(row) * a.channels + c;
  uint64_t i = static_cast<uint64_t>(row) * a.time * a.channels + c;
  float h = a.state != nullptr ? a.state[at] : 0.0f;
  for (uint32_t t = 0; t < n; ++t, i += a.channels) {
    const Gate k = gate_of(widen(a.g[i]));
    h = fmaf(k.keep, h, k.take * widen(a.u[i]));
    a.h[i] = static_cast<T>(h);
  }
  for (uint32_t t = n; t < a.time; ++t, i += a.channels) a.h[i] = static_cast<T>(0.0f);
  if (a.final != nullptr) a.final[at] = h;
}

template <typename T>
struct Backward {
  const T *dh, *u, *g, *h;
  const float *state, *dfinal;
  T *du, *dg;
  float *dstate;
  const int32_t *lengths;
  uint32_t time, channels;
};

template <typename T>
__global__ __launch_bounds__(64) void recurrence_backward_kernel(Backward<T> a) {
  const uint32_t c = blockIdx.x * 64 + threadIdx.x, row = blockIdx.y;
  if (c >= a.channels) return;
  const uint32_t n = length_of(a.lengths, row, a.time);
  const uint64_t at = static_cast<uint64_t>(row) * a.channels + c;
  const uint64_t first = static_cast<uint64_t>(row) * a.time * a.channels + c;
  for (uint32_t t = n; t < a.time; ++t) {
    const uint64_t i = first + static_cast<uint64_t>(t) * a.channels;
    a.du[i] = a.dg[i] = static_cast<T>(0.0f);
  }
  float l = a.dfinal != nullptr ? a.dfinal[at] : 0.0f;
  for (uint32_t t = n; t-- > 0;) {
    const uint64_t i = first + static_cast<uint64_t>(t) * a.channels;
    const Gate k = gate_of(widen(a.g[i]));
    const float before = t != 0              ? widen(a.h[i - a.channels])
                         : a.state != nullptr ? a.state[at]
                                              : 0.0f;
    l += widen(a.dh[i]);
    const float taken = k.take * l;
    a.du[i] = static_cast<T>(taken);
    a.dg[i] = static_cast<T>(k.keep * taken * (before - widen(a.u[i])));
    l *= k.keep;
  }
  if (a.dstate != nullptr) a.dstate[at] = l;
}

struct Span {
  const void *p;
  uint64_t n;
};

// Outputs distinct from the operands and from each other; `same` names pairs that may be the same
// buffer (not overlap partly).
oxh_status check_apart(const std::string &what, const Span *in, int ins, const Span *out,
                       int outs, int same_in, int same_out) {
  for (int o = 0; o < outs; ++o) {
    if (out[o].p == nullptr || out[o].n == 0) continue;
    for (int i = 0; i < ins; ++i) {
      if (in[i].p == nullptr || in[i].n == 0) continue;
      if (i == same_in && o == same_out && in[i].p == out[o].p) continue;
      OXH_REQUIRE(!oxh::any_overlap(out[o].p, out[o].n, in[i].p, in[i].n), OXH_INVALID_SHAPE,
                  what + ": an output overlaps an operand");
    }
    for (int k = 0; k < o; ++k)
      OXH_REQUIRE(out[k].p == nullptr || out[k].n == 0 ||
                      !oxh::any_overlap(out[o].p, out[o].n, out[k].p, out[k].n),
                  OXH_INVALID_SHAPE, what + ": two outputs overlap");
  }
  return oxh::ok();
}

bool aligned_to(const void *p, uint64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

oxh_status check_shape(const std::string &what, int dtype, uint64_t batch, uint64_t time,
                       uint64_t channels) {
  OXH_REQUIRE(oxh::storage::valid(dtype), OXH_INVALID_SHAPE,
              what + ": dtype is neither OXH_F32 nor OXH_BF16");
  OXH_REQUIRE(batch <= 65535, OXH_INVALID_SHAPE, what + ": batch above 65535");
  OXH_REQUIRE(time < (1ull << 31) && channels < (1ull << 31), OXH_INVALID_SHAPE,
              what + ": time or channels too large");
  OXH_REQUIRE(channels == 0 || batch * time <= (1ull << 58) / channels, OXH_INVALID_SHAPE,
              what + ": element count overflow");
  return oxh::ok();
}

template <typename T>
oxh_status forward(hipStream_t stream, uint64_t batch, const Forward<T> &a) {
  oxh::launch(recurrence_forward_kernel<T>,
              dim3((a.channels + 63) / 64, static_cast<uint32_t>(batch)), dim3(64), 0, stream,
              a);
  return oxh::launched("gated_recurrence_forward");
}

template <typename T>
oxh_status backward(hipStream_t stream, uint64_t batch, const Backward<T> &a) {
  oxh::launch(recurrence_backward_kernel<T>,
              dim3((a.channels + 63) / 64, static_cast<uint32_t>(batch)), dim3(64), 0, stream,
              a);
  return oxh::launched("gated_recurrence_backward");
}

}  // namespace

extern "C" {

oxh_status oxh_gated_recurrence_workspace_size(uint64_t batch, uint64_t time, uint64_t channels,
                                               uint64_t *bytes) {
  OXH_REQUIRE(bytes != nullptr, OXH_INVALID_SHAPE, "bytes is null");
  oxh_status st = check_shape("gated recurrence", OXH_F32, batch, time, channels);
  if (st != OXH_OK) return st;
  *bytes = 256;
  return oxh::ok();
}

oxh_status oxh_gated_recurrence_forward(oxh_stream stream, int dtype, uint64_t batch,
                                        uint64_t time, uint64_t channels, const void *input,
                                        const void *gate, const float *initial_state,
                                        const int32_t *lengths, void *output,
                                        float *final_state, void *workspace,
                                        uint64_t workspace_bytes) {
  const std::string what = "gated recurrence";
  oxh_status st = check_shape(what, dtype, batch, time, channels);
  if (st != OXH_OK) return st;
  if (batch == 0 || channels == 0) return oxh::ok();
  const uint64_t element = oxh::storage::bytes_of(dtype),
                 bytes = batch * time * channels * element, states = batch * channels * 4;
  OXH_REQUIRE(time == 0 || (input != nullptr && gate != nullptr && output != nullptr),
              OXH_INVALID_SHAPE, what + ": null pointer");
  OXH_REQUIRE(aligned_to(input, element) && aligned_to(gate, element) &&
                  aligned_to(output, element) && aligned_to(initial_state, 4) &&
                  aligned_to(final_state, 4) && aligned_to(lengths, 4),
              OXH_INVALID_SHAPE, what + ": a pointer is not aligned to its elements");
  uint64_t needed = 0;
  st = oxh_gated_recurrence_workspace_size(batch, time, channels, &needed);
  if (st != OXH_OK) return st;
  OXH_REQUIRE(workspace != nullptr && workspace_bytes >= needed && oxh::aligned16(workspace),
              OXH_INVALID_SHAPE, what + ": workspace too small or misaligned");
  const Span in[] = {{input, bytes}, {gate, bytes}, {initial_state, states}, {lengths, batch * 4}};
  const Span out[] = {{output, bytes}, {final_state, states}, {workspace, needed}};
  st = check_apart(what, in, 4, out, 3, 2, 1);
  if (st != OXH_OK) return st;
  const uint32_t t = static_cast<uint32_t>(time), c = static_cast<uint32_t>(channels);
  if (dtype == OXH_F32)
    return forward<float>(oxh::as_stream(stream), batch,
                          {static_cast<const float *>(input), static_cast<const float *>(gate),
                           initial_state, static_cast<float *>(output), final_state, lengths, t,
                           c});
  return forward<bf16>(oxh::as_stream(stream), batch,
                       {static_cast<const bf16 *>(input), static_cast<const bf16 *>(gate),
                        initial_state, static_cast<bf16 *>(output), final_state, lengths, t, c});
}

oxh_status oxh_gated_recurrence_backward(
    oxh_stream stream, int dtype, uint64_t batch, uint64_t time, uint64_t channels,
    const void *gradient, const void *input, const void *gate, const void *output,
    const float *initial_state, const float *final_state_gradient, const int32_t *lengths,
    void *input_gradient, void *gate_gradient, float *initial_state_gradient, void *workspace,
    uint64_t workspace_bytes) {
  const std::string what = "gated recurrence backward";
  oxh_status st = check_shape(what, dtype, batch, time, channels);
  if (st != OXH_OK) return st;
  if (batch == 0 || channels == 0) return oxh::ok();
  const uint64_t element = oxh::storage::bytes_of(dtype),
                 bytes = batch * time * channels * element, states = batch * channels * 4;
  OXH_REQUIRE(time == 0 || (gradient != nullptr && input != nullptr && gate != nullptr &&
                            output != nullptr && input_gradient != nullptr &&
                            gate_gradient != nullptr),
              OXH_INVALID_SHAPE, what + ": null pointer");
  OXH_REQUIRE(aligned_to(gradient, element) && aligned_to(input, element) &&
                  aligned_to(gate, element) && aligned_to(output, element) &&
                  aligned_to(input_gradient, element) && aligned_to(gate_gradient, element) &&
                  aligned_to(initial_state, 4) && aligned_to(final_state_gradient, 4) &&
                  aligned_to(initial_state_gradient, 4) && aligned_to(lengths, 4),
              OXH_INVALID_SHAPE, what + ": a pointer is not aligned to its elements");
  uint64_t needed = 0;
  st = oxh_gated_recurrence_workspace_size(batch, time, channels, &needed);
  if (st != OXH_OK) return st;
  OXH_REQUIRE(workspace != nullptr && workspace_bytes >= needed && oxh::aligned16(workspace),
              OXH_INVALID_SHAPE, what + ": workspace too small or misaligned");
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
  if (dtype == OXH_F32)
    return backward<float>(
        oxh::as_stream(stream), batch,
        {static_cast<const float *>(gradient), static_cast<const float *>(input),
         static_cast<const float *>(gate), static_cast<const float *>(output), initial_state,
         final_state_gradient, static_cast<float *>(input_gradient),
         static_cast<float *>(gate_gradient), initial_state_gradient, lengths, t, c});
  return backward<bf16>(
      oxh::as_stream(stream), batch,
      {static_cast<const bf16 *>(gradient), static_cast<const bf16 *>(input),
       static_cast<const bf16 *>(gate), static_cast<const bf16 *>(output), initial_state,
       final_state_gradient, static_cast<bf16 *>(input_gradient),
       static_cast<bf16 *>(gate_gradient), initial_state_gradient, lengths, t, c});
}

}  // extern "C"
