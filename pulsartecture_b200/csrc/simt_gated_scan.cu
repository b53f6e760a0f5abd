// Gated linear recurrence on CUDA cores: per batch row and channel
//
//   a_t = sigmoid(gate_t) or gate_t,  b_t = (1 - a_t) x_t or x_t
//   h_t = a_t h_{t-1} + b_t
//
// and its gradient, with G_t = dout_t + a_{t+1} G_{t+1} (dstate added at the
// last token):
//
//   dx_t = G_t (1 - a_t) or G_t          da_t = G_t (h_{t-1} - x_t) or G_t h_{t-1}
//   dgate_t = da_t a_t (1 - a_t) or da_t  dstate_in = a_1 G_1
//
// h, G and all products are fp32 for either type; out, dx and dgate are
// rounded once. The forward keeps h before every kTile-th token in `saved`;
// the backward rebuilds the states in between from there, so it reads no
// rounded state.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "fakla_common.cuh"
#include "fakla_kernels.h"

namespace fakla {
namespace {

constexpr int kTile = 128;  // tokens between two kept states
constexpr int kThreads = 128;

// a and 1 - a from one exponential of -|g|: neither cancels, and g = +-inf
// gives exactly 0 and 1.
// bf16 gates take the hardware's exponential and reciprocal, whose error (a few
// 2^-24 of 1 - a or of a) is far below the gate's own rounding.
template <int ACT, typename T>
__device__ __forceinline__ void gate_pair(float g, float& a, float& rest) {
  if constexpr (ACT == FAKLA_ACT_SIGMOID) {
    constexpr bool kFast = sizeof(T) == 2;
    const float e = kFast ? __expf(-fabsf(g)) : expf(-fabsf(g));
    const float big = kFast ? __fdividef(1.f, 1.f + e) : 1.f / (1.f + e), small = e * big;
    a = g >= 0.f ? big : small;
    rest = g >= 0.f ? small : big;
  } else {
    a = g;
    rest = 1.f - g;
  }
}

template <typename T, int ACT, bool MIX>
__global__ void __launch_bounds__(kThreads) scan_forward_kernel(GatedScanArgs p) {
  const int64_t blocks = (p.D + kThreads - 1) / kThreads;
  const int64_t d = blockIdx.x % blocks * kThreads + threadIdx.x, b = blockIdx.x / blocks;
  if (d >= p.D) return;
  const T* x = (const T*)p.x + b * p.x_batch + d;
  const T* gate = (const T*)p.gate + b * p.gate_batch + d;
  T* out = (T*)p.out + b * p.T * p.D + d;
  float* saved = p.saved ? p.saved + b * ((p.T + kTile - 1) / kTile) * p.D + d : nullptr;
  float h = p.state_in ? p.state_in[b * p.D + d] : 0.f;
  for (int64_t t = 0; t < p.T; ++t) {
    if (saved && t % kTile == 0) saved[t / kTile * p.D] = h;
    float a, rest;
    gate_pair<ACT, T>(to_f32(gate[t * p.gate_time]), a, rest);
    const float v = to_f32(x[t * p.x_time]);
    h = fmaf(a, h, MIX ? rest * v : v);
    out[t * p.D] = from_f32<T>(h);
  }
  if (p.state_out) p.state_out[b * p.D + d] = h;
}

template <typename T, int ACT, bool MIX>
__global__ void __launch_bounds__(kThreads) scan_backward_kernel(GatedScanArgs p) {
  const int64_t blocks = (p.D + kThreads - 1) / kThreads;
  const int64_t d = blockIdx.x % blocks * kThreads + threadIdx.x, b = blockIdx.x / blocks;
  if (d >= p.D) return;
  const T* x = (const T*)p.x + b * p.x_batch + d;
  const T* gate = (const T*)p.gate + b * p.gate_batch + d;
  const T* dout = (const T*)p.dout + b * p.T * p.D + d;
  T* dx = (T*)p.dx + b * p.T * p.D + d;
  T* dgate = (T*)p.dgate + b * p.T * p.D + d;
  const int64_t tiles = (p.T + kTile - 1) / kTile;
  const float* saved = p.saved + b * tiles * p.D + d;
  float carry = p.dstate_out ? p.dstate_out[b * p.D + d] : 0.f;  // a_{t+1} G_{t+1}
  float before[kTile];
  for (int64_t tile = tiles - 1; tile >= 0; --tile) {
    const int64_t t0 = tile * kTile;
    const int n = (int)(p.T - t0 < kTile ? p.T - t0 : kTile);
    float h = saved[tile * p.D];
    for (int i = 0; i < n; ++i) {
      before[i] = h;
      float a, rest;
      gate_pair<ACT, T>(to_f32(gate[(t0 + i) * p.gate_time]), a, rest);
      const float v = to_f32(x[(t0 + i) * p.x_time]);
      h = fmaf(a, h, MIX ? rest * v : v);
    }
    for (int i = n - 1; i >= 0; --i) {
      float a, rest;
      gate_pair<ACT, T>(to_f32(gate[(t0 + i) * p.gate_time]), a, rest);
      const float v = to_f32(x[(t0 + i) * p.x_time]);
      const float G = to_f32(dout[(t0 + i) * p.D]) + carry;
      carry = a * G;
      const float da = G * (MIX ? before[i] - v : before[i]);
      dx[(t0 + i) * p.D] = from_f32<T>(MIX ? G * rest : G);
      dgate[(t0 + i) * p.D] = from_f32<T>(ACT == FAKLA_ACT_SIGMOID ? da * a * rest : da);
    }
  }
  if (p.dstate_in) p.dstate_in[b * p.D + d] = carry;
}

template <typename T, int ACT, bool MIX>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(GatedScanArgs p) {
  const int64_t blocks = (p.D + kThreads - 1) / kThreads;
  const int64_t d = blockIdx.x % blocks * kThreads + threadIdx.x, b = blockIdx.x / blocks;
  if (d >= p.D) return;
  float a, rest;
  gate_pair<ACT, T>(to_f32(((const T*)p.gate)[b * p.gate_batch + d]), a, rest);
  const float v = to_f32(((const T*)p.x)[b * p.x_batch + d]);
  const float h = fmaf(a, p.state_in[b * p.D + d], MIX ? rest * v : v);
  p.state_out[b * p.D + d] = h;
  ((T*)p.out)[b * p.D + d] = from_f32<T>(h);
}

// Runs f with the type, gate activation and input form as constants.
template <typename F>
void dispatch(int dtype, int act, bool mix, F f) {
  auto by_form = [&](auto t, auto a) {
    if (mix) f(t, a, std::true_type{}); else f(t, a, std::false_type{});
  };
  auto by_act = [&](auto t) {
    if (act == FAKLA_ACT_SIGMOID) by_form(t, std::integral_constant<int, FAKLA_ACT_SIGMOID>{});
    else by_form(t, std::integral_constant<int, FAKLA_ACT_IDENTITY>{});
  };
  if (dtype == FAKLA_BF16) by_act(__nv_bfloat16{}); else by_act(float{});
}

}  // namespace

size_t gated_scan_saved_bytes(int64_t B, int64_t T, int64_t D) {
  return (size_t)B * (size_t)((T + kTile - 1) / kTile) * (size_t)D * sizeof(float);
}

cudaError_t launch_gated_scan(int dtype, const GatedScanArgs& p, cudaStream_t stream) {
  const unsigned grid = (unsigned)((p.D + kThreads - 1) / kThreads * p.B);
  dispatch(dtype, p.act, p.mix, [&](auto t, auto act, auto mix) {
    scan_forward_kernel<decltype(t), act(), mix()><<<grid, kThreads, 0, stream>>>(p);
  });
  return cudaGetLastError();
}

cudaError_t launch_gated_scan_backward(int dtype, const GatedScanArgs& p, cudaStream_t stream) {
  const unsigned grid = (unsigned)((p.D + kThreads - 1) / kThreads * p.B);
  dispatch(dtype, p.act, p.mix, [&](auto t, auto act, auto mix) {
    scan_backward_kernel<decltype(t), act(), mix()><<<grid, kThreads, 0, stream>>>(p);
  });
  return cudaGetLastError();
}

cudaError_t launch_gated_scan_step(int dtype, const GatedScanArgs& p, cudaStream_t stream) {
  const unsigned grid = (unsigned)((p.D + kThreads - 1) / kThreads * p.B);
  dispatch(dtype, p.act, p.mix, [&](auto t, auto act, auto mix) {
    scan_step_kernel<decltype(t), act(), mix()><<<grid, kThreads, 0, stream>>>(p);
  });
  return cudaGetLastError();
}

}  // namespace fakla
