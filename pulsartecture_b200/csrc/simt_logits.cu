// Rows of logits on CUDA cores: token log probabilities with entropy and the
// largest entries, and the divergence from a teacher's largest logits, with
// their gradients.
//
// With y = x / temperature, m = max y and s = sum_j e^{y_j - m}:
//   log p_j = (y_j - m) - log s,  H = log s - (sum_j e^{y_j - m} (y_j - m)) / s,
// both sums of one sign, so neither cancels. The backward recomputes p from m
// and log s. Everything is fp32; dlogits are rounded once.
//
// A row of nothing but -inf (s = 0) keeps log s = +inf, which makes every p 0.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "fakla_common.cuh"
#include "fakla_kernels.h"

namespace fakla {
namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ const T* row_of(const LogitsArgs& p, int64_t row) {
  return (const T*)p.logits + row / p.rows * p.batch_stride + row % p.rows * p.row_stride;
}

template <typename V, typename F>
__device__ V block_reduce(V v, F f) {
  __shared__ V part[32];
  __syncthreads();
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
  __syncthreads();
  v = part[0];
  for (int i = 1; i < blockDim.x / 32; ++i) v = f(v, part[i]);
  return v;
}
__device__ float block_sum(float v) { return block_reduce(v, [](float a, float b) { return a + b; }); }
__device__ float block_max(float v) { return block_reduce(v, [](float a, float b) { return fmaxf(a, b); }); }

// Order of the values (-0 as 0), then of the lower index.
__device__ __forceinline__ uint64_t order_key(float x, int j) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)o << 32 | (uint32_t)~j;
}

struct RowStats {
  float m;     // max x, or 0 in a row of nothing but -inf
  float logs;  // log s; +inf in such a row, NaN in one with a NaN or +inf
  float ws;    // sum e (y - m) / s
};

template <typename T>
__device__ RowStats row_stats(const T* x, int64_t V, float inv_t) {
  float m = -CUDART_INF_F;
  for (int64_t j = threadIdx.x; j < V; j += blockDim.x) m = fmaxf(m, to_f32(x[j]));
  m = block_max(m);
  if (m == -CUDART_INF_F) m = 0.f;
  float s = 0.f, w = 0.f;
  for (int64_t j = threadIdx.x; j < V; j += blockDim.x) {
    const float d = (to_f32(x[j]) - m) * inv_t, e = expf(d);
    s += e;
    w += e == 0.f ? 0.f : e * d;
  }
  s = block_sum(s);
  w = block_sum(w);
  if (s == 0.f) return {m, CUDART_INF_F, 0.f};
  return {m, logf(s), w / s};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(LogitsArgs p) {
  const int64_t row = blockIdx.x;
  const T* x = row_of<T>(p, row);
  const RowStats r = row_stats(x, p.vocab, p.inv_temperature);
  const bool empty = r.logs == CUDART_INF_F;
  auto logprob = [&](int64_t j) {
    return empty ? -CUDART_INF_F : (to_f32(x[j]) - r.m) * p.inv_temperature - r.logs;
  };
  if (threadIdx.x == 0) {
    const int64_t t = p.targets[row];
    float lp = 0.f;
    if (t != p.ignore_index) {
      if (t >= 0 && t < p.vocab) {
        lp = logprob(t);
      } else {
        lp = CUDART_NAN_F;
        report_status(p.status, FAKLA_ERR_INVALID_ARG);
      }
    }
    p.logprobs[row] = lp;
    p.entropy[row] = empty ? 0.f : r.logs - r.ws;
    if (p.stats) {
      p.stats[row * kTokenStats] = r.m;
      p.stats[row * kTokenStats + 1] = r.logs;
    }
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < p.top_k; ++k) {
    uint64_t best = 0;
    for (int64_t j = threadIdx.x; j < p.vocab; j += blockDim.x) {
      const uint64_t key = order_key(to_f32(x[j]), (int)j);
      if (key < last && key > best) best = key;
    }
    last = block_reduce(best, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    if (threadIdx.x == 0) {
      const bool bad = isnan(r.logs);
      const int64_t j = ~(uint32_t)last;
      p.top_ids[row * p.top_k + k] = bad ? -1 : j;
      p.top_logprobs[row * p.top_k + k] = bad ? CUDART_NAN_F : logprob(j);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_backward_kernel(LogitsArgs p) {
  const int64_t row = blockIdx.x;
  const T* x = row_of<T>(p, row);
  T* dx = (T*)p.dlogits + row * p.vocab;
  const float m = p.stats[row * kTokenStats], logs = p.stats[row * kTokenStats + 1];
  const int64_t t = p.targets[row];
  const bool counted = t != p.ignore_index;
  float w = counted && p.dlogprobs ? p.dlogprobs[row] : 0.f;
  if (counted && (t < 0 || t >= p.vocab)) w = CUDART_NAN_F;
  const float h = p.dentropy ? p.dentropy[row] : 0.f, H = p.entropy[row];
  float total = w;
  if (p.dtop_logprobs)
    for (int k = 0; k < p.top_k; ++k) total += p.dtop_logprobs[row * p.top_k + k];
  const bool empty = logs == CUDART_INF_F;
  for (int64_t j = threadIdx.x; j < p.vocab; j += blockDim.x) {
    const float lp = (to_f32(x[j]) - m) * p.inv_temperature - logs, e = expf(lp);
    float dz = (counted && j == t ? w : 0.f) - total * e - (e == 0.f ? 0.f : h * e * (lp + H));
    if (p.dtop_logprobs)
      for (int k = 0; k < p.top_k; ++k)
        if (p.top_ids[row * p.top_k + k] == j) dz += p.dtop_logprobs[row * p.top_k + k];
    dx[j] = from_f32<T>(empty ? 0.f : dz * p.inv_temperature);
  }
}

// The teacher's side of a row: q_k = e^{t_k / temperature - m - logs}.
struct Teacher {
  float m, logs;  // logs +inf: no distribution, every q is 0
  float mass;     // sum of the q
  float rest;     // what is left for the other entries (teacher_lse given)
  bool bad;       // an id out of range
};

__device__ __forceinline__ float teacher_q(const LogitsArgs& p, int64_t row, int k, float m, float logs, float& lq) {
  lq = -CUDART_INF_F;
  if (p.teacher_ids[row * p.entries + k] < 0) return 0.f;
  lq = (p.teacher_logits[row * p.entries + k] - m) * p.inv_temperature - logs;
  return expf(lq);
}

__device__ Teacher teacher_stats(const LogitsArgs& p, int64_t row) {
  Teacher t = {0.f, 0.f, 0.f, 0.f, false};
  float m = -CUDART_INF_F;
  int bad = 0, some = 0;
  for (int k = threadIdx.x; k < p.entries; k += blockDim.x) {
    const int64_t id = p.teacher_ids[row * p.entries + k];
    bad |= id < -1 || id >= p.vocab;
    if (id < 0) continue;
    some = 1;
    m = fmaxf(m, p.teacher_logits[row * p.entries + k]);
  }
  t.bad = __syncthreads_or(bad);
  some = __syncthreads_or(some);
  if (p.teacher_lse) {
    t.logs = some ? p.teacher_lse[row] : CUDART_INF_F;
  } else {
    m = block_max(m);
    t.m = m == -CUDART_INF_F ? 0.f : m;
  }
  float s = 0.f, lq;
  for (int k = threadIdx.x; k < p.entries; k += blockDim.x) s += teacher_q(p, row, k, t.m, t.logs, lq);
  s = block_sum(s);
  if (p.teacher_lse) {
    t.mass = s;
    t.rest = some ? fmaxf(0.f, 1.f - s) : 0.f;
  } else {
    t.logs = s == 0.f ? CUDART_INF_F : logf(s);
    t.mass = s == 0.f ? 0.f : 1.f;
  }
  return t;
}

__device__ bool is_member(const LogitsArgs& p, int64_t row, int64_t j) {
  for (int k = 0; k < p.entries; ++k)
    if (p.teacher_ids[row * p.entries + k] == j) return true;
  return false;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_kernel(LogitsArgs p) {
  const int64_t row = blockIdx.x;
  const T* x = row_of<T>(p, row);
  const RowStats r = row_stats(x, p.vocab, p.inv_temperature);
  const Teacher t = teacher_stats(p, row);
  auto logprob = [&](int64_t j) {
    return r.logs == CUDART_INF_F ? -CUDART_INF_F : (to_f32(x[j]) - r.m) * p.inv_temperature - r.logs;
  };
  float loss = 0.f;
  if (!t.bad)
    for (int k = threadIdx.x; k < p.entries; k += blockDim.x) {
      float lq;
      const float q = teacher_q(p, row, k, t.m, t.logs, lq);
      if (q != 0.f) loss += q * (lq - logprob(p.teacher_ids[row * p.entries + k]));
    }
  loss = block_sum(loss);
  float ratio = 0.f;  // q_r / p_r
  if (p.teacher_lse && !t.bad) {
    float s = 0.f;
    for (int64_t j = threadIdx.x; j < p.vocab; j += blockDim.x)
      if (!is_member(p, row, j)) s += expf((to_f32(x[j]) - r.m) * p.inv_temperature - r.logs);
    s = block_sum(s);
    if (t.rest > 0.f) {
      ratio = t.rest / s;
      loss += t.rest * logf(ratio);
    }
  }
  if (threadIdx.x != 0) return;
  if (t.bad) {
    loss = CUDART_NAN_F;
    report_status(p.status, FAKLA_ERR_INVALID_ARG);
  }
  p.loss[row] = loss;
  if (p.stats) {
    float* st = p.stats + row * kDistillStats;
    st[0] = r.m;
    st[1] = r.logs;
    st[2] = t.m;
    st[3] = t.logs;
    st[4] = t.bad ? CUDART_NAN_F : t.mass + t.rest;
    st[5] = ratio;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(LogitsArgs p) {
  const int64_t row = blockIdx.x;
  const T* x = row_of<T>(p, row);
  T* dx = (T*)p.dlogits + row * p.vocab;
  const float* st = p.stats + row * kDistillStats;
  const float g = p.dloss[row] * p.inv_temperature;
  const bool empty = st[1] == CUDART_INF_F;
  for (int64_t j = threadIdx.x; j < p.vocab; j += blockDim.x) {
    const float e = empty ? 0.f : expf((to_f32(x[j]) - st[0]) * p.inv_temperature - st[1]);
    float dz = e * st[4];
    bool member = false;
    for (int k = 0; k < p.entries; ++k)
      if (p.teacher_ids[row * p.entries + k] == j) {
        float lq;
        dz -= empty ? 0.f : teacher_q(p, row, k, st[2], st[3], lq);
        member = true;
      }
    if (!member && e != 0.f) dz -= e * st[5];
    dx[j] = from_f32<T>(dz * g);
  }
}

}  // namespace

cudaError_t launch_token_logprobs(int dtype, const LogitsArgs& p, cudaStream_t stream) {
  const unsigned grid = (unsigned)(p.batch * p.rows);
  if (dtype == FAKLA_BF16) token_logprobs_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
  else token_logprobs_kernel<float><<<grid, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_token_logprobs_backward(int dtype, const LogitsArgs& p, cudaStream_t stream) {
  const unsigned grid = (unsigned)(p.batch * p.rows);
  if (dtype == FAKLA_BF16) token_logprobs_backward_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
  else token_logprobs_backward_kernel<float><<<grid, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_distill(int dtype, const LogitsArgs& p, cudaStream_t stream) {
  const unsigned grid = (unsigned)(p.batch * p.rows);
  if (dtype == FAKLA_BF16) distill_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
  else distill_kernel<float><<<grid, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_distill_backward(int dtype, const LogitsArgs& p, cudaStream_t stream) {
  const unsigned grid = (unsigned)(p.batch * p.rows);
  if (dtype == FAKLA_BF16) distill_backward_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
  else distill_backward_kernel<float><<<grid, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace fakla
