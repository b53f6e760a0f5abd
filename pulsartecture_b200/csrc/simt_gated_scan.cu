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
// rounded once. Memory is the bound: 3 tensors for the forward, 5 for the
// backward, so each is read once into registers, where it stays.
//
// Time is split, because a batch rarely has channels enough to keep 6 TB/s in
// flight: a run of tokens maps h to A h + H (A the product of its a, H its
// result from zero), and such maps compose. A thread takes a run of L tokens
// of its channels, the 8 warps of a block consecutive runs (a tile), and the
// C blocks of a cluster consecutive tiles; one round composes the runs through
// shared memory, the tiles through the cluster's distributed shared memory,
// and only then walks each run from its true initial state to write it. The
// cluster moves on along its sequence with the state in registers. Every
// composition is in the order of time, so results do not depend on timing, and
// a round's barrier waits for no block outside of the cluster.
//
// The backward walks the tiles from the last to the first. The states that it
// needs are rebuilt from those the forward kept in `saved`, one before every
// kKept-th token (fp32, 1 % of the traffic): it reads no rounded output and one
// tensor less than a backward that keeps h.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "fakla_common.cuh"
#include "fakla_kernels.h"

namespace fakla {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCluster = 8;  // the largest portable cluster
// Tokens per thread and round. The forward holds a and b of a run and the next
// round's raw values, the backward also h and dout: both fit 128 registers, two
// blocks on an SM.
constexpr int kForwardRun = 16;
constexpr int kBackwardRun = 8;
constexpr int kForwardTile = kWarps * kForwardRun;
constexpr int kBackwardTile = kWarps * kBackwardRun;
constexpr int kKept = kBackwardTile;  // tokens between two kept states
static_assert(kForwardTile % kKept == 0, "kept states start a forward warp's run");

// VEC channels of one token, as one register: two bf16 or one value.
template <typename T, int VEC>
struct Pack;
template <>
struct Pack<float, 1> {
  typedef float Raw;
  static __device__ __forceinline__ float get(Raw r, int) { return r; }
  static __device__ __forceinline__ Raw put(const float* v) { return v[0]; }
};
template <>
struct Pack<__nv_bfloat16, 1> {
  typedef unsigned short Raw;
  static __device__ __forceinline__ float get(Raw r, int) { return __uint_as_float((uint32_t)r << 16); }
  static __device__ __forceinline__ Raw put(const float* v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v[0])); }
};
template <>
struct Pack<__nv_bfloat16, 2> {
  typedef uint32_t Raw;
  static __device__ __forceinline__ float get(Raw r, int i) {
    return __uint_as_float(i == 0 ? r << 16 : r & 0xffff0000u);
  }
  static __device__ __forceinline__ Raw put(const float* v) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(v[0], v[1]);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};

// a and 1 - a from one exponential of -|g|: neither cancels, and g = +-inf
// gives exactly 0 and 1. bf16 gates take the hardware's exponential and
// reciprocal, whose error (a few 2^-24 of 1 - a or of a) is far below the
// gate's own rounding.
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

// A h + H, with 0 where h is 0 even if A is past fp32 (no token of the run
// meets that product).
__device__ __forceinline__ float carry_on(float A, float h, float H) { return h == 0.f ? H : fmaf(A, h, H); }

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Stores v at the address that `local` has in the shared memory of block `rank`.
__device__ __forceinline__ void store_peer(float2* local, uint32_t rank, float2 v) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(local);
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(v.x), "f"(v.y) : "memory");
}

// One block's place: its channels of its batch row, and its rank in time.
template <int VEC>
struct Place {
  int lane, warp, rank;
  int64_t b, d;  // batch row, first channel of this thread
  bool on;       // the channels exist
  __device__ Place(const GatedScanArgs& p, int C) {
    lane = threadIdx.x % 32;
    warp = threadIdx.x / 32;
    rank = C > 1 ? (int)cluster_rank() : 0;
    const int64_t groups = (p.D + 32 * VEC - 1) / (32 * VEC), id = blockIdx.x / C;
    b = id / groups;
    d = (id % groups * 32 + lane) * VEC;
    on = d < p.D;
  }
};

template <typename T, int VEC, int ACT, bool MIX>
__global__ void __launch_bounds__(kThreads, 2) scan_forward_kernel(GatedScanArgs p, int C) {
  typedef Pack<T, VEC> P;
  typedef typename P::Raw Raw;
  constexpr int L = kForwardRun;
  // (A, H) of every warp's run and of every block's tile, for two rounds: a
  // round's values are overwritten two barriers later, when all have read them
  __shared__ float2 runs[2][kWarps][VEC][32];
  __shared__ float2 tiles[2][kMaxCluster][VEC][32];
  const Place<VEC> at(p, C);
  griddep_wait();
  const int64_t n_tiles = (p.T + kForwardTile - 1) / kForwardTile, n_kept = (p.T + kKept - 1) / kKept;
  const int64_t rounds = (n_tiles + C - 1) / C;
  const T* x = (const T*)p.x + at.b * p.x_batch + at.d;
  const T* gate = (const T*)p.gate + at.b * p.gate_batch + at.d;
  T* out = (T*)p.out + at.b * p.T * p.D + at.d;

  Raw rx[L], rg[L];
  int n = 0;       // tokens of this thread's run that exist
  int64_t t0 = 0;  // its first token
  auto fetch = [&](int64_t round) {
    t0 = (round * C + at.rank) * kForwardTile + at.warp * L;
    n = !at.on || t0 >= p.T ? 0 : (int)(p.T - t0 < L ? p.T - t0 : L);
    const T* px = x + t0 * p.x_time;
    const T* pg = gate + t0 * p.gate_time;
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i < n) {
        rx[i] = __ldcs((const Raw*)(px + i * p.x_time));
        rg[i] = __ldcs((const Raw*)(pg + i * p.gate_time));
      }
  };
  fetch(0);
  float state[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) state[v] = p.state_in && at.on ? p.state_in[at.b * p.D + at.d + v] : 0.f;
  if (C > 1) {  // no store into a block that has not begun
    cluster_arrive();
    cluster_wait();
  }
  for (int64_t round = 0; round < rounds; ++round) {
    const int buf = (int)(round & 1);
    float a[L][VEC], b[L][VEC], A[VEC], H[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A[v] = 1.f;
      H[v] = 0.f;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        if (i < n) {
          float rest;
          const float value = P::get(rx[i], v);
          gate_pair<ACT, T>(P::get(rg[i], v), a[i][v], rest);
          b[i][v] = MIX ? rest * value : value;
          A[v] *= a[i][v];
          H[v] = fmaf(a[i][v], H[v], b[i][v]);
        }
      }
      runs[buf][at.warp][v][at.lane] = make_float2(A[v], H[v]);
    }
    const int64_t here = t0;
    const int count = n;
    if (round + 1 < rounds) fetch(round + 1);
    __syncthreads();
    // the block's runs before this warp's, and (last warp) all of them
    float h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float PA = 1.f, PH = 0.f;
      for (int w = 0; w < at.warp; ++w) {
        const float2 r = runs[buf][w][v][at.lane];
        PA *= r.x;
        PH = carry_on(r.x, PH, r.y);
      }
      if (C > 1) {
        if (at.warp == kWarps - 1) {
          const float2 all = make_float2(PA * A[v], carry_on(A[v], PH, H[v]));
          for (int r = 0; r < C; ++r) store_peer(&tiles[buf][at.rank][v][at.lane], r, all);
        }
      }
      A[v] = PA;
      h[v] = PH;
    }
    if (C > 1) {
      cluster_arrive();
      cluster_wait();
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float c = state[v], first = c;
        for (int r = 0; r < C; ++r) {
          if (r == at.rank) first = c;
          const float2 t = tiles[buf][r][v][at.lane];
          c = carry_on(t.x, c, t.y);
        }
        h[v] = carry_on(A[v], first, h[v]);
        state[v] = c;
      }
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        h[v] = carry_on(A[v], state[v], h[v]);
        for (int w = 0; w < kWarps; ++w) {
          const float2 r = runs[buf][w][v][at.lane];
          state[v] = carry_on(r.x, state[v], r.y);
        }
      }
    }
    if (p.saved && count > 0 && here % kKept == 0) {
      float* keep = p.saved + (at.b * n_kept + here / kKept) * p.D + at.d;
#pragma unroll
      for (int v = 0; v < VEC; ++v) keep[v] = h[v];
    }
    T* po = out + here * p.D;
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i < count) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = fmaf(a[i][v], h[v], b[i][v]);
        __stcs((Raw*)(po + i * p.D), P::put(h));
      }
  }
  if (p.state_out && at.on && at.warp == 0 && at.rank == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.state_out[at.b * p.D + at.d + v] = state[v];
  }
}

template <typename T, int VEC, int ACT, bool MIX>
__global__ void __launch_bounds__(kThreads, 2) scan_backward_kernel(GatedScanArgs p, int C) {
  typedef Pack<T, VEC> P;
  typedef typename P::Raw Raw;
  constexpr int L = kBackwardRun;
  // (A, H) of every warp's run; what its gradients hand to the token before
  // it, K + A r for the r that it is given from behind; the same of the tiles
  __shared__ float2 runs[2][kWarps][VEC][32];
  __shared__ float back[2][kWarps][VEC][32];
  __shared__ float2 tiles[2][kMaxCluster][VEC][32];
  const Place<VEC> at(p, C);
  griddep_wait();
  const int64_t n_tiles = (p.T + kBackwardTile - 1) / kBackwardTile;
  const int64_t rounds = (n_tiles + C - 1) / C;
  const T* x = (const T*)p.x + at.b * p.x_batch + at.d;
  const T* gate = (const T*)p.gate + at.b * p.gate_batch + at.d;
  const int64_t dense = at.b * p.T * p.D + at.d;
  const T* dout = (const T*)p.dout + dense;
  T* dx = (T*)p.dx + dense;
  T* dgate = (T*)p.dgate + dense;

  Raw rx[L], rg[L], rd[L];
  float kept[VEC];  // h before the tile
  int n = 0;
  int64_t t0 = 0;
  auto fetch = [&](int64_t round) {
    const int64_t tile = round * C + at.rank;
    t0 = tile * kBackwardTile + at.warp * L;
    n = !at.on || t0 >= p.T ? 0 : (int)(p.T - t0 < L ? p.T - t0 : L);
    const T* px = x + t0 * p.x_time;
    const T* pg = gate + t0 * p.gate_time;
    const T* pd = dout + t0 * p.D;
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i < n) {
        rx[i] = __ldcs((const Raw*)(px + i * p.x_time));
        rg[i] = __ldcs((const Raw*)(pg + i * p.gate_time));
        rd[i] = __ldcs((const Raw*)(pd + i * p.D));
      }
#pragma unroll
    for (int v = 0; v < VEC; ++v) kept[v] = n > 0 ? p.saved[(at.b * n_tiles + tile) * p.D + at.d + v] : 0.f;
  };
  fetch(rounds - 1);
  float carry[VEC];  // a_{t+1} G_{t+1} behind the round's last token
#pragma unroll
  for (int v = 0; v < VEC; ++v) carry[v] = p.dstate_out && at.on ? p.dstate_out[at.b * p.D + at.d + v] : 0.f;
  if (C > 1) {
    cluster_arrive();
    cluster_wait();
  }
  for (int64_t round = rounds - 1; round >= 0; --round) {
    const int buf = (int)(round & 1);
    float a[L][VEC], rest[L][VEC], A[VEC], H[VEC], K[VEC], h[VEC];
    Raw vx[L], vd[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      vx[i] = rx[i];
      vd[i] = rd[i];
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A[v] = 1.f;
      H[v] = K[v] = 0.f;
      h[v] = kept[v];
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (i < n) {
          const float value = P::get(vx[i], v);
          gate_pair<ACT, T>(P::get(rg[i], v), a[i][v], rest[i][v]);
          A[v] *= a[i][v];
          H[v] = fmaf(a[i][v], H[v], MIX ? rest[i][v] * value : value);
        }
#pragma unroll
      for (int i = L - 1; i >= 0; --i)
        if (i < n) K[v] = a[i][v] * (P::get(vd[i], v) + K[v]);
      runs[buf][at.warp][v][at.lane] = make_float2(A[v], H[v]);
      back[buf][at.warp][v][at.lane] = K[v];
    }
    const int64_t here = t0;
    const int count = n;
    if (round > 0) fetch(round - 1);
    __syncthreads();
    float r[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      for (int w = 0; w < at.warp; ++w) {
        const float2 run = runs[buf][w][v][at.lane];
        h[v] = carry_on(run.x, h[v], run.y);
      }
      float PA = 1.f, PK = 0.f;
      for (int w = kWarps - 1; w > at.warp; --w) {
        const float m = runs[buf][w][v][at.lane].x;
        PA *= m;
        PK = carry_on(m, PK, back[buf][w][v][at.lane]);
      }
      if (C > 1) {
        if (at.warp == 0) {
          const float2 all = make_float2(PA * A[v], carry_on(A[v], PK, K[v]));
          for (int c = 0; c < C; ++c) store_peer(&tiles[buf][at.rank][v][at.lane], c, all);
        }
      }
      A[v] = PA;
      r[v] = PK;
    }
    if (C > 1) {
      cluster_arrive();
      cluster_wait();
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float c = carry[v], first = c;
        for (int k = C - 1; k >= 0; --k) {
          if (k == at.rank) first = c;
          const float2 t = tiles[buf][k][v][at.lane];
          c = carry_on(t.x, c, t.y);
        }
        r[v] = carry_on(A[v], first, r[v]);
        carry[v] = c;
      }
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        r[v] = carry_on(A[v], carry[v], r[v]);
        for (int w = kWarps - 1; w >= 0; --w)
          carry[v] = carry_on(runs[buf][w][v][at.lane].x, carry[v], back[buf][w][v][at.lane]);
      }
    }
    float before[L][VEC];
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i < count)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float value = P::get(vx[i], v);
          before[i][v] = MIX ? h[v] - value : h[v];
          h[v] = fmaf(a[i][v], h[v], MIX ? rest[i][v] * value : value);
        }
    T* pdx = dx + here * p.D;
    T* pdg = dgate + here * p.D;
#pragma unroll
    for (int i = L - 1; i >= 0; --i)
      if (i < count) {
        float ox[VEC], og[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float G = P::get(vd[i], v) + r[v];
          r[v] = a[i][v] * G;
          ox[v] = MIX ? G * rest[i][v] : G;
          const float da = G * before[i][v];
          og[v] = ACT == FAKLA_ACT_SIGMOID ? da * a[i][v] * rest[i][v] : da;
        }
        __stcs((Raw*)(pdx + i * p.D), P::put(ox));
        __stcs((Raw*)(pdg + i * p.D), P::put(og));
      }
  }
  if (p.dstate_in && at.on && at.warp == 0 && at.rank == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.dstate_in[at.b * p.D + at.d + v] = carry[v];
  }
}

template <typename T, int VEC, int ACT, bool MIX>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(GatedScanArgs p) {
  typedef Pack<T, VEC> P;
  typedef typename P::Raw Raw;
  griddep_wait();
  const int64_t per_row = p.D / VEC;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= per_row * p.B) return;
  const int64_t b = i / per_row, d = i % per_row * VEC;
  const Raw rg = *(const Raw*)((const T*)p.gate + b * p.gate_batch + d);
  const Raw rx = *(const Raw*)((const T*)p.x + b * p.x_batch + d);
  float h[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float a, rest;
    gate_pair<ACT, T>(P::get(rg, v), a, rest);
    const float value = P::get(rx, v);
    h[v] = fmaf(a, p.state_in[b * p.D + d + v], MIX ? rest * value : value);
    p.state_out[b * p.D + d + v] = h[v];
  }
  *(Raw*)((T*)p.out + b * p.D + d) = P::put(h);
}

// Runs f with the type, channels per thread, gate activation and input form as
// constants. bf16 channels go in pairs where every row starts on 4 bytes.
template <typename F>
void dispatch(int dtype, const GatedScanArgs& p, F f) {
  auto by_form = [&](auto t, auto vec, auto a) {
    if (p.mix) f(t, vec, a, std::true_type{}); else f(t, vec, a, std::false_type{});
  };
  auto by_act = [&](auto t, auto vec) {
    if (p.act == FAKLA_ACT_SIGMOID) by_form(t, vec, std::integral_constant<int, FAKLA_ACT_SIGMOID>{});
    else by_form(t, vec, std::integral_constant<int, FAKLA_ACT_IDENTITY>{});
  };
  const int64_t steps = p.D | p.x_batch | p.x_time | p.gate_batch | p.gate_time;
  const uintptr_t bases = (uintptr_t)p.x | (uintptr_t)p.gate | (uintptr_t)p.out | (uintptr_t)p.dout |
                          (uintptr_t)p.dx | (uintptr_t)p.dgate;
  if (dtype != FAKLA_BF16) by_act(float{}, std::integral_constant<int, 1>{});
  else if (steps % 2 == 0 && bases % 4 == 0) by_act(__nv_bfloat16{}, std::integral_constant<int, 2>{});
  else by_act(__nv_bfloat16{}, std::integral_constant<int, 1>{});
}

// Blocks of a cluster, which share a sequence's time: as many as give each SM
// two blocks, and no more than there are tiles.
int cluster_size(int64_t groups, int64_t tiles) {
  int c = 1;
  while (c < kMaxCluster && 2 * c <= tiles && groups * c < 2 * fakla_sm_count()) c *= 2;
  return c;
}

template <typename K>
cudaError_t launch(K kernel, const GatedScanArgs& p, int vec, int tile, cudaStream_t stream) {
  const int64_t groups = p.B * ((p.D + 32 * vec - 1) / (32 * vec));
  const int c = cluster_size(groups, (p.T + tile - 1) / tile);
  return launch_chained(kernel, dim3((unsigned)(groups * c)), dim3(kThreads), 0, stream, (unsigned)c, p, c);
}

}  // namespace

size_t gated_scan_saved_bytes(int64_t B, int64_t T, int64_t D) {
  return (size_t)B * (size_t)((T + kKept - 1) / kKept) * (size_t)D * sizeof(float);
}

cudaError_t launch_gated_scan(int dtype, const GatedScanArgs& p, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  dispatch(dtype, p, [&](auto t, auto vec, auto act, auto mix) {
    e = launch(scan_forward_kernel<decltype(t), vec(), act(), mix()>, p, vec(), kForwardTile, stream);
  });
  return e;
}

cudaError_t launch_gated_scan_backward(int dtype, const GatedScanArgs& p, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  dispatch(dtype, p, [&](auto t, auto vec, auto act, auto mix) {
    e = launch(scan_backward_kernel<decltype(t), vec(), act(), mix()>, p, vec(), kBackwardTile, stream);
  });
  return e;
}

cudaError_t launch_gated_scan_step(int dtype, const GatedScanArgs& p, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  dispatch(dtype, p, [&](auto t, auto vec, auto act, auto mix) {
    const int64_t items = p.B * p.D / vec();
    e = launch_chained(scan_step_kernel<decltype(t), vec(), act(), mix()>,
                       dim3((unsigned)((items + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, 1u, p);
  });
  return e;
}

}  // namespace fakla
