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
// of its VEC channels, the 8 warps of a block consecutive runs (a tile), and
// the C blocks of a cluster consecutive tiles. A round
//   1. reduces every run to (A, H) and puts it into shared memory,
//   2. lets one thread per channel walk the runs from the tile's initial h
//      (from the blocks before it in the cluster through distributed shared
//      memory, from the round before in a register), leaving each run's h,
//   3. walks each run from there and writes it,
// while the next round's loads are in flight. Every composition is in the
// order of time, so results do not depend on timing, and a round waits for no
// block outside of the cluster.
//
// The backward walks the tiles from the last to the first. The states that it
// needs are rebuilt from those the forward kept in `saved`, one before every
// kKept-th token (fp32, 2 % of the traffic): it reads no rounded output and one
// tensor less than a backward that keeps h.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <type_traits>

#include "fakla_common.cuh"
#include "fakla_kernels.h"
#include "sm100_umma.cuh"

namespace fakla {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kPortableCluster = 8;
constexpr int kMaxCluster = 16;
// Tokens per thread and round. The forward holds a and b of a run and the next
// round's raw values, the backward a, 1 - a, h, and the raw x and dout: with
// four channels both fit 128 registers, two blocks on an SM.
constexpr int kForwardRun = 8;
constexpr int kBackwardRun = 4;
constexpr int kKept = kWarps * kBackwardRun;  // tokens between two kept states: the backward's tile

// VEC channels of one token as loaded, at most 8 bytes.
template <typename T, int VEC>
struct Pack;
template <int VEC>
struct Pack<float, VEC> {
  typedef typename std::conditional<VEC == 2, float2, float>::type Raw;
  static __device__ __forceinline__ float get(const Raw& r, int i) { return reinterpret_cast<const float*>(&r)[i]; }
  static __device__ __forceinline__ Raw put(const float* v) {
    Raw r;
    for (int i = 0; i < VEC; ++i) reinterpret_cast<float*>(&r)[i] = v[i];
    return r;
  }
};
template <>
struct Pack<__nv_bfloat16, 1> {
  typedef unsigned short Raw;
  static __device__ __forceinline__ float get(Raw r, int) { return __uint_as_float((uint32_t)r << 16); }
  static __device__ __forceinline__ Raw negative(Raw r) { return r | 0x8000u; }  // -|r|
  static __device__ __forceinline__ Raw put(const float* v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v[0])); }
};
template <int VEC>
struct Pack<__nv_bfloat16, VEC> {
  typedef typename std::conditional<VEC == 4, uint2, uint32_t>::type Raw;
  static __device__ __forceinline__ float get(const Raw& r, int i) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(&r)[i / 2];
    return __uint_as_float(i % 2 == 0 ? w << 16 : w & 0xffff0000u);
  }
  static __device__ __forceinline__ Raw negative(Raw r) {  // -|r|
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) reinterpret_cast<uint32_t*>(&r)[i] |= 0x80008000u;
    return r;
  }
  static __device__ __forceinline__ Raw put(const float* v) {
    Raw r;
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v[i], v[i + 1]);
      reinterpret_cast<uint32_t*>(&r)[i / 2] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return r;
  }
};

// Element-wise products and sums of VEC values, two to an instruction (the
// packed fp32 forms halve the arithmetic: the forward's 30 instructions per value became
// 25, where 33 would fill the issue slots at full memory speed).
__device__ __forceinline__ uint64_t pair(const float* v) {
  return sm100::f2_make(__float_as_uint(v[0]), __float_as_uint(v[1]));
}
__device__ __forceinline__ void unpair(uint64_t v, float* d) {
  const float2 f = sm100::f2_split(v);
  d[0] = f.x;
  d[1] = f.y;
}
template <int VEC>
__device__ __forceinline__ void mul(float* d, const float* a, const float* b) {
  if constexpr (VEC == 1) d[0] = a[0] * b[0];
  else
#pragma unroll
    for (int i = 0; i < VEC; i += 2) unpair(sm100::f2_mul(pair(a + i), pair(b + i)), d + i);
}
template <int VEC>
__device__ __forceinline__ void add(float* d, const float* a, const float* b) {
  if constexpr (VEC == 1) d[0] = a[0] + b[0];
  else
#pragma unroll
    for (int i = 0; i < VEC; i += 2) unpair(sm100::f2_add(pair(a + i), pair(b + i)), d + i);
}
template <int VEC>
__device__ __forceinline__ void fma(float* d, const float* a, const float* b, const float* c) {
  if constexpr (VEC == 1) d[0] = fmaf(a[0], b[0], c[0]);
  else
#pragma unroll
    for (int i = 0; i < VEC; i += 2) unpair(sm100::f2_fma(pair(a + i), pair(b + i), pair(c + i)), d + i);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// a and 1 - a from one exponential of -|g|: neither cancels, and g = +-inf
// gives exactly 0 and 1. bf16 gates take the hardware's exponential and
// reciprocal, whose error (a few 2^-24 of 1 - a or of a) is far below the
// gate's own rounding.
template <int ACT, typename T, int VEC>
__device__ __forceinline__ void gates(const typename Pack<T, VEC>::Raw& raw, float* a, float* rest) {
  typedef Pack<T, VEC> P;
  if constexpr (ACT == FAKLA_ACT_SIGMOID) {
    float e[VEC], big[VEC], small[VEC];
    if constexpr (sizeof(T) == 2) {
      const auto down = P::negative(raw);
      float c[VEC], one[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        e[v] = P::get(down, v);
        c[v] = 1.44269504f;  // log2(e)
        one[v] = 1.f;
      }
      mul<VEC>(e, e, c);
#pragma unroll
      for (int v = 0; v < VEC; ++v) e[v] = exp2_approx(e[v]);
      add<VEC>(big, e, one);
#pragma unroll
      for (int v = 0; v < VEC; ++v) big[v] = reciprocal(big[v]);
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        e[v] = expf(-fabsf(P::get(raw, v)));
        big[v] = 1.f / (1.f + e[v]);
      }
    }
    mul<VEC>(small, e, big);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const bool up = P::get(raw, v) >= 0.f;
      a[v] = up ? big[v] : small[v];
      rest[v] = up ? small[v] : big[v];
    }
  } else {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      a[v] = P::get(raw, v);
      rest[v] = 1.f - a[v];
    }
  }
}

// b = (1 - a) x or x
template <typename T, int VEC, bool MIX>
__device__ __forceinline__ void inputs(const typename Pack<T, VEC>::Raw& raw, const float* rest, float* b) {
#pragma unroll
  for (int v = 0; v < VEC; ++v) b[v] = Pack<T, VEC>::get(raw, v);
  if constexpr (MIX) mul<VEC>(b, rest, b);
}

// The product of a run's coefficients, held within fp32 so that 0 times it is
// 0. (A NaN among them is lost here, and kept by H.)
__device__ __forceinline__ float bounded(float A) { return fminf(fmaxf(A, -FLT_MAX), FLT_MAX); }

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  sm100::cluster_sync();
}

// One block's place: its channels of its batch row, and its rank in time.
template <int VEC>
struct Place {
  static constexpr int kChannels = 32 * VEC;
  int lane, warp, rank;
  int64_t b;
  int64_t d;  // first channel of this thread's runs; the last one's where it has none
  bool on;    // its channels exist
  int64_t c;  // channel that it walks in step 2
  bool walks;
  int walkers;  // threads of the block that do
  __device__ Place(const GatedScanArgs& p, int C) {
    lane = threadIdx.x % 32;
    warp = threadIdx.x / 32;
    rank = C > 1 ? (int)sm100::cluster_ctarank() : 0;
    const int64_t groups = (p.D + kChannels - 1) / kChannels, id = blockIdx.x / C;
    b = id / groups;
    const int64_t first = id % groups * kChannels;
    d = first + lane * VEC;
    on = d < p.D;
    if (!on) d = p.D - VEC;  // read like any other, never written
    c = first + threadIdx.x;
    walkers = (int)(p.D - first < kChannels ? p.D - first : kChannels);
    walks = threadIdx.x < walkers;
  }
};

// What the blocks of a cluster tell each other in step 2: every block's (A, H)
// of its tile, stored into all of them with the bytes counted on the receiver's
// barrier, so a round costs one trip between SMs and no fence (a cluster
// barrier per round, which also waits for the block's own global stores, took
// 17 % longer). Two rounds' worth: a block gets a round's last value
// from a peer only after that peer has read the round before.
struct Exchange {
  float2 tiles[2][kMaxCluster][128];
  uint64_t full[2];
};
constexpr uint64_t kWaitLimitNs = 2000000000ull;

__device__ __forceinline__ void exchange_begin(Exchange& x) {
  if (threadIdx.x == 0) {
    sm100::mbar_init(&x.full[0], 1);
    sm100::mbar_init(&x.full[1], 1);
    sm100::fence_mbar_init();
  }
  cluster_sync();  // no store into a block that has not begun
}

// For the `walkers` threads that walk a channel: gives `mine` to all blocks and
// returns this tile's incoming value; `carry` moves on by the whole round.
// `step` counts rounds from 0, `order` is 1 in the order of time, -1 against
// it. A wait that runs out reports it and sets `late`, after which nothing is
// waited for any more.
__device__ __forceinline__ float exchange(Exchange& x, float2 mine, float& carry, int C, int rank, int walkers,
                                          int64_t step, int order, bool& late, int* status) {
  const int buf = (int)(step & 1);
  if (threadIdx.x == 0) sm100::mbar_arrive_expect_tx(&x.full[buf], (uint32_t)(C * walkers) * (uint32_t)sizeof(float2));
  for (int r = 0; r < C; ++r)
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(
                     sm100::mapa_shared(&x.tiles[buf][rank][threadIdx.x], r)),
                 "f"(mine.x), "f"(mine.y), "r"(sm100::mapa_shared(&x.full[buf], r))
                 : "memory");
  if (!late && !sm100::mbar_wait_cluster(&x.full[buf], (uint32_t)(step >> 1) & 1u, kWaitLimitNs)) {
    late = true;
    report_status(status, FAKLA_ERR_TIMEOUT);
  }
  float first = carry;
  for (int i = 0; i < C; ++i) {
    const int r = order > 0 ? i : C - 1 - i;
    if (r == rank) first = carry;
    const float2 t = x.tiles[buf][r][threadIdx.x];
    carry = fmaf(t.x, carry, t.y);
  }
  return first;
}

// Two blocks of 128 registers with 8 bytes per thread and token, three of 80 below.
constexpr int blocks_per_sm(int bytes) { return bytes == 8 ? 2 : 3; }

template <typename T, int VEC, int ACT, bool MIX>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(VEC * sizeof(T))) scan_forward_kernel(GatedScanArgs p, int C) {
  typedef Pack<T, VEC> P;
  typedef typename P::Raw Raw;
  constexpr int L = kForwardRun, kTile = kWarps * L;
  __shared__ __align__(16) float runA[kWarps][32 * VEC], runH[kWarps][32 * VEC];
  __shared__ Exchange ex;
  const Place<VEC> at(p, C);
  griddep_wait();
  const int64_t n_tiles = (p.T + kTile - 1) / kTile, n_kept = (p.T + kKept - 1) / kKept;
  const int64_t rounds = (n_tiles + C - 1) / C;
  const T* x = (const T*)p.x + at.b * p.x_batch + at.d;
  const T* gate = (const T*)p.gate + at.b * p.gate_batch + at.d;
  T* out = (T*)p.out + at.b * p.T * p.D + at.d;

  Raw rx[L], rg[L];
  int n = 0;       // tokens of this warp's run that exist
  int64_t t0 = 0;  // its first token
  auto fetch = [&](int64_t round) {
    t0 = (round * C + at.rank) * kTile + at.warp * L;
    n = (int)(p.T - t0 < 0 ? 0 : p.T - t0 < L ? p.T - t0 : L);
    const T* px = x + t0 * p.x_time;
    const T* pg = gate + t0 * p.gate_time;
    if (n == L) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        rx[i] = __ldcs((const Raw*)px);
        rg[i] = __ldcs((const Raw*)pg);
        px += p.x_time;
        pg += p.gate_time;
      }
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (i < n) {
          rx[i] = __ldcs((const Raw*)(px + i * p.x_time));
          rg[i] = __ldcs((const Raw*)(pg + i * p.gate_time));
        }
    }
  };
  fetch(0);
  float state = p.state_in && at.walks ? p.state_in[at.b * p.D + at.c] : 0.f;
  if (C > 1) exchange_begin(ex);
  bool late = false;
  for (int64_t round = 0; round < rounds; ++round) {
    float a[L][VEC], b[L][VEC], A[VEC], H[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A[v] = 1.f;
      H[v] = 0.f;
    }
    auto reduce = [&](auto full) {
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (decltype(full)::value || i < n) {
          float rest[VEC];
          gates<ACT, T, VEC>(rg[i], a[i], rest);
          inputs<T, VEC, MIX>(rx[i], rest, b[i]);
          mul<VEC>(A, A, a[i]);
          fma<VEC>(H, a[i], H, b[i]);
        }
    };
    if (n == L) reduce(std::true_type{});
    else reduce(std::false_type{});
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      runA[at.warp][at.lane * VEC + v] = bounded(A[v]);
      runH[at.warp][at.lane * VEC + v] = H[v];
    }
    const int64_t here = t0;
    const int count = n;
    if (round + 1 < rounds) fetch(round + 1);
    __syncthreads();
    if (at.walks) {
      float h = state;
      if (C > 1) {
        float2 all = make_float2(1.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          all.x *= runA[w][threadIdx.x];
          all.y = fmaf(runA[w][threadIdx.x], all.y, runH[w][threadIdx.x]);
        }
        all.x = bounded(all.x);
        h = exchange(ex, all, state, C, at.rank, at.walkers, round, 1, late, p.status);
      }
      const int64_t tile0 = here - at.warp * L;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float wA = runA[w][threadIdx.x], wH = runH[w][threadIdx.x];
        if (w * L % kKept == 0 && p.saved && tile0 + w * L < p.T)
          p.saved[(at.b * n_kept + (tile0 + w * L) / kKept) * p.D + at.c] = h;
        runH[w][threadIdx.x] = h;
        h = fmaf(wA, h, wH);
      }
      if (C == 1) state = h;
    }
    __syncthreads();
    float hv[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) hv[v] = runH[at.warp][at.lane * VEC + v];
    T* po = out + here * p.D;
    auto write = [&](auto full) {
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (decltype(full)::value || i < count) {
          fma<VEC>(hv, a[i], hv, b[i]);
          if (at.on) __stcs((Raw*)po, P::put(hv));
          po += p.D;
        }
    };
    if (count == L) write(std::true_type{});
    else write(std::false_type{});
  }
  if (C > 1) cluster_sync();  // no block leaves while another could store into it
  if (p.state_out && at.walks && at.rank == 0) p.state_out[at.b * p.D + at.c] = state;
}

template <typename T, int VEC, int ACT, bool MIX>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(VEC * sizeof(T))) scan_backward_kernel(GatedScanArgs p, int C) {
  typedef Pack<T, VEC> P;
  typedef typename P::Raw Raw;
  constexpr int L = kBackwardRun, kTile = kKept;
  // (A, H) of every warp's run, and K: given r from behind, a run hands
  // K + A r to the token before it
  __shared__ __align__(16) float runA[kWarps][32 * VEC], runH[kWarps][32 * VEC], runK[kWarps][32 * VEC];
  __shared__ Exchange ex;
  const Place<VEC> at(p, C);
  griddep_wait();
  const int64_t n_tiles = (p.T + kTile - 1) / kTile;
  const int64_t rounds = (n_tiles + C - 1) / C;
  const T* x = (const T*)p.x + at.b * p.x_batch + at.d;
  const T* gate = (const T*)p.gate + at.b * p.gate_batch + at.d;
  const int64_t dense = at.b * p.T * p.D + at.d;
  const T* dout = (const T*)p.dout + dense;
  T* dx = (T*)p.dx + dense;
  T* dgate = (T*)p.dgate + dense;

  Raw rx[L], rg[L], rd[L];
  float kept = 0.f;  // h before the tile, of the channel that this thread walks
  int n = 0;
  int64_t t0 = 0;
  auto fetch = [&](int64_t round) {
    const int64_t tile = round * C + at.rank;
    t0 = tile * kTile + at.warp * L;
    n = (int)(p.T - t0 < 0 ? 0 : p.T - t0 < L ? p.T - t0 : L);
    const T* px = x + t0 * p.x_time;
    const T* pg = gate + t0 * p.gate_time;
    const T* pd = dout + t0 * p.D;
    if (n == L) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        rx[i] = __ldcs((const Raw*)px);
        rg[i] = __ldcs((const Raw*)pg);
        rd[i] = __ldcs((const Raw*)pd);
        px += p.x_time;
        pg += p.gate_time;
        pd += p.D;
      }
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (i < n) {
          rx[i] = __ldcs((const Raw*)(px + i * p.x_time));
          rg[i] = __ldcs((const Raw*)(pg + i * p.gate_time));
          rd[i] = __ldcs((const Raw*)(pd + i * p.D));
        }
    }
    if (at.walks && tile < n_tiles) kept = p.saved[(at.b * n_tiles + tile) * p.D + at.c];
  };
  fetch(rounds - 1);
  float carry = p.dstate_out && at.walks ? p.dstate_out[at.b * p.D + at.c] : 0.f;  // a_{t+1} G_{t+1}
  if (C > 1) exchange_begin(ex);
  bool late = false;
  for (int64_t round = rounds - 1; round >= 0; --round) {
    float a[L][VEC], rest[L][VEC], A[VEC], H[VEC], K[VEC];
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
    }
    auto reduce = [&](auto full) {
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (decltype(full)::value || i < n) {
          float b[VEC];
          gates<ACT, T, VEC>(rg[i], a[i], rest[i]);
          inputs<T, VEC, MIX>(vx[i], rest[i], b);
          mul<VEC>(A, A, a[i]);
          fma<VEC>(H, a[i], H, b);
        }
#pragma unroll
      for (int i = L - 1; i >= 0; --i)
        if (decltype(full)::value || i < n) {
          float d[VEC];
#pragma unroll
          for (int v = 0; v < VEC; ++v) d[v] = P::get(vd[i], v);
          add<VEC>(K, d, K);
          mul<VEC>(K, a[i], K);
        }
    };
    if (n == L) reduce(std::true_type{});
    else reduce(std::false_type{});
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      runA[at.warp][at.lane * VEC + v] = bounded(A[v]);
      runH[at.warp][at.lane * VEC + v] = H[v];
      runK[at.warp][at.lane * VEC + v] = K[v];
    }
    const int64_t here = t0;
    const int count = n;
    float h = kept;
    if (round > 0) fetch(round - 1);
    __syncthreads();
    if (at.walks) {
      float r = carry;
      if (C > 1) {
        float2 all = make_float2(1.f, 0.f);
#pragma unroll
        for (int w = kWarps - 1; w >= 0; --w) {
          all.x *= runA[w][threadIdx.x];
          all.y = fmaf(runA[w][threadIdx.x], all.y, runK[w][threadIdx.x]);
        }
        all.x = bounded(all.x);
        r = exchange(ex, all, carry, C, at.rank, at.walkers, rounds - 1 - round, -1, late, p.status);
      }
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float wH = runH[w][threadIdx.x];
        runH[w][threadIdx.x] = h;
        h = fmaf(runA[w][threadIdx.x], h, wH);
      }
#pragma unroll
      for (int w = kWarps - 1; w >= 0; --w) {
        const float wK = runK[w][threadIdx.x];
        runK[w][threadIdx.x] = r;
        r = fmaf(runA[w][threadIdx.x], r, wK);
      }
      if (C == 1) carry = r;
    }
    __syncthreads();
    float hv[VEC], rv[VEC], before[L][VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      hv[v] = runH[at.warp][at.lane * VEC + v];
      rv[v] = runK[at.warp][at.lane * VEC + v];
    }
    T* pdx = dx + (here + L - 1) * p.D;
    T* pdg = dgate + (here + L - 1) * p.D;
    auto write = [&](auto full) {
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (decltype(full)::value || i < count) {
          float b[VEC];
#pragma unroll
          for (int v = 0; v < VEC; ++v) before[i][v] = MIX ? hv[v] - P::get(vx[i], v) : hv[v];
          inputs<T, VEC, MIX>(vx[i], rest[i], b);
          fma<VEC>(hv, a[i], hv, b);
        }
#pragma unroll
      for (int i = L - 1; i >= 0; --i) {
        if (decltype(full)::value || i < count) {
          float G[VEC], rG[VEC], og[VEC];
#pragma unroll
          for (int v = 0; v < VEC; ++v) G[v] = P::get(vd[i], v);
          add<VEC>(G, G, rv);
          mul<VEC>(rv, a[i], G);
          mul<VEC>(rG, rest[i], G);
          if constexpr (ACT == FAKLA_ACT_SIGMOID) {
            mul<VEC>(og, rG, a[i]);
            mul<VEC>(og, og, before[i]);
          } else {
            mul<VEC>(og, G, before[i]);
          }
          if (at.on) {
            __stcs((Raw*)pdx, P::put(MIX ? rG : G));
            __stcs((Raw*)pdg, P::put(og));
          }
        }
        pdx -= p.D;
        pdg -= p.D;
      }
    };
    if (count == L) write(std::true_type{});
    else write(std::false_type{});
  }
  if (C > 1) cluster_sync();
  if (p.dstate_in && at.walks && at.rank == 0) p.dstate_in[at.b * p.D + at.c] = carry;
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
  for (int v = 0; v < VEC; ++v) h[v] = p.state_in[b * p.D + d + v];
  float a[VEC], rest[VEC], in[VEC];
  gates<ACT, T, VEC>(rg, a, rest);
  inputs<T, VEC, MIX>(rx, rest, in);
  fma<VEC>(h, a, h, in);
#pragma unroll
  for (int v = 0; v < VEC; ++v) p.state_out[b * p.D + d + v] = h[v];
  *(Raw*)((T*)p.out + b * p.D + d) = P::put(h);
}

// Runs f with the type, channels per thread, gate activation and input form as
// constants. Channels go in fours (bf16) or twos where every row starts on a
// multiple of their size, and, for a scan of `tiles` tiles (0: one token), where
// the blocks then still reach every SM: 8 bytes of channels with 8 blocks on a
// sequence, 4 bytes with 16. bf16 forward, one / two / four channels a thread:
// 1 x 8192 x 512 takes 21 / 22 / 25 us, 1 x 16384 x 1024 73 / 54 / 57,
// 4 x 2048 x 512 21 / 14 / 17, 64 x 64 x 1024 13 / 11 / 9.
template <typename F>
void dispatch(int dtype, const GatedScanArgs& p, int64_t tiles, F f) {
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
  auto fits = [&](int vec, int bytes) {
    if (steps % vec != 0 || bases % (vec * bytes) != 0) return false;
    const int64_t most = vec * bytes == 8 ? kPortableCluster : kMaxCluster;
    return tiles == 0 || p.B * (p.D / (32 * vec)) * (tiles < most ? tiles : most) >= fakla_sm_count();
  };
  if (dtype == FAKLA_BF16) {
    if (fits(4, 2)) by_act(__nv_bfloat16{}, std::integral_constant<int, 4>{});
    else if (fits(2, 2)) by_act(__nv_bfloat16{}, std::integral_constant<int, 2>{});
    else by_act(__nv_bfloat16{}, std::integral_constant<int, 1>{});
  } else {
    if (fits(2, 4)) by_act(float{}, std::integral_constant<int, 2>{});
    else by_act(float{}, std::integral_constant<int, 1>{});
  }
}

// Blocks of a cluster, which share a sequence's time: as few as give four SMs
// five blocks, and no more than there are tiles. More blocks fill the SMs but
// wait longer for one another: 8 x 4096 x 2048 bf16 takes 104 us with 2 and
// 109 with 4, 3 x 1001 x 515 fp32 (forward and backward) 23 us with 4 and 28
// with 8, 65536 x 4096 bf16 434 us with 8, 710 with 4 and 633 with 16,
// 65536 x 64 95 us with 16 and 169 with 8.
int cluster_size(int64_t groups, int64_t tiles) {
  int c = 1;
  while (c < kMaxCluster && 2 * c <= tiles && groups * c * 4 < (int64_t)fakla_sm_count() * 5) c *= 2;
  return c;
}

template <typename K>
cudaError_t launch(K kernel, const GatedScanArgs& p, int vec, int64_t tiles, cudaStream_t stream) {
  const int64_t groups = p.B * ((p.D + 32 * vec - 1) / (32 * vec));
  const int c = cluster_size(groups, tiles);
  if (c > kPortableCluster) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  return launch_chained(kernel, dim3((unsigned)(groups * c)), dim3(kThreads), 0, stream, (unsigned)c, p, c);
}

}  // namespace

size_t gated_scan_saved_bytes(int64_t B, int64_t T, int64_t D) {
  return (size_t)B * (size_t)((T + kKept - 1) / kKept) * (size_t)D * sizeof(float);
}

cudaError_t launch_gated_scan(int dtype, const GatedScanArgs& p, cudaStream_t stream) {
  constexpr int kTile = kWarps * kForwardRun;
  const int64_t tiles = (p.T + kTile - 1) / kTile;
  cudaError_t e = cudaSuccess;
  dispatch(dtype, p, tiles, [&](auto t, auto vec, auto act, auto mix) {
    e = launch(scan_forward_kernel<decltype(t), vec(), act(), mix()>, p, vec(), tiles, stream);
  });
  return e;
}

cudaError_t launch_gated_scan_backward(int dtype, const GatedScanArgs& p, cudaStream_t stream) {
  const int64_t tiles = (p.T + kKept - 1) / kKept;
  cudaError_t e = cudaSuccess;
  dispatch(dtype, p, tiles, [&](auto t, auto vec, auto act, auto mix) {
    e = launch(scan_backward_kernel<decltype(t), vec(), act(), mix()>, p, vec(), tiles, stream);
  });
  return e;
}

cudaError_t launch_gated_scan_step(int dtype, const GatedScanArgs& p, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  dispatch(dtype, p, 0, [&](auto t, auto vec, auto act, auto mix) {
    const int64_t items = p.B * p.D / vec();
    e = launch_chained(scan_step_kernel<decltype(t), vec(), act(), mix()>,
                       dim3((unsigned)((items + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, 1u, p);
  });
  return e;
}

}  // namespace fakla
