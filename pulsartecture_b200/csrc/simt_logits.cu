// Rows of logits on CUDA cores: token log probabilities with entropy and the
// largest entries, and the divergence from a teacher's largest logits, with
// their gradients.
//
// With c = log2(e) / temperature, m = max x, M = c m and y_j = c x_j - M (one
// fused multiply-add, so y is exact but for its own rounding):
//   s = sum_j 2^{y_j},  log p_j = ln 2 (y_j - log2 s),
//   H = ln 2 (log2 s - (sum_j 2^{y_j} y_j) / s),
// both parts of H of one sign, so they do not cancel. The forward reads a row
// once: a thread keeps the maximum of what it has seen and rescales its sums
// when that grows; threads, and the blocks of a cluster where a row is split,
// merge theirs at the end in a fixed order. The backward recomputes p from m
// and log2 s, reading the logits once more and storing nothing in between.
// Memory bounds both: bf16 logits at 6.5 TB/s are 11 instructions per value on
// 148 SMs, and the passes take 5 to 8. Everything is fp32; dlogits are rounded
// once.
//
// Rows whose maximum is past 10^6 / c (a temperature close to 0, masks of a
// type's lowest value over all of a row) lose y in that form; they are summed
// once more from (x - m) / temperature, by one block, scalar by scalar. A row
// of nothing but -inf keeps log2 s = +inf, which makes every p 0.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "fakla_common.cuh"
#include "fakla_kernels.h"
#include "sm100_umma.cuh"

namespace fakla {
namespace {

// Few threads to a row: what each does once (its place, the merge of its sums)
// is spread over more values. With 256, 32000 bf16 values per row cost 13
// instructions each and 76 us for 4096 rows.
constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;      // 16-byte loads of a thread in flight
constexpr int kMaxCluster = 8;  // the largest portable cluster
constexpr int kMaxTop = 32;     // as fakla_token_logprobs takes; also the lanes of a warp
constexpr int kMaxEntries = 256;  // as fakla_distill_topk takes
constexpr int kMaxVocab = 1 << 20;  // as all of them take
constexpr int kCandidates = 512;
constexpr int kOneWarp = 16;
constexpr float kInf = __builtin_huge_valf();
constexpr float kNaN = __builtin_nanf("");
constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.693147181f;
constexpr float kFar = 1e6f;         // |c x| up to which y is formed by one fma
constexpr float kNear = 0.99f * kFar;  // and which a row's maximum keeps within

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint4 load_vec(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// 16 bytes of logits as pairs of fp32.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ uint64_t pair(const uint4& v, int i) {
    return i == 0 ? sm100::f2_make(v.x, v.y) : sm100::f2_make(v.z, v.w);
  }
  static __device__ __forceinline__ float max(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  // not below `low`; NaN stays
  static __device__ __forceinline__ uint4 at_least(uint4 v, float low) {
    auto f = [&](uint32_t x) {
      float r;
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(x)), "f"(low));
      return __float_as_uint(r);
    };
    return make_uint4(f(v.x), f(v.y), f(v.z), f(v.w));
  }
  static __device__ __forceinline__ uint4 put(const uint64_t* p) {
    const float2 a = sm100::f2_split(p[0]), b = sm100::f2_split(p[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ uint32_t word(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
  }
  static __device__ __forceinline__ __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  static __device__ __forceinline__ uint32_t bits(__nv_bfloat162 h) { return *reinterpret_cast<uint32_t*>(&h); }
  static __device__ __forceinline__ uint64_t pair(const uint4& v, int i) { return sm100::f2_from_bf16x2(word(v, i)); }
  static __device__ __forceinline__ float max(const uint4& v) {
    const uint32_t w = bits(__hmax2(__hmax2(two(v.x), two(v.y)), __hmax2(two(v.z), two(v.w))));
    return fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 at_least(uint4 v, float low) {
    const __nv_bfloat162 l = __bfloat162bfloat162(__float2bfloat16_rd(low));  // at or below it: y stays at or below 0
    auto f = [&](uint32_t x) { return bits(__hmax2_nan(two(x), l)); };
    return make_uint4(f(v.x), f(v.y), f(v.z), f(v.w));
  }
  static __device__ __forceinline__ uint4 put(const uint64_t* p) {
    return make_uint4(sm100::pack_bf16x2(p[0]), sm100::pack_bf16x2(p[1]), sm100::pack_bf16x2(p[2]), sm100::pack_bf16x2(p[3]));
  }
};

// A row in 16-byte vectors, with up to E - 1 single values before and after
// them where the row does not start or end on 16 bytes.
template <typename T>
struct Row {
  static constexpr int E = Vec<T>::E;
  const T* x;
  int V, lead, vectors, singles;
  __device__ Row(const LogitsArgs& p, uint32_t row) {
    const uint32_t rows = (uint32_t)p.rows, i = p.batch == 1 ? 0 : row / rows;
    x = (const T*)p.logits + i * p.batch_stride + (row - i * rows) * p.row_stride;
    V = (int)p.vocab;
    lead = (int)(-(intptr_t)x & 15) / (int)sizeof(T);
    if (lead > V) lead = V;
    vectors = (V - lead) / E;
    singles = V - vectors * E;
  }
  __device__ const T* vec(int v) const { return x + lead + v * E; }
  __device__ int single(int i) const { return i < lead ? i : i + vectors * E; }
  // the place of value j: its vector, or -1 - (its number among the singles)
  __device__ int place(int j) const {
    if (j < lead) return -1 - j;
    const int v = (j - lead) / E;
    return v < vectors ? v : -1 - (j - vectors * E);
  }
};

__device__ __forceinline__ float scale_of(const LogitsArgs& p) { return kLog2e * p.inv_temperature; }

// What a row's values, or some of them, add up to.
struct Sums {
  float m;  // the largest value
  float s;  // sum 2^y
  float w;  // sum 2^y y
};

// M of a maximum m, kept finite for -inf.
__device__ __forceinline__ float base_of(float m, float c) { return fmaxf(__fmul_rn(m, c), -kFar); }

// The sums over `width` neighbouring lanes (a power of two), in each of them:
// all are moved to the largest value's base once, then added in a fixed order.
template <bool WEIGHTED>
__device__ __forceinline__ Sums merge_lanes(Sums a, float c, int width) {
  float m = a.m;
  for (int o = width / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  const float move = base_of(a.m, c) - base_of(m, c), f = exp2_approx(move);
  if (WEIGHTED) a.w = f * fmaf(move, a.s, a.w);
  a.s *= f;
  for (int o = width / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(~0u, a.s, o);
    if (WEIGHTED) a.w += __shfl_xor_sync(~0u, a.w, o);
  }
  a.m = m;
  return a;
}

// One thread's running sums. WEIGHTED: the entropy's.
template <typename T, bool WEIGHTED>
struct Running {
  static constexpr int E = Vec<T>::E;
  float m, M, c;
  uint64_t c2, s2, w2;
  __device__ explicit Running(float c_) : m(-kInf), M(-kFar), c(c_), c2(sm100::f2_splat(c_)) {
    s2 = w2 = sm100::f2_splat(0.f);
  }
  __device__ __forceinline__ void see(float most) {
    if (most > m) {
      m = most;
      const float to = base_of(m, c);
      const uint64_t f = sm100::f2_splat(exp2_approx(M - to));
      if (WEIGHTED) w2 = sm100::f2_mul(f, sm100::f2_fma(sm100::f2_splat(M - to), s2, w2));
      s2 = sm100::f2_mul(f, s2);
      M = to;
    }
  }
  __device__ __forceinline__ void add(uint4 v) {
    if (WEIGHTED) v = Vec<T>::at_least(v, -kFar / c);  // 2^y y is 0 there, not 0 times -inf
    const uint64_t nM = sm100::f2_splat(-M);
    uint64_t all = 0;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const uint64_t y = sm100::f2_fma(Vec<T>::pair(v, i), c2, nM);
      const float2 f = sm100::f2_split(y);
      const uint64_t e = sm100::f2_make(__float_as_uint(exp2_approx(f.x)), __float_as_uint(exp2_approx(f.y)));
      all = i == 0 ? e : sm100::f2_add(all, e);
      if (WEIGHTED) w2 = sm100::f2_fma(e, y, w2);
    }
    s2 = sm100::f2_add(s2, all);
  }
  __device__ __forceinline__ void add_single(float x) {
    see(x);
    const float y = fmaf(WEIGHTED ? (x < -kFar / c ? -kFar / c : x) : x, c, -M), e = exp2_approx(y);
    s2 = sm100::f2_add(s2, sm100::f2_make(__float_as_uint(e), 0u));
    if (WEIGHTED) w2 = sm100::f2_fma(sm100::f2_make(__float_as_uint(e), 0u), sm100::f2_make(__float_as_uint(y), 0u), w2);
  }
  __device__ Sums sums() const {
    auto both = [](uint64_t v) { const float2 f = sm100::f2_split(v); return f.x + f.y; };
    return {m, both(s2), WEIGHTED ? both(w2) : 0.f};
  }
};

// Runs f(vectors, the first one's number) on every thread's vectors of
// [v0, v1), kUnroll at a time, kThreads apart; the next ones are on their way
// meanwhile. Past v1 the values are -inf, which add nothing. `first` is done
// while the first of them are on their way.
template <typename T, typename G, typename F>
__device__ __forceinline__ void each_vectors(const Row<T>& row, int v0, int v1, G first, F f) {
  auto fetch = [&](uint4* raw, int v) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      constexpr uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
      raw[u] = make_uint4(none, none, none, none);
      if (v + u * kThreads < v1) raw[u] = load_vec(row.vec(v + u * kThreads));
    }
  };
  constexpr int step = kUnroll * kThreads;
  uint4 even[kUnroll], odd[kUnroll];
  int v = v0 + threadIdx.x;
  fetch(even, v);
  first();
  while (v < v1) {
    fetch(odd, v + step);
    f(even, v);
    v += step;
    if (v >= v1) break;
    fetch(even, v + step);
    f(odd, v);
    v += step;
  }
}

// The sums over the block, in every thread.
template <bool WEIGHTED>
__device__ __forceinline__ Sums merge_block(Sums a, float c) {
  __shared__ Sums part[kWarps];
  a = merge_lanes<WEIGHTED>(a, c, 32);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = a;
  __syncthreads();
  return merge_lanes<WEIGHTED>(part[threadIdx.x % kWarps], c, kWarps);
}

__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename V>
__device__ __forceinline__ V* in_block(V* mine, uint32_t rank) {
  uint64_t there;
  asm("mapa.u64 %0, %1, %2;" : "=l"(there) : "l"((uint64_t)mine), "r"(rank));
  return (V*)there;
}

// The finished statistics of a row: p_j = 2^{y_j - l2s}.
struct Stats {
  float m, M;
  float l2s;   // log2 s; +inf in a row of nothing but -inf, NaN in one with a NaN or +inf
  float mean;  // sum p y
  float s;     // sum 2^y (by `finish`)
  bool far;    // y from (x - m) / temperature
  float c, inv_t;
  __device__ bool empty() const { return l2s == kInf; }
  __device__ float y(float x) const { return far ? (x - m) * inv_t * kLog2e : fmaf(x, c, -M); }
  __device__ float logprob(float x) const {
    if (empty()) return -kInf;
    // c x may be past fp32 where the log probability is not
    if (far || !(fabsf(x * c) <= kFar)) return (x - m) * inv_t - kLn2 * l2s;
    return kLn2 * (y(x) - l2s);
  }
};

// Reads back what the forward kept of a row.
__device__ __forceinline__ Stats stats_of(const LogitsArgs& p, float m, float l2s) {
  Stats r;
  r.m = m;
  r.l2s = l2s;
  r.c = scale_of(p);
  r.inv_t = p.inv_temperature;
  r.far = !(fabsf(__fmul_rn(m, r.c)) <= kNear);
  r.M = base_of(m, r.c);
  return r;
}

// By all threads of the block.
template <typename T, bool WEIGHTED>
__device__ Stats finish(const LogitsArgs& p, const Row<T>& row, Sums a) {
  Stats r = stats_of(p, a.m == -kInf ? 0.f : a.m, 0.f);
  const bool none = a.m == -kInf && !isnan(a.s);
  if (r.far) {  // the same for every thread
    float s = 0.f, w = 0.f;
    for (int j = threadIdx.x; j < row.V; j += kThreads) {
      const float y = (to_f32(row.x[j]) - r.m) * r.inv_t * kLog2e, e = exp2f(y);
      s += e;
      if (WEIGHTED) w += e == 0.f ? 0.f : e * y;
    }
    __shared__ float part[2][kWarps];
    float v[2] = {s, w};
    for (int i = 0; i < 2; ++i) {
      for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(~0u, v[i], o);
      if (threadIdx.x % 32 == 0) part[i][threadIdx.x / 32] = v[i];
    }
    __syncthreads();
    a.s = a.w = 0.f;
    for (int i = 0; i < kWarps; ++i) {
      a.s += part[0][i];
      a.w += part[1][i];
    }
  }
  r.s = a.s;
  if (none || a.s == 0.f) {
    r.l2s = kInf;
    r.mean = 0.f;
  } else {
    r.l2s = log2f(a.s);
    r.mean = a.w / a.s;
  }
  return r;
}

// ---------------------------------------------------------------------------
// The largest values of a row
// ---------------------------------------------------------------------------
// Order of the values (-0 as 0), then of the lower index. No value has key 0.
__device__ __forceinline__ uint64_t order_key(float x, int j) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)o << 32 | (uint32_t)~j;
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// The pass that sums a row leaves the maximum of each vector in shared memory.
// The k-th largest of the threads' own largest maxima has k values at or above
// it, so only values from there up can be among the k largest: some 5 for k = 5
// and 37 for k = 32 in a random row. Up to kOneWarp the threads of a lane go
// together, and one warp finds the k-th of 32: 8192 x 32000 bf16 with k = 5
// takes 123 us so and 127 us from 128 keys; with k = 32 that leaves 130
// candidates, and 301 x 50257 fp32 takes 34 us so and 28 us from 128. The
// values are in the vectors whose maximum reaches the threshold; those are
// listed first and then read again all at once, by a thread per value. Keys,
// which hold the index too, differ even between equal values, so rows of ties
// fill no list: threads interleave finely, and a row of one value lists its
// first 256 or so.
struct TopSpace {
  uint64_t best[kWarps][32];
  uint64_t list[kCandidates];
  int vectors[kCandidates];
  uint64_t top[kMaxTop];
  uint64_t floor;
  int vector_count, count;
};

// Every key >= floor of the block's part of the row goes into the list; returns
// their number, more than kCandidates if that or their vectors are too many.
template <typename T>
__device__ __forceinline__ int collect(TopSpace& sp, const Row<T>& row, int v0, int v1, bool singles,
                                       const T* most) {
  constexpr int E = Row<T>::E;
  const uint64_t floor = sp.floor;
  const float least = floor == 0 ? -kInf : key_value(floor);
  // equal maxima count up to the vector of the floor's own index
  const int last = floor == 0 ? v1 : (key_index(floor) - row.lead) / E;
  for (int v = v0 + threadIdx.x; v < v1; v += kThreads)
    if (const float m = to_f32(most[v - v0]); m > least || (m == least && v <= last)) {
      const int at = atomicAdd(&sp.vector_count, 1);
      if (at < kCandidates) sp.vectors[at] = v;
    }
  __syncthreads();
  const int n = sp.vector_count;
  if (n > kCandidates) return n;
  auto take = [&](int j) {
    const uint64_t key = order_key(to_f32(row.x[j]), j);
    if (key >= floor) {
      const int at = atomicAdd(&sp.count, 1);
      if (at < kCandidates) sp.list[at] = key;
    }
  };
  for (int i = threadIdx.x; i < n * E; i += kThreads) take(row.lead + sp.vectors[i / E] * E + i % E);
  if (singles && threadIdx.x < row.singles) take(row.single(threadIdx.x));
  __syncthreads();
  return sp.count;
}

// Puts the k largest keys of list[0, n) in descending order into top; the
// rest of top is 0.
__device__ __forceinline__ void rank_list(const uint64_t* list, int n, int k, uint64_t* top) {
  if (threadIdx.x < kMaxTop && threadIdx.x >= min(n, k)) top[threadIdx.x] = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t key = list[i];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) above += list[j] > key;
    if (above < k) top[above] = key;
  }
  __syncthreads();
}

// The keys of a warp in descending order over its lanes, by exchanges over
// growing and shrinking distances (a bitonic network).
__device__ __forceinline__ uint64_t sort_warp(uint64_t key) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int run = 2; run <= 32; run *= 2)
#pragma unroll
    for (int o = run / 2; o > 0; o /= 2) {
      const uint64_t other = __shfl_xor_sync(~0u, key, o);
      const bool larger = ((lane & o) == 0) == ((lane & run) == 0);  // this lane keeps the larger one
      key = (other > key) == larger ? other : key;
    }
  return key;
}

// How many of 32 keys in descending order are above `key` (or equal to it).
__device__ __forceinline__ int count_above(const uint64_t* list, uint64_t key, bool or_equal) {
  int n = 0;
#pragma unroll
  for (int step = 16; step > 0; step /= 2)
    if (list[n + step - 1] > key || (or_equal && list[n + step - 1] == key)) n += step;
  return n + (list[n] > key || (or_equal && list[n] == key));
}

// The k largest of C blocks' top keys, each in descending order (kMaxTop
// apart), into top: a key's rank is its place in its own list and the number of
// larger ones in each other.
__device__ __forceinline__ void merge_lists(const uint64_t* lists, int C, int k, uint64_t* top) {
  for (int i = threadIdx.x; i < C * k; i += kThreads) {
    const int own = i / k;
    const uint64_t key = lists[own * kMaxTop + (i - own * k)];
    int above = 0;
    for (int c = 0; c < C; ++c) above += count_above(lists + c * kMaxTop, key, false);
    if (above < k) top[above] = key;
  }
  __syncthreads();
}

// The k largest keys of the block's part of the row, into sp.top.
template <typename T>
__device__ __forceinline__ void block_top(TopSpace& sp, const Row<T>& row, int v0, int v1, bool singles,
                                          const T* most, int k) {
  // the thread's largest maximum of a vector, with the last index it can have
  float best = -kInf;
  int at = -1;
  for (int v = v0 + threadIdx.x; v < v1; v += kThreads) {
    const float m = to_f32(most[v - v0]);
    if (m > best || at < 0) {
      best = m;
      at = v;
    }
  }
  uint64_t key = at < 0 ? 0 : order_key(best, row.lead + at * Row<T>::E + Row<T>::E - 1);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (threadIdx.x == 0) sp.count = sp.vector_count = 0;
  // Those without a vector share key 0, in the order of the threads: the k-th
  // is one of them where fewer have any, and then every value qualifies.
  if (k <= kOneWarp) {
    sp.best[warp][lane] = key;
    __syncthreads();
    if (warp == 0) {
      for (int w = 1; w < kWarps; ++w) key = sp.best[w][lane] > key ? sp.best[w][lane] : key;
      key = sort_warp(key);
      if (lane == k - 1) sp.floor = key;
    }
  } else {
    key = sort_warp(key);
    sp.best[warp][lane] = key;
    __syncthreads();
    int above = lane;
    for (int w = 0; w < kWarps; ++w)
      if (w != warp) above += count_above(sp.best[w], key, w < warp);
    if (above == k - 1) sp.floor = key;
  }
  __syncthreads();
  const int n = collect(sp, row, v0, v1, singles, most);
  if (n <= kCandidates) {
    rank_list(sp.list, n, k, sp.top);
    return;
  }
  __syncthreads();
  // More than the list holds (large values in few lanes): the largest below
  // the last one found, k times over the block's part.
  uint64_t last = ~0ull;
  for (int i = 0; i < kMaxTop; ++i) {
    uint64_t most_key = 0;
    if (i < k) {
      for (int v = v0 + threadIdx.x; v < v1; v += kThreads)
        for (int e = 0; e < Row<T>::E; ++e) {
          const int j = row.lead + v * Row<T>::E + e;
          const uint64_t q = order_key(to_f32(row.x[j]), j);
          if (q < last && q > most_key) most_key = q;
        }
      if (singles && threadIdx.x < row.singles) {
        const int j = row.single(threadIdx.x);
        const uint64_t q = order_key(to_f32(row.x[j]), j);
        if (q < last && q > most_key) most_key = q;
      }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t q = __shfl_xor_sync(~0u, most_key, o);
      most_key = q > most_key ? q : most_key;
    }
    __syncthreads();
    if (threadIdx.x % 32 == 0) sp.best[0][threadIdx.x / 32] = most_key;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) most_key = sp.best[0][w] > most_key ? sp.best[0][w] : most_key;
    last = most_key;
    if (threadIdx.x == 0) sp.top[i] = most_key;
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------
// Token log probabilities
// ---------------------------------------------------------------------------
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(LogitsArgs p, int C) {
  extern __shared__ __align__(16) unsigned char most_space[];
  T* most = reinterpret_cast<T*>(most_space);  // TOP: the maximum of each of the block's vectors
  __shared__ std::conditional_t<TOP, TopSpace, int> space;
  __shared__ Sums peers[kMaxCluster];
  __shared__ uint64_t peer_top[TOP ? kMaxCluster * kMaxTop : 1];
  griddep_wait();
  const uint32_t r = blockIdx.x / C;
  const int rank = C > 1 ? (int)sm100::cluster_ctarank() : 0;
  if (C > 1) cluster_arrive();
  const Row<T> row(p, r);
  const int per = (row.vectors + C - 1) / C;
  const int v0 = min(rank * per, row.vectors), v1 = min(v0 + per, row.vectors);
  Running<T, true> run(scale_of(p));
  const int64_t t = rank == 0 && threadIdx.x == 0 ? p.targets[r] : -1;
  each_vectors(row, v0, v1, [] {}, [&](const uint4* raw, int v) {
    float top = -kInf;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const float m = Vec<T>::max(raw[u]);
      if (TOP && v + u * kThreads < v1) most[v + u * kThreads - v0] = from_f32<T>(m);
      top = fmaxf(top, m);
    }
    run.see(top);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) run.add(raw[u]);
  });
  const bool singles = rank == 0;
  if (singles && threadIdx.x < row.singles) run.add_single(to_f32(row.x[row.single(threadIdx.x)]));
  const float target = t >= 0 && t < row.V ? to_f32(row.x[t]) : 0.f;
  Sums a = merge_block<true>(run.sums(), run.c);
  if constexpr (TOP) block_top(space, row, v0, v1, singles, most, p.top_k);
  if (C > 1) {
    cluster_wait();  // every block has begun
    if (threadIdx.x == 0) *in_block(&peers[rank], 0) = a;
    if constexpr (TOP)
      if (threadIdx.x < kMaxTop) *in_block(&peer_top[rank * kMaxTop + threadIdx.x], 0) = space.top[threadIdx.x];
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    a = merge_lanes<true>(peers[threadIdx.x % C], run.c, C);
    if constexpr (TOP) merge_lists(peer_top, C, p.top_k, space.top);
  }
  const Stats st = finish<T, true>(p, row, a);
  if (threadIdx.x == 0) {
    float lp = 0.f;
    if (t != p.ignore_index) {
      if (t >= 0 && t < row.V) {
        lp = st.logprob(target);
      } else {
        lp = kNaN;
        report_status(p.status, FAKLA_ERR_INVALID_ARG);
      }
    }
    p.logprobs[r] = lp;
    p.entropy[r] = st.empty() ? 0.f : kLn2 * (st.l2s - st.mean);
    if (p.stats) {
      p.stats[(int64_t)r * kTokenStats] = st.m;
      p.stats[(int64_t)r * kTokenStats + 1] = st.l2s;
    }
  }
  if constexpr (TOP)
    if (threadIdx.x < p.top_k) {
      const uint64_t key = space.top[threadIdx.x];
      const bool bad = isnan(st.l2s);
      p.top_ids[(int64_t)r * p.top_k + threadIdx.x] = bad ? -1 : key_index(key);
      p.top_logprobs[(int64_t)r * p.top_k + threadIdx.x] = bad ? kNaN : st.logprob(key_value(key));
    }
}

// ---------------------------------------------------------------------------
// Gradients: one block per `span` vectors of a row
// ---------------------------------------------------------------------------
constexpr int kRound = kUnroll * kThreads;  // vectors of a block's loads in flight

// Writes f(pair of logits) over the block's vectors [v0, v1) of a row, or zeros.
// Stores are as wide as the loads where both rows lie alike. `first` is done
// while the first loads are on their way, not with zeros; `patch` changes a
// vector's results (given its logits and number) before they are stored.
template <typename T, typename G, typename F, typename P>
__device__ __forceinline__ void map_vectors(const Row<T>& row, T* out, int v0, int v1, bool zero, G first, F f, P patch) {
  const bool wide = (((uintptr_t)row.x ^ (uintptr_t)out) & 15) == 0;
  auto put = [&](uint4 got, int v) {
    T* to = out + row.lead + v * Row<T>::E;
    if (wide) {
      __stcs(reinterpret_cast<uint4*>(to), got);
    } else {
      const T* e = reinterpret_cast<const T*>(&got);
#pragma unroll
      for (int i = 0; i < Row<T>::E; ++i) to[i] = e[i];
    }
  };
  if (zero) {
    for (int v = v0 + threadIdx.x; v < v1; v += kThreads) put(make_uint4(0, 0, 0, 0), v);
    return;
  }
  each_vectors(row, v0, v1, first, [&](const uint4* raw, int v) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v + u * kThreads < v1) {
        uint64_t d[Row<T>::E / 2];
#pragma unroll
        for (int i = 0; i < Row<T>::E / 2; ++i) d[i] = f(raw[u], i);
        uint4 got = Vec<T>::put(d);
        patch(got, raw[u], v + u * kThreads);
        put(got, v + u * kThreads);
      }
  });
}

// Whether value j of the row is written by the block of vectors [v0, v1).
template <typename T>
__device__ __forceinline__ bool writes(const Row<T>& row, int j, int chunk, int v0, int v1) {
  const int v = row.place(j);
  return v < 0 ? chunk == 0 : v >= v0 && v < v1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_backward_kernel(LogitsArgs p, int chunks, int span) {
  griddep_wait();
  const uint32_t r = blockIdx.x / chunks;
  const int chunk = blockIdx.x - r * chunks;
  const Row<T> row(p, r);
  const int v0 = min(chunk * span, row.vectors), v1 = min(v0 + span, row.vectors);
  T* out = (T*)p.dlogits + (int64_t)r * p.vocab;
  const Stats st = stats_of(p, p.stats[(int64_t)r * kTokenStats], p.stats[(int64_t)r * kTokenStats + 1]);
  const int64_t t = p.targets[r];
  const bool counted = t != p.ignore_index, good = t >= 0 && t < row.V;
  float w = counted && p.dlogprobs ? p.dlogprobs[r] : 0.f;
  if (w != 0.f && !good) w = kNaN;
  const float h = p.dentropy ? p.dentropy[r] : 0.f;
  float total = w;
  bool given = w != 0.f || h != 0.f;
  for (int k = 0; k < p.top_k; ++k) {
    const float d = p.dtop_logprobs[(int64_t)r * p.top_k + k];
    total += d;
    given |= d != 0.f;
  }
  // dlogits_j = p_j (flat + slope log2 p_j), and what is given to j itself
  const float flat = -(total + (h == 0.f ? 0.f : h * p.entropy[r])) * p.inv_temperature;
  const float slope = -h * kLn2 * p.inv_temperature;
  // 2^l is 0 from kNone down, whose product with the slope (up to 10^30 times
  // what is given, at the lowest temperature) is finite
  constexpr float kNone = -200.f;
  auto value = [&](float x) {
    const float l = st.y(x) - st.l2s;
    return exp2_approx(l) * fmaf(fmaxf(l, kNone), slope, flat);
  };
  // a row that is given nothing gets 0 even where its p are NaN
  const bool zero = st.empty() || !given;
  if (st.far) {
    for (int j = row.lead + v0 * Row<T>::E + threadIdx.x; j < row.lead + v1 * Row<T>::E; j += kThreads)
      out[j] = from_f32<T>(zero ? 0.f : value(to_f32(row.x[j])));
  } else {
    const uint64_t c2 = sm100::f2_splat(st.c), nM = sm100::f2_splat(-st.M), nl = sm100::f2_splat(-st.l2s);
    const uint64_t f2 = sm100::f2_splat(flat), s2 = sm100::f2_splat(slope);
    const float low = (st.M + kNone) / st.c;
    auto map = [&](auto sloped) {
      map_vectors(row, out, v0, v1, zero, [] {}, [&](const uint4& raw, int i) {
        uint4 v = raw;
        if constexpr (decltype(sloped)::value) v = Vec<T>::at_least(raw, low);  // p log p is 0 there
        const uint64_t l = sm100::f2_add(sm100::f2_fma(Vec<T>::pair(v, i), c2, nM), nl);
        const float2 f = sm100::f2_split(l);
        const uint64_t e = sm100::f2_make(__float_as_uint(exp2_approx(f.x)), __float_as_uint(exp2_approx(f.y)));
        if constexpr (decltype(sloped)::value) return sm100::f2_mul(e, sm100::f2_fma(l, s2, f2));
        else return sm100::f2_mul(e, f2);
      }, [](uint4&, const uint4&, int) {});
    };
    if (slope == 0.f) map(std::false_type{});
    else map(std::true_type{});
  }
  if (chunk == 0 && threadIdx.x < row.singles) {
    const int j = row.single(threadIdx.x);
    out[j] = from_f32<T>(zero ? 0.f : value(to_f32(row.x[j])));
  }
  if (zero) return;
  __syncthreads();
  // the target and the alternatives once more, with their own gradients
  if (threadIdx.x < p.top_k) {
    const int64_t j = p.top_ids[(int64_t)r * p.top_k + threadIdx.x];
    if (j >= 0 && j < row.V && writes(row, (int)j, chunk, v0, v1)) {
      float d = p.dtop_logprobs[(int64_t)r * p.top_k + threadIdx.x];
      if (counted && j == t) d += w;
      out[j] = from_f32<T>(fmaf(d, p.inv_temperature, value(to_f32(row.x[j]))));
    }
  } else if (threadIdx.x == kMaxTop && counted && good && w != 0.f && writes(row, (int)t, chunk, v0, v1)) {
    for (int k = 0; k < p.top_k; ++k)
      if (p.top_ids[(int64_t)r * p.top_k + k] == t) return;
    out[t] = from_f32<T>(fmaf(w, p.inv_temperature, value(to_f32(row.x[t]))));
  }
}

// ---------------------------------------------------------------------------
// Distillation
// ---------------------------------------------------------------------------
// The teacher's side of a row: q_k = e^{t_k / temperature - m / temperature - logs}.
struct Teacher {
  float m, logs;  // logs +inf: no distribution, every q is 0
  float mass;     // sum of the q
  float rest;     // what is left for the other entries (teacher_lse given)
  bool bad;       // an id out of range
  bool twice;     // an id that is there more than once
};

__device__ __forceinline__ float teacher_q(const LogitsArgs& p, int id, float logit, float m, float logs, float& lq) {
  lq = -kInf;
  if (id < 0) return 0.f;
  lq = (logit - m) * p.inv_temperature - logs;
  return expf(lq);
}

constexpr int kPerThread = kMaxEntries / kThreads;  // entries of a thread: threadIdx.x + i * kThreads

// A thread's entries of a row, read at the start, while the block has nothing
// else to do, for the end.
struct Entries {
  int id[kPerThread];  // -1: none
  float logit[kPerThread];
  bool bad;            // one of them is out of range
  float lse;           // the row's teacher_lse, or 0
  __device__ __forceinline__ void read(const LogitsArgs& p, uint32_t r) {
    bad = false;
    lse = p.teacher_lse ? p.teacher_lse[r] : 0.f;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int k = threadIdx.x + i * kThreads;
      id[i] = -1;
      logit[i] = 0.f;
      if (k < p.entries) {
        const int64_t got = p.teacher_ids[(int64_t)r * p.entries + k];
        logit[i] = p.teacher_logits[(int64_t)r * p.entries + k];
        if (got >= 0 && got < p.vocab) id[i] = (int)got;
        else bad |= got != -1;
      }
    }
  }
};

// The teacher's entries of a row as a set: a table of ids, at most half full,
// each with the first entry that names it. Which of several that is does not
// depend on which came first to the table.
constexpr int kSlots = 2 * kMaxEntries;
struct EntrySet {
  static constexpr uint32_t kFree = ~0u;
  uint32_t slot[kSlots];  // id * kMaxEntries + entry
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kSlots; i += kThreads) slot[i] = kFree;
  }
  static __device__ __forceinline__ uint32_t place(uint32_t id) { return id * 2654435769u >> 23; }
  // false where another entry of this id was in already
  __device__ __forceinline__ bool put(uint32_t id, uint32_t entry) {
    const uint32_t own = id * kMaxEntries + entry;
    for (uint32_t h = place(id);; h = (h + 1) % kSlots) {
      const uint32_t was = atomicCAS(&slot[h], kFree, own);
      if (was == kFree) return true;
      if (was / kMaxEntries != id) continue;
      atomicMin(&slot[h], own);
      return false;
    }
  }
  // the slot of id, or a free one
  __device__ __forceinline__ uint32_t find(uint32_t id) const {
    for (uint32_t h = place(id);; h = (h + 1) % kSlots) {
      const uint32_t in = slot[h];
      if (in == kFree || in / kMaxEntries == id) return in;
    }
  }
  __device__ __forceinline__ bool holds(int id) const { return find(id) != kFree; }
  __device__ __forceinline__ bool is_first(int id, int entry) const { return find(id) % kMaxEntries == entry; }
};
static_assert((uint64_t)kMaxVocab * kMaxEntries < EntrySet::kFree, "a slot holds an id and an entry");
static_assert(kSlots == 1 << (32 - 23), "place() gives a slot");

// Both sums over the block, in every thread; once per N in a kernel.
template <int N>
__device__ __forceinline__ float2 sum_block(float2 v) {
  __shared__ float2 part[kWarps];
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(~0u, v.x, o);
    v.y += __shfl_xor_sync(~0u, v.y, o);
  }
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) {
    v.x += part[i].x;
    v.y += part[i].y;
  }
  return v;
}

// By the whole block.
__device__ __forceinline__ Teacher teacher_stats(const LogitsArgs& p, const Entries& e, bool twice) {
  Teacher t;
  t.m = 0.f;
  t.logs = e.lse;
  if (!p.teacher_lse) {
    __shared__ float part[kWarps];
    float m = -kInf;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (e.id[i] >= 0) m = fmaxf(m, e.logit[i]);
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) m = fmaxf(m, part[i]);
    if (m != -kInf) t.m = m;
  }
  // sum q; how many threads have an entry, a repeated one (2^8 each), a bad one (2^16 each)
  float2 s = make_float2(0.f, (twice ? 256.f : 0.f) + (e.bad ? 65536.f : 0.f));
  bool some = false;
  float lq;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    some |= e.id[i] >= 0;
    s.x += teacher_q(p, e.id[i], e.logit[i], t.m, t.logs, lq);
  }
  s.y += some;
  s = sum_block<0>(s);
  const uint32_t threads = (uint32_t)s.y;
  some = threads % 256 != 0;
  t.twice = threads / 256 % 256 != 0;
  t.bad = threads / 65536 != 0;
  if (p.teacher_lse) {
    if (!some) t.logs = kInf;
    t.mass = some ? s.x : 0.f;
    t.rest = some ? fmaxf(0.f, 1.f - s.x) : 0.f;
  } else {
    t.logs = s.x == 0.f ? kInf : logf(s.x);
    t.mass = s.x == 0.f ? 0.f : 1.f;
    t.rest = 0.f;
  }
  return t;
}

// The logits that are no entries, of a row without NaN or +inf: the largest and
// the sum of e^{(x - m) / temperature}. By the whole block.
struct Outside {
  float m, s;
};
template <typename T>
__device__ __forceinline__ Outside sum_outside(const Row<T>& row, const EntrySet& set, const Stats& st) {
  __shared__ float part[kWarps];
  Outside r = {-kInf, 0.f};
  for (int j0 = threadIdx.x; j0 < row.V; j0 += kUnroll * kThreads) {
    float x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int j = j0 + u * kThreads;
      x[u] = j < row.V ? to_f32(row.x[j]) : -kInf;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const float y = (x[u] - r.m) * st.c;
      if (x[u] == -kInf || y < -150.f || set.holds(j0 + u * kThreads)) continue;
      if (x[u] > r.m) {
        r.s = fmaf(r.s, exp2_approx(-y), 1.f);
        r.m = x[u];
      } else {
        r.s += exp2_approx(y);
      }
    }
  }
  float m = r.m;
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) m = fmaxf(m, part[i]);
  return {m, sum_block<2>({r.m == -kInf ? 0.f : r.s * exp2_approx((r.m - m) * st.c), 0.f}).x};
}

// With teacher_lse, what is left over is one more class: q_r = 1 - Q against
// p_r = 1 - P, with P the sum of p at the entries, each once. An error d of P
// is one of d q_r / p_r of the loss, no more than those of its other terms
// unless the model leaves much less than the teacher; rows where it leaves less
// than a quarter of q_r are walked once more for p_r itself, from the largest
// logit outside: p_r may be far below the smallest fp32 number, where its
// logarithm and the p / p_r of the gradient still are ordinary ones. Below
// 2^-10^6 it counts as 0 (masks of a type's lowest value). (Keeping
// that sum in the pass, by a byte of marks per vector, took 8 us of the 59 of
// 4096 x 32000 bf16 with 64 entries.) The ratio q_r / p_r is 1 + (P - Q) / p_r, whose
// difference keeps its digits where the entries hold little: the quotient is
// off by up to 2 10^-5 of such a loss, this by 10^-6. Where every
// row is walked (K = 16), 4096 x 32000 bf16 takes 270 us instead of 50. Twelve
// blocks on an SM (40 registers a thread, 8 to 16 bytes of them spilled) or
// nine (56 registers): bf16 50 and 53 us, 2048 x 32000 fp32 51 and 47.
template <typename T>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 12 : 9) distill_kernel(LogitsArgs p, int C) {
  __shared__ EntrySet set;
  __shared__ Sums peers[kMaxCluster];
  griddep_wait();
  const uint32_t r = blockIdx.x / C;
  const int rank = C > 1 ? (int)sm100::cluster_ctarank() : 0;
  if (C > 1) cluster_arrive();
  const Row<T> row(p, r);
  const int per = (row.vectors + C - 1) / C;
  const int v0 = min(rank * per, row.vectors), v1 = min(v0 + per, row.vectors);
  Running<T, false> run(scale_of(p));
  Entries entries;
  float given[kPerThread];  // the model's logits there
  bool fresh[kPerThread];   // the first of its id: counted in P
  Teacher t;
  auto first = [&] {
    if (rank != 0) return;
    entries.read(p, r);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) given[i] = entries.id[i] >= 0 ? to_f32(row.x[entries.id[i]]) : 0.f;
    set.clear();
    __syncthreads();
    bool twice = false;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      if (entries.id[i] < 0) continue;
      twice |= !set.put(entries.id[i], threadIdx.x + i * kThreads);
    }
    __syncwarp();  // threads that looked further are waited for here, not all along the row
    t = teacher_stats(p, entries, twice);  // (has a barrier: the table is complete)
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      fresh[i] = entries.id[i] >= 0 && (!t.twice || set.is_first(entries.id[i], threadIdx.x + i * kThreads));
    __syncwarp();
  };
  each_vectors(row, v0, v1, first, [&](const uint4* raw, int v) {
    float top = -kInf;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) top = fmaxf(top, Vec<T>::max(raw[u]));
    run.see(top);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) run.add(raw[u]);
  });
  if (rank == 0 && threadIdx.x < row.singles) run.add_single(to_f32(row.x[row.single(threadIdx.x)]));
  Sums a = merge_block<false>(run.sums(), run.c);
  if (C > 1) {
    cluster_wait();
    if (threadIdx.x == 0) *in_block(&peers[rank], 0) = a;
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    a = merge_lanes<false>(peers[threadIdx.x % C], run.c, C);
  }
  const Stats st = finish<T, false>(p, row, a);
  float2 sums = make_float2(0.f, 0.f);  // of the entries' terms, and of 2^y at them
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    float lq;
    const float q = teacher_q(p, entries.id[i], entries.logit[i], t.m, t.logs, lq);
    if (q != 0.f) sums.x += q * (lq - st.logprob(given[i]));
    if (fresh[i]) sums.y += exp2_approx(st.y(given[i]));
  }
  sums = sum_block<1>(sums);
  float loss = sums.x;
  float outside = t.mass;  // what p outside of the entries is multiplied by: Q + q_r - q_r / p_r
  Outside rest = {-kInf, 0.f};
  if (t.rest > 0.f) {
    const float in = st.empty() ? 0.f : sums.y / st.s, out = st.empty() ? 0.f : 1.f - in;
    if (4.f * out < t.rest && !st.empty()) {  // the same for every thread
      rest = sum_outside(row, set, st);
      const float lpr = rest.m == -kInf ? -kInf : st.logprob(rest.m) + logf(rest.s);
      if (lpr >= -kLn2 * kFar) {
        loss += t.rest * (logf(t.rest) - lpr);
        outside = expf(lpr) * (t.mass + t.rest) - t.rest;  // of p / p_r
      } else {  // masked
        rest.m = -kInf;
        loss = kInf;
        outside = 0.f;
      }
    } else {
      const float more = out == 0.f ? kInf : (in - t.mass) / out;
      loss += t.rest * (fabsf(more) < 0.5f ? log1pf(more) : logf(t.rest / out));
      outside = isinf(more) ? 0.f : -more;  // infinite: every p outside is 0
    }
  }
  if (threadIdx.x != 0) return;
  if (t.bad) {
    loss = kNaN;
    report_status(p.status, FAKLA_ERR_INVALID_ARG);
  }
  p.loss[r] = loss;
  if (p.stats) {
    float* keep = p.stats + (int64_t)r * kDistillStats;
    keep[0] = st.m;
    keep[1] = st.l2s;
    keep[2] = t.m;
    keep[3] = t.logs;
    keep[4] = t.bad ? kNaN : t.mass + t.rest;
    keep[5] = t.bad ? kNaN : outside;
    keep[6] = t.twice;
    keep[7] = rest.m;  // -inf: p outside goes by the row's own maximum and sum
    if (rest.m != -kInf) keep[2] = log2f(rest.s) + stats_of(p, rest.m, 0.f).y(rest.m);  // (t.m is 0 with teacher_lse)
  }
}

// What a block's entries subtract from their p_j inner, kept by vector: one bit
// per vector says whether it has an entry (the 32 vectors of a warp share a word),
// and those that have take one of kMaxEntries cells each.
template <int E>
struct Cells {
  __align__(16) float q[kMaxEntries][E];
  uint32_t has[kMaxEntries];  // bit e: value e of the cell's vector is an entry
  uint32_t count;
  float single_q[2 * E];
  uint32_t single_has;
};

// The entries go out with the rest of their vectors. (Writing them once more
// behind the pass took 10 us more for 64 of them on 4096 x 32000 bf16 and 30
// us for 256: their lines had left the cache by then.)
template <typename T>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(LogitsArgs p, int chunks, int span) {
  constexpr int E = Row<T>::E;
  extern __shared__ uint32_t marks[];  // span / 32 words of bits, then each word's first cell
  __shared__ Cells<E> cells;
  __shared__ int id_of[kMaxEntries];
  __shared__ float q_of[kMaxEntries];
  uint8_t* base = reinterpret_cast<uint8_t*>(marks + span / 32);
  griddep_wait();
  const uint32_t r = blockIdx.x / chunks;
  const int chunk = blockIdx.x - r * chunks;
  const Row<T> row(p, r);
  const int v0 = min(chunk * span, row.vectors), v1 = min(v0 + span, row.vectors);
  T* out = (T*)p.dlogits + (int64_t)r * p.vocab;
  const float* keep = p.stats + (int64_t)r * kDistillStats;
  const Stats st = stats_of(p, keep[0], keep[1]);
  const bool apart = keep[7] != -kInf;  // p_r was summed on its own
  const Stats other = apart ? stats_of(p, keep[7], keep[2]) : st;
  const float teacher_m = apart ? 0.f : keep[2];
  const float g = p.dloss[r] * p.inv_temperature;
  // dlogits_j = p_j inner - its q for an entry; otherwise p_j outer or (apart)
  // p_j / p_r outer, in both cases 2^{y - log2 s} of `other`
  const float inner = keep[4] * g, outer = keep[5] * g;
  auto cell = [&](int v) { return base[v / 32] + __popc(marks[v / 32] & ((1u << v % 32) - 1)); };
  auto first = [&] {
    Entries entries;
    entries.read(p, r);
    const int words = (v1 - v0 + 31) / 32;
    for (int i = threadIdx.x; i < words; i += kThreads) marks[i] = 0;
    for (int i = threadIdx.x; i < kMaxEntries; i += kThreads) cells.has[i] = 0;
    if (threadIdx.x == 0) cells.count = cells.single_has = 0;
    const bool twice = keep[6] != 0.f;
    float q[kPerThread];
    int at[kPerThread];  // its vector in the span, -1 - its single, or none of both
    constexpr int kNone = INT32_MIN;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      float lq;
      const int j = entries.id[i];
      q[i] = teacher_q(p, j, entries.logit[i], teacher_m, keep[3], lq) * g;
      at[i] = kNone;
      if (j >= 0 && writes(row, j, chunk, v0, v1)) at[i] = row.place(j) < 0 ? row.place(j) : row.place(j) - v0;
      if (twice) {
        q_of[threadIdx.x + i * kThreads] = q[i];
        id_of[threadIdx.x + i * kThreads] = j;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      if (at[i] == kNone) continue;
      if (twice) {  // the first that names it, with the q of all that do, in their order
        const int j = entries.id[i], self = threadIdx.x + i * kThreads;
        int first = self;
        q[i] = 0.f;
        for (int k = 0; k < p.entries; ++k)
          if (id_of[k] == j) {
            first = min(first, k);
            q[i] += q_of[k];
          }
        if (first != self) {
          at[i] = kNone;
          continue;
        }
      }
      if (at[i] >= 0) {
        atomicOr(&marks[at[i] / 32], 1u << at[i] % 32);
      } else {
        atomicOr(&cells.single_has, 1u << (-1 - at[i]));
        cells.single_q[-1 - at[i]] = q[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < words; i += kThreads)
      if (const uint32_t word = marks[i]) base[i] = (uint8_t)atomicAdd(&cells.count, __popc(word));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (at[i] >= 0) {
        const int c = cell(at[i]), e = (entries.id[i] - row.lead) % E;
        cells.q[c][e] = q[i];
        atomicOr(&cells.has[c], 1u << e);
      }
    __syncthreads();
  };
  auto prob = [&](float x) { return exp2_approx(st.y(x) - st.l2s); };
  // given nothing, by the loss or by the teacher (Q + q_r is 0 in a row without
  // entries only), and rows of nothing but -inf
  const bool zero = g == 0.f || keep[4] == 0.f || (st.empty() && !isnan(inner));
  auto prob_out = [&](float x) { return exp2_approx(other.y(x) - other.l2s); };
  if (st.far || other.far) {
    if (!zero) first();
    for (int v = v0 + threadIdx.x; v < v1; v += kThreads)
      for (int e = 0; e < E; ++e) {
        const int j = row.lead + v * E + e;
        const float x = zero ? 0.f : to_f32(row.x[j]);
        const bool marked = !zero && marks[(v - v0) / 32] >> (v - v0) % 32 & 1;
        const int c = marked ? cell(v - v0) : 0;
        const bool given = marked && cells.has[c] >> e & 1;
        out[j] = from_f32<T>(zero ? 0.f : given ? prob(x) * inner - cells.q[c][e] : prob_out(x) * outer);
      }
  } else {
    const uint64_t c2 = sm100::f2_splat(st.c), nM = sm100::f2_splat(-other.M), nl = sm100::f2_splat(-other.l2s);
    const uint64_t o2 = sm100::f2_splat(outer);
    // (an entry's own place is patched, whatever 2^{y - log2 s} of `other` is there)
    map_vectors(row, out, v0, v1, zero, first, [&](const uint4& raw, int i) {
      const float2 f = sm100::f2_split(sm100::f2_add(sm100::f2_fma(Vec<T>::pair(raw, i), c2, nM), nl));
      return sm100::f2_mul(sm100::f2_make(__float_as_uint(exp2_approx(f.x)), __float_as_uint(exp2_approx(f.y))), o2);
    }, [&](uint4& got, const uint4& raw, int v) {
      if (marks[(v - v0) / 32] >> (v - v0) % 32 & 1) {
        const int c = cell(v - v0);
        const uint32_t has = cells.has[c];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float f = prob(to_f32(reinterpret_cast<const T*>(&raw)[e])) * inner - cells.q[c][e];
          if (has >> e & 1) reinterpret_cast<T*>(&got)[e] = from_f32<T>(f);
        }
      }
    });
  }
  if (chunk == 0 && threadIdx.x < row.singles) {
    const int j = row.single(threadIdx.x);
    const float x = zero ? 0.f : to_f32(row.x[j]);
    const bool given = !zero && cells.single_has >> threadIdx.x & 1;
    out[j] = from_f32<T>(zero ? 0.f : given ? prob(x) * inner - cells.single_q[threadIdx.x] : prob_out(x) * outer);
  }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
// Blocks of a cluster, which share a row: as many as give every SM kBlocks,
// while a thread keeps a vector or two, and as a block's shared memory asks for
// (`bytes` per vector). With 4, 2 and 6 blocks per SM 301 x 50257 fp32 with 32
// alternatives took 34, 34 and 41 us, 257 x 50257 bf16 distillation (forward and
// backward) 21, 22 and 21.
constexpr int kBlocks = 4;
constexpr int kClusterBytes = 48 << 10;
int cluster_size(int64_t rows, int64_t vectors, int bytes) {
  int c = 1;
  while (c < kMaxCluster && ((rows * c < kBlocks * fakla_sm_count() && vectors / (2 * c) >= kThreads) ||
                             vectors / c * bytes > kClusterBytes))
    c *= 2;
  return c;
}

template <typename K>
cudaError_t launch_rows(K kernel, const LogitsArgs& p, int per_vector, int bytes, cudaStream_t stream) {
  const int64_t vectors = p.vocab / per_vector;
  const int c = cluster_size(p.batch * p.rows, vectors, bytes);
  const size_t smem = ((size_t)((vectors + c - 1) / c + 1) * bytes + 15) / 16 * 16;
  if (smem > (32 << 10)) {
    // The limit belongs to the kernel, which other threads launch at the same
    // time: it is the most that any call asks for, never this call's size.
    const int most = std::max(kMaxVocab / per_vector / kMaxCluster * bytes, kClusterBytes) + 64;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
  }
  return launch_chained(kernel, dim3((unsigned)(p.batch * p.rows * c)), dim3(kThreads), smem, stream, (unsigned)c, p, c);
}

// A row's gradient is split into spans of whole rounds of loads, as long as
// every SM still gets kBlocks blocks. `marks`: 5 bytes of shared memory per 32
// vectors (a span is at most 2^20 / 4 vectors: 40 KB, and 8 KB beside them).
template <typename K>
cudaError_t launch_spans(K kernel, const LogitsArgs& p, int per_vector, bool marks, cudaStream_t stream) {
  const int64_t rows = p.batch * p.rows, rounds = (p.vocab / per_vector + kRound - 1) / kRound;
  int64_t chunks = (kBlocks * fakla_sm_count() + rows - 1) / rows;
  if (chunks > rounds) chunks = rounds;
  if (chunks < 1) chunks = 1;
  const int span = (int)((rounds + chunks - 1) / chunks) * kRound;
  return launch_chained(kernel, dim3((unsigned)(rows * chunks)), dim3(kThreads),
                        marks ? (size_t)span / 32 * 5 : 0, stream, 1u, p, (int)chunks, span);
}

template <typename F>
cudaError_t by_type(int dtype, F f) {
  return dtype == FAKLA_BF16 ? f(__nv_bfloat16{}) : f(float{});
}

}  // namespace

cudaError_t launch_token_logprobs(int dtype, const LogitsArgs& p, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (p.top_k > 0) return launch_rows(token_logprobs_kernel<T, true>, p, Vec<T>::E, (int)sizeof(T), stream);
    return launch_rows(token_logprobs_kernel<T, false>, p, Vec<T>::E, 0, stream);
  });
}

cudaError_t launch_token_logprobs_backward(int dtype, const LogitsArgs& p, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) {
    return launch_spans(token_logprobs_backward_kernel<decltype(t)>, p, Vec<decltype(t)>::E, false, stream);
  });
}

cudaError_t launch_distill(int dtype, const LogitsArgs& p, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    return launch_rows(distill_kernel<T>, p, Vec<T>::E, 0, stream);
  });
}

cudaError_t launch_distill_backward(int dtype, const LogitsArgs& p, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) {
    return launch_spans(distill_backward_kernel<decltype(t)>, p, Vec<decltype(t)>::E, true, stream);
  });
}

}  // namespace fakla
