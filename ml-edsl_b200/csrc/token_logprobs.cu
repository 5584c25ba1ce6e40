// Log probabilities of given tokens, entropy and most probable tokens of rows
// of logits (HBM-bound: every logit is read once).
//
// In powers of two, L = log2 e, with a shift c near m L for the row's maximum m:
//   t = x L - c (one fma),  S = sum 2^t,  D = sum t 2^t
//   log p(i) = x_i - m + (m L - c) ln 2 - ln 2 log2 S
//   entropy  = ln 2 (log2 S - D / S)   (two terms of one sign)
// The shift is m L rounded to f32: what the rounding leaves is the bracket
// above, so that t is as exact for logits near 1e4 as near 0. Each thread
// keeps m, S and D of its own logits and rescales them when m grows (for
// m' > m, d = c - c': S' = 2^d S, D' = 2^d (D + d S)); threads, warps and CTAs
// are joined the same way, in a fixed order. Five instructions and one
// exponential a logit: of bf16 logits an SM has 11.6 a clock to take at the
// measured bandwidth, of exponentials it has 16.
//
// A row is split over the CTAs of a cluster, which send what they have to the
// first one's shared memory: no scratch in device memory, one launch.
//
// The `top` most probable tokens need no second pass over the row. The k-th
// largest of 32 groups' maxima (a group: the threads of one lane number) is a
// lower bound of the k-th largest logit, and only threads whose own maximum
// reaches it hold logits that can be among the first k: their warps read these
// threads' logits again (L2), and each of the few that reach the bound finds
// its place by counting the larger ones. Order: by logit, then the lowest
// index; NaN ranks as -inf.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstdint>
#include "dtype.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace b200 {

namespace {

constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2E = 1.44269504f, kLn2 = 0.693147181f;
// Maxima beyond this make x L leave f32: t is then (x - m) L, two roundings.
constexpr float kWide = 1e38f;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float minus_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float nan_f32() { return __int_as_float(0x7fc00000); }
// 2^t for t <= 0 or so; 0 below -126.
__device__ __forceinline__ float exp2_fast(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}

// The shift c of a maximum m. Rounded by itself wherever it is used: a product
// contracted into an fma would be another number.
__device__ __forceinline__ float shift_of(float m) { return __fmul_rn(m, kLog2E); }

struct Soft {
  float m, s, d;  // max, sum 2^t, sum t 2^t
};

// c - c' of two maxima m <= m', at least -200, where 2^d is 0.
__device__ __forceinline__ float shift_between(float m, float to) {
  m = fmaxf(m, kLowest);
  to = fmaxf(to, kLowest);
  const bool wide = fabsf(m) > kWide || fabsf(to) > kWide;
  return fmaxf(wide ? (m - to) * kLog2E : __fsub_rn(shift_of(m), shift_of(to)), -200.0f);
}

// a's sums with the maximum m >= a.m.
__device__ __forceinline__ void rescale(Soft& a, float m) {
  const float d = shift_between(a.m, m), f = exp2_fast(d);
  a.d = f * fmaf(d, a.s, a.d);
  a.s *= f;
  a.m = m;
}

// The sums of a warp's lanes, in every lane.
__device__ __forceinline__ Soft warp_join(Soft a) {
  float m = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  rescale(a, m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(kFull, a.s, o);
    a.d += __shfl_xor_sync(kFull, a.d, o);
  }
  return a;
}

// The order of floats as that of unsigned integers; NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) x = __int_as_float(0xff800000);
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float((o >> 31) ? o ^ 0x80000000u : ~o);
}
// Larger is better: the larger logit, then the lower index. 0 is no entry.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  return (uint64_t)ordered(x) << 32 | (uint32_t)~index;
}

__device__ __forceinline__ uint64_t xor_max(uint64_t v, int o, bool take_max) {
  const uint64_t w = __shfl_xor_sync(kFull, v, o);
  return (v > w) == take_max ? v : w;
}
// The 32 keys of a warp in descending order of lanes.
__device__ __forceinline__ uint64_t warp_sort(uint64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o > 0; o /= 2)
      v = xor_max(v, o, ((lane & size) == 0) == ((lane & o) == 0));
  return v;
}
// The first 32 of two descending lists (lane i holds the i-th of each).
__device__ __forceinline__ uint64_t warp_merge(uint64_t a, uint64_t b) {
  const int lane = threadIdx.x & 31;
  const uint64_t r = __shfl_sync(kFull, b, 31 - lane);
  uint64_t v = a > r ? a : r;  // bitonic, and holds the largest 32
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v = xor_max(v, o, (lane & o) == 0);
  return v;
}

// The first 32 of the CTA's lists, one in each warp, in warp 0.
template <int NW>
__device__ __forceinline__ uint64_t cta_merge(uint64_t v, uint64_t (*sh)[32]) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int half = NW / 2; half > 0; half /= 2) {
    if (wid >= half && wid < 2 * half) sh[wid][lane] = v;
    __syncthreads();
    if (wid < half) v = warp_merge(v, sh[wid + half][lane]);
  }
  return v;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// VEC logits into a thread's sums.
template <int VEC>
__device__ __forceinline__ void add_chunk(Soft& a, const float* x) {
  float cm = x[0];
#pragma unroll
  for (int i = 1; i < VEC; ++i) cm = max_nan(cm, x[i]);
  if (!(cm <= a.m)) {  // a new maximum, or NaN
    float m = a.m;
#pragma unroll
    for (int i = 0; i < VEC; ++i) m = fmaxf(m, x[i]);
    if (m > a.m) rescale(a, m);
    if (cm != cm || cm == __int_as_float(0x7f800000)) a.s = nan_f32();  // no distribution
  }
  const float m = fmaxf(a.m, kLowest);
  float t[VEC];
  if (fabsf(m) <= kWide) {
    const float c = shift_of(m);
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = fmaf(x[i], kLog2E, -c);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = (x[i] - m) * kLog2E;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    t[i] = fmaxf(t[i], -200.0f);  // 2^-200 is 0: -inf adds 0
    const float e = exp2_fast(t[i]);
    a.s += e;
    a.d = fmaf(e, t[i], a.d);
  }
}

constexpr uint32_t kNoChunk = 0xffffffffu;
constexpr int kMaxCandidates = 256;
constexpr int kMaxCluster = 8;

// Chunk j of a row: its elements [j * VEC - cut, + VEC), which start on 16
// bytes; the row's first and last chunk may be cut.
template <class T, int NT>
__global__ void __launch_bounds__(NT)
    token_logprobs_kernel(const __grid_constant__ TokenLogprobsArgs p, int log_c) {
  constexpr int VEC = Chunk<T>::kElems, NW = NT / 32, U = 4;
  __shared__ Soft sh_soft[NW];
  __shared__ uint32_t sh_max[NT];
  __shared__ uint8_t sh_lanes[NW][32];
  __shared__ uint64_t sh_keys[NW][32];
  __shared__ uint64_t sh_candidates[kMaxCandidates];
  __shared__ int sh_found;
  // what the cluster's CTAs send to the first one
  __shared__ Soft sh_row[kMaxCluster];
  __shared__ uint64_t sh_row_keys[kMaxCluster * kMaxTop];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = 1 << log_c, rank = blockIdx.x & (C - 1);
  if (C > 1) cluster.barrier_arrive();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int64_t row = blockIdx.x >> log_c;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const uint32_t V = (uint32_t)p.V;
  const uint32_t cut = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const T* base = x - cut;  // read from its first whole chunk on
  const uint32_t chunks = (V + cut + VEC - 1) / VEC;
  const uint32_t j0 = (uint32_t)((uint64_t)chunks * rank >> log_c);
  const uint32_t j1 = (uint32_t)((uint64_t)chunks * (rank + 1) >> log_c);
  const bool cut_last = (V + cut) % VEC != 0;
  pdl_trigger();
  pdl_wait();

  // ---- one pass. The cut chunks at the row's ends belong to threads 0 and 32
  // of the first and the last CTA; the whole ones go round: w0 + tid, + NT, ...
  const uint32_t w0 = j0 == 0 && cut ? 1 : j0, w1 = j1 == chunks && cut_last ? j1 - 1 : j1;
  uint32_t edge = kNoChunk;
  if (tid == 0 && w0 != j0) edge = 0;
  if (tid == 32 && j1 > w0 && w1 != j1) edge = j1 - 1;
  float at_edge[VEC];
  if (edge != kNoChunk) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const uint32_t n = edge * VEC + i;
      at_edge[i] = n >= cut && n < V + cut ? to_f32(base[n]) : minus_inf();
    }
  }
  // the given token's logit, for the end
  int32_t token = -1;
  float given = 0.0f;
  if (rank == 0 && tid == NT - 1 && p.tokens) {
    token = p.tokens[row];
    if (token >= 0 && (uint32_t)token < V) given = to_f32(x[token]);
  }
  Soft a = {minus_inf(), 0.0f, 0.0f};
  uint32_t j = w0 + tid;
  const bool any = j < w1 || edge != kNoChunk;
  const uint4* v = reinterpret_cast<const uint4*>(base);
  // four chunks on their way while four are added
  uint4 c[U];
  bool have = j + (U - 1) * NT < w1;
  if (have) {
#pragma unroll
    for (int u = 0; u < U; ++u) c[u] = __ldg(v + j + u * NT);
  }
  while (have) {
    uint4 next[U];
    const uint32_t jn = j + U * NT;
    have = jn + (U - 1) * NT < w1;
    if (have) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = __ldg(v + jn + u * NT);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[VEC];
      unpack(c[u], (const T*)nullptr, f);
      add_chunk<VEC>(a, f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) c[u] = next[u];
    j = jn;
  }
  {  // the last ones, fewer than U
    uint4 r[U - 1];
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (j + u * NT < w1) r[u] = __ldg(v + j + u * NT);
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (j + u * NT < w1) {
        float f[VEC];
        unpack(r[u], (const T*)nullptr, f);
        add_chunk<VEC>(a, f);
      }
  }
  if (edge != kNoChunk) add_chunk<VEC>(a, at_edge);

  // ---- the warps' sums
  const uint32_t mine = any ? ordered(a.m) : 0;
  const Soft w = warp_join(a);
  if (lane == 0) sh_soft[wid] = w;
  sh_max[tid] = mine;
  if (tid == 0) sh_found = 0;
  __syncthreads();

  // ---- the CTA's candidates for the first `top`
  if (p.top > 0) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) most = max(most, sh_max[i * 32 + lane]);
    int place = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint32_t o = __shfl_sync(kFull, most, i);
      place += o > most || (o == most && i < lane);
    }
    const unsigned at = __ballot_sync(kFull, place == p.top - 1);
    // 0: fewer than `top` groups have logits, and all of them pass
    const uint32_t bound = __shfl_sync(kFull, most, __ffs(at) - 1);
    const float least = unordered(bound);
    const bool flagged = any && mine >= bound;
    const unsigned mask = __ballot_sync(kFull, flagged);
    if (flagged) sh_lanes[wid][__popc(mask & ((1u << lane) - 1))] = (uint8_t)lane;
    __syncwarp();
    const uint32_t per = (w1 - w0 + NT - 1) / NT;  // whole chunks of a thread, at most
    const uint32_t work = (w1 > w0 ? per : 0) * __popc(mask);
    const bool first_edge = wid == 0 && (mask & 1) && w0 != j0;
    const bool last_edge = wid == 1 && (mask & 1) && j1 > w0 && w1 != j1;
    // this lane's chunk number q of the warp's flagged threads
    auto load = [&](uint32_t q, float (&f)[VEC]) -> uint32_t {
      const uint32_t l = sh_lanes[wid][q / per];
      const uint64_t jj = (uint64_t)w0 + wid * 32 + l + (uint64_t)(q % per) * NT;
      if (jj >= w1) return kNoChunk;
      unpack(__ldg(v + jj), (const T*)nullptr, f);
      return (uint32_t)jj;
    };
    auto load_edge = [&](uint32_t n, float& f) {
      const bool is = lane < VEC && n >= cut && n < V + cut;
      if (is) f = to_f32(base[n]);
      return is;
    };
    auto offer = [&](float f, uint32_t n) {
      const int slot = atomicAdd(&sh_found, 1);
      if (slot < kMaxCandidates) sh_candidates[slot] = key_of(f, n - cut);
    };
    for (uint32_t q = lane; q < work; q += 32) {
      float f[VEC];
      const uint32_t jj = load(q, f);
      if (jj == kNoChunk) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (!(f[i] < least)) offer(f[i], jj * VEC + i);
    }
    float f1 = 0.0f;
    if (first_edge && load_edge(lane, f1) && !(f1 < least)) offer(f1, lane);
    if (last_edge && load_edge(w1 * VEC + lane, f1) && !(f1 < least)) offer(f1, w1 * VEC + lane);
    __syncthreads();
    if (sh_found > kMaxCandidates) {  // many alike: sorted as they are read
      uint64_t keys = 0;
      auto insert = [&](uint64_t key) {
        const uint64_t last = __shfl_sync(kFull, keys, p.top - 1);
        if (__any_sync(kFull, key > last)) keys = warp_merge(keys, warp_sort(key));
      };
      for (uint32_t q0 = 0; q0 < work; q0 += 32) {
        float f[VEC];
        const uint32_t jj = q0 + lane < work ? load(q0 + lane, f) : kNoChunk;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          insert(jj != kNoChunk ? key_of(f[i], jj * VEC + i - cut) : 0);
      }
      if (first_edge) insert(load_edge(lane, f1) ? key_of(f1, lane - cut) : 0);
      if (last_edge)
        insert(load_edge(w1 * VEC + lane, f1) ? key_of(f1, w1 * VEC + lane - cut) : 0);
      keys = cta_merge<NW>(keys, sh_keys);
      if (wid == 0) sh_candidates[lane] = keys;
      if (tid == 0) sh_found = 32;
      __syncthreads();
    }
  }

  // ---- the row's sums, in the first CTA
  if (C > 1) cluster.barrier_wait();  // every CTA of the cluster runs
  if (wid == 0) {
    const Soft r = warp_join(lane < NW ? sh_soft[lane] : Soft{minus_inf(), 0.0f, 0.0f});
    if (lane == 0) *(C > 1 ? cluster.map_shared_rank(&sh_row[rank], 0) : &sh_row[0]) = r;
  }
  // a candidate's place, by the number of larger ones
  uint64_t key = 0;
  int place = 0;
  const int found = p.top > 0 ? sh_found : 0;
  if (tid < found) {
    key = sh_candidates[tid];
#pragma unroll 8
    for (int i = 0; i < found; ++i) place += sh_candidates[i] > key;
  }
  if (C > 1) {
    if (p.top > 0) {
      uint64_t* to = cluster.map_shared_rank(&sh_row_keys[rank * p.top], 0);
      if (key && place < p.top) to[place] = key;
      if (tid < p.top && tid >= found) to[tid] = 0;
    }
    cluster.sync();
    if (rank != 0) return;
    // the CTAs' lists are in order: the place by a search in each
    key = tid < p.top << log_c ? sh_row_keys[tid] : 0;
    place = 0;
    if (key) {
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        if (c >= C) break;
        const uint64_t* list = sh_row_keys + c * p.top;
        int n = 0;  // of the list's that are larger
#pragma unroll
        for (int step = kMaxTop; step > 0; step /= 2)
          if (n + step <= p.top && list[n + step - 1] > key) n += step;
        place += n;
      }
    }
  } else {
    __syncthreads();
  }
  Soft r = sh_row[0];
  if (C > 1) r = warp_join(lane < C ? sh_row[lane] : Soft{minus_inf(), 0.0f, 0.0f});
  // a row whose logits are all -inf has s = 0 and no distribution
  const float m = fmaxf(r.m, kLowest);
  const float rest = fabsf(m) <= kWide ? fmaf(m, kLog2E, -shift_of(m)) : 0.0f;
  const float log2_s = log2f(r.s);
  auto log_p = [&](float e) {
    return r.s == 0.0f ? minus_inf() : (e - m) - kLn2 * (log2_s - rest);
  };
  if (tid == NT - 1) {
    if (p.entropy) {
      const float h = kLn2 * (log2_s - r.d / r.s);
      p.entropy[row] = r.s == 0.0f || h < 0.0f ? 0.0f : h;
    }
    if (p.tokens) {
      float lp = 0.0f;
      if (token >= 0) lp = (uint32_t)token < V ? log_p(given) : nan_f32();
      p.logprobs[row] = lp;
    }
  }
  if (key && place < p.top) {
    p.top_logprobs[row * p.top + place] = log_p(unordered((uint32_t)(key >> 32)));
    p.top_tokens[row * p.top + place] = (int32_t)~(uint32_t)key;
  }
}

template <class T, int NT>
int launch(const TokenLogprobsArgs& p, int log_c, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.T << log_c));
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1u << log_c;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, NT>, p, log_c);
  count_launch();
  return launch_result(e != cudaSuccess ? e : cudaGetLastError());
}

template <class T>
int run(const TokenLogprobsArgs& p, cudaStream_t st) {
  // One CTA a row where the rows fill the GPU or are short (64x8192 bf16 4.4 us,
  // 5.9 split in two); otherwise the row is split, as long as every thread keeps
  // two chunks (1x131072 bf16 6.2 us, one CTA 15.6; 256x131072: 24.7 and 32.0).
  const int64_t chunks = (p.V + Chunk<T>::kElems - 1) / Chunk<T>::kElems;
  int l = 0;
  while (l < 3 && chunks > 2048 && (p.T << l) < 148 * 2 && chunks >= (int64_t)1024 << l) ++l;
  return launch<T, 256>(p, l, st);
}

}  // namespace

int token_logprobs(const TokenLogprobsArgs& p, int dtype, cudaStream_t st) {
  if (dtype == kF32) return run<float>(p, st);
  if (dtype == kBF16) return run<bf16>(p, st);
  return run<f16>(p, st);
}

}  // namespace b200
