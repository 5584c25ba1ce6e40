// Log probabilities of given tokens, entropy and most probable tokens of rows
// of logits (HBM-bound: every logit is read once).
//
// With m = max x, t = x - m, S = sum e^t and D = sum t e^t over a row:
//   log p(i) = t_i - log S
//   entropy  = -sum p log p = log S - D / S   (two terms of one sign)
// Each thread keeps m, S and D of its own logits and rescales them when m
// grows (D of m' = m + d: e^-d (D - d S)); threads, warps and CTAs are joined
// the same way, in a fixed order.
//
// A row is split over the CTAs of a cluster, which join in the first CTA's
// shared memory: no scratch in device memory, one launch.
//
// The `top` most probable tokens need no second pass over the row. The k-th
// largest of the threads' maxima is a lower bound of the k-th largest logit,
// and only the k threads at or above it hold logits that can be among the
// first k: the warps read these threads' logits again (L2) and merge what is
// above the bound into sorted lists of 32. Order: by logit, then the lowest
// index; NaN ranks as -inf.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstdint>
#include "dtype.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace b200 {

namespace {

constexpr float kLowest = -3.402823466e38f;
constexpr unsigned kFull = 0xffffffffu;

struct Soft {
  float m, s, d;  // max, sum e^(x-m), sum (x-m) e^(x-m)
};

// a's sums with the maximum m >= a.m. The difference is cut at -200, where
// e^d is 0 in f32, so that infinite differences give 0 and not NaN.
__device__ __forceinline__ void rescale(Soft& a, float m) {
  const float d = fmaxf(fmaxf(a.m, kLowest) - fmaxf(m, kLowest), -200.0f);
  const float f = __expf(d);
  a.d = f * fmaf(d, a.s, a.d);
  a.s *= f;
  a.m = m;
}

__device__ __forceinline__ Soft join(Soft a, Soft b) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m);
  rescale(b, m);
  return {m, a.s + b.s, a.d + b.d};
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

template <class T>
__device__ __forceinline__ void add_chunk(Soft& a, uint32_t& best, uint32_t j, const float* x) {
  constexpr int VEC = Chunk<T>::kElems;
  float cm = x[0];
#pragma unroll
  for (int i = 1; i < VEC; ++i) cm = fmaxf(cm, x[i]);
  if (cm > a.m) {
    rescale(a, cm);
    best = j;
  }
  const float m = fmaxf(a.m, kLowest);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float t = x[i] - m;
    const float e = __expf(t);
    a.s += e;
    a.d = fmaf(e, fmaxf(t, -200.0f), a.d);  // e^-200 is 0: -inf adds 0
  }
}

// Chunk j of a row: its elements [j * VEC - shift, + VEC), which start on 16
// bytes; the row's first and last chunk may be cut.
template <class T>
__global__ void __launch_bounds__(512)
    token_logprobs_kernel(const __grid_constant__ TokenLogprobsArgs p) {
  constexpr int VEC = Chunk<T>::kElems, NT = 512, NW = NT / 32, U = 4;
  __shared__ Soft sh_soft[NW];
  __shared__ uint64_t sh_keys[NW][32];
  __shared__ int sh_flagged[kMaxTop];
  __shared__ int sh_count;
  __shared__ uint64_t sh_bound;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int64_t row = blockIdx.x / C;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const uint32_t V = (uint32_t)p.V;
  const uint32_t shift = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const T* base = x - shift;  // read from its first full chunk on
  const uint32_t chunks = (V + shift + VEC - 1) / VEC;
  const uint32_t j0 = (uint32_t)((uint64_t)chunks * rank / C);
  const uint32_t j1 = (uint32_t)((uint64_t)chunks * (rank + 1) / C);
  const bool cut_last = (V + shift) % VEC != 0;

  auto cut_chunk = [&](uint32_t j, float* f) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const uint32_t n = j * VEC + i;
      f[i] = n >= shift && n < V + shift ? to_f32(base[n]) : __int_as_float(0xff800000);
    }
  };

  // ---- one pass: this thread's chunks j0 + tid, + NT, ...
  Soft a = {__int_as_float(0xff800000), 0.0f, 0.0f};
  uint32_t j = j0 + tid, best = j;
  if (tid == 0 && j == 0 && j < j1 && shift) {
    float f[VEC];
    cut_chunk(0, f);
    add_chunk<T>(a, best, 0, f);
    j += NT;
  }
  const uint32_t full = j1 == chunks && cut_last ? j1 - 1 : j1;  // full chunks end here
  const uint4* v = reinterpret_cast<const uint4*>(base);
  if (full > 0)
    for (; j + (U - 1) * NT < full; j += U * NT) {
      uint4 c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) c[u] = __ldg(v + j + u * NT);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[VEC];
        unpack(c[u], (const T*)nullptr, f);
        add_chunk<T>(a, best, j + u * NT, f);
      }
    }
  for (; j < full; j += NT) {
    float f[VEC];
    unpack(__ldg(v + j), (const T*)nullptr, f);
    add_chunk<T>(a, best, j, f);
  }
  if (j < j1) {
    float f[VEC];
    cut_chunk(j, f);
    add_chunk<T>(a, best, j, f);
  }
  const bool any = j0 + tid < j1;

  // ---- the CTA's sums, in warp 0's lane 0
  Soft w = a;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Soft b = {__shfl_down_sync(kFull, w.m, o), __shfl_down_sync(kFull, w.s, o),
                    __shfl_down_sync(kFull, w.d, o)};
    w = join(w, b);
  }
  if (lane == 0) sh_soft[wid] = w;
  if (tid == 0) sh_count = 0;

  // ---- the CTA's first `top` keys, in warp 0
  uint64_t keys = 0;
  if (p.top > 0) {
    const uint64_t mine = any ? key_of(a.m, best) : 0;
    uint64_t b = cta_merge<NW>(warp_sort(mine), sh_keys);
    if (wid == 0) {
      const uint64_t bound = __shfl_sync(kFull, b, p.top - 1);
      if (lane == 0) sh_bound = bound;
    }
    __syncthreads();
    const uint64_t bound = sh_bound;  // 0: fewer threads than `top` have logits
    if (any && mine >= bound) sh_flagged[atomicAdd(&sh_count, 1)] = tid;
    __syncthreads();
    const int count = sh_count;
    const uint32_t bound_x = (uint32_t)(bound >> 32), bound_j = ~(uint32_t)bound;
    for (int f = wid; f < count; f += NW) {
      const uint32_t t = (uint32_t)sh_flagged[f];
      // lane's element of the thread's chunks: VEC lanes a chunk
      for (uint32_t jb = j0 + t; jb < j1; jb += 32 / VEC * NT) {
        const uint64_t jj = (uint64_t)jb + (uint64_t)(lane / VEC) * NT;
        const uint32_t n = (uint32_t)jj * VEC + lane % VEC;
        uint64_t key = 0;
        if (jj < j1 && n >= shift && n < V + shift) {
          const float e = to_f32(base[n]);
          const uint32_t o = ordered(e);
          if (o > bound_x || (o == bound_x && jj <= bound_j)) key = key_of(e, n - shift);
        }
        const uint64_t last = __shfl_sync(kFull, keys, p.top - 1);
        if (__any_sync(kFull, key > last)) keys = warp_merge(keys, warp_sort(key));
      }
    }
    __syncthreads();  // cta_merge above is done with sh_keys
    keys = cta_merge<NW>(keys, sh_keys);
  }
  __syncthreads();
  if (wid == 0) {
    w = lane < NW ? sh_soft[lane] : Soft{__int_as_float(0xff800000), 0.0f, 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Soft b = {__shfl_down_sync(kFull, w.m, o), __shfl_down_sync(kFull, w.s, o),
                      __shfl_down_sync(kFull, w.d, o)};
      w = join(w, b);
    }
  }

  // ---- the row's, in the first CTA's warp 0
  if (C > 1) {
    if (wid == 0) {
      sh_keys[0][lane] = keys;
      if (lane == 0) sh_soft[0] = w;
    }
    cluster.sync();
    if (rank == 0 && wid == 0)
      for (int r = 1; r < C; ++r) {
        w = join(w, *cluster.map_shared_rank(&sh_soft[0], r));
        if (p.top > 0) keys = warp_merge(keys, cluster.map_shared_rank(&sh_keys[0][0], r)[lane]);
      }
    cluster.sync();  // the other CTAs' shared memory has been read
  }
  if (rank != 0 || wid != 0) return;
  w.m = __shfl_sync(kFull, w.m, 0);
  w.s = __shfl_sync(kFull, w.s, 0);
  w.d = __shfl_sync(kFull, w.d, 0);
  // a row whose logits are all -inf has s = 0 and no distribution
  const float minus_inf = __int_as_float(0xff800000);
  const float log_s = logf(w.s);
  auto log_p = [&](float e) { return w.s == 0.0f ? minus_inf : (e - fmaxf(w.m, kLowest)) - log_s; };
  if (lane == 0) {
    if (p.entropy) {
      const float h = log_s - w.d / w.s;
      p.entropy[row] = w.s == 0.0f || h < 0.0f ? 0.0f : h;
    }
    if (p.tokens) {
      const int32_t t = p.tokens[row];
      float lp = 0.0f;
      if (t >= 0) lp = (uint32_t)t < V ? log_p(to_f32(x[t])) : __int_as_float(0x7fc00000);
      p.logprobs[row] = lp;
    }
  }
  if (lane < p.top) {
    p.top_logprobs[row * p.top + lane] = log_p(unordered((uint32_t)(keys >> 32)));
    p.top_tokens[row * p.top + lane] = (int32_t)~(uint32_t)keys;
  }
}

template <class T>
int run(const TokenLogprobsArgs& p, cudaStream_t st) {
  // One CTA a row where the rows fill the GPU; otherwise the row is split, as
  // long as every thread keeps two chunks.
  const int64_t chunks = (p.V + Chunk<T>::kElems - 1) / Chunk<T>::kElems;
  int C = 1;
  while (C < 8 && p.T * C < 148 * 4 && chunks >= (int64_t)C * 2 * 512 * 2) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.T * C));
  cfg.blockDim = dim3(512);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, p);
  count_launch();
  return launch_result(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace

int token_logprobs(const TokenLogprobsArgs& p, int dtype, cudaStream_t st) {
  if (dtype == kF32) return run<float>(p, st);
  if (dtype == kBF16) return run<bf16>(p, st);
  return run<f16>(p, st);
}

}  // namespace b200
