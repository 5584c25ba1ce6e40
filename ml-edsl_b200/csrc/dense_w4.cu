// Dense layer of few rows with 4-bit weights:
//
//   Y[m,n] = act( sum_k x[m,k] * s[k/G, n] * (q[k,n] - z[k/G, n]) + b[n] )
//
// q: codes 0..15; s: a scale for each group of G rows of W and each column;
// z: a zero 0..15 (8 without zeros). For single tokens the weights are the
// whole cost: K * N / 2 bytes are read once, so the kernel is built to be
// bound by HBM.
//
// Arithmetic. q - z is a whole number of at most 15, exact in bf16 and f16,
// so the products are taken by mma.sync m16n8k16 with the weights as the
// 16-row operand (16 columns of W) and the rows of X as its 8 columns:
// x of bf16 as it is; f16 and e4m3 as f16 (exact); f32 as the sum of three
// bf16 parts of 8 bits each (exact down to bf16's smallest value, 2^-133), in three
// columns that are added at the end. bf16 weights are (q - z) / 4096 until the end,
// so that no sum before the scale leaves f32's range; what that costs lies below
// 2^-137. No product is rounded; sums run in f32, in the tensor core within a
// group (or a 64-long part of one), then with ordinary adds after the scale
// is applied in f32. For up to 8 operand columns the codes go from HBM to
// registers and into the product within one warp; more columns are
// dense_w4_tc.cu's, where tcgen05 takes 16 to 128 of them at the price of
// handing the expanded weights from one warp to another.
//
// Layout (w4_pack): strips of 64 columns; in a strip, blocks of 64 of K; in a
// block, four 512-byte pieces of 16 columns, 16 bytes for each lane: the
// codes of its fragments of four k16 steps, in an order that takes one shift
// and one and-or for two weights. Scales and zeros lie in the order in which
// the lanes read them.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstdint>
#include "w4.cuh"

namespace cg = cooperative_groups;

namespace b200 {

cudaError_t allow_shared(const void* kernel, std::atomic<uint64_t>& allowed, int* device) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (device) *device = dev;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (allowed.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared);
  if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

Capacity capacity_of(const void* kernel, int threads, int smem) {
  Capacity c;
  for (int l = 0; l < 4; ++l) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(8u * 148);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1u << l;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const int clusters = ask_or(
        l == 0 ? 148 : 0,
        [&](int* n) { return cudaOccupancyMaxActiveClusters(n, kernel, &cfg) == cudaSuccess; },
        [] { cudaGetLastError(); });
    c.ctas[l] = (int64_t)clusters << l;
  }
  return c;
}

int choose_cluster(const Capacity& capacity, int64_t tiles, int64_t kblocks, int warps, int fixed) {
  int best = 0;
  int64_t least = INT64_MAX;
  for (int l = 0; l <= 3; ++l) {
    if (capacity.ctas[l] == 0) continue;
    const int64_t waves = ((tiles << l) + capacity.ctas[l] - 1) / capacity.ctas[l];
    const int64_t blocks = (kblocks + ((int64_t)warps << l) - 1) / ((int64_t)warps << l);
    const int64_t cost = waves * (blocks + fixed);
    if (cost < least) {
      least = cost;
      best = l;
    }
  }
  return best;
}

namespace {

// ------------------------------------------------------------------ packing

// Row of W (k) of nibble `nib` of word `j` of lane `lane`'s 16 bytes, within
// its block, and its column within the 16 columns of the piece.
__host__ __device__ __forceinline__ void code_place(int lane, int j, int nib, int* k, int* n) {
  const int g = lane >> 2, t = lane & 3, r = nib & 3;
  *k = j * 16 + t * 2 + (r >> 1) * 8 + (nib >> 2);
  *n = g + (r & 1) * 8;
}

__global__ void w4_pack_codes_kernel(const uint8_t* __restrict__ codes, int64_t ldc, int64_t K,
                                     int64_t N, int64_t kblocks, int64_t total,
                                     uint32_t* __restrict__ out) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int j = (int)(i & 3), lane = (int)(i >> 2 & 31), mt = (int)(i >> 7 & 3);
    const int64_t block = i >> 9, kb = block % kblocks, strip = block / kblocks;
    uint32_t w = 0;
#pragma unroll
    for (int nib = 0; nib < 8; ++nib) {
      int k, n;
      code_place(lane, j, nib, &k, &n);
      const int64_t gk = kb * kBlockK + k, gn = strip * kStripN + mt * 16 + n;
      const uint32_t c = gk < K && gn < N ? codes[gk * ldc + gn] & 15u : 8u;
      w |= c << (4 * nib);
    }
    out[i] = w;
  }
}

__global__ void w4_pack_columns_kernel(const void* __restrict__ in, int64_t ldi, int64_t groups,
                                       int64_t N, int64_t strips, int bytes,
                                       void* __restrict__ out) {
  const int64_t total = strips * groups * 64;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int n = (int)(i & 63);
    const int64_t g = (i >> 6) % groups, strip = (i >> 6) / groups;
    const int64_t gn = strip * 64 + n, from = g * ldi + gn, to = (i & ~int64_t(63)) + column_place(n);
    if (bytes == 4)
      static_cast<uint32_t*>(out)[to] = gn < N ? static_cast<const uint32_t*>(in)[from] : 0u;
    else if (bytes == 2)
      static_cast<uint16_t*>(out)[to] = gn < N ? static_cast<const uint16_t*>(in)[from] : 0;
    else
      static_cast<uint8_t*>(out)[to] = gn < N ? static_cast<const uint8_t*>(in)[from] & 15 : 8;
  }
}

// Codes and scales of W: s = max|w| / 7 over a group of one column, rounded
// to the scales' type; q = round(w / s) + 8 with ties to even. A group that holds
// an infinity or NaN has a NaN for a scale, so that it shows in every product. A
// thread has one column of one group.
__global__ void w4_quantize_kernel(const float* __restrict__ W, int64_t ldw, int64_t K, int64_t N,
                                   int group, int64_t groups, uint8_t* __restrict__ codes,
                                   int64_t ldc, void* __restrict__ scales, int64_t lds,
                                   int s_dtype) {
  const int64_t total = groups * N;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t g = i / N, n = i - g * N;
    const int64_t k0 = g * group, k1 = min(K, k0 + group);
    float most = 0.0f;
    bool finite = true;
    for (int64_t k = k0; k < k1; ++k) {
      const float a = fabsf(W[k * ldw + n]);
      finite &= a < __int_as_float(0x7f800000);
      most = fmaxf(most, a);
    }
    float s = finite ? most / 7.0f : __int_as_float(0x7fc00000);
    if (s_dtype == kBF16) {
      const bf16 r = __float2bfloat16_rn(s);
      static_cast<bf16*>(scales)[g * lds + n] = r;
      s = __bfloat162float(r);
    } else if (s_dtype == kF16) {
      const f16 r = __float2half_rn(s);
      static_cast<f16*>(scales)[g * lds + n] = r;
      s = __half2float(r);
    } else {
      static_cast<float*>(scales)[g * lds + n] = s;
    }
    for (int64_t k = k0; k < k1; ++k) {
      const float q = s > 0.0f ? rintf(W[k * ldw + n] / s) : 0.0f;
      codes[k * ldc + n] = (uint8_t)((int)fminf(fmaxf(q, -8.0f), 7.0f) + 8);
    }
  }
}

__device__ __forceinline__ float packed_scale(const char* scales, int s_dtype, int64_t i) {
  return load_as_f32(scales, s_dtype, i);
}

__global__ void w4_dequantize_kernel(const uint32_t* __restrict__ codes, const char* scales,
                                     const uint8_t* zeros, W4Layout w, int64_t kblocks,
                                     int64_t groups, int64_t total, float* __restrict__ W,
                                     int64_t ldw) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int j = (int)(i & 3), lane = (int)(i >> 2 & 31), mt = (int)(i >> 7 & 3);
    const int64_t block = i >> 9, kb = block % kblocks, strip = block / kblocks;
    const uint32_t word = codes[i];
#pragma unroll
    for (int nib = 0; nib < 8; ++nib) {
      int k, n;
      code_place(lane, j, nib, &k, &n);
      n += mt * 16;
      const int64_t gk = kb * kBlockK + k, gn = strip * kStripN + n;
      if (gk >= w.K || gn >= w.N) continue;
      const int64_t at = (strip * groups + gk / w.group) * 64 + column_place(n);
      const int z = zeros ? zeros[at] : 8;
      W[gk * ldw + gn] = packed_scale(scales, w.s_dtype, at) * (float)((int)(word >> (4 * nib) & 15) - z);
    }
  }
}

// ------------------------------------------------------------------ product

// Few rows: a CTA has one strip of 64 columns and at most 8 operand columns,
// and its eight warps split the blocks of its part of K; the CTAs of a cluster
// share K. Every lane copies the codes that it will use itself, kDepth blocks
// ahead, into shared memory (cp.async), so the loop over K has no barrier;
// scales follow one block behind in registers. The activations of the CTA's
// part of K are staged once, or stage_blocks of K at a time where that takes
// more than kXBytes.
//
// Bound by instructions, not yet by HBM: about 340 of a warp for a block and strip
// (4096 weights: 176 to expand them, 16 products, 16 sums, the rest copies and
// addresses), 2.6 of a thread for a weight; the schedulers issue in 51% of cycles
// (1x8192x16384). 1x4096x4096 bf16 5.3 us (floor 1.3), 1x8192x16384 22.2 us or
// 3.1 TB/s (floor 10.6); with four warps a CTA and four CTAs an SM 5.7 and 26.5 us,
// with six blocks ahead 32.5 us for the latter. 1x4096x11008 f32, whose variant
// spills 48 bytes, lost by it: 13.8 us with four warps, 14.5 with eight.
constexpr int kFewWarps = 8;
constexpr int kFewColumns = 8;  // operand columns of a CTA
constexpr int kDepth = 4;
constexpr int kXBytes = 24 * 1024;
constexpr int kFewCtas = 2;  // an SM
constexpr int kFewShared = 96 * 1024;  // at most: 64 copied ahead, kXBytes, sums

template <int XT, bool FINE>
__global__ void __launch_bounds__(kFewWarps * 32, kFewCtas)
    dense_w4_few_kernel(const __grid_constant__ W4Params p) {
  using X = XRow<XT>;
  using Mma = typename X::Mma;
  using Raw = typename X::Raw;
  constexpr int MT = 4, SUBS = FINE ? 2 : 1, THREADS = kFewWarps * 32;
  extern __shared__ __align__(16) char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int log_c = p.log_cluster, C = 1 << log_c, rank = blockIdx.x & (C - 1);
  if (C > 1) cluster.barrier_arrive();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const DenseW4Args& a = p.a;
  const int64_t strip = blockIdx.x >> log_c, n0 = strip * kStripN;
  const int64_t m0 = (int64_t)blockIdx.y * p.rows;
  const int mrows = (int)min((int64_t)p.rows, a.M - m0), cols = mrows * X::kParts;
  const int K = (int)a.w.K, kblocks = (int)p.kblocks;
  const int b0 = (int)((int64_t)kblocks * rank >> log_c);
  const int b1 = (int)((int64_t)kblocks * (rank + 1) >> log_c);
  const bool s32 = a.w.s_dtype == kF32;

  // shared memory: what the cluster's CTAs send, the codes, the activations
  char* ring = smem + p.recv_bytes;
  uint4* mine = reinterpret_cast<uint4*>(ring) + wid * (kDepth * 128) + lane;
  const uint4* codes = p.codes + (strip * kblocks + b0 + wid) * 128 + lane;  // next to fetch
  int fetched = b0 + wid;
  const int64_t col0 = strip * p.groups * 64 + g * 8;
  auto fetch = [&](int slot) {
    if (fetched < b1) {
#pragma unroll
      for (int i = 0; i < MT; ++i) cp_async16(mine + slot * 128 + i * 32, codes + i * 32);
    }
    codes += kFewWarps * 128;
    fetched += kFewWarps;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // a block's scales are asked for when the scales before them have been used,
  // its zeros one block ahead
  const char* lane_scales = p.scales + (s32 ? col0 * 4 : col0 * 2);
  const int scale_step = s32 ? 256 : 128;  // bytes of a group
  uint4 raw[SUBS][2];
  uint2 zraw[SUBS];
  auto fetch_scales = [&](int b) {
    if (b >= b1) return;
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
      const int k = b * kBlockK + sub * 32;
      if (FINE && k >= K) return;
      const uint4* sp =
          reinterpret_cast<const uint4*>(lane_scales + (int64_t)p.group_of(k) * scale_step);
      raw[sub][0] = __ldg(sp);
      if (s32) raw[sub][1] = __ldg(sp + 1);
    }
  };
  auto fetch_zeros = [&](int b) {
    if (!p.zeros || b >= b1) return;
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
      const int k = b * kBlockK + sub * 32;
      if (FINE && k >= K) return;
      zraw[sub] = __ldg(reinterpret_cast<const uint2*>(p.zeros + col0 + (int64_t)p.group_of(k) * 64));
    }
  };
  // until pdl_wait the previous kernel of the stream may still run
  if (tid == 0) prefetch_strip(p, strip, b0, b1, true);
  pdl_wait();

  // The activations that are staged first are asked for before the weights.
  int per_row = min(b1 - b0, p.stage_blocks) * 8;  // units of 8 elements
  const char* xrow = static_cast<const char*>(a.X) + m0 * a.ldx * X::kBytes;
  auto load_x = [&](int s0, int m, int c) {
    return X::load(xrow + m * a.ldx * X::kBytes, (int64_t)s0 * kBlockK + c * 8, K, p.x_aligned);
  };
  auto next_unit = [&](int& m, int& c) {
    while (c >= per_row) {
      c -= per_row;
      ++m;
    }
  };
  Raw first = {};
  int m = 0, c = tid;
  if (b0 < b1) {
    next_unit(m, c);
    if (m < mrows) first = load_x(b0, m, c);
  }
#pragma unroll
  for (int i = 0; i < kDepth; ++i) fetch(i);
  fetch_scales(b0 + wid);
  fetch_zeros(b0 + wid);

  char* xsm = ring + kFewWarps * kDepth * 2048;
  const int pitch = p.stage_blocks * 128 + 64;  // bytes of a staged column: 64 mod 128
  if (cols < kFewColumns && tid < 8)
    *reinterpret_cast<uint4*>(xsm + cols * pitch + tid * 16) = make_uint4(0, 0, 0, 0);
  float total[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) total[i][c] = 0.0f;

  int b = b0 + wid, slot = 0;
  for (int s0 = b0; s0 < b1; s0 += p.stage_blocks) {
    const int s1 = min(b1, s0 + p.stage_blocks);
    if (s0 != b0) __syncthreads();
    if (s0 != b0) {
      per_row = (s1 - s0) * 8;
      m = 0;
      c = tid;
      next_unit(m, c);
      if (m < mrows) first = load_x(s0, m, c);
    }
    auto store_x = [&](int m, int c, const Raw& e) {
      uint4 out[X::kParts];
      X::stage(e, out);
      // Pair t of piece c is word c % 4 of the 16 bytes that lane t of a column
      // reads for 32 of K.
#pragma unroll
      for (int q = 0; q < X::kParts; ++q) {
        uint32_t* to = reinterpret_cast<uint32_t*>(xsm + (m * X::kParts + q) * pitch +
                                                   (c >> 2) * 64 + (c & 3) * 4);
        to[0] = out[q].x;
        to[4] = out[q].y;
        to[8] = out[q].z;
        to[12] = out[q].w;
      }
    };
    if (m < mrows) store_x(m, c, first);
    while (m < mrows) {  // the others, four loads at a time
      constexpr int U = 4;
      Raw e[U];
      int um[U], uc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        c += THREADS;
        next_unit(m, c);
        um[u] = m;
        uc[u] = c;
        if (m < mrows) e[u] = load_x(s0, m, c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (um[u] < mrows) store_x(um[u], uc[u], e[u]);
    }
    __syncthreads();
    // operand column g; columns that no row has read zeros
    const char* xs = g < cols ? xsm + g * pitch + (b - s0) * 128 + t * 16 : xsm + cols * pitch;
    const int xstep = g < cols ? kFewWarps * 128 : 0;
    for (; b < s1; b += kFewWarps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      uint4 cur[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) cur[i] = mine[slot * 128 + i * 32];
      uint32_t zero[SUBS][2 * MT];
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)  // one byte of z under the magic number's
          zero[sub][i] = p.zeros ? __byte_perm(i < 4 ? zraw[sub].x : zraw[sub].y, Mma::kMagic,
                                               0x5050 | (i & 3) * 0x0101)
                                 : 0x00080008u | Mma::kMagic;
      fetch_zeros(b + kFewWarps);
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        const int k = b * kBlockK + sub * 32;
        if (FINE && k >= K) break;  // the second half of the last block
        float acc[MT][4];
#pragma unroll
        for (int h = FINE ? sub : 0; h < (FINE ? sub + 1 : 2); ++h) {
          const uint4 xb = *reinterpret_cast<const uint4*>(xs + h * 64);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const uint2 w = h == 0 ? make_uint2(cur[i].x, cur[i].y) : make_uint2(cur[i].z, cur[i].w);
#pragma unroll
            for (int step = 0; step < 2; ++step) {
              uint32_t f[4];
#pragma unroll
              for (int r = 0; r < 4; ++r)
                f[r] = Mma::sub(and_or((step == 0 ? w.x : w.y) >> (4 * r), 0x000f000fu, Mma::kMagic),
                                zero[sub][2 * i + (r & 1)]);
              const uint32_t x0 = step == 0 ? xb.x : xb.z, x1 = step == 0 ? xb.y : xb.w;
              if (step == 0 && (FINE || h == 0)) Mma::mma_first(acc[i], f, x0, x1);
              else Mma::mma(acc[i], f, x0, x1);
            }
          }
        }
        // scales of the rows of X, where they have one for each group of K
        if (XT == kE4M3 && a.x_group > 0) {
          const unsigned xg = (unsigned)k / (unsigned)a.x_group;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int m = t * 2 + c;
            const float s = m < mrows ? __ldg(a.x_scales + (m0 + m) * a.ldxs + xg) : 0.0f;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              acc[i][c] *= s;
              acc[i][2 + c] *= s;
            }
          }
        }
        float sc[2 * MT];
        if (s32) {
          unpack(raw[sub][0], (const float*)nullptr, sc);
          unpack(raw[sub][1], (const float*)nullptr, sc + 4);
        } else if (a.w.s_dtype == kBF16) {
          unpack(raw[sub][0], (const bf16*)nullptr, sc);
        } else {
          unpack(raw[sub][0], (const f16*)nullptr, sc);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            total[i][c] = fmaf(acc[i][c], sc[2 * i + (c >> 1)], total[i][c]);
      }
      fetch_scales(b + kFewWarps);
      fetch(slot);
      slot = (slot + 1) & (kDepth - 1);
      xs += xstep;
    }
  }

  // ---- add the warps' parts of K in order, then the CTAs'. Each 32 outputs
  // of a row belong to one CTA of the cluster, in turn: the others send it
  // their sums.
  __syncthreads();
  float* red = reinterpret_cast<float*>(ring);   // [warp][column][64]
  float* recv = reinterpret_cast<float*>(smem);  // [CTA][part][slot]
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = t * 2 + c;
    if (col < cols) {
      float* to = red + (wid * kFewColumns + col) * 64 + g;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        to[i * 16] = total[i][c];
        to[i * 16 + 8] = total[i][2 + c];
      }
    }
  }
  __syncthreads();
  const int outs = mrows * 64;
  const int slots = ((mrows * 2 + C - 1) >> log_c) * 32;  // outputs of a CTA
  if (C > 1) cluster.barrier_wait();                     // every CTA of the cluster runs
  for (int u = tid; u < outs * X::kParts; u += THREADS) {
    const int col = u >> 6, m = col / X::kParts, q = col - m * X::kParts;
    float v = red[u];
#pragma unroll
    for (int k = 1; k < kFewWarps; ++k) v += red[k * kFewColumns * 64 + u];
    const int chunk = m * 2 + (u >> 5 & 1);
    float* dst = recv + (rank * X::kParts + q) * slots + (chunk >> log_c) * 32 + (u & 31);
    *(C > 1 ? cluster.map_shared_rank(dst, chunk & (C - 1)) : dst) = v;
  }
  // the bias of this thread's first output is on its way meanwhile
  auto bias_of = [&](int u) {
    const int64_t n = n0 + (((u >> 5 << log_c) + rank) * 32 + (u & 31) & 63);
    return a.b && n < a.w.N ? load_as_f32(a.b, a.b_dtype, n) : 0.0f;
  };
  float bias = bias_of(tid);
  if (C > 1) cluster.sync();
  else __syncthreads();
  for (int u = tid; u < slots; u += THREADS) {
    if (u != tid) bias = bias_of(u);
    const int o = ((u >> 5 << log_c) + rank) * 32 + (u & 31), m = o >> 6, n = o & 63;
    if (o >= outs || n0 + n >= a.w.N) continue;
    float part[X::kParts];
#pragma unroll
    for (int q = 0; q < X::kParts; ++q) part[q] = recv[q * slots + u];
    for (int r = 1; r < C; ++r)
#pragma unroll
      for (int q = 0; q < X::kParts; ++q) part[q] += recv[(r * X::kParts + q) * slots + u];
    float y = part[X::kParts - 1];  // the smallest part first
#pragma unroll
    for (int q = X::kParts - 2; q >= 0; --q) y += part[q];
    y *= Mma::kUp;
    if (a.x_scales && a.x_group == 0) y *= __ldg(a.x_scales + (m0 + m) * a.ldxs);
    if (a.b) y += bias;
    y = activate(y, a.act, a.alpha);
    const int64_t at = (m0 + m) * a.ldy + n0 + n;
    if (a.y_dtype == kF32) static_cast<float*>(a.Y)[at] = y;
    else if (a.y_dtype == kBF16) static_cast<bf16*>(a.Y)[at] = __float2bfloat16_rn(y);
    else static_cast<f16*>(a.Y)[at] = __float2half_rn(y);
  }
}

template <int XT, bool FINE>
int launch_few(W4Params p, cudaStream_t st) {
  auto kernel = dense_w4_few_kernel<XT, FINE>;
  p.rows = kFewColumns / XRow<XT>::kParts;
  const int64_t tiles = p.a.w.strips();
  const int64_t chunks = (p.a.M + p.rows - 1) / p.rows;
  if (chunks > 65535) return kErrTooLarge;
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  const cudaError_t e0 = allow_shared(reinterpret_cast<const void*>(kernel), allowed, &dev);
  if (e0 != cudaSuccess) return launch_result(e0);
  static PerDevice<Capacity> capacities;
  const Capacity capacity = capacities.of(dev, [&] {
    return capacity_of(reinterpret_cast<const void*>(kernel), kFewWarps * 32, kFewShared);
  });
  const int best = choose_cluster(capacity, tiles * chunks, p.kblocks, kFewWarps, 4);
  const int C = 1 << best;
  p.log_cluster = best;
  const int64_t mine = (p.kblocks + C - 1) / C;
  const int rows = (int)std::min<int64_t>(p.rows, p.a.M), cols = rows * XRow<XT>::kParts;
  p.stage_blocks = (int)std::max<int64_t>(
      1, std::min<int64_t>(mine, std::max(kFewWarps, (kXBytes / cols - 64) / 128 / kFewWarps *
                                                         kFewWarps)));
  p.recv_bytes = C * XRow<XT>::kParts * ((rows * 2 + C - 1) / C * 32) * 4;
  const int smem = p.recv_bytes + kFewWarps * kDepth * 2048 + cols * (p.stage_blocks * 128 + 64) +
                   128;  // and the zeros of columns that no row has
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * C), (unsigned)chunks);
  cfg.blockDim = dim3(kFewWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  count_launch();
  return launch_result(e != cudaSuccess ? e : cudaGetLastError());
}

// Up to 8 operand columns on mma.sync, whose n it is; more on the tensor core
// (bf16 12x4096x4096: 7.7 us there, 9.7 with two tiles of 8 columns here).
template <int XT>
int dispatch(const W4Params& p, int* status, cudaStream_t st) {
  if (p.a.M * XRow<XT>::kParts > kFewColumns) return dense_w4_tc(p, status, st);
  return p.a.w.group == 32 || p.a.x_group == 32 ? launch_few<XT, true>(p, st)
                                                : launch_few<XT, false>(p, st);
}

unsigned grid_for(int64_t work) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((work + 255) / 256, 148 * 32));
}

}  // namespace

int dense_w4(const DenseW4Args& a, int* status, cudaStream_t st) {
  W4Params p;
  p.a = a;
  const char* base = static_cast<const char*>(a.packed);
  p.codes = reinterpret_cast<const uint4*>(base);
  p.scales = base + a.w.codes_bytes();
  p.zeros = a.w.has_zeros
                ? reinterpret_cast<const uint8_t*>(p.scales + a.w.scales_bytes())
                : nullptr;
  p.kblocks = a.w.kblocks();
  p.groups = a.w.groups();
  p.rows = p.stage_blocks = p.recv_bytes = p.log_cluster = 0;
  p.group_shift = -1;
  for (int l = 5; l < 31; ++l)
    if (a.w.group == 1 << l) p.group_shift = l;
  const int64_t bytes = dtype_bytes(a.x_dtype);
  const int64_t unit = a.x_dtype == kE4M3 ? 8 : 16;
  p.x_aligned = reinterpret_cast<uintptr_t>(a.X) % unit == 0 && a.ldx * bytes % unit == 0;
  switch (a.x_dtype) {
    case kF32: return dispatch<kF32>(p, status, st);
    case kBF16: return dispatch<kBF16>(p, status, st);
    case kF16: return dispatch<kF16>(p, status, st);
    default: return dispatch<kE4M3>(p, status, st);
  }
}

int w4_quantize(const float* W, int64_t ldw, int64_t K, int64_t N, int group, uint8_t* codes,
                int64_t ldc, void* scales, int64_t lds, int s_dtype, cudaStream_t st) {
  const int64_t groups = (K + group - 1) / group;
  w4_quantize_kernel<<<grid_for(groups * N), 256, 0, st>>>(W, ldw, K, N, group, groups, codes, ldc,
                                                           scales, lds, s_dtype);
  count_launch();
  return launch_result();
}

int w4_pack(const uint8_t* codes, int64_t ldc, const void* scales, int64_t lds,
            const uint8_t* zeros, int64_t ldz, const W4Layout& w, void* packed, cudaStream_t st) {
  char* base = static_cast<char*>(packed);
  const int64_t words = w.strips() * w.kblocks() * 512;
  w4_pack_codes_kernel<<<grid_for(words), 256, 0, st>>>(codes, ldc, w.K, w.N, w.kblocks(), words,
                                                        reinterpret_cast<uint32_t*>(base));
  count_launch();
  int rc = launch_result();
  if (rc) return rc;
  const int64_t columns = w.strips() * w.groups() * 64;
  base += w.codes_bytes();
  w4_pack_columns_kernel<<<grid_for(columns), 256, 0, st>>>(
      scales, lds, w.groups(), w.N, w.strips(), w.s_dtype == kF32 ? 4 : 2, base);
  count_launch();
  if ((rc = launch_result()) || !w.has_zeros) return rc;
  w4_pack_columns_kernel<<<grid_for(columns), 256, 0, st>>>(
      zeros, ldz, w.groups(), w.N, w.strips(), 1, base + w.scales_bytes());
  count_launch();
  return launch_result();
}

int w4_dequantize(const void* packed, const W4Layout& w, float* W, int64_t ldw, cudaStream_t st) {
  const char* base = static_cast<const char*>(packed);
  const char* scales = base + w.codes_bytes();
  const uint8_t* zeros =
      w.has_zeros ? reinterpret_cast<const uint8_t*>(scales + w.scales_bytes()) : nullptr;
  const int64_t words = w.strips() * w.kblocks() * 512;
  w4_dequantize_kernel<<<grid_for(words), 256, 0, st>>>(reinterpret_cast<const uint32_t*>(base),
                                                        scales, zeros, w, w.kblocks(), w.groups(),
                                                        words, W, ldw);
  count_launch();
  return launch_result();
}

}  // namespace b200
