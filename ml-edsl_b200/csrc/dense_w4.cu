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
// bf16 parts of 8 bits each (exact), in three columns that are added at the
// end. No product is rounded; sums run in f32, in the tensor core within a
// group (or a 64-long part of one), then with ordinary adds after the scale
// is applied in f32. An accumulator in TMEM would hold 128 columns of W by at
// least 8 rows of X, but its operands have to come from shared memory, and
// weights that are used once, by few rows, would be written there expanded
// four times only to be read again; here they go from HBM to registers and
// into the product.
//
// Layout (w4_pack): strips of 64 columns; in a strip, blocks of 64 of K; in a
// block, four 512-byte pieces of 16 columns, 16 bytes for each lane: the
// codes of its fragments of four k16 steps, in an order that takes one shift
// and one and-or for two weights. K inside a block is permuted so that a
// lane's activations are 16 contiguous bytes. Scales and zeros lie in the
// order in which the lanes read them.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstdint>
#include <cstdlib>
#include <mutex>
#include <set>
#include <utility>
#include "dtype.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace b200 {

namespace {

constexpr int kBlockK = 64;   // k of one packed block
constexpr int kStripN = 64;   // columns of one strip
constexpr int kWarps = 8;
constexpr int kMaxCluster = 8;

// ------------------------------------------------------------------ packing

// Row of W (k) of nibble `nib` of word `j` of lane `lane`'s 16 bytes, within
// its block, and its column within the 16 columns of the piece.
__host__ __device__ __forceinline__ void code_place(int lane, int j, int nib, int* k, int* n) {
  const int g = lane >> 2, t = lane & 3, r = nib & 3;
  *k = (j >> 1) * 32 + t * 8 + (j & 1) * 4 + (r >> 1) * 2 + (nib >> 2);
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

// Place of column n (within its strip) among a group's 64 scales or zeros:
// lane group g = n % 8 reads its eight values together.
__host__ __device__ __forceinline__ int column_place(int n) { return (n & 7) * 8 + (n >> 3); }

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
// to the scales' type; q = round(w / s) + 8 with ties to even. A thread has
// one column of one group.
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
    for (int64_t k = k0; k < k1; ++k) most = fmaxf(most, fabsf(W[k * ldw + n]));
    float s = most / 7.0f;
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

// (a & b) | c in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// The types of the product's operands.
struct MmaBF16 {
  static constexpr uint32_t kMagic = 0x43004300u;  // 128 + q in bf16: q in the low bits
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4],
                                                   uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  }
};
struct MmaF16 {
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024 + q in f16
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a),
                              *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4],
                                                   uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  }
};

// How rows of X become operand columns: kParts columns for a row. stage()
// takes 8 consecutive elements and gives 16 bytes for each column.
template <int XT>
struct XRow;
template <>
struct XRow<kBF16> {
  using Mma = MmaBF16;
  using T = uint16_t;
  static constexpr int kParts = 1;
  static __device__ __forceinline__ void stage(const T (&e)[8], uint4 (&out)[1]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
    out[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct XRow<kF16> : XRow<kBF16> {
  using Mma = MmaF16;
};
template <>
struct XRow<kE4M3> {
  using Mma = MmaF16;
  using T = uint8_t;
  static constexpr int kParts = 1;
  static __device__ __forceinline__ void stage(const T (&e)[8], uint4 (&out)[1]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          (__nv_fp8x2_storage_t)(e[2 * i] | (uint16_t)e[2 * i + 1] << 8), __NV_E4M3);
      w[i] = h.x | (uint32_t)h.y << 16;
    }
    out[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct XRow<kF32> {
  using Mma = MmaBF16;
  using T = uint32_t;
  static constexpr int kParts = 3;
  // x = hi + mid + lo, each the leading 8 bits of what is left (cut, so that
  // no part rounds up out of range). Infinities and NaN travel in hi.
  static __device__ __forceinline__ void stage(const T (&e)[8], uint4 (&out)[3]) {
    uint32_t p[3][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool finite = (e[i] & 0x7f800000u) != 0x7f800000u;
      const bool nan = !finite && (e[i] & 0x007fffffu);
      p[0][i] = nan ? 0x7fc0u : e[i] >> 16;
      const float r = __uint_as_float(e[i]) - __uint_as_float(e[i] & 0xffff0000u);
      const uint32_t rb = __float_as_uint(r) & 0xffff0000u;
      p[1][i] = finite ? rb >> 16 : 0u;
      p[2][i] = finite ? __float_as_uint(r - __uint_as_float(rb)) >> 16 : 0u;
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = p[q][2 * i] | p[q][2 * i + 1] << 16;
      out[q] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

// Eight elements of a row of X from column k on, 0 from `end` on.
template <class T>
__device__ __forceinline__ void load8(const T* row, int64_t k, int64_t end, bool aligned,
                                      T (&e)[8]) {
  if (aligned && k + 8 <= end) {
    if constexpr (sizeof(T) == 1) {
      *reinterpret_cast<uint2*>(e) = __ldg(reinterpret_cast<const uint2*>(row + k));
    } else {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(row + k) + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < end ? __ldg(row + k + i) : T(0);
  }
}

__device__ __forceinline__ float activate(float x, int act, float alpha) {
  if (act == kActRelu) return (x > 0.0f || x != x) ? x : 0.0f;
  if (act == kActLeakyRelu) {
    const float pos = (x > 0.0f || x != x) ? x : 0.0f;
    const float neg = (x < 0.0f || x != x) ? x : 0.0f;
    return pos + neg * alpha;
  }
  return x;
}

// Eight scales of a lane as floats: scale of fragment row `half` of 16-column
// piece mt is v[2 * mt + half].
template <int MT>
__device__ __forceinline__ void load_scales(const char* p, int s_dtype, float (&v)[2 * MT]) {
  if (s_dtype == kF32) {
#pragma unroll
    for (int i = 0; i < MT / 2; ++i) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p) + i);
      v[4 * i] = f.x;
      v[4 * i + 1] = f.y;
      v[4 * i + 2] = f.z;
      v[4 * i + 3] = f.w;
    }
    return;
  }
  uint32_t w[MT];
  if constexpr (MT == 4)
    *reinterpret_cast<uint4*>(w) = __ldg(reinterpret_cast<const uint4*>(p));
  else
    *reinterpret_cast<uint2*>(w) = __ldg(reinterpret_cast<const uint2*>(p));
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    if (s_dtype == kBF16) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

struct Params {
  DenseW4Args a;
  const uint4* codes;
  const char* scales;
  const uint8_t* zeros;
  int64_t kblocks, groups;
  int rows;          // rows of X for each blockIdx.y
  int stage_blocks;  // blocks of K whose activations are staged at once
  int x_aligned;
  int recv_bytes;    // of shared memory for other CTAs' sums
  int log_cluster;   // CTAs that share K
  int group_shift;   // log2 of the group, or -1
  __device__ __forceinline__ unsigned group_of(int k) const {
    return group_shift >= 0 ? (unsigned)k >> group_shift : (unsigned)k / (unsigned)a.w.group;
  }
};

// A CTA computes WN * MT * 16 columns of Y for `rows` rows of X, over its
// part of K (the CTAs of a cluster share K): WN warps side by side in N, the
// others of the eight split the blocks of K among them. Each warp keeps the
// next block's codes in flight in registers. The parts of K are added in
// shared memory, warps first, then the cluster's CTAs, in a fixed order.
template <int XT, int NT, int MT, int WN, bool FINE>
__global__ void __launch_bounds__(kWarps * 32)
    dense_w4_kernel(const __grid_constant__ Params p) {
  using X = XRow<XT>;
  using Mma = typename X::Mma;
  using T = typename X::T;
  constexpr int WK = kWarps / WN, COLS = NT * 8, ROWS = WN * MT * 16;
  constexpr int SUBS = FINE ? 2 : 1;  // scales applied every 32 or every 64 of K
  extern __shared__ __align__(16) char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wn = wid % WN, wk = wid / WN;
  const DenseW4Args& a = p.a;
  const int64_t n0 = (int64_t)(blockIdx.x / C) * ROWS;
  const int64_t m0 = (int64_t)blockIdx.y * p.rows;
  const int mrows = (int)min((int64_t)p.rows, a.M - m0);
  // blocks of K of this CTA
  const int K = (int)a.w.K, kblocks = (int)p.kblocks;
  const int b0 = (int)((int64_t)kblocks * rank / C), b1 = (int)((int64_t)kblocks * (rank + 1) / C);
  // this warp's 16-column pieces: MT of the four of a strip
  const int64_t nw = n0 + (int64_t)wn * MT * 16;
  const int64_t strip = nw / kStripN;
  const int mt0 = (int)(nw % kStripN) / 16;
  const bool live = nw < a.w.N;  // the last CTA may have warps past the last strip
  const uint4* codes = p.codes + (strip * p.kblocks * 4 + mt0) * 32 + lane;
  const int64_t col0 = strip * p.groups * 64 + g * 8 + mt0 * 2;
  const int sbytes = a.w.s_dtype == kF32 ? 4 : 2;

  const int pitch = p.stage_blocks * 128 + 64;  // bytes of a staged column: 64 mod 128
  float total[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) total[i][j][c] = 0.0f;

  uint4 next[MT];
  auto fetch = [&](int b) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
      next[i] = live && b < b1 ? __ldcs(codes + (int64_t)b * 128 + i * 32) : make_uint4(0, 0, 0, 0);
  };
  int b = b0 + wk;
  fetch(b);

  for (int s0 = b0; s0 < b1; s0 += p.stage_blocks) {
    const int s1 = min(b1, s0 + p.stage_blocks);
    // ---- stage the activations of blocks [s0, s1): column m * parts + part
    const int per_row = (s1 - s0) * 8;  // units of 8 elements
    if (s0 != b0) __syncthreads();
    for (int u = tid; u < per_row * (COLS / X::kParts); u += kWarps * 32) {
      const int m = u / per_row, c = u - m * per_row;
      uint4 out[X::kParts];
      if (m < mrows) {
        __align__(16) T e[8];
        load8(static_cast<const T*>(a.X) + (m0 + m) * a.ldx, (int64_t)s0 * kBlockK + c * 8, K,
              p.x_aligned, e);
        X::stage(e, out);
      } else {
#pragma unroll
        for (int q = 0; q < X::kParts; ++q) out[q] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int q = 0; q < X::kParts; ++q)
        *reinterpret_cast<uint4*>(smem + (m * X::kParts + q) * pitch + c * 16) = out[q];
    }
    if (X::kParts > 1)  // columns that no row has
      for (int u = tid; u < per_row * (COLS % X::kParts); u += kWarps * 32) {
        const int q = COLS - COLS % X::kParts + u / per_row;
        *reinterpret_cast<uint4*>(smem + q * pitch + u % per_row * 16) = make_uint4(0, 0, 0, 0);
      }
    __syncthreads();

    for (; b < s1; b += WK) {
      uint4 cur[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) cur[i] = next[i];
      fetch(b + WK);
      if (!live) continue;
      const char* xs = smem + g * pitch + (b - s0) * 128 + t * 16;
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        const int k = b * kBlockK + sub * 32;
        if (FINE && k >= K) break;  // the second half of the last block
        const int64_t at = col0 + (int64_t)((unsigned)k / (unsigned)a.w.group) * 64;
        float sc[2 * MT];
        load_scales<MT>(p.scales + at * sbytes, a.w.s_dtype, sc);
        uint32_t zero[2 * MT];
        if (p.zeros) {
          uint32_t z[2];
          if constexpr (MT == 4) {
            *reinterpret_cast<uint2*>(z) = __ldg(reinterpret_cast<const uint2*>(p.zeros + at));
          } else {
            z[0] = __ldg(reinterpret_cast<const uint32_t*>(p.zeros + at));
          }
#pragma unroll
          for (int i = 0; i < 2 * MT; ++i)
            zero[i] = ((z[i >> 2] >> (8 * (i & 3)) & 15u) * 0x00010001u) | Mma::kMagic;
        } else {
#pragma unroll
          for (int i = 0; i < 2 * MT; ++i) zero[i] = 0x00080008u | Mma::kMagic;
        }
        float acc[MT][NT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.0f;
#pragma unroll
        for (int h = FINE ? sub : 0; h < (FINE ? sub + 1 : 2); ++h) {
          uint4 xb[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j)
            xb[j] = *reinterpret_cast<const uint4*>(xs + j * 8 * pitch + h * 64);
#pragma unroll
          for (int step = 0; step < 2; ++step)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const uint32_t w = h == 0 ? (step == 0 ? cur[i].x : cur[i].y)
                                        : (step == 0 ? cur[i].z : cur[i].w);
              uint32_t f[4];
#pragma unroll
              for (int r = 0; r < 4; ++r)
                f[r] = Mma::sub((w >> (4 * r) & 0x000f000fu) | Mma::kMagic, zero[2 * i + (r & 1)]);
#pragma unroll
              for (int j = 0; j < NT; ++j)
                Mma::mma(acc[i][j], f, step == 0 ? xb[j].x : xb[j].z,
                         step == 0 ? xb[j].y : xb[j].w);
            }
        }
        // scales of the rows of X, where they have one for each group of K
        if (XT == kE4M3 && a.x_group > 0) {
          const unsigned xg = (unsigned)k / (unsigned)a.x_group;
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int m = j * 8 + t * 2 + c;
              const float s = m < mrows ? __ldg(a.x_scales + (m0 + m) * a.ldxs + xg) : 0.0f;
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                acc[i][j][c] *= s;
                acc[i][j][2 + c] *= s;
              }
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              total[i][j][c] = fmaf(acc[i][j][c], sc[2 * i + (c >> 1)], total[i][j][c]);
      }
    }
  }

  // ---- add the warps' parts of K, then the CTAs', in shared memory
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);  // [WK][COLS][ROWS]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        red[(wk * COLS + j * 8 + t * 2 + (c & 1)) * ROWS + wn * MT * 16 + i * 16 + (c >> 1) * 8 +
            g] = total[i][j][c];
  __syncthreads();
  const int cols = mrows * X::kParts;
  if (WK > 1) {
    for (int u = tid; u < cols * ROWS; u += kWarps * 32) {
      float v = red[u];
#pragma unroll
      for (int k = 1; k < WK; ++k) v += red[k * COLS * ROWS + u];
      red[u] = v;
    }
    if (C == 1) __syncthreads();
  }
  if (C > 1) cluster.sync();
  const int outs = mrows * ROWS;
  for (int u = rank * kWarps * 32 + tid; u < outs; u += C * kWarps * 32) {
    const int m = u / ROWS, n = u - m * ROWS;
    if (n0 + n >= a.w.N) continue;
    float part[X::kParts];
#pragma unroll
    for (int q = 0; q < X::kParts; ++q) part[q] = 0.0f;
    for (int r = 0; r < C; ++r) {
      const float* from = C > 1 ? cluster.map_shared_rank(red, r) : red;
#pragma unroll
      for (int q = 0; q < X::kParts; ++q) part[q] += from[(m * X::kParts + q) * ROWS + n];
    }
    float y = part[X::kParts - 1];  // the smallest part first
#pragma unroll
    for (int q = X::kParts - 2; q >= 0; --q) y += part[q];
    if (a.x_scales && a.x_group == 0) y *= __ldg(a.x_scales + (m0 + m) * a.ldxs);
    if (a.b) y += load_as_f32(a.b, a.b_dtype, n0 + n);
    y = activate(y, a.act, a.alpha);
    const int64_t at = (m0 + m) * a.ldy + n0 + n;
    if (a.y_dtype == kF32) static_cast<float*>(a.Y)[at] = y;
    else if (a.y_dtype == kBF16) static_cast<bf16*>(a.Y)[at] = __float2bfloat16_rn(y);
    else static_cast<f16*>(a.Y)[at] = __float2half_rn(y);
  }
  if (C > 1) cluster.sync();  // nobody reads this CTA's shared memory any more
}

// Lets `kernel` use 200 KB of dynamic shared memory on the current device.
cudaError_t allow_shared(const void* kernel) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lk(mu);
  if (done.count({kernel, dev})) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  if (e == cudaSuccess) done.insert({kernel, dev});
  return e;
}

__device__ __forceinline__ void cp_async16(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(smem_u32(smem)),
               "l"(global)
               : "memory");
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// Brings `bytes` (a multiple of 16) at a 16-byte aligned address into L2.
__device__ __forceinline__ void prefetch_l2_bulk(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// Few rows: a CTA has one strip of 64 columns and at most 8 * NT operand
// columns, and its four warps split the blocks of its part of K. Every lane
// copies the codes that it will use itself, kDepth blocks ahead, into shared
// memory (cp.async), so the loop over K has no barrier; scales and zeros are
// one block ahead in registers. The activations of the CTA's part of K are
// staged once, or stage_blocks of K at a time where that takes more than
// kXBytes. CTAs are small so that several share an SM and the last wave is
// short; the CTAs of a cluster share K.
#ifndef W4MINB
#define W4MINB 4
#define W4OCC 4
#endif
constexpr int kFewWarps = 4;
constexpr int kDepth = 4;
constexpr int kXBytes = 24 * 1024;

template <int XT, int NT, bool FINE>
__global__ void __launch_bounds__(kFewWarps * 32, W4MINB)
    dense_w4_few_kernel(const __grid_constant__ Params p) {
  using X = XRow<XT>;
  using Mma = typename X::Mma;
  using T = typename X::T;
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
  // What the CTA will read of the weights is contiguous. The previous kernel of
  // the stream may still run (and may have written them): until pdl_wait they
  // are only brought into L2.
  if (tid == 0 && b0 < b1)
    prefetch_l2_bulk(p.codes + (strip * kblocks + b0) * 128, (uint32_t)min(b1 - b0, 64) * 2048u);
  if (tid == 32 && b0 < b1) {
    const int64_t at = strip * p.groups * 64 + (int64_t)p.group_of(b0 * kBlockK) * 64;
    prefetch_l2(p.scales + (s32 ? at * 4 : at * 2));
  }
  pdl_wait();

  // The activations that are staged first are asked for before the weights.
  int per_row = min(b1 - b0, p.stage_blocks) * 8;  // units of 8 elements
  const T* xrow = static_cast<const T*>(a.X) + m0 * a.ldx;
  auto load_x = [&](int s0, int m, int c, T (&e)[8]) {
    load8(xrow + m * a.ldx, (int64_t)s0 * kBlockK + c * 8, K, p.x_aligned, e);
  };
  auto next_unit = [&](int& m, int& c) {
    while (c >= per_row) {
      c -= per_row;
      ++m;
    }
  };
  __align__(16) T first[8];
  int m = 0, c = tid;
  if (b0 < b1) {
    next_unit(m, c);
    if (m < mrows) load_x(b0, m, c, first);
  }
#pragma unroll
  for (int i = 0; i < kDepth; ++i) fetch(i);
  fetch_scales(b0 + wid);
  fetch_zeros(b0 + wid);

  char* xsm = ring + kFewWarps * kDepth * 2048;
  const int pitch = p.stage_blocks * 128 + 64;  // bytes of a staged column: 64 mod 128
  if (cols < NT * 8 && tid < 8)
    *reinterpret_cast<uint4*>(xsm + cols * pitch + tid * 16) = make_uint4(0, 0, 0, 0);
  float total[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) total[i][j][c] = 0.0f;

  int b = b0 + wid, slot = 0;
  for (int s0 = b0; s0 < b1; s0 += p.stage_blocks) {
    const int s1 = min(b1, s0 + p.stage_blocks);
    if (s0 != b0) __syncthreads();
    if (s0 != b0) {
      per_row = (s1 - s0) * 8;
      m = 0;
      c = tid;
      next_unit(m, c);
      if (m < mrows) load_x(s0, m, c, first);
    }
    auto store_x = [&](int m, int c, const T (&e)[8]) {
      uint4 out[X::kParts];
      X::stage(e, out);
#pragma unroll
      for (int q = 0; q < X::kParts; ++q)
        *reinterpret_cast<uint4*>(xsm + (m * X::kParts + q) * pitch + c * 16) = out[q];
    };
    if (m < mrows) store_x(m, c, first);
    while (m < mrows) {  // the others, four loads at a time
      constexpr int U = 4;
      __align__(16) T e[U][8];
      int um[U], uc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        c += THREADS;
        next_unit(m, c);
        um[u] = m;
        uc[u] = c;
        if (m < mrows) load_x(s0, m, c, e[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (um[u] < mrows) store_x(um[u], uc[u], e[u]);
    }
    __syncthreads();
    // operand column j * 8 + g; columns that no row has read zeros
    const char* xs[NT];
    int xstep[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const bool is = j * 8 + g < cols;
      xs[j] = is ? xsm + (j * 8 + g) * pitch + (b - s0) * 128 + t * 16 : xsm + cols * pitch;
      xstep[j] = is ? kFewWarps * 128 : 0;
    }
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
        float acc[MT][NT][4];
#pragma unroll
        for (int h = FINE ? sub : 0; h < (FINE ? sub + 1 : 2); ++h) {
          uint4 xb[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j) xb[j] = *reinterpret_cast<const uint4*>(xs[j] + h * 64);
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
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                const uint32_t b0 = step == 0 ? xb[j].x : xb[j].z;
                const uint32_t b1 = step == 0 ? xb[j].y : xb[j].w;
                if (step == 0 && (FINE || h == 0)) Mma::mma_first(acc[i][j], f, b0, b1);
                else Mma::mma(acc[i][j], f, b0, b1);
              }
            }
          }
        }
        // scales of the rows of X, where they have one for each group of K
        if (XT == kE4M3 && a.x_group > 0) {
          const unsigned xg = (unsigned)k / (unsigned)a.x_group;
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int m = j * 8 + t * 2 + c;
              const float s = m < mrows ? __ldg(a.x_scales + (m0 + m) * a.ldxs + xg) : 0.0f;
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                acc[i][j][c] *= s;
                acc[i][j][2 + c] *= s;
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
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              total[i][j][c] = fmaf(acc[i][j][c], sc[2 * i + (c >> 1)], total[i][j][c]);
      }
      fetch_scales(b + kFewWarps);
      fetch(slot);
      slot = (slot + 1) & (kDepth - 1);
#pragma unroll
      for (int j = 0; j < NT; ++j) xs[j] += xstep[j];
    }
  }

  // ---- add the warps' parts of K in order, then the CTAs'. Each 32 outputs
  // of a row belong to one CTA of the cluster, in turn: the others send it
  // their sums.
  __syncthreads();
  float* red = reinterpret_cast<float*>(ring);   // [warp][column][64]
  float* recv = reinterpret_cast<float*>(smem);  // [CTA][part][slot]
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = j * 8 + t * 2 + c;
      if (col < cols) {
        float* to = red + (wid * NT * 8 + col) * 64 + g;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          to[i * 16] = total[i][j][c];
          to[i * 16 + 8] = total[i][j][2 + c];
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
    for (int k = 1; k < kFewWarps; ++k) v += red[k * NT * 8 * 64 + u];
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
    if (a.x_scales && a.x_group == 0) y *= __ldg(a.x_scales + (m0 + m) * a.ldxs);
    if (a.b) y += bias;
    y = activate(y, a.act, a.alpha);
    const int64_t at = (m0 + m) * a.ldy + n0 + n;
    if (a.y_dtype == kF32) static_cast<float*>(a.Y)[at] = y;
    else if (a.y_dtype == kBF16) static_cast<bf16*>(a.Y)[at] = __float2bfloat16_rn(y);
    else static_cast<f16*>(a.Y)[at] = __float2half_rn(y);
  }
}

template <int XT, int NT, bool FINE>
int launch_few(Params p, cudaStream_t st) {
  auto kernel = dense_w4_few_kernel<XT, NT, FINE>;
  p.rows = NT * 8 / XRow<XT>::kParts;
  const int64_t tiles = p.a.w.strips();
  const int64_t chunks = (p.a.M + p.rows - 1) / p.rows;
  if (chunks > 65535) return kErrTooLarge;
  // CTAs that share K: the fewest waves of the GPU's 148 * W4OCC CTAs, each as
  // long as a warp's blocks and kFixed of setting up and adding.
  constexpr int kFixed = 4;
  int best = 0;
  int64_t least = INT64_MAX;
  for (int l = 0; l <= 3; ++l) {
    const int64_t waves = ((tiles * chunks << l) + 148 * W4OCC - 1) / (148 * W4OCC);
    const int64_t blocks = (p.kblocks + (kFewWarps << l) - 1) / (kFewWarps << l);
    const int64_t cost = waves * (blocks + kFixed);
    if (cost < least) {
      least = cost;
      best = l;
    }
  }
  static const int force = getenv("W4C") ? atoi(getenv("W4C")) : -1;
  if (force >= 0) best = force;
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
  const cudaError_t e0 = allow_shared(reinterpret_cast<const void*>(kernel));
  if (e0 != cudaSuccess) return launch_result(e0);
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

template <int XT, int NT, int MT, int WN, bool FINE>
int launch(Params p, cudaStream_t st) {
  constexpr int WK = kWarps / WN, COLS = NT * 8, ROWS = WN * MT * 16;
  auto kernel = dense_w4_kernel<XT, NT, MT, WN, FINE>;
  p.rows = COLS / XRow<XT>::kParts;
  const int64_t tiles = (p.a.w.N + ROWS - 1) / ROWS;
  const int64_t chunks = (p.a.M + p.rows - 1) / p.rows;
  if (chunks > 65535) return kErrTooLarge;
  // K is shared by the CTAs of a cluster until they fill the GPU twice or a
  // warp has less than one block of K.
  int C = 1;
  while (C < kMaxCluster && tiles * chunks * C < 148 * 2 && p.kblocks >= (int64_t)2 * C * WK) C *= 2;
  constexpr int kStage = 64 * 1024;
  const int64_t mine = (p.kblocks + C - 1) / C;
  p.stage_blocks = (int)std::max<int64_t>(
      WK, std::min<int64_t>((mine + WK - 1) / WK * WK, (kStage / COLS - 64) / 128 / WK * WK));
  const int smem = std::max(COLS * (p.stage_blocks * 128 + 64), WK * COLS * ROWS * 4);
  const cudaError_t e0 = allow_shared(reinterpret_cast<const void*>(kernel));
  if (e0 != cudaSuccess) return launch_result(e0);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * C), (unsigned)chunks);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  count_launch();
  return launch_result(e != cudaSuccess ? e : cudaGetLastError());
}

template <int XT, bool FINE>
int dispatch_rows(const Params& p, cudaStream_t st) {
  const int64_t cols = p.a.M * XRow<XT>::kParts;
  if (cols <= 8) return launch_few<XT, 1, FINE>(p, st);
  if (cols <= 16) return launch_few<XT, 2, FINE>(p, st);
  if (cols <= 32) return launch<XT, 4, 2, 2, FINE>(p, st);
  return launch<XT, 8, 2, 4, FINE>(p, st);
}

template <int XT>
int dispatch(const Params& p, cudaStream_t st) {
  const bool fine = p.a.w.group == 32 || p.a.x_group == 32;
  return fine ? dispatch_rows<XT, true>(p, st) : dispatch_rows<XT, false>(p, st);
}

unsigned grid_for(int64_t work) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((work + 255) / 256, 148 * 32));
}

}  // namespace

int dense_w4(const DenseW4Args& a, cudaStream_t st) {
  Params p;
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
    case kF32: return dispatch<kF32>(p, st);
    case kBF16: return dispatch<kBF16>(p, st);
    case kF16: return dispatch<kF16>(p, st);
    default: return dispatch<kE4M3>(p, st);
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
