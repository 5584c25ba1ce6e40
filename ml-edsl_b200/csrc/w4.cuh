// Shared by the 4-bit dense layer's kernels (dense_w4.cu, dense_w4_tc.cu): the
// packed layout, the operands' types and the staging of activations.
#pragma once
#include <cuda_runtime.h>
#include <atomic>
#include <cstdint>
#include "dtype.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace b200 {

constexpr int kBlockK = 64;     // k of one packed block
constexpr int kStripN = 64;     // columns of one strip
constexpr int kMaxCluster = 8;  // CTAs that share K

// Place of column n (within its strip) among a group's 64 scales or zeros:
// lane group g = n % 8 reads its eight values together.
__host__ __device__ __forceinline__ int column_place(int n) { return (n & 7) * 8 + (n >> 3); }

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

// A call's arguments and what the host derives from them.
struct W4Params {
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

// Lets `kernel` use 200 KB of dynamic shared memory on the current device.
// `allowed`: one bit a device that has been told.
cudaError_t allow_shared(const void* kernel, std::atomic<uint64_t>& allowed);

// Many rows, on the tensor core (dense_w4_tc.cu).
int dense_w4_tc(const W4Params& p, int* status, cudaStream_t st);

}  // namespace b200
