// Shared by the 4-bit dense layer's kernels (dense_w4.cu, dense_w4_tc.cu): the
// packed layout, the operands' types and the staging of activations.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include "device_facts.h"
#include "dtype.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace b200 {

constexpr int kBlockK = 64;     // k of one packed block
constexpr int kStripN = 64;     // columns of one strip

// Place of column n (within its strip) among a group's 64 scales or zeros:
// lane group g = n % 8 reads its eight values together.
__host__ __device__ __forceinline__ int column_place(int n) { return (n & 7) * 8 + (n >> 3); }

// (a & b) | c in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// The types of the product's operands. A weight enters the product as
// (q - z) / kUp and its sums are multiplied by kUp at the end, both exactly: with
// an x of f32's range, 128 products of up to 15 x have to fit f32 before the scale
// is applied. x of f16 and e4m3 stays far below it.
struct MmaBF16 {
  static constexpr uint32_t kMagic = 0x3d003d00u;  // (128 + q) / 4096 in bf16: q in the low bits
  static constexpr float kUp = 4096.0f;
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
  static constexpr float kUp = 1.0f;
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

// How rows of X become operand columns: kParts columns for a row. load() takes
// 8 consecutive elements of a row from column k on, 0 from `end` on, into
// registers (load_whole(): aligned ones, all there); stage() makes 16 bytes for each column of them.
template <int XT>
struct XRow;
template <>
struct XRow<kBF16> {
  using Mma = MmaBF16;
  using Raw = uint4;
  static constexpr int kParts = 1, kBytes = 2;
  static __device__ __forceinline__ Raw load_whole(const char* row, int64_t k) {
    return __ldg(reinterpret_cast<const uint4*>(row + k * 2));
  }
  static __device__ __forceinline__ Raw load(const char* row, int64_t k, int64_t end,
                                             bool aligned) {
    const uint16_t* e = reinterpret_cast<const uint16_t*>(row) + k;
    if (aligned && k + 8 <= end) return load_whole(row, k);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (k + 2 * i < end ? __ldg(e + 2 * i) : 0u) |
             (k + 2 * i + 1 < end ? (uint32_t)__ldg(e + 2 * i + 1) : 0u) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ void stage(const Raw& r, uint4 (&out)[1]) { out[0] = r; }
};
template <>
struct XRow<kF16> : XRow<kBF16> {
  using Mma = MmaF16;
};
template <>
struct XRow<kE4M3> {
  using Mma = MmaF16;
  using Raw = uint2;
  static constexpr int kParts = 1, kBytes = 1;
  static __device__ __forceinline__ Raw load_whole(const char* row, int64_t k) {
    return __ldg(reinterpret_cast<const uint2*>(row + k));
  }
  static __device__ __forceinline__ Raw load(const char* row, int64_t k, int64_t end,
                                             bool aligned) {
    const uint8_t* e = reinterpret_cast<const uint8_t*>(row) + k;
    if (aligned && k + 8 <= end) return load_whole(row, k);
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < end) w[i >> 2] |= (uint32_t)__ldg(e + i) << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
  }
  static __device__ __forceinline__ void stage(const Raw& r, uint4 (&out)[1]) {
    const uint32_t in[2] = {r.x, r.y};
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          (__nv_fp8x2_storage_t)(in[i >> 1] >> (16 * (i & 1)) & 0xffffu), __NV_E4M3);
      w[i] = h.x | (uint32_t)h.y << 16;
    }
    out[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct XRow<kF32> {
  using Mma = MmaBF16;
  struct Raw {
    uint4 a, b;
  };
  static constexpr int kParts = 3, kBytes = 4;
  static __device__ __forceinline__ Raw load_whole(const char* row, int64_t k) {
    const uint4* e = reinterpret_cast<const uint4*>(row + k * 4);
    return {__ldg(e), __ldg(e + 1)};
  }
  static __device__ __forceinline__ Raw load(const char* row, int64_t k, int64_t end,
                                             bool aligned) {
    const uint32_t* e = reinterpret_cast<const uint32_t*>(row) + k;
    if (aligned && k + 8 <= end) return load_whole(row, k);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = k + i < end ? __ldg(e + i) : 0u;
    return {make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
  }
  // x = hi + mid + lo, each the leading 8 bits of what is left (cut, so that
  // no part rounds up out of range). Infinities and NaN travel in hi.
  static __device__ __forceinline__ void stage(const Raw& r, uint4 (&out)[3]) {
    const uint32_t e[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t p[3][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = e[2 * i + h];
        const bool finite = (x & 0x7f800000u) != 0x7f800000u;
        const bool nan = !finite && (x & 0x007fffffu);
        p[0][h] = nan ? 0x7fc00000u : x;
        const float rest = __uint_as_float(x) - __uint_as_float(x & 0xffff0000u);
        const uint32_t mid = __float_as_uint(rest);
        const uint32_t lo = __float_as_uint(rest - __uint_as_float(mid & 0xffff0000u));
        p[1][h] = finite ? mid : 0u;
        p[2][h] = finite ? lo : 0u;
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) w[q][i] = __byte_perm(p[q][0], p[q][1], 0x7632);  // upper halves
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) out[q] = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
  }
};

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

// `bytes` (0 to 16) of them, zeros for the rest.
__device__ __forceinline__ void cp_async16_fill(void* smem, const void* global, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(global),
               "r"(bytes)
               : "memory");
}

// Brings `bytes` (a multiple of 16) at a 16-byte aligned address into L2.
__device__ __forceinline__ void prefetch_l2_bulk(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// Brings a strip's weights of blocks [b0, b1) of K into L2, by one thread: scales
// and zeros (64 and 16 KB at most) and, if asked, codes (128 KB at most), each
// contiguous there. Only L2: the kernel before in the stream may still be writing
// them. 16x11008x4096 with zeros 20.0 -> 16.5 us; the codes of the tensor core's
// kernel are copied far enough ahead as it is (64x8192x8192 22.9 us, prefetched
// 23.5).
__device__ __forceinline__ void prefetch_strip(const W4Params& p, int64_t strip, int b0, int b1,
                                               bool codes) {
  if (b0 >= b1) return;
  if (codes)
    prefetch_l2_bulk(p.codes + (strip * p.kblocks + b0) * 128, (uint32_t)min(b1 - b0, 64) * 2048u);
  const int last = min((int)p.a.w.K, b1 * kBlockK) - 1;
  const int64_t g0 = p.group_of(b0 * kBlockK), g1 = p.group_of(last) + 1;
  const int64_t at = (strip * p.groups + g0) * 64, elems = min((int64_t)(g1 - g0) * 64, (int64_t)16384);
  const int bytes = p.a.w.s_dtype == kF32 ? 4 : 2;
  prefetch_l2_bulk(p.scales + at * bytes, (uint32_t)(elems * bytes));
  if (p.zeros) prefetch_l2_bulk(p.zeros + at, (uint32_t)elems);
}

// How many CTAs of a kernel run at once in clusters of 1, 2, 4 and 8. GPUs differ
// in how many clusters fit, so the driver is asked, once a kernel and device.
struct Capacity {
  int64_t ctas[4];
};
Capacity capacity_of(const void* kernel, int threads, int smem);

// The log2 of the CTAs that share K, of `tiles` CTAs' work each `kblocks` long
// that `warps` warps split: the fewest waves, each as long as a warp's blocks
// and `fixed` of setting up and adding. Clusters of 8 take more waves than
// their number of CTAs lets expect (16x16384x2048 bf16: 22.3 us, in clusters of
// 4 18.4, alone 61; 16x4096x512: 5.3 us, in fours 7.0).
int choose_cluster(const Capacity& capacity, int64_t tiles, int64_t kblocks, int warps, int fixed);

// Many rows, on the tensor core (dense_w4_tc.cu).
int dense_w4_tc(const W4Params& p, int* status, cudaStream_t st);

}  // namespace b200
