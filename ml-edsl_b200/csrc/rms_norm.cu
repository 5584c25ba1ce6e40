// Root-mean-square norm of rows, with the residual's addition and an output
// of 8 bits (HBM-bound).
//
//   h = x + r                                  (r optional)
//   y = h / sqrt(mean(h^2) + eps) * w          (w optional)
//   q = e4m3(y / s),  s = max|y| / 448         over the row or over groups of
//                                              32, 64 or 128 columns
//
// h is summed in f32 and stays there until the end: y comes from the f32 sum,
// not from the h that is stored in x's type, and q from the f32 y, so each
// output is rounded once. The sum of squares is a tree over f32 partial sums
// of at most 32 terms.
#include <cuda_runtime.h>
#include <algorithm>
#include <atomic>
#include <cstdint>
#include "device_facts.h"
#include "dtype.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace b200 {

namespace {

constexpr float kE4M3Max = 448.0f;
// Outside these maxima 448 / max leaves the range of f32 or of the fast
// division.
constexpr float kTinyMax = 1e-30f, kHugeMax = 1e37f;

struct Sum {
  static __device__ __forceinline__ float id() { return 0.0f; }
  static __device__ __forceinline__ float op(float a, float b) { return a + b; }
};
struct Max {
  static __device__ __forceinline__ float id() { return 0.0f; }  // of absolute values
  static __device__ __forceinline__ float op(float a, float b) { return fmaxf(a, b); }
};

// Reduction over the TPR threads of a row. For TPR > 32 the CTA is one row;
// `sh` holds 32 floats and is used by one reduction at a time: the caller
// alternates between two.
template <class Op, int TPR>
__device__ __forceinline__ float row_reduce(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = Op::op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (TPR > 32) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < TPR / 32 ? sh[lane] : Op::id();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = Op::op(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  return v;
}

// How the rows lie: on 16 bytes; anyhow (element by element); or, rows of an
// odd length in a buffer that starts on 16 bytes, each with the same cut off
// 16 bytes in every tensor. A cut row's chunks are those of the memory, so
// that all but its first and last one are 16-byte accesses (4234x7710 f32 with
// residual to e4m3: 163 us element by element, 91 us cut; floor 65).
enum Rows { kAligned, kAnyhow, kCut };

// Chunks that lie outside the row altogether are told apart first: a thread may
// have several of them, and going through one element by element costs more
// than a whole one.
__device__ __forceinline__ bool outside(int64_t n, int vec, int64_t N) {
  return n >= N || n + vec <= 0;
}

// Elements [n, n + VEC) of a row as floats, 0 past N (and before 0).
template <class T, bool AL>
__device__ __forceinline__ void load_chunk(const T* row, int64_t n, int64_t N, float* f) {
  constexpr int VEC = Chunk<T>::kElems;
  if (AL && n >= 0 && n + VEC <= N) {
    // an ordinary load: h may be stored over x or over the residual
    unpack(*reinterpret_cast<const uint4*>(row + n), (const T*)nullptr, f);
  } else if (outside(n, VEC, N)) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = 0.0f;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = n + i >= 0 && n + i < N ? to_f32(row[n + i]) : 0.0f;
  }
}

template <class T, bool AL>
__device__ __forceinline__ void store_chunk(T* row, int64_t n, int64_t N, const float* f) {
  constexpr int VEC = Chunk<T>::kElems;
  if (AL && n >= 0 && n + VEC <= N) {
    // streaming: outputs do not push the rows that are still to be read out of
    // L2 (65536x4096 bf16 with residual: 370 -> 357 us; loads gain nothing)
    __stcs(reinterpret_cast<uint4*>(row + n), pack(f, (const T*)nullptr));
  } else if (!outside(n, VEC, N)) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (n + i >= 0 && n + i < N) row[n + i] = from_f32<T>(f[i]);
  }
}

// VEC elements of w (T or f32), 1 without one.
template <class T, bool AL>
__device__ __forceinline__ void load_weight(const RmsNormArgs& p, int64_t n, float* f) {
  constexpr int VEC = Chunk<T>::kElems;
  if (!p.w) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = 1.0f;
  } else if (sizeof(T) == 4 || !p.w_f32) {
    load_chunk<T, AL>(static_cast<const T*>(p.w), n, p.N, f);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4)
      load_chunk<float, AL>(static_cast<const float*>(p.w), n + i, p.N, f + i);
  }
}

// The weights of a chunk of a row that is cut off 16 bytes, n + cut a multiple of
// VEC: out of the two aligned chunks of w that hold them (16384x5003 bf16 138 ->
// 131 us, 4213x11811 bf16 with residual 125 -> 119; without weights 109 and 105).
template <class T>
__device__ __forceinline__ void load_weight_cut(const RmsNormArgs& p, int64_t n, int cut, float* f) {
  constexpr int VEC = Chunk<T>::kElems;
  const int64_t end = n + cut + VEC;  // of the second one
  if (!p.w || (sizeof(T) == 2 && p.w_f32) || reinterpret_cast<uintptr_t>(p.w) % 16 != 0 || n < 0 ||
      end > p.N)
    return load_weight<T, false>(p, n, f);
  if (cut == 0) return load_weight<T, true>(p, n, f);
  const uint4* at = reinterpret_cast<const uint4*>(static_cast<const T*>(p.w) + (end - 2 * VEC));
  const uint4 a = at[0], b = at[1];
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  // 16 bytes from `from` on, by two words, one and a half
  const int from = 16 - cut * (int)sizeof(T);
  uint32_t u[6], v[5], o[4];
#pragma unroll
  for (int i = 0; i < 6; ++i) u[i] = from & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = from & 4 ? u[i + 1] : u[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(v[i], v[i + 1], (from & 2) * 8);
  unpack(make_uint4(o[0], o[1], o[2], o[3]), (const T*)nullptr, f);
}

// Codes of VEC values; factor(i) scales value i into e4m3's range.
template <int VEC, bool AL, class Factor>
__device__ __forceinline__ void store_codes(uint8_t* row, int64_t n, int64_t N, const float* y,
                                            Factor factor) {
  if (outside(n, VEC, N)) return;
  float c[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) c[i] = factor(i, y[i]);
  uint32_t w[VEC / 4];
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i) {
    const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(c[4 * i], c[4 * i + 1]),
                                                __NV_SATFINITE, __NV_E4M3);
    const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(c[4 * i + 2], c[4 * i + 3]),
                                                __NV_SATFINITE, __NV_E4M3);
    w[i] = a | b << 16;
  }
  if (AL && n >= 0 && n + VEC <= N) {
    if constexpr (VEC == 8)
      *reinterpret_cast<uint2*>(row + n) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(row + n) = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (n + i >= 0 && n + i < N) row[n + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
  }
}

// The scale of a row or group whose largest absolute value is `most`, and the
// factors that bring its values into range: 448 / most, with the two units in
// the last place of the fast division. Where most is too small or too large
// for that the values are moved by 2^100 first.
struct Scale {
  float scale, pre, inv;
  __device__ __forceinline__ explicit Scale(float most) {
    const float s = most * (1.0f / kE4M3Max);
    scale = s > 0.0f ? s : 1.0f;  // nothing but zeros (or underflow): codes of y itself
    pre = 1.0f;
    inv = s > 0.0f ? __fdividef(kE4M3Max, most) : 1.0f;
    if (!(most > kTinyMax && most < kHugeMax) && s > 0.0f) {
      pre = most < 1.0f ? 1.26765060e30f : 7.88860905e-31f;
      inv = __fdividef(1.0f, scale * pre);
    }
  }
  __device__ __forceinline__ float operator()(float y) const { return y * pre * inv; }
};

// The largest of a group's absolute values: the group's lanes are
// group / VEC consecutive ones.
__device__ __forceinline__ float group_max(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// y = (h * pre) * inv with inv = 1 / sqrt(mean of squares + eps) and pre = 1.
// `squares(c)` sums the squares of h * c over the row again, where those of h leave
// f32's range: |h| > 1.8e19, with c = 2^-100, which then goes to both factors so
// that neither leaves the range (an h that pre makes subnormal has a y that is);
// or |h| < 2^-45 with an eps that does not hide what its squares lose, with
// c = 2^60.
struct Factor {
  float pre, inv;
};
template <class Fn>
__device__ __forceinline__ Factor factor(float ss, float N, float eps, Fn squares) {
  const float tiny = 0x1p-90f;
  const bool small = ss < tiny && eps < tiny;
  if (ss < __int_as_float(0x7f800000) && !small) return {1.0f, 1.0f / sqrtf(ss / N + eps)};
  const float c = small ? 0x1p60f : 0x1p-100f;
  const float inv = 1.0f / sqrtf(squares(c) / N + eps * c * c);
  return small ? Factor{c, inv} : Factor{0x1p-48f, 0x1p-52f * inv};
}

// A chunk of x (and of r) as it lies in memory, or as floats where it has to be
// read element by element.
template <class T, bool AL>
struct RawChunk {
  uint4 v;
  __device__ __forceinline__ void load(const T* row, int64_t n, int64_t N) {
    constexpr int VEC = Chunk<T>::kElems;
    if (n >= 0 && n + VEC <= N) {
      v = *reinterpret_cast<const uint4*>(row + n);
    } else if (outside(n, VEC, N)) {
      v = make_uint4(0, 0, 0, 0);
    } else {
      float f[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = n + i >= 0 && n + i < N ? to_f32(row[n + i]) : 0.0f;
      v = pack(f, (const T*)nullptr);  // the values are T's: nothing is rounded
    }
  }
  __device__ __forceinline__ void floats(float* f) const { unpack(v, (const T*)nullptr, f); }
};
template <class T>
struct RawChunk<T, false> {
  float v[Chunk<T>::kElems];
  __device__ __forceinline__ void load(const T* row, int64_t n, int64_t N) {
    if (n >= N) {
#pragma unroll
      for (int i = 0; i < Chunk<T>::kElems; ++i) v[i] = 0.0f;
      return;
    }
#pragma unroll
    for (int i = 0; i < Chunk<T>::kElems; ++i) v[i] = n + i < N ? to_f32(row[n + i]) : 0.0f;
  }
  __device__ __forceinline__ void floats(float* f) const {
#pragma unroll
    for (int i = 0; i < Chunk<T>::kElems; ++i) f[i] = v[i];
  }
};

// CTAs that the compiler has to leave registers for: cut rows take more of them
// than pays (1000x1001 f32 3.4 -> 3.1 us).
constexpr int ctas_at_once(int tpr, Rows how) {
  return how != kCut ? 0 : tpr == 32 ? 4 : 1024 / tpr;  // 0: the compiler's choice
}

// Rows by TPR threads each, E chunks of 16 bytes a thread: chunk e * TPR + t of
// a row is thread t's e-th. A row is read once and stays in registers; the next
// row of the CTA is on its way while one is summed, scaled and stored.
template <class T, int TPR, int E, Rows HOW>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, ctas_at_once(TPR, HOW))
    rms_norm_kernel(const __grid_constant__ RmsNormArgs p) {
  constexpr int VEC = Chunk<T>::kElems;
  constexpr bool AL = HOW != kAnyhow, WHOLE = HOW == kAligned;
  constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
  __shared__ float sh[2][3][32];  // in turn, for one row and the next
  constexpr int kRowGroups = ROWS > 1 ? 33 : 513;  // of 32 columns
  __shared__ uint32_t sh_groups[2][HOW == kCut ? ROWS * kRowGroups : 1];
  const int t = threadIdx.x % TPR;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  pdl_trigger();
  pdl_wait();
  RawChunk<T, AL> xs[E], rs[E];
  auto cut_of = [&](int64_t m) { return HOW == kCut ? (int)(m * p.ldx & (VEC - 1)) : 0; };
  auto load_row = [&](int64_t m) {
    const int cut = cut_of(m);
    const T* x = static_cast<const T*>(p.X) + m * p.ldx;
#pragma unroll
    for (int e = 0; e < E; ++e) xs[e].load(x, (int64_t)(e * TPR + t) * VEC - cut, p.N);
    if (p.R) {
      const T* r = static_cast<const T*>(p.R) + m * p.ldr;
#pragma unroll
      for (int e = 0; e < E; ++e) rs[e].load(r, (int64_t)(e * TPR + t) * VEC - cut, p.N);
    }
  };
  if (m < p.M) load_row(m);
  if (HOW == kCut && p.group) {
    for (int g = threadIdx.x; g < ROWS * kRowGroups; g += blockDim.x) sh_groups[0][g] = 0;
    __syncthreads();
  }
  // rows of whole warps: TPR is 32 where a CTA has several
  for (int odd = 0; m < p.M; m += step, odd ^= 1) {
    const int cut = cut_of(m);
    float h[E][VEC];
#pragma unroll
    for (int e = 0; e < E; ++e) xs[e].floats(h[e]);
    if (p.R) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float f[VEC];
        rs[e].floats(f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[e][i] += f[i];
      }
    }
    if (m + step < p.M) load_row(m + step);
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < VEC; ++i) ss = fmaf(h[e][i], h[e][i], ss);
    ss = row_reduce<Sum, TPR>(ss, sh[odd][0]);
    const Factor f = factor(ss, (float)p.N, p.eps, [&](float c) {
      float s = 0.0f;
      for (int e = 0; e < E; ++e)
        for (int i = 0; i < VEC; ++i) s = fmaf(h[e][i] * c, h[e][i] * c, s);
      return row_reduce<Sum, TPR>(s, sh[odd][1]);
    });

    if (p.H) {
      T* hrow = static_cast<T*>(p.H) + m * p.ldh;
#pragma unroll
      for (int e = 0; e < E; ++e)
        store_chunk<T, AL>(hrow, (int64_t)(e * TPR + t) * VEC - cut, p.N, h[e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float w[VEC];
      if (HOW == kCut) load_weight_cut<T>(p, (int64_t)(e * TPR + t) * VEC - cut, cut, w);
      else load_weight<T, WHOLE>(p, (int64_t)(e * TPR + t) * VEC, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[e][i] = h[e][i] * f.pre * f.inv * w[i];
    }
    if (!p.scales) {
      T* y = static_cast<T*>(p.Y) + m * p.ldy;
#pragma unroll
      for (int e = 0; e < E; ++e)
        store_chunk<T, AL>(y, (int64_t)(e * TPR + t) * VEC - cut, p.N, h[e]);
      continue;
    }
    uint8_t* q = static_cast<uint8_t*>(p.Y) + m * p.ldy;
    float* s = p.scales + m * p.lds;
    float most[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      most[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) most[e] = fmaxf(most[e], fabsf(h[e][i]));
    }
    if (p.group == 0) {
      float all = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) all = fmaxf(all, most[e]);
      all = row_reduce<Max, TPR>(all, sh[odd][2]);
      const Scale scale(all);
      if (t == 0) s[0] = scale.scale;
#pragma unroll
      for (int e = 0; e < E; ++e)
        store_codes<VEC, AL>(q, (int64_t)(e * TPR + t) * VEC - cut, p.N, h[e],
                             [&](int, float y) { return scale(y); });
    } else if constexpr (HOW == kCut) {
      // a chunk's elements lie in up to two groups: maxima in shared memory
      // (of bits, whose order is that of absolute values)
      uint32_t* gm = sh_groups[odd] + threadIdx.x / TPR * kRowGroups;
      uint32_t* next = sh_groups[odd ^ 1] + threadIdx.x / TPR * kRowGroups;
      const int groups = (int)((p.N + p.group - 1) >> p.group_shift);
      if (TPR == 32) __syncwarp();  // wider rows met at their sum
      for (int g = t; g < groups; g += TPR) next[g] = 0;  // the row before has been read
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t n = (int64_t)(e * TPR + t) * VEC - cut;
        if (n >= p.N) continue;
        const int g0 = n < 0 ? 0 : (int)(n >> p.group_shift);
        const int in_first = (int)(((int64_t)(g0 + 1) << p.group_shift) - n);
        float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (i < in_first) m0 = fmaxf(m0, fabsf(h[e][i]));
          else m1 = fmaxf(m1, fabsf(h[e][i]));
        atomicMax(gm + g0, __float_as_uint(m0));
        if (in_first < VEC && g0 + 1 < groups) atomicMax(gm + g0 + 1, __float_as_uint(m1));
      }
      if (TPR > 32) __syncthreads();
      else __syncwarp();
      for (int g = t; g < groups; g += TPR) s[g] = Scale(__uint_as_float(gm[g])).scale;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t n = (int64_t)(e * TPR + t) * VEC - cut;
        if (n >= p.N) continue;
        const int g0 = n < 0 ? 0 : (int)(n >> p.group_shift);
        const int in_first = (int)(((int64_t)(g0 + 1) << p.group_shift) - n);
        const Scale a(__uint_as_float(gm[g0])), b(__uint_as_float(gm[min(g0 + 1, groups - 1)]));
        store_codes<VEC, AL>(q, n, p.N, h[e],
                             [&](int i, float y) { return i < in_first ? a(y) : b(y); });
      }
    } else {
      const int lanes = p.group / VEC;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t n = (int64_t)(e * TPR + t) * VEC;
        const Scale scale(group_max(most[e], lanes));
        if ((t & (lanes - 1)) == 0 && n < p.N) s[n >> p.group_shift] = scale.scale;
        store_codes<VEC, AL>(q, n, p.N, h[e], [&](int, float y) { return scale(y); });
      }
    }
  }
}

// Rows that do not fit the registers of one CTA. KEPT: h stays in shared memory,
// in f32, each thread's chunks its own (4096x16383 f32 144 -> 121 us, floor 82;
// 4096x32768 bf16 with residual to e4m3 396 -> 302 us, floor 143). Wider rows,
// one CTA of which would fill an SM (2048x50000 f32 kept 256 us, otherwise 178),
// are read once for the sum, once more for a row's maximum, and once to be
// written.
constexpr int kKeptBytes = 144 * 1024;
template <class T, Rows HOW, bool KEPT>
__global__ void __launch_bounds__(KEPT ? 512 : 1024)
    rms_norm_long_kernel(const __grid_constant__ RmsNormArgs p) {
  constexpr int VEC = Chunk<T>::kElems, TPR = KEPT ? 512 : 1024;
  extern __shared__ float4 kept[];  // [VEC / 4][chunk]
  constexpr bool AL = HOW != kAnyhow, WHOLE = HOW == kAligned;
  __shared__ float sh[3][32];
  const int t = threadIdx.x;
  const int64_t m = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  const T* x = static_cast<const T*>(p.X) + m * p.ldx;
  const T* r = p.R ? static_cast<const T*>(p.R) + m * p.ldr : nullptr;
  const int cut = HOW == kCut ? (int)(m * p.ldx & (VEC - 1)) : 0;
  const int64_t chunks = (p.N + cut + VEC - 1) / VEC;
  auto load_h = [&](int64_t c, float* h) {
    if (KEPT) {
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) {
        const float4 v = c < chunks ? kept[i * chunks + c] : make_float4(0, 0, 0, 0);
        h[4 * i] = v.x;
        h[4 * i + 1] = v.y;
        h[4 * i + 2] = v.z;
        h[4 * i + 3] = v.w;
      }
      return;
    }
    load_chunk<T, AL>(x, c * VEC - cut, p.N, h);
    if (r) {
      float f[VEC];
      load_chunk<T, AL>(r, c * VEC - cut, p.N, f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] += f[i];
    }
  };
  auto squares = [&](float c, float* buf) {
    float s = 0.0f;
    for (int64_t j = t; j < chunks; j += TPR) {
      float h[VEC];
      load_h(j, h);
      float part = 0.0f;  // at most VEC terms, then into the thread's sum
#pragma unroll
      for (int i = 0; i < VEC; ++i) part = fmaf(h[i] * c, h[i] * c, part);
      s += part;
    }
    return row_reduce<Sum, TPR>(s, buf);
  };
  float ss = 0.0f;
  if (KEPT) {
    constexpr int U = 4;  // chunks that a thread has under way
    for (int64_t j0 = t; j0 < chunks; j0 += U * TPR) {
      RawChunk<T, AL> xs[U], rs[U];
#pragma unroll
      for (int u = 0; u < U; ++u) xs[u].load(x, (j0 + u * TPR) * VEC - cut, p.N);
      if (r) {
#pragma unroll
        for (int u = 0; u < U; ++u) rs[u].load(r, (j0 + u * TPR) * VEC - cut, p.N);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t c = j0 + u * TPR;
        if (c >= chunks) break;
        float h[VEC];
        xs[u].floats(h);
        if (r) {
          float f[VEC];
          rs[u].floats(f);
#pragma unroll
          for (int i = 0; i < VEC; ++i) h[i] += f[i];
        }
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) part = fmaf(h[i], h[i], part);
        ss += part;
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i)
          kept[i * chunks + c] = make_float4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
      }
    }
    ss = row_reduce<Sum, TPR>(ss, sh[0]);
  } else {
    ss = squares(1.0f, sh[0]);
  }
  const Factor f =
      factor(ss, (float)p.N, p.eps, [&](float c) { return squares(c, sh[1]); });
  float all = 0.0f;
  if (p.scales && p.group == 0) {
    for (int64_t j = t; j < chunks; j += TPR) {
      float h[VEC], w[VEC];
      load_h(j, h);
      if (HOW == kCut) load_weight_cut<T>(p, j * VEC - cut, cut, w);
      else load_weight<T, WHOLE>(p, j * VEC, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) all = fmaxf(all, fabsf(h[i] * f.pre * f.inv * w[i]));
    }
    all = row_reduce<Max, TPR>(all, sh[2]);
    if (t == 0) p.scales[m * p.lds] = Scale(all).scale;
  }
  // whole warps take part in every step: a group's lanes exchange their maxima
  for (int64_t j0 = 0; j0 < chunks; j0 += TPR) {
    const int64_t n = (j0 + t) * VEC - cut;
    float h[VEC], w[VEC];
    load_h(j0 + t, h);
    if (HOW == kCut) load_weight_cut<T>(p, n, cut, w);
    else load_weight<T, WHOLE>(p, n, w);
    if (p.H) store_chunk<T, AL>(static_cast<T*>(p.H) + m * p.ldh, n, p.N, h);
#pragma unroll
    for (int i = 0; i < VEC; ++i) h[i] = h[i] * f.pre * f.inv * w[i];
    if (!p.scales) {
      store_chunk<T, AL>(static_cast<T*>(p.Y) + m * p.ldy, n, p.N, h);
      continue;
    }
    float most = all;
    if (p.group) {
      most = 0.0f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) most = fmaxf(most, fabsf(h[i]));
      most = group_max(most, p.group / VEC);
    }
    const Scale s(most);
    if (p.group && n % p.group == 0 && n < p.N) p.scales[m * p.lds + (n >> p.group_shift)] = s.scale;
    store_codes<VEC, AL>(static_cast<uint8_t*>(p.Y) + m * p.ldy, n, p.N, h,
                         [&](int, float y) { return s(y); });
  }
}

// Launches `kernel`, which may start early (it waits for the kernel before it
// where it first reads memory).
template <class Kernel>
cudaError_t launch_kernel(Kernel kernel, unsigned grid, int threads, int smem,
                          const RmsNormArgs& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <class T, int TPR, int E, Rows HOW>
cudaError_t launch(const RmsNormArgs& p, cudaStream_t st) {
  constexpr int ROWS = TPR < 128 ? 128 / TPR : 1, THREADS = TPR < 128 ? 128 : TPR;
  auto kernel = rms_norm_kernel<T, TPR, E, HOW>;
  // as many CTAs as fit, each with the rows that fall to it
  static PerDevice<int> resident;
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int per_sm = resident.of(dev, [&] {
    return ask_or(
        1,
        [&](int* n) {
          return cudaOccupancyMaxActiveBlocksPerMultiprocessor(n, kernel, THREADS, 0) ==
                 cudaSuccess;
        },
        [] { cudaGetLastError(); });
  });
  const int64_t grid = std::min<int64_t>((p.M + ROWS - 1) / ROWS, (int64_t)148 * per_sm);
  return launch_kernel(kernel, (unsigned)grid, THREADS, 0, p, st);
}

template <class T, Rows HOW>
cudaError_t launch_long(const RmsNormArgs& p, bool anyhow, cudaStream_t st) {
  if constexpr (HOW == kCut) {
    if (anyhow) return launch_long<T, kAnyhow>(p, false, st);
  }
  constexpr int VEC = Chunk<T>::kElems;
  const int64_t bytes = ((p.N + VEC - 1 + (HOW == kCut ? VEC - 1 : 0)) / VEC) * VEC * 4;
  if (bytes > kKeptBytes)
    return launch_kernel(rms_norm_long_kernel<T, HOW, false>, (unsigned)p.M, 1024, 0, p, st);
  auto kernel = rms_norm_long_kernel<T, HOW, true>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_shared(reinterpret_cast<const void*>(kernel), allowed);
  return e != cudaSuccess ? e : launch_kernel(kernel, (unsigned)p.M, 512, (int)bytes, p, st);
}

template <class T, Rows HOW>
cudaError_t dispatch(const RmsNormArgs& p, cudaStream_t st) {
  constexpr int VEC = Chunk<T>::kElems;
  const int64_t c = (p.N + (HOW == kCut ? VEC - 1 : 0) + VEC - 1) / VEC;
  // Few rows: time is latency, so a thread has one chunk (148x800 bf16, plain and
  // with residual to e4m3: 1.9 and 2.2 us, with four chunks 3.0 and 4.4;
  // 148x4096: 2.1 and 2.6, with two chunks 2.4 and 3.0). More rows than CTAs
  // stay at once: what counts is how many rows are under way, so a row has the
  // fewest threads that hold it with two chunks each, or four of a warp
  // (8192x800: 8.8 and 16.0 us, with 128 threads 13.1 and 22.3; 1024x800, which
  // all run at once: 3.6 and 5.1 us, with 128 threads 2.8 and 4.0). The steps
  // between the powers of two: 8192x2056 25.4 -> 20.5 us, 8192x4104 48.8 -> 41.1,
  // 8192x8200 96.8 -> 84.5. Four chunks of 1024 threads are slower than
  // rows in shared memory (4096x32768 bf16 216 and 179 us).
  const bool few = p.M <= 148, wave = p.M <= 148 * 8;
  if (c <= 32) return launch<T, 32, 1, HOW>(p, st);
  if (c <= 256 && few) return launch<T, 256, 1, HOW>(p, st);
  if (c <= 512 && few) return launch<T, 512, 1, HOW>(p, st);
  if (c <= 128 && !wave) return launch<T, 32, 4, HOW>(p, st);
  if (c <= 256) return launch<T, 128, 2, HOW>(p, st);
  if (c <= 384) return launch<T, 192, 2, HOW>(p, st);
  if (c <= 512) return launch<T, 256, 2, HOW>(p, st);
  if (c <= 768) return launch<T, 384, 2, HOW>(p, st);
  if (c <= 1024) return launch<T, 512, 2, HOW>(p, st);
  if (c <= 1536) return launch<T, 768, 2, HOW>(p, st);
  if (c <= 2048) return launch<T, 1024, 2, HOW>(p, st);
  // groups of cut rows: element by element
  return launch_long<T, HOW>(p, HOW == kCut && p.group, st);
}

template <class T>
cudaError_t dispatch_aligned(const RmsNormArgs& p, cudaStream_t st) {
  auto ok = [](const void* q, int64_t ld, int64_t elems, int bytes) {
    return (reinterpret_cast<uintptr_t>(q) % bytes) == 0 && ld % elems == 0;
  };
  constexpr int VEC = Chunk<T>::kElems;
  const bool al = ok(p.X, p.ldx, VEC, 16) && (!p.R || ok(p.R, p.ldr, VEC, 16)) &&
                  (!p.H || ok(p.H, p.ldh, VEC, 16)) && (!p.w || ok(p.w, VEC, VEC, 16)) &&
                  (p.scales ? ok(p.Y, p.ldy, VEC, VEC) : ok(p.Y, p.ldy, VEC, 16));
  if (al) return dispatch<T, kAligned>(p, st);
  auto same = [](const void* q, int64_t ld, int64_t ldx, int bytes) {
    return (reinterpret_cast<uintptr_t>(q) % bytes) == 0 && (ld - ldx) % VEC == 0;
  };
  const bool cut = same(p.X, p.ldx, p.ldx, 16) &&
                   (!p.R || same(p.R, p.ldr, p.ldx, 16)) && (!p.H || same(p.H, p.ldh, p.ldx, 16)) &&
                   same(p.Y, p.ldy, p.ldx, p.scales ? VEC : 16);
  return cut ? dispatch<T, kCut>(p, st) : dispatch<T, kAnyhow>(p, st);
}

}  // namespace

int rms_norm(const RmsNormArgs& p, int dtype, cudaStream_t st) {
  const cudaError_t e = dtype == kF32    ? dispatch_aligned<float>(p, st)
                        : dtype == kBF16 ? dispatch_aligned<bf16>(p, st)
                                         : dispatch_aligned<f16>(p, st);
  count_launch();
  return launch_result(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace b200
