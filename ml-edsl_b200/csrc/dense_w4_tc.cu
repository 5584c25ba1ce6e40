// The 4-bit dense layer for more rows than dense_w4.cu's kernel takes at once,
// on the tensor core: tcgen05.mma with the weights as the 128-row operand, in
// TMEM, and the rows of X as its columns, in shared memory.
//
// With W^T as the first operand its 128 rows are columns of W, so a tile of 16
// to 128 rows of X fills the instruction. The codes go from HBM to registers,
// become bf16 or f16 there (the same fragments and the same two instructions a
// pair as in dense_w4.cu) and are stored to TMEM, never to shared memory.
//
// A CTA has 128 columns of W, up to NC operand columns and its part of K (the
// CTAs of a cluster share K), and 13 warps:
//   0-7   two sets of four, a set for every other block of 64 of K: codes
//         (copied ahead by the lanes that use them) to TMEM; then the sums of
//         a unit of K out of TMEM, times its scale, into registers, each set
//         half of the columns
//   8-11  activations, one block ahead in registers, into shared memory
//   12    issues the products
// A unit is what one scale covers, at most 128 of K: products are exact, the
// tensor core sums 8 k16 steps at most, and the rest is added in f32 as for
// few rows. Every wait is bounded; one that runs out ends all roles and is
// reported by b200_stream_sync.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstdint>
#include <cstdlib>
#include "w4.cuh"

namespace cg = cooperative_groups;

namespace b200 {

namespace {

constexpr int kTileN = 128;
constexpr int kStages = 4;         // blocks of K between the roles
constexpr int kWorkers = 8;        // warps that expand codes and fold sums
constexpr int kStagers = 4;        // warps that bring activations
constexpr int kThreads = (kWorkers + kStagers + 1) * 32;
constexpr int kCodeDepth = 4;      // blocks that a lane copies ahead
constexpr int kTmemA = kStages * 32;  // TMEM columns of the expanded weights

// TMEM columns: 256 where two CTAs fit an SM.
__host__ __device__ constexpr int tmem_columns(int NC) { return NC <= 64 ? 256 : 512; }
__host__ __device__ constexpr int sum_buffers(int NC) {
  return (tmem_columns(NC) - kTmemA) / NC < 4 ? (tmem_columns(NC) - kTmemA) / NC : 4;
}

struct Barriers {
  uint64_t full[kStages];   // codes and activations of a block are in place
  uint64_t empty[kStages];  // its products are done
  uint64_t sums[4];         // the sums of a unit are complete
  uint64_t taken[4];        // and have been read
  uint32_t tmem;
  int abort_flag;
};

template <int XT, int NC, int UNIT>
__global__ void __launch_bounds__(kThreads, NC <= 64 ? 2 : 1)
    dense_w4_tc_kernel(const __grid_constant__ W4Params p, int* status) {
  using X = XRow<XT>;
  using Mma = typename X::Mma;
  using Raw = typename X::Raw;
  constexpr int PARTS = X::kParts, HALF = NC / 2, SUMS = sum_buffers(NC);
  constexpr bool BF16 = Mma::kMagic == MmaBF16::kMagic;
  constexpr uint32_t kIdesc = idesc_16bit_f32(BF16, kTileN, NC);
  extern __shared__ __align__(1024) char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int log_c = p.log_cluster, C = 1 << log_c, rank = blockIdx.x & (C - 1);
  if (C > 1) cluster.barrier_arrive();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const DenseW4Args& a = p.a;
  const int64_t n0 = (int64_t)(blockIdx.x >> log_c) * kTileN;
  const int64_t m0 = (int64_t)blockIdx.y * p.rows;
  const int mrows = (int)min((int64_t)p.rows, a.M - m0);
  const int K = (int)a.w.K, kblocks = (int)p.kblocks;
  // blocks of K of this CTA, in whole units
  constexpr int UB = UNIT / 64 > 0 ? UNIT / 64 : 1;  // blocks of a unit
  const int groups_of_blocks = (kblocks + UB - 1) / UB;
  const int b0 = (int)((int64_t)groups_of_blocks * rank >> log_c) * UB;
  const int b1 = min(kblocks, (int)((int64_t)groups_of_blocks * (rank + 1) >> log_c) * UB);
  const int nb = b1 - b0;
  const int units = nb > 0 ? (min(K, b1 * kBlockK) - b0 * kBlockK + UNIT - 1) / UNIT : 0;

  // shared memory: activations (swizzled tiles of 64 k by NC columns), codes,
  // what the cluster's CTAs send, barriers
  char* xring = smem;
  char* cring = xring + kStages * NC * 128;
  float* recv = reinterpret_cast<float*>(cring + kWorkers * kCodeDepth * 1024);
  Barriers* bar = reinterpret_cast<Barriers*>(reinterpret_cast<char*>(recv) + p.recv_bytes);
  volatile int* abort_flag = &bar->abort_flag;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar->full[i], kWorkers / 2 + kStagers);
      mbar_init(&bar->empty[i], 1);
    }
    for (int i = 0; i < SUMS; ++i) {
      mbar_init(&bar->sums[i], 1);
      mbar_init(&bar->taken[i], kWorkers);
    }
    bar->abort_flag = 0;
    fence_barrier_init();
  }
  pdl_wait();
  if (wid == kWorkers + kStagers) tmem_alloc(&bar->tmem, tmem_columns(NC));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // only now: a kernel that starts early must not take TMEM that a CTA of this
  // one still waits for
  pdl_trigger();
  const uint32_t tmem = bar->tmem, tmem_sums = tmem + kTmemA;

  float total[HALF];
#pragma unroll
  for (int i = 0; i < HALF; ++i) total[i] = 0.0f;
  const int quarter = wid & 3, set = wid >> 2;  // of a worker

  if (wid < kWorkers) {
    const int64_t strip = n0 / kStripN + (quarter >> 1);
    const bool live = strip * kStripN < a.w.N;
    const int mt0 = (quarter & 1) * 2, g = lane >> 2;
    // ---- codes: two 16-column pieces of the quarter's 32 columns
    uint4* mine = reinterpret_cast<uint4*>(cring) + wid * (kCodeDepth * 64) + lane;
    const uint4* codes = p.codes + ((strip * kblocks + b0 + set) * 4 + mt0) * 32 + lane;
    int fetched = set;
    auto fetch = [&](int slot) {
      if (live && fetched < nb) {
        cp_async16(mine + slot * 64, codes);
        cp_async16(mine + slot * 64 + 32, codes + 32);
      }
      codes += 2 * 128;
      fetched += 2;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kCodeDepth; ++i) fetch(i);
    const uint8_t* zeros = p.zeros ? p.zeros + strip * p.groups * 64 + g * 8 + mt0 * 2 : nullptr;
    uint32_t znext[UNIT == 32 ? 2 : 1] = {};
    auto fetch_zeros = [&](int i) {
      if (!zeros || !live || i >= nb) return;
#pragma unroll
      for (int sub = 0; sub < (UNIT == 32 ? 2 : 1); ++sub) {
        const int k = (b0 + i) * kBlockK + sub * 32;
        if (sub && k >= K) return;
        znext[sub] =
            __ldg(reinterpret_cast<const uint32_t*>(zeros + (int64_t)p.group_of(k) * 64));
      }
    };
    fetch_zeros(set);
    // ---- scales: this lane's column of W, for the unit that is folded next
    const int n = (quarter & 1) * 32 + lane;  // within the strip
    const int64_t scale_col = strip * p.groups * 64 + column_place(n);
    auto scale_of_unit = [&](int u) {
      const int k = b0 * kBlockK + u * UNIT;
      return live && u < units
                 ? load_as_f32(p.scales, a.w.s_dtype, scale_col + (int64_t)p.group_of(k) * 64)
                 : 0.0f;
    };
    float scale_next = scale_of_unit(0);

    bool ok = true;
    int folded = 0, slot = 0;
    auto fold = [&](int u) {
      const int buf = u % SUMS;
      if (!mbar_wait(&bar->sums[buf], (u / SUMS) & 1, status, kDevTimeoutAccum, abort_flag))
        return false;
      tc_fence_after();
      const float scale = scale_next;
      scale_next = scale_of_unit(u + 1);
      const uint32_t from = tmem_sums + ((uint32_t)(quarter * 32) << 16) + buf * NC + set * HALF;
      constexpr int STEP = HALF < 16 ? 8 : 16;
#pragma unroll
      for (int c = 0; c < HALF; c += STEP) {
        uint32_t v[STEP];
        if constexpr (STEP == 8) tmem_ld_32x32b_x8(from + c, v);
        else tmem_ld_32x32b_x16(from + c, v);
        tmem_ld_wait();
        if (XT == kE4M3 && a.x_group > 0) {
          const unsigned xg = (unsigned)(b0 * kBlockK + u * UNIT) / (unsigned)a.x_group;
#pragma unroll
          for (int i = 0; i < STEP; ++i) {
            const int m = set * HALF + c + i;
            const float xs = m < mrows ? __ldg(a.x_scales + (m0 + m) * a.ldxs + xg) : 0.0f;
            total[c + i] = fmaf(__uint_as_float(v[i]) * xs, scale, total[c + i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < STEP; ++i)
            total[c + i] = fmaf(__uint_as_float(v[i]), scale, total[c + i]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->taken[buf]);
      return true;
    };
    for (int i = set; i < nb && ok; i += 2) {
      const int stage = i % kStages;
      asm volatile("cp.async.wait_group %0;" ::"n"(kCodeDepth - 1) : "memory");
      uint4 w[2];
      w[0] = mine[slot * 64];
      w[1] = mine[slot * 64 + 32];
      uint32_t z[UNIT == 32 ? 2 : 1][4];
#pragma unroll
      for (int sub = 0; sub < (UNIT == 32 ? 2 : 1); ++sub)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          z[sub][q] = zeros ? __byte_perm(znext[sub], Mma::kMagic, 0x5050 | q * 0x0101)
                            : 0x00080008u | Mma::kMagic;
      fetch_zeros(i + 2);
      if (i >= kStages && !mbar_wait(&bar->empty[stage], (i / kStages - 1) & 1, status,
                                     kDevTimeoutEmpty, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t words[4] = {w[q].x, w[q].y, w[q].z, w[q].w};
        uint32_t f[16];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            f[4 * j + r] = Mma::sub(and_or(words[j] >> (4 * r), 0x000f000fu, Mma::kMagic),
                                    z[UNIT == 32 ? j >> 1 : 0][2 * q + (r & 1)]);
        tmem_st_16x128b_x8(tmem + ((uint32_t)(quarter * 32 + q * 16) << 16) + stage * 32, f);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->full[stage]);
      fetch(slot);  // the slot's codes have been used
      slot = (slot + 1) % kCodeDepth;
      // fold what is complete two blocks behind: the products of blocks that
      // both sets have expanded
      const int upto = min(units, UNIT == 32 ? 2 * (i - 1) : (i - 1) / UB);
      while (folded < upto && ok) ok = fold(folded++);
    }
    while (folded < units && ok) ok = fold(folded++);
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (wid < kWorkers + kStagers) {
    // ---- activations: pieces of 8 elements, 8 of a row and block; 16 bytes
    // of the column's 128 in shared memory, swizzled as the tensor core reads
    // them
    constexpr int PER = (NC / PARTS * 8 + kStagers * 32 - 1) / (kStagers * 32);
    const int st = tid - kWorkers * 32;
    const int c = st & 7, row0 = st >> 3, rows_step = kStagers * 4;
    const char* x = static_cast<const char*>(a.X) + m0 * a.ldx * X::kBytes;
    auto place = [&](int stage, int col) {
      return xring + stage * NC * 128 + col * 128 + ((c ^ (col & 7)) << 4);
    };
    auto room = [&](int i) {
      return i < kStages || mbar_wait(&bar->empty[i % kStages], (i / kStages - 1) & 1, status,
                                      kDevTimeoutEmpty, abort_flag);
    };
    auto post = [&](int i) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->full[i % kStages]);
    };
    if (X::kBytes == 2 && p.x_aligned) {
      // 16-bit rows are copied as they are, kAhead blocks ahead
      constexpr int kAhead = 2;
      for (int i = 0; i < nb + kAhead; ++i) {
        if (i < nb) {
          if (!room(i)) break;
          const int k = (b0 + i) * kBlockK + c * 8;
          const int bytes = max(0, min(16, (K - k) * 2));
#pragma unroll
          for (int u = 0; u < PER; ++u) {
            const int m = row0 + u * rows_step;
            if (m < mrows)
              cp_async16_fill(place(i % kStages, m), x + ((int64_t)m * a.ldx + (bytes ? k : 0)) * 2,
                              bytes);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (i >= kAhead) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
          post(i - kAhead);
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
      // others pass through registers, asked for one block ahead
      Raw next[PER];
      auto load = [&](int i) {
        if (i >= nb) return;
        const int64_t k = (int64_t)(b0 + i) * kBlockK + c * 8;
        if (p.x_aligned && (b0 + i + 1) * kBlockK <= K) {
#pragma unroll
          for (int u = 0; u < PER; ++u)  // rows past the last: the last again
            next[u] = X::load_whole(x + min(row0 + u * rows_step, mrows - 1) * a.ldx * X::kBytes, k);
        } else {
#pragma unroll
          for (int u = 0; u < PER; ++u)
            next[u] = X::load(x + min(row0 + u * rows_step, mrows - 1) * a.ldx * X::kBytes, k, K,
                              false);
        }
      };
      load(0);
      for (int i = 0; i < nb; ++i) {
        if (!room(i)) break;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          const int m = row0 + u * rows_step;
          if (m >= mrows) continue;
          uint4 out[PARTS];
          X::stage(next[u], out);
#pragma unroll
          for (int q = 0; q < PARTS; ++q)
            *reinterpret_cast<uint4*>(place(i % kStages, m * PARTS + q)) = out[q];
        }
        load(i + 1);
        post(i);
      }
    }
  } else if (lane == 0) {
    // ---- products
    bool ok = true;
    int u = 0;
    for (int i = 0; i < nb && ok; ++i) {
      const int stage = i % kStages;
      if (!mbar_wait(&bar->full[stage], (i / kStages) & 1, status, kDevTimeoutFull,
                     abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t bdesc = umma_desc_k<2, 1024>(smem_u32(xring + stage * NC * 128));
      const uint32_t at = tmem + stage * 32;
      constexpr int SUBS = UNIT == 32 ? 2 : 1, STEPS = 4 / SUBS;
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        if (u >= units) break;  // the second half of K's last block
        const int buf = u % SUMS;
        const bool first = UNIT < 128 || i % UB == 0;
        if (first && u >= SUMS &&
            !mbar_wait(&bar->taken[buf], (u / SUMS - 1) & 1, status, kDevTimeoutAccum,
                       abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
          const int step = sub * STEPS + k;
          umma_f16_ts(tmem_sums + buf * NC, at + step * 8, bdesc + step * 2, kIdesc,
                      !(first && k == 0));
        }
        if (UNIT < 128 || i % UB == UB - 1 || i == nb - 1) {
          umma_commit(&bar->sums[buf]);
          ++u;
        }
      }
      umma_commit(&bar->empty[stage]);
    }
    // the last arrival is in before shared memory goes
    if (ok && nb > 0)
      mbar_wait(&bar->empty[(nb - 1) % kStages], ((nb - 1) / kStages) & 1, status,
                kDevTimeoutEmpty, abort_flag);
  }

  // ---- the CTAs' parts of K: each 32 outputs of a row belong to one CTA of
  // the cluster, in turn
  const int outs = mrows * kTileN;
  const int slots = ((mrows * 4 + C - 1) >> log_c) * 32;
  if (C > 1) cluster.barrier_wait();  // every CTA of the cluster runs
  if (wid < kWorkers) {
#pragma unroll
    for (int c = 0; c < HALF; ++c) {
      const int col = set * HALF + c, m = col / PARTS, q = col - m * PARTS;
      if (m >= mrows) break;
      const int chunk = m * 4 + quarter;
      float* dst = recv + (rank * PARTS + q) * slots + (chunk >> log_c) * 32 + lane;
      *(C > 1 ? cluster.map_shared_rank(dst, chunk & (C - 1)) : dst) = total[c];
    }
  }
  tc_fence_before();
  if (C > 1) cluster.sync();
  else __syncthreads();
  tc_fence_after();
  if (wid == kWorkers + kStagers) tmem_dealloc(tmem, tmem_columns(NC));
  for (int u = tid; u < slots; u += kThreads) {
    const int o = ((u >> 5 << log_c) + rank) * 32 + (u & 31), m = o >> 7, n = o & 127;
    if (o >= outs || n0 + n >= a.w.N) continue;
    float part[PARTS];
#pragma unroll
    for (int q = 0; q < PARTS; ++q) part[q] = recv[q * slots + u];
    for (int r = 1; r < C; ++r)
#pragma unroll
      for (int q = 0; q < PARTS; ++q) part[q] += recv[(r * PARTS + q) * slots + u];
    float y = part[PARTS - 1];  // the smallest part first
#pragma unroll
    for (int q = PARTS - 2; q >= 0; --q) y += part[q];
    if (a.x_scales && a.x_group == 0) y *= __ldg(a.x_scales + (m0 + m) * a.ldxs);
    if (a.b) y += load_as_f32(a.b, a.b_dtype, n0 + n);
    y = activate(y, a.act, a.alpha);
    const int64_t at = (m0 + m) * a.ldy + n0 + n;
    if (a.y_dtype == kF32) static_cast<float*>(a.Y)[at] = y;
    else if (a.y_dtype == kBF16) static_cast<bf16*>(a.Y)[at] = __float2bfloat16_rn(y);
    else static_cast<f16*>(a.Y)[at] = __float2half_rn(y);
  }
}

template <int XT, int NC, int UNIT>
int launch(W4Params p, int* status, cudaStream_t st) {
  auto kernel = dense_w4_tc_kernel<XT, NC, UNIT>;
  constexpr int PARTS = XRow<XT>::kParts, PER_SM = NC <= 64 ? 2 : 1;
  p.rows = NC / PARTS;
  const int64_t tiles = (p.a.w.N + kTileN - 1) / kTileN;
  const int64_t chunks = (p.a.M + p.rows - 1) / p.rows;
  if (chunks > 65535) return kErrTooLarge;
  // CTAs that share K: the fewest waves, each as long as a CTA's blocks and
  // kFixed of setting up and adding.
  constexpr int kFixed = 8;
  int best = 0;
  int64_t least = INT64_MAX;
  for (int l = 0; l <= 3; ++l) {
    const int64_t waves = ((tiles * chunks << l) + 148 * PER_SM - 1) / (148 * PER_SM);
    const int64_t blocks = (p.kblocks + (1 << l) - 1) >> l;
    const int64_t cost = waves * (blocks + kFixed);
    if (cost < least) {
      least = cost;
      best = l;
    }
  }
  if (const char* e = getenv("W4C"); e && atoi(e) >= 0) best = atoi(e);
  const int C = 1 << best;
  p.log_cluster = best;
  const int rows = (int)std::min<int64_t>(p.rows, p.a.M);
  p.recv_bytes = C * PARTS * ((rows * 4 + C - 1) / C * 32) * 4;
  const int smem = kStages * NC * 128 + kWorkers * kCodeDepth * 1024 + p.recv_bytes +
                   (int)sizeof(Barriers);
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e0 = allow_shared(reinterpret_cast<const void*>(kernel), allowed);
  if (e0 != cudaSuccess) return launch_result(e0);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * C), (unsigned)chunks);
  cfg.blockDim = dim3(kThreads);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, status);
  count_launch();
  return launch_result(e != cudaSuccess ? e : cudaGetLastError());
}

template <int XT, int UNIT>
int by_columns(const W4Params& p, int* status, cudaStream_t st) {
  const int64_t cols = p.a.M * XRow<XT>::kParts;
  if (cols <= 16) return launch<XT, 16, UNIT>(p, status, st);
  if (cols <= 32) return launch<XT, 32, UNIT>(p, status, st);
  if (cols <= 64) return launch<XT, 64, UNIT>(p, status, st);
  return launch<XT, 128, UNIT>(p, status, st);
}

template <int XT>
int by_unit(const W4Params& p, int* status, cudaStream_t st) {
  const int g = p.a.w.group, xg = p.a.x_group;
  if (g == 32 || xg == 32) return by_columns<XT, 32>(p, status, st);
  if (g % 128 == 0 && xg != 64) return by_columns<XT, 128>(p, status, st);
  return by_columns<XT, 64>(p, status, st);
}

}  // namespace

int dense_w4_tc(const W4Params& p, int* status, cudaStream_t st) {
  switch (p.a.x_dtype) {
    case kF32: return by_unit<kF32>(p, status, st);
    case kBF16: return by_unit<kBF16>(p, status, st);
    case kF16: return by_unit<kF16>(p, status, st);
    default: return by_unit<kE4M3>(p, status, st);
  }
}

}  // namespace b200
