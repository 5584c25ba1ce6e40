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
// CTAs of a cluster share K), and its warps one task each:
//   8 warps   codes, copied ahead by the lanes that use them, to TMEM
//   4 warps   activations, a stage ahead, into shared memory
//   1 warp    issues the products
//   4 or 8    sums out of TMEM, times their scales, into registers
// A unit is what one scale covers, at most 128 of K: products are exact, the
// tensor core sums 8 k16 steps at most, and the rest is added in f32 as for
// few rows. Measured on B200, a product of up to 64 columns takes 47 cycles to
// issue, a commit 190 and each meeting of two roles about as long, so they
// meet once for a stage of up to four blocks of K, with one commit for its
// operands and its sums. 17 or 21 warps leave 96 or 80 registers for every role:
// variants of 128 columns and most for e4m3 spill. 64x8192x8192 f16 23.1 us (floor
// 5.6), 5.7 thread instructions a weight in 57% of issue slots. Waits between the roles are bounded; one that runs out
// ends all of them, makes what the cluster stores NaN and is reported by
// b200_stream_sync. (The allocation of TMEM and the cluster's barriers wait for
// other CTAs to run or to end, which these bounds see to.)
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <atomic>
#include <cstdint>
#include "w4.cuh"

namespace cg = cooperative_groups;

namespace b200 {

namespace {

constexpr int kTileN = 128;
constexpr int kExpanders = 8;  // warps that expand codes, in two sets
constexpr int kStagers = 4;    // warps that bring activations
constexpr int kCodeDepth = 8;  // blocks that a lane copies ahead
constexpr int kMaxStages = 3;

// A stage: kBlocks blocks of 64 of K and the kUnits sums of NC columns that
// they take; as many blocks (1, 2 or 4) as let two stages fit TMEM's 512
// columns.
template <int NC, int UNIT>
struct Stage {
  static constexpr int columns(int blocks) {
    return 32 * blocks + (64 * blocks > UNIT ? 64 * blocks / UNIT : 1) * NC;
  }
  static constexpr int kBlocks = columns(4) <= 256 ? 4 : columns(2) <= 256 ? 2 : 1;
  static constexpr int kUnits = 64 * kBlocks > UNIT ? 64 * kBlocks / UNIT : 1;
  static constexpr int kColumns = 32 * kBlocks + kUnits * NC;
  static constexpr int kCount = 512 / kColumns < kMaxStages ? 512 / kColumns : kMaxStages;
  static constexpr int kFolders = NC <= 32 ? 4 : 8;  // warps that fold sums
  static constexpr int kThreads = (kExpanders + kStagers + 1 + kFolders) * 32;
  static_assert(kCount >= 2, "two stages fit TMEM");
};

struct Barriers {
  uint64_t full[kMaxStages];   // codes and activations of a stage are in place
  uint64_t done[kMaxStages];   // its products are done, its sums complete
  uint64_t taken[kMaxStages];  // its sums have been read
  uint64_t unheard[kMaxStages];  // in place of done, where products do not report their end
  uint64_t drained;            // after a wait that ran out: products under way are done
  uint32_t tmem;
  int abort_flag;
};

// expire_ns > 0: waits run out after it, and products never report their end
// (b200_debug_w4_expire).
template <int XT, int NC, int UNIT>
__global__ void __launch_bounds__(Stage<NC, UNIT>::kThreads, 1)
    dense_w4_tc_kernel(const __grid_constant__ W4Params p, int* status, int64_t expire_ns) {
  using X = XRow<XT>;
  using Mma = typename X::Mma;
  using Raw = typename X::Raw;
  using S = Stage<NC, UNIT>;
  constexpr int PARTS = X::kParts, OWN = NC / (S::kFolders / 4), STAGES = S::kCount, SB = S::kBlocks;
  constexpr int kMmaWarp = kExpanders + kStagers, kFoldWarp = kMmaWarp + 1;
  constexpr int SUBS = UNIT == 32 ? 2 : 1;  // scales of a block
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
  // this CTA's blocks of K, in whole stages (and so whole units)
  const int all_stages = (kblocks + SB - 1) / SB;
  const int b0 = (int)((int64_t)all_stages * rank >> log_c) * SB;
  const int b1 = min(kblocks, (int)((int64_t)all_stages * (rank + 1) >> log_c) * SB);
  const int nb = max(0, b1 - b0), stages = (nb + SB - 1) / SB;
  const int units = nb > 0 ? (min(K, b1 * kBlockK) - b0 * kBlockK + UNIT - 1) / UNIT : 0;

  // shared memory: activations (swizzled tiles of 64 k by NC columns), codes,
  // what the cluster's CTAs send, barriers
  char* xring = smem;
  char* cring = xring + STAGES * SB * NC * 128;
  float* recv = reinterpret_cast<float*>(cring + kExpanders * kCodeDepth * 1024);
  Barriers* bar = reinterpret_cast<Barriers*>(reinterpret_cast<char*>(recv) + p.recv_bytes);
  volatile int* abort_flag = &bar->abort_flag;
  const uint64_t limit_ns = expire_ns > 0 ? (uint64_t)expire_ns : B200_WAIT_NS;
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&bar->full[i], (SB > 1 ? kExpanders : kExpanders / 2) + kStagers);
      mbar_init(&bar->done[i], 1);
      mbar_init(&bar->unheard[i], 1);
      mbar_init(&bar->taken[i], S::kFolders);
    }
    mbar_init(&bar->drained, 1);
    bar->abort_flag = 0;
    fence_barrier_init();
  }
  // one thread for each of the CTA's strips
  if (tid >= 32 && tid < 34 && n0 + (tid - 32) * kStripN < a.w.N)
    prefetch_strip(p, n0 / kStripN + tid - 32, b0, b1, false);
  pdl_wait();
  if (wid == kMmaWarp) tmem_alloc(&bar->tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // only now: a kernel that starts early must not take TMEM that a CTA of this
  // one still waits for
  pdl_trigger();
  const uint32_t tmem = bar->tmem, tmem_sums = tmem + STAGES * SB * 32;
  auto wait = [&](uint64_t* b, int phase, int code) {
    return mbar_wait_warp(b, phase & 1, status, code, abort_flag, limit_ns);
  };
  // the products of stage t's predecessor in the ring are done
  auto reusable = [&](int t) {
    return t < STAGES || wait(&bar->done[t % STAGES], t / STAGES - 1, kDevTimeoutEmpty);
  };

  const int quarter = wid & 3;  // of TMEM's lanes, where a warp has one
  float total[OWN];             // of a folding warp
#pragma unroll
  for (int i = 0; i < OWN; ++i) total[i] = 0.0f;
  const int fold_set = (wid - kFoldWarp) >> 2;
  bool ran_out = false;  // a wait of the CTA; its sums are NaN then

  const int64_t strip = n0 / kStripN + (quarter >> 1);
  const bool live = strip * kStripN < a.w.N;
  if (wid < kExpanders) {
    const int set = wid >> 2, mt0 = (quarter & 1) * 2, g = lane >> 2;
    // ---- codes: two 16-column pieces of the quarter's 32 columns; the set's
    // blocks are every other one
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
    uint32_t znext[SUBS] = {};
    auto fetch_zeros = [&](int i) {
      if (!zeros || !live || i >= nb) return;
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        const int k = (b0 + i) * kBlockK + sub * 32;
        if (sub && k >= K) return;
        znext[sub] =
            __ldg(reinterpret_cast<const uint32_t*>(zeros + (int64_t)p.group_of(k) * 64));
      }
    };
    fetch_zeros(set);
    int slot = 0;
    // block i (of the set's) to the columns of TMEM from `to` on
    auto expand = [&](int i, uint32_t to) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kCodeDepth - 1) : "memory");
      const uint4 w[2] = {mine[slot * 64], mine[slot * 64 + 32]};
      uint32_t z[SUBS][4];
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          z[sub][q] = zeros ? __byte_perm(znext[sub], Mma::kMagic, 0x5050 | q * 0x0101)
                            : 0x00080008u | Mma::kMagic;
      fetch_zeros(i + 2);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t words[4] = {w[q].x, w[q].y, w[q].z, w[q].w};
        uint32_t f[16];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            f[4 * j + r] = Mma::sub(and_or(words[j] >> (4 * r), 0x000f000fu, Mma::kMagic),
                                    z[SUBS == 2 ? j >> 1 : 0][2 * q + (r & 1)]);
        tmem_st_16x128b_x8(to + ((uint32_t)(quarter * 32 + q * 16) << 16), f);
      }
      fetch(slot);  // the slot's codes have been used
      slot = (slot + 1) % kCodeDepth;
    };

    for (int t = 0; t < stages; ++t) {
      if (SB == 1 && (t & 1) != set) continue;
      if (!reusable(t)) break;
      tc_fence_after();
#pragma unroll
      for (int b = 0; b < (SB + 1) / 2; ++b) {
        const int in_stage = SB > 1 ? 2 * b + set : 0, i = t * SB + in_stage;
        if (i < nb) expand(i, tmem + (t % STAGES * SB + in_stage) * 32);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->full[t % STAGES]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (wid < kMmaWarp) {
    // ---- activations: pieces of 8 elements, 8 of a row and block; 16 bytes
    // of the column's 128 in shared memory, swizzled as the tensor core reads
    // them
    constexpr int PER = (NC / PARTS * 8 + kStagers * 32 - 1) / (kStagers * 32);
    const int st = tid - kExpanders * 32;
    const int c = st & 7, row0 = st >> 3, rows_step = kStagers * 4;
    const char* x = static_cast<const char*>(a.X) + m0 * a.ldx * X::kBytes;
    // column `col` of block i
    auto place = [&](int i, int col) {
      return xring + (i / SB % STAGES * SB + i % SB) * (NC * 128) + col * 128 +
             ((c ^ (col & 7)) << 4);
    };
    auto post = [&](int t) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->full[t % STAGES]);
    };
    if (X::kBytes == 2 && p.x_aligned) {
      // 16-bit rows are copied as they are
      const int k0 = b0 * kBlockK + c * 8;
      const int64_t step = (int64_t)rows_step * a.ldx * 2;
      const char* from = x + ((int64_t)row0 * a.ldx + k0) * 2;
      int left = K - k0;            // elements of the row from here on; K may reach 2^31 - 64
      int64_t at_start = x - from;  // a valid address where nothing is read
      for (int t = 0; t < stages; ++t) {
        if (!reusable(t)) break;
#pragma unroll
        for (int sb = 0; sb < SB; ++sb) {
          const int bytes = max(0, min(8, left)) * 2;
          char* to = place(t * SB + sb, row0);  // rows_step is a multiple of the swizzle's 8
#pragma unroll
          for (int u = 0; u < PER; ++u)
            if (row0 + u * rows_step < mrows)
              cp_async16_fill(to + u * (rows_step * 128), from + (bytes ? u * step : at_start),
                              bytes);
          from += kBlockK * 2;
          at_start -= kBlockK * 2;
          left -= kBlockK;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        post(t);
      }
    } else {
      // others pass through registers: blocks whose 64 columns are all there and
      // aligned are asked for ahead, as many as fit 32 registers, without a
      // branch that would wait for them
      constexpr int WORDS = PER * (int)sizeof(Raw) / 4;
      constexpr int AHEAD = SB >= 4 && 4 * WORDS <= 32 ? 4 : SB >= 2 && 2 * WORDS <= 32 ? 2 : 1;
      const int whole = p.x_aligned ? min(nb, (K - b0 * kBlockK) / kBlockK) : 0;
      const char* rows[PER];
#pragma unroll
      for (int u = 0; u < PER; ++u)  // rows past the last: the last again
        rows[u] = x + ((int64_t)min(row0 + u * rows_step, mrows - 1) * a.ldx + b0 * kBlockK + c * 8) *
                          X::kBytes;
      Raw ahead[AHEAD][PER];
      auto load = [&](int i, Raw (&next)[PER]) {
#pragma unroll
        for (int u = 0; u < PER; ++u) next[u] = X::load_whole(rows[u], min(i, whole - 1) * kBlockK);
      };
      auto put = [&](int i, const Raw (&raw)[PER]) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          const int m = row0 + u * rows_step;
          if (m >= mrows) continue;
          uint4 out[PARTS];
          X::stage(raw[u], out);
#pragma unroll
          for (int q = 0; q < PARTS; ++q)
            *reinterpret_cast<uint4*>(place(i, m * PARTS + q)) = out[q];
        }
      };
      if (whole > 0) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) load(i, ahead[i]);
      }
      for (int t = 0; t < stages; ++t) {
        // few enough words: made ready, and the next stage's asked for, before the
        // wait (16x11008x4096 e4m3 18.4 -> 16.9 us)
        constexpr bool EARLY = AHEAD == SB && SB * PER * PARTS <= 4;
        uint4 ready[EARLY ? SB * PER : 1][PARTS];
        if constexpr (EARLY) {
#pragma unroll
          for (int sb = 0; sb < SB; ++sb)
            if (t * SB + sb < whole) {
#pragma unroll
              for (int u = 0; u < PER; ++u) X::stage(ahead[sb][u], ready[sb * PER + u]);
              load(t * SB + sb + AHEAD, ahead[sb]);
            }
        }
        if (!reusable(t)) break;
#pragma unroll
        for (int sb = 0; sb < SB; ++sb) {
          const int i = t * SB + sb;
          if (EARLY && i < whole) {
#pragma unroll
            for (int u = 0; u < PER; ++u) {
              const int m = row0 + u * rows_step;
              if (m >= mrows) continue;
#pragma unroll
              for (int q = 0; q < PARTS; ++q)
                *reinterpret_cast<uint4*>(place(i, m * PARTS + q)) = ready[EARLY ? sb * PER + u : 0][q];
            }
          } else if (i < whole) {
            put(i, ahead[sb % AHEAD]);
            load(i + AHEAD, ahead[sb % AHEAD]);
          } else if (i < nb) {
            Raw raw[PER];
#pragma unroll
            for (int u = 0; u < PER; ++u)
              raw[u] = X::load(rows[u] - c * 8 * X::kBytes, (int64_t)i * kBlockK + c * 8,
                               K - b0 * kBlockK, false);
            put(i, raw);
          }
        }
        post(t);
      }
    }
  } else if (wid == kMmaWarp) {
    // ---- products
    uint64_t* done = expire_ns > 0 ? bar->unheard : bar->done;
    for (int t = 0; lane == 0 && t < stages; ++t) {
      const int s = t % STAGES;
      if (!mbar_wait_long(&bar->full[s], (t / STAGES) & 1, status, kDevTimeoutFull, abort_flag,
                          limit_ns) ||
          (t >= STAGES && !mbar_wait_long(&bar->taken[s], (t / STAGES - 1) & 1, status,
                                          kDevTimeoutAccum, abort_flag, limit_ns)))
        break;
      tc_fence_after();
      const uint64_t bdesc = umma_desc_k<2, 1024>(smem_u32(xring + s * SB * NC * 128));
      const uint32_t from = tmem + s * SB * 32, to = tmem_sums + s * S::kUnits * NC;
#pragma unroll
      for (int k = 0; k < SB * 4; ++k) {  // k16 steps
        constexpr int PER_UNIT = UNIT / 16;
        const int unit = k / PER_UNIT;
        if (t * SB + k / 4 >= nb || t * S::kUnits + unit >= units) break;
        umma_f16_ts(to + unit * NC, from + k * 8, bdesc + (k / 4) * (NC * 8) + (k % 4) * 2, kIdesc,
                    k % PER_UNIT != 0);
      }
      umma_commit(&done[s]);
    }
  } else {
    // ---- sums: this lane's column of W, OWN operand columns of it
    const int n = (quarter & 1) * 32 + lane;  // within the strip
    // their scales, asked for a stage ahead; bits, so that nothing waits for
    // them before they are used (past the last unit or strip: the last again)
    const bool s32 = a.w.s_dtype == kF32;
    const int64_t last_strip = (a.w.N - 1) / kStripN;
    const int64_t scale_col = min(strip, last_strip) * p.groups * 64 + column_place(n);
    auto scale_bits = [&](int u) -> uint32_t {
      const int k = b0 * kBlockK + max(0, min(u, units - 1)) * UNIT;
      const int64_t at = scale_col + (int64_t)p.group_of(min(k, K - 1)) * 64;
      return s32 ? __ldg(reinterpret_cast<const uint32_t*>(p.scales) + at)
                 : (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p.scales) + at);
    };
    uint32_t next[S::kUnits];
    if (units > 0) {
#pragma unroll
      for (int j = 0; j < S::kUnits; ++j) next[j] = scale_bits(j);
    }
    for (int t = 0; t < stages; ++t) {
      const int s = t % STAGES;
      float scale[S::kUnits];
#pragma unroll
      for (int j = 0; j < S::kUnits; ++j)
        scale[j] = s32                        ? __uint_as_float(next[j])
                   : a.w.s_dtype == kBF16     ? __uint_as_float(next[j] << 16)
                                              : __half2float(__ushort_as_half((unsigned short)next[j]));
#pragma unroll
      for (int j = 0; j < S::kUnits; ++j) next[j] = scale_bits((t + 1) * S::kUnits + j);
      if (!wait(&bar->done[s], t / STAGES, kDevTimeoutAccum)) {
        ran_out = true;  // whichever wait of the CTA did, this one follows
        break;
      }
      tc_fence_after();
      const uint32_t at =
          tmem_sums + ((uint32_t)(quarter * 32) << 16) + s * S::kUnits * NC + fold_set * OWN;
#pragma unroll
      for (int j = 0; j < S::kUnits; ++j) {
        const int u = t * S::kUnits + j;
        if (u >= units) break;
        constexpr int STEP = OWN < 32 ? OWN : OWN == 32 ? 32 : 16;
#pragma unroll
        for (int c = 0; c < OWN; c += STEP) {
          uint32_t v[STEP];
          if constexpr (STEP == 16) tmem_ld_32x32b_x16(at + j * NC + c, v);
          else tmem_ld_32x32b_x32(at + j * NC + c, v);
          tmem_ld_wait();
          if (XT == kE4M3 && a.x_group > 0) {
            const unsigned xg = (unsigned)(b0 * kBlockK + u * UNIT) / (unsigned)a.x_group;
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
              const int m = fold_set * OWN + c + i;
              const float xs = m < mrows ? __ldg(a.x_scales + (m0 + m) * a.ldxs + xg) : 0.0f;
              total[c + i] = fmaf(__uint_as_float(v[i]) * xs, scale[j], total[c + i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < STEP; ++i)
              total[c + i] = fmaf(__uint_as_float(v[i]), scale[j], total[c + i]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->taken[s]);
    }
  }

  __syncwarp();
  // TMEM goes back before this CTA waits for others: two clusters that share
  // SMs must not hold it while each waits for a CTA that waits for it
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (wid == kMmaWarp) {
    if (lane == 0 && *abort_flag) {  // set before the barrier, if at all
      umma_commit(&bar->drained);
      const uint64_t since = globaltimer();
      while (!mbar_try_wait(&bar->drained, 0) && globaltimer() - since < B200_WAIT_NS) {
      }
    }
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
  // ---- the CTAs' parts of K: each 32 outputs of a row belong to one CTA of
  // the cluster, in turn
  const int chunks = mrows * 4;
  const int slots = ((chunks + C - 1) >> log_c) * 32;
  if (C > 1) cluster.barrier_wait();  // every CTA of the cluster runs
  if (wid >= kFoldWarp) {
    float* mine = recv + rank * PARTS * slots + lane;
    float* to[2];  // for even and odd rows
#pragma unroll
    for (int o = 0; o < 2; ++o)
      to[o] = C > 1 ? cluster.map_shared_rank(mine, (o * 4 + quarter) & (C - 1)) : mine;
#pragma unroll
    for (int c = 0; c < OWN; ++c) {
      const int col = fold_set * OWN + c, m = col / PARTS, q = col - m * PARTS;
      if (m < mrows) {
        const int at = q * slots + ((m * 4 + quarter) >> log_c) * 32;
        (m & 1 ? to[1] : to[0])[at] = ran_out ? __int_as_float(0x7fc00000) : total[c];
      }
    }
  }
  if (C > 1) cluster.sync();
  else __syncthreads();
  // four outputs a thread
  const int64_t y_bytes = a.y_dtype == kF32 ? 4 : 2;
  const bool whole = reinterpret_cast<uintptr_t>(a.Y) % (4 * y_bytes) == 0 && a.ldy % 4 == 0;
  for (int u = tid * 4; u < slots; u += S::kThreads * 4) {
    const int chunk = (u >> 5 << log_c) + rank, m = chunk >> 2;
    const int64_t n = n0 + (chunk & 3) * 32 + (u & 31);
    if (chunk >= chunks || n >= a.w.N) continue;
    float4 part[PARTS];
#pragma unroll
    for (int q = 0; q < PARTS; ++q) part[q] = *reinterpret_cast<const float4*>(recv + q * slots + u);
    for (int r = 1; r < C; ++r)
#pragma unroll
      for (int q = 0; q < PARTS; ++q) {
        const float4 v = *reinterpret_cast<const float4*>(recv + (r * PARTS + q) * slots + u);
        part[q].x += v.x;
        part[q].y += v.y;
        part[q].z += v.z;
        part[q].w += v.w;
      }
    float y[4] = {part[PARTS - 1].x, part[PARTS - 1].y, part[PARTS - 1].z, part[PARTS - 1].w};
#pragma unroll
    for (int q = PARTS - 2; q >= 0; --q) {  // the smallest part first
      y[0] += part[q].x;
      y[1] += part[q].y;
      y[2] += part[q].z;
      y[3] += part[q].w;
    }
    const float xs = a.x_scales && a.x_group == 0 ? __ldg(a.x_scales + (m0 + m) * a.ldxs) : 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] *= Mma::kUp;
      if (a.x_scales && a.x_group == 0) y[i] *= xs;
      if (a.b && n + i < a.w.N) y[i] += load_as_f32(a.b, a.b_dtype, n + i);
      y[i] = activate(y[i], a.act, a.alpha);
    }
    char* at = static_cast<char*>(a.Y) + ((m0 + m) * a.ldy + n) * y_bytes;
    if (a.y_dtype == kF32) {
      if (whole && n + 4 <= a.w.N) {
        *reinterpret_cast<float4*>(at) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
        for (int i = 0; i < 4 && n + i < a.w.N; ++i) reinterpret_cast<float*>(at)[i] = y[i];
      }
      continue;
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (a.y_dtype == kBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if (whole && n + 4 <= a.w.N) {
      *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
    } else {
      for (int i = 0; i < 4 && n + i < a.w.N; ++i)
        reinterpret_cast<uint16_t*>(at)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

std::atomic<int64_t> g_expire_ns{0};  // b200_debug_w4_expire

template <int XT, int NC, int UNIT>
int launch(W4Params p, int* status, cudaStream_t st) {
  auto kernel = dense_w4_tc_kernel<XT, NC, UNIT>;
  using S = Stage<NC, UNIT>;
  constexpr int PARTS = XRow<XT>::kParts;
  p.rows = NC / PARTS;
  const int64_t tiles = (p.a.w.N + kTileN - 1) / kTileN;
  const int64_t chunks = (p.a.M + p.rows - 1) / p.rows;
  if (chunks > 65535) return kErrTooLarge;
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  const cudaError_t e0 = allow_shared(reinterpret_cast<const void*>(kernel), allowed, &dev);
  if (e0 != cudaSuccess) return launch_result(e0);
  static PerDevice<Capacity> capacities;
  const Capacity capacity = capacities.of(dev, [&] {
    return capacity_of(reinterpret_cast<const void*>(kernel), S::kThreads, kMaxShared);
  });
  const int best = choose_cluster(capacity, tiles * chunks, p.kblocks, 1, 8);
  const int C = 1 << best;
  p.log_cluster = best;
  const int rows = (int)std::min<int64_t>(p.rows, p.a.M);
  p.recv_bytes = C * PARTS * ((rows * 4 + C - 1) / C * 32) * 4;
  const int smem = S::kCount * S::kBlocks * NC * 128 + kExpanders * kCodeDepth * 1024 + p.recv_bytes +
                   (int)sizeof(Barriers);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * C), (unsigned)chunks);
  cfg.blockDim = dim3(S::kThreads);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, status,
                                          g_expire_ns.load(std::memory_order_relaxed));
  count_launch();
  return launch_result(e != cudaSuccess ? e : cudaGetLastError());
}

template <int XT, int UNIT>
int by_columns(const W4Params& p, int* status, cudaStream_t st) {
  const int64_t cols = p.a.M * XRow<XT>::kParts;
  if (cols <= 16) return launch<XT, 16, UNIT>(p, status, st);
  if (cols <= 32) return launch<XT, 32, UNIT>(p, status, st);
  if (cols <= 64) return launch<XT, 64, UNIT>(p, status, st);
  // 64 at a time where the sums of 128 do not fit TMEM twice
  return launch<XT, UNIT == 32 ? 64 : 128, UNIT>(p, status, st);
}

template <int XT>
int by_unit(const W4Params& p, int* status, cudaStream_t st) {
  const int g = p.a.w.group, xg = p.a.x_group;
  if (g == 32 || xg == 32) return by_columns<XT, 32>(p, status, st);
  if (g % 128 == 0 && xg != 64) return by_columns<XT, 128>(p, status, st);
  return by_columns<XT, 64>(p, status, st);
}

}  // namespace

void w4_expire(int64_t limit_ns) { g_expire_ns.store(limit_ns, std::memory_order_relaxed); }

int dense_w4_tc(const W4Params& p, int* status, cudaStream_t st) {
  switch (p.a.x_dtype) {
    case kF32: return by_unit<kF32>(p, status, st);
    case kBF16: return by_unit<kBF16>(p, status, st);
    case kF16: return by_unit<kF16>(p, status, st);
    default: return by_unit<kE4M3>(p, status, st);
  }
}

}  // namespace b200
