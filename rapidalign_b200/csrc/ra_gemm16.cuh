// ra_gemm16.cuh -- persistent tensor-core matrix product with a fused
// epilogue: the three products of the linear cross entropy (ra_ce.cuh).
//
//   D[m, n] = sum_k A[m, k] B[n, k]      16-bit operands, fp32 accumulators
//
// Either operand may lie K-major (rows of K in memory) or MN-major (rows of
// M or N), so that G W and G^T X need no transposed copies.  Operands come
// as tensor maps with 128-byte swizzle; elements outside a map read as zero,
// so no edge of M, N or K is special before the epilogue.
//
// fp32 inputs come as two fp16 halves (a = hi + lo, 22 significant bits, one
// power-of-two scale per tensor) and three products, hi hi, hi lo and lo hi,
// from one copy of the four tiles; the two small ones have an accumulator of
// their own.  The tensor core drops the bits below an accumulator's last one
// instead of rounding them: over a long K the loss adds up (2.5e-5 of dw at
// K = 65537 in one chain of all three, where fp32 sums keep 1e-6).  So a unit of
// pairs is cut into rounds of kGmRound k steps; each round starts fresh
// accumulators and the epilogue adds the rounds in registers, rounding to
// nearest.
//
// Roles (576 threads, one CTA per SM, persistent over (tile, K slice) units):
//   warps 0-15 epilogue: warp w reads TMEM lanes 32 (w % 4).. and quarter w / 4
//              of the tile's columns.  Sixteen, because over a short K (D = 128:
//              1,500 cycles of MMAs a tile) the epilogue's own latency is what
//              a tile takes.
//   warp 16    lane 0 copies operand tiles into the shared-memory ring
//   warp 17    lane 0 issues the MMAs
// Two accumulators in TMEM (two pairs of them): the epilogue of one unit runs
// under the MMAs of the next; what it reads of its rows besides is loaded before
// it waits.  Every wait is bounded; on expiry the CTA records the timeout,
// drains its copies, frees its TMEM and returns.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ra_common.cuh"
#include "ra_tcprim.cuh"

namespace ra {

constexpr int kGmM = 128, kGmK = 64;
constexpr int kGmEpiWarps = 16, kGmLoadWarp = 16, kGmMmaWarp = 17, kGmThreads = 576;
constexpr int kGmParts = kGmEpiWarps / 4;  // column parts of a tile
constexpr int kGmABytes = kGmM * kGmK * 2;
constexpr int kGmRound = 4;  // k steps (of 64) of a round of pairs

// 192 KB of operand tiles: 4 stages of 128 x 256 tiles, 6 of 128 x 128, 3 of
// pairs (128 x 128 only)
__host__ __device__ constexpr int gm_stage_bytes(int TN, bool pairs) {
  return (kGmABytes + TN * kGmK * 2) * (pairs ? 2 : 1);
}
__host__ __device__ constexpr int gm_stages(int TN, bool pairs) {
  return 192 * 1024 / gm_stage_bytes(TN, pairs);
}
constexpr int kGmStageOut = 2048;  // a warp's 32 rows of 64 bytes on their way out
constexpr size_t kGmSmem = 1024 + 192 * 1024 + kGmEpiWarps * kGmStageOut + 256;

// The units of one launch: tiles of 128 x TN, each cut into `slices` of K.
// m runs fastest where the B operand is the large one (m_fast), so that
// concurrent CTAs share a B tile.
struct GmShape {
  int m_tiles, n_tiles, k_steps, slices;
  int m_fast;
  unsigned spin_limit;  // polls of one wait before giving up
  int no_mma;           // test hook: no products, so that the waits for them expire
  int *status;
};

struct GmMaps {
  CUtensorMap a_hi, a_lo, b_hi, b_lo;
};

__host__ __device__ constexpr uint32_t gm_idesc(int N, bool bf16, bool a_mn, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) |
         (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kGmM >> 4) << 24);
}
// 128-byte swizzled operand tiles.  K-major: rows of 64 k (128 bytes), eight
// rows an atom, atoms 1024 bytes apart.  MN-major: chunks of 64 m (or n),
// each 64 k rows of 128 bytes; 8-k groups 1024 bytes apart, chunks 8192.
__device__ __forceinline__ uint64_t gm_desc(uint32_t saddr, bool mn) {
  const uint64_t lbo = mn ? 8192u >> 4 : 1u, sbo = 1024u >> 4;
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (lbo << 16) | (sbo << 32) | (1ull << 46) |
         (2ull << 61);
}
__device__ __forceinline__ void gm_mma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, int x, int y,
                                       uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(mbar)
      : "memory");
}

struct GmUnit {
  int m, n, slice, k0, k1;
};
__device__ __forceinline__ GmUnit gm_unit(const GmShape &s, int u) {
  GmUnit r;
  r.slice = u % s.slices;
  const int t = u / s.slices;
  if (s.m_fast) {
    r.m = t % s.m_tiles;
    r.n = t / s.m_tiles;
  } else {
    r.n = t % s.n_tiles;
    r.m = t / s.n_tiles;
  }
  r.k0 = (int)((int64_t)s.k_steps * r.slice / s.slices);
  r.k1 = (int)((int64_t)s.k_steps * (r.slice + 1) / s.slices);
  return r;
}

// The thread's row of a finished tile, 32 columns at a time: straight from
// TMEM (which a warp reads together, whatever branches its lanes took before), or
// from the registers that joined the rounds.
struct GmFromTmem {
  uint32_t taddr;
  static constexpr int unroll = 1;
  __device__ __forceinline__ void get(int c, float (&v)[32]) const {
    __syncwarp();
    tmem_ld32(taddr + c, v);
  }
};
struct GmFromPairs {  // one round of pairs: both accumulators
  uint32_t taddr, small;
  static constexpr int unroll = 1;
  __device__ __forceinline__ void get(int c, float (&v)[32]) const {
    float x[32];
    __syncwarp();
    tmem_ld32(taddr + c, v);
    tmem_ld32(small + c, x);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] += x[j];
  }
};
template <int NC>
struct GmFromRegs {
  const float (&acc)[NC];
  static constexpr int unroll = NC / 32;
  __device__ __forceinline__ void get(int c, float (&v)[32]) const {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = acc[c + j];
  }
};
// A warp's way to global memory: every lane gives 64 bytes of its row, and four
// lanes at a time take a whole row's (a lane's own 16-byte stores would write
// half sectors of 32 rows).  put(row of the warp, 16-byte chunk, bits).
struct GmOut {
  uint8_t *p;  // kGmStageOut bytes of this warp
  template <class Put>
  __device__ __forceinline__ void rows64(const uint4 (&x)[4], Put put) const {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4 *>(p + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = x[j];
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = (lane >> 2) + 8 * k, j = lane & 3;
      put(row, j, *reinterpret_cast<const uint4 *>(p + row * 64 + ((j ^ ((row >> 1) & 3)) << 4)));
    }
  }
};

// Epi: `Fixed fixed()` once per thread; `Row begin(unit, row)` loads what the
// row needs; run<TN>(fixed, row state, unit, row, col, source, out) works on one
// thread's row of the tile and its quarter of the columns, all lanes of a warp
// together.  OP: one product; three products of pairs in one round, or in more.
enum GmOp { kGmOne, kGmPairs1, kGmPairs };
template <int TN, bool BF16, GmOp OP, bool A_MN, bool B_MN, class Epi>
__global__ void __launch_bounds__(kGmThreads, 1)
    gemm16_kernel(const __grid_constant__ GmMaps maps, const GmShape s,
                  const __grid_constant__ Epi epi) {
  extern __shared__ uint8_t gm_raw[];
  const uint32_t raw = smem_u32(gm_raw);
  const uint32_t base = (raw + 1023) & ~1023u;
  constexpr bool PAIRS = OP != kGmOne;
  static_assert(!PAIRS || TN == 128, "TMEM holds two pairs of 128 columns");
  constexpr int kStage = gm_stage_bytes(TN, PAIRS), kGmStages = gm_stages(TN, PAIRS);
  constexpr int kAccCols = PAIRS ? 2 * TN : TN;  // PAIRS: hi hi, then the small ones
  constexpr int kTmemCols = 2 * kAccCols;
  constexpr int kBBytes = TN * kGmK * 2;
  constexpr int kRound = OP == kGmPairs ? kGmRound : 1 << 30;
  const uint32_t outs = base + kGmStages * kStage, bars = outs + kGmEpiWarps * kGmStageOut;
  // full, empty [stages], accfull[2] accempty[2], then the TMEM address and abort flag
  const uint32_t full = bars, empty = bars + 8 * kGmStages, accfull = bars + 16 * kGmStages,
                 accempty = accfull + 16, tmem_slot = accempty + 16;
  volatile int *abort_flag = (volatile int *)(gm_raw + (tmem_slot + 4 - raw));
  volatile uint32_t *tmem_addr = (volatile uint32_t *)(gm_raw + (tmem_slot - raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = s.m_tiles * s.n_tiles * s.slices;

  if (warp == kGmMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     tmem_slot),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kGmStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(accfull + 8 * i, 1);
      mbar_init(accempty + 8 * i, kGmEpiWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_addr;

  if (warp == kGmLoadWarp) {
    if (lane == 0) {
      int issued = 0;  // operand tiles issued; tile i sits in stage i % kGmStages
      bool ok = true;
      for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
        const GmUnit w = gm_unit(s, u);
        for (int k = w.k0; k < w.k1; ++k, ++issued) {
          const int st = issued % kGmStages;
          if (issued >= kGmStages &&
              !ws_wait(empty + 8 * st, ((issued / kGmStages) - 1) & 1, abort_flag, s.spin_limit)) {
            ok = false;
            break;
          }
          const uint32_t a = base + st * kStage, b = a + (PAIRS ? 2 : 1) * kGmABytes,
                         bar = full + 8 * st;
          mbar_expect_tx(bar, kStage);
#pragma unroll
          for (int p = 0; p < (PAIRS ? 2 : 1); ++p) {
            const CUtensorMap *ma = p ? &maps.a_lo : &maps.a_hi, *mb = p ? &maps.b_lo : &maps.b_hi;
            if (A_MN) {
#pragma unroll
              for (int c = 0; c < kGmM / 64; ++c)
                tma_2d(a + p * kGmABytes + c * 8192, ma, w.m * kGmM + c * 64, k * kGmK, bar);
            } else {
              tma_2d(a + p * kGmABytes, ma, k * kGmK, w.m * kGmM, bar);
            }
            if (B_MN) {
#pragma unroll
              for (int c = 0; c < TN / 64; ++c)
                tma_2d(b + p * kBBytes + c * 8192, mb, w.n * TN + c * 64, k * kGmK, bar);
            } else {
              tma_2d(b + p * kBBytes, mb, k * kGmK, w.n * TN, bar);
            }
          }
        }
      }
      if (!ok) *abort_flag = 1;
      // a CTA does not leave while copies into its shared memory are in flight
      const int first = issued > kGmStages ? issued - kGmStages : 0;
      for (int i = first; i < issued; ++i)
        if (!mbar_wait(full + 8 * (i % kGmStages), (i / kGmStages) & 1)) ok = false;
      if (!ok) atomicOr(s.status, 1);
    }
  } else if (warp == kGmMmaWarp) {
    if (lane == 0 && !s.no_mma) {
      constexpr uint32_t idesc = gm_idesc(TN, BF16, A_MN, B_MN);
      int used = 0, t = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
        const GmUnit w = gm_unit(s, u);
        for (int k0 = w.k0; ok && k0 < w.k1; k0 += kRound, ++t) {
          const int buf = t & 1;
          if (t >= 2 &&
              !ws_wait(accempty + 8 * buf, ((t >> 1) - 1) & 1, abort_flag, s.spin_limit)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t acc = tmem + buf * kAccCols;
          const int steps = min(k0 + kRound, w.k1) - k0;
          for (int i = 0; i < steps; ++i, ++used) {
            const int st = used % kGmStages;
            if (!ws_wait(full + 8 * st, (used / kGmStages) & 1, abort_flag, s.spin_limit)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t a = base + st * kStage, b = a + (PAIRS ? 2 : 1) * kGmABytes;
            const uint64_t da = gm_desc(a, A_MN), db = gm_desc(b, B_MN);
#pragma unroll
            for (int kk = 0; kk < kGmK / 16; ++kk) {
              // 16 k: 32 bytes along a K-major row, two 8-k groups MN-major
              const uint64_t ka = da + (uint64_t)(kk * (A_MN ? 2048 : 32) >> 4),
                             kb = db + (uint64_t)(kk * (B_MN ? 2048 : 32) >> 4);
              gm_mma(acc, ka, kb, idesc, i > 0 || kk > 0);
              if (PAIRS) {
                gm_mma(acc + TN, ka + (kGmABytes >> 4), kb, idesc, i > 0 || kk > 0);
                gm_mma(acc + TN, ka, kb + (kBBytes >> 4), idesc, 1);
              }
            }
            tc_commit(empty + 8 * st);
          }
          if (ok) tc_commit(accfull + 8 * buf);
        }
      }
      if (!ok) {
        *abort_flag = 1;
        atomicOr(s.status, 1);
      }
    }
  } else {
    constexpr int kCols = TN / kGmParts;  // columns of a thread
    const int col = (warp >> 2) * kCols;
    const GmOut out{gm_raw + (outs - raw) + warp * kGmStageOut};
    const int row = 32 * (warp & 3) + lane;
    const uint32_t lane_addr =
        tmem + col + ((uint32_t)(32 * (warp & 3)) << 16);
    int t = 0;
    // waits for round t's accumulator; false (for the whole warp) on expiry
    auto ready = [&]() {
      const bool got = ws_wait(accfull + 8 * (t & 1), (t >> 1) & 1, abort_flag, s.spin_limit);
      if (!__all_sync(kFull, got)) {
        *abort_flag = 1;
        if (lane == 0) atomicOr(s.status, 1);
        return false;
      }
      tc_fence_after();
      return true;
    };
    auto release = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(accempty + 8 * (t & 1));
      ++t;
    };
    bool ok = true;
    const auto fixed = epi.fixed();
    for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
      const GmUnit w = gm_unit(s, u);
      const auto state = epi.begin(w, row);
      if constexpr (OP == kGmPairs) {
        float acc[kCols];
        for (int k0 = w.k0; k0 < w.k1; k0 += kRound) {
          if (!(ok = ready())) break;
          const uint32_t from = lane_addr + (t & 1) * kAccCols;
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            float v[32], x[32];
            tmem_ld32(from + c, v);
            tmem_ld32(from + TN + c, x);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              v[j] += x[j];
              acc[c + j] = k0 == w.k0 ? v[j] : acc[c + j] + v[j];
            }
          }
          release();
        }
        if (ok)
          epi.template run<TN>(fixed, state, w, row, col, GmFromRegs<kCols>{acc}, out);
      } else {
        if (!(ok = ready())) break;
        const uint32_t from = lane_addr + (t & 1) * kAccCols;
        if constexpr (OP == kGmPairs1)
          epi.template run<TN>(fixed, state, w, row, col, GmFromPairs{from, from + TN}, out);
        else
          epi.template run<TN>(fixed, state, w, row, col, GmFromTmem{from}, out);
        release();
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (*abort_flag && warp == kGmMmaWarp && lane == 0) {
    // products in flight still write TMEM and read shared memory: one more
    // commit completes after all of them
    const uint32_t bar = accempty;  // no role uses it any more
    asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
    mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc_commit(bar);
    mbar_wait(bar, 0);
  }
  __syncthreads();
  if (warp == kGmMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols));
  }
}

}  // namespace ra
