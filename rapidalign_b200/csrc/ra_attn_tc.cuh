// ra_attn_tc.cuh -- kernel attention on the tensor cores: head widths that are
// multiples of 8 up to 128 (padded to DP = 32, 64 or 128 with zeros).
//
// A CTA owns a tile of 128 rows of one graph and head (rows = TMEM lanes) and
// streams the other side in tiles of KT rows:
//   forward   rows = queries:  S = Q K^T;  P to TMEM;  O += P V
//   dq        rows = queries:  S = Q K^T, dP = dO V^T;  dU to TMEM;  dQ += dU K
//   dk, dv    rows = keys:     S^T = K Q^T, dP^T = V dO^T;  P^T, dU^T to TMEM;
//                              dV += P^T dO, dK += dU^T Q
// The two backward kernels each make S and dP (7 products instead of 5), so
// every result has one writer: no atomics, bitwise repeatable.
// What bounds them is not the tensor core (S and P V take 2 x 128 cycles a
// 128 x 64 tile at DP = 64) but the chain of a tile: products, TMEM load, 10 fp32
// operations and an EX2 a score with positions (17 instructions in all, the
// packed two-lane forms counted once), barrier.  So the flow within a CTA is
// simple -- all threads wait for the products, work on the scores, one thread
// issues the next products -- and two to four CTAs on an SM hide each other's
// waits: 0.41 to 0.47 instructions a cycle and scheduler, 10 % less with three
// CTAs in place of four.
// Measured, forward / dq / dk, dv in us: 512 graphs of 64-512 points, 4 heads on 2
// of 64, positions, bf16 293 / 329 / 368; 32 graphs of 33-2048, 8 heads of 128, cap,
// bf16 498 / 539 / 682 (322 TFLOP/s of 14 D operations a score); 256 graphs of
// 64-512, 4 heads of 32, positions, fp32 143 / 218 / 276.
//
// Tiles come by TMA in boxes of 64 columns (32 at DP = 32) with 128-byte (64)
// swizzle and are read K-major (S, dP) and MN-major (P V, dU K) from one copy.
// (Copied by the threads with cp.async 16 bytes each, the issue alone took 2,000
// to 3,000 cycles a tile.)  A streamed tile's rows behind the graph's end and
// masked rows are set to zero in shared memory before any product, so whatever
// those hold reaches none.  What a tile needs of its rows besides (positions,
// statistics) is loaded into registers an iteration ahead.
//
// fp32 inputs are fp16 pairs (hi + lo, one power of two for each graph and key head
// of a tensor, so that a graph's precision is its own), three products for one; the
// two small ones have an accumulator of their own where TMEM has room (the tensor
// core drops the bits below an accumulator's last one at each step: a third of the
// steps on the large sums, a third of the loss).  That loss grows with the sum (of
// dk over 5000 queries 5e-6, of 128-wide heads 1.5e-5), so a sum of fp32 is taken
// in rounds, which are added up in the results' memory with rounding: 512 rows for
// the output, dk and dv, 256 for dq, whose D and dP add their own errors, 128 for dk
// and dv without the second accumulator.  Then each is off by 3e-7 to 9e-7 at any
// length.  (256 rows for all cost 12 % of a step on graphs of 64-512 points.)
// P of 16-bit inputs is a pair too where the output is kept unrounded for a
// backward (D_i = do.o wants it); dU is one 16-bit number for 16-bit inputs (half
// a step, independent between elements).  The dq kernel also sums dS: the sum
// is what D_i was off by, since each row's P add up to 1, and it puts D_i right
// for the positions and for the dk, dv kernel.
// In fp16 P is held 2^7 up, and dU in units of the power of two that keeps
// 2 dim max |do| max |v| >= |dU| / slope below 2^14: v of the graph and key head,
// do of the row for dq (rows are lanes, the unit comes out of a lane's results) and
// of the graph's rows for dk, which adds them up.
#pragma once

#include <new>

#include <cuda.h>

#include "ra_attn.cuh"
#include "ra_tcprim.cuh"

namespace ra {

// Bounds: bits of the largest finite magnitude of each tensor in each graph and key
// head (for q and do: in the heads that share it), [4][graphs][kv_heads].
enum AttnWord { kWq = 0, kWk = 1, kWv = 2, kWdo = 3 };

struct AttnMap {  // 16-bit operand, or its halves
  CUtensorMap hi, lo;
};
struct AttnTcArgs {
  AttnMap q, k, v, go;
  const unsigned *words;  // bounds; not read where nothing is scaled
  int splits;             // forward: key ranges of a row tile
  float *part_o;          // [splits][num_q][heads][dim], unnormalised
  float2 *part_s;         // [splits][heads][num_q] (m, l)
  int pair_p;             // forward of 16-bit inputs: P as a pair
  int no_mma;             // test hook: no products, so that the waits for them expire
};

// Bounded waits, which end early where no products are made (the test hook).  With
// a limit in a register the dq kernel spilled, 11 % of its time at 64-wide heads;
// with tile_wait's test in its loop the dk, dv kernel did, 4 %.
__device__ __forceinline__ bool tile_wait(const AttnTcArgs &X, uint32_t bar, uint32_t parity) {
  for (unsigned it = 0; it < kTcSpinLimit; ++it) {
    if (mbar_wait(bar, parity, 1)) return true;
    if ((it & 4095) == 4095 && X.no_mma) return false;
  }
  return false;
}
__device__ __forceinline__ bool products_done(const AttnTcArgs &X, uint32_t bar, uint32_t parity) {
  return !X.no_mma && mbar_wait(bar, parity);
}

struct KindBf16 {
  using T = __nv_bfloat16;
  static constexpr bool bf16 = true, pair = false;
};
struct KindF16 {
  using T = __half;
  static constexpr bool bf16 = false, pair = false;
};
struct KindF32 {
  using T = float;
  static constexpr bool bf16 = false, pair = true;
};

// exponent that brings a largest magnitude into [2^13, 2^14)
__device__ __forceinline__ int attn_exp(float top) {
  if (!(top > 0.f)) return 0;
  int e;
  frexpf(top, &e);
  e = 14 - e;
  return e > 100 ? 100 : (e < -100 ? -100 : e);
}
// Scales of one graph and key head.
template <class Kind>
struct AttnScales {
  const unsigned *words;  // of this graph and head
  int64_t n;
  __device__ __forceinline__ void init(const AttnArgs &A, const AttnTcArgs &X, const AttnSegs &rows,
                                       int64_t tile, int64_t row, int hk) {
    if (Kind::bf16) return;
    n = A.graphs * A.kv_heads;
    words = X.words + rows.graph_of_tile(A.graphs, tile, row) * A.kv_heads + hk;
  }
  __device__ __forceinline__ float top(int w) const { return __uint_as_float(words[w * n]); }
  // of a tensor's halves
  __device__ __forceinline__ int elem(int w) const { return Kind::pair ? attn_exp(top(w)) : 0; }
  // of dU: 2 dim max |do| max |v| bounds |dP - D|
  __device__ __forceinline__ int du(float top_do, int dim) const {
    return Kind::bf16 ? 0 : attn_exp(2.f * dim * top_do * top(kWv));
  }
};

// Swizzled tiles: [chunk of CW columns][row][CW]; eight rows make an atom.
template <int DP>
constexpr int kCw = DP >= 64 ? 64 : 32;  // columns of a box
template <int DP>
__device__ __forceinline__ uint64_t tile_desc(uint32_t s, uint32_t lbo) {
  constexpr uint64_t sbo = 8 * kCw<DP> * 2, mode = DP >= 64 ? 2 : 4;
  return (uint64_t)((s >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) | ((sbo >> 4) << 32) |
         (1ull << 46) | (mode << 61);
}
// byte offset of 16 columns (K-major) in a tile of ROWS rows
template <int ROWS, int DP>
__host__ __device__ constexpr int k_step(int k) {
  return k * 16 / kCw<DP> * (ROWS * kCw<DP> * 2) + k * 16 % kCw<DP> * 2;
}
__host__ __device__ constexpr uint32_t attn_idesc(int N, bool bf16, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) |
         ((uint32_t)(N >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// One operand tile in shared memory: hi, then lo (pairs only).
template <int ROWS, int DP>
constexpr int tile_bytes = ROWS * DP * 2;

__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap *map, int col, int head,
                                         int row, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(col), "r"(head), "r"(row), "r"(mbar)
      : "memory");
}
// One thread: rows row0 .. of a head into a tile, BR rows a box; the barrier
// expects tile_bytes (twice for pairs).
template <class Kind, int ROWS, int DP, int BR>
__device__ __forceinline__ void load_tile(uint32_t dst, const AttnMap &op, int head, int row0,
                                          uint32_t mbar) {
#pragma unroll
  for (int h = 0; h < (Kind::pair ? 2 : 1); ++h)
#pragma unroll
    for (int c = 0; c < DP / kCw<DP>; ++c)
#pragma unroll
      for (int r = 0; r < ROWS; r += BR)
        tma_rows(dst + h * tile_bytes<ROWS, DP> + (c * ROWS + r) * kCw<DP> * 2,
                 h ? &op.lo : &op.hi, c * kCw<DP>, head, row0 + r, mbar);
}
// This thread's row of a streamed tile to zero.
template <class Kind, int ROWS, int DP>
__device__ __forceinline__ void zero_row(uint8_t *tile, int row) {
#pragma unroll 1
  for (int h = 0; h < (Kind::pair ? 2 : 1); ++h)
#pragma unroll 1
    for (int c = 0; c < DP / kCw<DP>; ++c) {
      uint4 *p = reinterpret_cast<uint4 *>(tile + h * tile_bytes<ROWS, DP> +
                                           (c * ROWS + row) * kCw<DP> * 2);
#pragma unroll
      for (int k = 0; k < kCw<DP> / 8; ++k) p[k] = make_uint4(0, 0, 0, 0);
    }
}

// D (+)= A B^T over the head width: A 128 rows, B N rows, both K-major
template <class Kind, int N, int DP>
__device__ __forceinline__ void products_rows(uint32_t d, uint32_t a, uint32_t b) {
  constexpr uint32_t idesc = attn_idesc(N, Kind::bf16, false);
  constexpr int P = Kind::pair ? 3 : 1;
#pragma unroll
  for (int p = 0; p < P; ++p) {  // lo hi, hi lo, hi hi: the small ones first
    const uint32_t ap = a + (Kind::pair && p == 0 ? tile_bytes<128, DP> : 0);
    const uint32_t bp = b + (Kind::pair && p == 1 ? tile_bytes<N, DP> : 0);
    const uint64_t da = tile_desc<DP>(ap, 16), db = tile_desc<DP>(bp, 16);
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
      mma_ss(d, da + (uint64_t)(k_step<128, DP>(k) >> 4), db + (uint64_t)(k_step<N, DP>(k) >> 4),
             idesc, p > 0 || k > 0);
  }
}
// D[128, DP] (+)= W[128, KT] X[KT, DP]: W in TMEM (per 32 columns of the
// scores 16 columns of hi, 16 of lo), X a streamed tile read MN-major
// SMALL: the small products of pairs go to the accumulator behind D
template <class Kind, int KT, int DP, bool SMALL>
__device__ __forceinline__ void products_weighted(uint32_t d, uint32_t w, uint32_t x, bool w_pair,
                                                  bool more) {
  constexpr uint32_t idesc = attn_idesc(DP, Kind::bf16, true);
  const int first = Kind::pair || w_pair ? 0 : 2;
  uint32_t acc = more;
#pragma unroll
  for (int p = 0; p < 3; ++p) {  // lo hi, hi lo (pairs of x only), hi hi
    if (p < first || (p == 1 && !Kind::pair)) continue;
    const uint64_t dx = tile_desc<DP>(x + (Kind::pair && p == 1 ? tile_bytes<KT, DP> : 0),
                                      KT * kCw<DP> * 2);
    if (SMALL && p == 2) acc = more;
#pragma unroll
    for (int k = 0; k < KT / 16; ++k) {
      mma_ts(SMALL && p < 2 ? d + DP : d, w + (k >> 1) * 32 + (k & 1) * 8 + (p == 0 ? 16 : 0),
             dx + (uint64_t)(k * 16 * kCw<DP> * 2 >> 4), idesc, acc);
      acc = 1;
    }
  }
}

template <class Kind>
__device__ __forceinline__ uint32_t pack_kind(float a, float b) {
  if (Kind::bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return bits_as<uint32_t>(v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return bits_as<uint32_t>(v);
}
template <class Kind>
__device__ __forceinline__ float2 unpack_kind(uint32_t u) {
  if (Kind::bf16) {
    return __bfloat1622float2(bits_as<__nv_bfloat162>(u));
  }
  return __half22float2(bits_as<__half2>(u));
}
// 32 weights of this lane's row to TMEM: hi, and lo where a pair is wanted
template <class Kind>
__device__ __forceinline__ void put_weights(uint32_t taddr, const float (&v)[32], bool pair) {
  uint32_t h[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) h[j] = pack_kind<Kind>(v[2 * j], v[2 * j + 1]);
  tmem_st16(taddr, h);
  if (pair) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 b = unpack_kind<Kind>(h[j]);
      h[j] = pack_kind<Kind>(v[2 * j] - b.x, v[2 * j + 1] - b.y);
    }
    tmem_st16(taddr + 16, h);
  }
}

// Positions of a streamed tile in shared memory: x, y, z of its rows.
template <int R>
struct TilePos {
  float c[3][R];
  __device__ __forceinline__ void put(int r, const AttnPos &p) {
    c[0][r] = p.x, c[1][r] = p.y, c[2][r] = p.z;
  }
};
__device__ __forceinline__ f2_t two(float v) { return pk(v, v); }
struct RowPos {  // -p of this thread's row, twice
  f2_t x, y, z;
  __device__ __forceinline__ void set(const AttnPos &p) {
    x = two(-p.x), y = two(-p.y), z = two(-p.z);
  }
};
// p_c - p_row and its square for columns c .. c + 3
struct Diff4 {
  f2_t x[2], y[2], z[2], r2[2];
  template <int R>
  __device__ __forceinline__ Diff4(const TilePos<R> &t, int c, const RowPos &p) {
    const ulonglong2 tx = *reinterpret_cast<const ulonglong2 *>(t.c[0] + c);
    const ulonglong2 ty = *reinterpret_cast<const ulonglong2 *>(t.c[1] + c);
    const ulonglong2 tz = *reinterpret_cast<const ulonglong2 *>(t.c[2] + c);
    x[0] = add2(tx.x, p.x), x[1] = add2(tx.y, p.x);
    y[0] = add2(ty.x, p.y), y[1] = add2(ty.y, p.y);
    z[0] = add2(tz.x, p.z), z[1] = add2(tz.y, p.z);
#pragma unroll
    for (int k = 0; k < 2; ++k) r2[k] = fma2(z[k], z[k], fma2(y[k], y[k], mul2(x[k], x[k])));
  }
};

// raw products of 32 scores -> base-2 scores
template <class Kind, int R>
__device__ __forceinline__ void scores32(const float (&v)[32], f2_t (&t)[16], const AttnScore &sc,
                                         bool pos, const TilePos<R> &tp, int c0,
                                         const RowPos &rp) {
  const f2_t su = two(sc.su);
  if (sc.capl > 0.f) {
    const f2_t capl = two(sc.capl);
    if (all_small(v, sc.su)) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        t[j] = mul2(capl, tanh_small2(mul2(pk(v[2 * j], v[2 * j + 1]), su)));
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        t[j] = mul2(capl, tanh2(mul2(pk(v[2 * j], v[2 * j + 1]), su)));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) t[j] = mul2(pk(v[2 * j], v[2 * j + 1]), su);
  }
  if (pos) {
    const f2_t nw = two(-sc.w);
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const Diff4 d(tp, c0 + j, rp);
      t[j / 2] = fma2(nw, d.r2[0], t[j / 2]);
      t[j / 2 + 1] = fma2(nw, d.r2[1], t[j / 2 + 1]);
    }
  }
}

// One past the last row of [0, n) that the mask leaves, for the whole CTA:
// padded tails cost nothing.  `slot`: an int in shared memory.
__device__ __forceinline__ int64_t masked_extent(const uint8_t *mask, int64_t n, int nt,
                                                 unsigned long long *slot) {
  if (mask == nullptr) return n;
  if (threadIdx.x == 0) *slot = 0;
  __syncthreads();
  int64_t last = 0;
  for (int64_t i = threadIdx.x; i < n; i += nt)
    if (mask[i]) last = i + 1;
  if (last) atomicMax(slot, (unsigned long long)last);
  __syncthreads();
  return (int64_t)*slot;
}

template <int COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
               "r"(COLS)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int COLS>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
}
__host__ __device__ constexpr int tmem_round(int c) {
  return c <= 32 ? 32 : c <= 64 ? 64 : c <= 128 ? 128 : c <= 256 ? 256 : 512;
}

// dim of a row's fp32 values (from TMEM, times f) to T and to fp32
template <class T, int DP, bool SMALL>
__device__ __forceinline__ void write_row(uint32_t taddr, float f, bool on, bool zero, int dim,
                                          T *out, float *out32, int c0 = 0, int c1 = DP) {
#pragma unroll 1
  for (int c = c0; c < c1; c += 32) {
    float v[32];
    __syncwarp();  // TMEM is read by whole warps
    tmem_ld32(taddr + c, v);
    if (SMALL) {
      float u[32];
      tmem_ld32(taddr + DP + c, u);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] += u[j];
    }
    if (!on || c >= dim) continue;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = zero ? 0.f : v[j] * f;
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      if (c + j >= dim) break;  // dim is a multiple of 8
      if (out != nullptr) {
        if (sizeof(T) == 4) {
          *reinterpret_cast<float4 *>(out + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          *reinterpret_cast<float4 *>(out + c + j + 4) =
              make_float4(v[j + 4], v[j + 5], v[j + 6], v[j + 7]);
        } else {
          T t[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) put(t + k, v[j + k]);
          uint4 u;
          memcpy(&u, t, 16);
          *reinterpret_cast<uint4 *>(out + c + j) = u;
        }
      }
      if (out32 != nullptr) {
        *reinterpret_cast<float4 *>(out32 + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        *reinterpret_cast<float4 *>(out32 + c + j + 4) =
            make_float4(v[j + 4], v[j + 5], v[j + 6], v[j + 7]);
      }
    }
  }
}

// A round of this lane's row to the sums in global memory, which only this thread
// writes: out = (keep out + f v) post, or zeros; keep 0: nothing is there yet.
template <int DP, bool SMALL>
__device__ __forceinline__ void add_round(uint32_t taddr, float f, float keep, float post, bool on,
                                          bool zero, int dim, float *out, int c0 = 0,
                                          int c1 = DP) {
#pragma unroll 1
  for (int c = c0; c < c1; c += 32) {
    float v[32];
    __syncwarp();
    tmem_ld32(taddr + c, v);
    if (SMALL) {
      float u[32];
      tmem_ld32(taddr + DP + c, u);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] += u[j];
    }
    if (!on || c >= dim) continue;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      if (c + j >= dim) break;
      float4 *at = reinterpret_cast<float4 *>(out + c + j);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      if (keep != 0.f) o = *at;
      o.x = fmaf(o.x, keep, v[j] * f) * post;
      o.y = fmaf(o.y, keep, v[j + 1] * f) * post;
      o.z = fmaf(o.z, keep, v[j + 2] * f) * post;
      o.w = fmaf(o.w, keep, v[j + 3] * f) * post;
      *at = zero ? make_float4(0.f, 0.f, 0.f, 0.f) : o;
    }
  }
}

// ---- bounds and halves ---------------------------------------------------------

struct AttnPrep {
  const void *x[4];
  int64_t row[4], head[4];
  int heads[4];
  AttnSegs segs[4];
  int64_t tiles[4];
  const uint8_t *mask[4];
  int word[4];
  uint16_t *hi[4], *lo[4];  // [rows][heads][dim]
  int64_t graphs;
  int kv_heads, dim, count;
};

// A CTA's share: a tile of 128 rows of a graph and the heads of a key head.
struct PrepUnit {
  int64_t tile_no, row0;
  int hk, group, dim8, n;  // n chunks of 8
  __device__ __forceinline__ PrepUnit(const AttnPrep &p, int t) {
    hk = (int)(blockIdx.x % p.kv_heads);
    tile_no = blockIdx.x / p.kv_heads;
    n = 0;
    if (tile_no >= p.tiles[t]) return;
    const int4 tile = p.segs[t].tile(tile_no, p.segs[t]);
    group = p.heads[t] / p.kv_heads;
    dim8 = p.dim >> 3;
    row0 = tile.x;
    n = tile.y * group * dim8;
  }
  __device__ __forceinline__ unsigned *word(const AttnPrep &p, int t, unsigned *words) const {
    const int64_t g = p.segs[t].graph_of_tile(p.graphs, tile_no, row0);
    return words + (p.word[t] * p.graphs + g) * p.kv_heads + hk;
  }
  // row, head and chunk of the e-th chunk
  __device__ __forceinline__ void at(int e, int64_t &i, int &h, int &c) const {
    const unsigned r = (unsigned)e / dim8, k = r / group;
    c = e - r * dim8;
    i = row0 + k;
    h = hk * group + (r - k * group);
  }
};
template <class T>
__device__ __forceinline__ void load8(const T *x, bool wide, float (&v)[8]) {
  if (wide) {
    uint4 u[sizeof(T) / 2];
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) u[k] = reinterpret_cast<const uint4 *>(x)[k];
    T t[8];
    memcpy(t, u, sizeof(t));
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = to_f(t[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = to_f(x[k]);
  }
}
template <class T>
__device__ __forceinline__ bool rows_wide(const AttnPrep &p, int t) {
  constexpr int e = 16 / sizeof(T);
  return ((uintptr_t)p.x[t] & 15) == 0 && p.row[t] % e == 0 && p.head[t] % e == 0;
}

// Bounds and halves, of q, k, v and do of 256 graphs of 64-512 points, 4 heads of 32:
// 43 and 50 us (one scale a tensor, without tiles: 45 and 40).
constexpr int kPrepThreads = 128;
// largest finite magnitude of each tensor in each graph and key head
template <class T>
__global__ void __launch_bounds__(kPrepThreads)
    attn_bounds_kernel(const AttnPrep p, unsigned *words) {
  const int t = blockIdx.y;
  const PrepUnit u(p, t);
  if (u.n == 0) return;
  const bool wide = rows_wide<T>(p, t);
  float top = 0.f;
#pragma unroll 4
  for (int e = threadIdx.x; e < u.n; e += kPrepThreads) {
    int64_t i;
    int h, c;
    u.at(e, i, h, c);
    if (p.mask[t] != nullptr && p.mask[t][i] == 0) continue;
    float v[8];
    load8((const T *)p.x[t] + i * p.row[t] + h * p.head[t] + c * 8, wide, v);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (fabsf(v[k]) < INFINITY) top = fmaxf(top, fabsf(v[k]));
  }
  __syncwarp();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
  unsigned *word = u.word(p, t, words);
  // maxima of bits: any order
  if ((threadIdx.x & 31) == 0 && top > 0.f) atomicMax(word, __float_as_uint(top));
}

// x 2^e = hi + lo in fp16
__global__ void __launch_bounds__(kPrepThreads)
    attn_halves_kernel(const AttnPrep p, unsigned *words) {
  const int t = blockIdx.y;
  const PrepUnit u(p, t);
  if (u.n == 0) return;
  const bool wide = rows_wide<float>(p, t);
  constexpr int B = 4;  // chunks in flight, the first ones during the search
  float v[B][8];
  int64_t to[B];
  auto load = [&](int e0) {
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int e = e0 + b * kPrepThreads;
      if (e >= u.n) break;
      int64_t i;
      int h, c;
      u.at(e, i, h, c);
      load8((const float *)p.x[t] + i * p.row[t] + h * p.head[t] + c * 8, wide, v[b]);
      to[b] = (i * p.heads[t] + h) * u.dim8 + c;
    }
  };
  load(threadIdx.x);
  __syncwarp();
  const float sc = ldexpf(1.f, attn_exp(__uint_as_float(*u.word(p, t, words))));
  for (int e0 = threadIdx.x; e0 < u.n; e0 += B * kPrepThreads) {
    if (e0 != threadIdx.x) load(e0);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (e0 + b * kPrepThreads >= u.n) break;
      __half hi[8], lo[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float y = v[b][k] * sc;
        hi[k] = __float2half_rn(y);
        lo[k] = __float2half_rn(y - __half2float(hi[k]));
      }
      uint4 w[2];
      memcpy(w, hi, 16);
      memcpy(w + 1, lo, 16);
      reinterpret_cast<uint4 *>(p.hi[t])[to[b]] = w[0];
      reinterpret_cast<uint4 *>(p.lo[t])[to[b]] = w[1];
    }
  }
}

// D_i = do_i . o_i, and the largest finite |do_i|: 2^k lanes a row and head, 8
// elements each
template <class T>
__global__ void __launch_bounds__(256) attn_delta8_kernel(const T *dout, const float *out32,
                                                          int64_t num_q, int heads, int dim,
                                                          int lanes, float *neg_d,
                                                          float *do_top) {
  const int l = threadIdx.x % lanes;
  const int64_t n = num_q * heads, step = gridDim.x * 256LL / lanes;
  // all lanes of a warp go round together: the shuffles need them
  for (int64_t r0 = (blockIdx.x * 256LL + (threadIdx.x & ~31)) / lanes; r0 < n; r0 += step) {
    const int64_t r = r0 + (threadIdx.x & 31) / lanes;
    float s = 0.f, top = 0.f;
    if (r < n && l * 8 < dim) {
      float a[8], b[8];
      load8(dout + r * dim + l * 8, true, a);
      load8(out32 + r * dim + l * 8, true, b);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        s = fmaf(a[k], b[k], s);
        if (fabsf(a[k]) < INFINITY) top = fmaxf(top, fabsf(a[k]));
      }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      s += __shfl_xor_sync(kFull, s, o);
      top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    }
    if (r < n && l == 0) {
      neg_d[(r % heads) * num_q + r / heads] = -s;
      if (do_top != nullptr) do_top[(r % heads) * num_q + r / heads] = top;
    }
  }
}

// ---- forward --------------------------------------------------------------------

// Rows of a streamed tile of the backward, with 128 threads of the CTA for every 32
// of them (32 columns of the scores a thread).  What counts is
// that warps wait at different times: 32 where four CTAs then share an SM's TMEM
// (dq of 64-wide bf16 heads: 318 us, with 64 and two CTAs 387); 128 where one
// CTA holds the TMEM anyhow (dk, dv of 128-wide heads: 671 us, with 64 756);
// else 64.
template <class Kind, int DP>
constexpr int dq_rows = 64 + (Kind::pair ? 2 : 1) * DP <= 128 ? 32 : 64;
template <class Kind, int DP>
constexpr int dkv_rows = 64 + (Kind::pair ? 4 : 2) * DP <= 128          ? 32
                         : !Kind::pair && DP == 128 || Kind::pair && DP == 64 ? 128
                                                                        : 64;
// Tiles of a round of `rows` (a power of two): 16-bit inputs have one, whose loss
// stays below their own rounding.
template <class Kind, int ROWS>
constexpr int round_tiles(int rows) {
  return Kind::pair ? rows / ROWS : 1 << 30;
}
// CTAs that fit an SM beside each other, with `regs` registers a thread
constexpr int attn_ctas(int smem, int tmem, int threads, int regs = 128) {
  int n = 65536 / (regs * threads);
  if (n > 512 / tmem) n = 512 / tmem;
  while (n > 1 && n * (smem + 1024) > 228 * 1024) --n;
  return n;
}

template <class Kind, int DP>
struct FwdCfg {
  static constexpr int KT = 64;
  static constexpr int HALF = Kind::pair ? 2 : 1;
  static constexpr int BR = KT;  // rows of a TMA box
  static constexpr int Q = HALF * tile_bytes<128, DP>, KV = HALF * tile_bytes<KT, DP>;
  static constexpr bool SMALL = Kind::pair;
  static constexpr int ROUND = round_tiles<Kind, KT>(512);
  static constexpr int TMEM = tmem_round(KT + (SMALL ? 2 : 1) * DP);
  static constexpr int pos = Q + 4 * KV;                 // TilePos<KT> [2]
  static constexpr int val = pos + 2 * KT * 12;          // unsigned [2][2]
  static constexpr int bar = val + 16, slot = bar + 40;  // slot: also the mask's extent
  static constexpr int top = slot + 8;                   // float [PARTS][128]
  // threads of a row: half of the columns each where TMEM or shared memory holds
  // fewer than four CTAs
  static constexpr int PARTS = attn_ctas(Q + 4 * KV, TMEM, 128) < 4 ? 2 : 1;
  static constexpr int NT = 128 * PARTS, C = KT / 32 / PARTS;  // 32-column chunks a thread
  static constexpr int smem = top + PARTS * 512 + 1024;        // 1024: the tiles' alignment
  static constexpr int CTAS = attn_ctas(smem, TMEM, NT, 128);
};

// Work for one thread, on the last two of NT threads' warps: issuing a tile's
// products takes 200 to 1,400 cycles, its copies 500, and the first warps fetch
// the rows.
template <int NT>
constexpr int kMmaThread = NT - 64;
template <int NT>
constexpr int kTmaThread = NT - 32;
// After an expired wait: a CTA does not leave while its copies write its shared
// memory, nor free TMEM that its products write.  The last copies of either
// buffer (`full`: the barriers; tiles t0 .. copied were asked for), and one more
// commit, which arrives after all products.
template <int NT>
__device__ __forceinline__ void drain(uint32_t full, int copied, int t0, int stages) {
  if (threadIdx.x == kTmaThread<NT> && copied >= t0) {
    if (stages == 1) mbar_wait(full, copied & 1);
    else
      for (int t = copied > t0 ? copied - 1 : t0; t <= copied; ++t)
        mbar_wait(full + 8 * (t & 1), ((t - t0) >> 1) & 1);
  }
  if (threadIdx.x == kMmaThread<NT>) {
    tc_commit(full + 16);
    mbar_wait(full + 16, 0);
  }
  __syncthreads();
  tc_fence_after();
}
// This thread's row of the next streamed tile, fetched an iteration ahead.
struct NextRow {
  AttnPos p;
  float nm, rl, nd;  // dk, dv: the query's statistics
  bool on;
};
__device__ __forceinline__ uint8_t *align1024(uint8_t *p) {
  return p + ((1024 - (smem_u32(p) & 1023)) & 1023);
}

template <class Kind, int DP>
__global__ void __launch_bounds__(FwdCfg<Kind, DP>::NT, FwdCfg<Kind, DP>::CTAS)
    attn_tc_fwd_kernel(const AttnArgs A, const __grid_constant__ AttnTcArgs X) {
  using C = FwdCfg<Kind, DP>;
  constexpr int KT = C::KT, NT = C::NT, PARTS = C::PARTS;
  extern __shared__ uint8_t raw_sm[];
  uint8_t *sm = align1024(raw_sm);
  const uint32_t base = smem_u32(sm);
  const uint32_t sQ = base, sK = base + C::Q, sV = sK + 2 * C::KV, bar = base + C::bar,
                 full = bar + 8;
  TilePos<KT> *kpos = reinterpret_cast<TilePos<KT> *>(sm + C::pos);
  unsigned *kval = reinterpret_cast<unsigned *>(sm + C::val);
  float *top = reinterpret_cast<float *>(sm + C::top);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = threadIdx.x & 127, part = warp >> 2;  // its share of the columns

  const int64_t item = blockIdx.x;
  const int split = (int)(item % X.splits);
  const int h = (int)(item / X.splits % A.heads), hk = h / (A.heads / A.kv_heads);
  const int4 tile = A.qs.tile(item / X.splits / A.heads, A.ks);
  const int i0 = tile.x, nq = tile.y, j0 = tile.z;
  const int64_t i = i0 + row;
  const bool row_on = row < nq && (A.q_mask == nullptr || A.q_mask[i] != 0);
  const int nk = (int)masked_extent(A.k_mask ? A.k_mask + j0 : nullptr, tile.w, NT,
                                    reinterpret_cast<unsigned long long *>(sm + C::slot));
  // no row to work for: no keys to see
  const int64_t all = __syncthreads_or(row_on) ? (nk + KT - 1) / KT : 0;
  const int t0 = (int)(all * split / X.splits);
  int t1 = (int)(all * (split + 1) / X.splits);

  volatile int *copied = reinterpret_cast<int *>(sm + C::bar + 32);  // the last tile asked for
  auto issue = [&](int t, uint32_t more) {
    const uint32_t fb = full + 8 * (t & 1);
    *copied = t;
    mbar_expect_tx(fb, more + 2 * C::KV);
    load_tile<Kind, KT, DP, C::BR>(sK + (t & 1) * C::KV, X.k, hk, j0 + t * KT, fb);
    load_tile<Kind, KT, DP, C::BR>(sV + (t & 1) * C::KV, X.v, hk, j0 + t * KT, fb);
  };
  NextRow nx;
  auto fetch = [&](int t) {
    const int r = threadIdx.x;
    if (r >= KT) return;
    const int64_t j = j0 + t * KT + r;
    nx.on = t * KT + r < nk && (A.k_mask == nullptr || A.k_mask[j] != 0);
    nx.p = nx.on ? pos_of(A.k_pos, A.pos_dim, j) : AttnPos{0.f, 0.f, 0.f};
  };
  auto settle = [&](int t) {  // the tile is there: its rows' marks and positions
    const int r = threadIdx.x, b = t & 1;
    if (r < KT) {
      const unsigned bits = __ballot_sync(kFull, nx.on);
      if (lane == 0) kval[2 * b + warp] = bits;
      if (A.pos_dim > 0) kpos[b].put(r, nx.p);
      if (!nx.on) {
        zero_row<Kind, KT, DP>(sm + C::Q + b * C::KV, r);
        zero_row<Kind, KT, DP>(sm + C::Q + (2 + b) * C::KV, r);
      }
    }
    fence_async_smem();
  };
  if (warp == 1) tmem_alloc<C::TMEM>(base + C::slot);
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    mbar_init(full, 1);
    mbar_init(full + 8, 1);
    mbar_init(full + 16, 1);
    *copied = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (t0 < t1) {
      issue(t0, C::Q);
      load_tile<Kind, 128, DP, C::BR>(sQ, X.q, h, i0, full + 8 * (t0 & 1));
    }
  }
  bool bad = false;
  if (t0 < t1) fetch(t0);
  __syncwarp();
  AttnScales<Kind> scl;
  scl.init(A, X, A.qs, item / X.splits / A.heads, i0, hk);
  const int es = scl.elem(kWq) + scl.elem(kWk), ev = scl.elem(kWv);
  __syncthreads();
  if (t0 < t1) {
    bad = !tile_wait(X, full + 8 * (t0 & 1), 0);
    settle(t0);
  }
  tc_fence_before();
  if ((bad = __syncthreads_or(bad))) t1 = t0;  // no first tile
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + C::slot);
  const uint32_t tS = tmem, tO = tmem + KT, lane_off = (uint32_t)(32 * (warp & 3)) << 16;

  AttnScore sc;
  sc.init(A, h);
  sc.su *= ldexpf(1.f, -es);
  RowPos rp;
  rp.set(row_on ? pos_of(A.q_pos, A.pos_dim, i) : AttnPos{0.f, 0.f, 0.f});
  constexpr float kUp = Kind::bf16 ? 0.f : 7.f;  // P is held 2^kUp up
  const bool p_pair = Kind::pair || X.pair_p;
  float m = -INFINITY, l = 0.f;  // m: the reference the sums are relative to; l: this part's
  float keep = 0.f;              // of earlier rounds, which are relative to earlier references
  // the row's columns: every PARTS-th 32, or what there is
  constexpr int W = DP / PARTS < 32 ? 32 : DP / PARTS;
  const int c0 = W * part, c1 = DP < c0 + W ? DP : c0 + W;
  auto dest = [&]() {  // of the sums: the output, or this range's
    return X.splits > 1 ? X.part_o + ((split * A.num_q + i) * A.heads + h) * A.dim
                        : (float *)A.out + (i * A.heads + h) * A.dim;
  };
  unsigned phase = 0;

  auto mma = [&]() { return threadIdx.x == kMmaThread<NT> && !X.no_mma; };
  if (t0 < t1 && mma()) {
    products_rows<Kind, KT, DP>(tS, sQ, sK + (t0 & 1) * C::KV);
    tc_commit(bar);
  }
  for (int t = t0; t < t1; ++t) {
    const int b = t & 1;
    bad |= !tile_wait(X, bar, phase);
    phase ^= 1;
    tc_fence_after();
    if (t + 1 < t1) {  // the products on its buffers are done
      if (threadIdx.x == kTmaThread<NT> && !bad) issue(t + 1, 0);
      fetch(t + 1);
    }
    if (Kind::pair && t > t0 && (t - t0) % C::ROUND == 0) {
      add_round<DP, C::SMALL>(tO + lane_off, ldexpf(1.f, -ev), keep, 1.f, row_on, false, A.dim,
                              dest(), c0, c1);
      keep = 1.f;
    }
    __syncwarp();
    f2_t s2[C::C][16];
    float mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < C::C; ++c) {
      const int at = C::C * part + c;
      float v[32];
      tmem_ld32(tS + lane_off + 32 * at, v);
      scores32<Kind>(v, s2[c], sc, A.pos_dim > 0, kpos[b], 32 * at, rp);
      const unsigned bits = kval[2 * b + at];
      if (bits != kFull) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float x, y;
          upk(s2[c][j], x, y);
          s2[c][j] = pk((bits >> (2 * j)) & 1 ? x : -INFINITY,
                        (bits >> (2 * j + 1)) & 1 ? y : -INFINITY);
        }
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) mx = fmaxf(mx, fmaxf(lo_of(s2[c][j]), hi_of(s2[c][j])));
    }
    if (PARTS > 1) {  // the row's: the four pairs of warps that share rows
      top[part * 128 + row] = mx;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
      mx = fmaxf(mx, top[(part ^ 1) * 128 + row]);
    }
    // the reference follows the maximum only where it grew by more than 2^8:
    // sums and O stay relative to one reference, whichever it is
    const bool grow = mx > m + 8.f;  // also from -inf
    const float mn = grow ? mx : m;
    if (__any_sync(kFull, grow)) {
      const float f = m > -INFINITY ? ex2(m - mn) : 0.f;
      l *= f;
      if (Kind::pair) keep *= f;
      if ((t - t0) % C::ROUND != 0) {
#pragma unroll 1
        for (int c = 32 * part; c < (C::SMALL ? 2 : 1) * DP; c += 32 * PARTS) {
          float o[32];
          tmem_ld32(tO + lane_off + c, o);
          uint32_t u[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) u[j] = __float_as_uint(o[j] * f);
          tmem_st32(tO + lane_off + c, u);
        }
      }
      m = mn;
    }
    const f2_t ref = two(kUp - (m > -INFINITY ? m : 0.f));
    f2_t sum[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < C::C; ++c) {
      float v[32];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float x, y;
        upk(add2(s2[c][j], ref), x, y);
        v[2 * j] = ex2(x);
        v[2 * j + 1] = ex2(y);
        sum[j & 1] = add2(sum[j & 1], pk(v[2 * j], v[2 * j + 1]));
      }
      put_weights<Kind>(tS + lane_off + 32 * (C::C * part + c), v, p_pair);
    }
    const f2_t both = add2(sum[0], sum[1]);
    l += lo_of(both) + hi_of(both);
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    if (t + 1 < t1) {
      // (copies that are not asked for any more are not waited for)
      bad = bad || !tile_wait(X, full + 8 * (b ^ 1), ((t + 1 - t0) >> 1) & 1);
      settle(t + 1);
    }
    tc_fence_before();
    if ((bad = __syncthreads_or(bad))) break;
    if (mma()) {
      tc_fence_after();
      products_weighted<Kind, KT, DP, C::SMALL>(tO, tS, sV + b * C::KV, p_pair,
                                                (t - t0) % C::ROUND != 0);
      if (t + 1 < t1) products_rows<Kind, KT, DP>(tS, sQ, sK + (b ^ 1) * C::KV);
      tc_commit(bar);
    }
  }
  if (t0 < t1 && !bad) {
    bad = !tile_wait(X, bar, phase);
    tc_fence_after();
  }
  if ((bad = __syncthreads_or(bad))) {
    if (threadIdx.x == 0) atomicOr(A.status, 1);
    drain<NT>(full, *copied, t0, 2);
  }

  if (PARTS > 1) {
    if (part > 0) top[row] = l;
    __syncthreads();
    if (part == 0) top[row] = l += top[row];
    __syncthreads();
    l = top[row];
  }
  const bool any = l > 0.f || l != l;
  const bool empty = !row_on || !any || t0 >= t1;
  using T = typename Kind::T;
  const float unscale = ldexpf(1.f, -ev);
  const bool in = row < nq;
  const float r = empty ? 0.f : 1.f / l;
  const bool rounds = Kind::pair && t1 - t0 > C::ROUND;
  if (rounds)
    add_round<DP, C::SMALL>(tO + lane_off, unscale, keep, X.splits > 1 ? 1.f : r, in, empty, A.dim,
                            dest(), c0, c1);
  if (X.splits > 1) {
    if (!rounds)
      write_row<float, DP, C::SMALL>(tO + lane_off, unscale, in, empty, A.dim, dest(), nullptr, c0,
                                     c1);
    if (in && part == 0)
      X.part_s[((int64_t)split * A.heads + h) * A.num_q + i] =
          make_float2(empty ? -INFINITY : (m > -INFINITY ? m : 0.f) - kUp, empty ? 0.f : l);
  } else {
    const int64_t at = (i * A.heads + h) * A.dim;
    if (!rounds)
      write_row<T, DP, C::SMALL>(tO + lane_off, unscale * r, in, empty, A.dim, (T *)A.out + at,
                                 A.out32 ? A.out32 + at : nullptr, c0, c1);
    if (in && part == 0 && A.neg_m)
      A.put_stats(h, i, empty ? INFINITY : (m > -INFINITY ? m : 0.f) - kUp, r);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<C::TMEM>(tmem);
  }
}

// One more key range (its maximum and sum st, its values x) joined to a row's.
template <int COLS>
__device__ __forceinline__ void join_range(float2 st, const float (&x)[COLS], float &m, float &l,
                                           float (&acc)[COLS]) {
  const float mx = fmaxf(m, st.x);
  const float keep = m > -INFINITY ? ex2(m - mx) : 0.f;
  const float f = st.x > -INFINITY ? ex2(st.x - mx) : 0.f;  // else l and o are 0
  l = fmaf(st.y, f, l * keep);
#pragma unroll
  for (int c = 0; c < COLS; ++c) acc[c] = fmaf(f, x[c], acc[c] * keep);
  m = mx;
}
constexpr int kJoinCols = 128 / 32;  // columns a lane: ranges are for widths up to 128
// Joins the key ranges of the rows, a warp a row, the maximum as it goes.
template <class T>
__global__ void __launch_bounds__(256)
    attn_join_kernel(const AttnArgs A, int splits, const float *part_o, const float2 *part_s) {
  const int lane = threadIdx.x & 31;
  const int64_t n = A.num_q * A.heads, r = blockIdx.x * 8LL + (threadIdx.x >> 5), i = r / A.heads;
  if (r >= n) return;
  const int h = (int)(r % A.heads);
  const float2 *ps = part_s + (int64_t)h * A.num_q + i;
  float m = -INFINITY, l = 0.f, acc[kJoinCols] = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float *po = part_o + (s * n + r) * A.dim;
    float x[kJoinCols];
#pragma unroll
    for (int c = 0; c < kJoinCols; ++c)
      x[c] = lane + 32 * c < A.dim ? po[lane + 32 * c] : 0.f;
    join_range(ps[s * n], x, m, l, acc);
  }
  const bool any = l > 0.f || l != l;
  const float rl = any ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < kJoinCols; ++c)
    if (lane + 32 * c < A.dim) {
      const float o = any ? acc[c] * rl : 0.f;
      put((T *)A.out + r * A.dim + lane + 32 * c, o);
      if (A.out32) A.out32[r * A.dim + lane + 32 * c] = o;
    }
  if (lane == 0 && A.neg_m) A.put_stats(h, i, any ? m : INFINITY, rl);
}
// The same with 32 warps a row, for many ranges: a warp takes every 32nd, then
// the warps are joined, a column a warp.
template <class T>
__global__ void __launch_bounds__(1024)
    attn_join_many_kernel(const AttnArgs A, int splits, const float *part_o, const float2 *part_s) {
  constexpr int WARPS = 32;
  __shared__ float so[WARPS][kJoinCols * 32 + 1];
  __shared__ float2 sl[WARPS];
  constexpr int COLS = kJoinCols;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n = A.num_q * A.heads, r = blockIdx.x, i = r / A.heads;
  const int h = (int)(r % A.heads);
  const float2 *ps = part_s + (int64_t)h * A.num_q + i;
  float m = -INFINITY, l = 0.f, acc[COLS] = {};
#pragma unroll 8
  for (int s = warp; s < splits; s += WARPS) {
    const float2 st = ps[s * n];
    const float *po = part_o + (s * n + r) * A.dim;
    float x[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) x[c] = lane + 32 * c < A.dim ? po[lane + 32 * c] : 0.f;
    join_range(st, x, m, l, acc);
  }
#pragma unroll
  for (int c = 0; c < COLS; ++c)
    if (lane + 32 * c < A.dim) so[warp][lane + 32 * c] = acc[c];
  if (lane == 0) sl[warp] = make_float2(m, l);
  __syncthreads();
  const float2 st = sl[lane];
  m = st.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  const float f = st.x > -INFINITY ? ex2(st.x - m) : 0.f;
  l = warp_sum(st.y * f);
  const bool any = l > 0.f || l != l;
  const float rl = any ? 1.f / l : 0.f;
  for (int d = warp; d < A.dim; d += WARPS) {
    float o = warp_sum(so[lane][d] * f);
    o = any ? o * rl : 0.f;
    if (lane == 0) {
      put((T *)A.out + r * A.dim + d, o);
      if (A.out32) A.out32[r * A.dim + d] = o;
    }
  }
  if (threadIdx.x == 0 && A.neg_m) A.put_stats(h, i, any ? m : INFINITY, rl);
}

// ---- backward -------------------------------------------------------------------

// The elementwise part of 32 scores of a row, four at a time, all in one pass
// so that only the scores and dP are held.  `v` raw products, `dp` raw dP; out:
// dU in dp (and P in v where the rows are keys).
// CAP: no cap; capped, all products small; capped.  POS, PG: positions and
// their gradients are there.
enum AttnCap { kNoCap, kCapSmall, kCapAny };
template <AttnCap CAP>
__device__ __forceinline__ f2_t cap_tanh(f2_t u) {
  return CAP == kCapSmall ? tanh_small2(u) : tanh2(u);
}
struct BwdRow {
  AttnScore sc;
  float dps, up;  // of raw dP; of dU
  RowPos p;
};
// dq: the row's statistics, and its sums of dS, dS (p_j - p_i), dS r^2 and of
// P (p_j - p_i), P r^2, each in two lanes
struct DqSums {
  f2_t ds = 0, g[4] = {}, q[4] = {};
};
// MASKED: some of the 32 columns are not there (`bits`).
template <class Kind, AttnCap CAP, bool POS, bool PG, bool MASKED, int R>
__device__ __forceinline__ void dq_elements(float (&v)[32], float (&dp)[32], const BwdRow &B,
                                            float m, float rl, float delta, unsigned bits,
                                            const TilePos<R> &tp, int c0, DqSums &S) {
  const f2_t su = two(B.sc.su), nm = two(-m), nw = two(-B.sc.w), dps = two(B.dps),
             nd = two(-delta), r2l = two(rl), up = two(B.up);
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    Diff4 *d = nullptr;
    alignas(Diff4) char raw[sizeof(Diff4)];
    if (POS) d = new (raw) Diff4(tp, c0 + j, B.p);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = j + 2 * k;
      f2_t t, th;
      if (CAP != kNoCap) {
        th = cap_tanh<CAP>(mul2(pk(v[e], v[e + 1]), su));
        t = fma2(th, two(B.sc.capl), nm);
      } else {
        t = fma2(pk(v[e], v[e + 1]), su, nm);
      }
      if (POS) t = fma2(nw, d->r2[k], t);
      float x, y;
      upk(t, x, y);
      x = ex2(x), y = ex2(y);
      if (MASKED) {
        x = (bits >> e) & 1 ? x : 0.f;
        y = (bits >> (e + 1)) & 1 ? y : 0.f;
      }
      const f2_t p = mul2(pk(x, y), r2l);
      f2_t ds = mul2(p, fma2(pk(dp[e], dp[e + 1]), dps, nd));
      S.ds = add2(S.ds, ds);
      if (PG) {
        S.g[0] = fma2(ds, d->x[k], S.g[0]), S.q[0] = fma2(p, d->x[k], S.q[0]);
        S.g[1] = fma2(ds, d->y[k], S.g[1]), S.q[1] = fma2(p, d->y[k], S.q[1]);
        S.g[2] = fma2(ds, d->z[k], S.g[2]), S.q[2] = fma2(p, d->z[k], S.q[2]);
        S.g[3] = fma2(ds, d->r2[k], S.g[3]), S.q[3] = fma2(p, d->r2[k], S.q[3]);
      }
      if (CAP != kNoCap) ds = mul2(ds, fma2(mul2(th, two(-1.f)), th, two(1.f)));
      if (!Kind::bf16) ds = mul2(ds, up);
      upk(ds, dp[e], dp[e + 1]);
    }
  }
}
// dk, dv: the columns' (queries') statistics in shared memory
template <int R>
struct TileStat {
  float nm[R], rl[R], nd[R];  // -m, 1 / l, -D
};
template <class Kind, AttnCap CAP, bool POS, bool PG, int R>
__device__ __forceinline__ void dkv_elements(float (&v)[32], float (&dp)[32], const BwdRow &B,
                                             float p_up, const TileStat<R> &st,
                                             const TilePos<R> &tp, int c0, f2_t (&g)[3]) {
  const f2_t su = two(B.sc.su), nw = two(-B.sc.w), dps = two(B.dps), up = two(B.up);
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    Diff4 *d = nullptr;
    alignas(Diff4) char raw[sizeof(Diff4)];
    if (POS) d = new (raw) Diff4(tp, c0 + j, B.p);
    const ulonglong2 nm = *reinterpret_cast<const ulonglong2 *>(st.nm + c0 + j);
    const ulonglong2 rl = *reinterpret_cast<const ulonglong2 *>(st.rl + c0 + j);
    const ulonglong2 nd = *reinterpret_cast<const ulonglong2 *>(st.nd + c0 + j);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = j + 2 * k;
      f2_t t, th;
      if (CAP != kNoCap) {
        th = cap_tanh<CAP>(mul2(pk(v[e], v[e + 1]), su));
        t = fma2(th, two(B.sc.capl), k ? nm.y : nm.x);
      } else {
        t = fma2(pk(v[e], v[e + 1]), su, k ? nm.y : nm.x);
      }
      if (POS) t = fma2(nw, d->r2[k], t);
      float x, y;
      upk(t, x, y);
      f2_t p = mul2(pk(ex2(x), ex2(y)), k ? rl.y : rl.x);
      f2_t ds = mul2(p, fma2(pk(dp[e], dp[e + 1]), dps, k ? nd.y : nd.x));
      if (PG) {
        g[0] = fma2(ds, d->x[k], g[0]);
        g[1] = fma2(ds, d->y[k], g[1]);
        g[2] = fma2(ds, d->z[k], g[2]);
      }
      if (CAP != kNoCap) ds = mul2(ds, fma2(mul2(th, two(-1.f)), th, two(1.f)));
      if (!Kind::bf16) {
        ds = mul2(ds, up);
        p = mul2(p, two(p_up));
      }
      upk(ds, dp[e], dp[e + 1]);
      upk(p, v[e], v[e + 1]);
    }
  }
}
__device__ __forceinline__ float sum_of(f2_t v) { return lo_of(v) + hi_of(v); }

template <class Kind, int DP>
struct DqCfg {
  static constexpr int KT = dq_rows<Kind, DP>;
  static constexpr int HALF = Kind::pair ? 2 : 1;
  static constexpr int BR = KT < dkv_rows<Kind, DP> ? KT : dkv_rows<Kind, DP>;
  static constexpr int Q = HALF * tile_bytes<128, DP>, KV = HALF * tile_bytes<KT, DP>;
  // two CTAs on an SM are worth more than a second buffer
  static constexpr int STAGES = 2 * Q + 4 * KV <= 100 * 1024 ? 2 : 1;
  static constexpr bool SMALL = Kind::pair;
  static constexpr int ROUND = round_tiles<Kind, KT>(256);
  static constexpr int TMEM = tmem_round(2 * KT + (SMALL ? 2 : 1) * DP);
  static constexpr int NT = 128 * (KT / 32);
  static constexpr int pos = 2 * Q + 2 * STAGES * KV;  // TilePos<KT> [2]
  static constexpr int val = pos + 2 * KT * 12;
  static constexpr int bar = val + 16, slot = bar + 40;
  static constexpr int smem = slot + 8 + 1024;
  static constexpr int CTAS = attn_ctas(smem, TMEM, NT);
};

template <class Kind, int DP>
__global__ void __launch_bounds__(DqCfg<Kind, DP>::NT, DqCfg<Kind, DP>::CTAS)
    attn_tc_dq_kernel(const AttnArgs A, const __grid_constant__ AttnTcArgs X) {
  using C = DqCfg<Kind, DP>;
  constexpr int KT = C::KT, NT = C::NT;
  extern __shared__ uint8_t raw_sm[];
  uint8_t *sm = align1024(raw_sm);
  const uint32_t base = smem_u32(sm);
  const uint32_t sQ = base, sG = base + C::Q, sK = sG + C::Q, sV = sK + C::STAGES * C::KV,
                 bar = base + C::bar, full = bar + 8;
  TilePos<KT> *kpos = reinterpret_cast<TilePos<KT> *>(sm + C::pos);
  unsigned *kval = reinterpret_cast<unsigned *>(sm + C::val);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp >> 2, row = threadIdx.x & 127;  // columns 32 part.. of the tile

  const int64_t item = blockIdx.x;
  const int h = (int)(item % A.heads), hk = h / (A.heads / A.kv_heads);
  const int4 tile = A.qs.tile(item / A.heads, A.ks);
  const int i0 = tile.x, nq = tile.y, j0 = tile.z;
  const int nk = (int)masked_extent(A.k_mask ? A.k_mask + j0 : nullptr, tile.w, NT,
                                    reinterpret_cast<unsigned long long *>(sm + C::slot));
  const int64_t i = i0 + row;
  const bool in = row < nq;
  float2 st = make_float2(INFINITY, 0.f);
  if (in) st = A.stats(h, i);
  const bool live = st.y != 0.f;  // has keys, and is not masked
  int t1 = __syncthreads_or(live) ? (nk + KT - 1) / KT : 0;

  volatile int *copied = reinterpret_cast<int *>(sm + C::bar + 32);  // the last tile asked for
  auto issue = [&](int t, uint32_t more) {
    const int b = C::STAGES == 1 ? 0 : t & 1;
    const uint32_t fb = full + 8 * b;
    *copied = t;
    mbar_expect_tx(fb, more + 2 * C::KV);
    load_tile<Kind, KT, DP, C::BR>(sK + b * C::KV, X.k, hk, j0 + t * KT, fb);
    load_tile<Kind, KT, DP, C::BR>(sV + b * C::KV, X.v, hk, j0 + t * KT, fb);
  };
  NextRow nx;
  auto fetch = [&](int t) {
    const int r = threadIdx.x;
    if (r >= KT) return;
    const int64_t j = j0 + t * KT + r;
    nx.on = t * KT + r < nk && (A.k_mask == nullptr || A.k_mask[j] != 0);
    nx.p = nx.on ? pos_of(A.k_pos, A.pos_dim, j) : AttnPos{0.f, 0.f, 0.f};
  };
  auto settle = [&](int t) {
    const int r = threadIdx.x, pb = t & 1, b = C::STAGES == 1 ? 0 : pb;
    if (r < KT) {
      const unsigned bits = __ballot_sync(kFull, nx.on);
      if (lane == 0) kval[2 * pb + warp] = bits;
      if (A.pos_dim > 0) kpos[pb].put(r, nx.p);
      if (!nx.on) {
        zero_row<Kind, KT, DP>(sm + 2 * C::Q + b * C::KV, r);
        zero_row<Kind, KT, DP>(sm + 2 * C::Q + (C::STAGES + b) * C::KV, r);
      }
    }
    fence_async_smem();
  };
  auto landed = [&](int t) {
    return C::STAGES == 1 ? tile_wait(X, full, t & 1)
                          : tile_wait(X, full + 8 * (t & 1), (t >> 1) & 1);
  };
  if (warp == 1) tmem_alloc<C::TMEM>(base + C::slot);
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    mbar_init(full, 1);
    mbar_init(full + 8, 1);
    mbar_init(full + 16, 1);
    *copied = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (t1 > 0) {
      issue(0, 2 * C::Q);
      load_tile<Kind, 128, DP, C::BR>(sQ, X.q, h, i0, full);
      load_tile<Kind, 128, DP, C::BR>(sG, X.go, h, i0, full);
    }
  }
  bool bad = false;
  if (t1 > 0) fetch(0);
  __syncwarp();
  AttnScales<Kind> scl;
  scl.init(A, X, A.qs, item / A.heads, i0, hk);
  const int ek = scl.elem(kWk), es = scl.elem(kWq) + ek, ep = scl.elem(kWdo) + scl.elem(kWv);
  const int eu = Kind::bf16 || !live ? 0 : scl.du(A.do_top[h * A.num_q + i], A.dim);
  __syncthreads();
  if (t1 > 0) {
    bad = !landed(0);
    settle(0);
  }
  tc_fence_before();
  if ((bad = __syncthreads_or(bad))) t1 = 0;  // no first tile
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + C::slot);
  const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
  const uint32_t tS = tmem, tP = tmem + KT, tD = tmem + 2 * KT;

  const float delta = live ? -A.neg_d[h * A.num_q + i] : 0.f;
  BwdRow B;
  B.sc.init(A, h);
  B.sc.su *= ldexpf(1.f, -es);
  B.dps = ldexpf(1.f, -ep);
  B.up = ldexpf(1.f, eu);
  B.p.set(live ? pos_of(A.q_pos, A.pos_dim, i) : AttnPos{0.f, 0.f, 0.f});
  constexpr int W = DP / (NT / 128) < 32 ? 32 : DP / (NT / 128);  // columns of a thread's rounds
  DqSums S;
  const bool pos_grad = A.pos_q != nullptr;
  unsigned phase = 0;

  auto mma = [&]() { return threadIdx.x == kMmaThread<NT> && !X.no_mma; };
  if (t1 > 0 && mma()) {
    products_rows<Kind, KT, DP>(tS, sQ, sK);
    products_rows<Kind, KT, DP>(tP, sG, sV);
    tc_commit(bar);
  }
  for (int t = 0; t < t1; ++t) {
    const int pb = t & 1, b = C::STAGES == 1 ? 0 : pb;
    bad |= !tile_wait(X, bar, phase);
    phase ^= 1;
    tc_fence_after();
    if (t + 1 < t1) {
      if (C::STAGES > 1 && threadIdx.x == kTmaThread<NT> && !bad) issue(t + 1, 0);
      fetch(t + 1);
    }
    if (Kind::pair && t > 0 && t % C::ROUND == 0 && A.dq != nullptr)
      add_round<DP, C::SMALL>(tD + lane_off, A.scale * ldexpf(1.f, -eu - ek), t > C::ROUND, 1.f,
                              live, false, A.dim, (float *)A.dq + (i * A.heads + h) * A.dim,
                              W * part, W * part + W);
    __syncwarp();
    float v[32], dp[32];
    tmem_ld32(tS + lane_off + 32 * part, v);
    tmem_ld32(tP + lane_off + 32 * part, dp);
    const unsigned bits = kval[2 * pb + part];  // the same for the warp
#define RA_DQ_(C, P, G, M) \
  dq_elements<Kind, C, P, G, M>(v, dp, B, st.x, st.y, delta, bits, kpos[pb], 32 * part, S)
#define RA_DQ(C, P, G) RA_DQ_(C, P, G, false)
#define RA_DQ_POS(C)                             \
  do {                                           \
    if (pos_grad) RA_DQ(C, true, true);          \
    else if (A.pos_dim > 0) RA_DQ(C, true, false); \
    else RA_DQ(C, false, false);                 \
  } while (0)
    // a last or masked tile: fewer forms.  (A row that is not there spoils its own
    // lane only, which nothing reads.)
    if (bits != kFull) {
      const bool cap = B.sc.capl > 0.f, pos = A.pos_dim > 0;
      if (cap && pos) RA_DQ_(kCapAny, true, true, true);
      else if (cap) RA_DQ_(kCapAny, false, false, true);
      else if (pos) RA_DQ_(kNoCap, true, true, true);
      else RA_DQ_(kNoCap, false, false, true);
    } else if (!(B.sc.capl > 0.f)) RA_DQ_POS(kNoCap);
    else if (all_small(v, B.sc.su)) RA_DQ_POS(kCapSmall);
    else RA_DQ_POS(kCapAny);
#undef RA_DQ_POS
#undef RA_DQ
#undef RA_DQ_
    put_weights<Kind>(tS + lane_off + 32 * part, dp, Kind::pair);
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    if (C::STAGES > 1 && t + 1 < t1) {
      bad = bad || !landed(t + 1);
      settle(t + 1);
    }
    tc_fence_before();
    if ((bad = __syncthreads_or(bad))) break;
    if (mma()) {
      tc_fence_after();
      products_weighted<Kind, KT, DP, C::SMALL>(tD, tS, sK + b * C::KV, false,
                                                t % C::ROUND != 0);
      if (C::STAGES > 1 && t + 1 < t1) {
        products_rows<Kind, KT, DP>(tS, sQ, sK + (b ^ 1) * C::KV);
        products_rows<Kind, KT, DP>(tP, sG, sV + (b ^ 1) * C::KV);
      }
      tc_commit(bar);
    }
    if (C::STAGES == 1 && t + 1 < t1) {  // one buffer: its products first
      bad |= !tile_wait(X, bar, phase);
      phase ^= 1;
      if (threadIdx.x == kTmaThread<NT> && !bad) issue(t + 1, 0);
      bad = bad || !landed(t + 1);
      settle(t + 1);
      if ((bad = __syncthreads_or(bad))) break;
      if (mma()) {
        tc_fence_after();
        products_rows<Kind, KT, DP>(tS, sQ, sK);
        products_rows<Kind, KT, DP>(tP, sG, sV);
        tc_commit(bar);
      }
    }
  }
  if (t1 > 0 && !bad) {
    bad = !tile_wait(X, bar, phase);
    tc_fence_after();
  }
  if ((bad = __syncthreads_or(bad))) {
    if (threadIdx.x == 0) atomicOr(A.status, 1);
    drain<NT>(full, *copied, 0, C::STAGES);
  }
  using T = typename Kind::T;
  if (A.dq != nullptr) {
    const float f = A.scale * ldexpf(1.f, -eu - ek);
    T *out = (T *)A.dq + (i * A.heads + h) * A.dim;
    if (Kind::pair && t1 > C::ROUND)
      add_round<DP, C::SMALL>(tD + lane_off, f, 1.f, 1.f, in, !live, A.dim, (float *)out, W * part,
                              W * part + W);
    else if (part == 0)
      write_row<T, DP, C::SMALL>(tD + lane_off, f, in, !live || t1 == 0, A.dim, out, nullptr);
  }
  // both halves of the columns; what the row's dS add up to is D's error
  float all[9] = {sum_of(S.ds)};
#pragma unroll
  for (int k = 0; k < 4; ++k) all[1 + k] = sum_of(S.g[k]), all[5 + k] = sum_of(S.q[k]);
  float *other = reinterpret_cast<float *>(sm);  // [9][128]: the tiles are done with
  if (part > 0) {
#pragma unroll
    for (int k = 0; k < 9; ++k) other[k * 128 + row] = all[k];
  }
  __syncthreads();
  if (part == 0 && in) {
    if (KT > 32) {
#pragma unroll
      for (int k = 0; k < 9; ++k) all[k] += other[k * 128 + row];
    }
    A.neg_d[h * A.num_q + i] = live ? -(delta + all[0]) : 0.f;
    if (pos_grad) {
#pragma unroll
      for (int k = 0; k < 4; ++k) all[1 + k] = live ? fmaf(-all[0], all[5 + k], all[1 + k]) : 0.f;
      const float s = A.sigma[h], w = 1.f / (s * s);
      A.pos_q[h * A.num_q + i] = make_float4(w * all[1], w * all[2], w * all[3], all[4]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<C::TMEM>(tmem);
  }
}

template <class Kind, int DP>
struct DkvCfg {
  static constexpr int QT = dkv_rows<Kind, DP>;
  static constexpr int HALF = Kind::pair ? 2 : 1;
  // one set of maps for both backward kernels
  static constexpr int BR = QT < dq_rows<Kind, DP> ? QT : dq_rows<Kind, DP>;
  static constexpr int K = HALF * tile_bytes<128, DP>, QG = HALF * tile_bytes<QT, DP>;
  static constexpr bool SMALL = Kind::pair && DP <= 64;  // at 128 TMEM is full
  static constexpr int ROUND = round_tiles<Kind, QT>(SMALL ? 512 : 128);
  static constexpr int TMEM = tmem_round(2 * QT + (SMALL ? 4 : 2) * DP);
  static constexpr int STAGES =
      2 * K + 4 * QG <= (TMEM == 512 ? 200 : 100) * 1024 ? 2 : 1;
  static constexpr int NT = 128 * (QT / 32);
  static constexpr int pos = 2 * K + 2 * STAGES * QG;  // TilePos<QT> [2]
  static constexpr int stt = pos + 2 * QT * 12;        // TileStat<QT> [2]
  static constexpr int bar = stt + 2 * QT * 12, slot = bar + 40;
  static constexpr int smem = slot + 8 + 1024;
  static constexpr int CTAS = attn_ctas(smem, TMEM, NT);
};

template <class Kind, int DP>
__global__ void __launch_bounds__(DkvCfg<Kind, DP>::NT, DkvCfg<Kind, DP>::CTAS)
    attn_tc_dkv_kernel(const AttnArgs A, const __grid_constant__ AttnTcArgs X) {
  using C = DkvCfg<Kind, DP>;
  constexpr int QT = C::QT, NT = C::NT;
  extern __shared__ uint8_t raw_sm[];
  uint8_t *sm = align1024(raw_sm);
  const uint32_t base = smem_u32(sm);
  const uint32_t sK = base, sV = base + C::K, sQ = sV + C::K, sG = sQ + C::STAGES * C::QG,
                 bar = base + C::bar, full = bar + 8;
  TilePos<QT> *qpos = reinterpret_cast<TilePos<QT> *>(sm + C::pos);
  TileStat<QT> *qst = reinterpret_cast<TileStat<QT> *>(sm + C::stt);
  const int warp = threadIdx.x >> 5;
  const int part = warp >> 2, row = threadIdx.x & 127;

  const int64_t item = blockIdx.x;
  const int hk = (int)(item % A.kv_heads), group = A.heads / A.kv_heads;
  const int4 tile = A.ks.tile(item / A.kv_heads, A.qs);
  const int j0 = tile.x, nk = tile.y, i0 = tile.z;
  const int64_t j = j0 + row;
  const bool in = row < nk;
  const bool live = in && (A.k_mask == nullptr || A.k_mask[j] != 0);
  const int nq = (int)masked_extent(A.q_mask ? A.q_mask + i0 : nullptr, tile.w, NT,
                                    reinterpret_cast<unsigned long long *>(sm + C::slot));
  const int per = (nq + QT - 1) / QT;
  int t1 = __syncthreads_or(live) ? per * group : 0;  // query tiles, head by head

  volatile int *copied = reinterpret_cast<int *>(sm + C::bar + 32);  // the last tile asked for
  auto issue = [&](int t, uint32_t more) {
    const int b = C::STAGES == 1 ? 0 : t & 1, h = hk * group + t / per, r0 = i0 + t % per * QT;
    const uint32_t fb = full + 8 * b;
    *copied = t;
    mbar_expect_tx(fb, more + 2 * C::QG);
    load_tile<Kind, QT, DP, C::BR>(sQ + b * C::QG, X.q, h, r0, fb);
    load_tile<Kind, QT, DP, C::BR>(sG + b * C::QG, X.go, h, r0, fb);
  };
  NextRow nx;
  auto fetch = [&](int t) {
    if (threadIdx.x >= QT) return;
    const int h = hk * group + t / per, r = t % per * QT + threadIdx.x;
    const int64_t i = i0 + r, at = h * A.num_q + i;
    nx.on = r < nq && (A.q_mask == nullptr || A.q_mask[i] != 0);
    // a row that is not there is all zero: P = 2^(score <= 0) 0 = 0
    nx.nm = nx.on ? A.neg_m[at] : 0.f;
    nx.rl = nx.on ? A.rl[at] : 0.f;
    nx.nd = nx.on ? A.neg_d[at] : 0.f;
    nx.p = nx.on ? pos_of(A.q_pos, A.pos_dim, i) : AttnPos{0.f, 0.f, 0.f};
  };
  auto settle = [&](int t) {
    const int r = threadIdx.x, pb = t & 1, b = C::STAGES == 1 ? 0 : pb;
    if (r < QT) {
      qst[pb].nm[r] = nx.nm, qst[pb].rl[r] = nx.rl, qst[pb].nd[r] = nx.nd;
      if (A.pos_dim > 0) qpos[pb].put(r, nx.p);
      if (!nx.on) {
        zero_row<Kind, QT, DP>(sm + 2 * C::K + b * C::QG, r);
        zero_row<Kind, QT, DP>(sm + 2 * C::K + (C::STAGES + b) * C::QG, r);
      }
    }
    fence_async_smem();
  };
  auto landed = [&](int t) {
    return C::STAGES == 1 ? mbar_wait(full, t & 1) : mbar_wait(full + 8 * (t & 1), (t >> 1) & 1);
  };
  if (warp == 1) tmem_alloc<C::TMEM>(base + C::slot);
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    mbar_init(full, 1);
    mbar_init(full + 8, 1);
    mbar_init(full + 16, 1);
    *copied = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (t1 > 0) {
      issue(0, 2 * C::K);
      load_tile<Kind, 128, DP, C::BR>(sK, X.k, hk, j0, full);
      load_tile<Kind, 128, DP, C::BR>(sV, X.v, hk, j0, full);
    }
  }
  bool bad = false;
  if (t1 > 0) fetch(0);
  __syncwarp();
  AttnScales<Kind> scl;
  scl.init(A, X, A.ks, item / A.kv_heads, j0, hk);
  __syncthreads();
  if (t1 > 0) {
    bad = !landed(0);
    settle(0);
  }
  tc_fence_before();
  if ((bad = __syncthreads_or(bad))) t1 = 0;  // no first tile
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + C::slot);
  const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
  const uint32_t tS = tmem, tP = tmem + QT, tDk = tmem + 2 * QT, tDv = tDk + (C::SMALL ? 2 : 1) * DP;

  // (read here: before the first wait, as the other kernels do, they spill)
  const int eu = Kind::bf16 ? 0 : scl.du(scl.top(kWdo), A.dim);
  const int eq = scl.elem(kWq), eg = scl.elem(kWdo);
  constexpr float kUp = Kind::bf16 ? 1.f : 8192.f;  // of P
  BwdRow B;
  const float us = ldexpf(1.f, -eq - scl.elem(kWk));
  B.dps = ldexpf(1.f, -eg - scl.elem(kWv));
  B.up = ldexpf(1.f, eu);
  B.p.set(live ? pos_of(A.k_pos, A.pos_dim, j) : AttnPos{0.f, 0.f, 0.f});
  float px = 0.f, py = 0.f, pz = 0.f;  // over all heads, times 1 / sigma^2
  f2_t g[3] = {};                      // of the current head
  const bool pos_grad = A.pos_k != nullptr;
  unsigned phase = 0;
  int cur = -1;

  auto mma = [&]() { return threadIdx.x == kMmaThread<NT> && !X.no_mma; };
  if (t1 > 0 && mma()) {
    products_rows<Kind, QT, DP>(tS, sK, sQ);
    products_rows<Kind, QT, DP>(tP, sV, sG);
    tc_commit(bar);
  }
  auto close_head = [&]() {
    if (cur >= 0 && pos_grad) {
      const float s = A.sigma[cur], w = 1.f / (s * s);
      px = fmaf(w, sum_of(g[0]), px);
      py = fmaf(w, sum_of(g[1]), py);
      pz = fmaf(w, sum_of(g[2]), pz);
    }
    g[0] = g[1] = g[2] = 0;
  };
  const int64_t at = (j * A.kv_heads + hk) * A.dim;
  constexpr int last = QT / 32 - 1;
  auto f_dk = [&]() { return A.scale * ldexpf(1.f, -eu - eq); };
  auto f_dv = [&]() { return ldexpf(1.f, -eg) / kUp; };
  auto add_rounds = [&](float keep, bool on, bool zero) {
    if (A.dk != nullptr && part == 0)
      add_round<DP, C::SMALL>(tDk + lane_off, f_dk(), keep, 1.f, on, zero, A.dim,
                              (float *)A.dk + at);
    if (A.dv != nullptr && part == last)
      add_round<DP, C::SMALL>(tDv + lane_off, f_dv(), keep, 1.f, on, zero, A.dim,
                              (float *)A.dv + at);
  };
  for (int t = 0; t < t1; ++t) {
    const int pb = t & 1, b = C::STAGES == 1 ? 0 : pb;
    const int h = hk * group + t / per;
    if (h != cur) {
      close_head();
      cur = h;
      B.sc.init(A, h);
      B.sc.su *= us;
    }
    bad |= !products_done(X, bar, phase);
    phase ^= 1;
    tc_fence_after();
    if (t + 1 < t1) {
      if (C::STAGES > 1 && threadIdx.x == kTmaThread<NT> && !bad) issue(t + 1, 0);
      fetch(t + 1);
    }
    if (Kind::pair && t > 0 && t % C::ROUND == 0) add_rounds(t > C::ROUND, live, false);
    __syncwarp();
    float v[32], dp[32];
    tmem_ld32(tS + lane_off + 32 * part, v);
    tmem_ld32(tP + lane_off + 32 * part, dp);
#define RA_DKV(C, P, G) \
  dkv_elements<Kind, C, P, G>(v, dp, B, kUp, qst[pb], qpos[pb], 32 * part, g)
#define RA_DKV_POS(C)                             \
  do {                                           \
    if (pos_grad) RA_DKV(C, true, true);          \
    else if (A.pos_dim > 0) RA_DKV(C, true, false); \
    else RA_DKV(C, false, false);                 \
  } while (0)
    if (!(B.sc.capl > 0.f)) RA_DKV_POS(kNoCap);
    else if (all_small(v, B.sc.su)) RA_DKV_POS(kCapSmall);
    else RA_DKV_POS(kCapAny);
#undef RA_DKV_POS
#undef RA_DKV
    put_weights<Kind>(tS + lane_off + 32 * part, v, Kind::pair);
    put_weights<Kind>(tP + lane_off + 32 * part, dp, Kind::pair);
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    if (C::STAGES > 1 && t + 1 < t1) {
      bad = bad || !landed(t + 1);
      settle(t + 1);
    }
    tc_fence_before();
    if ((bad = __syncthreads_or(bad))) break;
    if (mma()) {
      tc_fence_after();
      products_weighted<Kind, QT, DP, C::SMALL>(tDv, tS, sG + b * C::QG, false,
                                                t % C::ROUND != 0);
      products_weighted<Kind, QT, DP, C::SMALL>(tDk, tP, sQ + b * C::QG, false,
                                                t % C::ROUND != 0);
      if (C::STAGES > 1 && t + 1 < t1) {
        products_rows<Kind, QT, DP>(tS, sK, sQ + (b ^ 1) * C::QG);
        products_rows<Kind, QT, DP>(tP, sV, sG + (b ^ 1) * C::QG);
      }
      tc_commit(bar);
    }
    if (C::STAGES == 1 && t + 1 < t1) {
      bad |= !products_done(X, bar, phase);
      phase ^= 1;
      if (threadIdx.x == kTmaThread<NT> && !bad) issue(t + 1, 0);
      bad = bad || !landed(t + 1);
      settle(t + 1);
      if ((bad = __syncthreads_or(bad))) break;
      if (mma()) {
        tc_fence_after();
        products_rows<Kind, QT, DP>(tS, sK, sQ);
        products_rows<Kind, QT, DP>(tP, sV, sG);
        tc_commit(bar);
      }
    }
  }
  close_head();
  if (t1 > 0 && !bad) {
    bad = !products_done(X, bar, phase);
    tc_fence_after();
  }
  if ((bad = __syncthreads_or(bad))) {
    if (threadIdx.x == 0) atomicOr(A.status, 1);
    drain<NT>(full, *copied, 0, C::STAGES);
  }
  using T = typename Kind::T;
  const bool zero = !live || t1 == 0;
  if (Kind::pair && t1 > C::ROUND) {
    add_rounds(1.f, in, zero);
  } else {
    if (A.dk != nullptr && part == 0)
      write_row<T, DP, C::SMALL>(tDk + lane_off, f_dk(), in, zero, A.dim, (T *)A.dk + at, nullptr);
    if (A.dv != nullptr && part == last)
      write_row<T, DP, C::SMALL>(tDv + lane_off, f_dv(), in, zero, A.dim, (T *)A.dv + at, nullptr);
  }
  if (pos_grad) {
    float4 *sum = reinterpret_cast<float4 *>(sm);  // [parts - 1][128]
    if (part > 0) sum[(part - 1) * 128 + row] = make_float4(px, py, pz, 0.f);
    __syncthreads();
    if (part == 0 && in) {
#pragma unroll
      for (int k = 0; k < QT / 32 - 1; ++k) {
        const float4 o = sum[k * 128 + row];
        px += o.x, py += o.y, pz += o.z;
      }
      if (!live) px = py = pz = 0.f;
      A.pos_k[hk * A.num_k + j] = make_float4(px, py, pz, 0.f);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<C::TMEM>(tmem);
  }
}

}  // namespace ra
