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
// What bounds them is not the tensor core (S and P V take 2 x 64 cycles a
// 128 x 64 tile at DP = 64) but the elementwise part: about 12 fp32 operations
// and an EX2 a score with positions, 800 issue slots of each SM quarter a tile.
// So the flow within a CTA is simple -- all threads wait for the products, work
// on the scores, one thread issues the next products -- and two to four CTAs on
// an SM hide each other's waits.
//
// Tiles lie in shared memory in the canonical no-swizzle layout, 16-byte chunk
// (d / 8, row) at (d / 8 * rows + row) * 16: read K-major (S, dP) and MN-major
// (P V, dU K) from one copy.  cp.async copies 16 bytes a thread and fills rows
// behind the graph's end and masked rows with zeros, so whatever those hold
// reaches no product.
//
// fp32 inputs are fp16 pairs (hi + lo, one power of two per tensor), three
// products for one.  P of 16-bit inputs is a pair too where the output is kept
// unrounded for a backward (D_i = do.o must be as exact as dP); dU is one
// 16-bit number for 16-bit inputs (half a step, independent between elements).
// In fp16 P is held 2^7 up, and dU in units of the power of two that keeps
// 2 max |do| max |v| >= |dU| / slope below 2^14.
#pragma once

#include "ra_attn.cuh"
#include "ra_tcprim.cuh"

namespace ra {

// words of the bounds (bits of non-negative floats): largest finite element
// and row norm of each tensor
enum AttnWord { kWq = 0, kWk = 2, kWv = 4, kWdo = 6, kWords = 8 };

struct AttnOp {  // 16-bit operand, or its halves
  const uint16_t *hi, *lo;
  int64_t row, head;  // element strides
};
struct AttnTcArgs {
  AttnOp q, k, v, go;
  const unsigned *words;  // null where nothing is scaled
  int splits;             // forward: key ranges of a row tile
  float *part_o;          // [splits][num_q][heads][dim], unnormalised
  float2 *part_s;         // [splits][heads][num_q] (m, l)
  int pair_p;             // forward of 16-bit inputs: P as a pair
};

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
template <class Kind>
__device__ __forceinline__ int elem_exp(const AttnTcArgs &X, int w) {
  return Kind::pair ? attn_exp(__uint_as_float(X.words[w])) : 0;
}
// of dU: 2 |do| |v| bounds |dP - D|
template <class Kind>
__device__ __forceinline__ int du_exp(const AttnTcArgs &X) {
  if (Kind::bf16) return 0;
  return attn_exp(2.f * __uint_as_float(X.words[kWdo + 1]) * __uint_as_float(X.words[kWv + 1]));
}

// no-swizzle descriptor of a tile of `rows` rows
__device__ __forceinline__ uint64_t tile_desc_k(uint32_t s, int rows) {
  return tc_desc(s, (uint32_t)rows * 16, 128);
}
__device__ __forceinline__ uint64_t tile_desc_mn(uint32_t s, int rows) {
  return tc_desc(s, 128, (uint32_t)rows * 16);
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

template <int ROWS, int DP, int NT>
__device__ __forceinline__ void load_half(uint32_t dst, const uint16_t *src, int64_t row0, int n,
                                          int64_t stride, int dim8, const uint8_t *mask) {
  constexpr int kChunks = ROWS * DP / 8;
#pragma unroll 4
  for (int c = threadIdx.x; c < kChunks; c += NT) {
    // 16 rows x 2 chunks a warp: whole 32-byte sectors, no bank conflicts
    const int rest = c >> 5, row = (rest / (DP / 16)) * 16 + (c & 15),
              d8 = (rest % (DP / 16)) * 2 + ((c >> 4) & 1);
    const bool on = row < n && d8 < dim8 && (mask == nullptr || mask[row0 + row] != 0);
    const uint16_t *from = on ? src + (row0 + row) * stride + d8 * 8 : src;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (d8 * ROWS + row) * 16),
                 "l"(from), "r"(on ? 16 : 0)
                 : "memory");
  }
}
template <class Kind, int ROWS, int DP, int NT>
__device__ __forceinline__ void load_tile(uint32_t dst, const AttnOp &op, int head, int64_t row0,
                                          int n, int dim8, const uint8_t *mask) {
  load_half<ROWS, DP, NT>(dst, op.hi + head * op.head, row0, n, op.row, dim8, mask);
  if (Kind::pair)
    load_half<ROWS, DP, NT>(dst + tile_bytes<ROWS, DP>, op.lo + head * op.head, row0, n, op.row,
                            dim8, mask);
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
    const uint64_t da = tile_desc_k(ap, 128), db = tile_desc_k(bp, N);
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
      mma_ss(d, da + (uint64_t)(k * 2 * 128 * 16 >> 4), db + (uint64_t)(k * 2 * N * 16 >> 4), idesc,
             p > 0 || k > 0);
  }
}
// D[128, DP] (+)= W[128, KT] X[KT, DP]: W in TMEM (per 32 columns of the
// scores 16 columns of hi, 16 of lo), X a streamed tile read MN-major
template <class Kind, int KT, int DP>
__device__ __forceinline__ void products_weighted(uint32_t d, uint32_t w, uint32_t x, bool w_pair,
                                                  uint32_t acc) {
  constexpr uint32_t idesc = attn_idesc(DP, Kind::bf16, true);
  const int first = Kind::pair || w_pair ? 0 : 2;
#pragma unroll
  for (int p = 0; p < 3; ++p) {  // lo hi, hi lo (pairs of x only), hi hi
    if (p < first || (p == 1 && !Kind::pair)) continue;
    const uint64_t dx = tile_desc_mn(x + (Kind::pair && p == 1 ? tile_bytes<KT, DP> : 0), KT);
#pragma unroll
    for (int k = 0; k < KT / 16; ++k) {
      mma_ts(d, w + (k >> 1) * 32 + (k & 1) * 8 + (p == 0 ? 16 : 0), dx + (uint64_t)(k * 256 >> 4),
             idesc, acc);
      acc = 1;
    }
  }
}

template <class Kind>
__device__ __forceinline__ uint32_t pack_kind(float a, float b) {
  if (Kind::bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <class Kind>
__device__ __forceinline__ float2 unpack_kind(uint32_t u) {
  if (Kind::bf16) {
    const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162 *>(&u);
    return __bfloat1622float2(v);
  }
  return __half22float2(*reinterpret_cast<const __half2 *>(&u));
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

// tanh to 2^-22 of 1 (16-bit inputs) or to a few steps (fp32)
template <class Kind>
__device__ __forceinline__ float tanh_kind(float u) {
  if (Kind::pair) return tanhf(u);
  const float e = ex2(u * (2.f * kAttnLog2e));
  const float big = 1.f - __fdividef(2.f, 1.f + e);
  const float u2 = u * u;
  const float small = u * fmaf(u2, fmaf(u2, fmaf(u2, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  return fabsf(u) < 0.1f ? small : big;
}

// raw products of 32 scores -> base-2 scores before the distances; th: tanh
// where capped
template <class Kind>
__device__ __forceinline__ void scores32(float (&v)[32], float su, float capl) {
  if (capl > 0.f) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = capl * tanh_kind<Kind>(v[j] * su);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= su;
  }
}

__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

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
template <class T, int DP>
__device__ __forceinline__ void write_row(uint32_t taddr, float f, bool on, bool zero, int dim,
                                          T *out, float *out32) {
#pragma unroll 1
  for (int c = 0; c < DP; c += 32) {
    float v[32];
    tmem_ld32(taddr + c, v);
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
          alignas(16) T t[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) put(t + k, v[j + k]);
          *reinterpret_cast<uint4 *>(out + c + j) = *reinterpret_cast<const uint4 *>(t);
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

// ---- bounds and halves ---------------------------------------------------------

struct AttnPrep {
  const void *x[4];
  int64_t rows[4], row[4], head[4];
  int heads[4];
  const uint8_t *mask[4];
  int word[4];
  uint16_t *hi[4], *lo[4];  // [rows][heads][dim]
  int dim, count;
};

// largest finite element and row norm of each tensor; one warp a row and head
template <class T>
__global__ void __launch_bounds__(256) attn_bounds_kernel(const AttnPrep p, unsigned *words) {
  const int t = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t n = p.rows[t] * p.heads[t];
  float top = 0.f, norm = 0.f;
  for (int64_t r = blockIdx.x * 8LL + (threadIdx.x >> 5); r < n; r += gridDim.x * 8LL) {
    const int64_t i = r / p.heads[t];
    if (p.mask[t] != nullptr && p.mask[t][i] == 0) continue;
    const T *x = (const T *)p.x[t] + i * p.row[t] + (r % p.heads[t]) * p.head[t];
    float m = 0.f, s = 0.f;
    for (int d = lane; d < p.dim; d += 32) {
      const float v = to_f(x[d]);
      if (fabsf(v) < INFINITY) m = fmaxf(m, fabsf(v));
      s = fmaf(v, v, s);
    }
    s = warp_sum(s);
    top = fmaxf(top, m);
    if (s < INFINITY) norm = fmaxf(norm, s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
  if (lane == 0) {  // maxima of bits: any order
    if (top > 0.f) atomicMax(words + p.word[t], __float_as_uint(top));
    norm = sqrtf(norm) * 1.001f;
    if (norm > 0.f) atomicMax(words + p.word[t] + 1, __float_as_uint(norm));
  }
}

__global__ void __launch_bounds__(256) attn_halves_kernel(const AttnPrep p, const unsigned *words) {
  const int t = blockIdx.y;
  const float sc = ldexpf(1.f, attn_exp(__uint_as_float(words[p.word[t]])));
  const int64_t n = p.rows[t] * p.heads[t] * p.dim;
  const int64_t per = (int64_t)p.heads[t] * p.dim;
  for (int64_t e = blockIdx.x * 256LL + threadIdx.x; e < n; e += gridDim.x * 256LL) {
    const int64_t i = e / per;
    const int r = (int)(e - i * per), h = r / p.dim, d = r - h * p.dim;
    const float v = ((const float *)p.x[t])[i * p.row[t] + h * p.head[t] + d] * sc;
    const __half hi = __float2half_rn(v);
    p.hi[t][e] = __half_as_ushort(hi);
    p.lo[t][e] = __half_as_ushort(__float2half_rn(v - __half2float(hi)));
  }
}

// ---- forward --------------------------------------------------------------------

template <class Kind, int DP>
struct FwdCfg {
  static constexpr int KT = Kind::pair && DP == 128 ? 32 : 64;
  static constexpr int HALF = Kind::pair ? 2 : 1;
  static constexpr int Q = HALF * tile_bytes<128, DP>, KV = HALF * tile_bytes<KT, DP>;
  static constexpr int TMEM = tmem_round(KT + DP);
  static constexpr int pos = Q + 4 * KV;                 // float4 [2][KT]
  static constexpr int val = pos + 2 * KT * 16;          // unsigned [2][2]
  static constexpr int bar = val + 16, slot = bar + 8;
  static constexpr int smem = slot + 8;
};

template <class Kind, int DP>
__global__ void __launch_bounds__(128) attn_tc_fwd_kernel(const AttnArgs A, const AttnTcArgs X) {
  using C = FwdCfg<Kind, DP>;
  constexpr int KT = C::KT;
  extern __shared__ __align__(1024) uint8_t sm[];
  const uint32_t base = smem_u32(sm);
  const uint32_t sQ = base, sK = base + C::Q, sV = sK + 2 * C::KV, bar = base + C::bar;
  float4 *kpos = reinterpret_cast<float4 *>(sm + C::pos);
  unsigned *kval = reinterpret_cast<unsigned *>(sm + C::val);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int64_t item = blockIdx.x;
  const int split = (int)(item % X.splits);
  const int h = (int)(item / X.splits % A.heads), hk = h / (A.heads / A.kv_heads);
  const int2 tile = A.qs.tile(item / X.splits / A.heads);
  const int64_t i0 = A.qs.begin(tile.x) + 128LL * tile.y, j0 = A.ks.begin(tile.x);
  const int nq = (int)min((int64_t)128, A.qs.end(tile.x) - i0);
  const int64_t nk = A.ks.end(tile.x) - j0;
  const int64_t all = (nk + KT - 1) / KT;
  const int64_t t0 = all * split / X.splits, t1 = all * (split + 1) / X.splits;
  const int dim8 = A.dim >> 3;

  if (warp == 0) tmem_alloc<C::TMEM>(base + C::slot);
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  auto load_keys = [&](int64_t t) {
    const int b = (int)(t & 1);
    const int64_t r0 = j0 + t * KT;
    const int n = (int)min((int64_t)KT, nk - t * KT);
    load_tile<Kind, KT, DP, 128>(sK + b * C::KV, X.k, hk, r0, n, dim8, A.k_mask);
    load_tile<Kind, KT, DP, 128>(sV + b * C::KV, X.v, hk, r0, n, dim8, A.k_mask);
    if (warp < KT / 32) {
      const int r = threadIdx.x;
      const bool on = r < n && (A.k_mask == nullptr || A.k_mask[r0 + r] != 0);
      const unsigned bits = __ballot_sync(kFull, on);
      if (lane == 0) kval[2 * b + warp] = bits;
      AttnPos p{0.f, 0.f, 0.f};
      if (on) p = pos_of(A.k_pos, A.pos_dim, r0 + r);
      kpos[b * KT + r] = make_float4(p.x, p.y, p.z, 0.f);
    }
  };
  load_tile<Kind, 128, DP, 128>(sQ, X.q, h, i0, nq, dim8, A.q_mask);
  if (t0 < t1) load_keys(t0);
  cp_wait_all();
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + C::slot);
  const uint32_t tS = tmem, tO = tmem + KT, lane_off = (uint32_t)(32 * warp) << 16;

  const int64_t i = i0 + threadIdx.x;
  const bool row_on = threadIdx.x < nq && (A.q_mask == nullptr || A.q_mask[i] != 0);
  AttnScore sc;
  sc.init(A, h);
  sc.su *= ldexpf(1.f, -elem_exp<Kind>(X, kWq) - elem_exp<Kind>(X, kWk));
  AttnPos pi{0.f, 0.f, 0.f};
  if (row_on) pi = pos_of(A.q_pos, A.pos_dim, i);
  constexpr float kUp = Kind::bf16 ? 0.f : 7.f;  // P is held 2^kUp up
  const bool p_pair = Kind::pair || X.pair_p;
  float m = -INFINITY, l = 0.f;  // m: the reference the sums are relative to
  bool bad = false;
  unsigned phase = 0;

  if (t0 < t1 && threadIdx.x == 0) {
    products_rows<Kind, KT, DP>(tS, sQ, sK + (int)(t0 & 1) * C::KV);
    tc_commit(bar);
  }
  for (int64_t t = t0; t < t1; ++t) {
    const int b = (int)(t & 1);
    bad = !mbar_wait(bar, phase);
    phase ^= 1;
    tc_fence_after();
    if (t + 1 < t1) load_keys(t + 1);  // its buffers' products are done
    float v[KT / 32][32];
    const unsigned vb[2] = {kval[2 * b], KT > 32 ? kval[2 * b + 1] : 0u};
#pragma unroll
    for (int c = 0; c < KT / 32; ++c) {
      tmem_ld32(tS + lane_off + 32 * c, v[c]);
      scores32<Kind>(v[c], sc.su, sc.capl);
      if (A.pos_dim > 0) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float4 p = kpos[b * KT + 32 * c + j];
          const float dx = pi.x - p.x, dy = pi.y - p.y, dz = pi.z - p.z;
          v[c][j] = fmaf(-sc.w, fmaf(dz, dz, fmaf(dy, dy, dx * dx)), v[c][j]);
        }
      }
      if (vb[c] != kFull) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!((vb[c] >> j) & 1)) v[c][j] = -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < KT / 32; ++c)
#pragma unroll
      for (int j = 0; j < 32; ++j) mx = fmaxf(mx, v[c][j]);
    // the reference follows the maximum only where it grew by more than 2^8:
    // sums and O stay relative to one reference, whichever it is
    const bool grow = mx > m + 8.f;  // also from -inf
    const float mn = grow ? mx : m;
    if (__any_sync(kFull, grow)) {
      const float f = m > -INFINITY ? ex2(m - mn) : 0.f;
      l *= f;
      if (t > t0) {
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
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
    const float ref = (m > -INFINITY ? m : 0.f) - kUp;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int c = 0; c < KT / 32; ++c) {
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        v[c][j] = ex2(v[c][j] - ref);
        v[c][j + 1] = ex2(v[c][j + 1] - ref);
        s0 += v[c][j];
        s1 += v[c][j + 1];
      }
      put_weights<Kind>(tS + lane_off + 32 * c, v[c], p_pair);
    }
    l += s0 + s1;
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    cp_wait_all();
    fence_async_smem();
    tc_fence_before();
    if ((bad = __syncthreads_or(bad))) break;
    if (threadIdx.x == 0) {
      tc_fence_after();
      products_weighted<Kind, KT, DP>(tO, tS, sV + b * C::KV, p_pair, t > t0);
      if (t + 1 < t1) products_rows<Kind, KT, DP>(tS, sQ, sK + (b ^ 1) * C::KV);
      tc_commit(bar);
    }
  }
  if (t0 < t1 && !bad) {
    bad = !mbar_wait(bar, phase);
    tc_fence_after();
  }
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0) atomicOr(A.status, 1);

  const bool any = l > 0.f || l != l;
  const bool empty = !row_on || !any || t0 >= t1;
  using T = typename Kind::T;
  const float unscale = ldexpf(1.f, -elem_exp<Kind>(X, kWv));
  const bool in = threadIdx.x < nq;
  if (X.splits > 1) {
    float *po = X.part_o + ((split * A.num_q + i) * A.heads + h) * A.dim;
    write_row<float, DP>(tO + lane_off, unscale, in, empty, A.dim, po, nullptr);
    if (in)
      X.part_s[((int64_t)split * A.heads + h) * A.num_q + i] =
          make_float2(empty ? -INFINITY : (m > -INFINITY ? m : 0.f) - kUp, empty ? 0.f : l);
  } else {
    const float r = empty ? 0.f : 1.f / l;
    const int64_t at = (i * A.heads + h) * A.dim;
    write_row<T, DP>(tO + lane_off, unscale * r, in, empty, A.dim, (T *)A.out + at,
                     A.out32 ? A.out32 + at : nullptr);
    if (in && A.stats)
      A.stats[h * A.num_q + i] =
          make_float2(empty ? INFINITY : (m > -INFINITY ? m : 0.f) - kUp, r);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_free<C::TMEM>(tmem);
  }
}

// Joins the key ranges of a row: one warp a row and head, ranges in order.
template <class T>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs A, int splits,
                                                        const float *part_o, const float2 *part_s) {
  const int lane = threadIdx.x & 31;
  const int64_t n = A.num_q * A.heads;
  for (int64_t r = blockIdx.x * 8LL + (threadIdx.x >> 5); r < n; r += gridDim.x * 8LL) {
    const int64_t i = r / A.heads;
    const int h = (int)(r % A.heads);
    float m = -INFINITY;
    for (int s = lane; s < splits; s += 32) m = fmaxf(m, part_s[((int64_t)s * A.heads + h) * A.num_q + i].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    float l = 0.f, acc[kAttnMaxDim / 32] = {};
    for (int s = 0; s < splits; ++s) {
      const float2 st = part_s[((int64_t)s * A.heads + h) * A.num_q + i];
      if (!(st.x > -INFINITY)) continue;
      const float f = ex2(st.x - m);
      l = fmaf(st.y, f, l);
      const float *po = part_o + (s * n + r) * A.dim;
#pragma unroll
      for (int c = 0; c < kAttnMaxDim / 32; ++c)
        if (lane + 32 * c < A.dim) acc[c] = fmaf(f, po[lane + 32 * c], acc[c]);
    }
    const bool any = l > 0.f || l != l;
    const float rl = any ? 1.f / l : 0.f;
#pragma unroll
    for (int c = 0; c < kAttnMaxDim / 32; ++c)
      if (lane + 32 * c < A.dim) {
        const float o = any ? acc[c] * rl : 0.f;
        put((T *)A.out + r * A.dim + lane + 32 * c, o);
        if (A.out32) A.out32[r * A.dim + lane + 32 * c] = o;
      }
    if (lane == 0 && A.stats) A.stats[h * A.num_q + i] = make_float2(any ? m : INFINITY, rl);
  }
}

// ---- backward -------------------------------------------------------------------

// The elementwise part of 32 scores of a row, all in one pass so that only the
// scores and dP are held.  `v` raw products, `dp` raw dP; out: dU in dp (and P
// in v where the rows are keys).  g: the sums of dS (p_i - p_j) [, dS r^2].
// CAP, POS, PG: the cap, positions and their gradients are there.
struct BwdRow {
  float su, capl, w, dps, up;
  AttnPos p;
};
template <class Kind, bool CAP, bool POS, bool PG>
__device__ __forceinline__ void dq_elements(float (&v)[32], float (&dp)[32], const BwdRow &R,
                                            float m, float rl, float delta, unsigned bits,
                                            const float4 *kpos, float (&g)[4]) {
  const bool every = bits == kFull;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    float t = v[j] * R.su, th = 0.f, r2 = 0.f, dx = 0.f, dy = 0.f, dz = 0.f;
    if (CAP) {
      th = tanh_kind<Kind>(t);
      t = th * R.capl;
    }
    if (POS) {
      const float4 p = kpos[j];
      dx = R.p.x - p.x, dy = R.p.y - p.y, dz = R.p.z - p.z;
      r2 = fmaf(dz, dz, fmaf(dy, dy, dx * dx));
      t = fmaf(-R.w, r2, t);
    }
    float ds = ex2(t - m) * rl * fmaf(dp[j], R.dps, -delta);
    if (!every) ds = (bits >> j) & 1 ? ds : 0.f;
    if (PG) {
      g[0] = fmaf(ds, dx, g[0]);
      g[1] = fmaf(ds, dy, g[1]);
      g[2] = fmaf(ds, dz, g[2]);
      g[3] = fmaf(ds, r2, g[3]);
    }
    if (CAP) ds *= fmaf(-th, th, 1.f);
    dp[j] = Kind::bf16 ? ds : ds * R.up;
  }
}
template <class Kind, bool CAP, bool POS, bool PG>
__device__ __forceinline__ void dkv_elements(float (&v)[32], float (&dp)[32], const BwdRow &R,
                                             float p_up, const float2 *qst, const float4 *qpos,
                                             float (&g)[4]) {
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    float t = v[c] * R.su, th = 0.f, dx = 0.f, dy = 0.f, dz = 0.f;
    const float4 p = qpos[c];
    const float2 st = qst[c];
    if (CAP) {
      th = tanh_kind<Kind>(t);
      t = th * R.capl;
    }
    if (POS) {
      dx = p.x - R.p.x, dy = p.y - R.p.y, dz = p.z - R.p.z;
      t = fmaf(-R.w, fmaf(dz, dz, fmaf(dy, dy, dx * dx)), t);
    }
    const float pr = ex2(t - st.x) * st.y;
    float ds = pr * fmaf(dp[c], R.dps, -p.w);
    if (PG) {
      g[0] = fmaf(ds, dx, g[0]);
      g[1] = fmaf(ds, dy, g[1]);
      g[2] = fmaf(ds, dz, g[2]);
    }
    if (CAP) ds *= fmaf(-th, th, 1.f);
    v[c] = Kind::bf16 ? pr : pr * p_up;
    dp[c] = Kind::bf16 ? ds : ds * R.up;
  }
}

template <class Kind, int DP>
struct DqCfg {
  static constexpr int KT = Kind::pair && DP == 128 ? 32 : 64;
  static constexpr int HALF = Kind::pair ? 2 : 1;
  static constexpr int Q = HALF * tile_bytes<128, DP>, KV = HALF * tile_bytes<KT, DP>;
  static constexpr int STAGES = Kind::pair && DP == 128 ? 1 : 2;
  static constexpr int TMEM = tmem_round(2 * KT + DP);
  static constexpr int NT = 128 * (KT / 32);
  static constexpr int pos = 2 * Q + 2 * STAGES * KV;
  static constexpr int val = pos + 2 * KT * 16;
  static constexpr int bar = val + 16, slot = bar + 8;
  static constexpr int smem = slot + 8;
};

template <class Kind, int DP>
__global__ void __launch_bounds__(DqCfg<Kind, DP>::NT) attn_tc_dq_kernel(const AttnArgs A,
                                                                         const AttnTcArgs X) {
  using C = DqCfg<Kind, DP>;
  constexpr int KT = C::KT, NT = C::NT;
  extern __shared__ __align__(1024) uint8_t sm[];
  const uint32_t base = smem_u32(sm);
  const uint32_t sQ = base, sG = base + C::Q, sK = sG + C::Q, sV = sK + C::STAGES * C::KV,
                 bar = base + C::bar;
  float4 *kpos = reinterpret_cast<float4 *>(sm + C::pos);
  unsigned *kval = reinterpret_cast<unsigned *>(sm + C::val);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp >> 2, row = threadIdx.x & 127;  // columns 32 part.. of the tile

  const int64_t item = blockIdx.x;
  const int h = (int)(item % A.heads), hk = h / (A.heads / A.kv_heads);
  const int2 tile = A.qs.tile(item / A.heads);
  const int64_t i0 = A.qs.begin(tile.x) + 128LL * tile.y, j0 = A.ks.begin(tile.x);
  const int nq = (int)min((int64_t)128, A.qs.end(tile.x) - i0);
  const int64_t nk = A.ks.end(tile.x) - j0;
  const int64_t t1 = (nk + KT - 1) / KT;
  const int dim8 = A.dim >> 3;

  if (warp == 0) tmem_alloc<C::TMEM>(base + C::slot);
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  auto load_keys = [&](int64_t t) {
    const int b = C::STAGES == 1 ? 0 : (int)(t & 1), pb = (int)(t & 1);
    const int64_t r0 = j0 + t * KT;
    const int n = (int)min((int64_t)KT, nk - t * KT);
    load_tile<Kind, KT, DP, NT>(sK + b * C::KV, X.k, hk, r0, n, dim8, A.k_mask);
    load_tile<Kind, KT, DP, NT>(sV + b * C::KV, X.v, hk, r0, n, dim8, A.k_mask);
    if (warp < KT / 32) {
      const int r = threadIdx.x;
      const bool on = r < n && (A.k_mask == nullptr || A.k_mask[r0 + r] != 0);
      const unsigned bits = __ballot_sync(kFull, on);
      if (lane == 0) kval[2 * pb + warp] = bits;
      AttnPos p{0.f, 0.f, 0.f};
      if (on) p = pos_of(A.k_pos, A.pos_dim, r0 + r);
      kpos[pb * KT + r] = make_float4(p.x, p.y, p.z, 0.f);
    }
  };
  load_tile<Kind, 128, DP, NT>(sQ, X.q, h, i0, nq, dim8, A.q_mask);
  load_tile<Kind, 128, DP, NT>(sG, X.go, h, i0, nq, dim8, A.q_mask);
  if (t1 > 0) load_keys(0);
  cp_wait_all();
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + C::slot);
  const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
  const uint32_t tS = tmem, tP = tmem + KT, tD = tmem + 2 * KT;

  const int64_t i = i0 + row;
  const bool in = row < nq;
  float2 st = make_float2(INFINITY, 0.f);
  if (in) st = A.stats[h * A.num_q + i];
  const bool live = st.y != 0.f;  // has keys, and is not masked
  const float delta = live ? A.delta[h * A.num_q + i] : 0.f;
  AttnScore sc;
  sc.init(A, h);
  sc.su *= ldexpf(1.f, -elem_exp<Kind>(X, kWq) - elem_exp<Kind>(X, kWk));
  const int eu = du_exp<Kind>(X);
  BwdRow R{sc.su, sc.capl, sc.w,
           ldexpf(1.f, -elem_exp<Kind>(X, kWdo) - elem_exp<Kind>(X, kWv)), ldexpf(1.f, eu),
           {0.f, 0.f, 0.f}};
  if (live) R.p = pos_of(A.q_pos, A.pos_dim, i);
  float g[4] = {};
  const bool pos_grad = A.pos_q != nullptr;
  bool bad = false;
  unsigned phase = 0;

  if (t1 > 0 && threadIdx.x == 0) {
    products_rows<Kind, KT, DP>(tS, sQ, sK);
    products_rows<Kind, KT, DP>(tP, sG, sV);
    tc_commit(bar);
  }
  for (int64_t t = 0; t < t1; ++t) {
    const int pb = (int)(t & 1), b = C::STAGES == 1 ? 0 : pb;
    bad = !mbar_wait(bar, phase);
    phase ^= 1;
    tc_fence_after();
    if (C::STAGES > 1 && t + 1 < t1) load_keys(t + 1);
    float v[32], dp[32];
    tmem_ld32(tS + lane_off + 32 * part, v);
    tmem_ld32(tP + lane_off + 32 * part, dp);
    const unsigned bits = live ? kval[2 * pb + part] : 0u;
    const float4 *kp = kpos + pb * KT + 32 * part;
#define RA_DQ(C, P, G) \
  dq_elements<Kind, C, P, G>(v, dp, R, st.x, st.y, delta, bits, kp, g)
    if (R.capl > 0.f) {
      if (pos_grad) RA_DQ(true, true, true);
      else if (A.pos_dim > 0) RA_DQ(true, true, false);
      else RA_DQ(true, false, false);
    } else {
      if (pos_grad) RA_DQ(false, true, true);
      else if (A.pos_dim > 0) RA_DQ(false, true, false);
      else RA_DQ(false, false, false);
    }
#undef RA_DQ
    put_weights<Kind>(tS + lane_off + 32 * part, dp, Kind::pair);
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    cp_wait_all();
    fence_async_smem();
    tc_fence_before();
    if ((bad = __syncthreads_or(bad))) break;
    if (threadIdx.x == 0) {
      tc_fence_after();
      products_weighted<Kind, KT, DP>(tD, tS, sK + b * C::KV, false, t > 0);
      if (C::STAGES > 1 && t + 1 < t1) {
        products_rows<Kind, KT, DP>(tS, sQ, sK + (b ^ 1) * C::KV);
        products_rows<Kind, KT, DP>(tP, sG, sV + (b ^ 1) * C::KV);
      }
      tc_commit(bar);
    }
    if (C::STAGES == 1 && t + 1 < t1) {  // one buffer: its products first
      bad = !mbar_wait(bar, phase);
      phase ^= 1;
      load_keys(t + 1);
      cp_wait_all();
      fence_async_smem();
      if ((bad = __syncthreads_or(bad))) break;
      if (threadIdx.x == 0) {
        tc_fence_after();
        products_rows<Kind, KT, DP>(tS, sQ, sK);
        products_rows<Kind, KT, DP>(tP, sG, sV);
        tc_commit(bar);
      }
    }
  }
  if (t1 > 0 && !bad) {
    bad = !mbar_wait(bar, phase);
    tc_fence_after();
  }
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0) atomicOr(A.status, 1);
  using T = typename Kind::T;
  if (A.dq != nullptr && part == 0)
    write_row<T, DP>(tD + lane_off, A.scale * ldexpf(1.f, -eu - elem_exp<Kind>(X, kWk)), in,
                     !live || t1 == 0, A.dim, (T *)A.dq + (i * A.heads + h) * A.dim, nullptr);
  if (pos_grad) {
    float4 *sum = reinterpret_cast<float4 *>(sm);  // the tiles are done with
    if (part > 0) sum[row] = make_float4(g[0], g[1], g[2], g[3]);
    __syncthreads();
    if (part == 0 && in) {
      if (KT > 32) {
        const float4 o = sum[row];
        g[0] += o.x, g[1] += o.y, g[2] += o.z, g[3] += o.w;
      }
      const float s = A.sigma[h], w = 1.f / (s * s);
      A.pos_q[h * A.num_q + i] = make_float4(-w * g[0], -w * g[1], -w * g[2], g[3]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_free<C::TMEM>(tmem);
  }
}

template <class Kind, int DP>
struct DkvCfg {
  static constexpr int QT = Kind::pair && DP == 128 ? 32 : 64;
  static constexpr int HALF = Kind::pair ? 2 : 1;
  static constexpr int K = HALF * tile_bytes<128, DP>, QG = HALF * tile_bytes<QT, DP>;
  static constexpr int STAGES = Kind::pair && DP == 128 ? 1 : 2;
  static constexpr int TMEM = tmem_round(2 * QT + 2 * DP);
  static constexpr int NT = 128 * (QT / 32);
  static constexpr int pos = 2 * K + 2 * STAGES * QG;  // float4 [2][QT]: x y z delta
  static constexpr int stt = pos + 2 * QT * 16;        // float2 [2][QT]: m, 1 / l
  static constexpr int bar = stt + 2 * QT * 8, slot = bar + 8;
  static constexpr int smem = slot + 8;
};

template <class Kind, int DP>
__global__ void __launch_bounds__(DkvCfg<Kind, DP>::NT) attn_tc_dkv_kernel(const AttnArgs A,
                                                                           const AttnTcArgs X) {
  using C = DkvCfg<Kind, DP>;
  constexpr int QT = C::QT, NT = C::NT;
  extern __shared__ __align__(1024) uint8_t sm[];
  const uint32_t base = smem_u32(sm);
  const uint32_t sK = base, sV = base + C::K, sQ = sV + C::K, sG = sQ + C::STAGES * C::QG,
                 bar = base + C::bar;
  float4 *qpos = reinterpret_cast<float4 *>(sm + C::pos);
  float2 *qst = reinterpret_cast<float2 *>(sm + C::stt);
  const int warp = threadIdx.x >> 5;
  const int part = warp >> 2, row = threadIdx.x & 127;

  const int64_t item = blockIdx.x;
  const int hk = (int)(item % A.kv_heads), group = A.heads / A.kv_heads;
  const int2 tile = A.ks.tile(item / A.kv_heads);
  const int64_t j0 = A.ks.begin(tile.x) + 128LL * tile.y, i0 = A.qs.begin(tile.x);
  const int nk = (int)min((int64_t)128, A.ks.end(tile.x) - j0);
  const int64_t nq = A.qs.end(tile.x) - i0;
  const int64_t per = (nq + QT - 1) / QT, t1 = per * group;  // query tiles, head by head
  const int dim8 = A.dim >> 3;

  if (warp == 0) tmem_alloc<C::TMEM>(base + C::slot);
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  auto load_queries = [&](int64_t t) {
    const int b = C::STAGES == 1 ? 0 : (int)(t & 1), pb = (int)(t & 1);
    const int h = hk * group + (int)(t / per);
    const int64_t q0 = (t % per) * QT, r0 = i0 + q0;
    const int n = (int)min((int64_t)QT, nq - q0);
    load_tile<Kind, QT, DP, NT>(sQ + b * C::QG, X.q, h, r0, n, dim8, A.q_mask);
    load_tile<Kind, QT, DP, NT>(sG + b * C::QG, X.go, h, r0, n, dim8, A.q_mask);
    if (threadIdx.x < QT) {
      const int r = threadIdx.x;
      float2 st = make_float2(INFINITY, 0.f);  // P = 0
      if (r < n) st = A.stats[h * A.num_q + r0 + r];
      AttnPos p{0.f, 0.f, 0.f};
      float d = 0.f;
      if (st.y != 0.f) {
        p = pos_of(A.q_pos, A.pos_dim, r0 + r);
        d = A.delta[h * A.num_q + r0 + r];
      }
      qst[pb * QT + r] = st;
      qpos[pb * QT + r] = make_float4(p.x, p.y, p.z, d);
    }
  };
  load_tile<Kind, 128, DP, NT>(sK, X.k, hk, j0, nk, dim8, A.k_mask);
  load_tile<Kind, 128, DP, NT>(sV, X.v, hk, j0, nk, dim8, A.k_mask);
  if (t1 > 0) load_queries(0);
  cp_wait_all();
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + C::slot);
  const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
  const uint32_t tS = tmem, tP = tmem + QT, tDk = tmem + 2 * QT, tDv = tDk + DP;

  const int64_t j = j0 + row;
  const bool in = row < nk;
  const bool live = in && (A.k_mask == nullptr || A.k_mask[j] != 0);
  const float us = ldexpf(1.f, -elem_exp<Kind>(X, kWq) - elem_exp<Kind>(X, kWk));
  const int eu = du_exp<Kind>(X);
  constexpr float kUp = Kind::bf16 ? 1.f : 8192.f;  // of P
  BwdRow R{0.f, 0.f, 0.f, ldexpf(1.f, -elem_exp<Kind>(X, kWdo) - elem_exp<Kind>(X, kWv)),
           ldexpf(1.f, eu), {0.f, 0.f, 0.f}};
  if (live) R.p = pos_of(A.k_pos, A.pos_dim, j);
  float px = 0.f, py = 0.f, pz = 0.f;  // over all heads, times 1 / sigma^2
  float g[4] = {};                     // of the current head
  const bool pos_grad = A.pos_k != nullptr;
  bool bad = false;
  unsigned phase = 0;
  int cur = -1;

  if (t1 > 0 && threadIdx.x == 0) {
    products_rows<Kind, QT, DP>(tS, sK, sQ);
    products_rows<Kind, QT, DP>(tP, sV, sG);
    tc_commit(bar);
  }
  auto close_head = [&]() {
    if (cur >= 0 && pos_grad) {
      const float s = A.sigma[cur], w = 1.f / (s * s);
      px = fmaf(w, g[0], px), py = fmaf(w, g[1], py), pz = fmaf(w, g[2], pz);
    }
    g[0] = g[1] = g[2] = 0.f;
  };
  for (int64_t t = 0; t < t1; ++t) {
    const int pb = (int)(t & 1), b = C::STAGES == 1 ? 0 : pb;
    const int h = hk * group + (int)(t / per);
    if (h != cur) {
      close_head();
      cur = h;
      AttnScore sc;
      sc.init(A, h);
      R.su = sc.su * us, R.capl = sc.capl, R.w = sc.w;
    }
    bad = !mbar_wait(bar, phase);
    phase ^= 1;
    tc_fence_after();
    if (C::STAGES > 1 && t + 1 < t1) load_queries(t + 1);
    float v[32], dp[32];
    tmem_ld32(tS + lane_off + 32 * part, v);
    tmem_ld32(tP + lane_off + 32 * part, dp);
    const float4 *qp = qpos + pb * QT + 32 * part;
    const float2 *qs = qst + pb * QT + 32 * part;
#define RA_DKV(C, P, G) dkv_elements<Kind, C, P, G>(v, dp, R, kUp, qs, qp, g)
    if (R.capl > 0.f) {
      if (pos_grad) RA_DKV(true, true, true);
      else if (A.pos_dim > 0) RA_DKV(true, true, false);
      else RA_DKV(true, false, false);
    } else {
      if (pos_grad) RA_DKV(false, true, true);
      else if (A.pos_dim > 0) RA_DKV(false, true, false);
      else RA_DKV(false, false, false);
    }
#undef RA_DKV
    put_weights<Kind>(tS + lane_off + 32 * part, v, Kind::pair);
    put_weights<Kind>(tP + lane_off + 32 * part, dp, Kind::pair);
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    cp_wait_all();
    fence_async_smem();
    tc_fence_before();
    if ((bad = __syncthreads_or(bad))) break;
    if (threadIdx.x == 0) {
      tc_fence_after();
      products_weighted<Kind, QT, DP>(tDv, tS, sG + b * C::QG, false, t > 0);
      products_weighted<Kind, QT, DP>(tDk, tP, sQ + b * C::QG, false, t > 0);
      if (C::STAGES > 1 && t + 1 < t1) {
        products_rows<Kind, QT, DP>(tS, sK, sQ + (b ^ 1) * C::QG);
        products_rows<Kind, QT, DP>(tP, sV, sG + (b ^ 1) * C::QG);
      }
      tc_commit(bar);
    }
    if (C::STAGES == 1 && t + 1 < t1) {
      bad = !mbar_wait(bar, phase);
      phase ^= 1;
      load_queries(t + 1);
      cp_wait_all();
      fence_async_smem();
      if ((bad = __syncthreads_or(bad))) break;
      if (threadIdx.x == 0) {
        tc_fence_after();
        products_rows<Kind, QT, DP>(tS, sK, sQ);
        products_rows<Kind, QT, DP>(tP, sV, sG);
        tc_commit(bar);
      }
    }
  }
  close_head();
  if (t1 > 0 && !bad) {
    bad = !mbar_wait(bar, phase);
    tc_fence_after();
  }
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0) atomicOr(A.status, 1);
  using T = typename Kind::T;
  const int64_t at = (j * A.kv_heads + hk) * A.dim;
  const bool zero = !live || t1 == 0;
  constexpr int last = QT / 32 - 1;
  if (A.dk != nullptr && part == 0)
    write_row<T, DP>(tDk + lane_off, A.scale * ldexpf(1.f, -eu - elem_exp<Kind>(X, kWq)), in, zero,
                     A.dim, (T *)A.dk + at, nullptr);
  if (A.dv != nullptr && part == last)
    write_row<T, DP>(tDv + lane_off, ldexpf(1.f, -elem_exp<Kind>(X, kWdo)) / kUp, in, zero, A.dim,
                     (T *)A.dv + at, nullptr);
  if (pos_grad) {
    float4 *sum = reinterpret_cast<float4 *>(sm);
    if (part > 0) sum[row] = make_float4(px, py, pz, 0.f);
    __syncthreads();
    if (part == 0 && in) {
      if (QT > 32) {
        const float4 o = sum[row];
        px += o.x, py += o.y, pz += o.z;
      }
      if (!live) px = py = pz = 0.f;
      A.pos_k[hk * A.num_k + j] = make_float4(px, py, pz, 0.f);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_free<C::TMEM>(tmem);
  }
}

}  // namespace ra
