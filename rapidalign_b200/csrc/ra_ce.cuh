// ra_ce.cuh -- softmax cross entropy of rows x_i against a table of vectors
// w_v (a large vocabulary), without the logits in memory.
//
//   z_iv = s x_i.w_v            or  c tanh(s x_i.w_v / c)   (soft cap c)
//   lse_i = log sum_v e^z_iv    loss_i = lse_i - z_{i,t_i}
//   dz_iv = (gl_i + ge_i) e^(z_iv - lse_i) - gl_i [v = t_i]
//   du_iv = dz_iv (1 - (z_iv / c)^2)
//   dx_i = s sum_v du_iv w_v    dw_v = s sum_i du_iv x_i
// with gl, ge the upstream gradients of loss and lse.
//
// Forward: one product (ra_gemm16.cuh) whose epilogue keeps a running maximum
// and sum of exponentials of each row over its columns; `ce_rows_kernel`
// joins the column tiles.  All in base 2: t = z log2 e, 2^(t - m).
// Backward: the vocabulary in pieces; per piece the logits again, du in 16
// bits (with the rows' coefficients, so both products read it as it is), then
// dx += du W and dw = du^T X.  Sums over pieces and K slices have one writer
// each and a fixed order: no atomics, bitwise repeatable.
// du is rounded to the operands' 16-bit type (half a step, 2^-8 or 2^-11 of an
// element).  It is held divided by the largest coefficient: a mean's rows then
// have coefficient 1, and the label's element, which outweighs the others, is
// near -1 and exact, where 1 / count would round alike in every row (bf16
// gradients off by 3.9e-3 instead of 2e-3).  In fp16 2^13 more keeps small
// elements normal, and where the rows' coefficients may lie apart (a loss of each
// row, gradients of lse) each row has a power of two of its own in the place of the
// largest: dx takes it back by rows, and dw multiplies a copy of x whose rows have
// taken it, so that a row of small coefficients keeps its bits.  For fp32 inputs
// du, x and w are fp16 pairs hi + lo (22 bits).
// Bound by the tensor cores over a long width, by du's bytes over a short one.
// Measured, logits / du / dx / dw: 8192 x 131072 x 1024 bf16 1.55 / 1.78 / 1.74 /
// 1.64 ms (1.42 to 1.23 PFLOP/s); 65537 x 4099 x 128 fp32 270 / 410 / 290 / 241 us
// (du is 1.07 GB: 164 us each time it passes).
#pragma once

#include "ra_gemm16.cuh"
#include "ra_host.h"

namespace ra {

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;

// header of the state buffer
struct CeHead {
  unsigned amax_x, amax_w;  // bits of the largest finite |x|, |w| (fp32 inputs)
  unsigned amax_g;          // bits of the largest finite coefficient (backward)
  unsigned ticket;          // blocks of ce_rows_kernel done
  long long count;          // rows with a label
  unsigned amax_xu;         // bits of the largest finite |x_i| u_i (rows in units u_i)
};

// Power of two that brings a largest magnitude into [2^13, 2^14), below the
// fp16 maximum 65504.
__device__ __forceinline__ int ce_exp(unsigned amax_bits) {
  if (amax_bits == 0) return 0;
  int e;
  frexpf(__uint_as_float(amax_bits), &e);  // amax = f 2^e, f in [1/2, 1)
  e = 14 - e;
  return e > 100 ? 100 : (e < -100 ? -100 : e);
}
__device__ __forceinline__ float ce_pow2(int e) { return ldexpf(1.f, e); }

__device__ __forceinline__ unsigned finite_bits(float v) {
  const unsigned b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// Eight columns of a row, zeros behind its last; `wide`: rows of 16-byte aligned
// addresses and whole eights.
__device__ __forceinline__ void ce_load8(const float *a, int64_t ld, int cols, int64_t r, int c,
                                         bool wide, float (&v)[8]) {
  const float *p = a + r * ld + c;
  if (wide) {
    const float4 x = __ldg(reinterpret_cast<const float4 *>(p));
    const float4 y = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? p[k] : 0.f;
  }
}
__device__ __forceinline__ void ce_load8(const __half *a, int64_t ld, int cols, int64_t r, int c,
                                         bool wide, float (&v)[8]) {
  const __half *p = a + r * ld + c;
  if (wide) {
    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
    __half h[8];
    memcpy(h, &u, 16);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __half2float(h[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? __half2float(p[k]) : 0.f;
  }
}
template <class T>
struct CeMatrix {
  const T *a;
  int64_t rows, ld;
  int cols;
  const float *unit;  // of each row, or null: 1
  unsigned *word;
  __half *hi, *lo;  // [rows, 8 eights]; lo null: hi alone
  __device__ __forceinline__ bool wide() const {
    return ((uintptr_t)a & 15) == 0 && ld % (16 / (int)sizeof(T)) == 0 && (cols & 7) == 0;
  }
  __device__ __forceinline__ void load(int64_t r, int c, bool wide, float (&v)[8]) const {
    ce_load8(a, ld, cols, r, c, wide, v);
    if (unit != nullptr) {
      const float u = unit[r];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= u;
    }
  }
};

// largest finite |a| of x (blockIdx.y = 0) and w into their words
template <class T>
__global__ void __launch_bounds__(256) ce_amax_kernel(const CeMatrix<T> x, const CeMatrix<T> w) {
  const CeMatrix<T> &m = blockIdx.y ? w : x;
  const int eights = (m.cols + 7) >> 3;
  const bool wide = m.wide();
  unsigned best = 0;
  const int64_t n = m.rows * eights;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = n < ((int64_t)1 << 31) ? (unsigned)i / (unsigned)eights : i / eights;
    float v[8];
    m.load(r, (int)(i - r * eights) * 8, wide, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned b = finite_bits(v[k]);
      best = b > best ? b : best;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned b = __shfl_xor_sync(kFull, best, o);
    best = b > best ? b : best;
  }
  if ((threadIdx.x & 31) == 0 && best) atomicMax(m.word, best);  // a maximum: any order
}

// a 2^e = hi + lo in fp16, rows padded with zeros to whole eights
template <class T>
__global__ void __launch_bounds__(256) ce_split_kernel(const CeMatrix<T> x, const CeMatrix<T> w) {
  const CeMatrix<T> &m = blockIdx.y ? w : x;
  const int eights = (m.cols + 7) >> 3;
  const bool wide = m.wide();
  const float sc = ce_pow2(ce_exp(*m.word));
  const int64_t n = m.rows * eights;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = n < ((int64_t)1 << 31) ? (unsigned)i / (unsigned)eights : i / eights;
    float v[8];
    m.load(r, (int)(i - r * eights) * 8, wide, v);
    __half h[8], l[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float y = v[k] * sc;
      h[k] = __float2half_rn(y);
      l[k] = __float2half_rn(y - __half2float(h[k]));
    }
    uint4 u;
    memcpy(&u, h, 16);
    reinterpret_cast<uint4 *>(m.hi)[i] = u;
    if (m.lo == nullptr) continue;
    memcpy(&u, l, 16);
    reinterpret_cast<uint4 *>(m.lo)[i] = u;
  }
}

// z = s acc or c tanh(s acc / c), in units of log 2.  PAIRS: fp32 inputs.
template <bool PAIRS>
struct CeLogit {
  float scale, cap;
  const CeHead *head;  // split scales of pairs
  struct Fixed {
    float f, capl;  // t = acc f, or capl tanh(acc f)
  };
  __device__ __forceinline__ Fixed fixed() const {
    const float f = PAIRS ? ce_pow2(-ce_exp(head->amax_x) - ce_exp(head->amax_w)) : 1.f;
    return cap > 0.f ? Fixed{scale * f / cap, cap * kLog2e} : Fixed{scale * f * kLog2e, 0.f};
  }
};

// Forward epilogue: maximum and sum of 2^(t - m) over the thread's columns.
template <bool PAIRS>
struct CeEpiLse {
  CeLogit<PAIRS> lg;
  int64_t rows, vocab;
  const int64_t *target;
  float2 *part;  // [kGmParts n_tiles][ld]
  int64_t ld;
  float *zt;  // [rows] t at the label
  using Fixed = typename CeLogit<PAIRS>::Fixed;
  struct Row {
    int64_t target;
  };
  __device__ __forceinline__ Fixed fixed() const { return lg.fixed(); }
  __device__ __forceinline__ Row begin(const GmUnit &w, int row) const {
    const int64_t r = (int64_t)w.m * kGmM + row;
    return {r < rows ? target[r] : -1};
  }
  template <int TN, class Src>
  __device__ __forceinline__ void run(const Fixed &F, const Row &R, const GmUnit &w, int row,
                                      int col, const Src &src, const GmOut &out_rows) const {
    const int64_t r = (int64_t)w.m * kGmM + row, c0 = (int64_t)w.n * TN + col;
    const f2_t f2 = pk(F.f, F.f);
    float m = -INFINITY, s = 0.f;
#pragma unroll Src::unroll
    for (int c = 0; c < TN / kGmParts; c += 32) {
      float v[32];
      src.get(c, v);
      const int64_t left = vocab - (c0 + c);
      if (F.capl > 0.f) {
        const f2_t capl = pk(F.capl, F.capl);
        if (all_small(v, F.f)) {
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            upk(mul2(capl, tanh_small2(mul2(pk(v[j], v[j + 1]), f2))), v[j], v[j + 1]);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            upk(mul2(capl, tanh2(mul2(pk(v[j], v[j + 1]), f2))), v[j], v[j + 1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; j += 2) upk(mul2(pk(v[j], v[j + 1]), f2), v[j], v[j + 1]);
      }
      if (left < 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j >= left) v[j] = -INFINITY;
      }
      const int64_t at = R.target - (c0 + c);
      if (at >= 0 && at < 32 && at < left) {
        float z = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j)  // not v[at]: that would put v into local memory
          asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, %2;\n\t@p mov.f32 %0, %3;\n\t}"
                       : "+f"(z)
                       : "r"((int)at), "r"(j), "f"(v[j]));
        zt[r] = z;
      }
      float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
      for (int j = 4; j < 32; ++j) mx[j & 3] = fmaxf(mx[j & 3], v[j]);
      mx[0] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const float mn = fmaxf(m, mx[0]);
      if (mn > -INFINITY || mx[0] != mx[0]) {
        const f2_t ref = pk(-mn, -mn);
        f2_t sum[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float x, y;
          upk(add2(pk(v[j], v[j + 1]), ref), x, y);
          sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], pk(ex2(x), ex2(y)));
        }
        const f2_t both = add2(sum[0], sum[1]);
        s = s * (m > -INFINITY ? ex2(m - mn) : 0.f) + (lo_of(both) + hi_of(both));
        m = mn;
      }
    }
    part[((int64_t)w.n * kGmParts + col / (TN / kGmParts)) * ld + r] = make_float2(m, s);
  }
};

// Joins the parts of TX rows of a pass over rows [r0, r0 + pass_rows), TY threads
// a row; losses, lse, the rows' (m, sum) for the
// backward, and the sum or mean of the losses (block sums in fp64, added in
// block order by the block that finishes last).
template <int TX, int TY>
__global__ void __launch_bounds__(TX * TY) ce_rows_kernel(const float2 *part, int64_t ld, int parts,
                                                          int64_t r0, int64_t pass_rows,
                                                          int64_t rows, int64_t vocab,
                                                          const int64_t *target, int64_t ignore,
                                                          const float *zt, int reduction,
                                                          float *loss, float *lse, float2 *stats,
                                                          CeHead *head, double2 *blocks) {
  __shared__ float2 sh[TY][TX + 1];
  __shared__ double red[TX * TY / 32 * 2];
  __shared__ bool last;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int64_t in_pass = blockIdx.x * (int64_t)TX + tx, r = r0 + in_pass;
  const unsigned all_blocks = (unsigned)ceil_div(rows, (int64_t)TX);
  float m = -INFINITY, s = 0.f;
  if (in_pass < pass_rows) {
    for (int p = ty; p < parts; p += TY * 8) {  // eight loads in flight
      float2 v[8];
      float mn = m;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = p + TY * k < parts ? part[(int64_t)(p + TY * k) * ld + in_pass]
                                  : make_float2(-INFINITY, 0.f);
        mn = fmaxf(mn, v[k].x);
      }
      // no finite maximum yet: the sums are 0, or NaN
      const float ref = mn > -INFINITY ? mn : 0.f;
      s *= m > -INFINITY ? ex2(m - ref) : 1.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s = fmaf(v[k].y, v[k].x > -INFINITY ? ex2(v[k].x - ref) : 1.f, s);
      m = mn;
    }
  }
  sh[ty][tx] = make_float2(m, s);
  __syncthreads();
  // the first warp: 32 / TX threads a row, in order
  if (threadIdx.x < 32) {
    constexpr int kSide = 32 / TX;
    float M = -INFINITY;
    for (int k = ty; k < TY; k += kSide) M = fmaxf(M, sh[k][tx].x);
#pragma unroll
    for (int o = TX; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(kFull, M, o));
    float S = 0.f;
    for (int k = ty; k < TY; k += kSide) {
      const float2 v = sh[k][tx];
      S += v.x > -INFINITY ? v.y * ex2(v.x - M) : v.y;
    }
#pragma unroll
    for (int o = TX; o < 32; o <<= 1) S += __shfl_xor_sync(kFull, S, o);
    double row_loss = 0.0;
    long long labelled = 0;
    if (ty == 0 && in_pass < pass_rows) {
      const double l = (double)M * kLn2 + log((double)S);
      const int64_t t = target[r];
      if (t != ignore) {
        labelled = 1;
        // a label outside the table is never read: its loss is NaN
        row_loss = t >= 0 && t < vocab ? l - (double)zt[r] * kLn2 : (double)NAN;
      }
      lse[r] = (float)l;
      stats[r] = make_float2(M, S);
      if (reduction == RA_REDUCE_NONE) loss[r] = (float)row_loss;
    }
    if (reduction != RA_REDUCE_NONE) {
      const double sum = warp_sum(row_loss);
      const double cnt = warp_sum((double)labelled);
      if (threadIdx.x == 0) {
        blocks[r0 / TX + blockIdx.x] = make_double2(sum, cnt);
        __threadfence();
        last = atomicAdd(&head->ticket, 1u) == all_blocks - 1;
      }
    }
  }
  if (reduction == RA_REDUCE_NONE) return;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double acc[2] = {0.0, 0.0};
  for (int64_t b = threadIdx.x; b < all_blocks; b += TX * TY) {
    const double2 v = __ldcg(blocks + b);
    acc[0] += v.x;
    acc[1] += v.y;
  }
  block_sum_n<2>(acc, red);
  if (threadIdx.x == 0) {
    *loss = (float)(reduction == RA_REDUCE_MEAN ? acc[0] / acc[1] : acc[0]);
    head->count = (long long)acc[1];
  }
}

// Per row (gl + ge, gl) of the backward; 0 for a row without a label, NaN
// for a label outside the table (as its loss).  `unit`: null, or the rows' powers
// of two, that are taken out here; the largest coefficient then counts as 1.
__global__ void __launch_bounds__(256) ce_coef_kernel(const int64_t *target, int64_t rows,
                                                      int64_t vocab, int64_t ignore, int reduction,
                                                      const float *g_loss, const float *g_lse,
                                                      CeHead *head, float2 *coef, float *unit) {
  unsigned best = 0;
  for (int64_t r = blockIdx.x * (int64_t)256 + threadIdx.x; r < rows;
       r += (int64_t)gridDim.x * 256) {
    const int64_t t = target[r];
    float gl = 0.f;
    if (g_loss != nullptr && t != ignore) {
      gl = g_loss[reduction == RA_REDUCE_NONE ? r : 0];
      if (reduction == RA_REDUCE_MEAN) gl = (float)((double)gl / (double)head->count);
      if (t < 0 || t >= vocab) gl = NAN;
    }
    float c = gl + (g_lse != nullptr ? g_lse[r] : 0.f);
    const unsigned a = finite_bits(c), b = finite_bits(gl), top = a > b ? a : b;
    if (unit != nullptr) {
      // in [1, 2) of the unit, so that fp16's smallest step is no more of it than of
      // the largest coefficient elsewhere; of a row without coefficients 0, so that
      // its x counts for nothing
      int e = 1;
      if (top) frexpf(__uint_as_float(top), &e);
      e = e > 127 ? 126 : (e < -99 ? -100 : e - 1);
      const float u = top ? ce_pow2(e) : c == 0.f && gl == 0.f ? 0.f : 1.f;
      unit[r] = u;
      if (top) {
        const float inv = ce_pow2(-e);
        c *= inv;
        gl *= inv;
      }
    } else {
      best = top > best ? top : best;
    }
    coef[r] = make_float2(c, gl);
  }
  if (unit != nullptr) {
    if (blockIdx.x == 0 && threadIdx.x == 0) head->amax_g = __float_as_uint(1.f);
    return;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned b = __shfl_xor_sync(kFull, best, o);
    best = b > best ? b : best;
  }
  if ((threadIdx.x & 31) == 0 && best) atomicMax(&head->amax_g, best);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return bits_as<uint32_t>(v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return bits_as<uint32_t>(v);
}

template <bool BF16>
constexpr float kCeGradScale = BF16 ? 1.f : 8192.f;  // |du| < 2 times this (4, in rows' units)

// Backward epilogue: du of one piece of the vocabulary, in 16 bits.
template <bool BF16, bool PAIRS>
struct CeEpiGrad {
  CeLogit<PAIRS> lg;
  int64_t rows, vocab, v0;  // v0: the piece's first column
  const int64_t *target;
  const float2 *stats, *coef;
  const CeHead *head;
  uint16_t *hi, *lo;  // [128 m_tiles, ldg]
  int64_t ldg;
  struct Fixed {
    typename CeLogit<PAIRS>::Fixed lg;
    float top;  // the largest coefficient
  };
  struct Row {
    float2 cf, st;
    int64_t target;
  };
  __device__ __forceinline__ Fixed fixed() const {
    return {lg.fixed(), __uint_as_float(head->amax_g)};
  }
  __device__ __forceinline__ Row begin(const GmUnit &w, int row) const {
    const int64_t r = (int64_t)w.m * kGmM + row;
    if (r >= rows) return {make_float2(0.f, 0.f), make_float2(0.f, 1.f), -1};
    return {coef[r], stats[r], target[r] - v0};
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return BF16 ? pack_bf16(a, b) : pack_f16(a, b);
  }
  // the halves that `hi` left over
  static __device__ __forceinline__ uint32_t rest(uint32_t hi, float a, float b) {
    const float2 f = __half22float2(bits_as<__half2>(hi));
    return pack_f16(a - f.x, b - f.y);
  }
  template <int TN, class Src>
  __device__ __forceinline__ void run(const Fixed &F, const Row &R, const GmUnit &w, int row,
                                      int col, const Src &src, const GmOut &out_rows) const {
    const int64_t r = (int64_t)w.m * kGmM + row, c0 = (int64_t)w.n * TN + col;
    // c / top before the scale: 1 where all coefficients are alike
    const float gl = R.cf.y / F.top * kCeGradScale<BF16>, m = -R.st.x;
    const float cp = R.cf.x / F.top * kCeGradScale<BF16> / R.st.y;
    const bool off = R.cf.x == 0.f && R.cf.y == 0.f;
    const f2_t f2 = pk(F.lg.f, F.lg.f), nm = pk(m, m), pc = pk(cp, cp);
#pragma unroll Src::unroll
    for (int c = 0; c < TN / kGmParts; c += 32) {
      float v[32];
      src.get(c, v);
      const int64_t at = R.target - (c0 + c);
      const bool hit = at >= 0 && at < 32;
      if (F.lg.capl > 0.f) {
        const f2_t capl = pk(F.lg.capl, F.lg.capl), one = pk(1.f, 1.f), neg = pk(-1.f, -1.f);
        const bool small = all_small(v, F.lg.f);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const f2_t u = mul2(pk(v[j], v[j + 1]), f2);
          const f2_t th = small ? tanh_small2(u) : tanh2(u);
          float x, y;
          upk(fma2(th, capl, nm), x, y);
          f2_t g = mul2(pk(ex2(x), ex2(y)), pc);
          if (hit) {
            upk(g, x, y);
            g = pk(j == (int)at ? x - gl : x, j + 1 == (int)at ? y - gl : y);
          }
          upk(mul2(g, fma2(mul2(th, neg), th, one)), v[j], v[j + 1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float x, y;
          upk(fma2(pk(v[j], v[j + 1]), f2, nm), x, y);
          upk(mul2(pk(ex2(x), ex2(y)), pc), v[j], v[j + 1]);
        }
        if (hit) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = j == (int)at ? v[j] - gl : v[j];
        }
      }
      if (off) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0.f;
      }
      uint4 h[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        h[q] = make_uint4(pack(v[8 * q], v[8 * q + 1]), pack(v[8 * q + 2], v[8 * q + 3]),
                          pack(v[8 * q + 4], v[8 * q + 5]), pack(v[8 * q + 6], v[8 * q + 7]));
      const int64_t at0 = (r - (threadIdx.x & 31)) * ldg + c0 + c;
      out_rows.rows64(h, [&](int row_, int j, uint4 x) {
        *reinterpret_cast<uint4 *>(hi + at0 + row_ * ldg + 8 * j) = x;
      });
      if (PAIRS) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          h[q] = make_uint4(rest(h[q].x, v[8 * q], v[8 * q + 1]),
                            rest(h[q].y, v[8 * q + 2], v[8 * q + 3]),
                            rest(h[q].z, v[8 * q + 4], v[8 * q + 5]),
                            rest(h[q].w, v[8 * q + 6], v[8 * q + 7]));
        out_rows.rows64(h, [&](int row_, int j, uint4 x) {
          *reinterpret_cast<uint4 *>(lo + at0 + row_ * ldg + 8 * j) = x;
        });
      }
    }
  }
};

__device__ __forceinline__ void store_as(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_as(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// what undoes the scales of a product: s top / kCeGradScale 2^-exponent
struct CeAlpha {
  float scale;
  const unsigned *top;    // the largest coefficient
  const unsigned *other;  // amax word of the other operand, or null
  __device__ __forceinline__ float value() const {
    return scale * __uint_as_float(*top) * ce_pow2(other ? -ce_exp(*other) : 0);
  }
};

// Gradient epilogue: the finished product, or one K slice's sum over the
// pieces (`add`: later pieces).
template <class T>
struct CeEpiOut {
  CeAlpha alpha;
  int64_t rows, cols;
  T *out;       // [rows, cols], or null
  float *part;  // [slices][rows, cols]
  int add;
  const float *unit;  // of the rows, or null
  struct Fixed {
    float al;
  };
  struct Row {
    float unit;
  };
  __device__ __forceinline__ Fixed fixed() const { return {out ? alpha.value() : 1.f}; }
  __device__ __forceinline__ Row begin(const GmUnit &w, int row) const {
    const int64_t r = (int64_t)w.m * kGmM + row;
    return {unit != nullptr && r < rows ? unit[r] : 1.f};
  }
  template <int TN, class Src>
  __device__ __forceinline__ void run(const Fixed &F, const Row &R, const GmUnit &w, int row,
                                      int col, const Src &src, const GmOut &out_rows) const {
    const float al = F.al * R.unit;
    const int64_t r = (int64_t)w.m * kGmM + row, c0 = (int64_t)w.n * TN + col;
    const int64_t w0 = r - (threadIdx.x & 31);  // the warp's first row
    // 16-byte aligned rows: fp32 sums, or results; 8-byte ones of 16-bit results
    const bool wide = cols % (out != nullptr ? 16 / (int)sizeof(T) : 4) == 0;
    const bool half = cols % 4 == 0;
#pragma unroll Src::unroll
    for (int c = 0; c < TN / kGmParts; c += 32) {
      float v[32];
      src.get(c, v);
      const int64_t left = cols - (c0 + c);
      if (left <= 0) break;  // the same for the warp
      if (out != nullptr && sizeof(T) == 2) {
        uint4 x[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          T t[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) store_as(t + k, v[8 * q + k] * al);
          memcpy(&x[q], t, 16);
        }
        out_rows.rows64(x, [&](int row_, int j, uint4 u) {
          if (w0 + row_ >= rows) return;
          T *q = out + (w0 + row_) * cols + c0 + c + 8 * j;
          const int n = (int)min((int64_t)8, left - 8 * j);
          if (wide && n == 8) {
            *reinterpret_cast<uint4 *>(q) = u;
          } else if (half) {  // n is a multiple of 4
            if (n >= 4) *reinterpret_cast<uint2 *>(q) = make_uint2(u.x, u.y);
            if (n == 8) *reinterpret_cast<uint2 *>(q + 4) = make_uint2(u.z, u.w);
          } else {
            T t[8];
            memcpy(t, &u, 16);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k < n) q[k] = t[k];
          }
        });
      } else {
        float *base = out != nullptr ? reinterpret_cast<float *>(out)
                                     : part + (int64_t)w.slice * rows * cols;
        const bool more = out == nullptr && add;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint4 x[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            x[q] = make_uint4(__float_as_uint(v[16 * hf + 4 * q] * al),
                              __float_as_uint(v[16 * hf + 4 * q + 1] * al),
                              __float_as_uint(v[16 * hf + 4 * q + 2] * al),
                              __float_as_uint(v[16 * hf + 4 * q + 3] * al));
          out_rows.rows64(x, [&](int row_, int j, uint4 u) {
            if (w0 + row_ >= rows) return;
            float *q = base + (w0 + row_) * cols + c0 + c + 16 * hf + 4 * j;
            const int64_t n = left - 16 * hf - 4 * j;
            if (wide && n >= 4) {
              float4 *q4 = reinterpret_cast<float4 *>(q);
              float4 o = more ? *q4 : make_float4(0.f, 0.f, 0.f, 0.f);
              *q4 = make_float4(o.x + __uint_as_float(u.x), o.y + __uint_as_float(u.y),
                                o.z + __uint_as_float(u.z), o.w + __uint_as_float(u.w));
            } else {
              const float t[4] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z),
                                  __uint_as_float(u.w)};
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < n) q[k] = (more ? q[k] : 0.f) + t[k];
            }
          });
        }
      }
    }
  }
};

// out = alpha (sum of the K slices, in order)
template <class T>
__global__ void __launch_bounds__(256) ce_join_kernel(const float *part, int slices, int64_t n,
                                                      CeAlpha alpha, T *out) {
  const float al = alpha.value();
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int s = 0; s < slices; ++s) v += part[s * n + i];
    store_as(out + i, v * al);
  }
}

}  // namespace ra
