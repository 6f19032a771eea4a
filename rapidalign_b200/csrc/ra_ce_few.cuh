// ra_ce_few.cuh -- forward of the linear cross entropy for up to eight rows:
// scoring a few tokens against the whole table; fp32 inputs, and what it shares
// with the 16-bit form (ra_ce_few16.cuh).
//
// Bound by the table's bytes, each read once.  x stays in shared memory in fp32;
// LPK lanes (by the width: whole rows narrower than 256 side by side) take R rows
// of the table at a time, 8 columns a lane, with all N dots of the R in
// registers.  The R N dots are joined over the lanes by halving, so that each
// lane ends with one logit (or a copy of one, or two of one row) and its own
// running maximum and sum; those are joined over the warp and the CTA, and the
// CTAs by ce_rows_kernel.  Exact products of the inputs, fp32 sums: no halves.
// Measured: 5 rows against 131072 x 1024 (537 MB): 98 us (5.5 TB/s), 8 rows
// 113 us (bound by the reads of x in shared memory); 8 rows against 2097152 x 64
// 148 us, with 32 lanes a row whatever its width 646 us.
#pragma once

#include "ra_ce.cuh"
#include "ra_few.cuh"

namespace ra {

constexpr int kCeFewRows = 8, kCeFewWarps = 8;
constexpr size_t kCeFewSmem = 64 * 1024;  // most of x in shared memory: three CTAs an SM

// one more logit (base 2) to a running maximum and sum
__device__ __forceinline__ void ce_few_add(float &m, float &l, float z) {
  const float mx = fmaxf(m, z);
  if (mx > -INFINITY) {
    l = (m > -INFINITY ? l * ex2(m - mx) : l) + ex2(z - mx);
    m = mx;
  } else {
    l += z != z ? z : 0.f;
  }
}
// those of the lanes FROM, 2 FROM .. apart, below TO
template <int FROM, int TO>
__device__ __forceinline__ void ce_few_join(float &m, float &l) {
  float mx = m;
#pragma unroll
  for (int o = FROM; o < TO; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
  l *= m > -INFINITY ? ex2(m - mx) : 1.f;  // without a maximum: 0, or NaN
#pragma unroll
  for (int o = FROM; o < TO; o <<= 1) l += __shfl_xor_sync(kFull, l, o);
  m = mx;
}
// and of the warps (sml[warp * ld]), to the CTA's part of row n
__device__ __forceinline__ void ce_few_cta(const float2 *sml, int ld, float2 *part, int n) {
  float M = -INFINITY, S = 0.f;
  for (int k = 0; k < kCeFewWarps; ++k) M = fmaxf(M, sml[k * ld].x);
  for (int k = 0; k < kCeFewWarps; ++k) {
    const float2 s = sml[k * ld];
    S += s.x > -INFINITY ? s.y * ex2(s.x - M) : s.y;
  }
  part[blockIdx.x * kCeFewRows + n] = make_float2(M, S);
}

template <int N, int LPK>
__global__ void __launch_bounds__(32 * kCeFewWarps, 2)
    ce_few_kernel(const float *x, int64_t ldx, const float *w, int64_t ldw, int rows, int64_t vocab,
                  int dim, float scale, float cap, const int64_t *target, float2 *part, float *zt) {
  constexpr int R = N > 4 ? 2 : 4, SUBS = 32 / LPK, NV = R * N;
  constexpr int V = NV > LPK ? NV / LPK : 1;  // logits a lane finishes, all of one row
  constexpr int kDup = NV < LPK ? LPK / NV : 1;  // lanes with the same logit
  static_assert(V <= R, "a lane's logits are of one row");
  // x: of each eight columns the first four, then (dim / 2 floats on) the others,
  // so that lanes side by side read 16 bytes side by side
  extern __shared__ float xs[];  // [rows][2][dim / 8][4]
  __shared__ float2 sml[kCeFewWarps][N];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane % LPK, sub = lane / LPK;
  for (int e = threadIdx.x; e < rows * dim; e += 32 * kCeFewWarps) {
    const int n = e / dim, d = e - n * dim;
    xs[n * dim + (d & 4 ? dim / 2 : 0) + (d >> 3) * 4 + (d & 3)] = x[n * ldx + d];
  }
  __syncthreads();
  // this lane's row of x, and its first table row of R
  const int idx = c * NV / LPK, mn = idx / R, mr = idx % R;
  const float f = cap > 0.f ? scale / cap : scale * kLog2e, capl = cap * kLog2e;
  const int64_t tg = mn < rows ? target[mn] : -1;
  float m = -INFINITY, l = 0.f;
  const int64_t step = (int64_t)gridDim.x * kCeFewWarps * (R * SUBS);
  const int chunks = (dim + 8 * LPK - 1) / (8 * LPK);
  // the loads run one chunk ahead, over the ends of the rows
  Few8<float> nx[R];
  auto fetch = [&](int64_t v, int k) {
    const int col = (k * LPK + c) * 8;
    const float *p = w + v * ldw + col;
#pragma unroll
    for (int r = 0; r < R; ++r)  // dim is a multiple of 8
      nx[r].load(p + r * SUBS * ldw, col < dim && v + r * SUBS < vocab);
  };
  int64_t v0 = ((int64_t)blockIdx.x * kCeFewWarps + warp) * (R * SUBS) + sub;
  fetch(v0, 0);
  for (; v0 - sub < vocab; v0 += step) {
    f2_t acc[N][R] = {};
    for (int k = 0; k < chunks; ++k) {
      f2_t wv[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r) nx[r].get(wv[r]);
      if (k + 1 < chunks) fetch(v0, k + 1);
      else fetch(v0 + step, 0);
      const int col = (k * LPK + c) * 8;
      if (col >= dim) continue;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (n >= rows) break;  // the same for all: five rows cost five
        const float *xn = xs + n * dim + col / 2;
        const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(xn);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2 *>(xn + dim / 2);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          acc[n][r] = fma2(a.x, wv[r][0], acc[n][r]);
          acc[n][r] = fma2(a.y, wv[r][1], acc[n][r]);
          acc[n][r] = fma2(b.x, wv[r][2], acc[n][r]);
          acc[n][r] = fma2(b.y, wv[r][3], acc[n][r]);
        }
      }
    }
    float t[NV];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < R; ++r) t[n * R + r] = lo_of(acc[n][r]) + hi_of(acc[n][r]);
    few_halve<NV, LPK>(t, c);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int64_t v = v0 + (mr + e) * SUBS;
      float z = t[e] * f;
      if (cap > 0.f) z = capl * tanh_step(z);
      if (v < vocab) {
        if (tg == v) zt[mn] = z;
        ce_few_add(m, l, z);
      }
    }
  }
  // the lanes of a row of x, then the warps
  ce_few_join<kDup, LPK / N>(m, l);
  ce_few_join<LPK, 32>(m, l);
  if (sub == 0 && c % (LPK / N) == 0) sml[warp][mn] = make_float2(m, l);
  __syncthreads();
  if (threadIdx.x < rows) ce_few_cta(&sml[0][threadIdx.x], N, part, threadIdx.x);
}

}  // namespace ra
