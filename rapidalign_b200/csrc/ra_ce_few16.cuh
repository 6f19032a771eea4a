// ra_ce_few16.cuh -- forward of the linear cross entropy for up to eight rows,
// 16-bit inputs.
//
// Bound by the table's bytes, each read once.  A warp takes 16 rows of the table
// at a time: 128 columns (4 KB) a step, copied steps ahead into a ring in shared
// memory (16 bytes a lane, 256 in a row), and warp-wide 16 x 8 x 16 products with
// the table as the 16 rows and x as the eight columns, so that none of a product
// is idle but the rows that x lacks.  A step's sums are the tensor core's, the
// steps are added in fp32.  Each lane ends with the logits of two table rows for
// two rows of x, and keeps their running maxima and sums; those are joined over
// the warp and the CTA, and the CTAs by ce_rows_kernel.
// Measured: 5 rows against 131072 x 1024 in bf16 (268 MB) 45 us (6.0 TB/s); in the FMA form
// (ra_ce_few.cuh) 62 us; the product kernel of ra_gemm16.cuh, 128 rows for these
// few, 66 us.
#pragma once

#include "ra_ce_few.cuh"

namespace ra {

constexpr int kCeFew16K = 128, kCeFew16Rows = 16, kCeFew16Stages = 4;
constexpr int kCeFew16Step = kCeFew16Rows * kCeFew16K * 2;  // bytes
constexpr int kCeFew16Ring = kCeFewWarps * kCeFew16Stages * kCeFew16Step;
// bytes of a row of x in shared memory: whole steps, an odd number of 16s so that
// eight rows lie in eight bank groups
__host__ __device__ constexpr int ce_few16_row(int dim) {
  return (dim + kCeFew16K - 1) / kCeFew16K * kCeFew16K * 2 + 16;
}
// the most of it: x up to kCeFewSmem in fp32
constexpr int kCeFew16MostSmem =
    kCeFew16Ring + (int)kCeFewSmem / 2 + kCeFewRows * (2 * kCeFew16K + 16);
constexpr int ce_few16_smem(int rows, int dim) { return kCeFew16Ring + rows * ce_few16_row(dim); }

template <class T>
__global__ void __launch_bounds__(32 * kCeFewWarps, 1)
    ce_few16_kernel(const T *x, int64_t ldx, const T *w, int64_t ldw, int rows, int64_t vocab,
                    int dim, float scale, float cap, const int64_t *target, float2 *part,
                    float *zt) {
  constexpr int S = kCeFew16Stages;
  extern __shared__ uint4 few16_sm[];
  __shared__ float2 sml[kCeFewWarps][kCeFewRows];
  uint8_t *sm = reinterpret_cast<uint8_t *>(few16_sm);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lr = lane & 7, lm = lane >> 3, g = lane >> 2, n0 = 2 * (lane & 3);
  const uint32_t ring = smem_u32(sm) + warp * S * kCeFew16Step;
  const int xrow = ce_few16_row(dim), chunks = (dim + kCeFew16K - 1) / kCeFew16K;
  const int64_t step = (int64_t)gridDim.x * kCeFewWarps * kCeFew16Rows;
  const int64_t first = ((int64_t)blockIdx.x * kCeFewWarps + warp) * kCeFew16Rows;
  // what is copied next: rows from iv on, chunk ik
  int64_t iv = first;
  int ik = 0;
  auto issue = [&](int slot) {
    if (iv < vocab) {
      const uint32_t at = ring + slot * kCeFew16Step;
      const int c = lane & 15, col = ik * kCeFew16K + c * 8;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const int r = 2 * p + (lane >> 4);
        const bool on = iv + r < vocab && col < dim;  // dim is a multiple of 8
        few_copy(at + few_at<128>(r, c), on ? w + (iv + r) * ldw + col : w, on);
      }
      if (++ik == chunks) ik = 0, iv += step;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) issue(s);
  for (int e = threadIdx.x; e < rows * (xrow / 2); e += 32 * kCeFewWarps) {
    const int n = e / (xrow / 2), d = e - n * (xrow / 2);
    reinterpret_cast<uint16_t *>(sm + kCeFew16Ring)[e] =
        d < dim ? reinterpret_cast<const uint16_t *>(x)[n * ldx + d] : (uint16_t)0;
  }
  __syncthreads();
  // row lr of x; of the rows that are not there the first, which nothing reads
  const uint32_t sx = smem_u32(sm) + kCeFew16Ring + (lr < rows ? lr : 0) * xrow + lm * 16;
  const float f = cap > 0.f ? scale / cap : scale * kLog2e, capl = cap * kLog2e;
  int64_t tg[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) tg[e] = n0 + e < rows ? target[n0 + e] : -1;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  int slot = 0;
  for (int64_t v0 = first; v0 < vocab; v0 += step) {
    float sum[4] = {};
    for (int k = 0; k < chunks; ++k) {
      __syncwarp();  // the slot before this one has been read
      issue((slot + S - 1) % S);
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
      __syncwarp();
      const uint32_t at = ring + slot * kCeFew16Step, xk = sx + k * kCeFew16K * 2;
      float d[2][4] = {};
#pragma unroll
      for (int s = 0; s < kCeFew16K / 16; s += 2) {
        uint32_t a[4], b[4];
        few_ldm<false>(b, xk + s * 32);
        few_ldm<false>(a, at + few_at<128>(8 * (lm & 1) + lr, 2 * s + (lm >> 1)));
        few_mma<T>(d[0], a, b[0], b[1]);
        few_ldm<false>(a, at + few_at<128>(8 * (lm & 1) + lr, 2 * s + 2 + (lm >> 1)));
        few_mma<T>(d[1], a, b[2], b[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += d[0][e] + d[1][e];
      slot = (slot + 1) % S;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t v = v0 + g + 8 * (e >> 1);
      float z = sum[e] * f;
      if (cap > 0.f) z = capl * tanh_step(z);
      if (v < vocab) {
        if (tg[e & 1] == v) zt[n0 + (e & 1)] = z;
        ce_few_add(m[e & 1], l[e & 1], z);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    ce_few_join<4, 32>(m[e], l[e]);
    if (g == 0) sml[warp][n0 + e] = make_float2(m[e], l[e]);
  }
  __syncthreads();
  if (threadIdx.x < rows) ce_few_cta(&sml[0][threadIdx.x], kCeFewRows, part, threadIdx.x);
}

}  // namespace ra
