// ra_attn.cuh -- kernel attention over ragged batches of graphs.
//
// For query i and key j of one graph, head h (key head h' = h / (H / H')):
//   u = a q_i.k_j,   s = u  or  c tanh(u / c)   (soft cap c)
//   s -= |p_i - p_j|^2 / (2 sigma_h^2)          (positions, if given)
//   P_ij = e^s / sum_j e^s over the keys the mask leaves,  o_i = sum_j P_ij v_j
// a query without keys (or masked) gives 0.  Backward, with D_i = do_i.o_i:
//   dP = do_i.v_j,   dS = P (dP - D_i),   dU = dS (1 - (s / c)^2) a
//   dq_i = sum_j dU k_j,  dk_j = sum_i dU q_i,  dv_j = sum_i P do_i
//   dp_i = -sum_hj dS (p_i - p_j) / sigma_h^2,  dp_j the same with + over i
//   dsigma_h = sum_ij dS |p_i - p_j|^2 / sigma_h^3
// Scores are kept in base 2 (t = s log2 e), statistics per row as m and 1 / l
// with l = sum 2^(t - m); a row without keys has +inf and 0, so that every P of
// it is 0.  All sums are in fp32 or more; one writer per result, no atomics.
//
// This file: the parts every variant shares, and the kernels with one warp a
// row (any head width up to 256, any strides).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ra_common.cuh"
#include "ra_few.cuh"

namespace ra {

constexpr int kAttnMaxDim = 256;
constexpr int kAttnWarps = 4;  // rows a CTA of the warp-per-row kernels
constexpr float kAttnLog2e = 1.4426950408889634f;

// Rows of graph g, and the 128-row tiles of all graphs: from offsets and a
// list (ragged), or of `per` rows each (padded clouds).
struct AttnSegs {
  const int64_t *ptr;  // [graphs + 1], or null
  const int4 *tiles;   // (first row, rows, the other side's first row and rows)
  int64_t per;
  __device__ __forceinline__ int64_t begin(int64_t g) const { return ptr ? ptr[g] : g * per; }
  __device__ __forceinline__ int64_t end(int64_t g) const { return ptr ? ptr[g + 1] : (g + 1) * per; }
  __device__ __forceinline__ int4 tile(int64_t t, const AttnSegs &other) const {
    if (ptr) return tiles[t];
    const int64_t each = (per + 127) >> 7, g = t / each, n = t % each;
    return make_int4((int)(g * per + 128 * n), (int)min((int64_t)128, per - 128 * n),
                     (int)(g * other.per), (int)other.per);
  }
  // the graph of tile t, whose first row is `row`: a search with the whole warp,
  // two dependent loads for a thousand graphs
  __device__ __forceinline__ int64_t graph_of_tile(int64_t graphs, int64_t t, int64_t row) const {
    if (!ptr) return t / ((per + 127) >> 7);
    int64_t lo = 0, hi = graphs;
    while (hi - lo > 1) {
      const int64_t step = (hi - lo + 31) >> 5, at = lo + (threadIdx.x & 31) * step;
      const int under = __popc(__ballot_sync(kFull, at < hi && ptr[at] <= row));
      lo += (under - 1) * step;  // the first probe always is
      hi = min(hi, lo + step);
    }
    return lo;
  }
  // the graph of row i (skips empty graphs)
  __device__ __forceinline__ int64_t graph_of(int64_t graphs, int64_t i) const {
    if (!ptr) return i / per;
    int64_t lo = 0, hi = graphs;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (ptr[mid] <= i) lo = mid;
      else hi = mid;
    }
    return lo;
  }
};

struct AttnArgs {
  int64_t graphs, num_q, num_k;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // element strides
  const void *q, *k, *v;
  AttnSegs qs, ks;                      // rows of each graph
  int64_t n_q_tiles, n_k_tiles;
  const float *q_pos, *k_pos, *sigma;   // [num][pos_dim], [heads]
  const uint8_t *q_mask, *k_mask;
  int heads, kv_heads, dim, pos_dim;
  float scale, cap;
  // forward results
  void *out;        // [num_q][heads][dim]
  float *out32;     // the same unrounded, or null
  float *neg_m, *rl;  // [heads][num_q]: -m and 1 / l, or null
  // backward
  const void *dout;         // [num_q][heads][dim]
  float *neg_d;             // [heads][num_q]: -D
  float *do_top;            // [heads][num_q]: largest finite |do|; null where nothing is scaled
  void *dq, *dk, *dv;       // contiguous
  float4 *pos_q, *pos_k;    // [heads][num_q], [kv_heads][num_k]; or null
  int *status;

  __device__ __forceinline__ float2 stats(int h, int64_t i) const {
    return make_float2(-neg_m[h * num_q + i], rl[h * num_q + i]);
  }
  __device__ __forceinline__ void put_stats(int h, int64_t i, float m, float r) const {
    neg_m[h * num_q + i] = -m;
    rl[h * num_q + i] = r;
  }
};

__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

struct AttnPos {
  float x, y, z;
};
__device__ __forceinline__ AttnPos pos_of(const float *p, int dim, int64_t i) {
  AttnPos r{0.f, 0.f, 0.f};
  if (p == nullptr) return r;
  p += i * dim;
  r.x = p[0];
  if (dim > 1) r.y = p[1];
  if (dim > 2) r.z = p[2];
  return r;
}

// (p_i - p_j) and its square; the score t of raw product `dot` in base 2 and
// the cap's slope
struct AttnScore {
  float su;     // a log2 e, or a / c where capped
  float capl;   // c log2 e, or 0
  float w;      // log2 e / (2 sigma^2)
  __device__ __forceinline__ void init(const AttnArgs &A, int h) {
    su = A.cap > 0.f ? A.scale / A.cap : A.scale * kAttnLog2e;
    capl = A.cap > 0.f ? A.cap * kAttnLog2e : 0.f;
    w = 0.f;
    if (A.pos_dim > 0) {
      const float s = A.sigma[h];
      w = kAttnLog2e / (2.f * s * s);
    }
  }
  __device__ __forceinline__ float operator()(float dot, float r2, float &slope) const {
    float t = dot * su;
    slope = 1.f;
    if (capl > 0.f) {
      const float th = tanh_step(t);
      slope = 1.f - th * th;
      t = th * capl;
    }
    return fmaf(-w, r2, t);
  }
};

// D_i = do_i . o_i, one warp a row and head
template <class T>
__global__ void __launch_bounds__(256) attn_delta_kernel(const T *dout, const float *out32,
                                                         int64_t num_q, int heads, int dim,
                                                         float *neg_d) {
  const int lane = threadIdx.x & 31;
  const int64_t n = num_q * heads;
  for (int64_t r = blockIdx.x * 8LL + (threadIdx.x >> 5); r < n; r += gridDim.x * 8LL) {
    float s = 0.f;
    for (int d = lane; d < dim; d += 32) s = fmaf(to_f(dout[r * dim + d]), out32[r * dim + d], s);
    s = warp_sum(s);
    if (lane == 0) neg_d[(r % heads) * num_q + r / heads] = -s;
  }
}

// Gradients of positions and sigmas from the rows' partials.  blockIdx.y = 0, 1:
// queries' and keys' positions, the heads in order; 2: dsigma_h = sum_i w_i /
// sigma^3 in fp64, one CTA a head, in a fixed order.
struct AttnPosGrads {
  const float4 *part[2];  // [heads][num]
  int64_t num[2];
  int heads[2];
  int pos_dim;
  float *grad[2], *dsigma;  // or null
  const float *sigma;
};
__global__ void __launch_bounds__(512) attn_pos_kernel(const AttnPosGrads P) {
  __shared__ double sh[16];
  const int y = blockIdx.y;
  if (y < 2) {
    if (P.grad[y] == nullptr) return;
    const int64_t num = P.num[y];
    for (int64_t i = blockIdx.x * 512LL + threadIdx.x; i < num; i += gridDim.x * 512LL) {
      float x = 0.f, yy = 0.f, z = 0.f;
      for (int h = 0; h < P.heads[y]; ++h) {
        const float4 v = P.part[y][h * num + i];
        x += v.x;
        yy += v.y;
        z += v.z;
      }
      float *g = P.grad[y] + i * P.pos_dim;
      g[0] = x;
      if (P.pos_dim > 1) g[1] = yy;
      if (P.pos_dim > 2) g[2] = z;
    }
  } else if (P.dsigma != nullptr) {
    for (int h = blockIdx.x; h < P.heads[0]; h += gridDim.x) {
      const float4 *p = P.part[0] + h * P.num[0];
      double s = 0.0;
      for (int64_t i = threadIdx.x; i < P.num[0]; i += 512) s += (double)p[i].w;
      s = block_sum(s, sh);
      if (threadIdx.x == 0) {
        const double sg = (double)P.sigma[h];
        P.dsigma[h] = (float)(s / (sg * sg * sg));
      }
      __syncthreads();
    }
  }
}

// ---- one warp a row ---------------------------------------------------------
// For any width and strides, not for speed: every lane reads another row of the
// other side, an element at a time (64 graphs of 64-512 points, 4 heads of 100, bf16:
// 5.2 ms forward, 26 ms forward and backward).

template <class T>
__global__ void __launch_bounds__(32 * kAttnWarps) attn_row_fwd_kernel(const AttnArgs A) {
  __shared__ float rows[kAttnWarps][kAttnMaxDim];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int64_t item = blockIdx.x * (int64_t)kAttnWarps + wp;
  if (item >= A.num_q * A.heads) return;
  const int64_t i = item / A.heads;
  const int h = (int)(item % A.heads), hk = h / (A.heads / A.kv_heads), D = A.dim;
  const int64_t g = A.qs.graph_of(A.graphs, i);
  const int64_t j0 = A.ks.begin(g), j1 = A.ks.end(g);
  const bool live = A.q_mask == nullptr || A.q_mask[i] != 0;
  const T *q = (const T *)A.q + i * A.q_row + h * A.q_head;
  const T *k = (const T *)A.k + hk * A.k_head, *v = (const T *)A.v + hk * A.v_head;
  float *qv = rows[wp];
  for (int d = lane; d < D; d += 32) qv[d] = to_f(q[d]);
  __syncwarp();
  AttnScore sc;
  sc.init(A, h);
  const AttnPos pi = pos_of(A.q_pos, A.pos_dim, i);
  float acc[kAttnMaxDim / 32] = {};
  float m = -INFINITY, l = 0.f;
  for (int64_t jb = j0; live && jb < j1; jb += 32) {
    const int64_t j = jb + lane;
    const bool on = j < j1 && (A.k_mask == nullptr || A.k_mask[j] != 0);
    float t = -INFINITY;
    if (on) {
      float dot = 0.f, slope;
      for (int d = 0; d < D; ++d) dot = fmaf(qv[d], to_f(k[j * A.k_row + d]), dot);
      const AttnPos pj = pos_of(A.k_pos, A.pos_dim, j);
      const float dx = pi.x - pj.x, dy = pi.y - pj.y, dz = pi.z - pj.z;
      t = sc(dot, dx * dx + dy * dy + dz * dz, slope);
    }
    const unsigned keys = __ballot_sync(kFull, on);
    if (keys == 0) continue;
    float mx = t;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
    const float mn = fmaxf(m, mx);
    // all scores so far -inf (or NaN): nothing to subtract
    const float ref = mn > -INFINITY ? mn : 0.f;
    const float p = on ? ex2(t - ref) : 0.f, keep = m > -INFINITY ? ex2(m - ref) : 0.f;
    l = l * keep + warp_sum(p);
    m = mn;
#pragma unroll
    for (int c = 0; c < kAttnMaxDim / 32; ++c) acc[c] *= keep;
    for (unsigned left = keys; left; left &= left - 1) {
      const int s = __ffs(left) - 1;
      const float pj = __shfl_sync(kFull, p, s);
#pragma unroll
      for (int c = 0; c < kAttnMaxDim / 32; ++c)
        if (lane + 32 * c < D) acc[c] = fmaf(pj, to_f(v[(jb + s) * A.v_row + lane + 32 * c]), acc[c]);
    }
  }
  // l = 0: no key (NaN scores give l = NaN)
  const bool any = l > 0.f || l != l;
  const float r = any ? 1.f / l : 0.f;
  T *out = (T *)A.out + item * D;
#pragma unroll
  for (int c = 0; c < kAttnMaxDim / 32; ++c)
    if (lane + 32 * c < D) {
      const float o = any ? acc[c] * r : 0.f;
      put(out + lane + 32 * c, o);
      if (A.out32) A.out32[item * D + lane + 32 * c] = o;
    }
  if (lane == 0 && A.neg_m) A.put_stats(h, i, any ? m : INFINITY, r);
}

template <class T>
__global__ void __launch_bounds__(32 * kAttnWarps) attn_row_dq_kernel(const AttnArgs A) {
  __shared__ float rows[kAttnWarps][2][kAttnMaxDim];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int64_t item = blockIdx.x * (int64_t)kAttnWarps + wp;
  if (item >= A.num_q * A.heads) return;
  const int64_t i = item / A.heads;
  const int h = (int)(item % A.heads), hk = h / (A.heads / A.kv_heads), D = A.dim;
  const int64_t g = A.qs.graph_of(A.graphs, i);
  const int64_t j0 = A.ks.begin(g), j1 = A.ks.end(g);
  const T *q = (const T *)A.q + i * A.q_row + h * A.q_head;
  const T *go = (const T *)A.dout + item * D;
  const T *k = (const T *)A.k + hk * A.k_head, *v = (const T *)A.v + hk * A.v_head;
  float *qv = rows[wp][0], *gv = rows[wp][1];
  for (int d = lane; d < D; d += 32) {
    qv[d] = to_f(q[d]);
    gv[d] = to_f(go[d]);
  }
  __syncwarp();
  AttnScore sc;
  sc.init(A, h);
  const AttnPos pi = pos_of(A.q_pos, A.pos_dim, i);
  const float2 st = A.stats(h, i);
  const float delta = -A.neg_d[h * A.num_q + i];
  const bool live = st.y != 0.f;  // no key, or masked
  float acc[kAttnMaxDim / 32] = {};
  float gx = 0.f, gy = 0.f, gz = 0.f, gs = 0.f;
  for (int64_t jb = j0; live && jb < j1; jb += 32) {
    const int64_t j = jb + lane;
    const bool on = j < j1 && (A.k_mask == nullptr || A.k_mask[j] != 0);
    float du = 0.f;
    if (on) {
      float dot = 0.f, dp = 0.f, slope;
      for (int d = 0; d < D; ++d) {
        dot = fmaf(qv[d], to_f(k[j * A.k_row + d]), dot);
        dp = fmaf(gv[d], to_f(v[j * A.v_row + d]), dp);
      }
      const AttnPos pj = pos_of(A.k_pos, A.pos_dim, j);
      const float dx = pi.x - pj.x, dy = pi.y - pj.y, dz = pi.z - pj.z;
      const float r2 = dx * dx + dy * dy + dz * dz;
      const float t = sc(dot, r2, slope);
      const float ds = ex2(t - st.x) * st.y * (dp - delta);
      gx = fmaf(ds, dx, gx);
      gy = fmaf(ds, dy, gy);
      gz = fmaf(ds, dz, gz);
      gs = fmaf(ds, r2, gs);
      du = ds * slope;
    }
    for (unsigned left = __ballot_sync(kFull, on); left; left &= left - 1) {
      const int s = __ffs(left) - 1;
      const float dj = __shfl_sync(kFull, du, s);
#pragma unroll
      for (int c = 0; c < kAttnMaxDim / 32; ++c)
        if (lane + 32 * c < D) acc[c] = fmaf(dj, to_f(k[(jb + s) * A.k_row + lane + 32 * c]), acc[c]);
    }
  }
  if (A.dq) {
    T *dq = (T *)A.dq + item * D;
#pragma unroll
    for (int c = 0; c < kAttnMaxDim / 32; ++c)
      if (lane + 32 * c < D) put(dq + lane + 32 * c, acc[c] * A.scale);
  }
  if (A.pos_q) {
    const float s = A.sigma[h], w = 1.f / (s * s);
    gx = warp_sum(gx), gy = warp_sum(gy), gz = warp_sum(gz), gs = warp_sum(gs);
    if (lane == 0) A.pos_q[h * A.num_q + i] = make_float4(-w * gx, -w * gy, -w * gz, gs);
  }
}

template <class T>
__global__ void __launch_bounds__(32 * kAttnWarps) attn_row_dkv_kernel(const AttnArgs A) {
  __shared__ float rows[kAttnWarps][2][kAttnMaxDim];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int64_t item = blockIdx.x * (int64_t)kAttnWarps + wp;
  if (item >= A.num_k * A.kv_heads) return;
  const int64_t j = item / A.kv_heads;
  const int hk = (int)(item % A.kv_heads), group = A.heads / A.kv_heads, D = A.dim;
  const int64_t g = A.ks.graph_of(A.graphs, j);
  const int64_t i0 = A.qs.begin(g), i1 = A.qs.end(g);
  const bool live = A.k_mask == nullptr || A.k_mask[j] != 0;
  float *kv = rows[wp][0], *vv = rows[wp][1];
  for (int d = lane; d < D; d += 32) {
    kv[d] = to_f(((const T *)A.k)[j * A.k_row + hk * A.k_head + d]);
    vv[d] = to_f(((const T *)A.v)[j * A.v_row + hk * A.v_head + d]);
  }
  __syncwarp();
  const AttnPos pj = pos_of(A.k_pos, A.pos_dim, j);
  float dk[kAttnMaxDim / 32] = {}, dv[kAttnMaxDim / 32] = {};
  float px = 0.f, py = 0.f, pz = 0.f;
  for (int h = hk * group; live && h < (hk + 1) * group; ++h) {
    AttnScore sc;
    sc.init(A, h);
    const T *q = (const T *)A.q + h * A.q_head;
    const T *go = (const T *)A.dout + h * D;
    float gx = 0.f, gy = 0.f, gz = 0.f;
    for (int64_t ib = i0; ib < i1; ib += 32) {
      const int64_t i = ib + lane;
      float p = 0.f, du = 0.f;
      bool on = i < i1;
      if (on) {
        const float2 st = A.stats(h, i);
        on = st.y != 0.f;
        if (on) {
          float dot = 0.f, dp = 0.f, slope;
          for (int d = 0; d < D; ++d) {
            dot = fmaf(to_f(q[i * A.q_row + d]), kv[d], dot);
            dp = fmaf(to_f(go[i * A.heads * D + d]), vv[d], dp);
          }
          const AttnPos pi = pos_of(A.q_pos, A.pos_dim, i);
          const float dx = pi.x - pj.x, dy = pi.y - pj.y, dz = pi.z - pj.z;
          const float t = sc(dot, dx * dx + dy * dy + dz * dz, slope);
          p = ex2(t - st.x) * st.y;
          const float ds = p * (dp + A.neg_d[h * A.num_q + i]);
          gx = fmaf(ds, dx, gx);
          gy = fmaf(ds, dy, gy);
          gz = fmaf(ds, dz, gz);
          du = ds * slope;
        }
      }
      for (unsigned left = __ballot_sync(kFull, on); left; left &= left - 1) {
        const int s = __ffs(left) - 1;
        const float pi_ = __shfl_sync(kFull, p, s), di = __shfl_sync(kFull, du, s);
        const T *qr = q + (ib + s) * A.q_row, *gr = go + (ib + s) * A.heads * D;
#pragma unroll
        for (int c = 0; c < kAttnMaxDim / 32; ++c)
          if (lane + 32 * c < D) {
            dk[c] = fmaf(di, to_f(qr[lane + 32 * c]), dk[c]);
            dv[c] = fmaf(pi_, to_f(gr[lane + 32 * c]), dv[c]);
          }
      }
    }
    if (A.pos_k) {
      const float s = A.sigma[h], w = 1.f / (s * s);
      px = fmaf(w, warp_sum(gx), px);
      py = fmaf(w, warp_sum(gy), py);
      pz = fmaf(w, warp_sum(gz), pz);
    }
  }
#pragma unroll
  for (int c = 0; c < kAttnMaxDim / 32; ++c)
    if (lane + 32 * c < D) {
      if (A.dk) put((T *)A.dk + item * D + lane + 32 * c, dk[c] * A.scale);
      if (A.dv) put((T *)A.dv + item * D + lane + 32 * c, dv[c]);
    }
  if (A.pos_k && lane == 0) A.pos_k[hk * A.num_k + j] = make_float4(px, py, pz, 0.f);
}

}  // namespace ra
