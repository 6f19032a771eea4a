// ra_attn_few.cuh -- forward of kernel attention for a few query rows a graph
// (one query a graph: pooling, scoring, single new tokens), fp32 inputs without
// a backward; and what it shares with the 16-bit form (ra_attn_few16.cuh).
//
// Bound by the bytes of the keys and values, each read once for all the
// query heads of a key head.  A CTA takes one graph, key head and range of keys;
// its N = queries x group rows stay in registers.  LPK lanes share a key, eight
// columns (two 16-byte pieces) each, so a warp reads 32 / LPK whole rows an
// instruction, copied steps ahead into a ring in shared memory where a lane reads
// only what it copied itself.  The N U dots of a step are joined over the LPK
// lanes by halving (each exchange leaves a lane half of its values), so that
// every lane finishes N U / LPK scores of one row and none is worked on twice;
// their weights go back by shuffles.  Every lane group keeps the maximum and sums
// of its own keys, joined at the end over the warp, the CTA (shared memory) and
// the key ranges (attn_join_kernel).
// Measured: one query of 8 heads on 2 key heads of 64 against 262144 keys (272 MB
// with positions) 84 us, 3.2 TB/s; 8 rows a key head 87 us.
#pragma once

#include "ra_attn.cuh"
#include "ra_few.cuh"

namespace ra {

constexpr int kFewRows = 8;    // most rows (queries of a graph x heads a key head)
constexpr int kFewWarps = 4;

constexpr int kFewKeys = 2;  // U: keys of a step a lane
// CTAs of an SM, and steps in flight: 12 KB a warp of four, 16 of two
constexpr int few_ctas(int64_t rows) { return rows > 4 ? 2 : 4; }
constexpr int kFewStage = 2 * kFewKeys * 1024;  // bytes of a warp's step
template <int N>
constexpr int few_stages = (N > 4 ? 16384 : 12288) / kFewStage;
template <int N>
constexpr int few_smem = kFewWarps * few_stages<N> * kFewStage;

// Joins the warps of a CTA: their sums acc and (maximum, sum) sml of n rows.
template <class T>
__device__ __forceinline__ void few_finish(const AttnArgs &A, int n, int hk, int64_t i0, int splits,
                                           int split, const float *acc, int acc_warp, int acc_row,
                                           const float2 *sml, int ml_warp, float *part_o,
                                           float2 *part_s) {
  const int D = A.dim, group = A.heads / A.kv_heads;
  for (int e = threadIdx.x; e < n * D; e += 32 * kFewWarps) {
    const int r = e / D, d = e % D;
    float mx = -INFINITY;
    for (int k = 0; k < kFewWarps; ++k) mx = fmaxf(mx, sml[k * ml_warp + r].x);
    float ls = 0.f, o = 0.f;
    for (int k = 0; k < kFewWarps; ++k) {
      const float2 s = sml[k * ml_warp + r];
      const float f = s.x > -INFINITY ? ex2(s.x - mx) : s.y != s.y ? 1.f : 0.f;
      ls = fmaf(s.y, f, ls);
      o = fmaf(acc[k * acc_warp + r * acc_row + d], f, o);
    }
    const int64_t i = i0 + r / group;
    const int h = hk * group + r % group;
    const bool on = A.q_mask == nullptr || A.q_mask[i] != 0;
    const bool any = on && (ls > 0.f || ls != ls);
    const float ref = mx > -INFINITY ? mx : 0.f;
    const int64_t at = (i * A.heads + h) * D + d;
    if (splits > 1) {
      part_o[split * A.num_q * A.heads * D + at] = any ? o : 0.f;
      if (d == 0)
        part_s[((int64_t)split * A.heads + h) * A.num_q + i] =
            make_float2(any ? ref : -INFINITY, any ? ls : 0.f);
    } else {
      const float rl = any ? 1.f / ls : 0.f;
      const float v = any ? o * rl : 0.f;
      put((T *)A.out + at, v);
      if (A.out32) A.out32[at] = v;
      if (d == 0 && A.neg_m) A.put_stats(h, i, any ? ref : INFINITY, rl);
    }
  }
}

template <int N, int LPK>
__global__ void __launch_bounds__(32 * kFewWarps, few_ctas(N))
    attn_few_kernel(const AttnArgs A, int splits, float *part_o, float2 *part_s) {
  using T = float;
  constexpr int KPW = 32 / LPK, U = kFewKeys, NV = N * U;
  constexpr int V = NV >= LPK ? NV / LPK : 1;  // scores a lane finishes, all of one row
  static_assert(V <= U, "a lane's scores are of one row");
  extern __shared__ uint4 few_ring[];
  __shared__ float sacc[kFewWarps][N][LPK * 8];
  __shared__ float2 sml[kFewWarps][N];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = lane % LPK, sub = lane / LPK, D = A.dim;
  // the key heads of a range side by side: their rows are
  const int hk = (int)(blockIdx.x % A.kv_heads), group = A.heads / A.kv_heads;
  const int split = (int)(blockIdx.x / A.kv_heads % splits);
  const int64_t g = blockIdx.x / A.kv_heads / splits;
  const int64_t i0 = A.qs.begin(g), j0 = A.ks.begin(g), nk = A.ks.end(g) - j0;
  const int n = (int)min((int64_t)N, (A.qs.end(g) - i0) * group);
  const int64_t k0 = nk * split / splits, k1 = nk * (split + 1) / splits;
  const bool cols = c * 8 < D, pos = A.pos_dim > 0, capped = A.cap > 0.f;
  const float su = capped ? A.scale / A.cap : A.scale * kAttnLog2e, capl = A.cap * kAttnLog2e;

  f2_t q[N][4];
#pragma unroll
  for (int r = 0; r < N; ++r) {
    const int64_t i = i0 + r / group;
    const int h = hk * group + r % group;
    const bool live = r < n && (A.q_mask == nullptr || A.q_mask[i] != 0);
    Few8<T> x;
    x.load((const T *)A.q + (live ? i * A.q_row + h * A.q_head + c * 8 : 0), live && cols);
    x.get(q[r]);
#pragma unroll
    for (int k = 0; k < 4; ++k) q[r][k] = mul2(q[r][k], pk(su, su));
  }
  // the scores this lane finishes: row mr, keys u0 .. u0 + V - 1
  const int first = c * NV / LPK, mr = first / U, u0 = first % U;
  AttnPos pi{0.f, 0.f, 0.f};
  float w = 0.f;
  if (pos && mr < n) {
    const int64_t i = i0 + mr / group;
    if (A.q_mask == nullptr || A.q_mask[i] != 0) {
      pi = pos_of(A.q_pos, A.pos_dim, i);
      const float s = A.sigma[hk * group + mr % group];
      w = kAttnLog2e / (2.f * s * s);
    }
  }
  float mm = -INFINITY, ml = 0.f;  // of row mr, this lane group's keys; ml: this lane's part
  f2_t acc[N][4] = {};
  // This lane's keys of a step: rows u KPW apart from kp, vp.  A lane copies its
  // columns of S - 1 steps ahead into shared memory and reads only what it copied.
  constexpr int kStep = kFewWarps * KPW * U, S = few_stages<N>, W = sizeof(T) / 2;
  constexpr int kSlot = 2 * U * W * 32;  // 16-byte pieces of a warp's step
  const int64_t start = j0 + k0 + warp * (KPW * U) + sub;
  const T *kp = (const T *)A.k + hk * A.k_head + c * 8 + start * A.k_row;
  const T *vp = (const T *)A.v + hk * A.v_head + c * 8 + start * A.v_row;
  const float *pp = pos ? A.k_pos + (start + u0 * KPW) * A.pos_dim : nullptr;
  const uint8_t *mp = A.k_mask ? A.k_mask + start : nullptr;
  int left = (int)(k1 - k0) - warp * (KPW * U) - sub;  // keys from the next copied on
  const int steps = (int)((k1 - k0) - warp * (KPW * U) + kStep - 1) / kStep;  // the warp's
  uint4 *ring = few_ring + warp * S * kSlot + lane;
  unsigned marks = 0;  // U bits a slot
  unsigned next = 0;   // of the step to be copied next
  auto look = [&]() {
    next = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      next |= (unsigned)(u * KPW < left && (mp == nullptr || mp[u * KPW] != 0)) << u;
  };
  auto issue = [&](int t) {
    if (t < steps) {
      const int slot = t % S;
      const uint32_t at = smem_u32(ring + slot * kSlot);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool on = ((next >> u) & 1) && cols;
        const T *ku = on ? kp + u * KPW * A.k_row : (const T *)A.k;
        const T *vu = on ? vp + u * KPW * A.v_row : (const T *)A.v;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          few_copy(at + (u * W + w) * 512, ku + w * (16 / sizeof(T)), on);
          few_copy(at + ((U + u) * W + w) * 512, vu + w * (16 / sizeof(T)), on);
        }
      }
      marks = (marks & ~(((1u << U) - 1) << (slot * U))) | next << (slot * U);
      kp += kStep * A.k_row;
      vp += kStep * A.v_row;
      if (mp) mp += kStep;
      left -= kStep;
      look();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  AttnPos pj[V];
  auto place = [&](int t) {  // positions of step t, that has been copied
    const unsigned on = marks >> (t % S * U);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      pj[e] = AttnPos{0.f, 0.f, 0.f};
      if (pos && ((on >> (u0 + e)) & 1)) pj[e] = pos_of(pp + e * KPW * A.pos_dim, A.pos_dim, 0);
    }
    if (pos) pp += kStep * A.pos_dim;
  };
  look();
#pragma unroll
  for (int t = 0; t < S - 1; ++t) issue(t);
  if (steps > 0) place(0);
  for (int step = 0; step < steps; ++step) {
    issue(step + S - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    const unsigned on = marks >> (step % S * U);
    const uint4 *at = ring + step % S * kSlot;
    float t[NV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      f2_t x[4];
      Few8<T> kx;
#pragma unroll
      for (int e = 0; e < W; ++e) kx.u[e] = at[(u * W + e) * 32];
      kx.get(x);
#pragma unroll
      for (int r = 0; r < N; ++r) {
        f2_t s = mul2(q[r][0], x[0]);
#pragma unroll
        for (int k = 1; k < 4; ++k) s = fma2(q[r][k], x[k], s);
        t[r * U + u] = lo_of(s) + hi_of(s);
      }
    }
    few_halve<NV, LPK>(t, c);
    float mx = mm;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float s = t[e];
      if (capped) s = capl * tanh_step(s);
      if (pos) {
        const float dx = pi.x - pj[e].x, dy = pi.y - pj[e].y, dz = pi.z - pj[e].z;
        s = fmaf(-w, fmaf(dz, dz, fmaf(dy, dy, dx * dx)), s);
      }
      t[e] = (on >> (u0 + e)) & 1 ? s : -INFINITY;
      mx = fmaxf(mx, t[e]);
    }
    if (step + 1 < steps) place(step + 1);
    // the row's other lanes: U keys (or, of duplicates, the same)
#pragma unroll
    for (int o = 1; o < LPK / N; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
    const float ref = mx > -INFINITY ? mx : 0.f;
    if (__any_sync(kFull, mx > mm)) {
      const float keep = mm > -INFINITY ? ex2(mm - ref) : 0.f;
      ml *= keep;
#pragma unroll
      for (int r = 0; r < N; ++r) {
        const float f = __shfl_sync(kFull, keep, sub * LPK + r * U * LPK / NV);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[r][k] = mul2(acc[r][k], pk(f, f));
      }
      mm = mx;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      t[e] = ex2(t[e] - ref);
      ml += t[e];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      f2_t x[4];
      Few8<T> vx;
#pragma unroll
      for (int e = 0; e < W; ++e) vx.u[e] = at[((U + u) * W + e) * 32];
      vx.get(x);
#pragma unroll
      for (int r = 0; r < N; ++r) {
        const int v = r * U + u;
        const float p = __shfl_sync(kFull, t[v % V], sub * LPK + v * LPK / NV);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[r][k] = fma2(pk(p, p), x[k], acc[r][k]);
      }
    }
  }
  // each row's maximum and sum to all lanes of the group
  constexpr int kDup = NV >= LPK ? 1 : LPK / NV;  // lanes that finish the same score
#pragma unroll
  for (int o = kDup; o < LPK / N; o <<= 1) ml += __shfl_xor_sync(kFull, ml, o);
  float m[N], l[N];
#pragma unroll
  for (int r = 0; r < N; ++r) {
    m[r] = __shfl_sync(kFull, mm, sub * LPK + r * U * LPK / NV);
    l[r] = __shfl_sync(kFull, ml, sub * LPK + r * U * LPK / NV);
  }
  // the lane groups of the warp, then the warps, in a fixed order
#pragma unroll
  for (int r = 0; r < N; ++r) {
    float mx = m[r];
#pragma unroll
    for (int o = 16; o >= LPK; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
    const float f = m[r] > -INFINITY ? ex2(m[r] - mx) : l[r] != l[r] ? 1.f : 0.f;
    l[r] *= f;
#pragma unroll
    for (int o = 16; o >= LPK; o >>= 1) l[r] += __shfl_xor_sync(kFull, l[r], o);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float a = (k & 1 ? hi_of(acc[r][k / 2]) : lo_of(acc[r][k / 2])) * f;
#pragma unroll
      for (int o = 16; o >= LPK; o >>= 1) a += __shfl_xor_sync(kFull, a, o);
      if (sub == 0) sacc[warp][r][c * 8 + k] = a;
    }
    if (lane == 0) sml[warp][r] = make_float2(mx, l[r]);
  }
  __syncthreads();
  few_finish<T>(A, n, hk, i0, splits, split, &sacc[0][0][0], N * LPK * 8, LPK * 8, &sml[0][0], N,
                part_o, part_s);
}

}  // namespace ra
