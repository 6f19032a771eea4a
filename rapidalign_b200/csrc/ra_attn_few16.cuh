// ra_attn_few16.cuh -- forward of kernel attention for at most eight rows a graph
// and key head (queries x heads of the key head), 16-bit inputs.
//
// Bound by the bytes of the keys and values, each read once.  A CTA takes one
// graph, key head and range of keys; its warps take steps of KT keys in turn and
// share nothing until the end.  A warp copies its steps into a ring in shared
// memory (16 bytes a lane, masked keys as zeros) and works on them with the
// warp-wide 16 x 8 x 16 products: the rows are the upper eight of the 16,
//   S = Q K^T (keys as columns; accumulators lie as the next product wants P),
//   O += P V, with P's rounding error as the lower eight rows: P to 2^-17 (bf16)
//   for nothing.
// (The eight rows would be 1/16 of a tcgen05 tile, and P would travel through
// TMEM; in the FMA form of ra_attn_few.cuh, 745 instructions for 16 keys of 64
// and four rows, the issue slots were as busy as the memory.)  A step's sum is
// rounded by the tensor core, the steps are added in fp32.
// The warps, then the key ranges (attn_join_kernel) are joined in a fixed order.
// Measured: one query of 8 heads on 2 key heads of 64 against 262144 keys (137 MB
// with positions) 26 us, 5.3 TB/s, and 6.5 us joining (FMA form: 38 and 9);
// 1024 graphs of 64-512 keys 39 us, 4.0 TB/s (63).
#pragma once

#include "ra_attn_few.cuh"

namespace ra {

template <int DP>
struct Few16Cfg {
  static constexpr int KT = DP == 128 ? 16 : 32;  // keys a step
  static constexpr int TILE = KT * DP * 2;        // bytes of K, or V
  static constexpr int STAGES = 16384 / (2 * TILE);
  static constexpr int ring = kFewWarps * 16384;  // at the end: [warp][8][DP] floats
  static constexpr int pos = ring;                // float [warp][3][KT]
  static constexpr int ml = pos + kFewWarps * 3 * KT * 4;  // float2 [warp][8]
  static constexpr int smem = ml + kFewWarps * 8 * 8;
};
constexpr int kFew16Ctas = 3;

template <class T>
__device__ __forceinline__ uint32_t few_pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t few_pack<__half>(float a, float b) {
  return bits_as<uint32_t>(__floats2half2_rn(a, b));
}
template <>
__device__ __forceinline__ uint32_t few_pack<__nv_bfloat16>(float a, float b) {
  return bits_as<uint32_t>(__floats2bfloat162_rn(a, b));
}
template <class T>
__device__ __forceinline__ float2 few_unpack(uint32_t u);
template <>
__device__ __forceinline__ float2 few_unpack<__half>(uint32_t u) {
  return __half22float2(bits_as<__half2>(u));
}
template <>
__device__ __forceinline__ float2 few_unpack<__nv_bfloat16>(uint32_t u) {
  return __bfloat1622float2(bits_as<__nv_bfloat162>(u));
}
template <class T, int DP>
__global__ void __launch_bounds__(32 * kFewWarps, kFew16Ctas)
    attn_few16_kernel(const AttnArgs A, int splits, float *part_o, float2 *part_s) {
  using C = Few16Cfg<DP>;
  constexpr int KT = C::KT, S = C::STAGES, NT = KT / 8, CH = DP / 8, RP = 32 / CH;
  // P of fp16 is held 2^10 up, so that its rounding error has bits left
  constexpr float kUp = std::is_same<T, __half>::value ? 10.f : 0.f;
  extern __shared__ uint4 few_ring[];
  uint8_t *sm = reinterpret_cast<uint8_t *>(few_ring);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = lane >> 2, t2 = 2 * (lane & 3);
  const uint32_t ring = smem_u32(sm) + warp * 16384;
  float *kpos = reinterpret_cast<float *>(sm + C::pos) + warp * 3 * KT;
  float2 *sml = reinterpret_cast<float2 *>(sm + C::ml);
  // the key heads of a range side by side: their rows are
  const int hk = (int)(blockIdx.x % A.kv_heads), group = A.heads / A.kv_heads;
  const int split = (int)(blockIdx.x / A.kv_heads % splits);
  const int64_t g = blockIdx.x / A.kv_heads / splits;
  const int64_t i0 = A.qs.begin(g), j0 = A.ks.begin(g), nk = A.ks.end(g) - j0;
  const int n = (int)min((int64_t)8, (A.qs.end(g) - i0) * group);
  const int64_t k0 = nk * split / splits, k1 = nk * (split + 1) / splits;
  const bool pos = A.pos_dim > 0, capped = A.cap > 0.f;
  const float su = capped ? A.scale / A.cap : A.scale * kAttnLog2e, capl = A.cap * kAttnLog2e;

  // this lane's row
  const int64_t i = i0 + row / group;
  const int h = hk * group + row % group;
  const bool live = row < n && (A.q_mask == nullptr || A.q_mask[i] != 0);
  AttnPos pi{0.f, 0.f, 0.f};
  float w = 0.f;
  if (pos && live) {
    pi = pos_of(A.q_pos, A.pos_dim, i);
    const float s = A.sigma[h];
    w = kAttnLog2e / (2.f * s * s);
  }
  uint32_t q[DP / 16][2];
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = 16 * k + 8 * e + t2;
      q[k][e] = live && col < A.dim ? *reinterpret_cast<const uint32_t *>(
                                          (const T *)A.q + i * A.q_row + h * A.q_head + col)
                                    : 0u;
    }

  // Step t of the warp: KT keys from (t kFewWarps + warp) KT of the range.
  constexpr int kStep = kFewWarps * KT;
  const int64_t start = j0 + k0 + warp * KT;
  const int cc = lane % CH, cr = lane / CH;  // the piece and first row it copies
  const T *kp = (const T *)A.k + hk * A.k_head + cc * 8 + (start + cr) * A.k_row;
  const T *vp = (const T *)A.v + hk * A.v_head + cc * 8 + (start + cr) * A.v_row;
  const uint8_t *mp = A.k_mask ? A.k_mask + start + lane : nullptr;
  const int64_t mine = k1 - k0 - warp * KT;
  const int64_t steps = mine > 0 ? (mine + kStep - 1) / kStep : 0;
  int64_t left = mine - lane;  // keys from this lane's of the next copied step on
  unsigned marks[S];           // which keys of a slot's step are there
  bool next = false;
  auto look = [&]() { next = lane < KT && left > 0 && (mp == nullptr || *mp != 0); };
  auto issue = [&](int64_t t, int slot, unsigned &bits) {
    if (t < steps) {
      bits = __ballot_sync(kFull, next);
      const uint32_t at = ring + slot * 2 * C::TILE;
#pragma unroll
      for (int p = 0; p < KT / RP; ++p) {
        const int r = cr + p * RP;
        const bool on = ((bits >> r) & 1) && cc * 8 < A.dim;
        few_copy(at + few_at<DP>(r, cc), on ? kp + p * RP * A.k_row : (const T *)A.k, on);
        few_copy(at + C::TILE + few_at<DP>(r, cc), on ? vp + p * RP * A.v_row : (const T *)A.v, on);
      }
      kp += kStep * A.k_row;
      vp += kStep * A.v_row;
      if (mp) mp += kStep;
      left -= kStep;
      look();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  AttnPos np{0.f, 0.f, 0.f};
  auto place = [&](int64_t t, unsigned bits) {  // the position of this lane's key of step t
    np = pos && ((bits >> lane) & 1) ? pos_of(A.k_pos, A.pos_dim, start + t * kStep + lane)
                                     : AttnPos{0.f, 0.f, 0.f};
  };

  float mm = -INFINITY, ml = 0.f;  // of the row, and this lane's part of its sum
  float o[DP / 8][2] = {};
  look();
#pragma unroll
  for (int t = 0; t < S; ++t) marks[t] = 0;
#pragma unroll
  for (int t = 0; t < S - 1; ++t) issue(t, t, marks[t]);
  place(0, marks[0]);
  for (int64_t base = 0; base < steps; base += S) {
#pragma unroll
    for (int slot = 0; slot < S; ++slot) {
      const int64_t step = base + slot;
      if (step >= steps) break;
      __syncwarp();  // the last step's tiles and positions have been read
      if (pos && lane < KT) {
        kpos[lane] = np.x;
        kpos[KT + lane] = np.y;
        kpos[2 * KT + lane] = np.z;
      }
      issue(step + S - 1, (slot + S - 1) % S, marks[(slot + S - 1) % S]);
      if (step + 1 < steps) place(step + 1, marks[(slot + 1) % S]);
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
      __syncwarp();
      const unsigned bits = marks[slot];
      const uint32_t sk = ring + slot * 2 * C::TILE, sv = sk + C::TILE;
      const int lr = lane & 7, lm = lane >> 3;
      float s[NT][4] = {};
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
          uint32_t b[4];
          const uint32_t a[4] = {q[k][0], 0u, q[k][1], 0u};
          few_ldm<false>(b, sk + few_at<DP>(8 * (j + (lm >> 1)) + lr, 2 * k + (lm & 1)));
          few_mma<T>(s[j], a, b[0], b[1]);
          few_mma<T>(s[j + 1], a, b[2], b[3]);
        }
      float mx = mm;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float x[2] = {s[j][0] * su, s[j][1] * su};
        if (capped) {
          const f2_t th = tanh2(pk(x[0], x[1]));
          x[0] = capl * lo_of(th);
          x[1] = capl * hi_of(th);
        }
        if (pos) {
          const float2 px = *reinterpret_cast<const float2 *>(kpos + 8 * j + t2);
          const float2 py = *reinterpret_cast<const float2 *>(kpos + KT + 8 * j + t2);
          const float2 pz = *reinterpret_cast<const float2 *>(kpos + 2 * KT + 8 * j + t2);
          const float x0 = pi.x - px.x, y0 = pi.y - py.x, z0 = pi.z - pz.x;
          const float x1 = pi.x - px.y, y1 = pi.y - py.y, z1 = pi.z - pz.y;
          x[0] = fmaf(-w, fmaf(z0, z0, fmaf(y0, y0, x0 * x0)), x[0]);
          x[1] = fmaf(-w, fmaf(z1, z1, fmaf(y1, y1, x1 * x1)), x[1]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[j][e] = (bits >> (8 * j + t2 + e)) & 1 ? x[e] : -INFINITY;
          mx = fmaxf(mx, s[j][e]);
        }
      }
      mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 2));
      const float ref = mx > -INFINITY ? mx - kUp : 0.f;
      const float keep = mm > -INFINITY ? ex2(mm - mx) : 0.f;
      mm = mx;
      ml *= keep;
      uint32_t hi[NT], lo[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float a = ex2(s[j][0] - ref), b = ex2(s[j][1] - ref);
        ml += a + b;
        hi[j] = few_pack<T>(a, b);
        const float2 r = few_unpack<T>(hi[j]);
        lo[j] = few_pack<T>(a - r.x, b - r.y);
      }
#pragma unroll
      for (int d = 0; d < DP / 8; d += 2) {
        float c[2][4] = {};
#pragma unroll
        for (int k = 0; k < KT / 16; ++k) {
          uint32_t v[4];
          const uint32_t a[4] = {hi[2 * k], lo[2 * k], hi[2 * k + 1], lo[2 * k + 1]};
          few_ldm<true>(v, sv + few_at<DP>(16 * k + 8 * (lm & 1) + lr, d + (lm >> 1)));
          few_mma<T>(c[0], a, v[0], v[1]);
          few_mma<T>(c[1], a, v[2], v[3]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          o[d + e][0] = fmaf(o[d + e][0], keep, c[e][0] + c[e][2]);
          o[d + e][1] = fmaf(o[d + e][1], keep, c[e][1] + c[e][3]);
        }
      }
    }
  }
  ml += __shfl_xor_sync(kFull, ml, 1);
  ml += __shfl_xor_sync(kFull, ml, 2);
  __syncwarp();
  float *acc = reinterpret_cast<float *>(sm);
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
    *reinterpret_cast<float2 *>(acc + warp * 4096 + row * DP + 8 * d + t2) =
        make_float2(o[d][0], o[d][1]);
  if ((lane & 3) == 0) sml[warp * 8 + row] = make_float2(mm > -INFINITY ? mm - kUp : mm, ml);
  __syncthreads();
  few_finish<T>(A, n, hk, i0, splits, split, acc, 4096, DP, sml, 8, part_o, part_s);
}

}  // namespace ra
