// ra_few.cuh -- parts of the kernels for a few rows (ra_attn_few.cuh,
// ra_ce_few.cuh): loads of eight columns, sums over lanes by halving, and the
// warp-wide products of 16-bit inputs.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "ra_common.cuh"
#include "ra_tcprim.cuh"

namespace ra {

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <class T>
struct Few8 {  // eight columns of a row, as loaded
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p, bool on) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k)
      u[k] = on ? __ldg(reinterpret_cast<const uint4 *>(p) + k) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(f2_t (&f)[4]) const {
    T t[8];
    memcpy(t, u, sizeof(t));
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = pk(to_f(t[2 * k]), to_f(t[2 * k + 1]));
  }
};

// Sums v[0 .. NV) over LPK lanes; lane c is left with v[0 .. max(1, NV / LPK)),
// the values c NV / LPK ...
template <int NV, int LPK, int S = LPK / 2, int CNT = NV>
__device__ __forceinline__ void few_halve(float (&v)[NV], int c) {
  if constexpr (S >= 1) {
    if constexpr (CNT > 1) {
      const bool up = c & S;
#pragma unroll
      for (int k = 0; k < CNT / 2; ++k) {
        const float mine = up ? v[CNT / 2 + k] : v[k], send = up ? v[k] : v[CNT / 2 + k];
        v[k] = mine + __shfl_xor_sync(kFull, send, S);
      }
      few_halve<NV, LPK, S / 2, CNT / 2>(v, c);
    } else {
      v[0] += __shfl_xor_sync(kFull, v[0], S);
      few_halve<NV, LPK, S / 2, 1>(v, c);
    }
  }
}

// 16 bytes global to shared, or zeros
__device__ __forceinline__ void few_copy(uint32_t dst, const void *src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}

// d += a b, 16 x 8 x 16: lane 4 g + t holds d of rows g and g + 8, columns 2 t, 2 t + 1
template <class T>
__device__ __forceinline__ void few_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// four 8 x 8 matrices; lane 8 m + r gives the address of row r of matrix m
template <bool TRANS>
__device__ __forceinline__ void few_ldm(uint32_t (&v)[4], uint32_t at) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(at)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(at)
                 : "memory");
}
// byte of 16-byte piece c of row r: eight rows' pieces in eight bank groups
template <int DP>
__device__ __forceinline__ int few_at(int r, int c) {
  return r * DP * 2 + (c ^ (DP >= 64 ? r & 7 : (r >> 1) & 3)) * 16;
}

}  // namespace ra
