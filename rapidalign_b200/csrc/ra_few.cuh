// ra_few.cuh -- parts of the kernels for a few rows (ra_attn_few.cuh,
// ra_ce_few.cuh): loads of eight columns, and sums over lanes by halving.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ra_common.cuh"

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

}  // namespace ra
