// fp16 / bf16 values of the kernels that serve both types: 16-byte loads and stores of eight numbers as fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace bsb {

__device__ __forceinline__ float2 to_f2(__half2 h) { return __half22float2(h); }
__device__ __forceinline__ float2 to_f2(__nv_bfloat162 h) { return __bfloat1622float2(h); }
__device__ __forceinline__ float to_f(__half h) { return __half2float(h); }
__device__ __forceinline__ float to_f(__nv_bfloat16 h) { return __bfloat162float(h); }
__device__ __forceinline__ float to_f(float h) { return h; }
template <typename T> struct Pair;
template <> struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ __half2 make(float a, float b) { return __floats2half2_rn(a, b); }
};
template <> struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ __nv_bfloat162 make(float a, float b) { return __floats2bfloat162_rn(a, b); }
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& raw, float (&out)[8]) {
  const typename Pair<T>::type* p = reinterpret_cast<const typename Pair<T>::type*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = to_f2(p[i]);
    out[2 * i] = f.x;
    out[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&in)[8]) {
  uint4 raw;
  typename Pair<T>::type* p = reinterpret_cast<typename Pair<T>::type*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = Pair<T>::make(in[2 * i], in[2 * i + 1]);
  return raw;
}
template <typename T>
__device__ __forceinline__ void load8(const T* src, float (&out)[8]) {
  unpack8<T>(*reinterpret_cast<const uint4*>(src), out);
}
template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&in)[8]) {
  *reinterpret_cast<uint4*>(dst) = pack8<T>(in);
}

}  // namespace bsb
