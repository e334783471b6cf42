// Device helpers shared by the convolution and scan kernels: eight elements at a time whatever their type and alignment,
// silu, and the sum of per-block partial results in a fixed order.
#pragma once

#include "../../include/flare_b200_mixers.h"
#include "flare_common.cuh"

namespace flare {
namespace mixer {

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Eight elements as they lie in memory, so that loads can be in flight while the eight before are worked on.
template <typename T>
struct alignas(16) Raw8 {
  T v[8];
};

// `count` elements (the rest 0) from p; `wide`: p is 16-byte aligned and all eight lie inside the tensor.
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p, int count, bool wide) {
  Raw8<T> r;
  if (wide && count >= 8) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * 8 / 16); ++i) reinterpret_cast<uint4*>(r.v)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < count ? p[i] : from_float<T>(0.0f);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&out)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = to_float<T>(r.v[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8], int count, bool wide) {
  if (wide && count >= 8) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = from_float<T>(x[i]);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * 8 / 16); ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(r.v)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < count) p[i] = from_float<T>(x[i]);
  }
}

// 1 / (1 + exp(-x)): both functions within a few units in the last place, exp(-x) = inf gives 0
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

// may all rows of this tensor be read in 16-byte pieces?  (strides in elements)
inline bool rows_wide(const void* p, int dtype, std::initializer_list<int64_t> strides) {
  const int64_t per = 16 / dtype_size(dtype);
  if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  for (int64_t s : strides)
    if (s % per) return false;
  return true;
}

// out[i] = sum over p of in[p * stride + i], in the order of p (so the same call always gives the same bits)
struct SumList {
  struct Part {
    const float* in;
    void* out;
    int64_t count, stride;
    int parts, dtype;
  } part[4];
};
int launch_sum_parts(const SumList& list, int n, cudaStream_t stream);

}  // namespace mixer
}  // namespace flare
