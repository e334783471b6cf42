// Device helpers shared by the convolution and scan kernels: eight elements at a time whatever their type and alignment,
// silu, and the sum of per-block partial results in a fixed order.
#pragma once

#include "../../include/flare_b200_mixers.h"
#include "flare_common.cuh"
#include "sm100_ptx.cuh"

#include <type_traits>

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

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  return std::is_same<T, __half>::value ? sm100::pack_f16(lo, hi) : sm100::pack_bf16(lo, hi);
}

// V elements (8 unless said otherwise) as they lie in memory, so that loads can be in flight while others are worked on.
template <typename T, int V = 8>
struct Raw {
  static constexpr int WORDS = sizeof(T) * V / 4;
  uint32_t w[WORDS];
};
template <typename T>
using Raw8 = Raw<T, 8>;

__device__ __forceinline__ uint32_t word_of(__nv_bfloat16 lo, __nv_bfloat16 hi) {
  return (uint32_t)__bfloat16_as_ushort(lo) | (uint32_t)__bfloat16_as_ushort(hi) << 16;
}
__device__ __forceinline__ uint32_t word_of(__half lo, __half hi) {
  return (uint32_t)__half_as_ushort(lo) | (uint32_t)__half_as_ushort(hi) << 16;
}

// `count` elements (the rest 0) from p; `wide`: p is aligned to 16 bytes (or to the V elements, if those are fewer), and `count` is V or 0.
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p, int count, bool wide) {
  Raw<T, V> r;
  if (wide) {
    if constexpr (Raw<T, V>::WORDS == 2) {
      const uint2 v = count >= V ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
      r.w[0] = v.x; r.w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < Raw<T, V>::WORDS / 4; ++i) {
        const uint4 v = count >= V ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
        r.w[4 * i] = v.x; r.w[4 * i + 1] = v.y; r.w[4 * i + 2] = v.z; r.w[4 * i + 3] = v.w;
      }
    }
  } else {
    const T zero = from_float<T>(0.0f);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) r.w[i] = __float_as_uint(i < count ? (float)p[i] : 0.0f);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) r.w[i] = word_of(2 * i < count ? p[2 * i] : zero, 2 * i + 1 < count ? p[2 * i + 1] : zero);
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p, int count, bool wide) { return load_raw<T, 8>(p, count, wide); }

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&out)[V]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = __uint_as_float(r.w[i]);
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      out[2 * i] = __uint_as_float(r.w[i] << 16);
      out[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
      out[2 * i] = f.x;
      out[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&out)[8]) { unpack<T, 8>(r, out); }

// `wide`: all V go out in wide pieces (or, with count < V, nothing does)
template <typename T, int V>
__device__ __forceinline__ void store_all(T* p, const float (&x)[V], int count, bool wide) {
  if (wide) {
    if (count < V) return;
    uint32_t w[Raw<T, V>::WORDS];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = pack_pair<T>(x[2 * i], x[2 * i + 1]);
    }
    if constexpr (Raw<T, V>::WORDS == 2) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < Raw<T, V>::WORDS / 4; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
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
