// What the tensor-core attention kernels share: scores and their slopes, tensor maps, shared-memory rows.
#pragma once
#include "attention.cuh"
#include "prefill_tc.cuh"
#include "tc_device.cuh"

namespace flare {
namespace attn {

using namespace tc;

// Scores, in units of log 2 once they are multiplied by `unit`.  CAP: cap tanh(x), x = scale <q, k> / cap.  The special-function
// unit would give tanh as 1 - 2 / (exp(2 x) + 1), two results of it per score where the softmax itself takes one (tanh.approx is off by 2^-11 of
// cap, hundredths of a nat); for |x| <= 0.35, where caps leave nearly all scores, an odd polynomial does it on the FMA pipe: a
// weighted least-squares fit of x p(x^2) with four coefficients, repeated until its error was level (5.9e-9).  With the first one in fp32 it is off by 1.5e-8 at
// most (1.8e-7 of small x), in fp32 arithmetic by 4.8e-8.  A warp that meets a larger |x| takes the exponential form.
struct ScoreScale {
  float unit;   // scale log2 e, or cap log2 e
  float in;     // scale / cap
  float slope;  // of the head, log2 e times
};
__device__ __forceinline__ ScoreScale score_scale(const AttnParams& p, int h) {
  ScoreScale s;
  s.unit = (p.cap > 0.0f ? p.cap : p.scale) * kLog2e;
  s.in = p.cap > 0.0f ? p.scale / p.cap : 0.0f;
  s.slope = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.0f;
  return s;
}
__device__ __forceinline__ uint64_t twice(float x) { return f2_pack(x, x); }
// the polynomial's coefficients, for raw products.  The last one holds in^7: where that is no normal number of fp32 (scale / cap below 2^-17 or above 2^17)
// the coefficients would be rounded to multiples of the smallest one, or infinite, and no score is small enough for them.
struct CapSeries {
  uint64_t c[4];
  float in, limit;  // of |x|
  __device__ __forceinline__ explicit CapSeries(float in_) : in(in_), limit(in_ >= 0x1p-17f && in_ <= 0x1p17f ? 0.35f : -1.0f) {
    const float q = in * in;
    c[0] = twice(0.9999998211860657f * in);
    c[1] = twice(-0.3333165645599365f * in * q);
    c[2] = twice(0.13283318281173706f * in * q * q);
    c[3] = twice(-0.04837666451931f * in * q * q * q);
  }
  __device__ __forceinline__ uint64_t operator()(uint64_t x) const {
    const uint64_t q = f2_mul(x, x);
    uint64_t t = f2_fma(q, c[3], c[2]);
    t = f2_fma(q, t, c[1]);
    return f2_mul(x, f2_fma(q, t, c[0]));
  }
};
__device__ __forceinline__ float tanh_any(float x) { return fmaf(-2.0f, rcp_approx(ex2_approx(x * (2.0f * kLog2e)) + 1.0f), 1.0f); }

template <int N>
__device__ __forceinline__ float largest(const uint32_t (&s)[N]) {
  float most = 0.0f;
#pragma unroll
  for (int k = 0; k < N; k += 2) most = fmax3(most, fabsf(__uint_as_float(s[k])), fabsf(__uint_as_float(s[k + 1])));
  return most;
}
// may the whole warp's raw products take the polynomial?
__device__ __forceinline__ bool all_small(const uint32_t (&a)[32], const uint32_t (&b)[32], const CapSeries& series) {
  return __all_sync(0xffffffffu, fmaxf(largest(a), largest(b)) * series.in <= series.limit) != 0;
}

// raw products, in place: tanh of the capped score.  Whole warp.
template <int N>
__device__ __forceinline__ void cap_scores(uint32_t (&s)[N], const CapSeries& series) {
  if (__all_sync(0xffffffffu, largest(s) * series.in <= series.limit)) {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      float lo, hi;
      f2_unpack(series(f2_pack(__uint_as_float(s[k]), __uint_as_float(s[k + 1]))), lo, hi);
      s[k] = __float_as_uint(lo);
      s[k + 1] = __float_as_uint(hi);
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = __float_as_uint(tanh_any(__uint_as_float(s[k]) * series.in));
  }
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return F16 ? pack_f16(lo, hi) : pack_bf16(lo, hi);
}
template <bool F16>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if (F16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  } else {
    lo = bf16_lo(w);
    hi = bf16_hi(w);
  }
}
template <bool F16>
constexpr uint32_t make_idesc(int M, int N, int a_mn, int b_mn) {
  return F16 ? make_idesc_f16(M, N, a_mn, b_mn) : make_idesc_bf16(M, N, a_mn, b_mn);
}

// [B, N, heads, D] as tiles of 64 columns and `rows` tokens of a head: columns behind D and rows behind N read as zero
inline bool head_map(CUtensorMap* map, const void* base, int B, int N, int heads, int D, int64_t sb, int64_t sn, int64_t sh, uint32_t rows) {
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)heads, (uint64_t)N, (uint64_t)B};
  const int64_t strides[3] = {heads > 1 ? sh : 8, N > 1 ? sn : 8, B > 1 ? sb : 8};
  const uint32_t box[4] = {64, 1, rows, 1};
  return make_map_bf16(map, base, 4, dims, strides, box);
}

// Clears a row of a staged tile ([DB][ROWS][64 elements]) if its token belongs to nobody: its weights are 0, but 0 times what
// may lie there need not be.  The caller orders the async proxy behind it.
template <int DB, int ROWS>
__device__ __forceinline__ void clear_row(uint8_t* tile, const Masks& m, int b, int64_t per_row, int first, int r) {
  if (m.owned(b, per_row, first + r)) return;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(tile + (d * ROWS + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
}

// Which of a row's tiles of 64 tokens hold some that belong to nobody: 32 tiles at a time, a bit each.  Whole warps.
struct DirtyTiles {
  const uint8_t* flags;
  int count, base;
  unsigned bits;
  __device__ __forceinline__ DirtyTiles(const Masks& m, int b) : flags(m.dirty + (int64_t)b * (m.Nkp >> 6)), count(m.Nkp >> 6), base(-32), bits(0) {}
  __device__ __forceinline__ bool operator()(int tile) {
    if ((unsigned)(tile - base) >= 32u) {
      base = tile;
      const int at = tile + (threadIdx.x & 31);
      bits = __ballot_sync(0xffffffffu, at < count && flags[at] != 0);
    }
    return bits >> (tile - base) & 1;
  }
};

// 32 columns of fp32 times `f`, rounded, to a row of an output (columns from D on left out; D is a multiple of 8)
template <bool F16>
__device__ __forceinline__ void store_columns(void* row, int first, int D, const uint32_t (&r)[32], float f) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (first + c * 8 < D) {
      uint4 v;
      v.x = pack2<F16>(__uint_as_float(r[c * 8 + 0]) * f, __uint_as_float(r[c * 8 + 1]) * f);
      v.y = pack2<F16>(__uint_as_float(r[c * 8 + 2]) * f, __uint_as_float(r[c * 8 + 3]) * f);
      v.z = pack2<F16>(__uint_as_float(r[c * 8 + 4]) * f, __uint_as_float(r[c * 8 + 5]) * f);
      v.w = pack2<F16>(__uint_as_float(r[c * 8 + 6]) * f, __uint_as_float(r[c * 8 + 7]) * f);
      reinterpret_cast<uint4*>(row)[(first >> 3) + c] = v;
    }
}

}  // namespace attn
}  // namespace flare
