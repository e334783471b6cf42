// What the tensor-core attention kernels share: scores and their slopes, tensor maps, shared-memory rows.
#pragma once
#include "attention.cuh"
#include "prefill_tc.cuh"
#include "tc_device.cuh"

namespace flare {
namespace attn {

using namespace tc;

// Scores in units of log 2.  CAP: cap tanh(s / cap) = cap (1 - 2 r) with r = 1 / (exp(2 s / cap) + 1); the absolute error is a few
// 2^-24 of cap whatever s is (tanh.approx would be off by 2^-11 of it, hundredths of a nat).
struct ScoreScale {
  float plain;     // scale log2 e
  float cap_in;    // 2 log2 e scale / cap
  float cap_out;   // cap log2 e
  float slope;     // of the head, log2 e times
};
__device__ __forceinline__ ScoreScale score_scale(const AttnParams& p, int h) {
  ScoreScale s;
  s.plain = p.scale * kLog2e;
  s.cap_in = p.cap > 0.0f ? 2.0f * kLog2e * p.scale / p.cap : 0.0f;
  s.cap_out = p.cap * kLog2e;
  s.slope = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.0f;
  return s;
}
// r of the capped score
__device__ __forceinline__ float cap_weight(float s, const ScoreScale& c) { return rcp_approx(ex2_approx(s * c.cap_in) + 1.0f); }
__device__ __forceinline__ float capped(float r, const ScoreScale& c) { return fmaf(-2.0f * c.cap_out, r, c.cap_out); }

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return F16 ? pack_f16(lo, hi) : pack_bf16(lo, hi);
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

// Clears the rows of a staged tile ([DB][ROWS][64 elements]) whose keys belong to nobody: their weights are 0, but 0 times what
// may lie there need not be.  Whole warp; the caller orders the async proxy behind it.
template <int DB, int ROWS>
__device__ __forceinline__ void clear_rows(uint8_t* tile, const Masks& m, int b, int64_t per_row, int first, int lane) {
#pragma unroll 1
  for (int r = lane; r < ROWS; r += 32)
    if (!m.owned(b, per_row, first + r)) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(tile + (d * ROWS + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
    }
}

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
