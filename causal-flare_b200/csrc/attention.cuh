// Parameters and launchers of the attention kernels (attention.cu: who sees whom, caches, single tokens; attention_fwd.cu,
// attention_bwd.cu: the tensor-core kernels).
#pragma once
#include "mixer_common.cuh"

namespace flare {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

// Powers of two by which fp16 weights are laid down above their value, so that those far below one (long rows, a key that takes nearly all) are normal
// numbers too: forward, where the frame lets them grow to 2^8, and backward, where they are at most one (with a factor of four in hand).
template <bool F16>
constexpr float kFrameLift = F16 ? 7.0f : 0.0f;
constexpr int kWeightLift = 14;

// Which keys a query sees is always one interval, and both its ends grow with the query: whatever the mask, it is two numbers
// per query, and the keys of a tile of queries (the queries of a tile of keys) are one interval too.
struct Masks {
  const int2* range;       // [B][Nqp] keys [x, y) of a query
  const int2* query_span;  // [B][Nqp / 128] keys of 128 queries
  const int2* key_span;    // [B][Nkp / 128] queries of 128 keys
  const uint8_t* dirty;    // [B][Nkp / 64] 1: some of the 64 keys belong to nobody and may hold anything
  const int32_t* ends;     // [B] keys that a row has
  const int32_t* documents;
  const int32_t* cached;
  int Nqp, Nkp;  // rounded up to 128
  __device__ __forceinline__ bool owned(int b, int64_t row, int j) const {
    return j < ends[b] && (documents == nullptr || documents[row * b + j] >= 0);
  }
};

struct AttnParams {
  Masks masks;
  const float* slopes;
  float* lse;          // forward: written, may be null; backward: read
  const float* delta;  // backward: [B][H][Nqp] -<dy, y>
  // backward, fp16: |dy|^2 of every query and head, [B][H][Nqp]; the largest |dy|^2 and |v|^2 of a key head's tokens, [B][J][2].  Padding, and norms
  // that are not finite, count as 0.
  const float *dy_norm, *largest_norms;
  const float* lse_lifted;  // backward, fp16: lse + kWeightLift, for the kernel that lays weights down
  void *y, *dq, *dk, *dv;
  int* err;
  int B, Nq, Nk, H, J, D;
  float scale, cap;
};

int launch_forward_tc(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream);
int launch_backward_tc(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream);

}  // namespace attn
}  // namespace flare
