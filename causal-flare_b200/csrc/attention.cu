// Attention, everything but the tensor-core walks: who sees whom, <dy, y>, caches, single tokens, and the entry points.
#include "attention.cuh"

#include <limits.h>
#include <math.h>
#include <string.h>

#include "prefill_tc.cuh"

namespace flare {
namespace attn {
namespace {

using namespace mixer;

// ---- who sees whom ---------------------------------------------------------------------------------------------------

struct PlanParams {
  Masks m;
  int2* range;
  int2* query_span;
  int2* key_span;
  uint8_t* dirty;
  int32_t* ends;
  const uint8_t* prefix;
  const int32_t* lengths;
  int Nq, Nk, window;
};

constexpr int kPlanThreads = 1024, kPlanPer = 4, kPlanChunk = kPlanThreads * kPlanPer;

// Running maximum over a block's threads (MIN: minimum, from the last thread to the first): what lies in front of (MIN: behind)
// this thread's values, `carry` included; `carry` then takes the whole chunk in.
template <bool MIN>
__device__ __forceinline__ int block_running(int v, int& carry, int* warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const auto pick = [](int a, int b) { return MIN ? min(a, b) : max(a, b); };
  int run = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int got = MIN ? __shfl_down_sync(0xffffffffu, run, o) : __shfl_up_sync(0xffffffffu, run, o);
    if (MIN ? lane + o < 32 : lane >= o) run = pick(run, got);
  }
  __syncthreads();
  if (lane == (MIN ? 0 : 31)) warps[warp] = run;
  __syncthreads();
  int before = carry, all = carry;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (MIN ? w > warp : w < warp) before = pick(before, warps[w]);
    all = pick(all, warps[w]);
  }
  carry = all;
  const int next = MIN ? __shfl_down_sync(0xffffffffu, run, 1) : __shfl_up_sync(0xffffffffu, run, 1);
  return lane == (MIN ? 31 : 0) ? before : pick(before, next);
}

// One block per row.  A token's keys begin with its run of ids (or its window) and end behind itself, or behind the prefix
// that it is part of: the next token that is none, or that begins another run.  Bound by the latency of a few dozen steps on one SM: 10 us for 2 049 tokens.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  pdl_begin();
  __shared__ int warps[kPlanThreads / 32];
  const int b = blockIdx.x, tid = threadIdx.x, Nqp = p.m.Nqp;
  const int32_t* ids = p.m.documents != nullptr ? p.m.documents + (int64_t)b * p.Nq : nullptr;
  const uint8_t* prefix = p.prefix != nullptr ? p.prefix + (int64_t)b * p.Nq : nullptr;
  int cached = 0, len = p.Nq;
  if (p.m.cached != nullptr) cached = p.m.cached[b];
  if (p.lengths != nullptr) len = max(0, min(p.Nq, p.lengths[b]));
  if (cached < 0 || cached > p.Nk) len = 0;
  len = min(len, p.Nk - cached);
  const int end = len > 0 ? cached + len : 0;
  int2* const range = p.range + (int64_t)b * Nqp;
  if (tid == 0) p.ends[b] = end;
  const auto border = [&](int i) { return i == 0 || (ids != nullptr && ids[i] != ids[i - 1]); };
  // forward: first token of the run, last token that is no prefix
  int start_carry = 0, gap_carry = -1;
  for (int c0 = 0; c0 < Nqp; c0 += kPlanChunk) {
    const int i0 = c0 + tid * kPlanPer;
    int start[kPlanPer], gap[kPlanPer], s = -1, g = -1;
#pragma unroll
    for (int k = 0; k < kPlanPer; ++k) {
      const int i = i0 + k;
      if (i < len) {
        if (border(i)) s = i;
        if (prefix == nullptr || prefix[i] == 0) g = i;
      }
      start[k] = s;
      gap[k] = g;
    }
    const int s0 = block_running<false>(s, start_carry, warps), g0 = block_running<false>(g, gap_carry, warps);
#pragma unroll
    for (int k = 0; k < kPlanPer; ++k) {
      const int i = i0 + k;
      if (i >= Nqp) break;
      int2 r = make_int2(end, end);  // nobody
      if (i < len) {
        const int at = cached + i;
        if (ids != nullptr && ids[i] < 0) {
          r = make_int2(i, i);
        } else {
          const int begin = max(s0, start[k]);
          r.x = p.m.cached != nullptr ? 0 : begin;
          if (p.window > 0) r.x = max(r.x, at - p.window + 1);
          r.y = max(g0, gap[k]) < begin ? -1 : at + 1;  // (-1: part of the prefix, see below)
        }
      }
      range[i] = r;
    }
  }
  if (prefix != nullptr) {
    int stop_carry = len;
    for (int c0 = (Nqp - 1) / kPlanChunk * kPlanChunk; c0 >= 0; c0 -= kPlanChunk) {
      const int i0 = c0 + tid * kPlanPer;
      int stop[kPlanPer], s = INT_MAX;  // first stop behind token i
#pragma unroll
      for (int k = kPlanPer - 1; k >= 0; --k) {
        stop[k] = s;
        const int i = i0 + k;
        if (i < len && (prefix[i] == 0 || border(i))) s = i;
      }
      const int s0 = block_running<true>(s, stop_carry, warps);
#pragma unroll
      for (int k = 0; k < kPlanPer; ++k) {
        const int i = i0 + k;
        if (i < len && range[i].y == -1) range[i].y = cached + min(s0, stop[k]);
      }
    }
  }
  __syncthreads();
  // tiles of 128 queries: a warp each
  const int lane = tid & 31;
  for (int t = tid >> 5; t < Nqp / 128; t += kPlanThreads / 32) {
    int lo = INT_MAX, hi = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int2 r = range[t * 128 + k * 32 + lane];
      if (r.y > r.x) {
        lo = min(lo, r.x);
        hi = max(hi, r.y);
      }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) p.query_span[(int64_t)b * (Nqp / 128) + t] = hi > lo ? make_int2(lo, hi) : make_int2(0, 0);
  }
  // tiles of 128 keys: the first query whose keys end behind the tile's first, and the first whose keys begin behind its last.  Both
  // ends grow with the query, so every tile's two queries are where an end passes the tile: each query looks at the one before it.
  int2* const key_span = p.key_span + (int64_t)b * (p.m.Nkp / 128);
  for (int t = tid; t < p.m.Nkp / 128; t += kPlanThreads) key_span[t] = p.m.cached == nullptr ? make_int2(p.Nq, p.Nq) : make_int2(0, 0);
  __syncthreads();
  if (p.m.cached == nullptr) {
    for (int i = tid; i < p.Nq; i += kPlanThreads) {
      const int2 r = range[i], before = i > 0 ? range[i - 1] : make_int2(0, 0);
      for (int t = (before.y + 127) / 128; t * 128 < r.y; ++t) key_span[t].x = i;
      for (int t = before.x / 128; t * 128 + 128 <= r.x; ++t) key_span[t].y = i;
    }
  }
  for (int t = tid >> 5; t < p.m.Nkp / 64; t += kPlanThreads / 32) {
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = t * 64 + k * 32 + lane;
      bad |= j < p.Nk && (j >= end || (ids != nullptr && ids[j] < 0));
    }
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) p.dirty[(int64_t)b * (p.m.Nkp / 64) + t] = bad;
  }
}

struct DeltaParams {
  AttnParams p;
  const void *q, *k, *v, *dy;
  int64_t q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h, dy_b, dy_n, dy_h;
  float *delta, *dy_norm, *v_norm;  // (v_norm: [B][J][Nqp])
};
// Keys up to which a row's delta is the sum of P dP itself.  <dy, y> has y's rounding and that of the weights in y, about 2^-9 |dy| |v| / sqrt(keys),
// which dS = P (dP - delta) keeps: with two to five keys dQ and dK were 1.7 to 4 times as far off as their own rounding, with 50 and more 1.1.
constexpr int kFewKeys = 32;
constexpr int kRows = 32768;  // rows of the batch along a grid's second dimension

// -delta, delta = sum P dP = <dy, y>, LANES threads per row and head; 0 for queries without keys (their dy may hold anything).  For fp16 the norms too
// from which the kernels behind it know how large dS can be.  Bound by memory: B=2 N=4096 H=16 D=128 29 us, in fp16 with the values' rows 46.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) delta_kernel(const __grid_constant__ DeltaParams d) {
  pdl_begin();
  const AttnParams& p = d.p;
  const int lane = threadIdx.x % LANES, b = blockIdx.z * kRows + blockIdx.y;  // (a grid's second dimension ends at 65 535)
  if (b >= p.B) return;
  const unsigned idx = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int i = (int)(idx / (unsigned)p.H), h = (int)(idx % (unsigned)p.H);
  const bool live = i < p.masks.Nqp, mine = live && i < p.Nq && lane * 8 < p.D;
  const int2 r = live && i < p.Nq ? p.masks.range[(int64_t)b * p.masks.Nqp + i] : make_int2(0, 0);
  const auto eight = [&](const void* base, int64_t at, float (&out)[8]) {  // of a row
    unpack8(load_raw8<T>(reinterpret_cast<const T*>(base) + at + lane * 8, 8, true), out);
  };
  const auto dot = [](const float (&a)[8], const float (&c)[8]) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fmaf(a[k], c[k], s);
    return s;
  };
  const auto joined = [](float s) {  // over the row's threads
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  };
  float dy[8] = {}, sum = 0.0f;
  constexpr bool NORMS = std::is_same<T, __half>::value;
  const int keys = r.y - r.x, kv = h / (p.H / p.J);
  const bool value = NORMS && mine && h == kv * (p.H / p.J);  // (one of its heads looks at the token's value)
  Raw8<T> own_value;
  const bool few = keys <= kFewKeys;
  if (mine) {  // (the loads do not wait for the row's keys)
    float y[8];
    eight(d.dy, b * d.dy_b + i * d.dy_n + h * d.dy_h, dy);
    eight(p.y, (((int64_t)b * p.Nq + i) * p.H + h) * p.D, y);
    sum = dot(dy, y);
  }
  if (NORMS) own_value = load_raw8<T>(reinterpret_cast<const T*>(d.v) + b * d.v_b + i * d.v_n + kv * d.v_h + lane * 8, value ? 8 : 0, true);
  sum = joined(sum);
  const int steps = __reduce_max_sync(0xffffffffu, few ? max(keys, 0) : 0);
  if (steps > 0) {
    float q[8] = {}, weights = 0.0f, weighted = 0.0f;
    if (mine) eight(d.q, b * d.q_b + i * d.q_n + h * d.q_h, q);
    const float lse = few && keys > 0 ? p.lse[((int64_t)b * p.H + h) * p.masks.Nqp + i] : 0.0f, slope = p.slopes != nullptr ? p.slopes[h] : 0.0f;
    constexpr int GROUP = 4;  // keys on their way together
    for (int t0 = 0; t0 < steps; t0 += GROUP) {
      Raw8<T> k[GROUP], v[GROUP];
#pragma unroll
      for (int g = 0; g < GROUP; ++g) {
        const int64_t j = r.x + t0 + g;
        const int count = mine && few && t0 + g < keys ? 8 : 0;
        k[g] = load_raw8<T>(reinterpret_cast<const T*>(d.k) + b * d.k_b + j * d.k_n + kv * d.k_h + lane * 8, count, true);
        v[g] = load_raw8<T>(reinterpret_cast<const T*>(d.v) + b * d.v_b + j * d.v_n + kv * d.v_h + lane * 8, count, true);
      }
#pragma unroll
      for (int g = 0; g < GROUP; ++g) {
        const bool on = few && t0 + g < keys;
        float f[8];
        unpack8(k[g], f);
        float s = joined(dot(q, f)) * p.scale;
        unpack8(v[g], f);
        const float dp = joined(dot(dy, f));
        if (p.cap > 0.0f) s = p.cap * tanhf(s / p.cap);
        s = fmaf(-slope, (float)abs(i - (r.x + t0 + g)), s);
        const float w = on ? exp2f(fmaf(s, kLog2e, lse)) : 0.0f;
        weights += w;
        weighted = on ? fmaf(w, dp, weighted) : weighted;
      }
    }
    if (few) sum = weights == 0.0f ? 0.0f : weighted / weights;  // (0: no score above -infinity, and y is 0)
  }
  if (keys <= 0) sum = 0.0f;
  const int64_t at = ((int64_t)b * p.H + h) * p.masks.Nqp + i;
  if (live && lane == 0) d.delta[at] = -sum;
  if constexpr (NORMS) {
    float v[8];
    unpack8(own_value, v);
    const float dy_norm = joined(dot(dy, dy)), v_norm = joined(dot(v, v));
    if (live && lane == 0) {  // (comparisons with what is no number are false)
      d.dy_norm[at] = keys > 0 && dy_norm < INFINITY ? dy_norm : 0.0f;
      if (h == kv * (p.H / p.J)) d.v_norm[((int64_t)b * p.J + kv) * p.masks.Nqp + i] = keys > 0 && v_norm < INFINITY ? v_norm : 0.0f;
    }
  }
}

// The largest norms of a key head's tokens: |dy|^2 of its query heads, |v|^2; on the way the queries' lse for lifted weights (rows of [.., Nqp], as the
// norms are).  One block for a key head: two times 4 096 norms are 7 us at most (the wait for the kernel in front is part of it).
__global__ void __launch_bounds__(1024) largest_norms_kernel(const float* dy_norm, const float* v_norm, const float* lse, float* lse_lifted, float* out, int group,
                                                             int Nqp) {
  pdl_wait();
  pdl_trigger();
  const int64_t head = blockIdx.x;  // key head of the batch
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ float tops[2][32];
  const auto largest = [&](const float* from, int64_t n) {  // (n: a multiple of 128)
    float top = 0.0f;
    for (int64_t i = threadIdx.x; i < n / 4; i += 1024) {
      const float4 v = reinterpret_cast<const float4*>(from)[i];
      top = fmaxf(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    return top;
  };
  const int64_t first = head * group * Nqp, queries = (int64_t)group * Nqp;
  for (int64_t i = threadIdx.x; i < queries / 4; i += 1024) {
    constexpr float up = (float)kWeightLift;
    const float4 v = reinterpret_cast<const float4*>(lse + first)[i];
    reinterpret_cast<float4*>(lse_lifted + first)[i] = make_float4(v.x + up, v.y + up, v.z + up, v.w + up);
  }
  const float dy = largest(dy_norm + first, queries), v = largest(v_norm + head * Nqp, Nqp);
  if (lane == 0) {
    tops[0][warp] = dy;
    tops[1][warp] = v;
  }
  __syncthreads();
  if (warp < 2) {
    float top = tops[warp][lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) out[head * 2 + warp] = top;
  }
}

struct Layout {
  size_t range, query_span, key_span, dirty, ends, plan_bytes;      // in `plan`, or in front of the workspace
  size_t delta, dy_norm, v_norm, largest_norms, lse_lifted, bytes;  // in the workspace
  int Nqp, Nkp;
};
Layout layout(const flare_attention_args_t& a, bool backward) {
  Layout l;
  l.Nqp = (a.Nq + 127) / 128 * 128;
  l.Nkp = (a.Nk + 127) / 128 * 128;
  size_t at = 0;
  const auto take = [&](size_t n) {
    const size_t here = at;
    at += align_up(n, 256);
    return here;
  };
  l.range = take((size_t)a.B * l.Nqp * sizeof(int2));
  l.query_span = take((size_t)a.B * (l.Nqp / 128) * sizeof(int2));
  l.key_span = take((size_t)a.B * (l.Nkp / 128) * sizeof(int2));
  l.dirty = take((size_t)a.B * (l.Nkp / 64));
  l.ends = take((size_t)a.B * 4);
  l.plan_bytes = at;
  if (a.plan != nullptr) at = 0;
  const bool f16 = backward && a.dtype == FLARE_F16;
  l.delta = take(backward ? (size_t)a.B * a.H * l.Nqp * 4 : 0);
  l.dy_norm = take(f16 ? (size_t)a.B * a.H * l.Nqp * 4 : 0);
  l.lse_lifted = take(f16 ? (size_t)a.B * a.H * l.Nqp * 4 : 0);
  l.v_norm = take(f16 ? (size_t)a.B * a.J * l.Nqp * 4 : 0);
  l.largest_norms = take(f16 ? (size_t)a.B * a.J * 8 : 0);
  l.bytes = at;
  return l;
}

// Scores and caps that fp32 holds.  Behind a cap a score is off by up to cap 2^-21: from 1024 on that would be more than the rounding of
// the weights.
bool bad_scores(float scale, float cap, int window) {
  return !(scale > 0.0f) || !isfinite(scale) || !(cap >= 0.0f) || cap > 1024.0f || (cap > 0.0f && !isfinite(4.0f * scale / cap)) || window < 0;
}

bool strides_fit(const void* p, std::initializer_list<int64_t> strides) {
  if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15u)) return false;
  for (int64_t s : strides)
    if (s < 0 || s % 8) return false;
  return true;
}

int check(const flare_attention_args_t* args) {
  if (args == nullptr) return FLARE_ERR_BAD_POINTER;
  const flare_attention_args_t& a = *args;
  if (a.B <= 0 || a.Nq <= 0 || a.Nk <= 0 || a.H <= 0 || a.J <= 0 || a.D <= 0 || a.H % a.J) return FLARE_ERR_BAD_SHAPE;
  if (a.D % 8 || a.D > 128 || a.Nq > INT_MAX - 8192 || a.Nk > INT_MAX - 8192) return FLARE_ERR_UNSUPPORTED;
  if (a.dtype != FLARE_BF16 && a.dtype != FLARE_F16) return FLARE_ERR_BAD_DTYPE;
  if (bad_scores(a.scale, a.cap, a.window)) return FLARE_ERR_BAD_CONFIG;
  if (a.cached == nullptr ? a.Nk != a.Nq : a.documents != nullptr) return FLARE_ERR_BAD_CONFIG;
  if (reinterpret_cast<uintptr_t>(a.plan) & 255u) return FLARE_ERR_BAD_POINTER;
  if (!strides_fit(a.q, {a.q_stride_b, a.q_stride_n, a.q_stride_h}) || !strides_fit(a.k, {a.k_stride_b, a.k_stride_n, a.k_stride_h}) ||
      !strides_fit(a.v, {a.v_stride_b, a.v_stride_n, a.v_stride_h}) || !strides_fit(a.y, {}))
    return FLARE_ERR_BAD_POINTER;
  return FLARE_OK;
}

bool workspace_fits(const flare_attention_args_t& a, const Layout& l) {
  return l.bytes == 0 || (a.workspace != nullptr && a.workspace_bytes >= l.bytes && (reinterpret_cast<uintptr_t>(a.workspace) & 255u) == 0);
}

// parameters, and the masks' kernel (unless the forward left what it finds)
int begin(const flare_attention_args_t& a, const Layout& l, AttnParams& p, bool backward, cudaStream_t stream) {
  memset(&p, 0, sizeof(p));
  uint8_t* const ws = reinterpret_cast<uint8_t*>(a.plan != nullptr ? a.plan : a.workspace);
  PlanParams plan;
  plan.range = reinterpret_cast<int2*>(ws + l.range);
  plan.query_span = reinterpret_cast<int2*>(ws + l.query_span);
  plan.key_span = reinterpret_cast<int2*>(ws + l.key_span);
  plan.dirty = ws + l.dirty;
  plan.ends = reinterpret_cast<int32_t*>(ws + l.ends);
  p.masks = {plan.range, plan.query_span, plan.key_span, plan.dirty, plan.ends, a.documents, a.cached, l.Nqp, l.Nkp};
  plan.m = p.masks;
  plan.prefix = a.prefix;
  plan.lengths = a.lengths;
  plan.Nq = a.Nq; plan.Nk = a.Nk; plan.window = a.window;
  p.slopes = a.slopes;
  p.lse = a.lse;
  p.y = a.y; p.dq = a.dq; p.dk = a.dk; p.dv = a.dv;
  p.B = a.B; p.Nq = a.Nq; p.Nk = a.Nk; p.H = a.H; p.J = a.J; p.D = a.D;
  p.scale = a.scale; p.cap = a.cap;
  if (const int rc = tc_error_word(&p.err)) return rc;
  if (backward && a.plan != nullptr) return FLARE_OK;
  LaunchTimer timer("attention_plan_kernel", stream);
  FLARE_CUDA_CHECK(launch_pdl(plan_kernel, dim3((unsigned)a.B), dim3(kPlanThreads), 0, stream, plan));
  return FLARE_OK;
}

// ---- caches and single tokens --------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(256) append_kernel(const flare_cache_args_t a) {
  pdl_begin();
  const int pieces = a.D >> 3;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t per = (int64_t)a.N * a.J * pieces;
  if (idx >= a.B * per) return;
  const int64_t b = idx / per;
  int64_t r = idx - b * per;
  const int t = (int)(r / (a.J * pieces));
  r -= (int64_t)t * a.J * pieces;
  const int j = (int)(r / pieces), c = (int)(r % pieces) * 8;
  const int len = a.lengths != nullptr ? a.lengths[b] : a.N;
  const int64_t at = (int64_t)(a.cached != nullptr ? a.cached[b] : 0) + t;
  // (a row that begins outside its cache is left alone: its tokens see nothing, either)
  if (t >= len || at - t < 0 || at >= a.L) return;
  const uint16_t* k = reinterpret_cast<const uint16_t*>(a.new_k) + b * a.new_k_stride_b + t * a.new_k_stride_n + j * a.new_k_stride_h + c;
  const uint16_t* v = reinterpret_cast<const uint16_t*>(a.new_v) + b * a.new_v_stride_b + t * a.new_v_stride_n + j * a.new_v_stride_h + c;
  uint16_t* ko = reinterpret_cast<uint16_t*>(a.k_cache) + b * a.k_stride_b + at * a.k_stride_n + j * a.k_stride_h + c;
  uint16_t* vo = reinterpret_cast<uint16_t*>(a.v_cache) + b * a.v_stride_b + at * a.v_stride_n + j * a.v_stride_h + c;
  *reinterpret_cast<uint4*>(ko) = *reinterpret_cast<const uint4*>(k);
  *reinterpret_cast<uint4*>(vo) = *reinterpret_cast<const uint4*>(v);
}

struct DecodeParams {
  flare_cache_args_t a;
  float* part;  // [splits][B][H][D + 2]: unnormalised sums, maximum (log 2), denominator; null: y is written
  int splits, head_groups;
  bool cluster;  // a row's splits form a cluster
};

constexpr int kDecodeWarps = 4, kHeads = 16;  // heads of a block: the rows of a product
constexpr int kCluster = 8;                   // (what a cluster may have without being asked for more)

// rows 8 to 15 of the product: none of them has a head (EIGHT), or they are there
template <bool F16, bool EIGHT>
__device__ __forceinline__ void mma16816(float (&d)[EIGHT ? 2 : 4], const uint32_t (&a)[EIGHT ? 2 : 4], uint32_t b0, uint32_t b1) {
  if constexpr (EIGHT) {
    float none0, none1;
    if constexpr (F16)
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%0, %1, %9, %9};"
                   : "+f"(d[0]), "+f"(d[1]), "=f"(none0), "=f"(none1) : "r"(a[0]), "r"(0), "r"(a[1]), "r"(b0), "r"(b1), "f"(0.0f));
    else
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%0, %1, %9, %9};"
                   : "+f"(d[0]), "+f"(d[1]), "=f"(none0), "=f"(none1) : "r"(a[0]), "r"(0), "r"(a[1]), "r"(b0), "r"(b1), "f"(0.0f));
  } else {
    if constexpr (F16)
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                   : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                   : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// One token.  Bound by memory: every key and value in sight is read once, by one block for up to 16 query heads that share
// them.  A warp takes 16 keys at a time, straight from memory into the operands of m16n8k16 products: heads are the rows, so the
// scores come out as the A operand that the product with V takes.  A thread's 16-byte piece of a key covers the contraction in an
// order of its own (the queries are laid out in the same one); pairs of keys of V are formed by byte permutes.  Rows are cut into `splits` parts
// for the SMs; the warps of a block join theirs in shared memory, the blocks of a row theirs in a second kernel or, where all of them run
// at once, as a cluster that reads one another's shared memory (plan_decode).  B=32 H=32 J=8 D=128, caches of 4 096 filled to different
// lengths: 90 us, 4.5 TB/s (the same loads without the work between them: 67).
template <int DB, bool F16, bool EIGHT>
__global__ void __launch_bounds__(32 * kDecodeWarps) decode_kernel(const DecodeParams p) {
  constexpr int HALVES = EIGHT ? 1 : 2;  // of the sixteen rows
  using T = typename std::conditional<F16, __half, __nv_bfloat16>::type;
  pdl_begin();
  const flare_cache_args_t& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, j = blockIdx.y / p.head_groups, b = blockIdx.z, group = a.H / a.J;
  const int h0 = j * group + (blockIdx.y % p.head_groups) * kHeads, heads = min(kHeads, (j + 1) * group - h0);
  const int position = a.cached[b];
  const bool idle = position < 0 || position >= a.L;
  __shared__ float joined[kDecodeWarps][8 * HALVES][64 * DB + 2], block_ends[8 * HALVES][2];
  const uint16_t* const new_k = reinterpret_cast<const uint16_t*>(a.new_k) + b * a.new_k_stride_b + j * a.new_k_stride_h;
  const uint16_t* const new_v = reinterpret_cast<const uint16_t*>(a.new_v) + b * a.new_v_stride_b + j * a.new_v_stride_h;
  const uint16_t* const keys = reinterpret_cast<const uint16_t*>(a.k_cache) + b * a.k_stride_b + j * a.k_stride_h;
  const uint16_t* const values = reinterpret_cast<const uint16_t*>(a.v_cache) + b * a.v_stride_b + j * a.v_stride_h;
  // the token's row of the cache, which no block of this launch reads
  if (!idle && split == 0 && blockIdx.y % p.head_groups == 0 && threadIdx.x < (a.D >> 3)) {
    const int d = threadIdx.x * 8;
    uint16_t* ko = reinterpret_cast<uint16_t*>(a.k_cache) + b * a.k_stride_b + position * a.k_stride_n + j * a.k_stride_h + d;
    uint16_t* vo = reinterpret_cast<uint16_t*>(a.v_cache) + b * a.v_stride_b + position * a.v_stride_n + j * a.v_stride_h + d;
    *reinterpret_cast<uint4*>(ko) = *reinterpret_cast<const uint4*>(new_k + d);
    *reinterpret_cast<uint4*>(vo) = *reinterpret_cast<const uint4*>(new_v + d);
  }
  const int first = a.window > 0 ? max(0, position - a.window + 1) : 0;
  const int chunks = idle ? 0 : (position - first + 16) / 16;  // of 16 keys, the new one among them
  const int per = (chunks + p.splits - 1) / p.splits, begin = split * per, end = min(chunks, begin + per);

  // queries: k-step s of segment g (32 columns) takes columns 8 c + 4 s .. + 3
  uint32_t q[2 * DB][2][2 * HALVES];
#pragma unroll
  for (int g = 0; g < 2 * DB; ++g)
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {  // rows r and r + 8
      const int h = r + half * 8, d = g * 32 + c * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (h < heads && d < a.D) v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + b * a.q_stride_b + (h0 + h) * a.q_stride_h + d);
      q[g][0][half] = v.x; q[g][0][half + HALVES] = v.y;
      q[g][1][half] = v.z; q[g][1][half + HALVES] = v.w;
    }
  const float plain = a.scale * kLog2e, cap_in = a.cap > 0.0f ? 2.0f * kLog2e * a.scale / a.cap : 0.0f, cap_out = a.cap * kLog2e;
  float slope[HALVES] = {};
  if (a.slopes != nullptr)
    for (int half = 0; half < HALVES; ++half)
      if (r + half * 8 < heads) slope[half] = a.slopes[h0 + r + half * 8] * kLog2e;
  float o[DB * 8][2 * HALVES] = {}, top[HALVES], sum[HALVES] = {};
#pragma unroll
  for (int half = 0; half < HALVES; ++half) top[half] = -INFINITY;

  // The keys of the chunk after this one are fetched as soon as this one's have met the queries, the values as soon as this one's
  // have met the weights: both are on their way all the time, in the registers that they leave.
  uint4 kr[2][2 * DB], vr[4][DB];
  const int64_t last_row = position - 1;  // of the cache
  const auto fetch_keys = [&](int chunk) {
    const int key0 = first + chunk * 16;
    if (key0 + 16 <= position && a.D == 64 * DB) {  // (whole chunks of the cache need no look at every piece)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint16_t* row = keys + (int64_t)(key0 + n * 8 + r) * a.k_stride_n + c * 8;
#pragma unroll
        for (int g = 0; g < 2 * DB; ++g) kr[n][g] = load_streaming(reinterpret_cast<const uint4*>(row + g * 32));
      }
    } else {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int key = key0 + n * 8 + r;
        const uint16_t* row = key < position ? keys + min((int64_t)key, last_row) * a.k_stride_n : new_k;
#pragma unroll
        for (int g = 0; g < 2 * DB; ++g) {
          const int d = g * 32 + c * 8;
          kr[n][g] = key <= position && d < a.D ? load_streaming(reinterpret_cast<const uint4*>(row + d)) : make_uint4(0, 0, 0, 0);
        }
      }
    }
  };
  const auto fetch_values = [&](int chunk) {
    const int key0 = first + chunk * 16;
    if (key0 + 16 <= position && a.D == 64 * DB) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint16_t* row = values + (int64_t)(key0 + 2 * c + (n & 1) + (n >> 1) * 8) * a.v_stride_n + r * 8;
#pragma unroll
        for (int g = 0; g < DB; ++g) vr[n][g] = load_streaming(reinterpret_cast<const uint4*>(row + g * 64));
      }
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int key = key0 + 2 * c + (n & 1) + (n >> 1) * 8;
        const uint16_t* row = key < position ? values + min((int64_t)key, last_row) * a.v_stride_n : new_v;
#pragma unroll
        for (int g = 0; g < DB; ++g) {
          const int d = g * 64 + r * 8;
          vr[n][g] = key <= position && d < a.D ? load_streaming(reinterpret_cast<const uint4*>(row + d)) : make_uint4(0, 0, 0, 0);
        }
      }
    }
  };
  if (begin + warp < end) {
    fetch_keys(begin + warp);
    fetch_values(begin + warp);
  }
#pragma unroll 1
  for (int chunk = begin + warp; chunk < end; chunk += kDecodeWarps) {
    const int key0 = first + chunk * 16;
    float s[2][2 * HALVES] = {};
#pragma unroll
    for (int g = 0; g < 2 * DB; ++g)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        mma16816<F16, EIGHT>(s[n], q[g][0], kr[n][g].x, kr[n][g].y);
        mma16816<F16, EIGHT>(s[n], q[g][1], kr[n][g].z, kr[n][g].w);
      }
    if (chunk + kDecodeWarps < end) fetch_keys(chunk + kDecodeWarps);
    // s[n][2 half + i]: head r + 8 half, key key0 + 8 n + 2 c + i
    float most[HALVES];
#pragma unroll
    for (int half = 0; half < HALVES; ++half) most[half] = -INFINITY;
    const bool whole = key0 + 15 <= position;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2 * HALVES; ++e) {
        const int key = key0 + n * 8 + 2 * c + (e & 1);
        float x = s[n][e];
        if (a.cap > 0.0f) x = fmaf(-2.0f * cap_out, sm100::rcp_approx(sm100::ex2_approx(x * cap_in) + 1.0f), cap_out);
        else x *= plain;
        x = fmaf(-slope[e >> 1], (float)(position - key), x);
        s[n][e] = whole || key <= position ? x : -INFINITY;
        most[e >> 1] = fmaxf(most[e >> 1], s[n][e]);
      }
    // the frame moves only where the maximum has grown by more than 2^8 (it cancels in the quotient)
    bool grow = false;
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
      most[half] = fmaxf(most[half], __shfl_xor_sync(0xffffffffu, most[half], 1));
      most[half] = fmaxf(most[half], __shfl_xor_sync(0xffffffffu, most[half], 2));
      grow |= most[half] > top[half] + 8.0f || (top[half] == -INFINITY && most[half] > top[half]);
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int half = 0; half < HALVES; ++half) {
        const float to = fmaxf(top[half], most[half]);
        const float scale = top[half] == -INFINITY ? 0.0f : exp2f(top[half] - to);
        top[half] = to;
        sum[half] *= scale;
#pragma unroll
        for (int n = 0; n < DB * 8; ++n) {
          o[n][2 * half] *= scale;
          o[n][2 * half + 1] *= scale;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2 * HALVES; ++e) {
        s[n][e] = sm100::ex2_approx(s[n][e] - (top[e >> 1] == -INFINITY ? 0.0f : top[e >> 1] - kFrameLift<F16>));
        sum[e >> 1] += s[n][e];
      }
    uint32_t w[2 * HALVES];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int half = 0; half < HALVES; ++half) w[n * HALVES + half] = pack_pair<T>(s[n][2 * half], s[n][2 * half + 1]);
#pragma unroll
    for (int g = 0; g < DB; ++g) {
      const uint32_t v0[4] = {vr[0][g].x, vr[0][g].y, vr[0][g].z, vr[0][g].w}, v1[4] = {vr[1][g].x, vr[1][g].y, vr[1][g].z, vr[1][g].w};
      const uint32_t v2[4] = {vr[2][g].x, vr[2][g].y, vr[2][g].z, vr[2][g].w}, v3[4] = {vr[3][g].x, vr[3][g].y, vr[3][g].z, vr[3][g].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
        mma16816<F16, EIGHT>(o[g * 8 + e], w, __byte_perm(v0[e >> 1], v1[e >> 1], sel), __byte_perm(v2[e >> 1], v3[e >> 1], sel));
      }
    }
    if (chunk + kDecodeWarps < end) fetch_values(chunk + kDecodeWarps);
  }
#pragma unroll
  for (int half = 0; half < HALVES; ++half) {
    sum[half] += __shfl_xor_sync(0xffffffffu, sum[half], 1);
    sum[half] += __shfl_xor_sync(0xffffffffu, sum[half], 2);
  }
  // o[g * 8 + e][2 half + i]: head r + 8 half, column 64 g + 8 (2 c + i) + e
#pragma unroll
  for (int half = 0; half < HALVES; ++half) {
    float* const row = joined[warp][r + half * 8];
#pragma unroll
    for (int n = 0; n < DB * 8; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) row[(n >> 3) * 64 + (2 * c + i) * 8 + (n & 7)] = o[n][2 * half + i];
    if (c == 0) {
      row[64 * DB] = top[half];
      row[64 * DB + 1] = sum[half];
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < heads * a.D; idx += 32 * kDecodeWarps) {
    const int h = idx / a.D, d = idx - h * a.D;
    float t = -INFINITY, l = 0.0f, v = 0.0f;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) t = fmaxf(t, joined[w][h][64 * DB]);
    const float frame = t == -INFINITY ? 0.0f : t;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      const float f = exp2f(joined[w][h][64 * DB] - frame);
      l = fmaf(joined[w][h][64 * DB + 1], f, l);
      v = fmaf(joined[w][h][d], f, v);
    }
    const int64_t row = (int64_t)b * a.H + h0 + h;
    if (p.splits == 1) {
      store1(a.y, a.dtype, row * a.D + d, l == 0.0f ? 0.0f : v / l);  // (0: an idle row, or no score above -infinity)
    } else if (p.cluster) {
      joined[0][h][d] = v;  // (no other thread reads this one)
      if (d == 0) {
        block_ends[h][0] = t;
        block_ends[h][1] = l;
      }
    } else {
      float* const out = p.part + ((int64_t)split * a.B * a.H + row) * (a.D + 2);
      out[d] = v;
      if (d == 0) {
        out[a.D] = t;
        out[a.D + 1] = l;
      }
    }
  }
  if (p.cluster) {
    __syncwarp();
    sm100::cluster_sync_all();
    const uint32_t sums = sm100::smem_u32(&joined[0][0][0]), ends = sm100::smem_u32(&block_ends[0][0]);
    for (int idx = split * 32 * kDecodeWarps + threadIdx.x; idx < heads * a.D; idx += p.splits * 32 * kDecodeWarps) {
      const int h = idx / a.D, d = idx - h * a.D;
      float top_of[kCluster], t = -INFINITY, l = 0.0f, v = 0.0f;
#pragma unroll
      for (int s = 0; s < kCluster; ++s) {
        top_of[s] = s < p.splits ? sm100::ld_cluster_f32(sm100::mapa_shared(ends + h * 8, s)) : -INFINITY;
        t = fmaxf(t, top_of[s]);
      }
      const float frame = t == -INFINITY ? 0.0f : t;
#pragma unroll
      for (int s = 0; s < kCluster; ++s)
        if (s < p.splits) {
          const float f = exp2f(top_of[s] - frame);
          l = fmaf(sm100::ld_cluster_f32(sm100::mapa_shared(ends + h * 8 + 4, s)), f, l);
          v = fmaf(sm100::ld_cluster_f32(sm100::mapa_shared(sums + (h * (64 * DB + 2) + d) * 4, s)), f, v);
        }
      store1(a.y, a.dtype, ((int64_t)b * a.H + h0 + h) * a.D + d, l == 0.0f ? 0.0f : v / l);  // (0: see above)
    }
    __syncwarp();
    sm100::cluster_sync_all();  // (a block's shared memory is read by others until here)
  }
}

__global__ void __launch_bounds__(256) decode_join_kernel(const DecodeParams p) {
  pdl_begin();
  const flare_cache_args_t& a = p.a;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.B * a.H;
  if (idx >= rows * a.D) return;
  const int64_t row = idx / a.D;
  const int d = (int)(idx - row * a.D);
  float t = -INFINITY, l = 0.0f, v = 0.0f;
  for (int s = 0; s < p.splits; ++s) t = fmaxf(t, p.part[(s * rows + row) * (a.D + 2) + a.D]);
  const float frame = t == -INFINITY ? 0.0f : t;
  for (int s = 0; s < p.splits; ++s) {
    const float* in = p.part + (s * rows + row) * (a.D + 2);
    const float f = exp2f(in[a.D] - frame);
    l = fmaf(in[a.D + 1], f, l);
    v = fmaf(in[d], f, v);
  }
  store1(a.y, a.dtype, idx, l == 0.0f ? 0.0f : v / l);  // (0: an idle row, or no score above -infinity)
}

int check_cache(const flare_cache_args_t* args, bool decode) {
  if (args == nullptr) return FLARE_ERR_BAD_POINTER;
  const flare_cache_args_t& a = *args;
  if (a.B <= 0 || a.J <= 0 || a.D <= 0 || a.L <= 0 || (decode ? a.H <= 0 || a.H % a.J : a.N <= 0)) return FLARE_ERR_BAD_SHAPE;
  if (a.D % 8 || a.D > 128 || a.L > INT_MAX - 8192 || a.B > 65535) return FLARE_ERR_UNSUPPORTED;
  if (a.dtype != FLARE_BF16 && a.dtype != FLARE_F16) return FLARE_ERR_BAD_DTYPE;
  if (!strides_fit(a.new_k, {a.new_k_stride_b, a.new_k_stride_n, a.new_k_stride_h}) || !strides_fit(a.new_v, {a.new_v_stride_b, a.new_v_stride_n, a.new_v_stride_h}) ||
      !strides_fit(a.k_cache, {a.k_stride_b, a.k_stride_n, a.k_stride_h}) || !strides_fit(a.v_cache, {a.v_stride_b, a.v_stride_n, a.v_stride_h}))
    return FLARE_ERR_BAD_POINTER;
  if (!decode) return FLARE_OK;
  if (bad_scores(a.scale, a.cap, a.window)) return FLARE_ERR_BAD_CONFIG;
  if (!strides_fit(a.q, {a.q_stride_b, a.q_stride_h}) || a.y == nullptr || a.cached == nullptr) return FLARE_ERR_BAD_POINTER;
  return FLARE_OK;
}

// Four blocks for every SM, of 64 keys at least: a block's warps then have 32 KB on their way.
DecodeParams plan_decode(const flare_cache_args_t& a) {
  DecodeParams p;
  p.a = a;
  p.part = nullptr;
  p.head_groups = (a.H / a.J + kHeads - 1) / kHeads;
  const int64_t blocks = (int64_t)a.B * a.J * p.head_groups;
  const int sight = a.window > 0 && a.window < a.L ? a.window : a.L;
  int64_t splits = ((int64_t)sm_count() * 4 + blocks - 1) / blocks;
  if (splits > (sight + 63) / 64) splits = (sight + 63) / 64;
  p.splits = (int)splits;
  // A cluster saves the second launch (B=1 H=8 D=64 L=512: 8.5 us, with it 11.3), but its blocks come and go together: where a grid takes
  // several rounds of two blocks per SM, that costs more (B=32 H=32 J=8 D=128 L=4096, rows of different lengths: 97 us, apart 87).
  p.cluster = splits > 1 && splits <= kCluster && splits * blocks <= 2 * (int64_t)sm_count();
  return p;
}

}  // namespace
}  // namespace attn
}  // namespace flare

using namespace flare;
using namespace flare::attn;

extern "C" {

size_t flare_attention_plan_bytes(const flare_attention_args_t* args) {
  if (args == nullptr || args->B <= 0 || args->Nq <= 0 || args->Nk <= 0) return 0;
  return layout(*args, false).plan_bytes;
}
size_t flare_attention_forward_workspace_bytes(const flare_attention_args_t* args) {
  if (args == nullptr || args->B <= 0 || args->Nq <= 0 || args->Nk <= 0) return 0;
  return layout(*args, false).bytes;
}
size_t flare_attention_backward_workspace_bytes(const flare_attention_args_t* args) {
  if (args == nullptr || args->B <= 0 || args->Nq <= 0 || args->Nk <= 0 || args->H <= 0 || args->J <= 0) return 0;
  return layout(*args, true).bytes;
}

int flare_attention_forward(const flare_attention_args_t* args, flare_stream_t stream) {
  if (const int rc = check(args)) return rc;
  const flare_attention_args_t& a = *args;
  const Layout l = layout(a, false);
  if (!workspace_fits(a, l)) return FLARE_ERR_WORKSPACE;
  AttnParams p;
  if (const int rc = begin(a, l, p, false, stream)) return rc;
  return launch_forward_tc(a, p, stream);
}

int flare_attention_backward(const flare_attention_args_t* args, flare_stream_t stream) {
  if (const int rc = check(args)) return rc;
  const flare_attention_args_t& a = *args;
  if (a.cached != nullptr || a.lengths != nullptr) return FLARE_ERR_BAD_CONFIG;
  if (!strides_fit(a.dy, {a.dy_stride_b, a.dy_stride_n, a.dy_stride_h}) || !strides_fit(a.dq, {}) || !strides_fit(a.dk, {}) ||
      !strides_fit(a.dv, {}) || !strides_fit(a.lse, {}))
    return FLARE_ERR_BAD_POINTER;
  const Layout l = layout(a, true);
  if (!workspace_fits(a, l)) return FLARE_ERR_WORKSPACE;
  AttnParams p;
  if (const int rc = begin(a, l, p, true, stream)) return rc;
  uint8_t* const ws = reinterpret_cast<uint8_t*>(a.workspace);
  const auto floats = [&](size_t at) { return reinterpret_cast<float*>(ws + at); };
  p.delta = floats(l.delta);
  p.dy_norm = floats(l.dy_norm);
  p.largest_norms = floats(l.largest_norms);
  p.lse_lifted = floats(l.lse_lifted);
  const int lanes = a.D <= 64 ? 8 : 16;
  const int64_t blocks = ((int64_t)l.Nqp * a.H * lanes + 255) / 256;
  if (blocks * (256 / lanes) > UINT_MAX - 256 || (int64_t)a.B * a.J > INT_MAX) return FLARE_ERR_UNSUPPORTED;
  {
    LaunchTimer timer("attention_delta_kernel", stream);
    const dim3 grid((unsigned)blocks, (unsigned)(a.B < kRows ? a.B : kRows), (unsigned)((a.B + (int64_t)kRows - 1) / kRows));
    DeltaParams d;
    d.p = p;
    d.q = a.q; d.k = a.k; d.v = a.v; d.dy = a.dy;
    d.q_b = a.q_stride_b; d.q_n = a.q_stride_n; d.q_h = a.q_stride_h;
    d.k_b = a.k_stride_b; d.k_n = a.k_stride_n; d.k_h = a.k_stride_h;
    d.v_b = a.v_stride_b; d.v_n = a.v_stride_n; d.v_h = a.v_stride_h;
    d.dy_b = a.dy_stride_b; d.dy_n = a.dy_stride_n; d.dy_h = a.dy_stride_h;
    d.delta = floats(l.delta);
    d.dy_norm = floats(l.dy_norm);
    d.v_norm = floats(l.v_norm);
    auto* const kernel = a.dtype == FLARE_F16 ? (lanes == 8 ? delta_kernel<__half, 8> : delta_kernel<__half, 16>)
                                              : (lanes == 8 ? delta_kernel<__nv_bfloat16, 8> : delta_kernel<__nv_bfloat16, 16>);
    FLARE_CUDA_CHECK(launch_pdl(kernel, grid, dim3(256), 0, stream, d));
  }
  if (a.dtype == FLARE_F16) {
    LaunchTimer timer("attention_largest_norms_kernel", stream);
    FLARE_CUDA_CHECK(launch_pdl(largest_norms_kernel, dim3((unsigned)(a.J * a.B)), dim3(1024), 0, stream, p.dy_norm, (const float*)floats(l.v_norm),
                                (const float*)a.lse, floats(l.lse_lifted), floats(l.largest_norms), a.H / a.J, l.Nqp));
  }
  return launch_backward_tc(a, p, stream);
}

int flare_attention_append(const flare_cache_args_t* args, flare_stream_t stream) {
  if (const int rc = check_cache(args, false)) return rc;
  const flare_cache_args_t& a = *args;
  const int64_t blocks = ((int64_t)a.B * a.N * a.J * (a.D >> 3) + 255) / 256;
  if (blocks > INT_MAX) return FLARE_ERR_UNSUPPORTED;
  LaunchTimer timer("attention_append_kernel", stream);
  FLARE_CUDA_CHECK(launch_pdl(append_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a));
  return FLARE_OK;
}

size_t flare_attention_decode_workspace_bytes(const flare_cache_args_t* args) {
  if (check_cache(args, true)) return 0;
  const DecodeParams p = plan_decode(*args);
  return p.splits > 1 && !p.cluster ? (size_t)p.splits * args->B * args->H * (args->D + 2) * sizeof(float) : 0;
}

int flare_attention_decode(const flare_cache_args_t* args, flare_stream_t stream) {
  if (const int rc = check_cache(args, true)) return rc;
  const flare_cache_args_t& a = *args;
  DecodeParams p = plan_decode(a);
  if (p.splits > 1 && !p.cluster) {
    if (a.workspace == nullptr || a.workspace_bytes < flare_attention_decode_workspace_bytes(args)) return FLARE_ERR_WORKSPACE;
    p.part = reinterpret_cast<float*>(a.workspace);
  }
  if ((int64_t)a.J * p.head_groups > 65535) return FLARE_ERR_UNSUPPORTED;
  const bool f16 = a.dtype == FLARE_F16, eight = a.H / a.J <= 8;
  auto* const kernel = a.D <= 64 ? (eight ? (f16 ? decode_kernel<1, true, true> : decode_kernel<1, false, true>)
                                          : (f16 ? decode_kernel<1, true, false> : decode_kernel<1, false, false>))
                                 : (eight ? (f16 ? decode_kernel<2, true, true> : decode_kernel<2, false, true>)
                                          : (f16 ? decode_kernel<2, true, false> : decode_kernel<2, false, false>));
  {
    LaunchTimer timer("attention_decode_kernel", stream);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.splits, (unsigned)(a.J * p.head_groups), (unsigned)a.B);
    cfg.blockDim = dim3(32 * kDecodeWarps);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.cluster ? 2 : 1;
    FLARE_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  }
  if (p.part == nullptr) return FLARE_OK;
  const int64_t blocks = ((int64_t)a.B * a.H * a.D + 255) / 256;
  if (blocks > INT_MAX) return FLARE_ERR_UNSUPPORTED;
  LaunchTimer timer("attention_decode_join_kernel", stream);
  FLARE_CUDA_CHECK(launch_pdl(decode_join_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p));
  return FLARE_OK;
}

}  // extern "C"
