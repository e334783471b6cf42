// Short causal convolution, one filter of W taps per channel: forward, backward, one token.
//
// All three are bound by memory: 2 W operations (6 W with gradients) on 4 (6) bytes.  A thread owns a few neighbouring channels and
// walks a run of tokens with the last W - 1 rows in registers, so every row is read once but for the W - 1 in front of a run (and behind
// it, backward); a warp reads 256 contiguous bytes of a row, eight rows in flight while eight are worked on.  The four warps of a block
// take runs behind one another.  A token's taps end at its document's first token: `reach` counts the tokens in front of it that
// belong to the same run of ids, and is the same for a whole warp.  What is issued weighs as much as the bytes (half of all slots, in both
// directions), so products are packed in pairs and whole groups of rows go without a look at every row.
#include <algorithm>

#include "mixer_common.cuh"

namespace flare {
namespace {

using namespace mixer;
using namespace sm100;

constexpr int kWarps = 4;
// Channels of a thread and blocks of an SM.  B200, B=4 N=4096 C=4096 W=4 bf16, forward: (4, 6) 55.5 us = 4.8 TB/s, (8, 4) 58.4, (8, 3) 68, (8, 5) 81;
// backward: (4, 3) 100 us = 4.0 TB/s, (8, 1) 110, (4, 4) with half the rows ahead 117.
constexpr int kForwardChannels = 4, kForwardBlocks = 6, kBackwardChannels = 4, kBackwardBlocks = 3;
constexpr int kAhead = 8;  // rows on their way while as many are worked on

struct ConvParams {
  flare_conv_args_t a;
  int run;        // tokens of a warp's run
  int blocks_n;   // blocks along a row's tokens
  int wide;       // rows of x, y, dy, dx, state in 16-byte pieces
  int wide_weights;
  int columns;    // blocks along the channels
  float* partial; // [B * blocks_n][C * W + C]
};

// What a walk carries from token to token: the ids in front of it and how many of them belong to its document.
template <int W, bool DOCS>
struct Reach {
  const int32_t* ids;  // of the row
  int last, reach;
  __device__ __forceinline__ void start(const int32_t* row, int t) {
    ids = row;
    reach = 0;
    last = -1;
    if (!DOCS) return;
    last = t > 0 ? ids[t - 1] : -1;
    for (int j = 2; j < W && t - j >= 0 && ids[t - j] == last; ++j) ++reach;
  }
  // the number of tokens in front of t that its taps may see; the id of t in `id`
  __device__ __forceinline__ int step(int t, int& id) {
    id = 0;
    if (!DOCS) return W - 1;
    id = ids[t];
    reach = t > 0 && id == last ? min(reach + 1, W - 1) : 0;
    last = id;
    return reach;
  }
};

// V channels as pairs: the packed operations halve what is issued
template <int V>
struct Pairs {
  uint64_t v[V / 2];
};
template <int V>
__device__ __forceinline__ Pairs<V> zero_pairs() {
  Pairs<V> p;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) p.v[i] = 0;
  return p;
}
template <typename T, int V>
__device__ __forceinline__ Pairs<V> to_pairs(const Raw<T, V>& r) {
  float f[V];
  unpack<T, V>(r, f);
  Pairs<V> p;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) p.v[i] = f2_pack(f[2 * i], f[2 * i + 1]);
  return p;
}
template <int V>
__device__ __forceinline__ void from_pairs(const Pairs<V>& p, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) f2_unpack(p.v[i], f[2 * i], f[2 * i + 1]);
}
template <int V>
__device__ __forceinline__ void fma_pairs(const Pairs<V>& a, const Pairs<V>& b, Pairs<V>& c) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) c.v[i] = f2_fma(a.v[i], b.v[i], c.v[i]);
}

// 1 / (1 + exp(-v)): exp2 and the reciprocal are off by a few units in the last place
__device__ __forceinline__ uint64_t sigmoid_pair(uint64_t v) {
  const float k = -1.4426950408889634f;
  float lo, hi;
  f2_unpack(f2_mul(v, f2_pack(k, k)), lo, hi);
  f2_unpack(f2_add(f2_pack(ex2_approx(lo), ex2_approx(hi)), f2_pack(1.0f, 1.0f)), lo, hi);
  return f2_pack(rcp_approx(lo), rcp_approx(hi));
}
template <int V>
__device__ __forceinline__ void silu_pairs(Pairs<V>& p) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) p.v[i] = f2_mul(p.v[i], sigmoid_pair(p.v[i]));
}

// The filters of neighbouring channels lie behind one another: V W elements, in 16-byte pieces where they are aligned.
template <int W, int V>
__device__ __forceinline__ void load_weights(const flare_conv_args_t& a, int c, int count, bool wide, Pairs<V> (&w)[W], Pairs<V>& bias) {
  float f[V * W], g[V];
  if (wide && a.weight_dtype == FLARE_F32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.weight) + (int64_t)c * W);
#pragma unroll
    for (int i = 0; i < V * W / 4; ++i) {
      const float4 v = p[i];
      f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V * W; ++i) f[i] = i < count * W ? load1(a.weight, a.weight_dtype, (int64_t)c * W + i) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) g[i] = i < count && a.bias != nullptr ? load1(a.bias, a.weight_dtype, c + i) : 0.0f;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j].v[i] = f2_pack(f[2 * i * W + j], f[(2 * i + 1) * W + j]);
    bias.v[i] = f2_pack(g[2 * i], g[2 * i + 1]);
  }
}

// row t of the row's tokens behind the carried state: t in [-(W - 1), N)
template <typename T, int W, int V>
__device__ __forceinline__ Raw<T, V> row_at(const flare_conv_args_t& a, const T* x, const T* state, int t, int end, int count, bool wide) {
  if (t >= 0) return load_raw<T, V>(x + (int64_t)t * a.x_stride_n, t < end ? count : 0, wide);
  return load_raw<T, V>(state + (int64_t)(W - 1 + t) * a.C, state != nullptr && t >= 1 - W ? count : 0, wide);
}

// x is summed newest tap first, bias in front: v = bias + w[W-1] x[t] + ... + w[0] x[t-W+1]; past[j]: token t - j
template <int W, int V>
__device__ __forceinline__ Pairs<V> taps(const Pairs<V> (&w)[W], const Pairs<V>& bias, const Pairs<V> (&past)[W], int reach) {
  Pairs<V> v = bias;
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (j <= reach) fma_pairs(w[W - 1 - j], past[j], v);
  return v;
}

// (WIDE: every thread has all of its channels, in one aligned piece: 16 bytes, or 8 for 16-bit types)
template <typename T, int W, bool DOCS, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps, kForwardBlocks) conv_forward_kernel(const ConvParams p) {
  constexpr int V = kForwardChannels;
  pdl_begin();
  const flare_conv_args_t& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.blocks_n, nb = blockIdx.x % p.blocks_n;
  const int c = (blockIdx.y * 32 + lane) * V;
  if (c >= a.C) return;
  const int count = WIDE ? V : min(V, a.C - c);
  const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)b * a.x_stride_b + c;
  const T* state = a.state_in != nullptr ? reinterpret_cast<const T*>(a.state_in) + (int64_t)b * (W - 1) * a.C + c : nullptr;
  T* y = reinterpret_cast<T*>(a.y) + (int64_t)b * a.N * a.C + c;
  const int len = a.lengths != nullptr ? max(0, min(a.N, a.lengths[b])) : a.N;
  if (nb == 0 && warp == 0 && a.state_out != nullptr) {
    T* out = reinterpret_cast<T*>(a.state_out) + (int64_t)b * (W - 1) * a.C + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      float v[V];
      unpack<T, V>(row_at<T, W, V>(a, x, state, len - (W - 1) + j, len, count, WIDE), v);
      store_all<T, V>(out + (int64_t)j * a.C, v, count, WIDE);
    }
  }
  const int t0 = (nb * kWarps + warp) * p.run, t1 = min(a.N, t0 + p.run);
  if (t0 >= t1) return;
  Raw<T, V> rows[kAhead], next[kAhead];
  const T* from = x + (int64_t)t0 * a.x_stride_n;
  const auto fetch = [&](int t) {  // the next rows, in order; whole groups need no look at every row
    if (t + kAhead <= t1) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k, from += a.x_stride_n) next[k] = load_raw<T, V>(from, count, WIDE);
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k, from += a.x_stride_n) next[k] = load_raw<T, V>(from, t + k < t1 ? count : 0, WIDE);
    }
  };
  fetch(t0);
  Pairs<V> w[W], bias, past[W];
  load_weights<W, V>(a, c, count, WIDE && p.wide_weights, w, bias);
  Reach<W, DOCS> docs;
  docs.start(DOCS ? a.documents + (int64_t)b * a.N : nullptr, t0);
#pragma unroll
  for (int j = 1; j < W; ++j) past[j - 1] = to_pairs<T, V>(row_at<T, W, V>(a, x, state, t0 - j, a.N, count, WIDE));
  y += (int64_t)t0 * a.C;
  const bool silu = a.activation == FLARE_SILU;
  const auto group = [&](auto whole, int t) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
#pragma unroll
      for (int j = W - 1; j > 0; --j) past[j] = past[j - 1];
      past[0] = to_pairs<T, V>(rows[k]);
      if (decltype(whole)::value || t + k < t1) {
        int id;
        const int reach = docs.step(t + k, id);
        Pairs<V> s = zero_pairs<V>();
        if ((!DOCS || id >= 0) && (decltype(whole)::value || t + k < len)) {
          s = taps<W, V>(w, bias, past, reach);
          if (silu) silu_pairs(s);
        }
        float v[V];
        from_pairs(s, v);
        store_all<T, V>(y, v, count, WIDE);
        y += a.C;
      }
    }
  };
#pragma unroll 1
  for (int t = t0; t < t1; t += kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) rows[k] = next[k];
    if (t + kAhead < t1) fetch(t + kAhead);
    if (t + kAhead <= min(t1, len)) group(std::true_type(), t);
    else group(std::false_type(), t);
  }
}

// g[t] = dy[t] act'(pre[t]); dx[t] = sum_j w[W-1-j] g[t+j]; dw[W-1-j] = sum_t g[t] x[t-j]; dbias = sum g.
// A run computes the g of the W - 1 tokens behind it as well (their rows are read twice), and adds only its own tokens' to
// the weights' gradients: one partial sum per block, added up in order afterwards.
template <typename T, int W, bool DOCS, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps, kBackwardBlocks) conv_backward_kernel(const ConvParams p) {
  constexpr int V = kBackwardChannels;
  pdl_begin();
  const flare_conv_args_t& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.blocks_n, nb = blockIdx.x % p.blocks_n;
  const int c = (blockIdx.y * 32 + lane) * V, count = c >= a.C ? 0 : WIDE ? V : min(V, a.C - c);
  const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)b * a.x_stride_b + c;
  const T* dy = reinterpret_cast<const T*>(a.dy) + (int64_t)b * a.dy_stride_b + c;
  T* dx = reinterpret_cast<T*>(a.dx) + (int64_t)b * a.N * a.C + c;
  const int t0 = (nb * kWarps + warp) * p.run, t1 = min(a.N, t0 + p.run), t2 = min(a.N, t1 + W - 1);
  Pairs<V> dw[W + 1];  // (the last one: bias)
#pragma unroll
  for (int j = 0; j <= W; ++j) dw[j] = zero_pairs<V>();
  if (t0 < t1 && count > 0) {
    Pairs<V> w[W], bias, past[W], acc[W];  // acc[j]: gradient of token t - j, as far as it is known
    load_weights<W, V>(a, c, count, WIDE && p.wide_weights, w, bias);
    Reach<W, DOCS> docs;
    docs.start(DOCS ? a.documents + (int64_t)b * a.N : nullptr, t0);
#pragma unroll
    for (int j = 1; j < W; ++j) {
      past[j - 1] = to_pairs<T, V>(row_at<T, W, V>(a, x, nullptr, t0 - j, a.N, count, WIDE));
      acc[j - 1] = zero_pairs<V>();
    }
    const int end = t1 + W - 1;  // the last run's gradients leave W - 1 steps behind its last token
    Raw<T, V> rows[kAhead], drows[kAhead], next[kAhead], dnext[kAhead];
    const T *from = x + (int64_t)t0 * a.x_stride_n, *dfrom = dy + (int64_t)t0 * a.dy_stride_n;
    const auto fetch = [&](int t) {
      if (t + kAhead <= t2) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k, from += a.x_stride_n, dfrom += a.dy_stride_n) {
          next[k] = load_raw<T, V>(from, count, WIDE);
          dnext[k] = load_raw<T, V>(dfrom, count, WIDE);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kAhead; ++k, from += a.x_stride_n, dfrom += a.dy_stride_n) {
          next[k] = load_raw<T, V>(from, t + k < t2 ? count : 0, WIDE);
          dnext[k] = load_raw<T, V>(dfrom, t + k < t2 ? count : 0, WIDE);
        }
      }
    };
    fetch(t0);
    dx += (int64_t)t0 * a.C;
    const bool silu = a.activation == FLARE_SILU;
    const auto group = [&](auto whole, int t) {  // (whole: own tokens all)
      constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
#pragma unroll
        for (int j = W - 1; j > 0; --j) {
          past[j] = past[j - 1];
          acc[j] = acc[j - 1];
        }
        past[0] = to_pairs<T, V>(rows[k]);
        acc[0] = zero_pairs<V>();
        int id = -1, reach = 0;
        if (WHOLE || t + k < t2) reach = docs.step(t + k, id);
        if (id >= 0) {
          Pairs<V> g = to_pairs<T, V>(drows[k]);
          if (silu) {
            const Pairs<V> v = taps<W, V>(w, bias, past, reach);
            const uint64_t one = f2_pack(1.0f, 1.0f), minus = f2_pack(-1.0f, -1.0f);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              const uint64_t r = sigmoid_pair(v.v[i]);
              g.v[i] = f2_mul(f2_mul(g.v[i], r), f2_fma(v.v[i], f2_fma(r, minus, one), one));
            }
          }
#pragma unroll
          for (int j = 0; j < W; ++j)
            if (j <= reach) fma_pairs<V>(w[W - 1 - j], g, acc[j]);
          if (WHOLE || t + k < t1) {
#pragma unroll
            for (int j = 0; j < W; ++j)
              if (j <= reach) fma_pairs<V>(g, past[j], dw[W - 1 - j]);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) dw[W].v[i] = f2_add(dw[W].v[i], g.v[i]);
          }
        }
        const int done = t + k - (W - 1);
        if (done >= t0 && (WHOLE || done < t1)) {
          float v[V];
          from_pairs(acc[W - 1], v);
          store_all<T, V>(dx, v, count, WIDE);
          dx += a.C;
        }
      }
    };
#pragma unroll 1
    for (int t = t0; t < end; t += kAhead) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        rows[k] = next[k];
        drows[k] = dnext[k];
      }
      if (t + kAhead < end) fetch(t + kAhead);
      if (t + kAhead <= t1) group(std::true_type(), t);
      else group(std::false_type(), t);
    }
  }
  // the block's four runs, in their order
  __shared__ float sums[kWarps - 1][32][V * (W + 1) + 1];
  if (warp > 0) {
#pragma unroll
    for (int j = 0; j <= W; ++j) {
      float v[V];
      from_pairs(dw[j], v);
#pragma unroll
      for (int i = 0; i < V; ++i) sums[warp - 1][lane][j * V + i] = v[i];
    }
  }
  __syncthreads();
  if (warp > 0) return;
  float* out = p.partial + (int64_t)blockIdx.x * a.C * (W + 1);
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    float v[V];
    from_pairs(dw[j], v);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < count) {
#pragma unroll
        for (int q = 0; q < kWarps - 1; ++q) v[i] += sums[q][lane][j * V + i];
        out[j < W ? (int64_t)(c + i) * W + j : (int64_t)a.C * W + c + i] = v[i];
      }
  }
}

// One token: the state's rows move up by one, the token's is the last.
template <typename T, int W>
__global__ void __launch_bounds__(128) conv_decode_kernel(const ConvParams p) {
  constexpr int V = 8;
  pdl_begin();
  const flare_conv_args_t& a = p.a;
  const int groups = (a.C + V - 1) / V;
  const int64_t idx = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (idx >= (int64_t)a.B * groups) return;
  const int64_t b = idx / groups;
  const int c = (int)(idx - b * groups) * V, count = min(8, a.C - c);
  const bool wide = p.wide != 0;
  T* state = reinterpret_cast<T*>(a.state_out) + b * (W - 1) * a.C + c;
  Raw<T, V> rows[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) rows[j] = load_raw<T, V>(state + (int64_t)j * a.C, count, wide);
  rows[W - 1] = load_raw<T, V>(reinterpret_cast<const T*>(a.x) + b * a.x_stride_b + c, count, wide);
  Pairs<V> w[W], bias, past[W];
  float v[V];
  load_weights<W, V>(a, c, count, wide && p.wide_weights, w, bias);
#pragma unroll
  for (int j = 0; j < W; ++j) past[j] = to_pairs<T, V>(rows[W - 1 - j]);
  Pairs<V> s = taps<W, V>(w, bias, past, W - 1);
  if (a.activation == FLARE_SILU) silu_pairs(s);
  from_pairs(s, v);
  store_all<T, V>(reinterpret_cast<T*>(a.y) + b * a.C + c, v, count, wide);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    from_pairs(past[W - 2 - j], v);
    store_all<T, V>(state + (int64_t)j * a.C, v, count, wide);
  }
}

// Runs as long as fill the SMs' places in whole rounds (what is read again in front of a run, and its weights, count for less the longer
// it is), up to 128 tokens; at least 8, where that leaves SMs idle.
void plan(ConvParams& p, const flare_conv_args_t& a, int channels, int places) {
  p.a = a;
  p.columns = (a.C + 32 * channels - 1) / (32 * channels);
  const int64_t lanes = (int64_t)a.B * p.columns;
  for (int64_t rounds = 1;; ++rounds) {
    const int64_t blocks = std::max<int64_t>(1, (int64_t)sm_count() * places * rounds / lanes) * kWarps;
    p.run = (int)std::max<int64_t>(8, ((a.N + blocks - 1) / blocks + 7) / 8 * 8);
    if (p.run <= 128) break;
  }
  const int per = p.run * kWarps;
  p.blocks_n = (a.N + per - 1) / per;
  p.partial = nullptr;
}

int check(const flare_conv_args_t* a) {
  if (a == nullptr) return FLARE_ERR_BAD_POINTER;
  if (a->B <= 0 || a->N <= 0 || a->C <= 0) return FLARE_ERR_BAD_SHAPE;
  if (a->W < 2 || a->W > 4) return FLARE_ERR_UNSUPPORTED;
  if (a->C > 0x7fffffff - 256 || (a->C + 127) / 128 > 65535) return FLARE_ERR_UNSUPPORTED;  // (what grid.y holds)
  if ((int64_t)a->B * ((a->N + 31) / 32) > 0x7fffffff || (int64_t)a->N > 0x7fffffff - 1024) return FLARE_ERR_UNSUPPORTED;
  if (a->dtype < 0 || a->dtype > 2 || a->weight_dtype < 0 || a->weight_dtype > 2) return FLARE_ERR_BAD_DTYPE;
  if (a->activation != FLARE_IDENTITY && a->activation != FLARE_SILU) return FLARE_ERR_BAD_CONFIG;
  if (a->x == nullptr || a->weight == nullptr) return FLARE_ERR_BAD_POINTER;
  return FLARE_OK;
}

template <typename F>
int by_type(int dtype, int W, F f) {
  const auto taps_of = [&](auto t) {
    using T = decltype(t);
    if (W == 2) return f(t, std::integral_constant<int, 2>());
    if (W == 3) return f(t, std::integral_constant<int, 3>());
    return f(T(), std::integral_constant<int, 4>());
  };
  if (dtype == FLARE_F32) return taps_of(float());
  if (dtype == FLARE_BF16) return taps_of(__nv_bfloat16());
  return taps_of(__half());
}

}  // namespace

namespace mixer {
namespace {
__global__ void __launch_bounds__(256) sum_parts_kernel(const __grid_constant__ SumList list) {
  pdl_begin();
  const SumList::Part& s = list.part[blockIdx.y];
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  __shared__ float sums[8][32];
  for (int64_t i0 = (int64_t)blockIdx.x * 32; i0 < s.count; i0 += (int64_t)gridDim.x * 32) {
    const int64_t i = i0 + col;
    float v = 0.0f;
    if (i < s.count)
      for (int p = row; p < s.parts; p += 8) v += s.in[p * s.stride + i];
    __syncthreads();
    sums[row][col] = v;
    __syncthreads();
    if (row == 0 && i < s.count) {
#pragma unroll
      for (int q = 1; q < 8; ++q) v += sums[q][col];
      store1(s.out, s.dtype, i, v);
    }
  }
}
}  // namespace

int launch_sum_parts(const SumList& list, int n, cudaStream_t stream) {
  int64_t most = 0;
  for (int i = 0; i < n; ++i) most = list.part[i].count > most ? list.part[i].count : most;
  int64_t blocks = (most + 31) / 32;
  if (blocks > (int64_t)sm_count() * 64) blocks = (int64_t)sm_count() * 64;
  if (blocks <= 0) return FLARE_OK;
  LaunchTimer timer("sum_parts_kernel", stream);
  FLARE_CUDA_CHECK(launch_pdl(sum_parts_kernel, dim3((unsigned)blocks, n), dim3(256), 0, stream, list));
  return FLARE_OK;
}
}  // namespace mixer
}  // namespace flare

using namespace flare;

extern "C" {

int flare_conv_forward(const flare_conv_args_t* args, flare_stream_t stream) {
  if (const int rc = check(args)) return rc;
  const flare_conv_args_t& a = *args;
  if (a.y == nullptr || (a.state_out != nullptr && a.state_out == a.state_in)) return FLARE_ERR_BAD_POINTER;
  if (a.documents != nullptr && (a.state_in != nullptr || a.state_out != nullptr)) return FLARE_ERR_BAD_CONFIG;
  ConvParams p;
  plan(p, a, kForwardChannels, kForwardBlocks);
  p.wide_weights = (reinterpret_cast<uintptr_t>(a.weight) & 15u) == 0;
  p.wide = a.C % 8 == 0 && rows_wide(a.x, a.dtype, {a.x_stride_b, a.x_stride_n}) && rows_wide(a.y, a.dtype, {}) &&
           rows_wide(a.state_in, a.dtype, {}) && rows_wide(a.state_out, a.dtype, {});
  const dim3 grid((unsigned)(a.B * (int64_t)p.blocks_n), (unsigned)p.columns);
  return by_type(a.dtype, a.W, [&](auto t, auto w) -> int {
    LaunchTimer timer("conv_forward_kernel", stream);
    using T = decltype(t);
    constexpr int W = decltype(w)::value;
    auto* const kernel = a.documents != nullptr ? (p.wide ? conv_forward_kernel<T, W, true, true> : conv_forward_kernel<T, W, true, false>)
                                                : (p.wide ? conv_forward_kernel<T, W, false, true> : conv_forward_kernel<T, W, false, false>);
    FLARE_CUDA_CHECK(launch_pdl(kernel, grid, dim3(32 * kWarps), 0, stream, p));
    return FLARE_OK;
  });
}

size_t flare_conv_backward_workspace_bytes(const flare_conv_args_t* args) {
  ConvParams p;
  if (args == nullptr || args->B <= 0 || args->N <= 0 || args->C <= 0 || args->W < 2 || args->W > 4) return 0;
  plan(p, *args, kBackwardChannels, kBackwardBlocks);
  return (size_t)args->B * p.blocks_n * args->C * (args->W + 1) * sizeof(float);
}

int flare_conv_backward(const flare_conv_args_t* args, flare_stream_t stream) {
  if (const int rc = check(args)) return rc;
  const flare_conv_args_t& a = *args;
  if (a.dy == nullptr || a.dx == nullptr || a.dweight == nullptr) return FLARE_ERR_BAD_POINTER;
  if (a.state_in != nullptr || a.state_out != nullptr || a.lengths != nullptr) return FLARE_ERR_BAD_CONFIG;
  if (a.workspace == nullptr || a.workspace_bytes < flare_conv_backward_workspace_bytes(args)) return FLARE_ERR_WORKSPACE;
  ConvParams p;
  plan(p, a, kBackwardChannels, kBackwardBlocks);
  p.partial = reinterpret_cast<float*>(a.workspace);
  p.wide_weights = (reinterpret_cast<uintptr_t>(a.weight) & 15u) == 0;
  p.wide = a.C % 8 == 0 && rows_wide(a.x, a.dtype, {a.x_stride_b, a.x_stride_n}) &&
           rows_wide(a.dy, a.dtype, {a.dy_stride_b, a.dy_stride_n}) && rows_wide(a.dx, a.dtype, {});
  const int parts = a.B * p.blocks_n;
  const dim3 grid((unsigned)parts, (unsigned)p.columns);
  const int rc = by_type(a.dtype, a.W, [&](auto t, auto w) -> int {
    LaunchTimer timer("conv_backward_kernel", stream);
    using T = decltype(t);
    constexpr int W = decltype(w)::value;
    auto* const kernel = a.documents != nullptr ? (p.wide ? conv_backward_kernel<T, W, true, true> : conv_backward_kernel<T, W, true, false>)
                                                : (p.wide ? conv_backward_kernel<T, W, false, true> : conv_backward_kernel<T, W, false, false>);
    FLARE_CUDA_CHECK(launch_pdl(kernel, grid, dim3(32 * kWarps), 0, stream, p));
    return FLARE_OK;
  });
  if (rc) return rc;
  const int64_t stride = (int64_t)a.C * (a.W + 1);
  SumList list = {};
  list.part[0] = {p.partial, a.dweight, (int64_t)a.C * a.W, stride, parts, a.weight_dtype};
  list.part[1] = {p.partial + (int64_t)a.C * a.W, a.dbias, a.C, stride, parts, a.weight_dtype};
  return launch_sum_parts(list, a.dbias != nullptr ? 2 : 1, stream);
}

int flare_conv_decode(const flare_conv_args_t* args, flare_stream_t stream) {
  if (args == nullptr) return FLARE_ERR_BAD_POINTER;
  flare_conv_args_t a = *args;
  a.N = 1;
  if (const int rc = check(&a)) return rc;
  if (a.y == nullptr || a.state_out == nullptr) return FLARE_ERR_BAD_POINTER;
  ConvParams p;
  p.a = a;
  p.run = p.blocks_n = 0;
  p.partial = nullptr;
  p.wide_weights = (reinterpret_cast<uintptr_t>(a.weight) & 15u) == 0;
  p.wide = a.C % 8 == 0 && rows_wide(a.x, a.dtype, {a.x_stride_b}) && rows_wide(a.y, a.dtype, {}) && rows_wide(a.state_out, a.dtype, {});
  const int64_t blocks = ((int64_t)a.B * ((a.C + 7) / 8) + 127) / 128;
  if (blocks > 0x7fffffff) return FLARE_ERR_UNSUPPORTED;
  return by_type(a.dtype, a.W, [&](auto t, auto w) -> int {
    LaunchTimer timer("conv_decode_kernel", stream);
    FLARE_CUDA_CHECK(launch_pdl(conv_decode_kernel<decltype(t), decltype(w)::value>, dim3((unsigned)blocks), dim3(128), 0, stream, p));
    return FLARE_OK;
  });
}

size_t flare_mixers_abi_sizeof(int which) {
  switch (which) {
    case 0: return sizeof(flare_conv_args_t);
    case 1: return sizeof(flare_scan_args_t);
    case 2: return sizeof(flare_attention_args_t);
    case 3: return sizeof(flare_cache_args_t);
    default: return 0;
  }
}

}  // extern "C"
