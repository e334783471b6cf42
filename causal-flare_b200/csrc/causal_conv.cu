// Short causal convolution, one filter of W taps per channel: forward, backward, one token.
//
// All three are bound by memory: 2 W operations (6 W with gradients) on 4 (10) bytes.  A thread owns eight channels (16
// bytes of a row) and walks a run of tokens with the last W - 1 rows in registers, so every row is read once but for the
// W - 1 in front of a run; a warp reads 512 contiguous bytes of a row, eight (backward: four) rows in flight.  The four warps of a block
// take runs behind one another.  A token's taps end at its document's first token: `reach` counts the tokens in front of it
// that belong to the same run of ids, and is the same for a whole warp.
#include "mixer_common.cuh"

namespace flare {
namespace {

using namespace mixer;
using namespace sm100;

constexpr int kWarps = 4;

struct ConvParams {
  flare_conv_args_t a;
  int run;        // tokens of a warp's run
  int blocks_n;   // blocks along a row's tokens
  int wide;       // rows of x, y, dy, dx, state in 16-byte pieces
  float* partial; // [B * blocks_n][C * W + C]
};

__device__ __forceinline__ float weight_at(const flare_conv_args_t& a, int64_t i) { return load1(a.weight, a.weight_dtype, i); }

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

// eight channels as four pairs: the packed operations halve what is issued
struct Pairs {
  uint64_t v[4];
};
__device__ __forceinline__ Pairs zero_pairs() { return Pairs{{0, 0, 0, 0}}; }
template <typename T>
__device__ __forceinline__ Pairs to_pairs(const Raw8<T>& r) {
  float f[8];
  unpack8(r, f);
  Pairs p;
#pragma unroll
  for (int i = 0; i < 4; ++i) p.v[i] = f2_pack(f[2 * i], f[2 * i + 1]);
  return p;
}
__device__ __forceinline__ void from_pairs(const Pairs& p, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_unpack(p.v[i], f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void fma_pairs(const Pairs& a, const Pairs& b, Pairs& c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c.v[i] = f2_fma(a.v[i], b.v[i], c.v[i]);
}

template <int W>
__device__ __forceinline__ void load_weights(const flare_conv_args_t& a, int c, int count, Pairs (&w)[W], Pairs& bias) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j)
      w[j].v[i] = f2_pack(2 * i < count ? weight_at(a, (int64_t)(c + 2 * i) * W + j) : 0.0f,
                          2 * i + 1 < count ? weight_at(a, (int64_t)(c + 2 * i + 1) * W + j) : 0.0f);
    bias.v[i] = f2_pack(2 * i < count && a.bias != nullptr ? load1(a.bias, a.weight_dtype, c + 2 * i) : 0.0f,
                        2 * i + 1 < count && a.bias != nullptr ? load1(a.bias, a.weight_dtype, c + 2 * i + 1) : 0.0f);
  }
}

// row t of the row's tokens behind the carried state: t in [-(W - 1), N)
template <typename T, int W>
__device__ __forceinline__ Raw8<T> row_at(const flare_conv_args_t& a, const T* x, const T* state, int t, int end, int count, bool wide) {
  if (t >= 0) return load_raw8<T>(x + (int64_t)t * a.x_stride_n, t < end ? count : 0, wide);
  return load_raw8<T>(state + (int64_t)(W - 1 + t) * a.C, state != nullptr && t >= 1 - W ? count : 0, wide);
}

// x is summed newest tap first, bias in front: v = bias + w[W-1] x[t] + ... + w[0] x[t-W+1]; past[j]: token t - j
template <int W>
__device__ __forceinline__ Pairs taps(const Pairs (&w)[W], const Pairs& bias, const Pairs (&past)[W], int reach) {
  Pairs v = bias;
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (j <= reach) fma_pairs(w[W - 1 - j], past[j], v);
  return v;
}

// (WIDE: every thread has eight channels and 16-byte pieces)
template <typename T, int W, bool DOCS, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps) conv_forward_kernel(const ConvParams p) {
  pdl_begin();
  const flare_conv_args_t& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.blocks_n, nb = blockIdx.x % p.blocks_n;
  const int c = (blockIdx.y * 32 + lane) * 8;
  if (c >= a.C) return;
  const int count = WIDE ? 8 : min(8, a.C - c);
  const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)b * a.x_stride_b + c;
  const T* state = a.state_in != nullptr ? reinterpret_cast<const T*>(a.state_in) + (int64_t)b * (W - 1) * a.C + c : nullptr;
  T* y = reinterpret_cast<T*>(a.y) + (int64_t)b * a.N * a.C + c;
  const int len = a.lengths != nullptr ? max(0, min(a.N, a.lengths[b])) : a.N;
  if (nb == 0 && warp == 0 && a.state_out != nullptr) {
    T* out = reinterpret_cast<T*>(a.state_out) + (int64_t)b * (W - 1) * a.C + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      float v[8];
      unpack8(row_at<T, W>(a, x, state, len - (W - 1) + j, len, count, WIDE), v);
      store8<T>(out + (int64_t)j * a.C, v, count, WIDE);
    }
  }
  const int t0 = (nb * kWarps + warp) * p.run, t1 = min(a.N, t0 + p.run);
  if (t0 >= t1) return;
  constexpr int kAhead = sizeof(T) == 4 ? 4 : 8;
  Raw8<T> rows[kAhead];
  const auto fetch = [&](int t) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) rows[k] = load_raw8<T>(x + (int64_t)(t + k) * a.x_stride_n, t + k < t1 ? count : 0, WIDE);
  };
  fetch(t0);
  Pairs w[W], bias, past[W];
  load_weights<W>(a, c, count, w, bias);
  Reach<W, DOCS> docs;
  docs.start(DOCS ? a.documents + (int64_t)b * a.N : nullptr, t0);
#pragma unroll
  for (int j = 1; j < W; ++j) past[j - 1] = to_pairs(row_at<T, W>(a, x, state, t0 - j, a.N, count, WIDE));
  for (int t = t0; t < t1; t += kAhead) {
    if (t > t0) fetch(t);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
#pragma unroll
      for (int j = W - 1; j > 0; --j) past[j] = past[j - 1];
      past[0] = to_pairs(rows[k]);
      if (t + k < t1) {
        int id;
        const int reach = docs.step(t + k, id);
        float v[8];
        from_pairs(taps<W>(w, bias, past, reach), v);
        const bool on = (!DOCS || id >= 0) && t + k < len;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (a.activation == FLARE_SILU) v[i] *= sigmoid(v[i]);
          if (!on) v[i] = 0.0f;
        }
        store8<T>(y + (int64_t)(t + k) * a.C, v, count, WIDE);
      }
    }
  }
}

// g[t] = dy[t] act'(pre[t]); dx[t] = sum_j w[W-1-j] g[t+j]; dw[W-1-j] = sum_t g[t] x[t-j]; dbias = sum g.
// A run computes the g of the W - 1 tokens behind it as well (their rows are read twice), and adds only its own tokens' to
// the weights' gradients: one partial sum per block, added up in order afterwards.
template <typename T, int W, bool DOCS, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps) conv_backward_kernel(const ConvParams p) {
  pdl_begin();
  const flare_conv_args_t& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.blocks_n, nb = blockIdx.x % p.blocks_n;
  const int c = (blockIdx.y * 32 + lane) * 8, count = c >= a.C ? 0 : WIDE ? 8 : min(8, a.C - c);
  const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)b * a.x_stride_b + c;
  const T* dy = reinterpret_cast<const T*>(a.dy) + (int64_t)b * a.dy_stride_b + c;
  T* dx = reinterpret_cast<T*>(a.dx) + (int64_t)b * a.N * a.C + c;
  const int t0 = (nb * kWarps + warp) * p.run, t1 = min(a.N, t0 + p.run), t2 = min(a.N, t1 + W - 1);
  Pairs dw[W + 1];  // (the last one: bias)
#pragma unroll
  for (int j = 0; j <= W; ++j) dw[j] = zero_pairs();
  if (t0 < t1 && count > 0) {
    Pairs w[W], bias, past[W], acc[W];  // acc[j]: gradient of token t - j, as far as it is known
    load_weights<W>(a, c, count, w, bias);
    Reach<W, DOCS> docs;
    docs.start(DOCS ? a.documents + (int64_t)b * a.N : nullptr, t0);
#pragma unroll
    for (int j = 1; j < W; ++j) {
      past[j - 1] = to_pairs(row_at<T, W>(a, x, nullptr, t0 - j, a.N, count, WIDE));
      acc[j - 1] = zero_pairs();
    }
    constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;
    const int end = t1 + W - 1;  // the last run's gradients leave W - 1 steps behind its last token
    for (int t = t0; t < end; t += kAhead) {
      Raw8<T> rows[kAhead], drows[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int n = t + k < t2 ? count : 0;
        rows[k] = load_raw8<T>(x + (int64_t)(t + k) * a.x_stride_n, n, WIDE);
        drows[k] = load_raw8<T>(dy + (int64_t)(t + k) * a.dy_stride_n, n, WIDE);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
#pragma unroll
        for (int j = W - 1; j > 0; --j) {
          past[j] = past[j - 1];
          acc[j] = acc[j - 1];
        }
        past[0] = to_pairs(rows[k]);
        acc[0] = zero_pairs();
        int id = -1, reach = 0;
        if (t + k < t2) reach = docs.step(t + k, id);
        if (id >= 0) {
          Pairs g = to_pairs(drows[k]);
          if (a.activation == FLARE_SILU) {
            float v[8], d[8];
            from_pairs(taps<W>(w, bias, past, reach), v);
            from_pairs(g, d);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float r = sigmoid(v[i]);
              d[i] *= r * fmaf(v[i], 1.0f - r, 1.0f);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) g.v[i] = f2_pack(d[2 * i], d[2 * i + 1]);
          }
#pragma unroll
          for (int j = 0; j < W; ++j)
            if (j <= reach) fma_pairs(w[W - 1 - j], g, acc[j]);
          if (t + k < t1) {
#pragma unroll
            for (int j = 0; j < W; ++j)
              if (j <= reach) fma_pairs(g, past[j], dw[W - 1 - j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) dw[W].v[i] = f2_add(dw[W].v[i], g.v[i]);
          }
        }
        const int done = t + k - (W - 1);
        if (done >= t0 && done < t1) {
          float v[8];
          from_pairs(acc[W - 1], v);
          store8<T>(dx + (int64_t)done * a.C, v, count, WIDE);
        }
      }
    }
  }
  // the block's four runs, in their order
  __shared__ float sums[kWarps - 1][32][8 * (W + 1) + 1];
  if (warp > 0) {
#pragma unroll
    for (int j = 0; j <= W; ++j) {
      float v[8];
      from_pairs(dw[j], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) sums[warp - 1][lane][j * 8 + i] = v[i];
    }
  }
  __syncthreads();
  if (warp > 0) return;
  float* out = p.partial + (int64_t)blockIdx.x * a.C * (W + 1);
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    float v[8];
    from_pairs(dw[j], v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < count) {
#pragma unroll
        for (int q = 0; q < kWarps - 1; ++q) v[i] += sums[q][lane][j * 8 + i];
        out[j < W ? (int64_t)(c + i) * W + j : (int64_t)a.C * W + c + i] = v[i];
      }
  }
}

// One token: the state's rows move up by one, the token's is the last.
template <typename T, int W>
__global__ void __launch_bounds__(128) conv_decode_kernel(const ConvParams p) {
  pdl_begin();
  const flare_conv_args_t& a = p.a;
  const int groups = (a.C + 7) / 8;
  const int64_t idx = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (idx >= (int64_t)a.B * groups) return;
  const int64_t b = idx / groups;
  const int c = (int)(idx - b * groups) * 8, count = min(8, a.C - c);
  const bool wide = p.wide != 0;
  T* state = reinterpret_cast<T*>(a.state_out) + b * (W - 1) * a.C + c;
  Raw8<T> rows[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) rows[j] = load_raw8<T>(state + (int64_t)j * a.C, count, wide);
  rows[W - 1] = load_raw8<T>(reinterpret_cast<const T*>(a.x) + b * a.x_stride_b + c, count, wide);
  Pairs w[W], bias, past[W];
  float v[8];
  load_weights<W>(a, c, count, w, bias);
#pragma unroll
  for (int j = 0; j < W; ++j) past[j] = to_pairs(rows[W - 1 - j]);
  from_pairs(taps<W>(w, bias, past, W - 1), v);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (a.activation == FLARE_SILU) v[i] *= sigmoid(v[i]);
  store8<T>(reinterpret_cast<T*>(a.y) + b * a.C + c, v, count, wide);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    from_pairs(past[W - 2 - j], v);
    store8<T>(state + (int64_t)j * a.C, v, count, wide);
  }
}

// Runs of 64 tokens where that leaves eight warps for every SM, of 8 where it does not: the W - 1 rows read again weigh less than idle SMs.
void plan(ConvParams& p, const flare_conv_args_t& a) {
  p.a = a;
  const int64_t columns = (a.C + 255) / 256;
  p.run = 64;
  while (p.run > 8 && (int64_t)a.B * ((a.N + p.run - 1) / p.run) * columns < (int64_t)sm_count() * 8) p.run /= 2;
  const int per = p.run * kWarps;
  p.blocks_n = (a.N + per - 1) / per;
  p.partial = nullptr;
}

int check(const flare_conv_args_t* a) {
  if (a == nullptr) return FLARE_ERR_BAD_POINTER;
  if (a->B <= 0 || a->N <= 0 || a->C <= 0) return FLARE_ERR_BAD_SHAPE;
  if (a->W < 2 || a->W > 4) return FLARE_ERR_UNSUPPORTED;
  if (a->C > 0x7fffffff - 256 || (a->C + 255) / 256 > 65535) return FLARE_ERR_UNSUPPORTED;  // (what grid.y holds)
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
  plan(p, a);
  p.wide = a.C % 8 == 0 && rows_wide(a.x, a.dtype, {a.x_stride_b, a.x_stride_n}) && rows_wide(a.y, a.dtype, {}) &&
           rows_wide(a.state_in, a.dtype, {}) && rows_wide(a.state_out, a.dtype, {});
  const dim3 grid((unsigned)(a.B * (int64_t)p.blocks_n), (unsigned)((a.C + 255) / 256));
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
  plan(p, *args);
  return (size_t)args->B * p.blocks_n * args->C * (args->W + 1) * sizeof(float);
}

int flare_conv_backward(const flare_conv_args_t* args, flare_stream_t stream) {
  if (const int rc = check(args)) return rc;
  const flare_conv_args_t& a = *args;
  if (a.dy == nullptr || a.dx == nullptr || a.dweight == nullptr) return FLARE_ERR_BAD_POINTER;
  if (a.state_in != nullptr || a.state_out != nullptr || a.lengths != nullptr) return FLARE_ERR_BAD_CONFIG;
  if (a.workspace == nullptr || a.workspace_bytes < flare_conv_backward_workspace_bytes(args)) return FLARE_ERR_WORKSPACE;
  ConvParams p;
  plan(p, a);
  p.partial = reinterpret_cast<float*>(a.workspace);
  p.wide = a.C % 8 == 0 && rows_wide(a.x, a.dtype, {a.x_stride_b, a.x_stride_n}) &&
           rows_wide(a.dy, a.dtype, {a.dy_stride_b, a.dy_stride_n}) && rows_wide(a.dx, a.dtype, {});
  const int parts = a.B * p.blocks_n;
  const dim3 grid((unsigned)parts, (unsigned)((a.C + 255) / 256));
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
  if (const int rc = check(args)) return rc;
  const flare_conv_args_t& a = *args;
  if (a.y == nullptr || a.state_out == nullptr) return FLARE_ERR_BAD_POINTER;
  ConvParams p;
  p.a = a;
  p.run = p.blocks_n = 0;
  p.partial = nullptr;
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
