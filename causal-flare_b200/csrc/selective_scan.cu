// Selective state space scan: forward, backward, one token.
//
//   h[t] = exp(delta A) h[t-1] + delta b[t] x[t],   y[t] = (<c[t], h[t]> + D x[t]) silu(z[t])
//
// Bound by the special-function unit: S exponentials for every token and channel, at 16 per cycle and SM, where the rows
// themselves are 6 to 8 bytes.  A channel belongs to four threads, S / 4 states each in registers; 64 channels make a block,
// which walks its tokens in tiles: delta, delta x, b and c of a tile are laid down in shared memory as fp32 (softplus once per
// token and channel, not once per state), the next tile's rows are fetched into registers meanwhile.  The recurrence's
// products are packed in pairs.  The sum over a channel's states is taken for four tokens at a time: three exchanges
// instead of eight.
//
// Few channels: a row's tokens are cut into segments that run side by side.  A first pass over all segments but the last forms
// what each leaves behind from a zero state (every exponential once more, no read-out), a small kernel joins them in order
// (a segment multiplies what enters it by exp(A sum of its deltas)), then every segment starts from its own carry.
//
// Backward: g[t] = c[t] gy[t] + exp(delta[t+1] A) g[t+1] in reverse, with the states that the forward kept in front of every
// tile.  A tile is walked forward once (which leaves the states in front of every eight tokens in shared memory), then eight
// tokens at a time are recomputed, with their factors, and walked in reverse.  The gradients of b and c are sums over channels: over the eight
// channels of a warp by seven exchanges for eight values, over a block's warps in shared memory, over blocks in order by a
// kernel of their own.  No atomics: the same call gives the same bits.
#include "selective_scan.cuh"

#include "sm100_ptx.cuh"

namespace flare {
namespace scan {

#ifdef FLARE_SCAN_TYPE

namespace {

using namespace mixer;
using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRow = kChannels + 8;  // padded rows: no bank is asked twice, neither by a token's threads nor by a channel's
__device__ __forceinline__ int padded(int c) { return c + 2 * (c >> 4); }

template <int NS>
struct Shape {
  static constexpr int S = NS * kLanes, TT = tile_tokens(S), SUB = NS <= 4 ? 8 : 4;
  static constexpr int BC = TT * S / kThreads;  // elements of b and of c that a thread stages
  static_assert(BC >= 1 && TT * S % kThreads == 0, "tile");
};

template <int NS>
struct Tile {
  float2 dd[Shape<NS>::TT][kRow];  // delta, delta x
  alignas(16) float b[Shape<NS>::TT][Shape<NS>::S];
  alignas(16) float c[Shape<NS>::TT][Shape<NS>::S];
  int reset[Shape<NS>::TT];
};
template <int NS>
struct ForwardSmem {
  Tile<NS> in;
  float y[Shape<NS>::TT][kRow];
};
template <int NS>
struct BackwardSmem {
  Tile<NS> in;
  float gy[Shape<NS>::TT][kRow];
  float p1[Shape<NS>::TT][kRow], p2[Shape<NS>::TT][kRow], y[Shape<NS>::TT][kRow];
  float bc[Shape<NS>::TT][kThreads / 32][2 * Shape<NS>::S];
  alignas(16) float starts[Shape<NS>::TT / Shape<NS>::SUB][kThreads][NS];  // (each thread its own)
};

// log(1 + exp(u)), the relative error a few 2^-24 for small values too (log1p); above 20 it is u to less than 2^-24 of it
__device__ __forceinline__ float softplus(float u) { return u > 20.0f ? u : log1pf(__expf(u)); }

// Where a block and a thread work.
template <typename T, int NS>
struct Place {
  int b, seg, t0, t1, len;   // tokens of the segment
  int group, c0;             // first channel of the block
  int token, cg, count;      // staging: token of the tile, first of eight channels, how many of them there are
  int ch, sub, channel;      // walking: channel of the block, quarter of its states, channel (-1: none)
  const int32_t* ids;
  __device__ __forceinline__ Place(const ScanParams& p) {
    const flare_scan_args_t& a = p.a;
    b = blockIdx.x / p.segments;
    seg = blockIdx.x % p.segments;
    t0 = seg * p.seg_tokens;
    t1 = min(a.N, t0 + p.seg_tokens);
    len = a.lengths != nullptr ? max(0, min(a.N, a.lengths[b])) : a.N;
    group = blockIdx.y / p.blocks_c;
    const int in_group = (blockIdx.y % p.blocks_c) * kChannels;
    c0 = group * p.channels + in_group;
    const int here = min(kChannels, p.channels - in_group);
    token = threadIdx.x >> 3;
    cg = (threadIdx.x & 7) * 8;
    count = token < Shape<NS>::TT ? max(0, min(8, here - cg)) : 0;
    ch = threadIdx.x >> 2;
    sub = threadIdx.x & 3;
    channel = ch < here ? c0 + ch : -1;
    ids = a.documents != nullptr ? a.documents + (int64_t)b * a.N : nullptr;
  }
  __device__ __forceinline__ bool on(int t) const { return t < t1 && t < len && (ids == nullptr || ids[t] >= 0); }
};

// A tile's rows on their way from memory.
template <typename T, int NS>
struct Rows {
  Raw8<T> x, dt;
  T b[Shape<NS>::BC], c[Shape<NS>::BC];
  bool on, bc_on[Shape<NS>::BC], reset;

  __device__ __forceinline__ void load(const ScanParams& p, const Place<T, NS>& at, int t0) {
    const flare_scan_args_t& a = p.a;
    const int t = t0 + at.token;
    on = at.token < Shape<NS>::TT && at.on(t);
    const int n = on ? at.count : 0;
    x = load_raw8<T>(reinterpret_cast<const T*>(a.x) + at.b * a.x_stride_b + t * a.x_stride_n + at.c0 + at.cg, n, p.wide);
    dt = load_raw8<T>(reinterpret_cast<const T*>(a.dt) + at.b * a.dt_stride_b + t * a.dt_stride_n + at.c0 + at.cg, n, p.wide);
#pragma unroll
    for (int i = 0; i < Shape<NS>::BC; ++i) {
      const int idx = threadIdx.x + i * kThreads, tt = t0 + idx / Shape<NS>::S, s = idx % Shape<NS>::S;
      bc_on[i] = at.on(tt);
      b[i] = c[i] = from_float<T>(0.0f);
      if (bc_on[i]) {
        b[i] = reinterpret_cast<const T*>(a.b)[at.b * a.b_stride_b + tt * a.b_stride_n + at.group * a.b_stride_g + s];
        c[i] = reinterpret_cast<const T*>(a.c)[at.b * a.c_stride_b + tt * a.c_stride_n + at.group * a.c_stride_g + s];
      }
    }
    const int r = t0 + threadIdx.x;
    reset = false;
    if (at.ids != nullptr && threadIdx.x < Shape<NS>::TT && r < at.t1) reset = r == 0 || at.ids[r] != at.ids[r - 1];
  }
  // into shared memory; padding: delta = delta x = b = c = 0, so that it leaves the state as it is
  __device__ __forceinline__ void stage(const ScanParams& p, const Place<T, NS>& at, const float (&bias)[8], Tile<NS>& to, float (&delta)[8],
                                        float (&xf)[8]) const {
    unpack8(x, xf);
    unpack8(dt, delta);
    if (at.token < Shape<NS>::TT) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        delta[i] += bias[i];
        if (p.a.dt_softplus) delta[i] = softplus(delta[i]);
        if (!on) delta[i] = 0.0f;
      }
      float4* const row = reinterpret_cast<float4*>(&to.dd[at.token][padded(at.cg)]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        row[i] = make_float4(delta[2 * i], delta[2 * i] * xf[2 * i], delta[2 * i + 1], delta[2 * i + 1] * xf[2 * i + 1]);
    }
#pragma unroll
    for (int i = 0; i < Shape<NS>::BC; ++i) {
      const int idx = threadIdx.x + i * kThreads;
      to.b[idx / Shape<NS>::S][idx % Shape<NS>::S] = to_float<T>(b[i]);
      to.c[idx / Shape<NS>::S][idx % Shape<NS>::S] = to_float<T>(c[i]);
    }
    if (threadIdx.x < Shape<NS>::TT) to.reset[threadIdx.x] = reset;
  }
};

template <int NS>
__device__ __forceinline__ void load_pairs(const float* p, uint64_t (&v)[NS / 2]) {
  if constexpr (NS == 2) {
    v[0] = *reinterpret_cast<const uint64_t*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < NS / 4; ++i) {
      const ulonglong2 r = reinterpret_cast<const ulonglong2*>(p)[i];
      v[2 * i] = r.x;
      v[2 * i + 1] = r.y;
    }
  }
}
template <int NS>
__device__ __forceinline__ void store_pairs(float* p, const uint64_t (&v)[NS / 2]) {
  if constexpr (NS == 2) {
    *reinterpret_cast<uint64_t*>(p) = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < NS / 4; ++i) reinterpret_cast<ulonglong2*>(p)[i] = make_ulonglong2(v[2 * i], v[2 * i + 1]);
  }
}

__device__ __forceinline__ uint64_t factor(uint64_t a2, uint64_t delta2) {
  float lo, hi;
  f2_unpack(f2_mul(a2, delta2), lo, hi);
  return f2_pack(ex2_approx(lo), ex2_approx(hi));
}
__device__ __forceinline__ float pair_sum(uint64_t v) {
  float lo, hi;
  f2_unpack(v, lo, hi);
  return lo + hi;
}

// v[k], summed over the four threads of a channel, for four tokens: thread `sub` gets token `sub`
__device__ __forceinline__ float four_sums(float (&v)[4], int sub) {
  const bool up = sub & 2, odd = sub & 1;
  const float s0 = __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], 2), s1 = __shfl_xor_sync(0xffffffffu, up ? v[1] : v[3], 2);
  const float k0 = (up ? v[2] : v[0]) + s0, k1 = (up ? v[3] : v[1]) + s1;
  return (odd ? k1 : k0) + __shfl_xor_sync(0xffffffffu, odd ? k0 : k1, 1);
}

// v[0..M), summed over the eight channels of a warp (lanes that differ in bits 2 to 4): afterwards v[0..max(1, M / 8)) holds
// the sums whose indexes begin at the returned one (-1: another lane has them)
template <int M>
__device__ __forceinline__ int channel_sums(float (&v)[M], int lane) {
  int first = 0, mine = 1;
#pragma unroll
  for (int step = 0; step < 3; ++step) {
    const int mask = 16 >> step, n = M >> step;
    const bool up = lane & mask;
    if (n > 1) {
#pragma unroll
      for (int i = 0; i < n / 2; ++i) {
        const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + n / 2], mask);
        v[i] = (up ? v[i + n / 2] : v[i]) + got;
      }
      if (up) first += n / 2;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], mask);
      if (up) mine = 0;
    }
  }
  return mine ? first : -1;
}

template <typename T, int NS, bool ENDS>
__global__ void __launch_bounds__(kThreads) forward_kernel(const ScanParams p) {
  pdl_wait();
  extern __shared__ __align__(16) uint8_t smem[];
  ForwardSmem<NS>& sm = *reinterpret_cast<ForwardSmem<NS>*>(smem);
  const flare_scan_args_t& a = p.a;
  const Place<T, NS> at(p);
  if (ENDS && at.seg == p.segments - 1) return;  // (nothing follows it)
  constexpr int TT = Shape<NS>::TT, S = Shape<NS>::S;
  float bias[8], D[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = at.c0 + at.cg + i;
    bias[i] = i < at.count && a.dt_bias != nullptr ? a.dt_bias[c] : 0.0f;
    D[i] = i < at.count && a.D != nullptr ? a.D[c] : 0.0f;
  }
  uint64_t A2[NS / 2], h[NS / 2];
  const int64_t weight_at = (int64_t)max(at.channel, 0) * S + at.sub * NS;
  float sum = 0.0f;  // of the deltas
#pragma unroll
  for (int i = 0; i < NS / 2; ++i) {
    const float* A = a.A + weight_at + 2 * i;
    A2[i] = f2_pack(A[0] * kLog2e, A[1] * kLog2e);
    h[i] = 0;
  }
  const int64_t state_at = (int64_t)at.b * a.C * S + weight_at;
  const int64_t carry_at = (int64_t)blockIdx.x * a.C * S + weight_at;
  if (!ENDS) {
    if (p.segments > 1) load_pairs<NS>(p.carry + carry_at, h);
    else if (a.state_in != nullptr) load_pairs<NS>(a.state_in + state_at, h);
  }
  Rows<T, NS> rows;
  rows.load(p, at, at.t0);
  Raw8<T> z, z_next;
  const T* const zp = reinterpret_cast<const T*>(a.z);
  const auto load_z = [&](int t0) {
    const int t = t0 + at.token;
    return load_raw8<T>(zp + at.b * a.z_stride_b + t * a.z_stride_n + at.c0 + at.cg, at.token < TT && at.on(t) ? at.count : 0, p.wide);
  };
  if (!ENDS && zp != nullptr) z_next = load_z(at.t0);
  const int tiles = (a.N + TT - 1) / TT;
  const bool docs = at.ids != nullptr;
#pragma unroll 1
  for (int t0 = at.t0; t0 < at.t1; t0 += TT) {
    float delta[8], x[8];
    rows.stage(p, at, bias, sm.in, delta, x);
    const bool on = rows.on;
    z = z_next;
    __syncthreads();
    if (t0 + TT < at.t1) {
      rows.load(p, at, t0 + TT);
      if (!ENDS && zp != nullptr) z_next = load_z(t0 + TT);
    }
    if (!ENDS && a.keep != nullptr && at.channel >= 0)
      store_pairs<NS>(a.keep + ((int64_t)at.b * tiles + t0 / TT) * a.C * S + weight_at, h);
#pragma unroll 2
    for (int t = 0; t < TT; t += 4) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (docs && sm.in.reset[t + k]) {
#pragma unroll
          for (int i = 0; i < NS / 2; ++i) h[i] = 0;
          if (ENDS) sum = -INFINITY;
        }
        const float2 dd = sm.in.dd[t + k][padded(at.ch)];
        const uint64_t d2 = f2_pack(dd.x, dd.x), x2 = f2_pack(dd.y, dd.y);
        uint64_t b[NS / 2], c[NS / 2], acc = 0;
        load_pairs<NS>(&sm.in.b[t + k][at.sub * NS], b);
        if (!ENDS) load_pairs<NS>(&sm.in.c[t + k][at.sub * NS], c);
        if (ENDS) sum += dd.x;
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) {
          h[i] = f2_fma(factor(A2[i], d2), h[i], f2_mul(x2, b[i]));
          if (!ENDS) acc = i ? f2_fma(h[i], c[i], acc) : f2_mul(h[i], c[i]);
        }
        v[k] = pair_sum(acc);
      }
      if (!ENDS) sm.y[t + at.sub][at.ch] = four_sums(v, at.sub);
    }
    __syncthreads();
    if (!ENDS) {
      const int t = t0 + at.token;
      if (at.token < TT && t < at.t1 && at.count > 0) {
        float y[8], g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = fmaf(D[i], x[i], sm.y[at.token][at.cg + i]);
        if (zp != nullptr) {
          unpack8(z, g);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] *= g[i] * sigmoid(g[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = on ? y[i] : 0.0f;
        store8<T>(reinterpret_cast<T*>(a.y) + ((int64_t)at.b * a.N + t) * a.C + at.c0 + at.cg, y, at.count, p.wide);
      }
    }
  }
  if (at.channel < 0) return;
  if (ENDS) {
    store_pairs<NS>(p.carry + carry_at, h);
    if (at.sub == 0) p.decay[(int64_t)blockIdx.x * a.C + at.channel] = sum < 0.0f ? -1.0f : sum;
  } else if (a.state_out != nullptr && at.seg == p.segments - 1) {
    store_pairs<NS>(a.state_out + state_at, h);
  }
}

template <typename T, int NS, bool ENDS>
__global__ void __launch_bounds__(kThreads) backward_kernel(const ScanParams p) {
  pdl_wait();
  extern __shared__ __align__(16) uint8_t smem[];
  BackwardSmem<NS>& sm = *reinterpret_cast<BackwardSmem<NS>*>(smem);
  const flare_scan_args_t& a = p.a;
  const Place<T, NS> at(p);
  if (ENDS && at.seg == 0) return;
  constexpr int TT = Shape<NS>::TT, S = Shape<NS>::S, SUB = Shape<NS>::SUB, P = NS / 2;
  float bias[8], D[8], sum_d[8], sum_bias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = at.c0 + at.cg + i;
    bias[i] = i < at.count && a.dt_bias != nullptr ? a.dt_bias[c] : 0.0f;
    D[i] = i < at.count && a.D != nullptr ? a.D[c] : 0.0f;
    sum_d[i] = sum_bias[i] = 0.0f;
  }
  uint64_t A2[P], G[P], dA[P];  // G: gradient of the state behind the token at hand, times that token's successor's factor
  const int64_t weight_at = (int64_t)max(at.channel, 0) * S + at.sub * NS;
  const int64_t carry_at = (int64_t)blockIdx.x * a.C * S + weight_at;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float* A = a.A + weight_at + 2 * i;
    A2[i] = f2_pack(A[0] * kLog2e, A[1] * kLog2e);
    G[i] = dA[i] = 0;
  }
  if (!ENDS && p.segments > 1) load_pairs<NS>(p.carry + carry_at, G);
  const T* const zp = reinterpret_cast<const T*>(a.z);
  const int tiles = (a.N + TT - 1) / TT;
  const bool docs = at.ids != nullptr;
  const int last = at.t0 + (at.t1 - at.t0 - 1) / TT * TT;
  Rows<T, NS> rows;
  Raw8<T> dy, z;
  uint64_t kept[P];
  const auto fetch = [&](int t0) {
    rows.load(p, at, t0);
    const int t = t0 + at.token, n = rows.on ? at.count : 0;
    dy = load_raw8<T>(reinterpret_cast<const T*>(a.dy) + at.b * a.dy_stride_b + t * a.dy_stride_n + at.c0 + at.cg, n, p.wide);
    if (zp != nullptr) z = load_raw8<T>(zp + at.b * a.z_stride_b + t * a.z_stride_n + at.c0 + at.cg, n, p.wide);
    if (!ENDS) load_pairs<NS>(a.keep + ((int64_t)at.b * tiles + t0 / TT) * a.C * S + weight_at, kept);
  };
  fetch(last);
#pragma unroll 1
  for (int t0 = last; t0 >= at.t0; t0 -= TT) {
    float delta[8], x[8];
    rows.stage(p, at, bias, sm.in, delta, x);
    const Raw8<T> dt_raw = rows.dt, dy_raw = dy, z_raw = z;
    const bool on = rows.on;
    if (at.token < TT) {
      float g[8], zf[8];
      unpack8(dy, g);
      if (zp != nullptr) {
        unpack8(z, zf);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= zf[i] * sigmoid(zf[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sm.gy[at.token][at.cg + i] = on ? g[i] : 0.0f;
    }
    uint64_t h[P];
#pragma unroll
    for (int i = 0; i < P; ++i) h[i] = kept[i];
    __syncthreads();
    if (t0 > at.t0) fetch(t0 - TT);
    if (ENDS) {
#pragma unroll 4
      for (int t = TT - 1; t >= 0; --t) {
        const float2 dd = sm.in.dd[t][padded(at.ch)];
        const uint64_t d2 = f2_pack(dd.x, dd.x), gy = f2_pack(sm.gy[t][at.ch], sm.gy[t][at.ch]);
        uint64_t c[P];
        load_pairs<NS>(&sm.in.c[t][at.sub * NS], c);
        sum += dd.x;
#pragma unroll
        for (int i = 0; i < P; ++i) G[i] = f2_mul(f2_fma(c[i], gy, G[i]), factor(A2[i], d2));
        if (docs && sm.in.reset[t]) {
#pragma unroll
          for (int i = 0; i < P; ++i) G[i] = 0;
          sum = -INFINITY;
        }
      }
    } else {
      const auto move = [&](int t, uint64_t (&f)[P], uint64_t (&before)[P]) {  // h over token t; its factors; what they multiply
        if (docs && sm.in.reset[t]) {
#pragma unroll
          for (int i = 0; i < P; ++i) h[i] = 0;
        }
        const float2 dd = sm.in.dd[t][padded(at.ch)];
        const uint64_t d2 = f2_pack(dd.x, dd.x), x2 = f2_pack(dd.y, dd.y);
        uint64_t b[P];
        load_pairs<NS>(&sm.in.b[t][at.sub * NS], b);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          f[i] = factor(A2[i], d2);
          before[i] = h[i];
          h[i] = f2_fma(f[i], h[i], f2_mul(x2, b[i]));
        }
      };
#pragma unroll 1
      for (int q = 0; q < TT / SUB; ++q) {
        store_pairs<NS>(sm.starts[q][threadIdx.x], h);
        if (q + 1 < TT / SUB) {
#pragma unroll
          for (int k = 0; k < SUB; ++k) {
            uint64_t f[P], before[P];
            move(q * SUB + k, f, before);
          }
        }
      }
#pragma unroll 1
      for (int q = TT / SUB - 1; q >= 0; --q) {
        uint64_t f[SUB][P], before[SUB][P];
        load_pairs<NS>(sm.starts[q][threadIdx.x], h);
#pragma unroll
        for (int k = 0; k < SUB; ++k) move(q * SUB + k, f[k], before[k]);
#pragma unroll
        for (int k4 = SUB - 4; k4 >= 0; k4 -= 4) {
          float p1[4], p2[4], yv[4];
#pragma unroll
          for (int k = 3; k >= 0; --k) {
            const int t = q * SUB + k4 + k;
            const float2 dd = sm.in.dd[t][padded(at.ch)];
            const float gys = sm.gy[t][at.ch];
            const uint64_t d2 = f2_pack(dd.x, dd.x), x2 = f2_pack(dd.y, dd.y), gy = f2_pack(gys, gys);
            uint64_t b[P], c[P], s1 = 0, s2 = 0, s3 = 0;
            load_pairs<NS>(&sm.in.b[t][at.sub * NS], b);
            load_pairs<NS>(&sm.in.c[t][at.sub * NS], c);
            float v[2 * NS];
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const uint64_t g = f2_fma(c[i], gy, G[i]);
              const uint64_t moved = f2_mul(f[k4 + k][i], before[k4 + k][i]);
              const uint64_t now = f2_fma(x2, b[i], moved);
              const uint64_t u = f2_mul(g, moved);
              s1 = i ? f2_fma(g, b[i], s1) : f2_mul(g, b[i]);
              s2 = i ? f2_fma(u, A2[i], s2) : f2_mul(u, A2[i]);
              s3 = i ? f2_fma(now, c[i], s3) : f2_mul(now, c[i]);
              dA[i] = f2_fma(u, d2, dA[i]);
              G[i] = f2_mul(g, f[k4 + k][i]);
              f2_unpack(f2_mul(g, x2), v[2 * i], v[2 * i + 1]);
              f2_unpack(f2_mul(now, gy), v[NS + 2 * i], v[NS + 2 * i + 1]);
            }
            if (docs && sm.in.reset[t]) {
#pragma unroll
              for (int i = 0; i < P; ++i) G[i] = 0;
            }
            p1[k] = pair_sum(s1);
            p2[k] = pair_sum(s2);
            yv[k] = pair_sum(s3);
            if (at.channel < 0) {
#pragma unroll
              for (int i = 0; i < 2 * NS; ++i) v[i] = 0.0f;
            }
            const int first = channel_sums(v, threadIdx.x & 31);
            if (first >= 0) {
              constexpr int R = 2 * NS >= 8 ? 2 * NS / 8 : 1;
#pragma unroll
              for (int i = 0; i < R; ++i) {
                const int j = first + i;  // (dB of this thread's states, then dC)
                sm.bc[t][threadIdx.x >> 5][(j / NS) * S + at.sub * NS + j % NS] = v[i];
              }
            }
          }
          const int t = q * SUB + k4 + at.sub;
          sm.p1[t][at.ch] = four_sums(p1, at.sub);
          sm.p2[t][at.ch] = four_sums(p2, at.sub);
          if (zp != nullptr) sm.y[t][at.ch] = four_sums(yv, at.sub);
        }
      }
    }
    __syncthreads();
    if (ENDS) continue;
    const int t = t0 + at.token;
    if (at.token < TT && t < at.t1 && at.count > 0) {
      float dx[8], ddt[8], dyf[8], gate[8], zf[8];
      unpack8(dy_raw, dyf);
      if (zp != nullptr) unpack8(z_raw, zf);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p1 = sm.p1[at.token][at.cg + i], gy = sm.gy[at.token][at.cg + i];
        ddt[i] = fmaf(x[i], p1, sm.p2[at.token][at.cg + i] * (1.0f / kLog2e));
        dx[i] = fmaf(delta[i], p1, D[i] * gy);
        if (!on) dx[i] = ddt[i] = 0.0f;
      }
      if (a.dt_softplus) {
        float u[8];
        unpack8(dt_raw, u);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (on) ddt[i] *= sigmoid(u[i] + bias[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum_bias[i] += ddt[i];
        if (on) sum_d[i] = fmaf(sm.gy[at.token][at.cg + i], x[i], sum_d[i]);
      }
      const int64_t row = ((int64_t)at.b * a.N + t) * a.C + at.c0 + at.cg;
      store8<T>(reinterpret_cast<T*>(a.dx) + row, dx, at.count, p.wide);
      store8<T>(reinterpret_cast<T*>(a.ddt) + row, ddt, at.count, p.wide);
      if (zp != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float r = sigmoid(zf[i]);
          gate[i] = on ? dyf[i] * fmaf(D[i], x[i], sm.y[at.token][at.cg + i]) * r * fmaf(zf[i], 1.0f - r, 1.0f) : 0.0f;
        }
        store8<T>(reinterpret_cast<T*>(a.dz) + row, gate, at.count, p.wide);
      }
    }
    for (int idx = threadIdx.x; idx < TT * 2 * S; idx += kThreads) {
      const int tt = idx / (2 * S), j = idx % (2 * S);
      if (t0 + tt < at.t1) {
        float v = sm.bc[tt][0][j];
#pragma unroll
        for (int w = 1; w < kThreads / 32; ++w) v += sm.bc[tt][w][j];
        p.partial_bc[(((int64_t)at.b * a.N + t0 + tt) * gridDim.y + blockIdx.y) * (2 * S) + j] = v;
      }
    }
  }
  if (ENDS) {
    if (at.channel >= 0) {
      store_pairs<NS>(p.carry + carry_at, G);
      if (at.sub == 0) p.decay[(int64_t)blockIdx.x * a.C + at.channel] = sum < 0.0f ? -1.0f : sum;
    }
    return;
  }
  float* out = p.partial_w + (int64_t)blockIdx.x * weight_sums(a);
  if (at.channel >= 0) store_pairs<NS>(out + weight_at, dA);
  // the sums that the staging threads hold, over the tokens of a tile
  __syncthreads();
  if (at.token < TT) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sm.p1[at.token][at.cg + i] = sum_d[i];
      sm.p2[at.token][at.cg + i] = sum_bias[i];
    }
  }
  __syncthreads();
  if (threadIdx.x < kChannels && (int)threadIdx.x < min(kChannels, p.channels - (int)(blockIdx.y % p.blocks_c) * kChannels)) {
    float d = 0.0f, e = 0.0f;
    for (int t = 0; t < TT; ++t) {
      d += sm.p1[t][threadIdx.x];
      e += sm.p2[t][threadIdx.x];
    }
    out[(int64_t)a.C * S + at.c0 + threadIdx.x] = d;
    out[(int64_t)a.C * (S + 1) + at.c0 + threadIdx.x] = e;
  }
}

// One token.  Bound by memory: every state is read and written once, 16 bytes of it by a thread.
template <typename T, int NS>
__global__ void __launch_bounds__(256) decode_kernel(const ScanParams p) {
  pdl_begin();
  constexpr int S = NS * kLanes;
  const flare_scan_args_t& a = p.a;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t channel = idx / kLanes;
  if (channel >= (int64_t)a.B * a.C) return;  // (whole groups of four lanes)
  const int64_t b = channel / a.C;
  const int c = (int)(channel - b * a.C), sub = threadIdx.x & 3, group = c / p.channels;
  float* state = a.state_out + channel * S + sub * NS;
  uint64_t h[NS / 2], acc = 0;
  load_pairs<NS>(state, h);
  const float x = to_float<T>(reinterpret_cast<const T*>(a.x)[b * a.x_stride_b + c]);
  float delta = to_float<T>(reinterpret_cast<const T*>(a.dt)[b * a.dt_stride_b + c]) + (a.dt_bias != nullptr ? a.dt_bias[c] : 0.0f);
  if (a.dt_softplus) delta = softplus(delta);
  const uint64_t d2 = f2_pack(delta, delta), x2 = f2_pack(delta * x, delta * x);
  const T* bp = reinterpret_cast<const T*>(a.b) + b * a.b_stride_b + group * a.b_stride_g + sub * NS;
  const T* cp = reinterpret_cast<const T*>(a.c) + b * a.c_stride_b + group * a.c_stride_g + sub * NS;
  const float* A = a.A + (int64_t)c * S + sub * NS;
#pragma unroll
  for (int i = 0; i < NS / 2; ++i) {
    const uint64_t A2 = f2_pack(A[2 * i] * kLog2e, A[2 * i + 1] * kLog2e);
    const uint64_t bv = f2_pack(to_float<T>(bp[2 * i]), to_float<T>(bp[2 * i + 1]));
    const uint64_t cv = f2_pack(to_float<T>(cp[2 * i]), to_float<T>(cp[2 * i + 1]));
    h[i] = f2_fma(factor(A2, d2), h[i], f2_mul(x2, bv));
    acc = i ? f2_fma(h[i], cv, acc) : f2_mul(h[i], cv);
  }
  store_pairs<NS>(state, h);
  float y = pair_sum(acc);
  const unsigned mask = __activemask();
  y += __shfl_xor_sync(mask, y, 1);
  y += __shfl_xor_sync(mask, y, 2);
  if (sub != 0) return;
  if (a.D != nullptr) y = fmaf(a.D[c], x, y);
  if (a.z != nullptr) {
    const float z = to_float<T>(reinterpret_cast<const T*>(a.z)[b * a.z_stride_b + c]);
    y *= z * sigmoid(z);
  }
  reinterpret_cast<T*>(a.y)[channel] = from_float<T>(y);
}

template <typename T, int NS>
int launch_ns(Pass pass, const ScanParams& p, cudaStream_t stream) {
  const flare_scan_args_t& a = p.a;
  if (pass == DECODE) {
    const int64_t blocks = ((int64_t)a.B * a.C * kLanes + 255) / 256;
    if (blocks > 0x7fffffff) return FLARE_ERR_UNSUPPORTED;
    LaunchTimer timer("scan_decode_kernel", stream);
    FLARE_CUDA_CHECK(launch_pdl(decode_kernel<T, NS>, dim3((unsigned)blocks), dim3(256), 0, stream, p));
    return FLARE_OK;
  }
  const char* const names[] = {"scan_forward_kernel", "scan_forward_kernel (ends)", "scan_backward_kernel", "scan_backward_kernel (ends)"};
  void (*const kernels[])(ScanParams) = {forward_kernel<T, NS, false>, forward_kernel<T, NS, true>, backward_kernel<T, NS, false>,
                                         backward_kernel<T, NS, true>};
  const size_t smem = pass == FORWARD || pass == FORWARD_ENDS ? sizeof(ForwardSmem<NS>) : sizeof(BackwardSmem<NS>);
  static_assert(sizeof(BackwardSmem<NS>) <= (size_t)kMaxDynamicSmem, "shared memory");
  const dim3 grid((unsigned)(a.B * (int64_t)p.segments), (unsigned)(a.G * p.blocks_c));
  FLARE_CUDA_CHECK(allow_smem(kernels[pass]));
  LaunchTimer timer(names[pass], stream);
  FLARE_CUDA_CHECK(launch_pdl(kernels[pass], grid, dim3(kThreads), smem, stream, p));
  return FLARE_OK;
}

}  // namespace

template <typename T>
int launch(Pass pass, const ScanParams& p, cudaStream_t stream) {
  switch (p.a.S) {
    case 8: return launch_ns<T, 2>(pass, p, stream);
    case 16: return launch_ns<T, 4>(pass, p, stream);
    default: return launch_ns<T, 8>(pass, p, stream);
  }
}
template int launch<FLARE_SCAN_TYPE>(Pass, const ScanParams&, cudaStream_t);

#else  // host side

extern template int launch<float>(Pass, const ScanParams&, cudaStream_t);
extern template int launch<__nv_bfloat16>(Pass, const ScanParams&, cudaStream_t);
extern template int launch<__half>(Pass, const ScanParams&, cudaStream_t);

namespace {

using namespace mixer;

// What enters a segment: what enters the one in front of it (REVERSE: behind it), decayed, plus what that one leaves behind.
template <bool REVERSE>
__global__ void __launch_bounds__(256) join_kernel(const ScanParams p) {
  pdl_begin();
  const flare_scan_args_t& a = p.a;
  const int64_t per = (int64_t)a.C * a.S, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.B * per) return;
  const int64_t b = i / per, cs = i - b * per, c = cs / a.S;
  const float A = a.A[cs];
  float in = !REVERSE && a.state_in != nullptr ? a.state_in[i] : 0.0f;
  for (int k = 0; k < p.segments; ++k) {
    const int64_t at = b * p.segments + (REVERSE ? p.segments - 1 - k : k);
    const bool ends = k + 1 < p.segments;  // (of the one behind which nothing follows there is no end)
    const float end = ends ? p.carry[at * per + cs] : 0.0f, sum = ends ? p.decay[at * a.C + c] : 0.0f;
    p.carry[at * per + cs] = in;
    in = sum < 0.0f ? end : fmaf(expf(A * sum), in, end);
  }
}

// db and dc: the blocks of a group's channels in their order
__global__ void __launch_bounds__(256) sum_bc_kernel(const ScanParams p) {
  pdl_begin();
  const flare_scan_args_t& a = p.a;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, total = (int64_t)a.B * a.N * a.G * 2 * a.S;
  if (i >= total) return;
  const int64_t tg = i / (2 * a.S);  // token and group
  const int j = (int)(i - tg * 2 * a.S);
  const float* in = p.partial_bc + tg * p.blocks_c * 2 * a.S + j;
  float v = in[0];
  for (int k = 1; k < p.blocks_c; ++k) v += in[(int64_t)k * 2 * a.S];
  store1(j < a.S ? a.db : a.dc, a.dtype, tg * a.S + (j < a.S ? j : j - a.S), v);
}

int check(const flare_scan_args_t* args) {
  if (args == nullptr) return FLARE_ERR_BAD_POINTER;
  const flare_scan_args_t& a = *args;
  if (a.B <= 0 || a.N <= 0 || a.C <= 0 || a.G <= 0 || a.C % a.G) return FLARE_ERR_BAD_SHAPE;
  if (a.S != 8 && a.S != 16 && a.S != 32) return FLARE_ERR_UNSUPPORTED;
  if (a.dtype < 0 || a.dtype > 2) return FLARE_ERR_BAD_DTYPE;
  if (a.N > 0x7fffffff - 1024 || (int64_t)a.G * ((a.C / a.G + kChannels - 1) / kChannels) > 65535) return FLARE_ERR_UNSUPPORTED;
  if (a.x == nullptr || a.dt == nullptr || a.A == nullptr || a.b == nullptr || a.c == nullptr) return FLARE_ERR_BAD_POINTER;
  for (const void* q : {(const void*)a.state_in, (const void*)a.state_out, (const void*)a.keep})
    if (reinterpret_cast<uintptr_t>(q) & 15u) return FLARE_ERR_BAD_POINTER;
  return FLARE_OK;
}

// Segments where the channels alone leave SMs idle: as many as fill two blocks per SM, of four tiles at least.  Below three they
// do not pay for the pass over their ends.
void plan(ScanParams& p, const flare_scan_args_t& a) {
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.channels = a.C / a.G;
  p.blocks_c = (p.channels + kChannels - 1) / kChannels;
  const int tile = tile_tokens(a.S);
  const int64_t blocks = (int64_t)a.B * a.G * p.blocks_c, tiles = (a.N + tile - 1) / tile;
  int64_t segments = 2 * (int64_t)sm_count() / blocks;
  if (segments > tiles / 4) segments = tiles / 4;
  if (segments < 3) segments = 1;
  const int64_t per = (tiles + segments - 1) / segments;
  p.seg_tokens = (int)(per * tile);
  p.segments = (int)((tiles + per - 1) / per);
}

size_t carry_bytes(const ScanParams& p) {
  if (p.segments == 1) return 0;
  return align_up((size_t)p.a.B * p.segments * p.a.C * p.a.S * 4, 256) + align_up((size_t)p.a.B * p.segments * p.a.C * 4, 256);
}
uint8_t* take_carry(ScanParams& p, uint8_t* ws) {
  p.carry = reinterpret_cast<float*>(ws);
  p.decay = reinterpret_cast<float*>(ws + align_up((size_t)p.a.B * p.segments * p.a.C * p.a.S * 4, 256));
  return ws + carry_bytes(p);
}
size_t partial_bc_bytes(const ScanParams& p) {
  return align_up((size_t)p.a.B * p.a.N * p.a.G * p.blocks_c * 2 * p.a.S * 4, 256);
}
size_t partial_w_bytes(const ScanParams& p) { return align_up((size_t)p.a.B * p.segments * weight_sums(p.a) * 4, 256); }

int run(Pass pass, const ScanParams& p, cudaStream_t stream) {
  switch (p.a.dtype) {
    case FLARE_F32: return launch<float>(pass, p, stream);
    case FLARE_BF16: return launch<__nv_bfloat16>(pass, p, stream);
    default: return launch<__half>(pass, p, stream);
  }
}

template <bool REVERSE>
int run_segments(const ScanParams& p, cudaStream_t stream) {
  if (p.segments > 1) {
    if (const int rc = run(REVERSE ? BACKWARD_ENDS : FORWARD_ENDS, p, stream)) return rc;
    const int64_t n = (int64_t)p.a.B * p.a.C * p.a.S;
    LaunchTimer timer("scan_join_kernel", stream);
    FLARE_CUDA_CHECK(launch_pdl(join_kernel<REVERSE>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p));
  }
  return run(REVERSE ? BACKWARD : FORWARD, p, stream);
}

}  // namespace
#endif

}  // namespace scan
}  // namespace flare

#ifndef FLARE_SCAN_TYPE
using namespace flare;
using namespace flare::scan;

extern "C" {

size_t flare_scan_keep_bytes(const flare_scan_args_t* args) {
  if (check(args)) return 0;
  const int tile = tile_tokens(args->S);
  return (size_t)args->B * ((args->N + tile - 1) / tile) * args->C * args->S * 4;
}

size_t flare_scan_forward_workspace_bytes(const flare_scan_args_t* args) {
  if (check(args)) return 0;
  ScanParams p;
  plan(p, *args);
  return carry_bytes(p);
}

int flare_scan_forward(const flare_scan_args_t* args, flare_stream_t stream) {
  if (const int rc = check(args)) return rc;
  const flare_scan_args_t& a = *args;
  if (a.y == nullptr || (a.state_out != nullptr && a.state_out == a.state_in)) return FLARE_ERR_BAD_POINTER;
  if (a.documents != nullptr && (a.state_in != nullptr || a.state_out != nullptr)) return FLARE_ERR_BAD_CONFIG;
  ScanParams p;
  plan(p, a);
  if (carry_bytes(p) > 0) {
    if (a.workspace == nullptr || a.workspace_bytes < carry_bytes(p)) return FLARE_ERR_WORKSPACE;
    take_carry(p, reinterpret_cast<uint8_t*>(a.workspace));
  }
  p.wide = p.channels % 8 == 0 && rows_wide(a.x, a.dtype, {a.x_stride_b, a.x_stride_n}) && rows_wide(a.dt, a.dtype, {a.dt_stride_b, a.dt_stride_n}) &&
           (a.z == nullptr || rows_wide(a.z, a.dtype, {a.z_stride_b, a.z_stride_n})) && rows_wide(a.y, a.dtype, {});
  return run_segments<false>(p, stream);
}

size_t flare_scan_backward_workspace_bytes(const flare_scan_args_t* args) {
  if (check(args)) return 0;
  ScanParams p;
  plan(p, *args);
  return carry_bytes(p) + partial_bc_bytes(p) + partial_w_bytes(p);
}

int flare_scan_backward(const flare_scan_args_t* args, flare_stream_t stream) {
  if (const int rc = check(args)) return rc;
  const flare_scan_args_t& a = *args;
  if (a.dy == nullptr || a.dx == nullptr || a.ddt == nullptr || a.db == nullptr || a.dc == nullptr || a.dA == nullptr || a.keep == nullptr ||
      (a.z != nullptr && a.dz == nullptr))
    return FLARE_ERR_BAD_POINTER;
  if (a.state_in != nullptr || a.state_out != nullptr || a.lengths != nullptr) return FLARE_ERR_BAD_CONFIG;
  ScanParams p;
  plan(p, a);
  if (a.workspace == nullptr || a.workspace_bytes < flare_scan_backward_workspace_bytes(args)) return FLARE_ERR_WORKSPACE;
  uint8_t* ws = take_carry(p, reinterpret_cast<uint8_t*>(a.workspace));
  p.partial_bc = reinterpret_cast<float*>(ws);
  p.partial_w = reinterpret_cast<float*>(ws + partial_bc_bytes(p));
  p.wide = p.channels % 8 == 0 && rows_wide(a.x, a.dtype, {a.x_stride_b, a.x_stride_n}) && rows_wide(a.dt, a.dtype, {a.dt_stride_b, a.dt_stride_n}) &&
           (a.z == nullptr || rows_wide(a.z, a.dtype, {a.z_stride_b, a.z_stride_n})) && rows_wide(a.dy, a.dtype, {a.dy_stride_b, a.dy_stride_n}) &&
           rows_wide(a.dx, a.dtype, {}) && rows_wide(a.ddt, a.dtype, {}) && rows_wide(a.dz, a.dtype, {});
  if (const int rc = run_segments<true>(p, stream)) return rc;
  const int64_t n = (int64_t)a.B * a.N * a.G * 2 * a.S;
  if ((n + 255) / 256 > 0x7fffffff) return FLARE_ERR_UNSUPPORTED;
  {
    LaunchTimer timer("scan_sum_bc_kernel", stream);
    FLARE_CUDA_CHECK(launch_pdl(sum_bc_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p));
  }
  const int64_t cs = (int64_t)a.C * a.S, stride = weight_sums(a);
  const int parts = a.B * p.segments;
  SumList list = {};
  int count = 0;
  list.part[count++] = {p.partial_w, a.dA, cs, stride, parts, FLARE_F32};
  if (a.dD != nullptr) list.part[count++] = {p.partial_w + cs, a.dD, a.C, stride, parts, FLARE_F32};
  if (a.ddt_bias != nullptr) list.part[count++] = {p.partial_w + cs + a.C, a.ddt_bias, a.C, stride, parts, FLARE_F32};
  return launch_sum_parts(list, count, stream);
}

int flare_scan_decode(const flare_scan_args_t* args, flare_stream_t stream) {
  flare_scan_args_t a;
  if (args == nullptr) return FLARE_ERR_BAD_POINTER;
  a = *args;
  a.N = 1;
  if (const int rc = check(&a)) return rc;
  if (a.y == nullptr || a.state_out == nullptr) return FLARE_ERR_BAD_POINTER;
  ScanParams p;
  plan(p, a);
  return run(DECODE, p, stream);
}

}  // extern "C"
#endif
