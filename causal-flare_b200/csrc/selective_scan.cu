// Selective state space scan: forward, backward, one token.
//
//   h[t] = exp(delta A) h[t-1] + delta b[t] x[t],   y[t] = (<c[t], h[t]> + D x[t]) silu(z[t])
//
// Bound by the special-function unit: S exponentials for every token and channel, at 16 per cycle and SM, where the rows
// themselves are 6 to 8 bytes.  A channel belongs to S / NS threads with NS states each in registers; a block walks its channels' tokens
// in tiles of 32: delta, delta x, b and c of a tile are laid down in shared memory as fp32 (softplus once per token and channel, not
// once per state), twice, so that the next tile is laid down while this one is walked (by threads of their own, where a block has an SM to itself) and a tile
// costs one barrier; the rows of the tile after that are on their way into registers meanwhile.  The recurrence's products are packed in pairs.  The sum over a
// channel's states is taken for as many tokens as the channel has threads at a time: three exchanges for four tokens.  B200, B=4 N=4096 C=2048 S=16
// bf16: 317 us (the exponentials alone: 120; what is issued and its latencies bound it).
//
// Few channels: a row's tokens are cut into segments that run side by side.  A first pass over all segments but the last forms
// what each leaves behind from a zero state (every exponential once more, no read-out), a small kernel joins them in order
// (a segment multiplies what enters it by exp(A sum of its deltas)), then every segment starts from its own carry.
//
// Backward: g[t] = c[t] gy[t] + exp(delta[t+1] A) g[t+1] in reverse, with the states that the forward kept in front of every
// tile.  A tile is walked forward once (which leaves the states in front of every eight tokens in shared memory), then eight
// tokens at a time are recomputed, with their factors, and walked in reverse.  The gradients of b and c are sums over channels: over
// the channels of a warp by exchanges that halve the values they carry, over a block's warps in shared memory, over blocks in order
// by a kernel of their own.  No atomics: the same call gives the same bits.  The same sizes: 1 053 us, bound by latencies: eight warps an SM walk,
// which is all that there are channels for.
#include "selective_scan.cuh"

#include "sm100_ptx.cuh"

namespace flare {
namespace scan {

#ifdef FLARE_SCAN_TYPE

namespace {

using namespace mixer;
using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f;

template <int S_, int NS_, int THREADS_, int BLOCKS_ = 1, int CT_ = 1, int STAGERS_ = 0>
struct Config {
  static constexpr int STAGERS = STAGERS_;  // of the backward: threads that stage while the others walk (0: all do both)
  static constexpr int BLOCKS = BLOCKS_;  // of an SM, at least
  static constexpr int CT = CT_;          // channels of a thread, CH / CT apart (1 in the forward)
  static constexpr int SUB = 8;           // tokens that the backward recomputes at a time
  static constexpr int S = S_, NS = NS_, THREADS = THREADS_, P = NS / 2, LANES = S / NS, CH = THREADS / LANES * CT, APART = CH / CT, WARPS = THREADS / 32;
  static constexpr int V = kTile * CH / THREADS;   // neighbouring channels of a token that a thread stages
  static constexpr int PER = CH / V;               // threads of a token, staging
  static constexpr int BC = kTile * S / THREADS;   // elements of b and of c that a thread stages
  static constexpr int ROW = CH + 32 / LANES;      // rows of one value per channel: neither staging nor walking asks a bank twice
  static constexpr int ROW4 = CH + CH / 8;         // rows of four, see padded()
  static_assert(kTile * CH % THREADS == 0 && (V == 4 || V == 8) && kTile * S % THREADS == 0 && NS % 2 == 0, "tile");
};
__device__ __forceinline__ int padded(int c) { return c + (c >> 3); }

template <typename K>
struct Tile {
  alignas(16) float4 dd[kTile][K::ROW4];       // delta, delta x, each twice: as the packed products take them
  alignas(16) float bc[kTile][K::S / 2][4];    // b, c of a pair of states
  int reset[kTile];
};
template <typename K>
struct ForwardSmem {
  Tile<K> in[2];
  float y[2][kTile][K::ROW];
};
template <typename K, bool SPLIT>
struct BackwardSmem {
  static constexpr int BUFFERS = SPLIT ? 2 : 1;
  Tile<K> in[BUFFERS];
  float gy[BUFFERS][kTile][K::ROW];
  float p1[BUFFERS][kTile][K::ROW], p2[BUFFERS][kTile][K::ROW], y[BUFFERS][kTile][K::ROW];
  float bc[BUFFERS][kTile][K::WARPS][2 * K::S];
  alignas(16) float starts[kTile / K::SUB - 1][K::THREADS][K::CT * K::NS];  // (each thread its own)
};

// softplus(u) = max(u, 0) + log(1 + t), t = exp(-|u|), and its slope 1 / (1 + exp(-u)).  log(1 + t) = 2 atanh(s) with s = t / (2 + t) <= 1 / 3: the
// terms of atanh's series up to s^13 leave less than 2e-8 of it, and small t keep their relative precision.
__device__ __forceinline__ float softplus(float u, float& slope) {
  const float t = ex2_approx(-kLog2e * fabsf(u)), s = t * rcp_approx(2.0f + t), q = s * s;
  float a = fmaf(q, 1.0f / 13.0f, 1.0f / 11.0f);
  a = fmaf(q, a, 1.0f / 9.0f);
  a = fmaf(q, a, 1.0f / 7.0f);
  a = fmaf(q, a, 1.0f / 5.0f);
  a = fmaf(q, a, 1.0f / 3.0f);
  const float r = rcp_approx(1.0f + t);
  slope = u >= 0.0f ? r : t * r;
  return fmaxf(u, 0.0f) + 2.0f * fmaf(s * q, a, s);
}

// Where a block and a thread work.  A thread is one of K::THREADS: itself, HALVES: one of the first half (which walks) or of the second (which
// stages), GIVEN: what the caller says.
enum Who { ITSELF, HALVES, GIVEN };
template <typename K, Who WHO = ITSELF>
struct Place {
  unsigned given;
  __device__ __forceinline__ unsigned tid() const { return WHO == GIVEN ? given : WHO == HALVES ? threadIdx.x % K::THREADS : threadIdx.x; }
  int b, seg, t0, t1, len;   // tokens of the segment
  int group, c0, here;       // first channel of the block, how many it has
  int token, cg, count;      // staging: token of the tile, first of V channels, how many of them there are
  int ch, sub, channel;      // walking: channel of the block, part of its states, channel (-1: none)
  const int32_t* ids;
  __device__ __forceinline__ explicit Place(const ScanParams& p, unsigned given_ = 0) : given(given_) {
    const flare_scan_args_t& a = p.a;
    b = blockIdx.x / p.segments;
    seg = blockIdx.x % p.segments;
    t0 = seg * p.seg_tokens;
    t1 = min(a.N, t0 + p.seg_tokens);
    len = a.lengths != nullptr ? max(0, min(a.N, a.lengths[b])) : a.N;
    group = blockIdx.y / p.blocks_c;
    const int in_group = (blockIdx.y % p.blocks_c) * K::CH;
    c0 = group * p.channels + in_group;
    here = min(K::CH, p.channels - in_group);
    token = tid() / K::PER;
    cg = tid() % K::PER * K::V;
    count = max(0, min(K::V, here - cg));
    ch = tid() / K::LANES;
    sub = tid() % K::LANES;
    channel = ch < here ? c0 + ch : -1;
    ids = a.documents != nullptr ? a.documents + (int64_t)b * a.N : nullptr;
  }
  __device__ __forceinline__ bool on(int t) const { return t < t1 && t < len && (ids == nullptr || ids[t] >= 0); }
};

// A tile's rows on their way from memory.
template <typename T, typename K, bool WIDE>
struct Rows {
  Raw<T, K::V> x, dt;
  T b[K::BC], c[K::BC];
  bool on, bc_on[K::BC], reset;

  template <typename At>
  __device__ __forceinline__ void load(const ScanParams& p, const At& at, int t0) {
    const flare_scan_args_t& a = p.a;
    const int t = t0 + at.token;
    on = at.on(t);
    const int n = on ? at.count : 0;
    x = load_raw<T, K::V>(reinterpret_cast<const T*>(a.x) + at.b * a.x_stride_b + t * a.x_stride_n + at.c0 + at.cg, n, WIDE);
    dt = load_raw<T, K::V>(reinterpret_cast<const T*>(a.dt) + at.b * a.dt_stride_b + t * a.dt_stride_n + at.c0 + at.cg, n, WIDE);
#pragma unroll
    for (int i = 0; i < K::BC; ++i) {
      const int idx = at.tid() + i * K::THREADS, tt = t0 + idx / K::S, s = idx % K::S;
      bc_on[i] = at.on(tt);
      b[i] = c[i] = from_float<T>(0.0f);
      if (bc_on[i]) {
        b[i] = reinterpret_cast<const T*>(a.b)[at.b * a.b_stride_b + tt * a.b_stride_n + at.group * a.b_stride_g + s];
        c[i] = reinterpret_cast<const T*>(a.c)[at.b * a.c_stride_b + tt * a.c_stride_n + at.group * a.c_stride_g + s];
      }
    }
    const int r = t0 + at.tid();
    reset = false;
    if (at.ids != nullptr && at.tid() < kTile && r < at.t1) reset = r == 0 || at.ids[r] != at.ids[r - 1];
  }
  // into shared memory; padding: delta = delta x = b = c = 0, so that it leaves the state as it is
  template <typename At>
  __device__ __forceinline__ void stage(const ScanParams& p, const At& at, const float (&bias)[K::V], Tile<K>& to, float (&delta)[K::V],
                                        float (&slope)[K::V], float (&xf)[K::V]) const {
    unpack<T, K::V>(x, xf);
    unpack<T, K::V>(dt, delta);
#pragma unroll
    for (int i = 0; i < K::V; ++i) {
      delta[i] += bias[i];
      slope[i] = 1.0f;
      if (p.a.dt_softplus) delta[i] = softplus(delta[i], slope[i]);
      if (!on) delta[i] = 0.0f;
    }
    float4* const row = &to.dd[at.token][padded(at.cg)];
#pragma unroll
    for (int i = 0; i < K::V; ++i) row[i] = make_float4(delta[i], delta[i], delta[i] * xf[i], delta[i] * xf[i]);
#pragma unroll
    for (int i = 0; i < K::BC; ++i) {
      const int idx = at.tid() + i * K::THREADS, s = idx % K::S;
      to.bc[idx / K::S][s >> 1][s & 1] = to_float<T>(b[i]);
      to.bc[idx / K::S][s >> 1][2 + (s & 1)] = to_float<T>(c[i]);
    }
    if (at.tid() < kTile) to.reset[at.tid()] = reset;
  }
};

template <int P>
__device__ __forceinline__ void load_pairs(const float* p, uint64_t (&v)[P]) {
  if constexpr (P == 1) {
    v[0] = *reinterpret_cast<const uint64_t*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      const ulonglong2 r = reinterpret_cast<const ulonglong2*>(p)[i];
      v[2 * i] = r.x;
      v[2 * i + 1] = r.y;
    }
  }
}
template <int P>
__device__ __forceinline__ void store_pairs(float* p, const uint64_t (&v)[P]) {
  if constexpr (P == 1) {
    *reinterpret_cast<uint64_t*>(p) = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) reinterpret_cast<ulonglong2*>(p)[i] = make_ulonglong2(v[2 * i], v[2 * i + 1]);
  }
}
// b and c of a thread's pairs
template <int P>
__device__ __forceinline__ void load_bc(const float (*p)[4], uint64_t (&b)[P], uint64_t (&c)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const ulonglong2 r = *reinterpret_cast<const ulonglong2*>(p[i]);
    b[i] = r.x;
    c[i] = r.y;
  }
}

__device__ __forceinline__ uint64_t twice(float x) { return f2_pack(x, x); }
// exp(delta A).  ex2.approx is low by 0.4 units in the last place on average (over arguments from -0.5 to 0 its error has mean -2.1e-8 and
// deviation 3.3e-8, measured against 64 bits), which adds up over the tokens that a state remembers: a shift of the argument takes the mean
// away.  (A factor of 1 stays 1: 2^shift is nearer to it than to its neighbour.)
constexpr float kShift = 3.3e-8f;
__device__ __forceinline__ uint64_t factor(uint64_t a2, uint64_t delta2) {
  float lo, hi;
  f2_unpack(f2_fma(a2, delta2, f2_pack(kShift, kShift)), lo, hi);
  return f2_pack(ex2_approx(lo), ex2_approx(hi));
}
__device__ __forceinline__ float low(uint64_t v) {
  float lo, hi;
  f2_unpack(v, lo, hi);
  return lo;
}
__device__ __forceinline__ float pair_sum(uint64_t v) {
  float lo, hi;
  f2_unpack(v, lo, hi);
  return lo + hi;
}

// v[k], summed over the L threads of a channel (neighbouring lanes), for L tokens: thread `sub` gets token `sub`
template <int L>
__device__ __forceinline__ float lane_sums(float (&v)[L], int sub) {
#pragma unroll
  for (int n = L; n > 1; n /= 2) {
    const bool up = sub & (n / 2);
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + n / 2], n / 2);
      v[i] = (up ? v[i + n / 2] : v[i]) + got;
    }
  }
  return v[0];
}

// v[0..M), summed over the channels of a warp (lanes that differ in bits above those of a channel's L threads): afterwards
// v[0..max(1, M L / 32)) holds the sums whose indexes begin at the returned one (-1: another lane has them)
template <int M, int L>
__device__ __forceinline__ int channel_sums(float (&v)[M], int lane) {
  int first = 0, mine = 1, n = M;
#pragma unroll
  for (int mask = 16; mask >= L; mask /= 2) {
    const bool up = lane & mask;
    if (n > 1) {
#pragma unroll
      for (int i = 0; i < M / 2; ++i)
        if (i < n / 2) {
          const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + n / 2], mask);
          v[i] = (up ? v[i + n / 2] : v[i]) + got;
        }
      n /= 2;
      if (up) first += n;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], mask);
      if (up) mine = 0;
    }
  }
  return mine ? first : -1;
}

// SPLIT: half of the threads walk, the others lay down the next tile and read out the last one meanwhile
template <typename T, typename K, bool ENDS, bool WIDE, bool DOCS, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 2 * K::THREADS : K::THREADS, SPLIT ? 1 : K::BLOCKS) forward_kernel(const ScanParams p) {
  pdl_wait();
  extern __shared__ __align__(16) uint8_t smem[];
  ForwardSmem<K>& sm = *reinterpret_cast<ForwardSmem<K>*>(smem);
  const flare_scan_args_t& a = p.a;
  const bool walks = !SPLIT || threadIdx.x < K::THREADS, stages = !SPLIT || !walks;
  const Place<K, SPLIT ? HALVES : ITSELF> at(p);
  if (ENDS && at.seg == p.segments - 1) return;  // (nothing follows it)
  constexpr int S = K::S, P = K::P, V = K::V, LANES = K::LANES;
  float bias[V], D[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = at.c0 + at.cg + i;
    bias[i] = i < at.count && a.dt_bias != nullptr ? a.dt_bias[c] : 0.0f;
    D[i] = i < at.count && a.D != nullptr ? a.D[c] : 0.0f;
  }
  uint64_t A2[P], h[P];
  const int64_t weight_at = (int64_t)max(at.channel, 0) * S + at.sub * K::NS;
  float sum = 0.0f;  // of the deltas
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float* A = a.A + weight_at + 2 * i;
    A2[i] = f2_pack(A[0] * kLog2e, A[1] * kLog2e);
    h[i] = 0;
  }
  const int64_t state_at = (int64_t)at.b * a.C * S + weight_at;
  const int64_t carry_at = (int64_t)blockIdx.x * a.C * S + weight_at;
  if (!ENDS) {
    if (p.segments > 1) load_pairs<P>(p.carry + carry_at, h);
    else if (a.state_in != nullptr) load_pairs<P>(a.state_in + state_at, h);
  }
  const T* const zp = reinterpret_cast<const T*>(a.z);
  const int tiles = (a.N + kTile - 1) / kTile;
  Rows<T, K, WIDE> rows;
  Raw<T, V> z;  // of the rows in `rows`
  const auto fetch = [&](int t0) {
    rows.load(p, at, t0);
    const int t = t0 + at.token;
    if (!ENDS && zp != nullptr)
      z = load_raw<T, V>(zp + at.b * a.z_stride_b + t * a.z_stride_n + at.c0 + at.cg, rows.on ? at.count : 0, WIDE);
  };
  const auto lay_down = [&](int buffer) {
    float delta[V], slope[V], x[V];
    rows.stage(p, at, bias, sm.in[buffer], delta, slope, x);
  };
  // what the read-out of a tile takes: of the tile that is walked, and of the one before it
  Raw<T, V> x_now, z_now, x_out, z_out;
  bool on_now = false, on_out = false;
  const auto read_out = [&](int t, int buffer) {
    if (ENDS || t >= at.t1 || at.count <= 0) return;
    float y[V], x[V], g[V];
    unpack<T, V>(x_out, x);
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = fmaf(D[i], x[i], sm.y[buffer][at.token][at.cg + i]);
    if (zp != nullptr) {
      unpack<T, V>(z_out, g);
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] *= g[i] * sigmoid(g[i]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = on_out ? y[i] : 0.0f;
    store_all<T, V>(reinterpret_cast<T*>(a.y) + ((int64_t)at.b * a.N + t) * a.C + at.c0 + at.cg, y, at.count, WIDE);
  };
  const auto walk = [&](int t0, int buffer) {
    const Tile<K>& in = sm.in[buffer];
    if (!ENDS && a.keep != nullptr && at.channel >= 0)
      store_pairs<P>(a.keep + ((int64_t)at.b * tiles + t0 / kTile) * a.C * S + weight_at, h);
    constexpr int STEP = ENDS ? 4 : LANES;
#pragma unroll(ENDS ? 4 : kTile / STEP)
    for (int t = 0; t < kTile; t += STEP) {
      float v[STEP];
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        if (DOCS && in.reset[t + k]) {
#pragma unroll
          for (int i = 0; i < P; ++i) h[i] = 0;
          if (ENDS) sum = -INFINITY;
        }
        const ulonglong2 dd = *reinterpret_cast<const ulonglong2*>(&in.dd[t + k][padded(at.ch)]);
        const uint64_t d2 = dd.x, x2 = dd.y;
        uint64_t b[P], c[P], acc = 0;
        load_bc<P>(&in.bc[t + k][at.sub * P], b, c);
        if (ENDS) sum += low(d2);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          h[i] = f2_fma(factor(A2[i], d2), h[i], f2_mul(x2, b[i]));
          if (!ENDS) acc = i ? f2_fma(h[i], c[i], acc) : f2_mul(h[i], c[i]);
        }
        v[k] = pair_sum(acc);
      }
      if constexpr (!ENDS) sm.y[buffer][t + at.sub][at.ch] = lane_sums<LANES>(v, at.sub);
    }
  };
  if (stages) {
    fetch(at.t0);
    lay_down(0);
    x_now = rows.x;
    z_now = z;
    on_now = rows.on;
    if (at.t0 + kTile < at.t1) fetch(at.t0 + kTile);
  }
  const auto stage = [&](int t0, int buffer) {  // the next tile, while this one is walked
    x_out = x_now;
    z_out = z_now;
    on_out = on_now;
    if (t0 + kTile < at.t1) {
      lay_down(buffer ^ 1);
      x_now = rows.x;
      z_now = z;
      on_now = rows.on;
      if (t0 + 2 * kTile < at.t1) fetch(t0 + 2 * kTile);
    }
  };
  int buffer = 0;
  if constexpr (SPLIT) {
    // (loops of their own: neither side's registers are the other's)
    const auto tile_done = [] { asm volatile("bar.sync 1, %0;" ::"n"(2 * K::THREADS) : "memory"); };
    tile_done();
    if (walks) {
#pragma unroll 1
      for (int t0 = at.t0; t0 < at.t1; t0 += kTile, buffer ^= 1) {
        walk(t0, buffer);
        tile_done();
      }
    } else {
#pragma unroll 1
      for (int t0 = at.t0; t0 < at.t1; t0 += kTile, buffer ^= 1) {
        if (t0 > at.t0) read_out(t0 - kTile + at.token, buffer ^ 1);
        stage(t0, buffer);
        tile_done();
      }
      read_out(at.t0 + (at.t1 - at.t0 - 1) / kTile * kTile + at.token, buffer ^ 1);
      return;
    }
  } else {
    __syncthreads();
#pragma unroll 1
    for (int t0 = at.t0; t0 < at.t1; t0 += kTile, buffer ^= 1) {
      walk(t0, buffer);
      stage(t0, buffer);
      __syncthreads();
      read_out(t0 + at.token, buffer);
    }
  }
  if (at.channel < 0) return;
  if (ENDS) {
    store_pairs<P>(p.carry + carry_at, h);
    if (at.sub == 0) p.decay[(int64_t)blockIdx.x * a.C + at.channel] = sum;
  } else if (a.state_out != nullptr && at.seg == p.segments - 1) {
    store_pairs<P>(a.state_out + state_at, h);
  }
}

// SPLIT: the first K::THREADS threads walk, K::STAGERS more lay down the next tile and form the gradients of the last one meanwhile, each for as
// many places of a tile as it takes
template <typename T, typename K, bool ENDS, bool WIDE, bool DOCS, bool SPLIT>
__global__ void __launch_bounds__(K::THREADS + (SPLIT ? K::STAGERS : 0), K::BLOCKS) backward_kernel(const ScanParams p) {
  pdl_wait();
  extern __shared__ __align__(16) uint8_t smem[];
  BackwardSmem<K, SPLIT>& sm = *reinterpret_cast<BackwardSmem<K, SPLIT>*>(smem);
  const flare_scan_args_t& a = p.a;
  constexpr int STAGERS = SPLIT ? K::STAGERS : K::THREADS, ROUNDS = K::THREADS / STAGERS;
  const bool walks = !SPLIT || threadIdx.x < K::THREADS, stages = !SPLIT || !walks;
  const unsigned self = SPLIT && !walks ? threadIdx.x - K::THREADS : threadIdx.x;
  const Place<K, SPLIT ? GIVEN : ITSELF> at(p, self);
  if (ENDS && at.seg == 0) return;
  constexpr int S = K::S, P = K::P, NS = K::NS, V = K::V, LANES = K::LANES, SUB = K::SUB, CT = K::CT, APART = K::APART;
  float bias[V], D[V], sum_d[V], sum_bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = at.c0 + at.cg + i;
    bias[i] = i < at.count && a.dt_bias != nullptr ? a.dt_bias[c] : 0.0f;
    D[i] = i < at.count && a.D != nullptr ? a.D[c] : 0.0f;
    sum_d[i] = sum_bias[i] = 0.0f;
  }
  // of channel ch + j APART.  G: gradient of the state behind the token at hand, times that token's successor's factor
  uint64_t A2[CT][P], G[CT][P], dA[CT][P];
  const auto there = [&](int j) { return at.ch + j * APART < at.here; };
  const auto weight_at = [&](int j) { return (int64_t)(at.c0 + (there(j) ? at.ch + j * APART : 0)) * S + at.sub * NS; };
  const int64_t carry_at = (int64_t)blockIdx.x * a.C * S;
  float sum[CT] = {};
#pragma unroll
  for (int j = 0; j < CT; ++j)
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float* A = a.A + weight_at(j) + 2 * i;
      A2[j][i] = f2_pack(A[0] * kLog2e, A[1] * kLog2e);
      G[j][i] = dA[j][i] = 0;
    }
  if (!ENDS && p.segments > 1)
    for (int j = 0; j < CT; ++j) load_pairs<P>(p.carry + carry_at + weight_at(j), G[j]);
  const T* const zp = reinterpret_cast<const T*>(a.z);
  const int tiles = (a.N + kTile - 1) / kTile;
  const int last = at.t0 + (at.t1 - at.t0 - 1) / kTile * kTile;
  // staging
  Rows<T, K, WIDE> rows[ROUNDS];
  Raw<T, V> dy[ROUNDS], z[ROUNDS];
  const auto place = [&](int round) { return Place<K, SPLIT ? GIVEN : ITSELF>(p, self + round * STAGERS); };
  const auto fetch = [&](int t0) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const auto here = place(r);
      rows[r].load(p, here, t0);
      const int t = t0 + here.token, n = rows[r].on ? here.count : 0;
      dy[r] = load_raw<T, V>(reinterpret_cast<const T*>(a.dy) + at.b * a.dy_stride_b + t * a.dy_stride_n + at.c0 + at.cg, n, WIDE);
      if (zp != nullptr) z[r] = load_raw<T, V>(zp + at.b * a.z_stride_b + t * a.z_stride_n + at.c0 + at.cg, n, WIDE);
    }
  };
  // what the gradients of a tile take (SPLIT: fetched and formed once more)
  float delta[V], slope[V], x[V];
  Raw<T, V> dy_raw, z_raw;
  bool on = false;
  const auto lay_down = [&](int buffer) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const auto here = place(r);
      rows[r].stage(p, here, bias, sm.in[buffer], delta, slope, x);
      dy_raw = dy[r];
      z_raw = z[r];
      on = rows[r].on;
      float g[V], zf[V];
      unpack<T, V>(dy_raw, g);
      if (zp != nullptr) {
        unpack<T, V>(z_raw, zf);
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] *= zf[i] * sigmoid(zf[i]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sm.gy[buffer][here.token][at.cg + i] = on ? g[i] : 0.0f;
    }
  };
  const auto gradients = [&](int t0, int buffer) {
#pragma unroll 1
    for (int r = 0; r < ROUNDS; ++r) {
      const int token = at.token + r * (STAGERS / K::PER), t = t0 + token;
      if (SPLIT) {
        on = at.on(t);
        const int n = on ? at.count : 0;
        const Raw<T, V> xr = load_raw<T, V>(reinterpret_cast<const T*>(a.x) + at.b * a.x_stride_b + t * a.x_stride_n + at.c0 + at.cg, n, WIDE);
        const Raw<T, V> dr = load_raw<T, V>(reinterpret_cast<const T*>(a.dt) + at.b * a.dt_stride_b + t * a.dt_stride_n + at.c0 + at.cg, n, WIDE);
        dy_raw = load_raw<T, V>(reinterpret_cast<const T*>(a.dy) + at.b * a.dy_stride_b + t * a.dy_stride_n + at.c0 + at.cg, n, WIDE);
        if (zp != nullptr) z_raw = load_raw<T, V>(zp + at.b * a.z_stride_b + t * a.z_stride_n + at.c0 + at.cg, n, WIDE);
        unpack<T, V>(xr, x);
        unpack<T, V>(dr, delta);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          delta[i] += bias[i];
          slope[i] = 1.0f;
          if (a.dt_softplus) delta[i] = softplus(delta[i], slope[i]);
        }
      }
      if (t >= at.t1 || at.count <= 0) continue;
      float dx[V], ddt[V], dyf[V], gate[V], zf[V];
      unpack<T, V>(dy_raw, dyf);
      if (zp != nullptr) unpack<T, V>(z_raw, zf);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float p1 = sm.p1[buffer][token][at.cg + i], gy = sm.gy[buffer][token][at.cg + i];
        ddt[i] = fmaf(x[i], p1, sm.p2[buffer][token][at.cg + i] * (1.0f / kLog2e)) * slope[i];
        dx[i] = fmaf(delta[i], p1, D[i] * gy);
        if (!on) dx[i] = ddt[i] = 0.0f;
        sum_bias[i] += ddt[i];
        if (on) sum_d[i] = fmaf(gy, x[i], sum_d[i]);
      }
      const int64_t row = ((int64_t)at.b * a.N + t) * a.C + at.c0 + at.cg;
      store_all<T, V>(reinterpret_cast<T*>(a.dx) + row, dx, at.count, WIDE);
      store_all<T, V>(reinterpret_cast<T*>(a.ddt) + row, ddt, at.count, WIDE);
      if (zp != nullptr) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float r = sigmoid(zf[i]);
          gate[i] = on ? dyf[i] * fmaf(D[i], x[i], sm.y[buffer][token][at.cg + i]) * r * fmaf(zf[i], 1.0f - r, 1.0f) : 0.0f;
        }
        store_all<T, V>(reinterpret_cast<T*>(a.dz) + row, gate, at.count, WIDE);
      }
    }
#pragma unroll (SPLIT ? 2 : 1)
    for (int idx = self; idx < kTile * 2 * S; idx += STAGERS) {
      const int tt = idx / (2 * S), j = idx % (2 * S);
      if (t0 + tt < at.t1) {
        float v = sm.bc[buffer][tt][0][j];
#pragma unroll
        for (int w = 1; w < K::WARPS; ++w) v += sm.bc[buffer][tt][w][j];
        p.partial_bc[(((int64_t)at.b * a.N + t0 + tt) * gridDim.y + blockIdx.y) * (2 * S) + j] = v;
      }
    }
  };
  uint64_t kept[CT][P];  // the states in front of a tile
  const auto fetch_states = [&](int t0) {
    if (ENDS) return;
#pragma unroll
    for (int j = 0; j < CT; ++j) load_pairs<P>(a.keep + ((int64_t)at.b * tiles + t0 / kTile) * a.C * S + weight_at(j), kept[j]);
  };
  const auto walk = [&](int t0, int buffer) {
    const Tile<K>& in = sm.in[buffer];
    const auto& gys = sm.gy[buffer];
    uint64_t h[CT][P], tile_dA[CT][P];  // (summed tile by tile: thousands of tokens one by one would lose digits)
#pragma unroll
    for (int j = 0; j < CT; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) {
        h[j][i] = kept[j][i];
        tile_dA[j][i] = 0;
      }
    uint64_t first[CT][P];
#pragma unroll
    for (int j = 0; j < CT; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) first[j][i] = kept[j][i];
    if (t0 > at.t0) fetch_states(t0 - kTile);
    if (ENDS) {
#pragma unroll 4
      for (int t = kTile - 1; t >= 0; --t) {
        uint64_t b[P], c[P];
        load_bc<P>(&in.bc[t][at.sub * P], b, c);
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          const uint64_t d2 = *reinterpret_cast<const uint64_t*>(&in.dd[t][padded(at.ch + j * APART)]), gy = twice(gys[t][at.ch + j * APART]);
          sum[j] += low(d2);
#pragma unroll
          for (int i = 0; i < P; ++i) G[j][i] = f2_mul(f2_fma(c[i], gy, G[j][i]), factor(A2[j][i], d2));
        }
        if (DOCS && in.reset[t]) {
#pragma unroll
          for (int j = 0; j < CT; ++j) {
#pragma unroll
            for (int i = 0; i < P; ++i) G[j][i] = 0;
            sum[j] = -INFINITY;
          }
        }
      }
    } else {
      const auto move = [&](int t, uint64_t (&f)[CT][P]) {  // h over token t; its factors
        if (DOCS && in.reset[t]) {
#pragma unroll
          for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int i = 0; i < P; ++i) h[j][i] = 0;
        }
        uint64_t b[P], c[P];
        load_bc<P>(&in.bc[t][at.sub * P], b, c);
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          const ulonglong2 dd = *reinterpret_cast<const ulonglong2*>(&in.dd[t][padded(at.ch + j * APART)]);
          const uint64_t d2 = dd.x, x2 = dd.y;
#pragma unroll
          for (int i = 0; i < P; ++i) {
            f[j][i] = factor(A2[j][i], d2);
            h[j][i] = f2_fma(f[j][i], h[j][i], f2_mul(x2, b[i]));
          }
        }
      };
#pragma unroll 1
      for (int q = 0; q < kTile / SUB; ++q) {
#pragma unroll
        for (int j = 0; j < CT; ++j)
          if (q > 0) store_pairs<P>(&sm.starts[q - 1][threadIdx.x][j * NS], h[j]);
        if (q + 1 < kTile / SUB) {
#pragma unroll
          for (int k = 0; k < SUB; ++k) {
            uint64_t f[CT][P];
            move(q * SUB + k, f);
          }
        }
      }
#pragma unroll 1
      for (int q = kTile / SUB - 1; q >= 0; --q) {
        uint64_t f[SUB][CT][P], behind[SUB][CT][P], start[CT][P];  // factors; states behind the tokens and in front of them all
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          if (q > 0) load_pairs<P>(&sm.starts[q - 1][threadIdx.x][j * NS], start[j]);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            if (q == 0) start[j][i] = first[j][i];
            h[j][i] = start[j][i];
          }
        }
#pragma unroll
        for (int k = 0; k < SUB; ++k) {
          move(q * SUB + k, f[k]);
#pragma unroll
          for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int i = 0; i < P; ++i) behind[k][j][i] = h[j][i];
        }
#pragma unroll
        for (int k0 = SUB - LANES; k0 >= 0; k0 -= LANES) {
          float p1[CT][LANES], p2[CT][LANES], yv[CT][LANES];
#pragma unroll
          for (int k = LANES - 1; k >= 0; --k) {
            const int t = q * SUB + k0 + k;
            uint64_t b[P], c[P], db[P], dc[P];
            load_bc<P>(&in.bc[t][at.sub * P], b, c);
#pragma unroll
            for (int j = 0; j < CT; ++j) {
              const ulonglong2 dd = *reinterpret_cast<const ulonglong2*>(&in.dd[t][padded(at.ch + j * APART)]);
              const uint64_t d2 = dd.x, x2 = dd.y, gy = twice(gys[t][at.ch + j * APART]);
              uint64_t s1 = 0, s2 = 0, s3 = 0;
#pragma unroll
              for (int i = 0; i < P; ++i) {
                const uint64_t g = f2_fma(c[i], gy, G[j][i]);
                const uint64_t before = DOCS && in.reset[t] ? 0 : k0 + k ? behind[k0 + k - 1][j][i] : start[j][i], now = behind[k0 + k][j][i];
                const uint64_t next = f2_mul(g, f[k0 + k][j][i]), u = f2_mul(next, before);
                s1 = i ? f2_fma(g, b[i], s1) : f2_mul(g, b[i]);
                s2 = i ? f2_fma(u, A2[j][i], s2) : f2_mul(u, A2[j][i]);
                s3 = i ? f2_fma(now, c[i], s3) : f2_mul(now, c[i]);
                tile_dA[j][i] = f2_fma(u, d2, tile_dA[j][i]);
                G[j][i] = next;
                db[i] = j ? f2_fma(g, x2, db[i]) : f2_mul(g, x2);
                dc[i] = j ? f2_fma(now, gy, dc[i]) : f2_mul(now, gy);
              }
              if (DOCS && in.reset[t]) {
#pragma unroll
                for (int i = 0; i < P; ++i) G[j][i] = 0;
              }
              p1[j][k] = pair_sum(s1);
              p2[j][k] = pair_sum(s2);
              yv[j][k] = pair_sum(s3);
            }
            float v[2 * NS];
#pragma unroll
            for (int i = 0; i < P; ++i) {
              f2_unpack(db[i], v[2 * i], v[2 * i + 1]);
              f2_unpack(dc[i], v[NS + 2 * i], v[NS + 2 * i + 1]);
            }
            // (a channel that does not exist has delta x = gy = 0: it adds nothing)
            const int first = channel_sums<2 * NS, LANES>(v, threadIdx.x & 31);
            if (first >= 0) {
              constexpr int R = 2 * NS * LANES >= 32 ? 2 * NS * LANES / 32 : 1;
#pragma unroll
              for (int i = 0; i < R; ++i) {
                const int j = first + i;  // (dB of this thread's states, then dC)
                sm.bc[buffer][t][threadIdx.x >> 5][(j / NS) * S + at.sub * NS + j % NS] = v[i];
              }
            }
          }
          const int t = q * SUB + k0 + at.sub;
#pragma unroll
          for (int j = 0; j < CT; ++j) {
            sm.p1[buffer][t][at.ch + j * APART] = lane_sums<LANES>(p1[j], at.sub);
            sm.p2[buffer][t][at.ch + j * APART] = lane_sums<LANES>(p2[j], at.sub);
            if (zp != nullptr) sm.y[buffer][t][at.ch + j * APART] = lane_sums<LANES>(yv[j], at.sub);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) dA[j][i] = f2_add(dA[j][i], tile_dA[j][i]);
    }
  };
  if (stages) fetch(last);
  if (walks) fetch_states(last);
  if (SPLIT) {
    if (stages) {
      lay_down(0);
      if (last > at.t0) fetch(last - kTile);
    }
    // (loops of their own: neither side's registers are the other's)
    const auto tile_done = [] { asm volatile("bar.sync 1, %0;" ::"n"(K::THREADS + K::STAGERS) : "memory"); };
    tile_done();
    int buffer = 0;
    if (walks) {
#pragma unroll 1
      for (int t0 = last; t0 >= at.t0; t0 -= kTile, buffer ^= 1) {
        walk(t0, buffer);
        tile_done();
      }
    } else {
#pragma unroll 1
      for (int t0 = last; t0 >= at.t0; t0 -= kTile, buffer ^= 1) {
        if (t0 < last) gradients(t0 + kTile, buffer ^ 1);
        if (t0 > at.t0) {
          lay_down(buffer ^ 1);
          if (t0 - kTile > at.t0) fetch(t0 - 2 * kTile);
        }
        tile_done();
      }
      gradients(at.t0, buffer ^ 1);
    }
  } else {
#pragma unroll 1
    for (int t0 = last; t0 >= at.t0; t0 -= kTile) {
      lay_down(0);
      __syncthreads();
      if (t0 > at.t0) fetch(t0 - kTile);
      walk(t0, 0);
      __syncthreads();
      if (!ENDS) gradients(t0, 0);
    }
  }
  if (ENDS) {
#pragma unroll
    for (int j = 0; j < CT; ++j)
      if (there(j)) {
        store_pairs<P>(p.carry + carry_at + weight_at(j), G[j]);
        if (at.sub == 0) p.decay[(int64_t)blockIdx.x * a.C + at.c0 + at.ch + j * APART] = sum[j];
      }
    return;
  }
  float* out = p.partial_w + (int64_t)blockIdx.x * weight_sums(a);
#pragma unroll
  for (int j = 0; j < CT; ++j)
    if (walks && there(j)) store_pairs<P>(out + weight_at(j), dA[j]);
  // the sums that the staging threads hold, over the tokens of a tile
  __syncthreads();
  if (stages) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sm.p1[0][at.token][at.cg + i] = sum_d[i];
      sm.p2[0][at.token][at.cg + i] = sum_bias[i];
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < at.here) {
    float d = 0.0f, e = 0.0f;
    for (int t = 0; t < STAGERS / K::PER; ++t) {
      d += sm.p1[0][t][threadIdx.x];
      e += sm.p2[0][t][threadIdx.x];
    }
    out[(int64_t)a.C * S + at.c0 + threadIdx.x] = d;
    out[(int64_t)a.C * (S + 1) + at.c0 + threadIdx.x] = e;
  }
}

// One token.  Bound by memory: every state is read and written once.  Four threads share four channels (eight apart, so that a warp's
// loads are contiguous): each prepares one of them (softplus, gate) and holds a quarter of the states of all four, for several rows of the
// batch one after the other, whose A is read once.  B=256 C=8192 S=16: 52.8 us, 5.1 TB/s.
template <typename T, int NS>
__global__ void __launch_bounds__(256) decode_kernel(const ScanParams p, int rows) {
  pdl_begin();
  constexpr int S = NS * 4, P = NS / 2;
  const flare_scan_args_t& a = p.a;
  const int lane = threadIdx.x & 31, quad = lane >> 2, sub = lane & 3;
  const int base = (blockIdx.x * 8 + (threadIdx.x >> 5)) * 32;
  if (base >= a.C) return;
  const int mine = base + quad + 8 * sub;  // the channel that this thread prepares
  const bool have = mine < a.C;
  const float bias = have && a.dt_bias != nullptr ? a.dt_bias[mine] : 0.0f, D = have && a.D != nullptr ? a.D[mine] : 0.0f;
  uint64_t A2[4][P];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = min(base + quad + 8 * k, a.C - 1);
    load_pairs<P>(a.A + (int64_t)c * S + sub * NS, A2[k]);
#pragma unroll
    for (int i = 0; i < P; ++i) A2[k][i] = f2_mul(A2[k][i], twice(kLog2e));
  }
  const int group = base / p.channels;
  const bool one_group = min(base + 31, a.C - 1) / p.channels == group;
  const int b_end = min(a.B, (int)(blockIdx.y + 1) * rows);
#pragma unroll 1
  for (int b = blockIdx.y * rows; b < b_end; ++b) {
    float* const states = a.state_out + ((int64_t)b * a.C + base + quad) * S + sub * NS;
    uint64_t h[4][P], bv[P], cv[P];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (base + quad + 8 * k < a.C) load_pairs<P>(states + 8 * k * S, h[k]);
    float x = 0.0f, delta = 0.0f, z = 0.0f, slope;
    if (have) {
      x = to_float<T>(reinterpret_cast<const T*>(a.x)[b * a.x_stride_b + mine]);
      delta = to_float<T>(reinterpret_cast<const T*>(a.dt)[b * a.dt_stride_b + mine]) + bias;
      if (a.z != nullptr) z = to_float<T>(reinterpret_cast<const T*>(a.z)[b * a.z_stride_b + mine]);
    }
    const auto projections = [&](int g) {
      const T* bp = reinterpret_cast<const T*>(a.b) + b * a.b_stride_b + g * a.b_stride_g + sub * NS;
      const T* cp = reinterpret_cast<const T*>(a.c) + b * a.c_stride_b + g * a.c_stride_g + sub * NS;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        bv[i] = f2_pack(to_float<T>(bp[2 * i]), to_float<T>(bp[2 * i + 1]));
        cv[i] = f2_pack(to_float<T>(cp[2 * i]), to_float<T>(cp[2 * i + 1]));
      }
    };
    if (one_group) projections(group);
    if (a.dt_softplus) delta = softplus(delta, slope);
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = base + quad + 8 * k;
      const float dk = __shfl_sync(0xffffffffu, delta, quad * 4 + k), xk = __shfl_sync(0xffffffffu, x, quad * 4 + k);
      y[k] = 0.0f;
      if (c < a.C) {
        if (!one_group) projections(c / p.channels);
        uint64_t acc = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          h[k][i] = f2_fma(factor(A2[k][i], twice(dk)), h[k][i], f2_mul(twice(dk * xk), bv[i]));
          acc = i ? f2_fma(h[k][i], cv[i], acc) : f2_mul(h[k][i], cv[i]);
        }
        store_pairs<P>(states + 8 * k * S, h[k]);
        y[k] = pair_sum(acc);
      }
    }
    float out = fmaf(D, x, lane_sums<4>(y, sub));
    if (a.z != nullptr) out *= z * sigmoid(z);
    if (have) reinterpret_cast<T*>(a.y)[(int64_t)b * a.C + mine] = from_float<T>(out);
  }
}

// Rows of the batch that a thread takes: four, where that leaves two blocks for every SM
template <typename T, int NS>
int launch_decode(const ScanParams& p, cudaStream_t stream) {
  const int64_t blocks = (p.a.C + 255) / 256;
  int rows = 4;
  while (rows > 1 && blocks * ((p.a.B + rows - 1) / rows) < 2 * (int64_t)sm_count()) rows /= 2;
  while ((p.a.B + rows - 1) / rows > 65535) rows *= 2;
  LaunchTimer timer("scan_decode_kernel", stream);
  FLARE_CUDA_CHECK(launch_pdl(decode_kernel<T, NS>, dim3((unsigned)blocks, (unsigned)((p.a.B + rows - 1) / rows)), dim3(256), 0, stream, p, rows));
  return FLARE_OK;
}

template <typename T, typename K, bool BACKWARD>
int launch_walk(bool ends, const ScanParams& p, cudaStream_t stream) {
  constexpr bool STAGERS = BACKWARD && K::STAGERS > 0;
  using Smem = typename std::conditional<BACKWARD, BackwardSmem<K, STAGERS>, ForwardSmem<K>>::type;
  static_assert(sizeof(Smem) <= (size_t)kMaxDynamicSmem, "shared memory");
  static_assert(K::CH == block_channels(K::S), "channels of a block");
  const dim3 grid((unsigned)(p.a.B * (int64_t)p.segments), (unsigned)(p.a.G * p.blocks_c));
  // Where every block has an SM of its own, twice the threads hide what lies between two walks (B=4 N=4096 C=2048 bf16: 317 us, 395 without; N=2048 fp32: 184,
  // 278); where blocks share one, they do that for one another (B=8 N=2048 C=4096: 666 us, 590 without).
  const bool split = !BACKWARD && !ends && p.wide && (int64_t)grid.x * grid.y <= sm_count();
  const auto pick = [&](auto ends_, auto wide, auto docs) -> void (*)(ScanParams) {
    constexpr bool E = decltype(ends_)::value, W = decltype(wide)::value, DOCS = decltype(docs)::value;
    if constexpr (BACKWARD) return backward_kernel<T, K, E, W, DOCS, STAGERS && !E>;
    else if constexpr (E) return forward_kernel<T, K, E, W, DOCS, false>;
    else return split ? forward_kernel<T, K, E, W, DOCS, true> : forward_kernel<T, K, E, W, DOCS, false>;
  };
  const auto with_docs = [&](auto ends_, auto wide) { return p.a.documents != nullptr ? pick(ends_, wide, std::true_type()) : pick(ends_, wide, std::false_type()); };
  const auto with_wide = [&](auto ends_) { return p.wide ? with_docs(ends_, std::true_type()) : with_docs(ends_, std::false_type()); };
  auto* const kernel = ends ? with_wide(std::true_type()) : with_wide(std::false_type());
  FLARE_CUDA_CHECK(allow_smem(kernel));
  LaunchTimer timer(BACKWARD ? (ends ? "scan_backward_kernel (ends)" : "scan_backward_kernel") : (ends ? "scan_forward_kernel (ends)" : "scan_forward_kernel"),
                    stream);
  FLARE_CUDA_CHECK(launch_pdl(kernel, grid, dim3(split ? 2 * K::THREADS : K::THREADS + (STAGERS && !ends ? K::STAGERS : 0)), sizeof(Smem), stream, p));
  return FLARE_OK;
}

}  // namespace

template <typename T>
int launch(Pass pass, const ScanParams& p, cudaStream_t stream) {
  constexpr int STAGERS = sizeof(T) == 2 ? 128 : 0;  // (the rows of fp32 take the registers that they would save: S=8 B=2 N=2048 C=2048 402 us, 321 without)
  const bool ends = pass == FORWARD_ENDS || pass == BACKWARD_ENDS;
  switch (pass) {
    case DECODE:
      return p.a.S == 8 ? launch_decode<T, 2>(p, stream) : p.a.S == 16 ? launch_decode<T, 4>(p, stream) : launch_decode<T, 8>(p, stream);
    case FORWARD:
    case FORWARD_ENDS:
      // (16 states in fours: B=8 N=2048 C=4096 594 us, B=1 N=8191 C=2048 241; in twos, with twice the threads: 705, 332)
      if (p.a.S == 8) return launch_walk<T, Config<8, 2, 256, 2>, false>(ends, p, stream);
      if (p.a.S == 16) return launch_walk<T, Config<16, 4, 256, 2>, false>(ends, p, stream);
      return launch_walk<T, Config<32, 4, 256, 2>, false>(ends, p, stream);
    default:
      if (p.a.S == 8) return launch_walk<T, Config<8, 2, 256, 1, 1, STAGERS>, true>(ends, p, stream);
      // (16 states in twos, two channels a thread, whose sums over channels cost half the exchanges, and four warps more that stage: B=4 N=4096 C=2048
      // 1 053 us; without those 1 169; one channel a thread and twice the threads 1 183; in fours 1 235 with the registers of one block on an SM, 2 000
      // where two share them.  With `setmaxnreg` between the two sides 1 711, spills; sums over lanes exchanged token by token, in fewer registers, 1 217)
      if (p.a.S == 16) return launch_walk<T, Config<16, 2, 256, 1, 2, STAGERS>, true>(ends, p, stream);
      return launch_walk<T, Config<32, 4, 256>, true>(ends, p, stream);
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
    in = sum == -INFINITY ? end : fmaf(expf(A * sum), in, end);
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
  if (a.N > 0x7fffffff - 1024 || (int64_t)a.G * ((a.C / a.G + 31) / 32) > 65535) return FLARE_ERR_UNSUPPORTED;
  if (a.x == nullptr || a.dt == nullptr || a.A == nullptr || a.b == nullptr || a.c == nullptr) return FLARE_ERR_BAD_POINTER;
  for (const void* q : {(const void*)a.A, (const void*)a.state_in, (const void*)a.state_out, (const void*)a.keep})
    if (reinterpret_cast<uintptr_t>(q) & 15u) return FLARE_ERR_BAD_POINTER;
  return FLARE_OK;
}

// Segments where the channels alone leave SMs idle: as many as fill two blocks per SM, of four tiles at least.  Below three they
// do not pay for the pass over their ends.
void plan(ScanParams& p, const flare_scan_args_t& a) {
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.channels = a.C / a.G;
  const int block = block_channels(a.S);
  p.blocks_c = (p.channels + block - 1) / block;
  const int64_t blocks = (int64_t)a.B * a.G * p.blocks_c, tiles = (a.N + kTile - 1) / kTile;
  int64_t segments = 2 * (int64_t)sm_count() / blocks;
  if (segments > tiles / 4) segments = tiles / 4;
  if (segments < 3) segments = 1;
  const int64_t per = (tiles + segments - 1) / segments;
  p.seg_tokens = (int)(per * kTile);
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
  return (size_t)args->B * ((args->N + kTile - 1) / kTile) * args->C * args->S * 4;
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
