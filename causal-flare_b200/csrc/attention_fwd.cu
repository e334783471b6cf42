// Attention forward on tcgen05: y = softmax(scores) V in one pass over the keys.
//
// One CTA per head and 256 queries, as two groups of 128 (a thread is a query is a lane of tensor memory).  Per tile of 64 keys and
// group: S = Q K^T into tensor memory, the group's threads read their rows, take the running maximum and lay P = exp2(S - m) down
// over S as packed 16-bit values, O += P V takes its A operand from there.  S has two buffers per group, so that a group finds its next
// scores when it is done with a tile; with one buffer of 128 keys it waited
// for its own two products and their hand-overs every time: 5 100 cycles for 128 keys, of which its own work took 3 000.
// O stays in tensor memory; it is rescaled only where the maximum has grown by
// more than 2^8 since the frame was set (exact: the frame cancels in O / l).  In fp16 P is laid down times 2^7: up to 2^15, and normal numbers down to
// 2^-21 (a weight of 1.4 2^-20 beside one of 1 was 1.4 % off).
// Sums are of the unrounded weights, in fp32; P is rounded once, to the type of V, which is what the products take.
//
// Tensor memory: S / P of the groups, two buffers each, at 0 and 128, O at 256 and 384.  Shared memory (D = 128): Q 64 KB, the
// first two tiles of K, four stages of a tile of V and one of K.  Floors per 64 keys and both groups, in cycles: products 1 024 (M = 128, N = 64 from shared memory: 1 280),
// exponentials 1 024.  B200, B=2 N=4096 H=16 D=128 bf16: 150 us (0.55 of the measured matrix rate), with a cap 192: the caps' seven
// products and sums for every score come on top of a group's own work, which is what bounds either.
#include <limits.h>

#include "attention_tc.cuh"

namespace flare {
namespace attn {

#ifdef FLARE_ATTN_DB

namespace {

constexpr int kThreads = 320;  // two groups of four warps, products, copies
constexpr int kWarpMma = 8, kWarpTma = 9;
constexpr float kGrowth = 8.0f;

constexpr int kKeys = 64, kStages = 4, kAhead = 2;

struct Misc {
  uint64_t q_full[2], head_full[kAhead], full[kStages], empty[kStages], s_full[2][2], p_ready[2][2], o_free[2], o_done[2];
  uint32_t tmem_base;
  volatile int abort_flag;
};

template <int DB>
struct Layout {
  static constexpr int Q = DB * 16384, TILE = DB * 8192;
  // keys of the first tiles, then stages: the values of tile n and the keys of tile n + 2, which are needed at the same time
  static constexpr int HEAD = 2 * Q, RING = HEAD + kAhead * TILE, STAGE = 2 * TILE, MISC = RING + kStages * STAGE, BYTES = MISC + (int)sizeof(Misc) + 1024;
  static_assert(BYTES <= kMaxDynamicSmem, "shared memory");
};

template <int DB, bool F16, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
attention_forward_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const AttnParams p) {
  using L = Layout<DB>;
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  Misc* const misc = reinterpret_cast<Misc*>(smem + L::MISC);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int g = 0; g < 2; ++g) {
      mbar_init(&misc->q_full[g], 1);
      mbar_init(&misc->o_free[g], 1);
      mbar_init(&misc->o_done[g], 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&misc->s_full[g][i], 1);
        mbar_init(&misc->p_ready[g][i], 4);
      }
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&misc->full[i], 1);
      mbar_init(&misc->empty[i], 1);
    }
    for (int i = 0; i < kAhead; ++i) mbar_init(&misc->head_full[i], 1);
    misc->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kWarpMma) {
    tmem_alloc(&misc->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = misc->tmem_base;
  pdl_wait();

  const int lanes = p.B * p.H, block = gridDim.x / lanes - 1 - blockIdx.x / lanes;  // (causal: the longest first)
  const int b = blockIdx.x % lanes / p.H, h = blockIdx.x % p.H, kv = h / (p.H / p.J), q0 = block * 256;
  // tiles of keys of each group: both begin with the first that one of them sees
  int last[2], j0 = INT_MAX;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int tile = block * 2 + g;
    const int2 s = tile * 128 < p.masks.Nqp ? p.masks.query_span[b * (p.masks.Nqp >> 7) + tile] : make_int2(0, 0);
    last[g] = s.y > s.x ? (s.y + kKeys - 1) / kKeys : 0;
    if (s.y > s.x) j0 = min(j0, s.x / kKeys);
  }
  const int tiles[2] = {max(0, last[0] - j0), max(0, last[1] - j0)}, total = max(tiles[0], tiles[1]);
  bool ok = true;
  const auto wait_one = [&](uint64_t* bar, uint32_t parity) { return wait_or_abort(bar, parity, &misc->abort_flag, 8); };
  // (whole warps give up together)
  const auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_one(bar, parity)) != 0; };

  if (warp == kWarpTma) {
    if (elect_one()) {
      const auto load = [&](const CUtensorMap* map, uint8_t* to, uint64_t* bar, int n) {
        for (int d = 0; d < DB; ++d) tma_load_4d(to + d * 8192, map, bar, d * 64, kv, (j0 + n) * kKeys, b);
      };
      for (int g = 0; g < 2; ++g)
        if (tiles[g] > 0) {
          mbar_arrive_expect_tx(&misc->q_full[g], L::Q);
          for (int d = 0; d < DB; ++d) tma_load_4d(smem + g * L::Q + d * 16384, &tm_q, &misc->q_full[g], d * 64, h, q0 + g * 128, b);
        }
      for (int n = 0; n < min(kAhead, total); ++n) {
        mbar_arrive_expect_tx(&misc->head_full[n], L::TILE);
        load(&tm_k, smem + L::HEAD + n * L::TILE, &misc->head_full[n], n);
      }
      for (int n = 0; n < total; ++n) {
        const int s = n % kStages;
        if (!(ok = wait_one(&misc->empty[s], ((n / kStages) & 1) ^ 1))) break;
        uint8_t* const stage = smem + L::RING + s * L::STAGE;
        const bool more = n + kAhead < total;
        mbar_arrive_expect_tx(&misc->full[s], more ? 2 * L::TILE : L::TILE);
        load(&tm_v, stage, &misc->full[s], n);
        if (more) load(&tm_k, stage + L::TILE, &misc->full[s], n + kAhead);
      }
    }
  } else if (warp == kWarpMma) {
    if (elect_one()) {  // (one thread all along: what it does between two products is on every tile's way)
      constexpr uint32_t ID_S = make_idesc<F16>(128, kKeys, 0, 0);    // Q, K: K-major
      constexpr uint32_t ID_O = make_idesc<F16>(128, 64 * DB, 0, 1);  // P (tensor memory), V: MN-major
      const uint64_t dq[2] = {make_desc_sw128(smem_u32(smem), 16, 1024), make_desc_sw128(smem_u32(smem + L::Q), 16, 1024)};
      const uint64_t dk0 = make_desc_sw128(smem_u32(smem), 16, 1024), dv0 = make_desc_sw128(smem_u32(smem + L::RING), 8192, 1024);
      const auto scores = [&](int g, int buffer, int at) {  // of the keys that lie at byte `at`
        const uint64_t dk = dk0 + (uint64_t)(at >> 4);
#pragma unroll
        for (int i = 0; i < 4 * DB; ++i)
          mma_ss(tmem + g * 128 + buffer * 64, kmaj_step(dq[g], i), dk + (uint64_t)(((i >> 2) * 8192 + (i & 3) * 32) >> 4), ID_S, i > 0);
        tc_commit(&misc->s_full[g][buffer]);
      };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        if (ok && n < total) ok = wait_one(&misc->head_full[n], 0);
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (ok && n < tiles[g] && (ok = wait_one(&misc->q_full[g], 0))) {
            tc_fence_after_sync();
            scores(g, n, L::HEAD + n * L::TILE);
          }
      }
#pragma unroll 1
      for (int n = 0; ok && n < total; ++n) {
        const int s = n % kStages, buffer = n & 1;
        if (!(ok = wait_one(&misc->full[s], (n / kStages) & 1))) break;
        const uint64_t dv = dv0 + (uint64_t)((s * L::STAGE) >> 4);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (n >= tiles[g]) continue;
          if (!(ok = wait_one(&misc->p_ready[g][buffer], (n >> 1) & 1))) break;
          tc_fence_after_sync();
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i)
            mma_ts(tmem + 256 + g * 128, tmem + g * 128 + buffer * 64 + i * 8, mnmaj_step(dv, i), ID_O, i > 0 || n > 0);
          tc_commit(&misc->o_free[g]);
          if (n + 1 == tiles[g]) tc_commit(&misc->o_done[g]);
          if (n + kAhead < tiles[g]) scores(g, buffer, L::RING + s * L::STAGE + L::TILE);  // (behind the product that reads P where S goes: products run in order)
        }
        if (ok) tc_commit(&misc->empty[s]);
      }
    }
  } else {
    const int g = warp >> 2, row = (warp & 3) * 32 + lane, i = q0 + g * 128 + row;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16), ts = tl + g * 128, to = tl + 256 + g * 128;
    const bool inside = i < p.masks.Nqp;
    const int2 keys = inside ? p.masks.range[(int64_t)b * p.masks.Nqp + i] : make_int2(0, 0);
    const int position = i + (p.masks.cached != nullptr ? p.masks.cached[b] : 0);
    const ScoreScale sc = score_scale(p, h);
    const CapSeries series(sc.in);
    DirtyTiles dirty(p.masks, b);
    float m = -INFINITY, sum = 0.0f;
#pragma unroll 1
    for (int n = 0; n < tiles[g]; ++n) {
      const int key0 = (j0 + n) * kKeys;
      const uint32_t tp = ts + (n & 1) * 64;
      if (!(ok = wait(&misc->s_full[g][n & 1], (n >> 1) & 1))) break;
      tc_fence_after_sync();
      uint32_t s[2][32];
      tmem_ld32(tp, s[0]);
      tmem_ld32(tp + 32, s[1]);
      if (dirty(j0 + n)) {  // (both groups may clear the same rows: zeros over zeros)
        const int stage = n % kStages;
        if (!(ok = wait(&misc->full[stage], (n / kStages) & 1))) break;
        if (row < kKeys) clear_row<DB, kKeys>(smem + L::RING + stage * L::STAGE, p.masks, b, p.Nk, key0, row);
        fence_proxy_async_smem();
      }
      tmem_wait_ld();
      tmem_fence_regs(s[0]);
      tmem_fence_regs(s[1]);
      const bool full = __all_sync(0xffffffffu, keys.x <= key0 && keys.y >= key0 + kKeys) != 0;
      unsigned in_sight[2];  // a bit for every key
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = min(max(keys.x - key0 - c * 32, 0), 32), to_ = min(max(keys.y - key0 - c * 32, 0), 32);
        in_sight[c] = (unsigned)(((1ull << to_) - 1) & ~((1ull << from) - 1));
      }
      // Weights are formed in the frame so far, caps and biases on the way, the maximum behind them: only where it has grown too far (a
      // few of the first tiles) are they formed once more.  So no exponential waits for the maximum, and caps, biases and exponentials,
      // which have pipes of their own, are worked on side by side.  Not so the first tile, and what needs masks or the other form of caps.
      const float unit = BIAS ? 1.0f : sc.unit, d0 = (float)(position - key0);
      uint32_t w[2][16];
      float part[4], t4[4];
      const auto weights = [&](auto raw_) {  // raw: the scores are products still
        constexpr bool RAW = decltype(raw_)::value;
        const uint64_t frame2 = twice(m == -INFINITY ? 0.0f : kFrameLift<F16> - m), unit2 = twice(unit);
        uint64_t sum2[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int col = c * 32 + 2 * k;
            uint64_t x = f2_pack(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1]));
            float lo, hi;
            if (RAW && (CAP || BIAS)) {
              if (CAP) x = series(x);
              if (BIAS) x = f2_fma(twice(-sc.slope), f2_pack(fabsf(d0 - (float)col), fabsf(d0 - (float)(col + 1))), f2_mul(x, twice(sc.unit)));
              f2_unpack(x, lo, hi);
              s[c][2 * k] = __float_as_uint(lo);
              s[c][2 * k + 1] = __float_as_uint(hi);
            }
            f2_unpack(BIAS ? f2_add(x, frame2) : f2_fma(x, unit2, frame2), lo, hi);
            lo = ex2_approx(lo);
            hi = ex2_approx(hi);
            sum2[k & 1] = f2_add(sum2[k & 1], f2_pack(lo, hi));
            w[c][k] = pack2<F16>(lo, hi);
          }
        f2_unpack(sum2[0], part[0], part[1]);
        f2_unpack(sum2[1], part[2], part[3]);
      };
      const bool at_once = n > 0 && full && (!CAP || all_small(s[0], s[1], series));
      if (at_once) {
        weights(std::true_type());
      } else {
        if (CAP) {
          if (!full) {  // (what lies out of sight does not choose the form)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!(in_sight[c] >> k & 1)) s[c][k] = 0u;
          }
          cap_scores(s[0], series);
          cap_scores(s[1], series);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            if (BIAS) s[c][k] = __float_as_uint(fmaf(-sc.slope, fabsf(d0 - (float)(c * 32 + k)), __uint_as_float(s[c][k]) * sc.unit));
            if (!(in_sight[c] >> k & 1)) s[c][k] = 0xff800000u;  // -inf
          }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t* const v = s[c >> 1] + (c & 1) * 16;
        t4[c] = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
#pragma unroll
        for (int k = 2; k < 16; k += 2) t4[c] = fmax3(t4[c], __uint_as_float(v[k]), __uint_as_float(v[k + 1]));
      }
      const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * unit;
      const bool grow = top > m + kGrowth || (m == -INFINITY && top > m), any = __any_sync(0xffffffffu, grow);
      if (any && n > 0) {
        // O is at rest once the product of the tile before is done.  (That of the one before it is: these scores were issued behind it,
        // so the barrier is in this phase or through with it.)
        if (!(ok = wait(&misc->o_free[g], (n - 1) & 1))) break;
        tc_fence_after_sync();
        const float f = grow ? ex2_approx(m - top) : 1.0f;
        sum *= f;
#pragma unroll 1
        for (int c = 0; c < 2 * DB; ++c) {
          uint32_t o[32];
          tmem_read<32>(to + c * 32, o);
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
          tmem_st32(to + c * 32, o);
        }
      }
      if (grow) m = top;
      if (any || !at_once) weights(std::false_type());
      tmem_st16(tp, w[0]);
      tmem_st16(tp + 16, w[1]);
      tmem_wait_st();
      tc_fence_before_sync();
      warp_arrive(&misc->p_ready[g][n & 1], lane);
      sum += (part[0] + part[1]) + (part[2] + part[3]);
    }
    if (ok && tiles[g] > 0) ok = wait(&misc->o_done[g], 0);
    if (ok) {
      tc_fence_after_sync();
      const float inv = sum > 0.0f ? 1.0f / sum : sum != sum ? sum : 0.0f;
      uint16_t* const y = reinterpret_cast<uint16_t*>(p.y) + (((int64_t)b * p.Nq + i) * p.H + h) * p.D;
#pragma unroll
      for (int c = 0; c < 2 * DB; ++c) {
        uint32_t o[32];
        if (tiles[g] > 0) {
          tmem_read<32>(to + c * 32, o);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
        }
        if (i < p.Nq) store_columns<F16>(y, c * 32, p.D, o, inv);
      }
      // with its sign changed, as the backward adds it (a query without keys: -inf, so that every weight formed with it is 0)
      if (p.lse != nullptr && inside) p.lse[((int64_t)b * p.H + h) * p.masks.Nqp + i] = sum == 0.0f ? -INFINITY : -(m + (__log2f(sum) - kFrameLift<F16>));
    }
  }
  if (!ok) {
    misc->abort_flag = 1;
    atomicOr(p.err, 1);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kWarpMma) tmem_dealloc(tmem, 512);
}

template <bool F16>
int launch(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream) {
  constexpr int DB = FLARE_ATTN_DB;
  CUtensorMap q, k, v;
  if (!head_map(&q, a.q, a.B, a.Nq, a.H, a.D, a.q_stride_b, a.q_stride_n, a.q_stride_h, 128) ||
      !head_map(&k, a.k, a.B, a.Nk, a.J, a.D, a.k_stride_b, a.k_stride_n, a.k_stride_h, kKeys) ||
      !head_map(&v, a.v, a.B, a.Nk, a.J, a.D, a.v_stride_b, a.v_stride_n, a.v_stride_h, kKeys))
    return FLARE_ERR_CUDA;
  const bool cap = p.cap > 0.0f, bias = p.slopes != nullptr;
  auto* const kernel = cap ? (bias ? attention_forward_kernel<DB, F16, true, true> : attention_forward_kernel<DB, F16, true, false>)
                           : (bias ? attention_forward_kernel<DB, F16, false, true> : attention_forward_kernel<DB, F16, false, false>);
  FLARE_CUDA_CHECK(allow_smem(kernel));
  const int64_t blocks = (int64_t)((a.Nq + 255) / 256) * a.B * a.H;
  if (blocks > 0x7fffffff) return FLARE_ERR_UNSUPPORTED;
  LaunchTimer timer("attention_forward_kernel", stream);
  FLARE_CUDA_CHECK(launch_pdl(kernel, dim3((unsigned)blocks), dim3(kThreads), Layout<DB>::BYTES, stream, q, k, v, p));
  return FLARE_OK;
}

}  // namespace

template <int DB>
int launch_forward_db(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream);
template <>
int launch_forward_db<FLARE_ATTN_DB>(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream) {
  return a.dtype == FLARE_F16 ? launch<true>(a, p, stream) : launch<false>(a, p, stream);
}

#else

template <int DB>
int launch_forward_db(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream);
template <>
int launch_forward_db<1>(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream);
template <>
int launch_forward_db<2>(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream);

int launch_forward_tc(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream) {
  return a.D <= 64 ? launch_forward_db<1>(a, p, stream) : launch_forward_db<2>(a, p, stream);
}

#endif

}  // namespace attn
}  // namespace flare
