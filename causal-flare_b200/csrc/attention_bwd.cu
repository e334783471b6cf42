// Attention backward on tcgen05, deterministic: one kernel for dK and dV, one for dQ, the same code on either side.
//
//   P = exp2(scores - lse),  dS = P (dP - delta), dP = dY V^T, delta = <dY, y>; behind the cap dS *= 1 - tanh^2
//   (of a saturated score that is off by up to 2^-23, as tanh itself is)
//   dV = P^T dY,  dK = scale dS^T Q,  dQ = scale dS K
//
// A CTA keeps 128 rows of its own side (KEYS: K and V; else Q and dY) and walks tiles of 64 rows of the other: S = X0 Y0^T and
// dP = X1 Y1^T into tensor memory, rows of the own side on the lanes; the threads turn them into P and dS, laid down over S and dP
// as packed 16-bit values, from where the products that are summed over the walk take their A operand (dV += P Y1,
// dK or dQ += dS Y0): neither P nor dS passes through shared memory, and no gradient is added by two CTAs (a key head's dK and dV walk its
// query heads one after the other).  The price is S and dP twice and dS in two parts: 18 D instead of 10 D operations for a pair.  Two slots take every
// other tile, with eight warps each (32 of the 64 columns a warp), so that one's exponentials run under the other's products.
// B200, B=2 N=4096 H=16 D=128 bf16: 550 us for both kernels (0.67 of the measured matrix rate for 18 D), with a cap 632.
//
// fp16 holds 40 powers of two, and dS of ordinary gradients (1e-6) and of scaled ones (1e5) lie at its ends or behind them: dS is laid down times a
// power of two, taken out again with the last product's factor.  |dS| <= 2 |dY| |V| of the longest rows, so 2^e |dS| <= 2^14 (and a factor of four
// in hand for P above 1, which is as far off as large scores are): one e for a query, and for a key head's dK one for the row of the batch.  The sizes above:
// 590 us in fp16, of which the norms that e is taken from are 20.
//
// Tensor memory: two slots of S 64, dP 64; sums of dS and P products at 256 and 384 (the queries' kernel: its own tiles at 384).  P is rounded once, to the type of the
// operands it meets (in fp16 times 2^14: weights of 1e-5, of rows of 1e5 keys, lost two bits); dS goes to its product as a rounded value and what that
// lost, rounded again: rounded once it made dK and dQ 1.6 times as far off as their own rounding does.  Everything in front of that, and the sums, is fp32.
#include "attention_tc.cuh"

namespace flare {
namespace attn {

#ifdef FLARE_ATTN_DB

namespace {

constexpr int kThreads = 576;  // four groups of four warps, products, copies
constexpr int kWarpMma = 16, kWarpTma = 17;
constexpr int kStages = 4, kWalk = 64;

struct Stats {  // of a tile of queries (KEYS); lse and delta with their signs changed
  float lse[kWalk], delta[kWalk];
  int2 keys[kWalk];
};
struct Misc {
  alignas(16) Stats stats[kStages];
  uint64_t own_full, own_ready, full[kStages], empty[kStages], s_full[2], w_ready[2], done;
  uint32_t tmem_base;
  volatile int abort_flag;
};

template <int DB>
struct Layout {
  static constexpr int OWN = DB * 16384, TILE = DB * 8192;
  static constexpr int Y = 2 * OWN, MISC = Y + kStages * 2 * TILE, BYTES = MISC + (int)sizeof(Misc) + 1024;
};

// e of 2^e |dS| <= 2^14, |dS| <= 2 |dy| |v| (squares given; nothing to scale: 0).  Norms of fp16 rows are below 2^20: e >= -28; up to 60, where fp32
// still holds everything.
__device__ __forceinline__ int range_exponent(float dy2, float v2) {
  const float bound = sqrtf(dy2) * sqrtf(v2);
  return bound > 0.0f ? min(12 - ilogbf(bound), 60) : 0;
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }

// contiguous bytes, 16-byte aligned on both sides
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int DB, bool F16, bool CAP, bool BIAS, bool KEYS>
__global__ void __launch_bounds__(kThreads, 1)
attention_backward_kernel(const __grid_constant__ CUtensorMap tm_x0, const __grid_constant__ CUtensorMap tm_x1,
                          const __grid_constant__ CUtensorMap tm_y0, const __grid_constant__ CUtensorMap tm_y1, const AttnParams p) {
  using L = Layout<DB>;
  constexpr uint32_t T_DS = 256, T_P = 384, T_X = 384;  // (queries: no sum of P products, their two own tiles instead)
  constexpr uint32_t LOW = KEYS ? 16 : 0;  // of the 32 columns of a half's scores: where the lower part of dS goes
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  Misc* const misc = reinterpret_cast<Misc*>(smem + L::MISC);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&misc->own_full, 1);
    mbar_init(&misc->own_ready, 16);
    mbar_init(&misc->done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&misc->s_full[i], 1);
      mbar_init(&misc->w_ready[i], 8);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&misc->full[i], 1);
      mbar_init(&misc->empty[i], 1);
    }
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

  // causal: the longest walks first, those of the first keys and of the last queries
  const int group = p.H / p.J, heads = KEYS ? p.J : p.H, lanes = p.B * heads;
  const int tile = KEYS ? blockIdx.x / lanes : gridDim.x / lanes - 1 - blockIdx.x / lanes;
  const int b = blockIdx.x % lanes / heads, head = blockIdx.x % heads, x0 = tile * 128;
  const int2 span = KEYS ? p.masks.key_span[b * (p.masks.Nkp >> 7) + tile] : p.masks.query_span[b * (p.masks.Nqp >> 7) + tile];
  const int first = span.x / kWalk, per_head = span.y > span.x ? (span.y + kWalk - 1) / kWalk - first : 0;
  const int total = KEYS ? per_head * group : per_head;
  const auto row_of = [&](int n) { return (first + (KEYS ? n % per_head : n)) * kWalk; };
  const auto head_of = [&](int n) { return KEYS ? head * group + n / per_head : head / group; };
  bool ok = true;
  const auto wait_one = [&](uint64_t* bar, uint32_t parity) { return wait_or_abort(bar, parity, &misc->abort_flag, 8); };
  // (whole warps give up together)
  const auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_one(bar, parity)) != 0; };

  if (warp == kWarpTma) {
    if (total > 0 && elect_one()) {
      mbar_arrive_expect_tx(&misc->own_full, 2 * L::OWN);
      for (int d = 0; d < DB; ++d) {
        tma_load_4d(smem + d * 16384, &tm_x0, &misc->own_full, d * 64, head, x0, b);
        tma_load_4d(smem + L::OWN + d * 16384, &tm_x1, &misc->own_full, d * 64, head, x0, b);
      }
      for (int n = 0; n < total; ++n) {
        const int s = n % kStages, row = row_of(n), hd = head_of(n);
        if (!(ok = wait_one(&misc->empty[s], ((n / kStages) & 1) ^ 1))) break;
        uint8_t* const y = smem + L::Y + s * 2 * L::TILE;
        mbar_arrive_expect_tx(&misc->full[s], 2 * L::TILE + (KEYS ? (uint32_t)sizeof(Stats) : 0u));
        for (int d = 0; d < DB; ++d) {
          tma_load_4d(y + d * 8192, &tm_y0, &misc->full[s], d * 64, hd, row, b);
          tma_load_4d(y + L::TILE + d * 8192, &tm_y1, &misc->full[s], d * 64, hd, row, b);
        }
        if (KEYS) {
          const int64_t at = ((int64_t)b * p.H + hd) * p.masks.Nqp + row;
          bulk_load(misc->stats[s].lse, (F16 ? p.lse_lifted : p.lse) + at, kWalk * 4, &misc->full[s]);
          bulk_load(misc->stats[s].delta, p.delta + at, kWalk * 4, &misc->full[s]);
          bulk_load(misc->stats[s].keys, p.masks.range + (int64_t)b * p.masks.Nqp + row, kWalk * 8, &misc->full[s]);
        }
      }
    }
  } else if (warp == kWarpMma) {
    if (total > 0 && elect_one()) {  // (one thread all along: what it does between two products is on every tile's way)
      constexpr uint32_t ID_S = make_idesc<F16>(128, kWalk, 0, 0);
      constexpr uint32_t ID_SUM = make_idesc<F16>(128, 64 * DB, 0, 1);
      const auto step_y = [](uint64_t desc, int i) { return desc + (uint64_t)(((i >> 2) * 8192 + (i & 3) * 32) >> 4); };
      const uint64_t dx0 = make_desc_sw128(smem_u32(smem), 16, 1024), dx1 = make_desc_sw128(smem_u32(smem + L::OWN), 16, 1024);
      const uint32_t y = smem_u32(smem + L::Y);
      const uint64_t k0 = make_desc_sw128(y, 16, 1024), k1 = make_desc_sw128(y + L::TILE, 16, 1024);      // K-major
      const uint64_t mn0 = make_desc_sw128(y, 8192, 1024), mn1 = make_desc_sw128(y + L::TILE, 8192, 1024);  // MN-major
      const auto scores = [&](int n) {
        const int s = n % kStages, slot = n & 1;
        if (!(ok = wait_one(&misc->full[s], (n / kStages) & 1))) return;
        tc_fence_after_sync();
        const uint64_t at = (uint64_t)((s * 2 * L::TILE) >> 4);
#pragma unroll
        for (int i = 0; i < 4 * DB; ++i) {
          if (KEYS) mma_ss(tmem + slot * 128, kmaj_step(dx0, i), step_y(k0 + at, i), ID_S, i > 0);
          else mma_ts(tmem + slot * 128, tmem + T_X + i * 8, step_y(k0 + at, i), ID_S, i > 0);
        }
#pragma unroll
        for (int i = 0; i < 4 * DB; ++i) {
          if (KEYS) mma_ss(tmem + slot * 128 + 64, kmaj_step(dx1, i), step_y(k1 + at, i), ID_S, i > 0);
          else mma_ts(tmem + slot * 128 + 64, tmem + T_X + 32 * DB + i * 8, step_y(k1 + at, i), ID_S, i > 0);
        }
        tc_commit(&misc->s_full[slot]);
      };
      ok = wait_one(KEYS ? &misc->own_full : &misc->own_ready, 0);
      tc_fence_after_sync();
      if (ok) scores(0);
      if (ok && total > 1) scores(1);
      for (int n = 0; ok && n < total; ++n) {
        const int s = n % kStages, slot = n & 1;
        if (!(ok = wait_one(&misc->w_ready[slot], (n >> 1) & 1))) break;
        tc_fence_after_sync();
        const uint64_t at = (uint64_t)((s * 2 * L::TILE) >> 4);
        if (KEYS) {
#pragma unroll
          for (int i = 0; i < kWalk / 16; ++i)
            mma_ts(tmem + T_P, tmem + slot * 128 + (i >> 1) * 32 + (i & 1) * 8, mnmaj_step(mn1 + at, i), ID_SUM, i > 0 || n > 0);
        }
#pragma unroll
        for (int i = 0; i < kWalk / 16; ++i)
          mma_ts(tmem + T_DS, tmem + slot * 128 + 64 + (i >> 1) * 32 + (i & 1) * 8, mnmaj_step(mn0 + at, i), ID_SUM, i > 0 || n > 0);
#pragma unroll
        for (int i = 0; i < kWalk / 16; ++i)
          mma_ts(tmem + T_DS, tmem + slot * 128 + LOW + (i >> 1) * 32 + (i & 1) * 8, mnmaj_step(mn0 + at, i), ID_SUM, 1);
        tc_commit(&misc->empty[s]);
        if (n + 1 == total) tc_commit(&misc->done);
        if (n + 2 < total) scores(n + 2);  // (behind the products that read P and dS where it goes: products run in order)
      }
    }
  } else {
    const int slot = (warp >> 2) & 1, half = warp >> 3, row = x0 + (warp & 3) * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16), ts = tl + slot * 128 + half * 32, td = ts + 64;
    float lse = -INFINITY, delta = 0.0f;  // (signs changed)
    int2 keys = make_int2(0, 0);
    // fp16: dS times `up`, the sums of its products times `down`.  (Queries: P is not laid down, so that `up` can be part of it.  Keys: P has a factor of
    // its own, which is part of lse.)
    float up = 1.0f, down = 1.0f;
    const float* const norms = F16 ? p.largest_norms + ((int64_t)b * p.J + (KEYS ? head : head / group)) * 2 : nullptr;
    if (!KEYS) {
      const int64_t at = ((int64_t)b * p.H + head) * p.masks.Nqp + row;
      lse = p.lse[at];
      delta = p.delta[at];
      keys = p.masks.range[(int64_t)b * p.masks.Nqp + row];
      if (F16) {
        const int e = range_exponent(p.dy_norm[at], norms[1]);
        lse += (float)e;
        down = power_of_two(-e);
      }
    } else if (F16) {
      const int e = range_exponent(norms[0], norms[1]);
      up = power_of_two(e - kWeightLift);
      down = power_of_two(-e);
    }
    ScoreScale sc = score_scale(p, KEYS ? head * group : head);
    const CapSeries series(sc.in);
    DirtyTiles dirty(p.masks, b);
    if (!KEYS && total > 0) {
      // the own tiles move to tensor memory, from where products of 64 columns take them at the full rate: with both operands in shared
      // memory they are bound by its bandwidth (128 + 64 rows of 32 bytes in 32 cycles).  A quarter of the columns a warp.
      if ((ok = wait(&misc->own_full, 0))) {
        const int r = (warp & 3) * 32 + lane;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint8_t* const from = smem + t * L::OWN + (DB == 2 ? half * 16384 : 0);
          const int part = DB == 2 ? slot : half * 2 + slot;  // of the row's 128 bytes there: a half, or a quarter
          constexpr int PIECES = DB == 2 ? 4 : 2;
          uint32_t w[PIECES * 4];
#pragma unroll
          for (int c = 0; c < PIECES; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(from + swz_chunk_off(r, part * PIECES + c));
            w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
          }
          tmem_write<PIECES * 4>(tl + T_X + t * 32 * DB + (DB == 2 ? half * 32 : 0) + part * PIECES * 4, w);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        warp_arrive(&misc->own_ready, lane);
      }
    }
#pragma unroll 1
    for (int n = slot; ok && n < total; n += 2) {
      const int y0 = row_of(n), s_ = n % kStages;
      if (KEYS && BIAS) sc = score_scale(p, head_of(n));
      // (the tile has been there since before its scores; the wait on `full` makes its statistics visible to this thread)
      const bool unclean = dirty(y0 / kWalk);
      if ((KEYS || unclean) && !(ok = wait(&misc->full[s_], (n / kStages) & 1))) break;
      if (!(ok = wait(&misc->s_full[slot], (n >> 1) & 1))) break;
      tc_fence_after_sync();
      if (unclean) {  // scores of rows that belong to nobody are masked, whatever they are; the products behind them take the rows themselves
        const int r = half * 32 + (warp & 3) * 8 + (lane >> 2);
        if ((lane & 3) < 2) clear_row<DB, kWalk>(smem + L::Y + (s_ * 2 + (lane & 1)) * L::TILE, p.masks, b, p.Nk, y0, r);
        fence_proxy_async_smem();
      }
      const Stats& st = misc->stats[s_];
      const bool all = KEYS ? st.keys[0].y >= x0 + 128 && st.keys[kWalk - 1].x <= x0
                            : __all_sync(0xffffffffu, keys.x <= y0 && keys.y >= y0 + kWalk) != 0;
      const float d0 = (float)(row - y0);
      // 16 columns at a time, of this warp's half; packed, they take the first of the columns that they were read from
      const auto columns = [&](auto masked_) {  // (apart for tiles in full sight: a look at every pair keeps the pairs from overlapping)
        constexpr bool MASKED = decltype(masked_)::value;
        uint32_t low[2][8];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col0 = half * 32 + c * 16;
          uint32_t s[16], d[16], pw[8], dw[8];
          tmem_ld16(ts + c * 16, s);
          tmem_ld16(td + c * 16, d);
          tmem_wait_ld();
          tmem_fence_regs16(s);
          tmem_fence_regs16(d);
          unsigned on = 0xffffu;
          if (MASKED) {
            on = 0;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int2 see = KEYS ? st.keys[col0 + k] : keys;
              const int key = KEYS ? row : y0 + col0 + k;
              on |= (unsigned)(key >= see.x && key < see.y) << k;
            }
          }
          if (CAP) {
            if (MASKED) {  // (what lies out of sight does not choose the form)
#pragma unroll
              for (int k = 0; k < 16; ++k)
                if (!(on >> k & 1)) s[k] = 0u;
            }
            cap_scores(s, series);
          }
#pragma unroll
          for (int k4 = 0; k4 < 16; k4 += 4) {
            ulonglong2 l4 = make_ulonglong2(twice(lse), twice(lse)), d4 = make_ulonglong2(twice(delta), twice(delta));
            if (KEYS) {
              l4 = *reinterpret_cast<const ulonglong2*>(&st.lse[col0 + k4]);
              d4 = *reinterpret_cast<const ulonglong2*>(&st.delta[col0 + k4]);
            }
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const int k = k4 + e, col = col0 + k;
              const uint64_t t = f2_pack(__uint_as_float(s[k]), __uint_as_float(s[k + 1]));
              uint64_t bias = e ? l4.y : l4.x;
              if (BIAS) bias = f2_fma(twice(-sc.slope), f2_pack(fabsf(d0 - (float)col), fabsf(d0 - (float)(col + 1))), bias);
              float w0, w1, g0, g1;
              f2_unpack(f2_fma(t, twice(sc.unit), bias), w0, w1);
              w0 = ex2_approx(w0);
              w1 = ex2_approx(w1);
              uint64_t g = f2_mul(f2_pack(w0, w1), f2_add(f2_pack(__uint_as_float(d[k]), __uint_as_float(d[k + 1])), e ? d4.y : d4.x));
              if (CAP) g = f2_mul(g, f2_fma(f2_mul(t, twice(-up)), t, twice(up)));
              else if (F16 && KEYS) g = f2_mul(g, twice(up));
              f2_unpack(g, g0, g1);
              if (MASKED) {
                w0 = on >> k & 1 ? w0 : 0.0f;
                g0 = on >> k & 1 ? g0 : 0.0f;
                w1 = on >> (k + 1) & 1 ? w1 : 0.0f;
                g1 = on >> (k + 1) & 1 ? g1 : 0.0f;
              }
              pw[k >> 1] = pack2<F16>(w0, w1);
              dw[k >> 1] = pack2<F16>(g0, g1);
              float h0, h1;
              unpack2<F16>(dw[k >> 1], h0, h1);
              low[c][k >> 1] = pack2<F16>(g0 - h0, g1 - h1);
            }
          }
          if (KEYS) tmem_st8(ts + c * 8, pw);
          tmem_st8(td + c * 8, dw);
        }
        // what dS lost in that rounding, behind P (which all scores of this half have been read from by now)
        tmem_st8(ts + LOW, low[0]);
        tmem_st8(ts + LOW + 8, low[1]);
      };
      if (all) columns(std::false_type());
      else columns(std::true_type());
      tmem_wait_st();
      tc_fence_before_sync();
      warp_arrive(&misc->w_ready[slot], lane);
    }
    if (ok && total > 0) ok = wait(&misc->done, 0);
    if (ok) {
      tc_fence_after_sync();
      const int rows = KEYS ? p.Nk : p.Nq;
      const int64_t at = (((int64_t)b * rows + row) * heads + head) * p.D;
      const auto put = [&](void* out, uint32_t t, int c, float f) {
        uint32_t r[32];
        if (total > 0) {
          tmem_read<32>(tl + t + c * 32, r);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0u;
        }
        if (row < rows) store_columns<F16>(reinterpret_cast<uint16_t*>(out) + at, c * 32, p.D, r, f);
      };
      if (KEYS) {  // a sum for the groups of a slot, half the columns each
#pragma unroll
        for (int c = 0; c < DB; ++c)
          if (slot == 0) put(p.dk, T_DS, half * DB + c, p.scale * down);
          else put(p.dv, T_P, half * DB + c, F16 ? power_of_two(-kWeightLift) : 1.0f);
      } else if (slot * 2 + half < 2 * DB) {  // 32 columns each
        put(p.dq, T_DS, slot * 2 + half, p.scale * down);
      }
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

template <bool F16, bool KEYS>
int launch(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream) {
  constexpr int DB = FLARE_ATTN_DB;
  const auto map = [&](CUtensorMap* m, int which, uint32_t rows) {
    switch (which) {
      case 0: return head_map(m, a.q, a.B, a.Nq, a.H, a.D, a.q_stride_b, a.q_stride_n, a.q_stride_h, rows);
      case 1: return head_map(m, a.dy, a.B, a.Nq, a.H, a.D, a.dy_stride_b, a.dy_stride_n, a.dy_stride_h, rows);
      case 2: return head_map(m, a.k, a.B, a.Nk, a.J, a.D, a.k_stride_b, a.k_stride_n, a.k_stride_h, rows);
      default: return head_map(m, a.v, a.B, a.Nk, a.J, a.D, a.v_stride_b, a.v_stride_n, a.v_stride_h, rows);
    }
  };
  CUtensorMap x0, x1, y0, y1;
  const int own = KEYS ? 2 : 0;
  if (!map(&x0, own, 128) || !map(&x1, own + 1, 128) || !map(&y0, 2 - own, kWalk) || !map(&y1, 3 - own, kWalk)) return FLARE_ERR_CUDA;
  const bool cap = p.cap > 0.0f, bias = p.slopes != nullptr;
  auto* const kernel = cap ? (bias ? attention_backward_kernel<DB, F16, true, true, KEYS> : attention_backward_kernel<DB, F16, true, false, KEYS>)
                           : (bias ? attention_backward_kernel<DB, F16, false, true, KEYS> : attention_backward_kernel<DB, F16, false, false, KEYS>);
  FLARE_CUDA_CHECK(allow_smem(kernel));
  const int64_t blocks = (int64_t)((KEYS ? a.Nk : a.Nq) + 127) / 128 * a.B * (KEYS ? a.J : a.H);
  if (blocks > 0x7fffffff) return FLARE_ERR_UNSUPPORTED;
  LaunchTimer timer(KEYS ? "attention_backward_kernel (keys)" : "attention_backward_kernel (queries)", stream);
  FLARE_CUDA_CHECK(launch_pdl(kernel, dim3((unsigned)blocks), dim3(kThreads), Layout<DB>::BYTES, stream, x0, x1, y0, y1, p));
  return FLARE_OK;
}

}  // namespace

template <int DB>
int launch_backward_db(const flare_attention_args_t& a, const AttnParams& p, bool keys, cudaStream_t stream);
template <>
int launch_backward_db<FLARE_ATTN_DB>(const flare_attention_args_t& a, const AttnParams& p, bool keys, cudaStream_t stream) {
  if (a.dtype == FLARE_F16) return keys ? launch<true, true>(a, p, stream) : launch<true, false>(a, p, stream);
  return keys ? launch<false, true>(a, p, stream) : launch<false, false>(a, p, stream);
}

#else

template <int DB>
int launch_backward_db(const flare_attention_args_t& a, const AttnParams& p, bool keys, cudaStream_t stream);
template <>
int launch_backward_db<1>(const flare_attention_args_t& a, const AttnParams& p, bool keys, cudaStream_t stream);
template <>
int launch_backward_db<2>(const flare_attention_args_t& a, const AttnParams& p, bool keys, cudaStream_t stream);

int launch_backward_tc(const flare_attention_args_t& a, const AttnParams& p, cudaStream_t stream) {
  for (const bool keys : {true, false})
    if (const int rc = a.D <= 64 ? launch_backward_db<1>(a, p, keys, stream) : launch_backward_db<2>(a, p, keys, stream)) return rc;
  return FLARE_OK;
}

#endif

}  // namespace attn
}  // namespace flare
