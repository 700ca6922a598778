// Attention backward on the tensor cores: 16-bit tensors.
//
// Two kernels, each of which recomputes the probabilities p = 2^(s scale
// log2 e - lse2) of a block of queries and keys from the rows' statistics and
// writes each gradient element once:
//   dK, dV: a CTA keeps 128 keys and streams the queries that see them, of
//           every head of the group, in blocks of 64: S^T = K Q^T,
//           dP^T = V dO^T, dV += P^T dO, dK += dS^T Q;
//   dQ:     a CTA keeps 128 queries and streams keys in blocks of 64:
//           S = Q K^T, dP = dO V^T, dQ += dS K.
// Seven products instead of the five of a single kernel, whose dQ would be a
// sum over CTAs: fp32 atomics, whose order changes the result, and a pass to
// clear and one to round them (12 bytes an element of dQ and 4 more an
// addition). The gradients here do not depend on scheduling.
//
// P^T, dS^T and dS are rounded to the tensors' type and stay in tensor memory,
// where S^T and dP lay, as the products' first operand; the streamed tiles are
// read by the products both by rows and by columns, so nothing is transposed
// or stored again. (Tiles of few keys, kFineKeys: as two terms, in the two
// halves of where S^T and dP lay. fp16: times powers of two that keep them in its
// range, kBwdShift and ds_scale.) Blocks alternate between two buffers of S and of dP in
// tensor memory and two groups of four warps (thread = row of the kept tile,
// 64 columns): a group has two blocks' time for its own, so neither the
// hand-over between warps nor its own latencies stop the tensor core. Warps 8
// and 9 issue the products, warp 10 the copies.
//
// At head_dim 256 the sums of dV and dK would fill tensor memory (512 columns),
// so they are two launches of the first kernel, one with S^T and dV, one with
// S^T, dP^T and dK: five products where one launch would need four.
//
// Bound: the products. 64 streamed rows against 128 kept ones in shared memory
// take the time of 128 (a step reads 4 KB of the kept tile whatever the
// streamed one has): 512 cycles each for S and dP at head_dim 128, 256 for dV
// or dK. With the kept tiles in tensor memory, where the sums leave room for
// them (dQ up to head_dim 128; dK and dV at head_dim 64), S and dP take 256 as
// well. Beside them 512 cycles a block for its exponentials.
// Measured at 8192 rows of 32/8 heads of 128 (bf16), from idle, at 1965 MHz: causal,
// dK and dV 830 us (four products, 1320 TFLOP/s), dQ 582 us (three, 1410); full rows,
// dQ 1120 us, with the kept tiles in shared memory 1370, and dK and dV 1700 to 1840 us,
// in blocks of 128 queries in single buffers 1826. In seconds of calls the 1 kW cap
// leaves 1470 to 1690 MHz: dQ 980 cycles a block and 11,500 a CTA beside them, dK and
// dV 1650 and 6,400. Sixteen softmax warps in place of eight were no faster.
#pragma once

#include <climits>

#include "attn_impl.cuh"
#include "tc.cuh"

namespace bloth {

// What a launch sums up.
enum BwdSums : int { kSumDQ = 0, kSumDV = 1, kSumDK = 2, kSumDKV = 3 };

template <int D, int SUMS>
struct BwdCfg {
  static constexpr int TILE = 128;             // rows of the kept tiles
  static constexpr int BLK = 64;               // rows of a streamed block
  static constexpr int THREADS = 352;
  static constexpr int OWNB = TILE * D * 2, STRB = BLK * D * 2;  // bytes of a tile
  static constexpr int OWN = SUMS == kSumDV ? 1 : 2;  // kept tiles: K and V, or Q and dO
  // Stages of A (Q, or K) and of B (dO, or V): as many as fit. Two of A at
  // least, which a block's last product reads; one of B where only dP reads it.
  static constexpr int NA = D == 64 ? 8 : D == 128 ? 5 : SUMS == kSumDV ? 3 : 2;
  static constexpr int NB = D == 64 ? 8 : D == 128 ? 5 : SUMS == kSumDV ? 2 : 1;
  static constexpr int OWN_OFF = 0;                    // the kept tiles
  static constexpr int A_OFF = OWN * OWNB;
  static constexpr int B_OFF = A_OFF + NA * STRB;
  static constexpr int STAT_OFF = B_OFF + NB * STRB;   // lse2 and delta, with A's stages
  static constexpr int BAR_OFF = STAT_OFF + NA * 512;
  static constexpr int BARS = 1 + 2 * NA + 2 * NB + 8 + 3 + 1;
  static constexpr int SMEM = BAR_OFF + BARS * 8 + 16;
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static_assert(OWN * OWNB >= 8 * 4096, "4 KB of the kept tiles for each warp's results");
  // tensor-memory columns: S (two buffers), dP (two buffers, not for dV alone),
  // the sums, and behind them, where there is room, the kept tiles
  static constexpr uint32_t COLS = 512;
  static constexpr uint32_t S_COL = 0, DP_COL = 128, ACC_COL = SUMS == kSumDV ? 128 : 256;
  static constexpr uint32_t OWN_COL = ACC_COL + (SUMS == kSumDKV ? 2 * D : D);
  static constexpr bool OWN_TMEM = OWN_COL + OWN * D / 2 <= COLS;
};

struct BwdMaps {
  CUtensorMap q, k, v, dout;
};

// Barriers of both kernels; A and B are the streamed tensors (Q and dO, or K
// and V), [2] one for each buffer.
template <int NA, int NB>
struct BwdBars {
  uint32_t own, a_full, a_free, b_full, b_free, s_full, p_full, dp_full, ds_full, acc, drained,
      there;
  __device__ __forceinline__ explicit BwdBars(uint32_t at) {
    own = at;
    a_full = own + 8;
    a_free = a_full + 8 * NA;
    b_full = a_free + 8 * NA;
    b_free = b_full + 8 * NB;
    s_full = b_free + 8 * NB;
    p_full = s_full + 16;
    dp_full = p_full + 16;
    ds_full = dp_full + 16;
    acc = ds_full + 16;
    drained = acc + 8;
    there = drained + 16;  // the kept tiles are in tensor memory
  }
  // b_free completes when `b_uses` products have, acc with `sums` of them
  __device__ __forceinline__ void init(int b_uses, int sums) const {
    bar_init(own, 1);
    bar_init(there, 8);
    for (int i = 0; i < NA; ++i) {
      bar_init(a_full + 8 * i, 1);
      bar_init(a_free + 8 * i, 1);
    }
    for (int i = 0; i < NB; ++i) {
      bar_init(b_full + 8 * i, 1);
      bar_init(b_free + 8 * i, b_uses);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(s_full + 8 * i, 1);
      bar_init(p_full + 8 * i, 4);
      bar_init(dp_full + 8 * i, 1);
      bar_init(ds_full + 8 * i, 4);
      bar_init(drained + 8 * i, 1);
    }
    bar_init(acc, sums);
  }
  // given up: not before the copies in flight have landed (blocks [0, it))
  __device__ __forceinline__ void drain_copies(int it, const Waits& w) const {
    bar_drain(own, 0, w);
    for (int i = max(0, it - NA); i < it; ++i)
      bar_drain(a_full + 8 * (i % NA), (uint32_t)(i / NA) & 1u, w);
    for (int i = max(0, it - NB); i < it; ++i)
      bar_drain(b_full + 8 * (i % NB), (uint32_t)(i / NB) & 1u, w);
  }
};

// COLS accumulator columns of the thread's row, times f, to 16-bit memory, or
// zeros (!keep): the warp's rows r < n at dst + r * ss, through 4 KB of shared
// memory `sm`. `any`, alike in the whole warp: there are sums.
template <int COLS, typename T>
__device__ __forceinline__ void store_sums(uint32_t at, float f, T* dst, int64_t ss, int n,
                                           bool keep, bool any, unsigned char* sm) {
  constexpr int CW = COLS < 64 ? COLS : 64;
#pragma unroll 1
  for (int c = 0; c < COLS; c += CW) {
    uint32_t w[CW / 2] = {};
    if (any) {
#pragma unroll
      for (int p = 0; p < CW; p += 32) {
        uint32_t r[32];
        tmem_ld32(at + c + p, r);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w[p / 2 + i] = keep ? pack2<T>(__uint_as_float(r[2 * i]) * f,
                                         __uint_as_float(r[2 * i + 1]) * f)
                              : 0u;
      }
    }
    store_rows<CW>(sm, w, dst + c, ss, n);
  }
}

// ------------------------------------------------------------------ dK, dV
template <typename T, int D, int SUMS>
__global__ void __launch_bounds__(352, 1)
    attn_dkv_kernel(const AttnArgs a, const __grid_constant__ BwdMaps maps) {
  using C = BwdCfg<D, SUMS>;
  constexpr bool DV = (SUMS & kSumDV) != 0, DK = (SUMS & kSumDK) != 0;
  constexpr int N = C::TILE, BLK = C::BLK, NA = C::NA, NB = C::NB;
  constexpr uint32_t DV_COL = C::ACC_COL, DK_COL = C::ACC_COL + (DV ? D : 0);
  constexpr bool OWN_TMEM = C::OWN_TMEM;
  constexpr uint32_t K_COL = C::OWN_COL, V_COL = K_COL + D / 2;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_addr(smem);
  const BwdBars<NA, NB> bar(base + C::BAR_OFF);
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + 8 * C::BARS);
  const Waits waits{reinterpret_cast<volatile int*>(tmem_ptr + 1), a.fault};

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int heads = a.Hk * a.B;
  const int hb = blockIdx.x % heads, h = hb % a.Hk;
  // the first keys are seen by most queries (causal): they start first
  const AttnSeq s = find_seq<false>(a, hb / a.Hk, (int)(blockIdx.x / heads), N);
  if (s.tile < 0) return;
  const int n0 = s.tile * N;
  const int limit = a.packed ? s.klen : a.Sk;
  if (n0 >= limit) return;
  int lo, hi;
  query_range(a, s, n0, min(n0 + N, s.klen), lo, hi);
  const int mb = lo / BLK, nm = hi > lo ? (hi + BLK - 1) / BLK - mb : 0;  // blocks per head
  const int total = nm * a.G;
  const bool fine = few_keys(a, s, hi);

  if (warp == 8) {
    tmem_alloc(tmem_ptr, C::COLS);
  } else if (threadIdx.x == 0) {
    bar.init(DV && DK ? 2 : 1, DV && DK ? 2 : 1);
    *waits.stop = 0;
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;

  if (warp == 10) {
    // ------------------------------------------------------------- copies
    if (lane == 0 && total > 0) {
      bar_expect(bar.own, C::OWN * C::OWNB);
      load_tile<D, N>(base + C::OWN_OFF, &maps.k, s.k0 + n0, h, s.b, bar.own);
      if (DK) load_tile<D, N>(base + C::OWN_OFF + C::OWNB, &maps.v, s.k0 + n0, h, s.b, bar.own);
      Ring<NA> qst;
      Ring<NB> ost;
      int it = 0, mi = 0, hq = h * a.G;
      for (; it < total; ++it, qst.next(), ost.next()) {
        const int m0 = (mb + mi) * BLK;
        const int64_t stat = (int64_t)hq * a.R + s.stat0 + m0;
        const uint32_t qf = bar.a_full + 8 * qst.at, of = bar.b_full + 8 * ost.at;
        const uint32_t sp = base + C::STAT_OFF + qst.at * 512;
        if (!bar_wait(bar.a_free + 8 * qst.at, qst.phase ^ 1u, waits)) break;
        bar_expect(qf, C::STRB + 512);
        run_load(sp, a.lse2 + stat, 256, qf);
        run_load(sp + 256, a.delta + stat, 256, qf);
        load_tile<D, BLK>(base + C::A_OFF + qst.at * C::STRB, &maps.q, s.q0 + m0, hq, s.b, qf);
        if (!bar_wait(bar.b_free + 8 * ost.at, ost.phase ^ 1u, waits)) {
          bar_drain(qf, qst.phase, waits);
          break;
        }
        bar_expect(of, C::STRB);
        load_tile<D, BLK>(base + C::B_OFF + ost.at * C::STRB, &maps.dout, s.q0 + m0, hq, s.b, of);
        if (++mi == nm) {
          mi = 0;
          ++hq;
        }
      }
      if (*waits.stop) bar.drain_copies(it, waits);
    }
  } else if (warp == 8) {
    // S^T and dV: P^T lies where S^T was, so S^T of block j follows dV of j - 2
    if (total > 0) {
      const uint32_t ka = base + C::OWN_OFF;
      const bool lead = elect();
      Ring<NA> qst, qold;
      Ring<NB> ost;
      Ring<2> buf, pbuf;
      bool ok = bar_wait(OWN_TMEM ? bar.there : bar.own, 0, waits);
      tc_fence_after();
      auto steps = [&](auto few) {
        constexpr bool FINE = decltype(few)::value;
        for (int j = 0; ok && j < total + 2; ++j) {
          if (j >= 2) {
            ok = (!DV || bar_wait(bar.b_full + 8 * ost.at, ost.phase, waits)) &&
                 bar_wait(bar.p_full + 8 * pbuf.at, pbuf.phase, waits);
            if (!ok) break;
            tc_fence_after();
            if (DV && lead) {
              const uint32_t p = tmem + C::S_COL + pbuf.at * BLK;
              const uint32_t ot = base + C::B_OFF + ost.at * C::STRB;
              product_cols<T, D>(tmem + DV_COL, p, ot, j > 2);
              if (FINE) product_cols<T, D>(tmem + DV_COL, p + 32, ot, true);
              mma_commit(bar.b_free + 8 * ost.at);
              // Q and the statistics went into P^T, which this product has read
              if (!DK) mma_commit(bar.a_free + 8 * qold.at);
            }
            ost.next();
            qold.next();
            pbuf.next();
          }
          if (j < total) {
            ok = bar_wait(bar.a_full + 8 * qst.at, qst.phase, waits);
            if (!ok) break;
            if (lead) {
              const uint32_t qt = base + C::A_OFF + qst.at * C::STRB;
              if constexpr (OWN_TMEM)
                product_rows_ts<T, D>(tmem + C::S_COL + buf.at * BLK, tmem + K_COL, qt);
              else
                product_rows<T, D>(tmem + C::S_COL + buf.at * BLK, ka, qt);
              mma_commit(bar.s_full + 8 * buf.at);
            }
            qst.next();
            buf.next();
          }
        }
      };
      if (fine) steps(std::true_type{});
      else steps(std::false_type{});
      if (lead && (DV || !ok)) {
        mma_commit(ok ? bar.acc : bar.drained);
        if (!ok) bar_drain(bar.drained, 0, waits);
      }
      __syncwarp();
    }
  } else if (warp == 9) {
    // dP^T and dK, dS^T where dP^T was
    if (DK && total > 0) {
      const uint32_t va = base + C::OWN_OFF + C::OWNB;
      const bool lead = elect();
      Ring<NA> qst;
      Ring<NB> ost;
      Ring<2> buf, dbuf;
      bool ok = bar_wait(OWN_TMEM ? bar.there : bar.own, 0, waits);
      tc_fence_after();
      auto steps = [&](auto few) {
        constexpr bool FINE = decltype(few)::value;
        for (int j = 0; ok && j < total + 2; ++j) {
          if (j >= 2) {
            ok = bar_wait(bar.a_full + 8 * qst.at, qst.phase, waits) &&
                 bar_wait(bar.ds_full + 8 * dbuf.at, dbuf.phase, waits);
            if (!ok) break;
            tc_fence_after();
            if (lead) {
              const uint32_t ds = tmem + C::DP_COL + dbuf.at * BLK;
              const uint32_t qt = base + C::A_OFF + qst.at * C::STRB;
              product_cols<T, D>(tmem + DK_COL, ds, qt, j > 2);
              if (FINE) product_cols<T, D>(tmem + DK_COL, ds + 32, qt, true);
              mma_commit(bar.a_free + 8 * qst.at);
            }
            qst.next();
            dbuf.next();
          }
          if (j < total) {
            ok = bar_wait(bar.b_full + 8 * ost.at, ost.phase, waits);
            if (!ok) break;
            if (lead) {
              const uint32_t ot = base + C::B_OFF + ost.at * C::STRB;
              if constexpr (OWN_TMEM)
                product_rows_ts<T, D>(tmem + C::DP_COL + buf.at * BLK, tmem + V_COL, ot);
              else
                product_rows<T, D>(tmem + C::DP_COL + buf.at * BLK, va, ot);
              mma_commit(bar.dp_full + 8 * buf.at);
              mma_commit(bar.b_free + 8 * ost.at);
            }
            ost.next();
            buf.next();
          }
        }
      };
      if (fine) steps(std::true_type{});
      else steps(std::false_type{});
      if (lead) {
        mma_commit(ok ? bar.acc : bar.drained + 8);
        if (!ok) bar_drain(bar.drained + 8, 0, waits);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------- blocks `group`, group + 2, ...
    const int group = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int key = n0 + r, off = s.klen - s.qlen;
    const uint32_t s_at = tmem + lanes + C::S_COL + group * BLK;
    const uint32_t dp_at = tmem + lanes + C::DP_COL + group * BLK;
    const float2 sc = f2s(a.scale_log2);
    const int seen0 = first_query(a, s);
    // fp16: dS times a power of two, by the largest bound of the CTA's
    float ds_up = 1.f;
    if constexpr (DK && kBwdShift<T> != 0.f) {
      if (total > 0) {
        const float2* top = a.qtop + (int64_t)h * a.G * stat_tiles(a.R) + s.stat0 / 128 + lo / 128;
        const int n = (hi + 127) / 128 - lo / 128;
        float2 most = f2(0.f, 0.f);
        for (int g = 0; g < a.G; ++g)
          for (int i = lane; i < n; i += 32) {
            const float2 u = __ldg(top + (int64_t)g * stat_tiles(a.R) + i);
            most = f2(fmaxf(most.x, u.x), fmaxf(most.y, u.y));
          }
        const float v = __ldg(a.vtop + (int64_t)h * stat_tiles(a.RK) + s.kstat0 / 128 + s.tile);
        ds_up = ds_scale(warp_top(most.x) * v + warp_top(most.y));
      }
    }
    Ring<NA> st;
    Ring<NB> ost;
    int mi = 0;
    if (group) {
      st.next();
      ost.next();
      mi = nm > 1 ? 1 : 0;
    }
    uint32_t ph = 0;
    bool ok = true;
    if (OWN_TMEM && total > 0) {
      ok = __all_sync(0xffffffffu, bar_wait(bar.own, 0, waits));
      if (ok) {
        if (group < C::OWN)
          copy_operand<D>(smem + C::OWN_OFF + group * C::OWNB, r,
                          tmem + lanes + K_COL + group * (D / 2));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar.there);
      }
    }
    auto blocks = [&](auto few) {  // two loops: as in the forward
      constexpr bool FINE = decltype(few)::value;
      for (int it = group; ok && it < total; it += 2, ph ^= 1u) {
        const int m0 = (mb + mi) * BLK;
        const float* stat = reinterpret_cast<const float*>(smem + C::STAT_OFF + st.at * 512);
        ok = bar_wait(bar.a_full + 8 * st.at, st.phase, waits) &&
             bar_wait(bar.s_full + 8 * group, ph, waits);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
        float x[BLK];
        load64(s_at, x);
#pragma unroll
        for (int i = 0; i < BLK; i += 4) {
          const float4 l = *reinterpret_cast<const float4*>(stat + i);
          const float2 u = f2_fma(f2(x[i], x[i + 1]), sc, f2(-l.x, -l.y));
          const float2 w = f2_fma(f2(x[i + 2], x[i + 3]), sc, f2(-l.z, -l.w));
          x[i] = ex2(u.x);
          x[i + 1] = ex2(u.y);
          x[i + 2] = ex2(w.x);
          x[i + 3] = ex2(w.y);
        }
        // the block's columns that see this thread's key: [from, to)
        const int from = a.causal ? key - off - m0 : 0;
        const int to = min(s.qlen, a.window ? key - off + a.window : s.qlen) - m0;
        const bool masked = m0 + BLK > s.qlen || s.klen == 1 ||
                            (a.causal && n0 + N - 1 - off > m0) ||
                            (a.window && n0 - off + a.window < m0 + BLK);
        // the block has rows that nothing may be read from (it is masked then): before
        // the first query that sees a key, or past the sequence's end where memory does
        // hold some
        const bool dead = m0 < seen0 || (m0 + BLK > s.qlen && s.q0 + s.qlen < a.Sq);
        // the query that sees one key only; INT_MAX: all do, -1: none of the block
        const int alone = s.klen == 1 || a.window == 1 ? INT_MAX : a.causal ? -off - m0 : -1;
        if (masked) {
#pragma unroll
          for (int i = 0; i < BLK; ++i)
            if (i < from || i >= to) x[i] = 0.f;
          if (DV && dead) {
            ok = __all_sync(0xffffffffu, bar_wait(bar.b_full + 8 * ost.at, ost.phase, waits));
            if (!ok) break;
            keep_rows<D>(smem + C::B_OFF + ost.at * C::STRB, seen0 - m0, s.qlen - m0);
          }
        }
        if (DV) {
          store64<T>(s_at, x);
          if (FINE) store64_rest<T>(s_at + 32, x);
        }
        const bool there = !DK || bar_test(bar.dp_full + 8 * group, ph);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar.p_full + 8 * group);
        ok = __all_sync(0xffffffffu, there || bar_wait(bar.dp_full + 8 * group, ph, waits));
        if (!ok) break;
        tc_fence_after();
        if constexpr (DK) {
          float y[BLK];
          load64(dp_at, y);
          if constexpr (kBwdShift<T> != 0.f) {
            const float2 down = f2s(ds_up * exp2f(-kBwdShift<T>));
#pragma unroll
            for (int i = 0; i < BLK; i += 2) {
              const float2 p = f2_mul(f2(x[i], x[i + 1]), down);
              x[i] = p.x;
              x[i + 1] = p.y;
            }
          }
#pragma unroll
          for (int i = 0; i < BLK; i += 4) {
            const float4 d = *reinterpret_cast<const float4*>(stat + 64 + i);
            const float2 u = f2_mul(f2(x[i], x[i + 1]), f2_add(f2(y[i], y[i + 1]), f2(-d.x, -d.y)));
            const float2 w =
                f2_mul(f2(x[i + 2], x[i + 3]), f2_add(f2(y[i + 2], y[i + 3]), f2(-d.z, -d.w)));
            y[i] = u.x;
            y[i + 1] = u.y;
            y[i + 2] = w.x;
            y[i + 3] = w.y;
          }
          if (masked) {
#pragma unroll
            for (int i = 0; i < BLK; ++i)
              if (i < from || i >= to || i == alone || alone == INT_MAX) y[i] = 0.f;
            if (dead) keep_rows<D>(smem + C::A_OFF + st.at * C::STRB, seen0 - m0, s.qlen - m0);
          }
          store64<T>(dp_at, y);
          if (FINE) store64_rest<T>(dp_at + 32, y);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(bar.ds_full + 8 * group);
        }
        st.next();
        st.next();
        ost.next();
        ost.next();
        mi += 2;
        if (mi >= nm) mi -= nm;
        if (mi >= nm) mi -= nm;  // nm == 1
      }
    };
    if (fine) blocks(std::true_type{});
    else blocks(std::false_type{});
    if (ok && total > 0) {
      ok = __all_sync(0xffffffffu, bar_wait(bar.acc, 0, waits));
      tc_fence_after();
    }
    if (ok) {
      // group 0 writes dV, group 1 dK, or each half of the one there is; keys
      // past the sequence's end (dense tensors) get zeros
      const bool is_k = DV && DK ? group != 0 : DK;
      constexpr int COLS = DV && DK ? D : D / 2;
      const int c0 = DV && DK ? 0 : group * COLS, key0 = n0 + (warp & 3) * 32;
      const HT& t = is_k ? a.dk : a.dv;
      T* dst = reinterpret_cast<T*>(const_cast<void*>(t.p)) + (int64_t)s.b * t.sb +
               (int64_t)h * t.sh + (int64_t)(s.k0 + key0) * t.ss + c0;
      // through the kept tiles, which every product has read
      store_sums<COLS>(tmem + lanes + (is_k ? DK_COL : DV_COL) + c0,
                       is_k ? a.scale / ds_up : exp2f(-kBwdShift<T>), dst, t.ss, limit - key0,
                       key < s.klen, total > 0, smem + C::OWN_OFF + warp * 4096);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_free(tmem, C::COLS);
}

// ---------------------------------------------------------------------- dQ
template <typename T, int D>
__global__ void __launch_bounds__(352, 1)
    attn_dq_kernel(const AttnArgs a, const __grid_constant__ BwdMaps maps) {
  using C = BwdCfg<D, kSumDQ>;
  constexpr int N = C::TILE, BLK = C::BLK, NA = C::NA, NB = C::NB;
  constexpr bool OWN_TMEM = C::OWN_TMEM;
  constexpr uint32_t Q_COL = C::OWN_COL, O_COL = Q_COL + D / 2;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_addr(smem);
  const BwdBars<NA, NB> bar(base + C::BAR_OFF);
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + 8 * C::BARS);
  const Waits waits{reinterpret_cast<volatile int*>(tmem_ptr + 1), a.fault};

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int heads = a.Hq * a.B;
  const int tiles = (int)(gridDim.x / heads);
  const int hb = blockIdx.x % heads, h = hb % a.Hq;
  // the last queries see most keys (causal): they start first
  const AttnSeq s = find_seq<true>(a, hb / a.Hq, tiles - 1 - (int)(blockIdx.x / heads), N);
  if (s.tile < 0) return;
  const int m0 = s.tile * N;
  const int limit = a.packed ? s.qlen : a.Sq;
  if (m0 >= limit) return;
  int lo, hi;
  key_range(a, s, m0, min(m0 + N, s.qlen), lo, hi);
  const int b0 = lo / BLK, total = hi > lo ? (hi + BLK - 1) / BLK - b0 : 0;
  const bool fine = few_keys(a, s, min(m0 + N, s.qlen));

  if (warp == 8) {
    tmem_alloc(tmem_ptr, C::COLS);
  } else if (threadIdx.x == 0) {
    bar.init(1, 1);
    *waits.stop = 0;
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;

  if (warp == 10) {
    // ------------------------------------------------------------- copies
    if (lane == 0 && total > 0) {
      bar_expect(bar.own, 2 * C::OWNB);
      load_tile<D, N>(base + C::OWN_OFF, &maps.q, s.q0 + m0, h, s.b, bar.own);
      load_tile<D, N>(base + C::OWN_OFF + C::OWNB, &maps.dout, s.q0 + m0, h, s.b, bar.own);
      const int hk = h / a.G;
      Ring<NA> kst;
      Ring<NB> vst;
      int it = 0, r0 = s.k0 + b0 * BLK;
      for (; it < total; ++it, r0 += BLK, kst.next(), vst.next()) {
        const uint32_t kf = bar.a_full + 8 * kst.at, vf = bar.b_full + 8 * vst.at;
        if (!bar_wait(bar.a_free + 8 * kst.at, kst.phase ^ 1u, waits)) break;
        bar_expect(kf, C::STRB);
        load_tile<D, BLK>(base + C::A_OFF + kst.at * C::STRB, &maps.k, r0, hk, s.b, kf);
        if (!bar_wait(bar.b_free + 8 * vst.at, vst.phase ^ 1u, waits)) {
          bar_drain(kf, kst.phase, waits);
          break;
        }
        bar_expect(vf, C::STRB);
        load_tile<D, BLK>(base + C::B_OFF + vst.at * C::STRB, &maps.v, r0, hk, s.b, vf);
      }
      if (*waits.stop) bar.drain_copies(it, waits);
    }
  } else if (warp == 8) {
    // S, into the buffer that the group has read when its dS is there
    if (total > 0) {
      const bool lead = elect();
      Ring<NA> st;
      Ring<2> buf;
      bool ok = bar_wait(OWN_TMEM ? bar.there : bar.own, 0, waits);
      tc_fence_after();
      for (int j = 0; ok && j < total; ++j) {
        ok = bar_wait(bar.a_full + 8 * st.at, st.phase, waits);
        if (ok && j >= 2) ok = bar_wait(bar.ds_full + 8 * buf.at, buf.phase ^ 1u, waits);
        if (!ok) break;
        tc_fence_after();
        if (lead) {
          const uint32_t kt = base + C::A_OFF + st.at * C::STRB;
          if constexpr (OWN_TMEM)
            product_rows_ts<T, D>(tmem + C::S_COL + buf.at * BLK, tmem + Q_COL, kt);
          else
            product_rows<T, D>(tmem + C::S_COL + buf.at * BLK, base + C::OWN_OFF, kt);
          mma_commit(bar.s_full + 8 * buf.at);
        }
        st.next();
        buf.next();
      }
      if (!ok && lead) {
        mma_commit(bar.drained);
        bar_drain(bar.drained, 0, waits);
      }
      __syncwarp();
    }
  } else if (warp == 9) {
    // dP and dQ: dS lies where dP was, so dP of block j follows dQ of j - 2
    if (total > 0) {
      const bool lead = elect();
      Ring<NA> kst;
      Ring<NB> vst;
      Ring<2> buf, dbuf;
      bool ok = bar_wait(OWN_TMEM ? bar.there : bar.own, 0, waits);
      tc_fence_after();
      auto steps = [&](auto few) {
        constexpr bool FINE = decltype(few)::value;
        for (int j = 0; ok && j < total + 2; ++j) {
          if (j >= 2) {
            ok = bar_wait(bar.a_full + 8 * kst.at, kst.phase, waits) &&
                 bar_wait(bar.ds_full + 8 * dbuf.at, dbuf.phase, waits);
            if (!ok) break;
            tc_fence_after();
            if (lead) {
              const uint32_t ds = tmem + C::DP_COL + dbuf.at * BLK;
              const uint32_t kt = base + C::A_OFF + kst.at * C::STRB;
              product_cols<T, D>(tmem + C::ACC_COL, ds, kt, j > 2);
              if (FINE) product_cols<T, D>(tmem + C::ACC_COL, ds + 32, kt, true);
              mma_commit(bar.a_free + 8 * kst.at);
            }
            kst.next();
            dbuf.next();
          }
          if (j < total) {
            ok = bar_wait(bar.b_full + 8 * vst.at, vst.phase, waits);
            if (!ok) break;
            if (lead) {
              const uint32_t vt = base + C::B_OFF + vst.at * C::STRB;
              if constexpr (OWN_TMEM)
                product_rows_ts<T, D>(tmem + C::DP_COL + buf.at * BLK, tmem + O_COL, vt);
              else
                product_rows<T, D>(tmem + C::DP_COL + buf.at * BLK, base + C::OWN_OFF + C::OWNB,
                                   vt);
              mma_commit(bar.dp_full + 8 * buf.at);
              mma_commit(bar.b_free + 8 * vst.at);
            }
            vst.next();
            buf.next();
          }
        }
      };
      if (fine) steps(std::true_type{});
      else steps(std::false_type{});
      if (lead) {
        mma_commit(ok ? bar.acc : bar.drained + 8);
        if (!ok) bar_drain(bar.drained + 8, 0, waits);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------- blocks `group`, group + 2, ...
    const int group = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int row = m0 + r, off = s.klen - s.qlen;
    const int64_t stat = (int64_t)h * a.R + s.stat0 + row;
    const float delta1 = __ldg(a.delta + stat), lse1 = __ldg(a.lse2 + stat);
    float v_top = 0.f, do_norm = 0.f;  // fp16; reduced below, while the tiles are on their way
    if constexpr (kBwdShift<T> != 0.f) {
      const float* top = a.vtop + (int64_t)(h / a.G) * stat_tiles(a.RK) + s.kstat0 / 128;
      for (int i = lo / 128 + lane; i < (hi + 127) / 128; i += 32)
        v_top = fmaxf(v_top, __ldg(top + i));
      do_norm = __ldg(a.donorm + stat);
    }
    const float2 sc = f2s(a.scale_log2);
    const uint32_t s_at = tmem + lanes + C::S_COL + group * BLK;
    const uint32_t dp_at = tmem + lanes + C::DP_COL + group * BLK;
    uint32_t ph = 0;
    bool ok = true;
    if (OWN_TMEM && total > 0) {
      ok = __all_sync(0xffffffffu, bar_wait(bar.own, 0, waits));
      if (ok) {
        copy_operand<D>(smem + C::OWN_OFF + group * C::OWNB, r,
                        tmem + lanes + Q_COL + group * (D / 2));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar.there);
      }
    }
    // fp16: dS times a power of two, by the row's bound, which is part of its p's
    // exponent
    float ds_up = 1.f, up = -kBwdShift<T>;
    if constexpr (kBwdShift<T> != 0.f) {
      ds_up = ds_scale(do_norm * warp_top(v_top) + fabsf(delta1));
      up += (float)((__float_as_int(ds_up) >> 23) - 127);
    }
    const float2 lse2 = f2s(up - lse1), delta = f2s(-delta1);
    auto blocks = [&](auto few) {  // two loops: as in the forward
      constexpr bool FINE = decltype(few)::value;
      for (int it = group; ok && it < total; it += 2, ph ^= 1u) {
        const int n0 = (b0 + it) * BLK;
        ok = __all_sync(0xffffffffu, bar_wait(bar.s_full + 8 * group, ph, waits));
        if (!ok) break;
        tc_fence_after();
        float x[BLK], y[BLK];
        load64(s_at, x);
        const bool there = bar_test(bar.dp_full + 8 * group, ph);
#pragma unroll
        for (int i = 0; i < BLK; i += 2) {
          const float2 u = f2_fma(f2(x[i], x[i + 1]), sc, lse2);
          x[i] = ex2(u.x);
          x[i + 1] = ex2(u.y);
        }
        ok = __all_sync(0xffffffffu, there || bar_wait(bar.dp_full + 8 * group, ph, waits));
        if (!ok) break;
        tc_fence_after();
        load64(dp_at, y);
#pragma unroll
        for (int i = 0; i < BLK; i += 2) {
          const float2 d = f2_mul(f2(x[i], x[i + 1]), f2_add(f2(y[i], y[i + 1]), delta));
          y[i] = d.x;
          y[i + 1] = d.y;
        }
        if (n0 + BLK > s.klen || (a.causal && n0 + BLK - 1 > m0 + off) ||
            (a.window && n0 <= m0 + N - 1 + off - a.window)) {
          const int to = (a.causal ? min(s.klen, row + off + 1) : s.klen) - n0;
          int from = a.window ? row + off - a.window + 1 - n0 : 0;
          if (sees_one(a, s, row)) from = BLK;
#pragma unroll
          for (int i = 0; i < BLK; ++i)
            if (i < from || i >= to) y[i] = 0.f;
          // rows of K that nothing may be read from: before the first key that a query
          // sees, and past the sequence's end where memory does hold some
          if (n0 < first_key(a, s) || (n0 + BLK > s.klen && s.k0 + s.klen < a.Sk))
            keep_rows<D>(smem + C::A_OFF + (it % NA) * C::STRB, first_key(a, s) - n0,
                         s.klen - n0);
        }
        store64<T>(dp_at, y);
        if (FINE) store64_rest<T>(dp_at + 32, y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar.ds_full + 8 * group);
      }
    };
    if (fine) blocks(std::true_type{});
    else blocks(std::false_type{});
    if (ok && total > 0) {
      ok = __all_sync(0xffffffffu, bar_wait(bar.acc, 0, waits));
      tc_fence_after();
    }
    if (ok) {
      const int row0 = m0 + (warp & 3) * 32;
      T* dst = reinterpret_cast<T*>(const_cast<void*>(a.dq.p)) + (int64_t)s.b * a.dq.sb +
               (int64_t)h * a.dq.sh + (int64_t)(s.q0 + row0) * a.dq.ss + group * (D / 2);
      // queries past the sequence's end (dense tensors) get zeros; through the
      // kept tiles, which every product has read
      store_sums<D / 2>(tmem + lanes + C::ACC_COL + group * (D / 2), a.scale / ds_up, dst, a.dq.ss,
                        limit - row0, row < s.qlen, total > 0, smem + C::OWN_OFF + warp * 4096);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_free(tmem, C::COLS);
}

template <typename T, int D>
int launch_attn_bwd(const AttnArgs& a0, cudaStream_t st) {
  AttnArgs a = a0;
  a.fault = fault_word();
  if (a.fault == nullptr) return cuda_status(cudaErrorInvalidDevice);
  BwdMaps m;
  const int dt = DTypeOf<T>::value;
  // no keys or no queries, hence no copies: maps of any memory
  if (a.Sk == 0) a.k = a.v = a.q;
  if (a.Sq == 0) a.q = a.dout = a.k;
  const int Sq = a.Sq > 0 ? a.Sq : 1, Sk = a.Sk > 0 ? a.Sk : 1;
  int rc = head_map(&m.q, a.q.p, a.q.sb, a.q.ss, a.q.sh, a.B, Sq, a.Hq, D, 64, dt);
  if (rc == BLOTH_OK)
    rc = head_map(&m.k, a.k.p, a.k.sb, a.k.ss, a.k.sh, a.B, Sk, a.Hk, D, 64, dt);
  if (rc == BLOTH_OK)
    rc = head_map(&m.v, a.v.p, a.v.sb, a.v.ss, a.v.sh, a.B, Sk, a.Hk, D, 64, dt);
  if (rc == BLOTH_OK)
    rc = head_map(&m.dout, a.dout.p, a.dout.sb, a.dout.ss, a.dout.sh, a.B, Sq, a.Hq, D, 64, dt);
  if (rc != BLOTH_OK) return rc;
  auto run = [&](auto kern, int smem, int threads, int64_t grid) {
    const int r = prepare_smem((const void*)kern, smem);
    if (r != BLOTH_OK) return r;
    if (grid == 0) return BLOTH_OK;
    if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
    kern<<<(unsigned)grid, threads, smem, st>>>(a, m);
    return launched(cudaGetLastError());
  };
  auto keys = [&](auto sums) {
    constexpr int S = decltype(sums)::value;
    using C = BwdCfg<D, S>;
    return run(attn_dkv_kernel<T, D, S>, C::SMEM, C::THREADS,
               attn_tiles(a.Sk, a.packed, C::TILE) * a.Hk * a.B);
  };
  if (a.dk.p != nullptr) {
    if constexpr (D == 256) {
      rc = keys(std::integral_constant<int, kSumDV>{});
      if (rc == BLOTH_OK) rc = keys(std::integral_constant<int, kSumDK>{});
    } else {
      rc = keys(std::integral_constant<int, kSumDKV>{});
    }
  }
  if (rc == BLOTH_OK && a.dq.p != nullptr) {
    using C = BwdCfg<D, kSumDQ>;
    rc = run(attn_dq_kernel<T, D>, C::SMEM, C::THREADS,
             attn_tiles(a.Sq, a.packed, C::TILE) * a.Hq * a.B);
  }
  return rc;
}

}  // namespace bloth
