// Attention backward on the tensor cores: 16-bit tensors, head_dim 64 or 128.
//
// Two kernels, each of which recomputes the probabilities p = 2^(s scale
// log2 e - lse2) of a block of 128 queries x 128 keys from the rows'
// statistics and writes each gradient element once:
//   dK, dV: a CTA keeps 128 keys and streams the queries that see them, of
//           every head of the group: S^T = K Q^T, dP^T = V dO^T,
//           dV += P^T dO, dK += dS^T Q;
//   dQ:     a CTA keeps 128 queries and streams keys: S = Q K^T,
//           dP = dO V^T, dQ += dS K.
// Seven products instead of the five of a single kernel, whose dQ would be a
// sum over CTAs: fp32 atomics, whose order changes the result, and a pass to
// clear and one to round them (12 bytes an element of dQ and 4 more an
// addition). The gradients here do not depend on scheduling.
//
// P^T, dS^T and dS are rounded to the tensors' type and stay in tensor memory
// as the products' first operand; the streamed tiles are read by the products
// both by rows and by columns, so nothing is transposed or stored again.
// Thread = row of the kept tile, 64 of the block's columns: warps 0-3 columns
// 0-63, warps 4-7 columns 64-127. Warp 8 issues the products, warp 9 the
// copies.
//
// Bound: the products (128 x 128 x 128 in 512 cycles), 2048 cycles a block
// for dK, dV and 1536 for dQ, beside 1024 for its exponentials.
#pragma once

#include "attn_impl.cuh"
#include "tc.cuh"

namespace bloth {

template <int D>
struct BwdCfg {
  static constexpr int TILE = 128;
  static constexpr int THREADS = 320;
  static constexpr int OPB = TILE * D * 2;     // bytes of one operand tile
  // Stages of Q (or K) and of dO (or V). Q and K are read by a block's first
  // and its last product, so two stages leave a copy less than a block's time;
  // dO and V are free after half of it. D = 128, 8192 full rows of 32/8 heads:
  // @@STAGES@@
  static constexpr int NA = D == 64 ? 4 : 3, NB = D == 64 ? 4 : 2;
  static constexpr int OWN_OFF = 0;                // the two kept tiles
  static constexpr int A_OFF = 2 * OPB;            // stages of Q (or K)
  static constexpr int B_OFF = A_OFF + NA * OPB;   // stages of dO (or V)
  static constexpr int STAT_OFF = B_OFF + NB * OPB;  // lse2 and delta, with dO's stages
  static constexpr int BAR_OFF = STAT_OFF + NB * 1024;
  static constexpr int BARS = 1 + 2 * NA + 2 * NB + 8;
  static constexpr int SMEM = BAR_OFF + BARS * 8 + 16;
  static constexpr uint32_t COLS = 512;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct BwdMaps {
  CUtensorMap q, k, v, dout;
};

// One operand tile: rows r0.. of a head, D / 64 boxes.
template <int D>
__device__ __forceinline__ void load_tile(unsigned char* dst, const CUtensorMap* map, int r0, int h,
                                          int b, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c) tma_load(dst + c * 128 * 128, map, c * 64, r0, h, b, bar);
}

// Rows [r0, 128) of an operand tile in shared memory become zeros (256 threads).
template <int D>
__device__ __forceinline__ void zero_rows(unsigned char* tile, int r0) {
  for (int c = threadIdx.x; c < (128 - r0) * (D / 8); c += 256) {
    const int r = r0 + c / (D / 8), b = c % (D / 8);
    *reinterpret_cast<uint4*>(tile + (b / 8) * (128 * 128) + r * 128 + (b % 8) * 16) =
        make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
}

// 64 columns of the thread's row.
__device__ __forceinline__ void load64(uint32_t at, float (&x)[64]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t r[32];
    tmem_ld32(at + c * 32, r);
#pragma unroll
    for (int i = 0; i < 32; ++i) x[c * 32 + i] = __uint_as_float(r[i]);
  }
  tmem_wait_ld();
}
template <typename T>
__device__ __forceinline__ void store64(uint32_t at, const float (&x)[64]) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
  tmem_st32(at, r);
  tmem_wait_st();
}

// `cols` accumulator columns of the thread's row, times f, to 16-bit memory
// (in), or zeros (!keep). `any`, alike in the whole warp: there are sums.
template <typename T>
__device__ __forceinline__ void store_row(uint32_t at, int cols, float f, T* dst, bool in,
                                          bool keep, bool any) {
  keep = keep && any;
#pragma unroll 1
  for (int c = 0; c < cols; c += 32) {
    uint32_t r[32];
    if (any) {
      tmem_ld32(at + c, r);
      tmem_wait_ld();
    }
    if (!in) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        w[u] = keep ? pack2<T>(__uint_as_float(r[8 * i + 2 * u]) * f,
                               __uint_as_float(r[8 * i + 2 * u + 1]) * f)
                    : 0u;
      *reinterpret_cast<uint4*>(dst + c + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// ------------------------------------------------------------------ dK, dV
template <typename T, int D>
__global__ void __launch_bounds__(320, 1)
    attn_dkv_kernel(const AttnArgs a, const __grid_constant__ BwdMaps maps) {
  using C = BwdCfg<D>;
  constexpr int N = C::TILE, NA = C::NA, NB = C::NB;
  // tensor-memory columns: S^T (then P^T), dP^T (then dS^T), dV, dK
  constexpr uint32_t S_COL = 0, DP_COL = 128, DV_COL = 256, DK_COL = 256 + D;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* own_full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* q_full = own_full + 1;
  uint64_t* q_free = q_full + NA;
  uint64_t* o_full = q_free + NA;  // dO and the statistics
  uint64_t* o_free = o_full + NB;
  uint64_t* s_full = o_free + NB;
  uint64_t* p_full = s_full + 1;
  uint64_t* dp_full = p_full + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* acc_full = ds_full + 1;
  uint64_t* drained = acc_full + 1;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(own_full + C::BARS);
  volatile int* stop = reinterpret_cast<volatile int*>(tmem_ptr + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  const int mb = lo / N, nm = hi > lo ? (hi + N - 1) / N - mb : 0;  // query blocks per head
  const int total = nm * a.G;

  if (warp == 8) {
    tmem_alloc(tmem_ptr, C::COLS);
  } else if (threadIdx.x == 0) {
    mbar_init(own_full, 1);
    for (int i = 0; i < NA; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_free[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(&o_full[i], 1);
      mbar_init(&o_free[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, 8);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 8);
    mbar_init(acc_full, 1);
    mbar_init(drained, 1);
    *stop = 0;
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;

  if (warp == 9) {
    if (lane == 0 && total > 0) {
      mbar_arrive_expect_tx(own_full, 2 * C::OPB);
      load_tile<D>(smem + C::OWN_OFF, &maps.k, s.k0 + n0, h, s.b, own_full);
      load_tile<D>(smem + C::OWN_OFF + C::OPB, &maps.v, s.k0 + n0, h, s.b, own_full);
      int it = 0;
      for (; it < total; ++it) {
        const int sa = it % NA, sb = it % NB;
        const uint32_t pa = (uint32_t)(it / NA) & 1u, pb = (uint32_t)(it / NB) & 1u;
        const int hq = h * a.G + it / nm, m0 = (mb + it % nm) * N;
        const int64_t stat = (int64_t)hq * a.R + s.stat0 + m0;
        unsigned char* sp = smem + C::STAT_OFF + sb * 1024;
        if (!tc_wait(&q_free[sa], pa ^ 1u, stop, a.fault)) break;
        mbar_arrive_expect_tx(&q_full[sa], C::OPB);
        load_tile<D>(smem + C::A_OFF + sa * C::OPB, &maps.q, s.q0 + m0, hq, s.b, &q_full[sa]);
        if (!tc_wait(&o_free[sb], pb ^ 1u, stop, a.fault)) {
          mbar_wait(&q_full[sa], pa, nullptr);
          break;
        }
        mbar_arrive_expect_tx(&o_full[sb], C::OPB + 1024);
        bulk_load(sp, a.lse2 + stat, 512, &o_full[sb]);
        bulk_load(sp + 512, a.delta + stat, 512, &o_full[sb]);
        load_tile<D>(smem + C::B_OFF + sb * C::OPB, &maps.dout, s.q0 + m0, hq, s.b, &o_full[sb]);
      }
      if (*stop) {  // given up: not before the copies in flight have landed
        mbar_wait(own_full, 0, nullptr);
        for (int i = max(0, it - NA); i < it; ++i)
          mbar_wait(&q_full[i % NA], (uint32_t)(i / NA) & 1u, nullptr);
        for (int i = max(0, it - NB); i < it; ++i)
          mbar_wait(&o_full[i % NB], (uint32_t)(i / NB) & 1u, nullptr);
      }
    }
  } else if (warp == 8) {
    if (lane == 0 && total > 0) {
      const uint32_t ka = smem_addr(smem + C::OWN_OFF), va = ka + C::OPB;
      const uint32_t qa = smem_addr(smem + C::A_OFF), oa = smem_addr(smem + C::B_OFF);
      bool ok = tc_wait(own_full, 0, stop, a.fault) && tc_wait(&q_full[0], 0, stop, a.fault);
      if (ok) {
        product_rows<T, D>(tmem + S_COL, ka, qa);
        mma_commit(s_full);
        ok = tc_wait(&o_full[0], 0, stop, a.fault);
      }
      if (ok) {
        product_rows<T, D>(tmem + DP_COL, va, oa);
        mma_commit(dp_full);
      }
      for (int it = 0; ok && it < total; ++it) {
        const int sa = it % NA, sb = it % NB, na = (it + 1) % NA, nb = (it + 1) % NB;
        if (!(ok = tc_wait(p_full, it & 1, stop, a.fault))) break;
        tc_fence_after();
        product_cols<T, D>(tmem + DV_COL, tmem + S_COL, 64, oa + sb * C::OPB, it > 0);
        if (it + 1 < total) {
          if (!(ok = tc_wait(&q_full[na], (uint32_t)((it + 1) / NA) & 1u, stop, a.fault))) break;
          product_rows<T, D>(tmem + S_COL, ka, qa + na * C::OPB);
          mma_commit(s_full);
        }
        if (!(ok = tc_wait(ds_full, it & 1, stop, a.fault))) break;
        tc_fence_after();
        product_cols<T, D>(tmem + DK_COL, tmem + DP_COL, 64, qa + sa * C::OPB, it > 0);
        mma_commit(&q_free[sa]);
        mma_commit(&o_free[sb]);  // not before dS: the statistics lie with dO
        if (it + 1 < total) {
          if (!(ok = tc_wait(&o_full[nb], (uint32_t)((it + 1) / NB) & 1u, stop, a.fault))) break;
          product_rows<T, D>(tmem + DP_COL, va, oa + nb * C::OPB);
          mma_commit(dp_full);
        }
      }
      mma_commit(ok ? acc_full : drained);
      if (!ok) mbar_wait(drained, 0, nullptr);
    }
  } else {
    const int half = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int key = n0 + r, off = s.klen - s.qlen;
    const uint32_t s_at = tmem + lanes + S_COL + half * 64;
    const uint32_t dp_at = tmem + lanes + DP_COL + half * 64;
    bool ok = true;
    for (int it = 0; it < total; ++it) {
      const int sa = it % NA, sb = it % NB;
      const int m0 = (mb + it % nm) * N;
      const float* stat = reinterpret_cast<const float*>(smem + C::STAT_OFF + sb * 1024);
      ok = tc_wait(&o_full[sb], (uint32_t)(it / NB) & 1u, stop, a.fault) &&
           tc_wait(s_full, it & 1, stop, a.fault);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      float x[64];
      load64(s_at, x);
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        const float4 l = *reinterpret_cast<const float4*>(stat + half * 64 + i);
        const float2 u = f2_fma(f2(x[i], x[i + 1]), f2s(a.scale_log2), f2(-l.x, -l.y));
        const float2 w = f2_fma(f2(x[i + 2], x[i + 3]), f2s(a.scale_log2), f2(-l.z, -l.w));
        x[i] = ex2(u.x);
        x[i + 1] = ex2(u.y);
        x[i + 2] = ex2(w.x);
        x[i + 3] = ex2(w.y);
      }
      // columns of this thread's 64 that see its key: [from, to)
      const int c0 = m0 + half * 64;
      const int from = a.causal ? key - off - c0 : 0;
      const int to = min(s.qlen, a.window ? key - off + a.window : s.qlen) - c0;
      const bool masked = m0 + N > s.qlen || (a.causal && n0 + N - 1 - off > m0) ||
                          (a.window && n0 - off + a.window < m0 + N);
      const bool tail = m0 + N > s.qlen && s.q0 + s.qlen < a.Sq;
      if (masked) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (i < from || i >= to) x[i] = 0.f;
        // rows of dO past the sequence's end that memory does hold
        if (tail) zero_rows<D>(smem + C::B_OFF + sb * C::OPB, s.qlen - m0);
      }
      store64<T>(s_at, x);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
      ok = __all_sync(0xffffffffu, tc_wait(dp_full, it & 1, stop, a.fault));
      if (!ok) break;
      tc_fence_after();
      float y[64];
      load64(dp_at, y);
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        const float4 d = *reinterpret_cast<const float4*>(stat + 128 + half * 64 + i);
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
        for (int i = 0; i < 64; ++i)
          if (i < from || i >= to) y[i] = 0.f;
        if (tail) zero_rows<D>(smem + C::A_OFF + sa * C::OPB, s.qlen - m0);
      }
      store64<T>(dp_at, y);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok && total > 0) {
      ok = __all_sync(0xffffffffu, tc_wait(acc_full, 0, stop, a.fault));
      tc_fence_after();
    }
    if (ok) {
      const HT& t = half ? a.dk : a.dv;
      T* dst = reinterpret_cast<T*>(const_cast<void*>(t.p)) + (int64_t)s.b * t.sb +
               (int64_t)h * t.sh + (int64_t)(s.k0 + key) * t.ss;
      // keys past the sequence's end (dense tensors) get zeros
      store_row<T>(tmem + lanes + (half ? DK_COL : DV_COL), D, half ? a.scale : 1.f, dst,
                   key < limit, key < s.klen, total > 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_free(tmem, C::COLS);
}

// ---------------------------------------------------------------------- dQ
template <typename T, int D>
__global__ void __launch_bounds__(320, 1)
    attn_dq_kernel(const AttnArgs a, const __grid_constant__ BwdMaps maps) {
  using C = BwdCfg<D>;
  constexpr int N = C::TILE, NA = C::NA, NB = C::NB;
  // tensor-memory columns: S, dP, dQ, and two buffers of dS
  constexpr uint32_t S_COL = 0, DP_COL = 128, DQ_COL = 256, DS_COL = 384;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* own_full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* k_full = own_full + 1;
  uint64_t* k_free = k_full + NA;
  uint64_t* v_full = k_free + NA;
  uint64_t* v_free = v_full + NB;
  uint64_t* sdp_full = v_free + NB;
  uint64_t* read = sdp_full + 1;  // S and dP are in registers
  uint64_t* ds_full = read + 1;
  uint64_t* acc_full = ds_full + 1;
  uint64_t* drained = acc_full + 1;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(own_full + C::BARS);
  volatile int* stop = reinterpret_cast<volatile int*>(tmem_ptr + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = a.Hq * a.B;
  const int tiles = (int)(gridDim.x / heads);
  const int hb = blockIdx.x % heads, h = hb % a.Hq;
  const AttnSeq s = find_seq<true>(a, hb / a.Hq, tiles - 1 - (int)(blockIdx.x / heads), N);
  if (s.tile < 0) return;
  const int m0 = s.tile * N;
  const int limit = a.packed ? s.qlen : a.Sq;
  if (m0 >= limit) return;
  int lo, hi;
  key_range(a, s, m0, min(m0 + N, s.qlen), lo, hi);
  const int b0 = lo / N, total = hi > lo ? (hi + N - 1) / N - b0 : 0;

  if (warp == 8) {
    tmem_alloc(tmem_ptr, C::COLS);
  } else if (threadIdx.x == 0) {
    mbar_init(own_full, 1);
    for (int i = 0; i < NA; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_free[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_free[i], 1);
    }
    mbar_init(sdp_full, 1);
    mbar_init(read, 8);
    mbar_init(ds_full, 8);
    mbar_init(acc_full, 1);
    mbar_init(drained, 1);
    *stop = 0;
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;

  if (warp == 9) {
    if (lane == 0 && total > 0) {
      mbar_arrive_expect_tx(own_full, 2 * C::OPB);
      load_tile<D>(smem + C::OWN_OFF, &maps.q, s.q0 + m0, h, s.b, own_full);
      load_tile<D>(smem + C::OWN_OFF + C::OPB, &maps.dout, s.q0 + m0, h, s.b, own_full);
      int it = 0;
      for (; it < total; ++it) {
        const int sa = it % NA, sb = it % NB;
        const uint32_t pa = (uint32_t)(it / NA) & 1u, pb = (uint32_t)(it / NB) & 1u;
        const int r0 = s.k0 + (b0 + it) * N;
        if (!tc_wait(&k_free[sa], pa ^ 1u, stop, a.fault)) break;
        mbar_arrive_expect_tx(&k_full[sa], C::OPB);
        load_tile<D>(smem + C::A_OFF + sa * C::OPB, &maps.k, r0, h / a.G, s.b, &k_full[sa]);
        if (!tc_wait(&v_free[sb], pb ^ 1u, stop, a.fault)) {
          mbar_wait(&k_full[sa], pa, nullptr);
          break;
        }
        mbar_arrive_expect_tx(&v_full[sb], C::OPB);
        load_tile<D>(smem + C::B_OFF + sb * C::OPB, &maps.v, r0, h / a.G, s.b, &v_full[sb]);
      }
      if (*stop) {
        mbar_wait(own_full, 0, nullptr);
        for (int i = max(0, it - NA); i < it; ++i)
          mbar_wait(&k_full[i % NA], (uint32_t)(i / NA) & 1u, nullptr);
        for (int i = max(0, it - NB); i < it; ++i)
          mbar_wait(&v_full[i % NB], (uint32_t)(i / NB) & 1u, nullptr);
      }
    }
  } else if (warp == 8) {
    if (lane == 0 && total > 0) {
      const uint32_t qa = smem_addr(smem + C::OWN_OFF), oa = qa + C::OPB;
      const uint32_t ka = smem_addr(smem + C::A_OFF), va = smem_addr(smem + C::B_OFF);
      bool ok = tc_wait(own_full, 0, stop, a.fault);
      // S and dP of block it are issued once those of it - 1 are in registers,
      // dQ's product of it - 1 after them
      for (int it = 0; ok && it <= total; ++it) {
        const int sa = it % NA, sb = it % NB, sp = (it + NA - 1) % NA;
        if (it < total) {
          if (!(ok = tc_wait(&k_full[sa], (uint32_t)(it / NA) & 1u, stop, a.fault))) break;
          if (it > 0 && !(ok = tc_wait(read, (it - 1) & 1, stop, a.fault))) break;
          tc_fence_after();
          product_rows<T, D>(tmem + S_COL, qa, ka + sa * C::OPB);
          if (!(ok = tc_wait(&v_full[sb], (uint32_t)(it / NB) & 1u, stop, a.fault))) break;
          product_rows<T, D>(tmem + DP_COL, oa, va + sb * C::OPB);
          mma_commit(sdp_full);
          mma_commit(&v_free[sb]);
        }
        if (it > 0) {
          if (!(ok = tc_wait(ds_full, (it - 1) & 1, stop, a.fault))) break;
          tc_fence_after();
          product_cols<T, D>(tmem + DQ_COL, tmem + DS_COL + ((it - 1) & 1) * 64, 32,
                             ka + sp * C::OPB, it > 1);
          mma_commit(&k_free[sp]);
        }
      }
      mma_commit(ok ? acc_full : drained);
      if (!ok) mbar_wait(drained, 0, nullptr);
    }
  } else {
    const int half = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int row = m0 + r, off = s.klen - s.qlen;
    const int64_t stat = (int64_t)h * a.R + s.stat0 + row;
    const float2 lse2 = f2s(-__ldg(a.lse2 + stat)), delta = f2s(-__ldg(a.delta + stat));
    bool ok = true;
    for (int it = 0; it < total; ++it) {
      const int n0 = (b0 + it) * N;
      ok = __all_sync(0xffffffffu, tc_wait(sdp_full, it & 1, stop, a.fault));
      if (!ok) break;
      tc_fence_after();
      float x[64], y[64];
      load64(tmem + lanes + S_COL + half * 64, x);
      load64(tmem + lanes + DP_COL + half * 64, y);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(read);
#pragma unroll
      for (int i = 0; i < 64; i += 2) {
        const float2 u = f2_fma(f2(x[i], x[i + 1]), f2s(a.scale_log2), lse2);
        const float2 d = f2_mul(f2(ex2(u.x), ex2(u.y)), f2_add(f2(y[i], y[i + 1]), delta));
        y[i] = d.x;
        y[i + 1] = d.y;
      }
      if (n0 + N > s.klen || (a.causal && n0 + N - 1 > m0 + off) ||
          (a.window && n0 <= m0 + N - 1 + off - a.window)) {
        const int to = (a.causal ? min(s.klen, row + off + 1) : s.klen) - n0 - half * 64;
        const int from = a.window ? row + off - a.window + 1 - n0 - half * 64 : 0;
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (i < from || i >= to) y[i] = 0.f;
        // rows of K past the sequence's end that memory does hold
        if (n0 + N > s.klen && s.k0 + s.klen < a.Sk)
          zero_rows<D>(smem + C::A_OFF + (it % NA) * C::OPB, s.klen - n0);
      }
      store64<T>(tmem + lanes + DS_COL + (it & 1) * 64 + half * 32, y);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok && total > 0) {
      ok = __all_sync(0xffffffffu, tc_wait(acc_full, 0, stop, a.fault));
      tc_fence_after();
    }
    if (ok) {
      T* dst = reinterpret_cast<T*>(const_cast<void*>(a.dq.p)) + (int64_t)s.b * a.dq.sb +
               (int64_t)h * a.dq.sh + (int64_t)(s.q0 + row) * a.dq.ss + half * (D / 2);
      // queries past the sequence's end (dense tensors) get zeros
      store_row<T>(tmem + lanes + DQ_COL + half * (D / 2), D / 2, a.scale, dst, row < limit,
                   row < s.qlen, total > 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_free(tmem, C::COLS);
}

template <typename T, int D>
int launch_attn_bwd(const AttnArgs& a0, cudaStream_t st) {
  using C = BwdCfg<D>;
  AttnArgs a = a0;
  a.fault = fault_word();
  if (a.fault == nullptr) return cuda_status(cudaErrorInvalidDevice);
  BwdMaps m;
  const int dt = DTypeOf<T>::value;
  int rc = head_map(&m.q, a.q.p, a.q.sb, a.q.ss, a.q.sh, a.B, a.Sq, a.Hq, D, C::TILE, dt);
  if (rc == BLOTH_OK)
    rc = head_map(&m.k, a.k.p, a.k.sb, a.k.ss, a.k.sh, a.B, a.Sk, a.Hk, D, C::TILE, dt);
  if (rc == BLOTH_OK)
    rc = head_map(&m.v, a.v.p, a.v.sb, a.v.ss, a.v.sh, a.B, a.Sk, a.Hk, D, C::TILE, dt);
  if (rc == BLOTH_OK)
    rc = head_map(&m.dout, a.dout.p, a.dout.sb, a.dout.ss, a.dout.sh, a.B, a.Sq, a.Hq, D, C::TILE,
                  dt);
  if (rc != BLOTH_OK) return rc;
  auto run = [&](auto kern, int64_t grid) {
    const int r = prepare_smem((const void*)kern, C::SMEM);
    if (r != BLOTH_OK) return r;
    if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
    kern<<<(unsigned)grid, C::THREADS, C::SMEM, st>>>(a, m);
    return launched(cudaGetLastError());
  };
  if (a.dk.p != nullptr)
    rc = run(attn_dkv_kernel<T, D>, attn_tiles(a.Sk, a.packed, C::TILE) * a.Hk * a.B);
  if (rc == BLOTH_OK && a.dq.p != nullptr)
    rc = run(attn_dq_kernel<T, D>, attn_tiles(a.Sq, a.packed, C::TILE) * a.Hq * a.B);
  return rc;
}

}  // namespace bloth
