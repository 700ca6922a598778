// Attention forward on the tensor cores: 16-bit tensors.
//
// A CTA takes 256 query rows of one head as two tiles of 128 (128 rows, one
// tile, at head_dim 256) and streams the keys they see in blocks of 64. Warps
// 0-3 and 4-7 are one softmax group per tile (thread = row), warps 8 and 9
// issue one tile's matrix products each, warp 10 the copies.
// Per tile t and block j:
//   S = Q_t K_j^T into tensor memory (64 columns of fp32),
//   the group reads its rows of S (S of block j + 1 may then follow), masks,
//   takes the running maximum m (base 2), p = 2^(S scale log2 e - m), adds the
//   row's p, and writes P, rounded to the tensors' type, to one of two buffers
//   of 32 columns,
//   O_t += P V_j with P read from tensor memory.
// What costs here is the hand-over between warps and the issuing warps' own
// instructions, one after the other. At 8192 full rows of 32/8 heads of 128
// (bf16): blocks of 128 keys in one buffer, P over S, and one issuing thread
// 1050 us; blocks of 64 in two buffers of S, P over S, and two issuing warps
// that run converged on uniform addresses 850 us; one buffer of S, freed when it
// has been read, and two of P 831 us (1323 TFLOP/s, 80% of cuBLAS's burst rate of
// 1660). These are from idle, at 1965 MHz; in seconds of calls the 1 kW cap leaves
// 1570 MHz, and 950 us.
//
// The running maximum moves only when a block's maximum exceeds it by more
// than 2^8 (then the group rescales O_t in tensor memory, after its last
// product). Until then p is at most 2^8, which costs no precision: p is
// rounded relative to its own size (fp16: times 2^7, kFwdShift), and sums are fp32.
//
// Tiles whose rows see few keys (kFineKeys) have P as two terms, which take both
// buffers: P of a block then waits for the product of the block before.
//
// Keys past the sequence's end, or below every query's window, are masked in S;
// their rows of V, which a probability of 0 would turn into NaN if they hold an
// infinity, are zeroed in shared memory by the groups (rows past the tensor's
// end are zero-filled by the copy).
//
// Bound at head_dim 128: the products. A block's for one tile take 392 cycles
// with K (a step reads 6 KB of shared memory for 32 cycles of arithmetic) and
// 263 with V, 1310 for both tiles; a block takes 1510 (at 1570 to 1690 MHz). At
// head_dim 64 the groups: 1460 to 1480 cycles a block (1920 to 1965 MHz), of them
// 730 for the exponentials (512 alone, at 16 a cycle and SM), 320 for maximum and
// mask, 130 for the wait for S and 130 to store P. A CTA takes 19,000 and 12,000
// beside its blocks. A quarter of the exponentials as polynomials on the FMA units
// made it slower (700 to 860 us at 8192 full rows), as did leaving the maximum
// out until a block's sum shows that it is needed.
#pragma once

#include "attn_impl.cuh"
#include "tc.cuh"

namespace bloth {

template <int D>
struct FwdCfg {
  static constexpr int TILE = 128;                   // query rows of a tile
  static constexpr int BLK = 64;                     // keys of a block
  static constexpr int THREADS = 352;
  static constexpr int TILES = D == 256 ? 1 : 2;     // tiles of a CTA
  static constexpr int QB = TILE * D * 2, KB = BLK * D * 2;  // bytes of an operand tile
  static constexpr int NST = D == 64 ? 8 : D == 128 ? 5 : 2;  // stages of K and of V
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = TILES * QB;
  static constexpr int V_OFF = K_OFF + NST * KB;
  static constexpr int BAR_OFF = V_OFF + NST * KB;
  static constexpr int BARS = 1 + 4 * NST + 4 + 4 + 2 + 2 + 2 + 1;
  // barriers, the tensor-memory address and the stop flag
  static constexpr int SMEM = BAR_OFF + BARS * 8 + 16;
  static_assert(SMEM <= 227 * 1024, "shared memory");
  // tensor-memory columns: for each tile 64 of S and two buffers of 32 of P, its O,
  // and where there is room its Q
  static constexpr bool Q_TMEM = D != 128;
  static constexpr uint32_t COLS = 512;
  static constexpr uint32_t S_COL = 0, O_COL = TILES * 128, Q_COL = 384;
};

struct FwdMaps {
  CUtensorMap q, k, v;
};

template <typename T, int D>
__global__ void __launch_bounds__(352, 1)
    attn_fwd_kernel(const AttnArgs a, const __grid_constant__ FwdMaps maps) {
  using C = FwdCfg<D>;
  constexpr int N = C::TILE, BLK = C::BLK, NST = C::NST;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_addr(smem);
  // barriers (8 bytes each)
  const uint32_t q_full = base + C::BAR_OFF;
  const uint32_t k_full = q_full + 8, k_free = k_full + 8 * NST;
  const uint32_t v_full = k_free + 8 * NST, v_free = v_full + 8 * NST;
  const uint32_t s_full = v_free + 8 * NST;  // [tile]
  const uint32_t s_read = s_full + 8 * 2;    // [tile]: S is in registers
  const uint32_t p_full = s_read + 8 * 2;    // [tile][buffer]
  const uint32_t o_done = p_full + 8 * 4;    // [tile]: a block's product with V has completed
  const uint32_t drained = o_done + 8 * 2;
  const uint32_t o_last = drained + 8 * 2;   // [tile]: all have
  const uint32_t q_there = o_last + 8 * 2;  // Q_TMEM: both tiles are in tensor memory
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + 8 * C::BARS);
  const Waits waits{reinterpret_cast<volatile int*>(tmem_ptr + 1), a.fault};

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int heads = a.Hq * a.B;
  const int tiles = (int)(gridDim.x / heads);
  const int hb = blockIdx.x % heads, h = hb % a.Hq;
  // the tiles that see most keys (causal) start first
  const AttnSeq s = find_seq<true>(a, hb / a.Hq, tiles - 1 - (int)(blockIdx.x / heads),
                                  C::TILES * N);
  if (s.tile < 0) return;
  const int m0 = s.tile * C::TILES * N;
  const int limit = a.packed ? s.qlen : a.Sq;
  if (m0 >= limit) return;

  // blocks of keys of each tile, and of the CTA
  int first[2], last[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    int lo, hi;
    const int r = m0 + t * N;
    key_range(a, s, r, min(r + N, s.qlen), lo, hi);
    first[t] = lo / BLK;
    last[t] = (hi + BLK - 1) / BLK;
    if (hi <= lo || t >= C::TILES) first[t] = last[t] = 0;
  }
  int b0 = first[0], b1 = last[0];
  if (last[1] > first[1]) {
    b0 = b1 > b0 ? min(b0, first[1]) : first[1];
    b1 = max(b1, last[1]);
  }
  const int nb = b1 - b0;

  if (warp == 8) {
    tmem_alloc(tmem_ptr, C::COLS);
  } else if (threadIdx.x == 0) {
    bar_init(q_full, 1);
    bar_init(q_there, 4 * C::TILES);
    for (int i = 0; i < NST; ++i) {
      bar_init(k_full + 8 * i, 1);
      bar_init(k_free + 8 * i, C::TILES);
      bar_init(v_full + 8 * i, 1);
      bar_init(v_free + 8 * i, C::TILES);
    }
    for (int i = 0; i < 4; ++i) bar_init(p_full + 8 * i, 4);
    for (int t = 0; t < 2; ++t) {
      bar_init(s_full + 8 * t, 1);
      bar_init(s_read + 8 * t, 4);
      bar_init(o_done + 8 * t, 1);
      bar_init(drained + 8 * t, 1);
      bar_init(o_last + 8 * t, 1);
    }
    *waits.stop = 0;
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;

  if (warp == 10) {
    // ------------------------------------------------------------- copies
    if (lane == 0 && nb > 0) {
      bar_expect(q_full, C::TILES * C::QB);
      load_tile<D, N>(base + C::Q_OFF, &maps.q, s.q0 + m0, h, s.b, q_full);
      if (C::TILES == 2)
        load_tile<D, N>(base + C::Q_OFF + C::QB, &maps.q, s.q0 + m0 + N, h, s.b, q_full);
      const int hk = h / a.G;
      int r0 = s.k0 + b0 * BLK, it = 0;
      Ring<NST> st;
      for (; it < nb; ++it, r0 += BLK, st.next()) {
        const uint32_t kf = k_full + 8 * st.at, vf = v_full + 8 * st.at;
        if (!bar_wait(k_free + 8 * st.at, st.phase ^ 1u, waits)) break;
        bar_expect(kf, C::KB);
        load_tile<D, BLK>(base + C::K_OFF + st.at * C::KB, &maps.k, r0, hk, s.b, kf);
        if (!bar_wait(v_free + 8 * st.at, st.phase ^ 1u, waits)) {
          bar_drain(kf, st.phase, waits);
          break;
        }
        bar_expect(vf, C::KB);
        load_tile<D, BLK>(base + C::V_OFF + st.at * C::KB, &maps.v, r0, hk, s.b, vf);
      }
      if (*waits.stop) {  // given up: not before the copies in flight have landed
        bar_drain(q_full, 0, waits);
        for (int i = max(0, it - NST); i < it; ++i) {
          bar_drain(k_full + 8 * (i % NST), (uint32_t)(i / NST) & 1u, waits);
          bar_drain(v_full + 8 * (i % NST), (uint32_t)(i / NST) & 1u, waits);
        }
      }
    }
  } else if (warp >= 8) {
    // ----------------------------------------------------------- products
    if (nb > 0 && warp - 8 < C::TILES) {
      const int t = warp - 8;
      const int f = (t ? first[1] : first[0]) - b0, e = (t ? last[1] : last[0]) - b0;
      const uint32_t qa = base + C::Q_OFF + t * C::QB;
      const uint32_t s_at = tmem + C::S_COL + t * N, o_at = tmem + C::O_COL + t * D;
      const bool lead = elect();
      Ring<NST> kst, vst;
      Ring<2> pb;
      bool ok = bar_wait(C::Q_TMEM ? q_there : q_full, 0, waits);
      tc_fence_after();
      // step j: S of block j, then O of block j - 1; of the CTA's blocks [f, e)
      // are this tile's
      auto steps = [&](auto few) {
        constexpr bool FINE = decltype(few)::value;
        for (int j = 0; ok && j <= nb; ++j) {
          if (j < nb) {
            const bool mine = j >= f && j < e;
            ok = bar_wait(k_full + 8 * kst.at, kst.phase, waits);
            if (ok && mine && j > f)
              ok = bar_wait(s_read + 8 * t, (uint32_t)(j - f - 1) & 1u, waits);
            if (!ok) break;
            tc_fence_after();
            if (lead) {
              if (mine) {
                const uint32_t kt = base + C::K_OFF + kst.at * C::KB;
                if constexpr (C::Q_TMEM)
                  product_rows_ts<T, D>(s_at, tmem + C::Q_COL + t * (D / 2), kt);
                else
                  product_rows<T, D>(s_at, qa, kt);
                mma_commit(s_full + 8 * t);
              }
              // (a commit completes with the products before it, if there are any)
              mma_commit(k_free + 8 * kst.at);
            }
            kst.next();
          }
          if (j > 0) {
            const bool mine = j - 1 >= f && j - 1 < e;
            ok = bar_wait(v_full + 8 * vst.at, vst.phase, waits);
            if (ok && mine) ok = bar_wait(p_full + 16 * t + 8 * pb.at, pb.phase, waits);
            if (!ok) break;
            tc_fence_after();
            if (lead) {
              if (mine) {
                const uint32_t vt = base + C::V_OFF + vst.at * C::KB;
                product_cols<T, D>(o_at, s_at + BLK + (FINE ? 0 : pb.at * 32), vt, j - 1 > f);
                if (FINE) product_cols<T, D>(o_at, s_at + BLK + 32, vt, true);
                mma_commit((j - 1 < e - 1 ? o_done : o_last) + 8 * t);
              }
              mma_commit(v_free + 8 * vst.at);
            }
            vst.next();
            if (mine) pb.next();
          }
        }
      };
      if (few_keys(a, s, min(m0 + t * N + N, s.qlen))) steps(std::true_type{});
      else steps(std::false_type{});
      if (!ok && lead) {  // given up: not before the products in flight have completed
        mma_commit(drained + 8 * t);
        bar_drain(drained + 8 * t, 0, waits);
      }
      __syncwarp();
    }
  } else if (warp < 4 * C::TILES) {
    // ------------------------------------------------------------ softmax
    const int t = warp >> 2;
    const int row = m0 + t * N + (threadIdx.x & 127);  // of the sequence
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_at = tmem + lanes + C::O_COL + t * D;
    const int f = t ? first[1] : first[0], e = t ? last[1] : last[0];
    const int off = s.klen - s.qlen;
    const float2 sc = f2s(a.scale_log2);
    // Every row of the tile sees every key of the blocks that start at keys
    // [clear0, clear1] (rows past the sequence's end do not count: they are not
    // written); in the others row sees keys [lo, hi).
    const int clear1 = min(s.klen, a.causal ? m0 + t * N + off + 1 : s.klen) - BLK;
    const int clear0 = a.window ? min(m0 + t * N + N, s.qlen) + off - a.window : 0;
    const int row_hi = a.causal ? min(s.klen, row + off + 1) : s.klen;
    const int row_lo = a.window ? row + off - a.window + 1 : 0;
    float m = -INFINITY, l = 0.f;
    bool ok = true, there = false;
    if (C::Q_TMEM && nb > 0) {
      ok = __all_sync(0xffffffffu, bar_wait(q_full, 0, waits));
      if (ok) {
        copy_operand<D>(smem + C::Q_OFF + t * C::QB, threadIdx.x & 127,
                        tmem + lanes + C::Q_COL + t * (D / 2));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(q_there);
      }
    }
    float x[BLK];
    const uint32_t s_at = tmem + lanes + C::S_COL + t * N;
    // Two loops, and two of the products: with a flag inside of them instead, the
    // softmax took 881 us for 727 (8192 full rows of 32/8 heads of 64), the products
    // 983 for 922 (of 128).
    auto blocks = [&](auto few) {
      constexpr bool FINE = decltype(few)::value;
      for (int j = f; j < e; ++j) {
        if (!there) there = ok && bar_wait(s_full + 8 * t, (uint32_t)(j - f) & 1u, waits);
        ok = __all_sync(0xffffffffu, there);
        if (!ok) break;
        tc_fence_after();
        load64(s_at, x);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(s_read + 8 * t);
        const int n0 = j * BLK;
        if (n0 > clear1 || n0 < clear0) {
          const int hi = row_hi - n0, lo = row_lo - n0;
#pragma unroll
          for (int i = 0; i < BLK; ++i)
            if (i >= hi || i < lo) x[i] = -INFINITY;
          // rows of V that nothing may be read from: before the first key that a query
          // sees, and past the sequence's end where memory does hold some
          const int seen0 = first_key(a, s);
          if (n0 < seen0 || (n0 + BLK > s.klen && s.k0 + s.klen < a.Sk)) {
            const int it = j - b0, st = it % NST;
            ok = __all_sync(0xffffffffu,
                            bar_wait(v_full + 8 * st, (uint32_t)(it / NST) & 1u, waits));
            if (!ok) break;
            unsigned char* vt = smem + C::V_OFF + st * C::KB;
            if (n0 < seen0) zero_rows<D>(vt, 0, seen0 - n0);
            if (n0 + BLK > s.klen) zero_rows<D>(vt, s.klen - n0, BLK);
          }
        }
        float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int i = 4; i + 8 <= BLK; i += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u) top[u] = max3(top[u], x[i + u], x[i + 4 + u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) top[u] = fmaxf(top[u], x[BLK - 4 + u]);
        const float mb = max3(fmaxf(top[0], top[1]), top[2], top[3]) * a.scale_log2;
        if (j == f) {
          m = mb;
        } else if (__any_sync(0xffffffffu, mb > m + 8.f)) {
          const float mn = mb > m + 8.f ? mb : m;
          const float w = mn == m ? 1.f : ex2(m - mn);
          m = mn;
          l *= w;
          // O_t, after the product of the block before; the one before that has
          // completed, since S of this block was issued after it
          ok = __all_sync(0xffffffffu, bar_wait(o_done + 8 * t, (uint32_t)(j - f - 1) & 1u, waits));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(o_at + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w);
            tmem_st16(o_at + c * 16, o);
          }
        }
        // whether the next block's S is there: asked before the exponentials, so
        // that the answer (200 cycles) comes during them
        there = j + 1 < e && bar_test(s_full + 8 * t, (uint32_t)(j + 1 - f) & 1u);
        // a row that has seen nothing (m = -inf) is masked everywhere: 2^(-inf - 0) = 0
        const float2 from = f2s(m == -INFINITY ? 0.f : kFwdShift<T> - m);
        float2 sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < BLK; i += 2) {
          const float2 y = f2_fma(f2(x[i], x[i + 1]), sc, from);
          x[i] = ex2(y.x);
          x[i + 1] = ex2(y.y);
          sum[(i / 2) & 1] = f2_add(sum[(i / 2) & 1], f2(x[i], x[i + 1]));
        }
        if constexpr (FINE) {
          if (j > f) {
            ok = __all_sync(0xffffffffu,
                            bar_wait(o_done + 8 * t, (uint32_t)(j - f - 1) & 1u, waits));
            if (!ok) break;
            tc_fence_after();
          }
          store64<T>(s_at + BLK, x);
          store64_rest<T>(s_at + BLK + 32, x);
        } else {
          store64<T>(s_at + BLK + ((j - f) & 1) * 32, x);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(p_full + 16 * t + 8 * ((j - f) & 1));
      }
    };
    if (few_keys(a, s, min(m0 + t * N + N, s.qlen))) blocks(std::true_type{});
    else blocks(std::false_type{});
    if (ok && e > f) {
      ok = __all_sync(0xffffffffu, bar_wait(o_last + 8 * t, 0, waits));
      tc_fence_after();
    } else if (ok && nb > 0) {  // no keys, but a copy of Q that its memory waits for
      ok = __all_sync(0xffffffffu, bar_wait(q_full, 0, waits));
    }
    if (ok) {
      const bool in = row < s.qlen, any = e > f && in;
      const float inv = any && l != 0.f ? 1.f / l : 0.f;
      // through the tile's Q, which every product with K has read
      const int row0 = m0 + t * N + (warp & 3) * 32;
      unsigned char* sm = smem + C::Q_OFF + t * C::QB + (warp & 3) * 4096;
      const int64_t at = (int64_t)s.b * a.o.sb + (int64_t)h * a.o.sh +
                         (int64_t)(s.q0 + row0) * a.o.ss;
      T* out = reinterpret_cast<T*>(const_cast<void*>(a.o.p)) + at;
#pragma unroll 1
      for (int c = 0; c < D; c += 64) {
        uint32_t w[32] = {}, v[32] = {};
        if (e > f) {  // the whole group alike
          load64(o_at + c, x);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            split2<T, kRestUp<T>>(x[2 * i] * inv, x[2 * i + 1] * inv, w[i], v[i]);
            if (inv == 0.f) w[i] = v[i] = 0u;
          }
        }
        store_rows<64>(sm, w, out + c, a.o.ss, limit - row0);
        if (a.rest != nullptr)
          store_rows<64>(sm, v, reinterpret_cast<T*>(a.rest) + at + c, a.o.ss, limit - row0);
      }
      if (row < limit && a.lse != nullptr)
        a.lse[((int64_t)s.b * a.Hq + h) * a.Sq + s.q0 + row] =
            inv != 0.f ? (m - kFwdShift<T> + log2f(l)) * kLn2 : -INFINITY;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_free(tmem, C::COLS);
}

template <typename T, int D>
int launch_attn_fwd(const AttnArgs& a0, cudaStream_t st) {
  using C = FwdCfg<D>;
  AttnArgs a = a0;
  a.fault = fault_word();
  if (a.fault == nullptr) return cuda_status(cudaErrorInvalidDevice);
  FwdMaps m;
  const int dt = DTypeOf<T>::value;
  int rc = head_map(&m.q, a.q.p, a.q.sb, a.q.ss, a.q.sh, a.B, a.Sq, a.Hq, D, 64, dt);
  if (a.Sk == 0) a.k = a.v = a.q;  // no keys, hence no copies: a map of any memory
  const int Sk = a.Sk > 0 ? a.Sk : 1;
  if (rc == BLOTH_OK)
    rc = head_map(&m.k, a.k.p, a.k.sb, a.k.ss, a.k.sh, a.B, Sk, a.Hk, D, 64, dt);
  if (rc == BLOTH_OK)
    rc = head_map(&m.v, a.v.p, a.v.sb, a.v.ss, a.v.sh, a.B, Sk, a.Hk, D, 64, dt);
  if (rc != BLOTH_OK) return rc;
  auto kern = attn_fwd_kernel<T, D>;
  if ((rc = prepare_smem((const void*)kern, C::SMEM)) != BLOTH_OK) return rc;
  const int64_t grid = attn_tiles(a.Sq, a.packed, C::TILES * C::TILE) * a.Hq * a.B;
  if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
  kern<<<(unsigned)grid, C::THREADS, C::SMEM, st>>>(a, m);
  return launched(cudaGetLastError());
}

}  // namespace bloth
