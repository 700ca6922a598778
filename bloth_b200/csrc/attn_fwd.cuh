// Attention forward on the tensor cores: 16-bit tensors, head_dim 64 or 128.
//
// A CTA takes 256 query rows of one head as two tiles of 128 and streams the
// keys they see in blocks of 128. Warps 0-3 and 4-7 are one softmax group per
// tile (thread = row), warp 8 issues the matrix products, warp 9 the copies
// (warps 10 and 11 only complete its warpgroup).
// Per tile t and block j:
//   S_t = Q_t K_j^T into tensor memory (128 columns of fp32),
//   the group reads its row of S_t, masks, takes the running maximum m (base
//   2), p = 2^(S scale log2 e - m), adds the row's p, and writes P_t, rounded
//   to the tensors' type, over the first 64 columns of S_t,
//   O_t += P_t V_j with P_t read from tensor memory.
// The tensor core works on one tile's products while the other tile's group
// computes: products are issued in the order PV_0(j), QK_0(j+1), PV_1(j),
// QK_1(j+1), each waiting for its own group only.
//
// The running maximum moves only when a block's maximum exceeds it by more
// than 2^8 (then O_t is rescaled in tensor memory by the group itself, whose
// previous product has completed because S_t's product was issued after it).
// Until then p is at most 2^8, which costs no precision: p is rounded
// relative to its own size, and sums are fp32.
//
// Keys past the sequence's end are masked in S; their rows of V, which a
// probability of 0 would turn into NaN if they hold an infinity, are zeroed
// in shared memory by the groups (rows past the tensor's end are zero-filled
// by the copy).
//
// Bound: the exponentials (16 a cycle and SM) and the products (128 x 128 x
// 128 in 512 cycles) take the same time at head_dim 128.
#pragma once

#include "attn_impl.cuh"
#include "tc.cuh"

namespace bloth {

template <int D>
struct FwdCfg {
  static constexpr int TILE = 128;
  static constexpr int THREADS = 384;
  // registers of a softmax thread, whose row of 128 scores stays in them, and
  // of the third warpgroup's (12 warps are launched with 168 each)
  static constexpr int SOFT_REGS = 224, ISSUE_REGS = 40;
  static constexpr int OPB = TILE * D * 2;           // bytes of one operand tile
  static constexpr int NK = D == 64 ? 4 : 3, NV = D == 64 ? 4 : 2;  // stages of K and V
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = 2 * OPB;
  static constexpr int V_OFF = K_OFF + NK * OPB;
  static constexpr int BAR_OFF = V_OFF + NV * OPB;
  static constexpr int BARS = 1 + 2 * NK + 2 * NV + 8 + 1;
  // barriers, the tensor-memory address and the stop flag
  static constexpr int SMEM = BAR_OFF + BARS * 8 + 16;
  static_assert(SMEM <= 227 * 1024, "shared memory");
  // tensor-memory columns: S_0, S_1, O_0, O_1
  static constexpr uint32_t COLS = 512;
  static constexpr uint32_t S_COL = 0, O_COL = 256;
};

struct FwdMaps {
  CUtensorMap q, k, v;
};

// Whether any (row, column) of rows [m0, m0 + 128) and keys [n0, n0 + 128) is
// not seen (rows past the sequence's end do not count: they are not written).
__device__ __forceinline__ bool block_masked(const AttnArgs& a, const AttnSeq& s, int m0, int n0) {
  const int off = s.klen - s.qlen;
  if (n0 + 128 > s.klen) return true;
  if (a.causal && n0 + 127 > m0 + off) return true;
  return a.window && n0 <= min(m0 + 127, s.qlen - 1) + off - a.window;
}

// p of quarter PART (32 columns) of a row of 128, packed into r, their sum
// added to `sum`. A row that has seen nothing (m = -inf) is masked
// everywhere: 2^(-inf - 0) = 0.
template <typename T, int PART>
__device__ __forceinline__ void softmax_part(const float (&x)[128], float2 sc, float m,
                                             uint32_t (&r)[16], float2& sum) {
  const float2 base = f2s(m == -INFINITY ? 0.f : -m);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 y = f2_fma(f2(x[PART * 32 + 2 * i], x[PART * 32 + 2 * i + 1]), sc, base);
    const float2 p = f2(ex2(y.x), ex2(y.y));
    sum = f2_add(sum, p);
    r[i] = pack2<T>(p.x, p.y);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(384, 1)
    attn_fwd_kernel(const AttnArgs a, const __grid_constant__ FwdMaps maps) {
  using C = FwdCfg<D>;
  constexpr int N = C::TILE, NK = C::NK, NV = C::NV;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;
  uint64_t* k_free = k_full + NK;
  uint64_t* v_full = k_free + NK;
  uint64_t* v_free = v_full + NV;
  uint64_t* s_full = v_free + NV;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 4;  // p_full: each tile's first half, then each one's second
  uint64_t* drained = o_full + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* stop = reinterpret_cast<volatile int*>(tmem_ptr + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = a.Hq * a.B;
  const int tiles = (int)(gridDim.x / heads);
  const int hb = blockIdx.x % heads, h = hb % a.Hq;
  // the tiles that see most keys (causal) start first
  const AttnSeq s = find_seq<true>(a, hb / a.Hq, tiles - 1 - (int)(blockIdx.x / heads), 2 * N);
  if (s.tile < 0) return;
  const int m0 = s.tile * 2 * N;
  const int limit = a.packed ? s.qlen : a.Sq;
  if (m0 >= limit) return;

  // blocks of keys of each tile, and of the CTA
  int first[2], last[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    int lo, hi;
    const int r = m0 + t * N;
    key_range(a, s, r, min(r + N, s.qlen), lo, hi);
    first[t] = lo / N;
    last[t] = (hi + N - 1) / N;
    if (hi <= lo) first[t] = last[t] = 0;
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
    mbar_init(q_full, 1);
    for (int i = 0; i < NK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_free[i], 1);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_free[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&p_full[2 + t], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(drained, 1);
    *stop = 0;
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;

  if (warp >= 8) {
    lower_registers<C::ISSUE_REGS>();
    if (warp == 9) {
      // ------------------------------------------------------------- copies
      if (lane == 0 && nb > 0) {
        mbar_arrive_expect_tx(q_full, 2 * C::OPB);
        for (int t = 0; t < 2; ++t)
          for (int c = 0; c < D / 64; ++c)
            tma_load(smem + C::Q_OFF + t * C::OPB + c * N * 128, &maps.q, c * 64,
                     s.q0 + m0 + t * N, h, s.b, q_full);
        int it = 0;
        for (; it < nb; ++it) {
          const int sk = it % NK, sv = it % NV;
          const uint32_t pk = (uint32_t)(it / NK) & 1u, pv = (uint32_t)(it / NV) & 1u;
          if (!tc_wait(&k_free[sk], pk ^ 1u, stop, a.fault)) break;
          mbar_arrive_expect_tx(&k_full[sk], C::OPB);
          for (int c = 0; c < D / 64; ++c)
            tma_load(smem + C::K_OFF + sk * C::OPB + c * N * 128, &maps.k, c * 64,
                     s.k0 + (b0 + it) * N, h / a.G, s.b, &k_full[sk]);
          if (!tc_wait(&v_free[sv], pv ^ 1u, stop, a.fault)) {
            mbar_wait(&k_full[sk], pk, nullptr);
            break;
          }
          mbar_arrive_expect_tx(&v_full[sv], C::OPB);
          for (int c = 0; c < D / 64; ++c)
            tma_load(smem + C::V_OFF + sv * C::OPB + c * N * 128, &maps.v, c * 64,
                     s.k0 + (b0 + it) * N, h / a.G, s.b, &v_full[sv]);
        }
        if (*stop) {  // given up: not before the copies in flight have landed
          mbar_wait(q_full, 0, nullptr);
          for (int i = max(0, it - NK); i < it; ++i)
            mbar_wait(&k_full[i % NK], (uint32_t)(i / NK) & 1u, nullptr);
          for (int i = max(0, it - NV); i < it; ++i)
            mbar_wait(&v_full[i % NV], (uint32_t)(i / NV) & 1u, nullptr);
        }
      }
    } else if (warp == 8) {
      // ----------------------------------------------------------- products
      if (lane == 0 && nb > 0) {
        const uint32_t qa = smem_addr(smem + C::Q_OFF), ka = smem_addr(smem + C::K_OFF),
                       va = smem_addr(smem + C::V_OFF);
        uint32_t p_ph[2] = {0, 0};
        bool ok = tc_wait(q_full, 0, stop, a.fault);
        for (int it = 0; ok && it <= nb; ++it) {
          const int sk = it % NK, sv = (it + NV - 1) % NV;  // K of block it, V of the one before
          if (it > 0) ok = tc_wait(&v_full[sv], (uint32_t)((it - 1) / NV) & 1u, stop, a.fault);
          if (ok && it < nb) ok = tc_wait(&k_full[sk], (uint32_t)(it / NK) & 1u, stop, a.fault);
          if (!ok) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int jp = b0 + it - 1, j = b0 + it;
            if (it > 0 && jp >= first[t] && jp < last[t]) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                ok = tc_wait(&p_full[2 * half + t], p_ph[t], stop, a.fault);
                if (!ok) break;
                tc_fence_after();
                if (half == 0)
                  product_cols<T, D, 0, 4>(tmem + C::O_COL + t * D, tmem + C::S_COL + t * N, 32,
                                           va + sv * C::OPB, jp > first[t]);
                else
                  product_cols<T, D, 4, 8>(tmem + C::O_COL + t * D, tmem + C::S_COL + t * N, 32,
                                           va + sv * C::OPB, true);
              }
              if (!ok) break;
              p_ph[t] ^= 1u;
              if (jp == last[t] - 1) mma_commit(&o_full[t]);
            }
            if (it < nb && j >= first[t] && j < last[t]) {
              product_rows<T, D>(tmem + C::S_COL + t * N, qa + t * C::OPB, ka + sk * C::OPB);
              mma_commit(&s_full[t]);
            }
          }
          if (!ok) break;
          if (it > 0) mma_commit(&v_free[sv]);
          if (it < nb) mma_commit(&k_free[sk]);
        }
        if (!ok) {  // given up: not before the products in flight have completed
          mma_commit(drained);
          mbar_wait(drained, 0, nullptr);
        }
      }
    }
  } else {
    raise_registers<C::SOFT_REGS>();
    // ------------------------------------------------------------ softmax
    const int t = warp >> 2;
    const int row = m0 + t * N + (threadIdx.x & 127);  // of the sequence
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + C::S_COL + t * N;
    const uint32_t o_at = tmem + lanes + C::O_COL + t * D;
    const int f = t ? first[1] : first[0], e = t ? last[1] : last[0];
    const int off = s.klen - s.qlen;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    uint32_t ph = 0;
    for (int j = f; j < e; ++j) {
      ok = __all_sync(0xffffffffu, tc_wait(&s_full[t], ph, stop, a.fault));
      if (!ok) break;
      ph ^= 1u;
      tc_fence_after();
      float x[N];
#pragma unroll
      for (int c = 0; c < N / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(s_at + c * 32, r);
#pragma unroll
        for (int i = 0; i < 32; ++i) x[c * 32 + i] = __uint_as_float(r[i]);
      }
      tmem_wait_ld();
      const int n0 = j * N;
      if (block_masked(a, s, m0 + t * N, n0)) {
        const int hi = (a.causal ? min(s.klen, row + off + 1) : s.klen) - n0;
        const int lo = a.window ? row + off - a.window + 1 - n0 : 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (i >= hi || i < lo) x[i] = -INFINITY;
        // rows of V past the sequence's end that memory does hold
        if (n0 + N > s.klen && s.k0 + s.klen < a.Sk) {
          const int it = j - b0, sv = it % NV;
          ok = __all_sync(0xffffffffu, tc_wait(&v_full[sv], (uint32_t)(it / NV) & 1u, stop, a.fault));
          if (!ok) break;
          const int r0 = s.klen - n0;
          for (int c = threadIdx.x & 127; c < (N - r0) * (D / 8); c += 128) {
            const int r = r0 + c / (D / 8), b = c % (D / 8);
            *reinterpret_cast<uint4*>(smem + C::V_OFF + sv * C::OPB + (b / 8) * (N * 128) +
                                      r * 128 + (b % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
      }
      // p of the first 32 columns with the maximum so far, while the block's
      // maximum is found: it seldom moves, and the exponentials' unit would
      // idle for 450 cycles otherwise
      const float2 sc = f2s(a.scale_log2);
      uint32_t r[16];
      float2 sum = f2(0.f, 0.f);
      if (j > f) softmax_part<T, 0>(x, sc, m, r, sum);
      float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int i = 4; i + 8 <= N; i += 8)
#pragma unroll
        for (int u = 0; u < 4; ++u) top[u] = max3(top[u], x[i + u], x[i + 4 + u]);
#pragma unroll
      for (int u = 0; u < 4; ++u) top[u] = fmaxf(top[u], x[N - 4 + u]);
      const float mb = max3(fmaxf(top[0], top[1]), top[2], top[3]) * a.scale_log2;
      if (j == f) {
        m = mb;
        softmax_part<T, 0>(x, sc, m, r, sum);
      } else if (__any_sync(0xffffffffu, mb > m + 8.f)) {
        const float mn = mb > m + 8.f ? mb : m;
        const float w = mn == m ? 1.f : ex2(m - mn);
        m = mn;
        l *= w;
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld16(o_at + c * 16, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w);
          tmem_st16(o_at + c * 16, o);
        }
        sum = f2(0.f, 0.f);
        softmax_part<T, 0>(x, sc, m, r, sum);
      }
      tmem_st16(s_at, r);
      softmax_part<T, 1>(x, sc, m, r, sum);
      tmem_st16(s_at + 16, r);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
      softmax_part<T, 2>(x, sc, m, r, sum);
      tmem_st16(s_at + 32, r);
      softmax_part<T, 3>(x, sc, m, r, sum);
      tmem_st16(s_at + 48, r);
      l += sum.x + sum.y;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[2 + t]);
    }
    if (ok && e > f) {
      ok = __all_sync(0xffffffffu, tc_wait(&o_full[t], 0, stop, a.fault));
      tc_fence_after();
    }
    if (ok) {
      const bool in = row < s.qlen, any = e > f && in;
      const float inv = any && l != 0.f ? 1.f / l : 0.f;
      T* out = reinterpret_cast<T*>(const_cast<void*>(a.o.p)) + (int64_t)s.b * a.o.sb +
               (int64_t)h * a.o.sh + (int64_t)(s.q0 + row) * a.o.ss;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (e > f) {  // the whole group alike
          tmem_ld32(o_at + c * 32, r);
          tmem_wait_ld();
        }
        if (row < limit) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              w[u] = inv != 0.f ? pack2<T>(__uint_as_float(r[8 * i + 2 * u]) * inv,
                                           __uint_as_float(r[8 * i + 2 * u + 1]) * inv)
                                : 0u;
            *reinterpret_cast<uint4*>(out + c * 32 + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (row < limit && a.lse != nullptr)
        a.lse[((int64_t)s.b * a.Hq + h) * a.Sq + s.q0 + row] =
            inv != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
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
  int rc = head_map(&m.q, a.q.p, a.q.sb, a.q.ss, a.q.sh, a.B, a.Sq, a.Hq, D, C::TILE, dt);
  if (rc == BLOTH_OK)
    rc = head_map(&m.k, a.k.p, a.k.sb, a.k.ss, a.k.sh, a.B, a.Sk, a.Hk, D, C::TILE, dt);
  if (rc == BLOTH_OK)
    rc = head_map(&m.v, a.v.p, a.v.sb, a.v.ss, a.v.sh, a.B, a.Sk, a.Hk, D, C::TILE, dt);
  if (rc != BLOTH_OK) return rc;
  auto kern = attn_fwd_kernel<T, D>;
  if ((rc = prepare_smem((const void*)kern, C::SMEM)) != BLOTH_OK) return rc;
  static const bool enough =
      registers_cover((const void*)kern, 3, 2 * C::SOFT_REGS + C::ISSUE_REGS);
  if (!enough) return cuda_status(cudaErrorLaunchOutOfResources);
  const int64_t grid = attn_tiles(a.Sq, a.packed, 2 * C::TILE) * a.Hq * a.B;
  if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
  kern<<<(unsigned)grid, C::THREADS, C::SMEM, st>>>(a, m);
  return launched(cudaGetLastError());
}

}  // namespace bloth
