// Attention on the fp32 units, forward and backward: fp32 tensors (whose
// products the tensor cores would round to 16 or 19 bits) and head_dim 256.
//
// A CTA of 256 threads keeps a tile of 64 rows of one head ("own" rows) in
// shared memory as fp32 and streams the rows of the other side past it in
// tiles. Thread (ty, tx) of 16 x 16 holds a 4 x (tile/16) block of a product
// of two tiles: own rows 4*ty.., streamed rows tx, tx + 16, ... Rows are
// padded by 4 floats, so the 16-byte reads of eight neighbouring rows fall in
// different banks. Rows past the sequence's end are zero in shared memory,
// whatever memory holds there.
//
// Bound: fp32 FMA issue. A product of two 4-wide rows costs one 16-byte read
// of each row per 4 values, so a 4 x 4 block does 64 FMA for 8 reads.
#pragma once

#include "attn_impl.cuh"

namespace bloth {

constexpr int kSimtOwn = 64;
constexpr int kSimtThreads = 256;

// `rows` rows of D of head tensor t (batch b, head h, rows r0..) as fp32 into
// dst [tile][D + 4], rows from `rows` on as zeros.
template <typename T, int D>
__device__ __forceinline__ void simt_load(float* dst, int tile, const HT& t, int b, int h, int r0,
                                          int rows) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const T* base = reinterpret_cast<const T*>(t.p) + (int64_t)b * t.sb + (int64_t)h * t.sh +
                  (int64_t)r0 * t.ss;
  for (int c = threadIdx.x; c < tile * (D / VEC); c += kSimtThreads) {
    const int r = c / (D / VEC), x = c % (D / VEC) * VEC;
    float f[VEC];
    if (r < rows) {
      unpack(ldg_pack<T, VEC>(base + (int64_t)r * t.ss + x), f);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < VEC; e += 4)
      *reinterpret_cast<float4*>(dst + r * (D + 4) + x + e) =
          make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
  }
}

// acc[i][j] = own row 4*ty + i . streamed row tx + 16*j
template <int D, int NJ>
__device__ __forceinline__ void simt_dot(const float* own, const float* str, int ty, int tx,
                                         float (&acc)[4][NJ]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = 0.f;
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float4 x[4], y[NJ];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = *reinterpret_cast<const float4*>(own + (4 * ty + i) * (D + 4) + d);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      y[j] = *reinterpret_cast<const float4*>(str + (tx + 16 * j) * (D + 4) + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]);
        acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
        acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]);
        acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
      }
  }
}

// acc[i][c] += sum over the streamed rows t of w[4*ty + i][t] * str[t][column
// of c], columns 64*(c / 4) + 4*tx + c % 4. w has rows of `ldw` floats.
template <int D, int NT>
__device__ __forceinline__ void simt_acc(const float* w, int ldw, const float* str, int ty, int tx,
                                         float (&acc)[4][D / 16]) {
#pragma unroll 2
  for (int t = 0; t < NT; t += 4) {
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(w + (4 * ty + i) * ldw + t);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const float4 y =
            *reinterpret_cast<const float4*>(str + (t + u) * (D + 4) + 64 * c + 4 * tx);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = u == 0 ? x[i].x : u == 1 ? x[i].y : u == 2 ? x[i].z : x[i].w;
          acc[i][4 * c + 0] = fmaf(p, y.x, acc[i][4 * c + 0]);
          acc[i][4 * c + 1] = fmaf(p, y.y, acc[i][4 * c + 1]);
          acc[i][4 * c + 2] = fmaf(p, y.z, acc[i][4 * c + 2]);
          acc[i][4 * c + 3] = fmaf(p, y.w, acc[i][4 * c + 3]);
        }
      }
    }
  }
}

// Row 4*ty + i of acc, times f, to row r0 + 4*ty + i of t (rows < `rows`).
template <typename T, int D>
__device__ __forceinline__ void simt_store(const HT& t, int b, int h, int r0, int rows, int ty,
                                           int tx, const float (&acc)[4][D / 16],
                                           const float (&f)[4]) {
  T* base = reinterpret_cast<T*>(const_cast<void*>(t.p)) + (int64_t)b * t.sb + (int64_t)h * t.sh +
            (int64_t)r0 * t.ss;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (4 * ty + i >= rows) continue;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[i][4 * c + e] * f[i];
      stg_pack<T, 4>(base + (int64_t)(4 * ty + i) * t.ss + 64 * c + 4 * tx, pack<T, 4>(v));
    }
  }
}

template <int D>
constexpr size_t simt_fwd_smem() {
  return (2 * kSimtOwn * (D + 4) + kSimtOwn * (kSimtOwn + 4)) * sizeof(float);
}

template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads) attn_simt_fwd_kernel(const AttnArgs a) {
  constexpr int N = kSimtOwn, LD = D + 4, LP = N + 4;
  extern __shared__ __align__(16) float sm[];
  float* qs = sm;
  float* ks = qs + N * LD;  // a tile of K, then the same rows of V
  float* ps = ks + N * LD;
  const int heads = a.Hq * a.B;
  const int tiles = (int)(gridDim.x / heads);
  const int hb = blockIdx.x % heads, h = hb % a.Hq;
  const AttnSeq s = find_seq<true>(a, hb / a.Hq, tiles - 1 - (int)(blockIdx.x / heads), N);
  if (s.tile < 0) return;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int m0 = s.tile * N;
  const int limit = a.packed ? s.qlen : a.Sq;  // dense: rows past qlen are written as zeros
  if (m0 >= limit) return;
  const int rows = max(0, min(N, s.qlen - m0));
  int lo, hi;
  key_range(a, s, m0, m0 + rows, lo, hi);
  simt_load<T, D>(qs, N, a.q, s.b, h, s.q0 + m0, rows);
  float acc[4][D / 16], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) acc[i][c] = 0.f;
  }
  for (int n0 = lo / N * N; n0 < hi; n0 += N) {
    const int nk = min(N, s.klen - n0);
    __syncthreads();
    simt_load<T, D>(ks, N, a.k, s.b, h / a.G, s.k0 + n0, nk);
    __syncthreads();
    float x[4][4];
    simt_dot<D, 4>(qs, ks, ty, tx, x);
    __syncthreads();
    simt_load<T, D>(ks, N, a.v, s.b, h / a.G, s.k0 + n0, nk);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[i][j] = see_keys(a, s, m0 + 4 * ty + i, n0 + tx + 16 * j) ? x[i][j] * a.scale : -INFINITY;
        top = fmaxf(top, x[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m[i], top);
      const float from = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: all terms are 0
      const float f = expf(m[i] - from);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = expf(x[i][j] - from);
        sum += p;
        ps[(4 * ty + i) * LP + tx + 16 * j] = p;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = fmaf(l[i], f, sum);
#pragma unroll
      for (int c = 0; c < D / 16; ++c) acc[i][c] *= f;
    }
    __syncthreads();
    simt_acc<D, N>(ps, LP, ks, ty, tx, acc);
  }
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = l[i] > 0.f || l[i] != l[i] ? 1.f / l[i] : 0.f;
  const int out_rows = min(N, limit - m0);
  simt_store<T, D>(a.o, s.b, h, s.q0 + m0, out_rows, ty, tx, acc, f);
  if constexpr (sizeof(T) == 2) {
    if (a.rest != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const float y = acc[i][c] * f[i];
          acc[i][c] = y - to_f(from_f<T>(y));
        }
        f[i] = 1.f;
      }
      HT rest = a.o;
      rest.p = a.rest;
      simt_store<T, D>(rest, s.b, h, s.q0 + m0, out_rows, ty, tx, acc, f);
    }
  }
  if (tx == 0 && a.lse != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * ty + i < out_rows)
        a.lse[((int64_t)s.b * a.Hq + h) * a.Sq + s.q0 + m0 + 4 * ty + i] =
            l[i] == 0.f ? -INFINITY : m[i] + logf(l[i]);
  }
}

// Rows of a streamed tile of the backward: two own tiles, two streamed ones
// and the two weight tiles have to fit in shared memory.
template <int D> constexpr int kSimtStr = D == 256 ? 32 : 64;

template <int D>
constexpr size_t simt_bwd_smem() {
  return (2 * (kSimtOwn + kSimtStr<D>) * (D + 4) + 2 * kSimtOwn * (kSimtStr<D> + 4)) *
         sizeof(float);
}

// DKV: own rows are keys (K, V), the queries of every head of the group (Q,
// dO) stream past, dk and dv are written. Else own rows are queries, the keys
// stream, dq is written.
template <typename T, int D, bool DKV>
__global__ void __launch_bounds__(kSimtThreads) attn_simt_bwd_kernel(const AttnArgs a) {
  constexpr int N = kSimtOwn, M = kSimtStr<D>, NJ = M / 16, LD = D + 4, LP = M + 4;
  extern __shared__ __align__(16) float sm[];
  float* own1 = sm;  // K or Q
  float* own2 = own1 + N * LD;  // V or dO
  float* str1 = own2 + N * LD;  // Q or K
  float* str2 = str1 + M * LD;  // dO or V
  float* ps = str2 + M * LD;
  float* ds = ps + N * LP;
  const int H = DKV ? a.Hk : a.Hq;
  const int heads = H * a.B;
  const int hb = blockIdx.x % heads, h = hb % H;
  const int tiles = (int)(gridDim.x / heads), bt = (int)(blockIdx.x / heads);
  const AttnSeq s = find_seq<!DKV>(a, hb / H, DKV ? bt : tiles - 1 - bt, N);
  if (s.tile < 0) return;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int r0 = s.tile * N;
  const int len = DKV ? s.klen : s.qlen;
  const int limit = a.packed ? len : (DKV ? a.Sk : a.Sq);
  if (r0 >= limit) return;
  const int rows = max(0, min(N, len - r0));
  int lo, hi;
  if (DKV) query_range(a, s, r0, r0 + rows, lo, hi);
  else key_range(a, s, r0, r0 + rows, lo, hi);
  const int own0 = (DKV ? s.k0 : s.q0) + r0, strb = DKV ? s.q0 : s.k0;
  simt_load<T, D>(own1, N, DKV ? a.k : a.q, s.b, h, own0, rows);
  simt_load<T, D>(own2, N, DKV ? a.v : a.dout, s.b, h, own0, rows);
  float acc1[4][D / 16], acc2[DKV ? 4 : 1][D / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      acc1[i][c] = 0.f;
      if (DKV) acc2[i][c] = 0.f;
    }
  const int h1 = DKV ? h * a.G : h / a.G;
  for (int g = 0; g < (DKV ? a.G : 1); ++g) {
    const int64_t stat = (int64_t)(DKV ? h1 + g : h) * a.R + s.stat0;
    for (int t0 = lo / M * M; t0 < hi; t0 += M) {
      const int nt = min(M, (DKV ? s.qlen : s.klen) - t0);
      __syncthreads();
      simt_load<T, D>(str1, M, DKV ? a.q : a.k, s.b, h1 + g, strb + t0, nt);
      simt_load<T, D>(str2, M, DKV ? a.dout : a.v, s.b, h1 + g, strb + t0, nt);
      __syncthreads();
      float x[4][NJ], y[4][NJ];
      simt_dot<D, NJ>(own1, str1, ty, tx, x);
      simt_dot<D, NJ>(own2, str2, ty, tx, y);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int ro = r0 + 4 * ty + i, rt = t0 + tx + 16 * j;
          const int qi = DKV ? rt : ro, kj = DKV ? ro : rt;
          float p = 0.f, d = 0.f;
          if (see_keys(a, s, qi, kj)) {
            // log2 and exp2 of the same numbers as the forward's, in fp32
            p = exp2f(fmaf(x[i][j], a.scale_log2, -__ldg(a.lse2 + stat + qi)));
            d = p * (y[i][j] - __ldg(a.delta + stat + qi));
          }
          if (DKV) ps[(4 * ty + i) * LP + tx + 16 * j] = p;
          ds[(4 * ty + i) * LP + tx + 16 * j] = d;
        }
      __syncthreads();
      simt_acc<D, M>(ds, LP, str1, ty, tx, acc1);
      if constexpr (DKV) simt_acc<D, M>(ps, LP, str2, ty, tx, acc2);
    }
  }
  const int out_rows = min(N, limit - r0);
  const float fs[4] = {a.scale, a.scale, a.scale, a.scale};
  simt_store<T, D>(DKV ? a.dk : a.dq, s.b, h, own0, out_rows, ty, tx, acc1, fs);
  if constexpr (DKV) {
    const float f1[4] = {1.f, 1.f, 1.f, 1.f};
    simt_store<T, D>(a.dv, s.b, h, own0, out_rows, ty, tx, acc2, f1);
  }
}

// delta = rowsum(dO * O) and lse in base 2 for the backward kernels, for every
// row of every 128-row tile of a sequence: a row past the sequence's end, or
// one that sees nothing, gets lse2 = +inf and delta = 0, so its recomputed
// probabilities are exp2(x - inf) = 0. HBM-bound: reads O, its rest and dO once. A row
// takes D / 8 lanes of 16-bit (D / 4 of fp32) elements, one 16-byte load of
// each tensor per lane and pass.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_stats_kernel(const AttnArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T), LPR = D / VEC < 32 ? D / VEC : 32;
  constexpr int PASS = D / (VEC * LPR), RPW = 32 / LPR;
  const int heads = a.Hq * a.B;
  const int hb = blockIdx.x % heads, h = hb % a.Hq;
  const AttnSeq s = find_seq<true>(a, hb / a.Hq, (int)(blockIdx.x / heads), 128);
  if (s.tile < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int m0 = s.tile * 128;
  const int64_t stat = (int64_t)h * a.R + s.stat0 + m0;
  const T* op = reinterpret_cast<const T*>(a.o.p) + (int64_t)s.b * a.o.sb + (int64_t)h * a.o.sh;
  const T* rp =
      reinterpret_cast<const T*>(a.rest) + (int64_t)s.b * a.o.sb + (int64_t)h * a.o.sh;
  const T* dp =
      reinterpret_cast<const T*>(a.dout.p) + (int64_t)s.b * a.dout.sb + (int64_t)h * a.dout.sh;
#pragma unroll
  for (int r = warp * 16 + lane / LPR; r < warp * 16 + 16; r += RPW) {
    const bool in = m0 + r < s.qlen;
    const int64_t row = s.q0 + m0 + r;
    float sum = 0.f;
    if (in) {
#pragma unroll
      for (int u = 0; u < PASS; ++u) {
        const int x = (u * LPR + lane % LPR) * VEC;
        float f[VEC], g[VEC];
        unpack(ldg_pack<T, VEC>(op + row * a.o.ss + x), f);
        unpack(ldg_pack<T, VEC>(dp + row * a.dout.ss + x), g);
        if (sizeof(T) == 2 && a.rest != nullptr) {
          float e[VEC];
          unpack(ldg_pack<T, VEC>(rp + row * a.o.ss + x), e);
#pragma unroll
          for (int i = 0; i < VEC; ++i) f[i] += e[i];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum = fmaf(f[e], g[e], sum);
      }
    }
    sum = group_lane_sum<LPR>(sum);
    if (lane % LPR == 0) {
      const float l = in ? a.lse[((int64_t)s.b * a.Hq + h) * a.Sq + row] : -INFINITY;
      const bool none = l == -INFINITY;
      a.lse2[stat + r] = none ? INFINITY : l * kLog2e;
      a.delta[stat + r] = none ? 0.f : sum;
    }
  }
}

template <typename F>
int attn_head_dim(int D, F&& f) {
  switch (D) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 256: return f(std::integral_constant<int, 256>{});
    default: return BLOTH_ERR_SHAPE;
  }
}

template <typename T>
int attn_simt_fwd(const AttnArgs& a, int D, cudaStream_t st) {
  return attn_head_dim(D, [&](auto dd) {
    constexpr int DD = decltype(dd)::value;
    auto kern = attn_simt_fwd_kernel<T, DD>;
    const int rc = prepare_smem((const void*)kern, simt_fwd_smem<DD>());
    if (rc != BLOTH_OK) return rc;
    const int64_t grid = attn_tiles(a.Sq, a.packed, kSimtOwn) * a.Hq * a.B;
    if (grid == 0) return BLOTH_OK;
    if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
    return launched(launch_ex(kern, (unsigned)grid, kSimtThreads, simt_fwd_smem<DD>(), st, a));
  });
}

template <typename T>
int attn_simt_bwd(const AttnArgs& a, int D, cudaStream_t st) {
  return attn_head_dim(D, [&](auto dd) {
    constexpr int DD = decltype(dd)::value;
    auto run = [&](auto kern, int64_t grid) {
      const int rc = prepare_smem((const void*)kern, simt_bwd_smem<DD>());
      if (rc != BLOTH_OK) return rc;
      if (grid == 0) return BLOTH_OK;
      if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
      return launched(launch_ex(kern, (unsigned)grid, kSimtThreads, simt_bwd_smem<DD>(), st, a));
    };
    int rc = BLOTH_OK;
    if (a.dk.p != nullptr)
      rc = run(attn_simt_bwd_kernel<T, DD, true>,
               attn_tiles(a.Sk, a.packed, kSimtOwn) * a.Hk * a.B);
    if (rc == BLOTH_OK && a.dq.p != nullptr)
      rc = run(attn_simt_bwd_kernel<T, DD, false>,
               attn_tiles(a.Sq, a.packed, kSimtOwn) * a.Hq * a.B);
    return rc;
  });
}

template <typename T>
int attn_stats(const AttnArgs& a, int D, cudaStream_t st) {
  return attn_head_dim(D, [&](auto dd) {
    constexpr int DD = decltype(dd)::value;
    const int64_t grid = attn_tiles(a.Sq, a.packed, 128) * a.Hq * a.B;
    if (grid == 0) return BLOTH_OK;
    if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
    return launched(launch_ex(attn_stats_kernel<T, DD>, (unsigned)grid, 256u, 0, st, a));
  });
}

}  // namespace bloth

#define BLOTH_INSTANTIATE_ATTN_SIMT(T)                                  \
  namespace bloth {                                                     \
  template int attn_simt_fwd<T>(const AttnArgs&, int, cudaStream_t);    \
  template int attn_simt_bwd<T>(const AttnArgs&, int, cudaStream_t);    \
  template int attn_stats<T>(const AttnArgs&, int, cudaStream_t);       \
  }
