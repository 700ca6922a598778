// Attention of fp32 tensors, on the fp32 units (the tensor cores would round
// the products' operands to 19 bits): forward and backward.
//
// A CTA keeps a tile of OWN rows of one head ("own" rows) in shared memory and
// streams the rows of the other side past it in tiles. Thread (ty, tx) of
// OWN/4 x 16 holds a 4 x (tile/16) block of a product of two tiles: own rows
// 4*ty.., streamed rows tx, tx + 16, ... Rows are padded by 4 floats, so the
// 16-byte reads of eight neighbouring rows fall in different banks. Rows past
// the sequence's end are zero in shared memory, whatever memory holds there, and
// so are queries before the first that sees a key, and keys before the first
// that a query sees.
//
// OWN is 64 where that gives a CTA for every SM, else 32: half the threads and
// half the work of a CTA (100 rows of 4 heads of 64: dK and dV 35 us with
// 64, 17 with 32).
// dK and dV are written by one CTA per key tile and key head, or, where those
// are fewer than two for an SM, by one per query head into fp32 partial sums
// that simt_sum_kernel adds over the group in order (2048 rows of 16/4 heads of 128: 2139 us
// without, 1035 us with).
//
// Bound: fp32 FMA issue; a 4 x 4 block does 64 FMA for 8 shared-memory reads of
// 16 bytes, which leaves about half of the FMA rate.
#pragma once

#include "attn_rows.cuh"

namespace bloth {

constexpr int kSimtKeys = 64;  // streamed rows of a forward tile

// `rows` rows of D of head tensor t (batch b, head h, rows r0..) as fp32 into
// dst [tile][D + 4], rows from `rows` on as zeros.
template <typename T, int D, int THREADS>
__device__ __forceinline__ void simt_load(float* dst, int tile, const HT& t, int b, int h, int r0,
                                          int rows) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const T* base = reinterpret_cast<const T*>(t.p) + (int64_t)b * t.sb + (int64_t)h * t.sh +
                  (int64_t)r0 * t.ss;
  for (int c = threadIdx.x; c < tile * (D / VEC); c += THREADS) {
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

// Rows before `first` of such a tile become zeros: each thread clears what it
// wrote itself. (2 x 1024 rows of 16/4 heads of 64, forward and backward: 738 us with
// this bound inside simt_load, 735 with a call that is not inlined, 663 so, and 663
// without.)
template <typename T, int D, int THREADS>
__device__ __forceinline__ void simt_clear(float* dst, int first) {
  constexpr int VEC = 16 / (int)sizeof(T);
  for (int c = threadIdx.x; c < first * (D / VEC); c += THREADS) {
    const int r = c / (D / VEC), x = c % (D / VEC) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; e += 4)
      *reinterpret_cast<float4*>(dst + r * (D + 4) + x + e) = make_float4(0.f, 0.f, 0.f, 0.f);
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

template <int D, int OWN>
constexpr size_t simt_fwd_smem() {
  return ((OWN + kSimtKeys) * (D + 4) + OWN * (kSimtKeys + 4)) * sizeof(float);
}

// One tile of keys for the own rows in qs: scores, running maximum m (natural
// logarithm's units) and sum l, and acc += p V. `sees(i, j)`: whether own row i
// sees key j of the tile; no query sees the first `front` (if positive).
template <typename T, int D, int THREADS, typename Sees>
__device__ __forceinline__ void simt_fwd_tile(const AttnArgs& a, const float* qs, float* ks,
                                              float* ps, int b, int h, int r0, int nk, int front,
                                              int ty, int tx, float (&acc)[4][D / 16],
                                              float (&m)[4], float (&l)[4], Sees sees) {
  constexpr int N = kSimtKeys, LP = N + 4;
  __syncthreads();
  simt_load<T, D, THREADS>(ks, N, a.k, b, h, r0, nk);
  __syncthreads();
  float x[4][4];
  simt_dot<D, 4>(qs, ks, ty, tx, x);
  __syncthreads();
  simt_load<T, D, THREADS>(ks, N, a.v, b, h, r0, nk);
  if (front > 0) simt_clear<T, D, THREADS>(ks, front);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[i][j] = sees(4 * ty + i, tx + 16 * j) ? x[i][j] * a.scale : -INFINITY;
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

template <typename T, int D, int OWN>
__global__ void __launch_bounds__(4 * OWN) attn_simt_fwd_kernel(const AttnArgs a) {
  constexpr int N = OWN, LD = D + 4, THREADS = 4 * OWN;
  extern __shared__ __align__(16) float sm[];
  float* qs = sm;
  float* ks = qs + N * LD;  // a tile of K, then the same rows of V
  float* ps = ks + kSimtKeys * LD;
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
  const int seen0 = first_key(a, s);
  simt_load<T, D, THREADS>(qs, N, a.q, s.b, h, s.q0 + m0, rows);
  float acc[4][D / 16], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) acc[i][c] = 0.f;
  }
  for (int n0 = lo / kSimtKeys * kSimtKeys; n0 < hi; n0 += kSimtKeys)
    simt_fwd_tile<T, D, THREADS>(
        a, qs, ks, ps, s.b, h / a.G, s.k0 + n0, min(kSimtKeys, s.klen - n0), seen0 - n0, ty,
        tx, acc, m, l,
        [&](int i, int j) { return see_keys(a, s, m0 + i, n0 + j); });
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = l[i] > 0.f || l[i] != l[i] ? 1.f / l[i] : 0.f;
  const int out_rows = min(N, limit - m0);
  simt_store<T, D>(a.o, s.b, h, s.q0 + m0, out_rows, ty, tx, acc, f);
  if (tx == 0 && a.lse != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * ty + i < out_rows)
        a.lse[((int64_t)s.b * a.Hq + h) * a.Sq + s.q0 + m0 + 4 * ty + i] =
            l[i] == 0.f ? -INFINITY : m[i] + logf(l[i]);
  }
}

// Few query rows over many keys: the group's rows (row r = query r / G of head
// h*G + r % G, at most 16) are one own tile, so K and V are read once for the
// group, and the keys are split over CTAs in chunks (as in attn_rows.cuh, whose
// join adds the chunks up). Bound: HBM, K and V once, and close to it the FMA
// of 16 rows.
constexpr int kSimtRows = 16;

template <typename T, int D>
__global__ void __launch_bounds__(4 * kSimtRows)
    attn_simt_rows_kernel(const AttnArgs a, const RowsPlan pl) {
  constexpr int N = kSimtRows, LD = D + 4, THREADS = 4 * N;
  extern __shared__ __align__(16) float sm[];
  allow_dependent_launch();
  float* qs = sm;
  float* ks = qs + N * LD;
  float* ps = ks + kSimtKeys * LD;
  const int bh = blockIdx.x % (a.B * a.Hk), split = blockIdx.x / (a.B * a.Hk);
  const int b = bh / a.Hk, h = bh % a.Hk;
  const AttnSeq s = find_seq<true>(a, b, 0, 1);
  const int rows = a.Sq * a.G;
  int lo, hi;
  key_range(a, s, 0, s.qlen, lo, hi);
  const int seen0 = lo;  // the first key that a query sees
  lo = max(lo, split * pl.chunk) / kSimtKeys * kSimtKeys;
  hi = min(hi, (split + 1) * pl.chunk);
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  for (int r = 0; r < N; ++r) {
    const bool in = r < rows;
    simt_load<T, D, THREADS>(qs + r * LD, 1, a.q, b, h * a.G + (in ? r % a.G : 0),
                             in ? r / a.G : 0, in ? 1 : 0);
  }
  float acc[4][D / 16], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) acc[i][c] = 0.f;
  }
  for (int n0 = lo; n0 < hi; n0 += kSimtKeys)
    simt_fwd_tile<T, D, THREADS>(
        a, qs, ks, ps, b, h, n0, min(kSimtKeys, s.klen - n0), seen0 - n0, ty, tx, acc, m, l,
        [&](int i, int j) { return i < rows && see_keys(a, s, i / a.G, n0 + j); });
  const int64_t part = ((int64_t)split * a.B * a.Hk + bh) * N;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i;
    if (r >= rows) continue;
    const float m2 = m[i] * kLog2e;  // the join's units
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
#pragma unroll
    for (int c = 0; c < D / 16; c += 2) {
      const int col = 64 * (c / 4) + 4 * tx + c % 4;
      if (pl.splits == 1) rows_out<T>(a, b, h, r, col, acc[i][c] * inv, acc[i][c + 1] * inv);
      else
        *reinterpret_cast<float2*>(pl.sums + (part + r) * D + col) = f2(acc[i][c], acc[i][c + 1]);
    }
    if (tx == 0) {
      if (pl.splits == 1) {
        rows_lse(a, b, h, r, m2, l[i]);
      } else {
        pl.stat[(part + r) * 2] = m2;
        pl.stat[(part + r) * 2 + 1] = l[i];
      }
    }
  }
}

// Rows of a streamed tile of the backward: two own tiles, two streamed ones
// and the two weight tiles have to fit in shared memory.
template <int D> constexpr int kSimtStr = D == 256 ? 32 : 64;

template <int D, int OWN>
constexpr size_t simt_bwd_smem() {
  return (2 * (OWN + kSimtStr<D>) * (D + 4) + 2 * OWN * (kSimtStr<D> + 4)) * sizeof(float);
}

// DKV: own rows are keys (K, V), the queries of every head of the group (Q,
// dO) stream past, dk and dv are written; SPLIT: of one head, whose sums go to
// head h of dk and dv (the partial sums). Else own rows are queries, the keys
// stream, dq is written.
template <typename T, int D, int OWN, bool DKV, bool SPLIT>
__global__ void __launch_bounds__(4 * OWN) attn_simt_bwd_kernel(const AttnArgs a) {
  constexpr int N = OWN, M = kSimtStr<D>, NJ = M / 16, LD = D + 4, LP = M + 4;
  constexpr int THREADS = 4 * OWN;
  extern __shared__ __align__(16) float sm[];
  float* own1 = sm;  // K or Q
  float* own2 = own1 + N * LD;  // V or dO
  float* str1 = own2 + N * LD;  // Q or K
  float* str2 = str1 + M * LD;  // dO or V
  float* ps = str2 + M * LD;
  float* ds = ps + N * LP;
  const int H = DKV && !SPLIT ? a.Hk : a.Hq;
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
  const int ho = SPLIT ? h / a.G : h;  // head of the own rows
  simt_load<T, D, THREADS>(own1, N, DKV ? a.k : a.q, s.b, ho, own0, rows);
  simt_load<T, D, THREADS>(own2, N, DKV ? a.v : a.dout, s.b, ho, own0, rows);
  float acc1[4][D / 16], acc2[DKV ? 4 : 1][D / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      acc1[i][c] = 0.f;
      if (DKV) acc2[i][c] = 0.f;
    }
  const int seen0 = DKV ? first_query(a, s) : first_key(a, s);
  const int h1 = !DKV ? h / a.G : SPLIT ? h : h * a.G;
  for (int g = 0; g < (DKV && !SPLIT ? a.G : 1); ++g) {
    const int64_t stat = (int64_t)(DKV ? h1 + g : h) * a.R + s.stat0;
    for (int t0 = lo / M * M; t0 < hi; t0 += M) {
      const int nt = min(M, (DKV ? s.qlen : s.klen) - t0);
      __syncthreads();
      simt_load<T, D, THREADS>(str1, M, DKV ? a.q : a.k, s.b, h1 + g, strb + t0, nt);
      simt_load<T, D, THREADS>(str2, M, DKV ? a.dout : a.v, s.b, h1 + g, strb + t0, nt);
      if (t0 < seen0) {
        simt_clear<T, D, THREADS>(str1, seen0 - t0);
        simt_clear<T, D, THREADS>(str2, seen0 - t0);
      }
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
            if (!sees_one(a, s, qi)) d = p * (y[i][j] - __ldg(a.delta + stat + qi));
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

// The group's partial sums of dk and dv [B, Hq, Sk, D], added in head order.
template <int D>
__global__ void __launch_bounds__(256) simt_sum_kernel(const float* pk, const float* pv, HT dk,
                                                       HT dv, int B, int Sk, int Hk, int G) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // 4 elements each
  const int c = (int)(i % (D / 4)) * 4;
  const int64_t row = i / (D / 4);  // (b * Hk + h) * Sk + key
  if (row >= (int64_t)B * Hk * Sk) return;
  const int key = (int)(row % Sk), h = (int)(row / Sk % Hk), b = (int)(row / Sk / Hk);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
  for (int g = 0; g < G; ++g) {
    const int64_t at = ((((int64_t)b * Hk + h) * G + g) * Sk + key) * D + c;
    const float4 u = *reinterpret_cast<const float4*>(pk + at);
    const float4 w = *reinterpret_cast<const float4*>(pv + at);
    x = make_float4(x.x + u.x, x.y + u.y, x.z + u.z, x.w + u.w);
    y = make_float4(y.x + w.x, y.y + w.y, y.z + w.z, y.w + w.w);
  }
  auto put = [&](const HT& t, float4 v) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(const_cast<void*>(t.p)) +
                               (int64_t)b * t.sb + (int64_t)key * t.ss + (int64_t)h * t.sh + c) = v;
  };
  put(dk, x);
  put(dv, y);
}

// Own rows of a tile: 64 where `tiles64` CTAs of 64 give every SM one.
inline int simt_own(int64_t tiles64) { return tiles64 >= device_sm_count() ? 64 : 32; }

template <typename F>
int simt_own_tile(int own, F&& f) {
  return own == 64 ? f(std::integral_constant<int, 64>{}) : f(std::integral_constant<int, 32>{});
}

template <typename T, int D>
int simt_rows(const AttnArgs& a, void* ws, cudaStream_t st) {
  auto kern = attn_simt_rows_kernel<T, D>;
  constexpr size_t smem = simt_fwd_smem<D, kSimtRows>();
  const RowsPlan pl = rows_plan(a, kSimtRows, D, ws);
  int rc = prepare_smem((const void*)kern, smem);
  if (rc != BLOTH_OK) return rc;
  const int64_t grid = (int64_t)pl.splits * a.B * a.Hk;
  if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
  rc = launched(launch_ex(kern, (unsigned)grid, 4 * kSimtRows, smem, st, a, pl));
  if (rc != BLOTH_OK || pl.splits == 1) return rc;
  return launch_attn_join<T, D>(a, pl, kSimtRows, st);
}

template <typename T>
int attn_simt_fwd(const AttnArgs& a, int D, void* ws, cudaStream_t st) {
  return attn_head_dim(D, [&](auto dd) {
    constexpr int DD = decltype(dd)::value;
    if (attn_simt_rows_take(a.Sq, a.G, a.packed) && a.Sk > 0) return simt_rows<T, DD>(a, ws, st);
    const int64_t heads = (int64_t)a.Hq * a.B;
    return simt_own_tile(simt_own(attn_tiles(a.Sq, a.packed, 64) * heads), [&](auto oo) {
      constexpr int OWN = decltype(oo)::value;
      auto kern = attn_simt_fwd_kernel<T, DD, OWN>;
      constexpr size_t smem = simt_fwd_smem<DD, OWN>();
      const int rc = prepare_smem((const void*)kern, smem);
      if (rc != BLOTH_OK) return rc;
      const int64_t grid = attn_tiles(a.Sq, a.packed, OWN) * heads;
      if (grid == 0) return BLOTH_OK;
      if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
      return launched(launch_ex(kern, (unsigned)grid, 4 * OWN, smem, st, a));
    });
  });
}

template <typename T>
int attn_simt_bwd(const AttnArgs& a0, int D, void* partial, cudaStream_t st) {
  return attn_head_dim(D, [&](auto dd) {
    constexpr int DD = decltype(dd)::value;
    AttnArgs a = a0;
    auto run = [&](auto dkv, auto split, int64_t heads, int64_t S) {
      constexpr bool DKV = decltype(dkv)::value, SPLIT = decltype(split)::value;
      return simt_own_tile(simt_own(attn_tiles(S, a.packed, 64) * heads), [&](auto oo) {
        constexpr int OWN = decltype(oo)::value;
        auto kern = attn_simt_bwd_kernel<T, DD, OWN, DKV, SPLIT>;
        constexpr size_t smem = simt_bwd_smem<DD, OWN>();
        const int rc = prepare_smem((const void*)kern, smem);
        if (rc != BLOTH_OK) return rc;
        const int64_t grid = attn_tiles(S, a.packed, OWN) * heads;
        if (grid == 0) return BLOTH_OK;
        if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
        return launched(launch_ex(kern, (unsigned)grid, 4 * OWN, smem, st, a));
      });
    };
    using Yes = std::true_type;
    using No = std::false_type;
    int rc = BLOTH_OK;
    if (a.dk.p != nullptr) {
      if (simt_split(a.B, a.Sk, a.Hk, a.G, a.packed)) {
        // partial sums [B, Hq, Sk, D] of dk, then of dv
        const int64_t n = (int64_t)a.B * a.Hq * a.Sk * DD;
        float* pk = reinterpret_cast<float*>(partial);
        a.dk = HT{pk, (int64_t)a.Hq * a.Sk * DD, DD, (int64_t)a.Sk * DD};
        a.dv = a.dk;
        a.dv.p = pk + n;
        rc = run(Yes{}, Yes{}, (int64_t)a.Hq * a.B, a.Sk);
        const int64_t four = (int64_t)a.B * a.Hk * a.Sk * (DD / 4);
        if (rc == BLOTH_OK)
          rc = launched(launch_ex(simt_sum_kernel<DD>, (unsigned)((four + 255) / 256), 256u, 0, st,
                                  pk, pk + n, a0.dk, a0.dv, a.B, a.Sk, a.Hk, a.G));
      } else {
        rc = run(Yes{}, No{}, (int64_t)a.Hk * a.B, a.Sk);
      }
    }
    if (rc == BLOTH_OK && a.dq.p != nullptr)
      rc = run(No{}, No{}, (int64_t)a.Hq * a.B, a.Sq);
    return rc;
  });
}

}  // namespace bloth
