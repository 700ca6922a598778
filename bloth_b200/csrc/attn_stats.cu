// Row statistics of the attention backward, every element type.
#include "attn_impl.cuh"

namespace bloth {

// Sum of squares over this lane's part of a row of D elements.
template <typename T, int D>
__device__ __forceinline__ float row_square(const T* p) {
  constexpr int VEC = 16 / (int)sizeof(T), LPR = D / VEC < 32 ? D / VEC : 32;
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < D / (VEC * LPR); ++u) {
    float g[VEC];
    unpack(ldg_pack<T, VEC>(p + (u * LPR + (threadIdx.x & 31) % LPR) * VEC), g);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum = fmaf(g[e], g[e], sum);
  }
  return sum;
}

// The largest of the CTA's 8 warps' numbers, x and y.
__device__ __forceinline__ float2 cta_top(float2 v, float2 (&sm)[8]) {
  v = f2(warp_top(v.x), warp_top(v.y));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[threadIdx.x & 7];
  return f2(warp_top(v.x), warp_top(v.y));
}
__device__ __forceinline__ float if_finite(float x) { return isfinite(x) ? x : 0.f; }

// Largest norm of V's rows in tile s.tile of keys of head h.
template <typename T, int D>
__device__ __forceinline__ void key_top(const AttnArgs& a, const AttnSeq& s, int h,
                                        float2 (&sm)[8]) {
  constexpr int VEC = 16 / (int)sizeof(T), LPR = D / VEC < 32 ? D / VEC : 32;
  const T* vp = reinterpret_cast<const T*>(a.v.p) + (int64_t)s.b * a.v.sb + (int64_t)h * a.v.sh +
                (int64_t)s.k0 * a.v.ss;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = 0.f;
#pragma unroll
  for (int r = warp * 16 + lane / LPR; r < warp * 16 + 16; r += 32 / LPR) {
    const int j = s.tile * 128 + r;
    const bool in = j < s.klen && j >= first_key(a, s);
    const float n = group_lane_sum<LPR>(in ? row_square<T, D>(vp + (int64_t)j * a.v.ss) : 0.f);
    top = fmaxf(top, if_finite(n));
  }
  top = cta_top(f2(top, 0.f), sm).x;
  if (threadIdx.x == 0)
    a.vtop[(int64_t)h * stat_tiles(a.RK) + s.kstat0 / 128 + s.tile] = sqrtf(top);
}

// delta = rowsum(dO * O) and lse in base 2 for the backward kernels, for every
// row of every 128-row tile of a sequence: a row past the sequence's end, or
// one that sees nothing, gets lse2 = +inf and delta = 0, so its recomputed
// probabilities are exp2(x - inf) = 0. HBM-bound: reads O, its rest and dO
// once. A row takes D / 8 lanes of 16-bit (D / 4 of fp32) elements, one 16-byte
// load of each tensor per lane and pass. 8192 rows of 32 heads of 128 (bf16),
// 201 MB: 45 us, 4.5 TB/s. A CTA has 128 rows, so that it needs one search for
// its sequence.
//
// fp16: also what bounds ds, |ds_ij| <= |do_i| |v_j| + |delta_i| (Cauchy-Schwarz, p
// is at most 1): the norms of the rows of dO, their largest and that of delta for
// every tile, and, by CTAs of their own (the first `key_ctas`; of packed sequences
// one for all heads, which then search the offsets once), the largest norm of V's
// rows for every tile of keys. Rows that are not finite do not count: what they
// reach is not finite whatever its scale, and other rows keep theirs.
template <typename T, int D>
__global__ void __launch_bounds__(256, 6) attn_stats_kernel(const AttnArgs a, int key_ctas) {
  constexpr int VEC = 16 / (int)sizeof(T), LPR = D / VEC < 32 ? D / VEC : 32;
  constexpr int PASS = D / (VEC * LPR), RPW = 32 / LPR;
  constexpr bool BOUND = std::is_same<T, __half>::value;
  __shared__ float2 sm[8];
  int x = (int)blockIdx.x;
  if constexpr (BOUND) {
    if (x < key_ctas) {
      const int heads = a.packed ? 1 : a.Hk, hb = x % (heads * a.B);
      const AttnSeq s = find_seq<false>(a, hb / heads, x / (heads * a.B), 128);
      if (s.tile < 0) return;
      if (!a.packed) key_top<T, D>(a, s, hb % heads, sm);
      else
        for (int h = 0; h < a.Hk; ++h) key_top<T, D>(a, s, h, sm);
      return;
    }
    x -= key_ctas;
  }
  const int heads = a.Hq * a.B;
  const int hb = x % heads, h = hb % a.Hq;
  const AttnSeq s = find_seq<true>(a, hb / a.Hq, x / heads, 128);
  if (s.tile < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int m0 = s.tile * 128;
  float do_top = 0.f, delta_top = 0.f;
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
    float sum = 0.f, square = 0.f;
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
          for (int i = 0; i < VEC; ++i) f[i] = fmaf(e[i], 1.f / kRestUp<T>, f[i]);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          sum = fmaf(f[e], g[e], sum);
          if (BOUND) square = fmaf(g[e], g[e], square);
        }
      }
    }
    sum = group_lane_sum<LPR>(sum);
    if constexpr (BOUND) square = group_lane_sum<LPR>(square);
    if (lane % LPR == 0) {
      const float l = in ? a.lse[((int64_t)s.b * a.Hq + h) * a.Sq + row] : -INFINITY;
      const bool none = l == -INFINITY;
      a.lse2[stat + r] = none ? INFINITY : l * kLog2e - kBwdShift<T>;
      a.delta[stat + r] = none ? 0.f : sum;
      if constexpr (BOUND) {
        const float n = none ? 0.f : if_finite(sqrtf(square));
        a.donorm[stat + r] = n;
        do_top = fmaxf(do_top, n);
        delta_top = fmaxf(delta_top, none ? 0.f : if_finite(fabsf(sum)));
      }
    }
  }
  if constexpr (BOUND) {
    const float2 top = cta_top(f2(do_top, delta_top), sm);
    if (threadIdx.x == 0) a.qtop[(int64_t)h * stat_tiles(a.R) + s.stat0 / 128 + s.tile] = top;
  }
}

template <typename T>
int attn_stats(const AttnArgs& a, int D, cudaStream_t st) {
  return attn_head_dim(D, [&](auto dd) {
    constexpr int DD = decltype(dd)::value;
    const int64_t q_ctas = attn_tiles(a.Sq, a.packed, 128) * a.Hq * a.B;
    if (q_ctas == 0) return BLOTH_OK;
    const int64_t key_ctas = a.vtop == nullptr ? 0
                                               : attn_tiles(a.Sk, a.packed, 128) * a.B *
                                                     (a.packed ? 1 : a.Hk);
    if (q_ctas + key_ctas > 0x7fffffff) return BLOTH_ERR_SHAPE;
    return launched(launch_ex(attn_stats_kernel<T, DD>, (unsigned)(q_ctas + key_ctas), 256u, 0, st,
                              a, (int)key_ctas));
  });
}
template int attn_stats<float>(const AttnArgs&, int, cudaStream_t);
template int attn_stats<__nv_bfloat16>(const AttnArgs&, int, cudaStream_t);
template int attn_stats<__half>(const AttnArgs&, int, cudaStream_t);

}  // namespace bloth
