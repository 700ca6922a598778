// Row statistics of the attention backward, every element type.
#include "attn_impl.cuh"

namespace bloth {

// delta = rowsum(dO * O) and lse in base 2 for the backward kernels, for every
// row of every 128-row tile of a sequence: a row past the sequence's end, or
// one that sees nothing, gets lse2 = +inf and delta = 0, so its recomputed
// probabilities are exp2(x - inf) = 0. HBM-bound: reads O, its rest and dO
// once. A row takes D / 8 lanes of 16-bit (D / 4 of fp32) elements, one 16-byte
// load of each tensor per lane and pass. 8192 rows of 32 heads of 128 (bf16),
// 201 MB: 45 us, 4.5 TB/s. A CTA has 128 rows, so that it needs one search for
// its sequence.
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
      a.lse2[stat + r] = none ? INFINITY : l * kLog2e - kBwdShift<T>;
      a.delta[stat + r] = none ? 0.f : sum;
    }
  }
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
template int attn_stats<float>(const AttnArgs&, int, cudaStream_t);
template int attn_stats<__nv_bfloat16>(const AttnArgs&, int, cudaStream_t);
template int attn_stats<__half>(const AttnArgs&, int, cudaStream_t);

}  // namespace bloth
