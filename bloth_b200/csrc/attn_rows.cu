// Few-row attention forward, instantiated.
#include "attn_rows.cuh"

namespace bloth {

// Whether the few-row kernel takes a call: up to 32 rows per key head (16 at
// head_dim 256, where two row tiles do not fit in registers). Heads of 128,
// 32/8, bf16, few-row kernel against the tile kernel: 16 caches of 8192, 4 rows
// 104 and 351 us, 32 rows 158 and 352; one cache of 1024, 9.6 and 16.6, and 15.0
// and 16.5.
bool attn_rows_take(int64_t Sq, int64_t G, int64_t D, int64_t packed) {
  return packed == 0 && Sq * G <= (D == 256 ? 16 : 32);
}

size_t attn_rows_workspace(int64_t B, int64_t Sk, int64_t Hk, int64_t D, int rows) {
  int64_t chunk, splits;
  if (B * Hk == 0) return 0;
  rows_split(B * Hk, Sk, chunk, splits);
  if (splits == 1) return 0;
  return (size_t)(splits * B * Hk * rows * (D + 2)) * sizeof(float);
}

template <typename T>
int attn_rows_fwd(const AttnArgs& a, int D, void* ws, cudaStream_t st) {
  const bool one = a.Sq * a.G <= 16;
  if (D == 64)
    return one ? launch_attn_rows<T, 64, 1>(a, ws, st) : launch_attn_rows<T, 64, 2>(a, ws, st);
  if (D == 128)
    return one ? launch_attn_rows<T, 128, 1>(a, ws, st) : launch_attn_rows<T, 128, 2>(a, ws, st);
  return launch_attn_rows<T, 256, 1>(a, ws, st);
}
template int attn_rows_fwd<__nv_bfloat16>(const AttnArgs&, int, void*, cudaStream_t);
template int attn_rows_fwd<__half>(const AttnArgs&, int, void*, cudaStream_t);

}  // namespace bloth
