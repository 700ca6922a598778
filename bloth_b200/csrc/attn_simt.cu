// fp32 attention, instantiated.
#include "attn_simt.cuh"

namespace bloth {

// Few-row kernel against the tile kernel: 16 rows per key head of 128, one cache
// of 1024, 50 and 119 us; 8 caches of 4096, 96 and 671 us (16/4 heads).
bool attn_simt_rows_take(int64_t Sq, int64_t G, int64_t packed) {
  return packed == 0 && Sq * G <= kSimtRows;
}

// One CTA per key tile and query head where those per key head would be fewer
// than two for an SM.
bool simt_split(int64_t B, int64_t Sk, int64_t Hk, int64_t G, int64_t packed) {
  return G > 1 && attn_tiles(Sk, packed, 64) * Hk * B < 2 * (int64_t)device_sm_count();
}

template int attn_simt_fwd<float>(const AttnArgs&, int, void*, cudaStream_t);
template int attn_simt_bwd<float>(const AttnArgs&, int, void*, cudaStream_t);

}  // namespace bloth
