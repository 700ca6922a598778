// Tensor-core attention backward, instantiated.
#include "attn_bwd.cuh"

namespace bloth {

template <typename T>
int attn_tc_bwd(const AttnArgs& a, int D, cudaStream_t st) {
  return D == 64    ? launch_attn_bwd<T, 64>(a, st)
         : D == 128 ? launch_attn_bwd<T, 128>(a, st)
                    : launch_attn_bwd<T, 256>(a, st);
}
template int attn_tc_bwd<__nv_bfloat16>(const AttnArgs&, int, cudaStream_t);
template int attn_tc_bwd<__half>(const AttnArgs&, int, cudaStream_t);

}  // namespace bloth
