// Tensor-core attention forward, instantiated.
#include "attn_fwd.cuh"

namespace bloth {

template <typename T>
int attn_tc_fwd(const AttnArgs& a, int D, cudaStream_t st) {
  return D == 64    ? launch_attn_fwd<T, 64>(a, st)
         : D == 128 ? launch_attn_fwd<T, 128>(a, st)
                    : launch_attn_fwd<T, 256>(a, st);
}
template int attn_tc_fwd<__nv_bfloat16>(const AttnArgs&, int, cudaStream_t);
template int attn_tc_fwd<__half>(const AttnArgs&, int, cudaStream_t);

}  // namespace bloth
