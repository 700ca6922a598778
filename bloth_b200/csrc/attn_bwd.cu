// Tensor-core attention backward, instantiated.
#include "attn_bwd.cuh"

namespace bloth {

template <typename T>
int attn_tc_bwd(const AttnArgs& a, int D, cudaStream_t st) {
  return attn_head_dim(D, [&](auto dd) {
    constexpr int DD = decltype(dd)::value;
    return launch_attn_bwd<T, DD>(a, st);
  });
}
template int attn_tc_bwd<__nv_bfloat16>(const AttnArgs&, int, cudaStream_t);
template int attn_tc_bwd<__half>(const AttnArgs&, int, cudaStream_t);

}  // namespace bloth
