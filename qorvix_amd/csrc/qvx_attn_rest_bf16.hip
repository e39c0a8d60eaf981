// qvx_attn_rest_bf16.hip -- the split attention kernel over BF16 keys and values (qvx_attn_split.hpp):
// what is behind a shared prefix.
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_rest_bf16(const AttnCall& c, dim3 grid, hipStream_t s) {
  return attn_split_dt<T_BF16, kMaskRest>(c, grid, s);
}

}  // namespace qvx
