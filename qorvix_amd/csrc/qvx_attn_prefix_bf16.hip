// qvx_attn_prefix_bf16.hip -- the split attention kernel over BF16 keys and values (qvx_attn_split.hpp):
// a prefix that sequences share.
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_prefix_bf16(const AttnCall& c, dim3 grid, hipStream_t s) {
  return attn_split_dt<T_BF16, kMaskPrefix>(c, grid, s);
}

}  // namespace qvx
