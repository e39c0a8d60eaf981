// qvx_attn_prefix_q8.hip -- the split attention kernel over Q8_0 keys and values (qvx_attn_split.hpp):
// a prefix that sequences share.
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_prefix_q8(const AttnCall& c, dim3 grid, hipStream_t s) {
  return attn_split_dt<T_Q8_0, kMaskPrefix>(c, grid, s);
}

}  // namespace qvx
