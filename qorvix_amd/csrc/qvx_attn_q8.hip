// qvx_attn_q8.hip -- the split attention kernel over Q8_0 keys and values (qvx_attn_split.hpp).
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_split_q8(const AttnCall& c, dim3 grid, hipStream_t s) {
  return attn_split_dt<T_Q8_0>(c, grid, s);
}

}  // namespace qvx
