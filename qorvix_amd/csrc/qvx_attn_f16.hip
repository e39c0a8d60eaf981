// qvx_attn_f16.hip -- the split attention kernel over F16 keys and values (qvx_attn_split.hpp).
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_split_f16(const AttnCall& c, dim3 grid, hipStream_t s) {
  return attn_split_dt<T_F16>(c, grid, s);
}

}  // namespace qvx
