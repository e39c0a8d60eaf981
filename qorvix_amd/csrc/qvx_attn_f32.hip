// qvx_attn_f32.hip -- the split attention kernel over F32 keys and values (qvx_attn_split.hpp).
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_split_f32(const AttnCall& c, dim3 grid, hipStream_t s) {
  return attn_split_dt<T_F32>(c, grid, s);
}

}  // namespace qvx
