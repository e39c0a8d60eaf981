// qvx_attn_window_bf16.hip -- the split attention kernel over BF16 keys and values (qvx_attn_split.hpp):
// rows that see a window and first tokens.
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_window_bf16(const AttnCall& c, dim3 grid, hipStream_t s) {
  return attn_split_dt<T_BF16, kMaskWindow>(c, grid, s);
}

}  // namespace qvx
