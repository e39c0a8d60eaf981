// qvx_attn_whole_bf16.hip -- the split attention kernel over BF16 keys and values (qvx_attn_split.hpp):
// sequences behind a shared prefix that read it each for itself.
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_whole_bf16(const AttnCall& c, dim3 grid, hipStream_t s) {
  return attn_split_dt<T_BF16, kMaskWhole>(c, grid, s);
}

}  // namespace qvx
