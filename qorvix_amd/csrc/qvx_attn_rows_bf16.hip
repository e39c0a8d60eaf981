// qvx_attn_rows_bf16.hip -- the kernel of many query rows over BF16 pages (qvx_attn_rows.hpp).
#include "qvx_attn_rows.hpp"

namespace qvx {

bool launch_attn_rows_bf16(const AttnCall& c, bool parts, dim3 grid, hipStream_t s) {
  return rows::launch_mode<T_BF16>(c, parts, grid, s);
}

}  // namespace qvx
