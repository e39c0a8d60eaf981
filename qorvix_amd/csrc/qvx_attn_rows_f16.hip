// qvx_attn_rows_f16.hip -- the kernel of many query rows over F16 pages (qvx_attn_rows.hpp).
#include "qvx_attn_rows.hpp"

namespace qvx {

bool launch_attn_rows_f16(const AttnCall& c, bool parts, dim3 grid, hipStream_t s) {
  return rows::launch_mode<T_F16>(c, parts, grid, s);
}

}  // namespace qvx
