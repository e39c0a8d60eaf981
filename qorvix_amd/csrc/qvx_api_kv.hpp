// qvx_api_kv.hpp -- argument checks that the calls of the paged cache share (include/qvx.h), and how a launch's
// outcome becomes a status.
#pragma once

#include "qvx_common.hpp"

#include "../../include/qvx.h"

#include <cstdio>

namespace qvx {

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline int attn_status(bool launched) {
  const hipError_t e = hipGetLastError();
  if (launched && e == hipSuccess) return QVX_OK;
  std::fprintf(stderr, "qvx: HIP error %d (%s)\n", (int)e, hipGetErrorString(e));
  return QVX_E_HIP;
}

// Bytes of n values of a cache or states type; 0 for another type.
inline int64_t value_bytes(uint32_t type, int64_t n) {
  switch (type) {
    case T_F32: return 4 * n;
    case T_F16: case T_BF16: return 2 * n;
    case T_Q8_0: return n + n / 16;
    default: return 0;
  }
}

inline bool head_dim_ok(uint32_t type, int d) { return d > 0 && d <= 256 && d % (type == T_Q8_0 ? 32 : 8) == 0; }

inline int64_t page_bytes(uint32_t type, int kv_heads, int page_size, int head_dim) {
  if (!value_bytes(type, 1) || kv_heads <= 0 || page_size <= 0 || !head_dim_ok(type, head_dim)) return 0;
  const int64_t rows = (int64_t)kv_heads * page_size;
  if (rows > (1ll << 40)) return 0;
  return (value_bytes(type, rows * head_dim) + 15) / 16 * 16;
}

inline int check_cache(const qvx_kv_cache* c, int64_t* stride) {
  if (!c) return QVX_E_NULL;
  if (!value_bytes(c->type, 1)) return QVX_E_TYPE;
  const int64_t packed = page_bytes(c->type, c->kv_heads, c->page_size, c->head_dim);
  if (!packed || c->n_pages <= 0) return QVX_E_SHAPE;
  if ((int64_t)c->n_pages * c->page_size > 0x7fffffffll) return QVX_E_RANGE;
  if (c->page_stride && (c->page_stride < packed || c->page_stride % 16)) return QVX_E_RANGE;
  if (!c->d_k || !c->d_v) return QVX_E_NULL;
  if (!aligned(c->d_k, 16) || !aligned(c->d_v, 16)) return QVX_E_RANGE;
  *stride = c->page_stride ? c->page_stride : packed;
  return QVX_OK;
}

}  // namespace qvx
