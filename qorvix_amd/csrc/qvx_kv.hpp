// qvx_kv.hpp -- the calls of the paged cache's upkeep (qvx_kv.hip) as the host checked them.
#pragma once

#include "qvx_common.hpp"

#include "../../include/qvx.h"

#include <algorithm>

namespace qvx {

enum { kMapTokens = 1, kMapSeqs = 2 };
constexpr int kRopeMaxPairs = 128, kRopeMaxTokens = 8;  // of a workgroup's table of cosines and sines

struct MapCall {
  const int32_t *held, *added;
  int n_seqs;
  int32_t* table;
  int table_width, page_size;
  const int32_t* free_list;
  int n_free;
  const int32_t* taken_in;
  int32_t *taken_out, *lens, *offsets, *slots, *pos, *seq;
  int max_tokens;
};

struct RopeCall {
  float* q_out;
  const float *q, *k, *v;
  int64_t q_out_stride, q_stride, k_stride, v_stride;
  int q_heads, kv_heads, head_dim, n_tokens;
  const double* inv_freq;
  const uint8_t* axis;
  int rot_dim, n_axes, halves;
  float scale;
  const int32_t* pos;
  int64_t pos_stride;
  const int32_t* slots;  // null: no cache, every row counts
  uint8_t *k_pages, *v_pages;
  int64_t page_stride, scale_off;
  int page_size;
  int64_t n_slots;
  int tokens_wg, rows_wg;
};

// With norms: the weights of a head are w_stride values from the last one's (0: all heads' alike), null: no norm.
struct NormRopeCall : RopeCall {
  void* q_typed;  // in place of q_out
  const float *q_w, *k_w;
  int w_stride, lanes_log;
  float eps;
  double inv_dim;
};

}  // namespace qvx
