// qvx_pages.hpp -- the calls that move the pages of a cache between sequences (qvx_pages.hip) as the host checked them.
#pragma once

#include "qvx_common.hpp"

#include "../../include/qvx.h"

#include <algorithm>

namespace qvx {

enum { kForkRows = 1, kForkTotals = 2 };

struct ForkCall {
  const int32_t *from, *to;
  int n;
  int32_t* table;
  int n_rows, table_width, page_size;
  int32_t *lens, *extra;
  int n_pages;
  const int32_t* free_list;
  int n_free;
  const int32_t* taken_in;
  int32_t *taken_out, *pairs, *n_pairs;
};

struct FreeCall {
  const int32_t *rows, *begin, *end;
  int n;
  int32_t* table;
  int n_rows, table_width;
  int32_t *lens, *extra;
  int n_pages;
  int32_t* free_list;
  int n_free;
  const int32_t* taken_in;
  int32_t *taken_out, *counts;
};

struct CompactCall {
  const int32_t* table;
  int32_t* table_out;
  int64_t entries;
  const int32_t* extra;
  int32_t* extra_out;
  int n_pages;
  const int32_t* free_list;
  int32_t* free_out;
  int n_free;
  const int32_t* taken;
  int32_t *pairs, *moved;
};

constexpr int kCopyCaches = 64;  // of a launch
struct CopyCall {
  const int32_t *pairs, *count;
  int most, n_pages, n_caches;
  int64_t page_bytes;
  struct {
    uint8_t *k, *v;
    int64_t stride;
  } cache[kCopyCaches];
};

constexpr int kFreePages = 8192;  // pages of a workgroup of the release's count
constexpr int kCompactPages = 1 << 20;

}  // namespace qvx
