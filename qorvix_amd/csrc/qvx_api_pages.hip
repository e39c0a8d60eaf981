// qvx_api_pages.hip -- the extern "C" boundary of the calls that move a cache's pages between sequences (include/qvx.h):
// argument checks, which run before any device work.
#include "qvx_api_kv.hpp"
#include "qvx_pages.hpp"

namespace qvx {
void launch_kv_fork(const ForkCall& c, bool alias, hipStream_t s);
void launch_kv_free(const FreeCall& c, hipStream_t s);
bool launch_kv_compact(const CompactCall& c, bool in_place, hipStream_t s);
void launch_kv_copy(const CopyCall& c, hipStream_t s);
}  // namespace qvx

using namespace qvx;

namespace {

constexpr int kMostForks = 16384, kMostColumns = 1 << 24;

struct Span {
  const void* p;
  int64_t bytes;
};
bool overlap(const Span& a, const Span& b) {
  const auto x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return a.p && b.p && a.bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}
template <size_t N, size_t M> bool any_overlap(const Span (&a)[N], const Span (&b)[M]) {
  for (const Span& x : a)
    for (const Span& y : b)
      if (overlap(x, y)) return true;
  return false;
}

int check_table(int n_rows, int table_width, int n_pages, int n_free) {
  if (n_rows <= 0 || table_width <= 0 || n_pages <= 0 || n_free < 0) return QVX_E_SHAPE;
  if (table_width > kMostColumns) return QVX_E_RANGE;
  return QVX_OK;
}

}  // namespace

#pragma GCC visibility push(default)
extern "C" {

int qvx_kv_fork(const int32_t* d_from, const int32_t* d_to, int n, int32_t* d_table, int n_rows, int table_width,
                int page_size, int32_t* d_lens, int32_t* d_extra, int n_pages, const int32_t* d_free, int n_free,
                const int32_t* d_taken_in, int32_t* d_taken_out, int32_t* d_pairs, int32_t* d_n_pairs, void* stream) {
  if (n <= 0) return QVX_E_NVEC;
  if (int rc = check_table(n_rows, table_width, n_pages, n_free); rc != QVX_OK) return rc;
  if (page_size <= 0) return QVX_E_SHAPE;
  if (n > kMostForks || (int64_t)n_pages * page_size > 0x7fffffffll) return QVX_E_RANGE;
  if (!d_from || !d_to || !d_table || !d_lens || !d_extra || (!d_free && n_free) || !d_taken_in || !d_taken_out || !d_pairs ||
      !d_n_pairs)
    return QVX_E_NULL;
  const int64_t rows = n_rows, entries = rows * table_width;
  const Span read[] = {{d_from, 4ll * n}, {d_to, 4ll * n}, {d_free, 4ll * n_free}};
  const Span kept[] = {{d_table, 4 * entries}, {d_lens, 4 * rows}, {d_extra, 4ll * n_pages}};
  const Span made[] = {{d_taken_out, 8}, {d_pairs, 8ll * n}, {d_n_pairs, 4}};
  const Span taken[] = {{d_taken_in, 8}};
  const bool alias = d_taken_in == d_taken_out;
  if (any_overlap(read, kept) || any_overlap(read, made) || any_overlap(kept, made) || any_overlap(taken, kept) ||
      overlap(made[1], made[2]) || overlap(made[0], made[1]) || overlap(made[0], made[2]) || overlap(taken[0], made[1]) ||
      overlap(taken[0], made[2]) || (!alias && overlap(taken[0], made[0])) || overlap(kept[0], kept[1]) ||
      overlap(kept[0], kept[2]) || overlap(kept[1], kept[2]))
    return QVX_E_RANGE;
  const ForkCall c{d_from, d_to,   n,      d_table, n_rows,     table_width, page_size, d_lens,
                   d_extra, n_pages, d_free, n_free,  d_taken_in, d_taken_out, d_pairs,   d_n_pairs};
  launch_kv_fork(c, alias, static_cast<hipStream_t>(stream));
  return attn_status(true);
}

size_t qvx_kv_free_ws(int n_pages) {
  return n_pages <= 2 * kFreePages ? 0 : 4 * (((size_t)n_pages + kFreePages - 1) / kFreePages + 1);
}

int qvx_kv_free(const int32_t* d_rows, const int32_t* d_begin, const int32_t* d_end, int n, int32_t* d_table, int n_rows,
                int table_width, int32_t* d_lens, int32_t* d_extra, int n_pages, int32_t* d_free, int n_free,
                const int32_t* d_taken_in, int32_t* d_taken_out, void* d_ws, size_t ws_bytes, void* stream) {
  if (n <= 0) return QVX_E_NVEC;
  if (int rc = check_table(n_rows, table_width, n_pages, n_free); rc != QVX_OK) return rc;
  if (n > kMostForks) return QVX_E_RANGE;
  const size_t need = qvx_kv_free_ws(n_pages);
  const bool whole = !d_begin && !d_end;
  if (!d_rows || (!d_begin) != (!d_end) || !d_table || (whole && !d_lens) || !d_extra || (!d_free && n_free) || !d_taken_in ||
      !d_taken_out || (need && !d_ws))
    return QVX_E_NULL;
  if (ws_bytes < need || !aligned(d_ws, 4)) return QVX_E_RANGE;
  const Span read[] = {{d_rows, 4ll * n}, {d_begin, 4ll * n}, {d_end, 4ll * n}};
  const Span kept[] = {{d_table, 4ll * n_rows * table_width}, {whole ? d_lens : nullptr, 4ll * n_rows},
                       {d_extra, 4ll * n_pages}, {d_free, 4ll * n_free}, {d_ws, (int64_t)need}};
  const Span taken[] = {{d_taken_in, 8}, {d_taken_out, 8}};
  // the totals may lie on each other: several workgroups read them where there are several
  if (any_overlap(read, kept) || any_overlap(read, taken) || any_overlap(taken, kept) ||
      (d_taken_in != d_taken_out && overlap(taken[0], taken[1])))
    return QVX_E_RANGE;
  for (int i = 0; i < 5; ++i)
    for (int j = 0; j < i; ++j)
      if (overlap(kept[i], kept[j])) return QVX_E_RANGE;
  const FreeCall c{d_rows,  d_begin, d_end,  n,      d_table,    n_rows,      table_width,               d_lens,
                   d_extra, n_pages, d_free, n_free, d_taken_in, d_taken_out, static_cast<int32_t*>(d_ws)};
  launch_kv_free(c, static_cast<hipStream_t>(stream));
  return attn_status(true);
}

int qvx_kv_compact(const int32_t* d_table, int32_t* d_table_out, int n_rows, int table_width, const int32_t* d_extra,
                   int32_t* d_extra_out, int n_pages, const int32_t* d_free, int32_t* d_free_out, int n_free,
                   const int32_t* d_taken, int32_t* d_pairs, int32_t* d_moved, void* stream) {
  if (int rc = check_table(n_rows, table_width, n_pages, n_free); rc != QVX_OK) return rc;
  if (n_pages > kCompactPages) return QVX_E_RANGE;
  if (!d_table || !d_table_out || !d_extra || !d_extra_out || ((!d_free || !d_free_out) && n_free) || !d_taken ||
      (!d_pairs && n_pages > 1) || !d_moved)
    return QVX_E_NULL;
  const int64_t entries = (int64_t)n_rows * table_width;
  const Span in[] = {{d_table, 4 * entries}, {d_extra, 4ll * n_pages}, {d_free, 4ll * n_free}, {d_taken, 4}};
  const Span out[] = {{d_table_out, 4 * entries}, {d_extra_out, 4ll * n_pages}, {d_free_out, 4ll * n_free},
                      {d_pairs, 8ll * (n_pages / 2)}, {d_moved, 8}};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 5; ++j)
      if (overlap(in[i], out[j]) && !(i == j && in[i].p == out[j].p)) return QVX_E_RANGE;
  for (int i = 0; i < 5; ++i)
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return QVX_E_RANGE;
  const CompactCall c{d_table, d_table_out, entries, d_extra, d_extra_out, n_pages, d_free, d_free_out,
                      n_free,  d_taken,     d_pairs, d_moved};
  return attn_status(launch_kv_compact(c, d_free == d_free_out, static_cast<hipStream_t>(stream)));
}

int qvx_kv_copy(const qvx_kv_cache* caches, int n_caches, const int32_t* d_pairs, const int32_t* d_n_pairs, int most_pairs,
                void* stream) {
  if (n_caches <= 0 || most_pairs < 0) return QVX_E_NVEC;
  if (!caches) return QVX_E_NULL;
  CopyCall c{};
  for (int i = 0; i < n_caches; ++i) {
    int64_t stride = 0;
    if (int rc = check_cache(caches + i, &stride); rc != QVX_OK) return rc;
    if (caches[i].type != caches->type || caches[i].n_pages != caches->n_pages || caches[i].page_size != caches->page_size ||
        caches[i].kv_heads != caches->kv_heads || caches[i].head_dim != caches->head_dim)
      return QVX_E_SHAPE;
  }
  c.page_bytes = page_bytes(caches->type, caches->kv_heads, caches->page_size, caches->head_dim);
  if (c.page_bytes > 1ll << 36) return QVX_E_RANGE;
  if (most_pairs == 0) return QVX_OK;
  if (!d_pairs) return QVX_E_NULL;
  c.pairs = d_pairs;
  c.count = d_n_pairs;
  c.most = most_pairs;
  c.n_pages = caches->n_pages;
  for (int i0 = 0; i0 < n_caches; i0 += kCopyCaches) {
    c.n_caches = std::min(kCopyCaches, n_caches - i0);
    for (int i = 0; i < c.n_caches; ++i) {
      const qvx_kv_cache& x = caches[i0 + i];
      c.cache[i].k = static_cast<uint8_t*>(x.d_k);
      c.cache[i].v = static_cast<uint8_t*>(x.d_v);
      check_cache(&x, &c.cache[i].stride);
    }
    launch_kv_copy(c, static_cast<hipStream_t>(stream));
  }
  return attn_status(true);
}

}  // extern "C"
#pragma GCC visibility pop
