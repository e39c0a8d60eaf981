// qvx_api_attn.hip -- the extern "C" boundary of the attention calls (include/qvx.h): argument checks,
// which run before any device work, and the bounds that the kernels' partition of the work needs.
#include "qvx_api_kv.hpp"
#include "qvx_attn.hpp"
#include "qvx_kv.hpp"

namespace qvx {
bool launch_attn_split(const AttnCall& c, uint32_t type, bool join, hipStream_t s);
void launch_attn_join(const AttnCall& c, hipStream_t s);
bool launch_attn_mask(const AttnCall& c, uint32_t type, bool join, hipStream_t s);
bool launch_attn16(const AttnCall& c, uint32_t type, hipStream_t s);
bool launch_kv_map(const MapCall& c, bool alias, hipStream_t s);
void launch_rope_kv(RopeCall c, uint32_t type, bool vec, hipStream_t s);
void launch_norm_rope(NormRopeCall c, uint32_t type, uint32_t q_type, bool vec, hipStream_t s);
}  // namespace qvx

using namespace qvx;

namespace {

constexpr int kAttnMaxSeqs = 65536, kMapMaxSeqs = 16384;
constexpr int kMaxLen = 0x7ffffff0;  // the kernels round lengths up to whole tiles
constexpr int kMaxTiles = 0x3fffffff;  // and add a chunk's first tile and length, each at most this
constexpr int64_t kMaxPitch = 64ll << 20;  // sixteen rows stay far inside 32-bit offsets
constexpr float kLeastScale = 1e-30f;       // far above the subnormal numbers

// The partition of a call whose heads, pages and sequences are filled in: how many work items are
// aimed at, and the bounds that grid and workspace are sized by.  Workgroups to fill the chip: two a CU.
// A chunk has at least 8 tiles (128 keys), two a wave: 2048 tokens of 8 heads of 128 11.3 us, with 4 tiles 12.0 and with 16
// 12.3; 8192 tokens 16.2, 17.7 and 16.1.
constexpr int kAttnWgs = 512, kMinChunk = 8;

// Rows of a row tile for sequences of `rows` rows.  Up to four rows run on a matrix instruction that computes
// four, a quarter the time of sixteen; up to eight on two of those: 2048 tokens, 4 heads a group, 11.2 us against 12.7 as 16
// rows, 8 heads 12.9 against 13.3.
int tile_rows(int64_t rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : 16; }

// Tiles of the longest sequence that the call allows; of a window, of what one of its row tiles may see.
int64_t tiles_of(const AttnCall& c, int len) {
  return (int64_t)len / c.page_size * c.page_tiles + (len % c.page_size + kAttnTile - 1) / kAttnTile;
}
int64_t most_tiles(const AttnCall& c) {
  const int64_t all = tiles_of(c, c.max_len) + (c.mode == kMaskWhole);  // where the shared keys end, a tile for both parts
  if (c.mode != kMaskWindow || c.window >= c.max_len) return all;
  const int64_t near = (int64_t)c.window + attn_span(c.tile_rows, c.group) - 1;
  return std::min<int64_t>(all, tiles_of(c, std::min(c.sinks, c.max_len)) +
                                    attn_most_tiles(c.page_size, c.page_tiles, std::max<int64_t>(near, 0)));
}

// The rest of a partition whose row tiles, target and min_chunk (0: one chunk, whatever the length) are chosen.
// False: it passes what a launch or 32 bits hold.
bool plan_items(AttnCall& c, int64_t row_tiles, bool* join, size_t* ws_bytes) {
  const int64_t tiles = most_tiles(c);
  *join = c.min_chunk && tiles > c.min_chunk;
  const int64_t most = *join ? (tiles + c.min_chunk - 1) / c.min_chunk : 1;  // chunks of a row tile
  const bool always = c.mode == kMaskPrefix;  // every item leaves a partial result
  const int64_t items = std::min(row_tiles + c.target, row_tiles * most);
  if (items * c.kv_heads > kMostWgs || tiles > kMaxTiles) return false;
  if (!*join) c.min_chunk = 0x7ffffff0;
  c.items = (int)items;
  c.most_tiles = (int)tiles;
  c.by_length = items * c.kv_heads > kAttnWgs;
  const int d16 = (c.head_dim + 15) / 16 * 16;
  c.small_sum = row_tiles * tiles <= 0x7fffffffll;
  c.read_once = row_tiles <= c.n_seqs;
  c.slots = (int)(always ? items : std::min<int64_t>(2 * (int64_t)c.target, row_tiles * most));
  *ws_bytes = *join || always ? sizeof(AttnPiece) * (1 + (size_t)c.slots) +
                          (size_t)c.slots * c.kv_heads * attn_part(c.tile_rows, d16) * sizeof(float)
                    : 0;
  return true;
}

// One workgroup reads some 45 GB/s, a split costs a launch of its own and the workspace's traffic, together 4 to 5 us.
// So sequences that cannot pass 320 KB of keys and values a head are left whole, and up to 640 KB those of calls that
// occupy a good part of the card all the same.  Head size 128, fp16, split against whole: 256 keys 11.3 and 8.3 us
// at 40 items, 21.4 and 13.5 at 320; 512 keys 12.2 and 11.1, 26.6 and 20.2; 1024 keys 15.0 and 15.8 at 40,
// 21.5 and 16.0 at 96, 27.5 and 20.6 at 160, 44.6 and 41.3 at 320; 2048 keys 16.0 and 24.2, 74.3 and 76.0.
// Between 40 and 96 items sequences of equal length would be faster whole from an item for each 8 KB on (672 keys at 88 items
// 19.3 and 13.1, 800 at 64 15.4 and 14.1, 1024 at 72 16.6 and 16.1), but mixed lengths split, the longest setting the time:
// up to 800 keys at 80 items 11.7 and 12.9, up to 1264 12.9 and 17.2, up to 2000 in Q8_0 15.9 and 27.9.  They lose more.
bool plan_split(AttnCall& c, int64_t row_tiles, bool* join, size_t* ws_bytes) {
  const int64_t bytes = most_tiles(c) * 2 * kAttnTile * c.key_bytes;
  const bool whole = bytes <= 320 << 10 || (bytes <= 640 << 10 && row_tiles * c.kv_heads >= 96);
  c.min_chunk = whole ? 0 : kMinChunk;
  c.target = std::max(1, kAttnWgs / c.kv_heads);
  return plan_items(c, row_tiles, join, ws_bytes);
}

// The 16-bit kernel's: row tiles of 128 rows.  Partial results of so many rows are dear, so they are split only where all of
// them find a place at once, one a CU, and the states are the longer the more of them there are; into chunks of 256 keys at
// least, one a CU (two, where row tiles are half empty in the mean).  Whole against split, a sequence a row tile of each of 8
// heads, head size 64 and 128: 8 row tiles on 700 states 14.4 and 20.3 us against 12.9 and 17.4, on 300 9.4 and 12.8 against 12.9
// and 17.6; 64 on 1500 25.9 and 37.5 against 22.3 and 30.7, on 700 15.2 and 21.9 against 16.3 and 23.4; 128 on 2500 39.2 and
// 61.9 against 36.7 and 60.6.  Above half the CUs lengths decide: 192 of equal length on 4000 states 62.5 and 103 against 67.9 and
// 114 (of one sequence 57.7 and 86.5 against 57.6 and 87.1), but seven ragged ones of 450 queries at most 57.3 and 85.3 against
// 45.3 and 68.2.  Chunks for two workgroups a CU: 32 on 4000 27.6 and 35.1 against 21.8 and 28.5; but 4 sequences of 32 rows on
// 1500, 20 heads of 64, 15.5 against 17.3.
// Row tiles of 64 rows leave the matrix cores time: two chunks a CU, up to one row tile a CU.  60 rows each over 16000 keys, 20
// sequences of 8 heads 423 us with a chunk a CU and 257 with two, 32 of 20 rows 441 and 364; but 40 of them over 5000 156 and 175.
// (Of as many queries each.  By offsets a row tile more a sequence has to be reckoned with, which passes that bound sooner: the first
// two 417 and 435 us.)
bool plan16(AttnCall& c, int64_t row_tiles, bool* join, size_t* ws_bytes) {
  const int64_t whole = row_tiles * c.kv_heads;
  const bool half = c.tile_rows < kAttnRows16;
  const bool split = (half ? whole <= kAttnWgs / 2 : whole < kAttnWgs / 2) && most_tiles(c) > 40 + whole / 2;
  c.min_chunk = split ? 16 : 0;
  const bool sparse = 2 * (int64_t)c.n_q * c.group <= c.tile_rows * row_tiles;
  c.target = std::max(1, (sparse || half ? kAttnWgs : kAttnWgs / 2) / c.kv_heads);
  return plan_items(c, row_tiles, join, ws_bytes);
}

// A call's cache and table, whatever its queries.
int check_pages(const qvx_kv_cache* cache, int q_heads, int n_seqs, int table_width, AttnCall& c) {
  if (n_seqs <= 0) return QVX_E_NVEC;
  if (int rc = check_cache(cache, &c.page_stride); rc != QVX_OK) return rc;
  if (q_heads <= 0 || q_heads % cache->kv_heads || table_width <= 0) return QVX_E_SHAPE;
  if (n_seqs > kAttnMaxSeqs || cache->kv_heads > 65535 || (int64_t)table_width * cache->page_size > kMaxLen)
    return QVX_E_RANGE;
  const int d = cache->head_dim;
  c.k = static_cast<const uint8_t*>(cache->d_k);
  c.v = static_cast<const uint8_t*>(cache->d_v);
  c.pitch = cache->type == T_Q8_0 ? d : (int)value_bytes(cache->type, d);
  c.key_bytes = (int)value_bytes(cache->type, d);
  c.head_stride = (int64_t)cache->page_size * c.pitch;
  c.scale_off = (int64_t)cache->kv_heads * c.head_stride;
  c.table_width = table_width;
  c.n_pages = cache->n_pages;
  c.page_size = cache->page_size;
  c.page_tiles = (cache->page_size + kAttnTile - 1) / kAttnTile;
  c.max_len = table_width * cache->page_size;
  c.n_seqs = c.n_q = n_seqs;
  c.q_each = 1;
  c.kv_heads = cache->kv_heads;
  c.group = q_heads / cache->kv_heads;
  c.head_dim = d;
  return QVX_OK;
}

int check_paged(const qvx_kv_cache* cache, int q_heads, int n_seqs, int table_width, AttnCall& c, bool* join,
                size_t* ws_bytes) {
  if (int rc = check_pages(cache, q_heads, n_seqs, table_width, c); rc != QVX_OK) return rc;
  c.tile_rows = tile_rows(c.group);
  const int64_t row_tiles = (int64_t)n_seqs * ((c.group + c.tile_rows - 1) / c.tile_rows);
  return plan_split(c, row_tiles, join, ws_bytes) ? QVX_OK : QVX_E_RANGE;
}

bool q_type_ok(uint32_t t) { return t == T_F32 || t == T_F16 || t == T_BF16; }

// Whether calls of so many rows a sequence (of a mean one) run on the kernel of many rows, and the partition's geometry there: keys
// in a row, whatever their pages.  Those of more than a row tile of the split kernel, which reads the keys again for each; up to 64
// rows in row tiles of 64, waves in two groups on other keys.  8 key heads of 128 in fp16, split kernel against this one, fp32 and
// fp16 queries: 8 sequences of 2000 tokens 20 rows 30.7 and 29.0, 30.4 and 28.2 us, 32 rows 30.9 and 32.2, 31.0 and 30.5, 48 rows
// 47.8 and 34.6, 47.8 and 31.7; 32 of 16000 20 rows 471 and 369, 469 and 444, 48 rows 699 and 431, 694 and 451.  One prefix of 30000
// tokens, 32 rows 52.8 and 41.2, 48 rows 61.4 and 42.8; 64 rows 43.8, in a row tile of 128 51.2.
bool many_rows(const qvx_kv_cache* cache, int64_t rows, AttnCall& c) {
  if ((cache->type != T_F16 && cache->type != T_BF16) || rows <= 16) return false;
  if (c.max_len > 0x7ffff000) return false;  // it looks up to 1024 keys past the last one by number
  c.table_page = c.page_size;
  c.page_size = c.max_len;
  c.page_tiles = (int)(((int64_t)c.max_len + kAttnTile - 1) / kAttnTile);
  c.tile_rows = rows <= kAttnRows16 / 2 ? kAttnRows16 / 2 : kAttnRows16;
  return true;
}

int check_window(const qvx_kv_cache* cache, uint32_t q_type, int q_heads, bool ragged, int n_q, int n_seqs, int table_width,
                 int window, int sinks, AttnCall& c, bool* join, size_t* ws_bytes) {
  if (int rc = check_pages(cache, q_heads, n_seqs, table_width, c); rc != QVX_OK) return rc;
  if (!q_type_ok(q_type)) return QVX_E_TYPE;
  if (n_q < 0 || (!ragged && n_q % n_seqs) || window < 0 || sinks < 0) return QVX_E_SHAPE;
  if ((int64_t)n_q * c.group > 0x7fffff00ll) return QVX_E_RANGE;
  c.mode = kMaskWindow;
  c.q_type = q_type;
  c.n_q = n_q;
  c.q_each = ragged ? 0 : n_q / n_seqs;
  c.window = std::min(window, kMaxLen);
  c.sinks = std::min(sinks, kMaxLen);
  const int64_t rows = (int64_t)(ragged ? n_q : n_q / n_seqs) * c.group;
  const int64_t mean = ragged ? (rows + n_seqs - 1) / n_seqs : rows;
  const bool many = many_rows(cache, mean, c);
  if (!many) c.tile_rows = tile_rows(mean);
  const int64_t row_tiles =
      ragged ? rows / c.tile_rows + n_seqs : n_seqs * ((rows + c.tile_rows - 1) / c.tile_rows);
  return (many ? plan16 : plan_split)(c, row_tiles, join, ws_bytes) ? QVX_OK : QVX_E_RANGE;
}

// Whether sequences read shared keys each for itself, in one launch (kMaskWhole): reading them once costs another launch and
// partial results of the prefix, which is worth it where the tables hold more than 128 MB of keys and values in all, or 256 MB in
// rows of up to 1024 tokens.  Past 256 sequences a thread looks for several groups, again and again.  Once against each for
// itself, 8 heads of 128 in fp16, 4 queries each: 4 sequences of 1000 tokens 19.0 and 12.8 us, 16 of 1600 21.9 and 20.9, of 3100 24.0
// and 28.0, 32 of 1600 24.9 and 27.6, 64 of 306 24.8 and 12.2, of 1000 29.8 and 24.8, of 1600 30.9 and 36.9, 100 of 1000 41.1 and
// 48.1, 200 of 306 54.3 and 43.8, in fifty groups 55.0 and 47.9.
bool read_whole(const AttnCall& c, int n_groups) {
  const int64_t bytes = (int64_t)c.n_seqs * c.max_len * 2 * c.key_bytes * c.kv_heads;
  return bytes <= (c.max_len <= 1024 ? 256ll : 128ll) << 20 && (c.n_seqs <= 256 || n_groups == 1);
}

// The two parts of qvx_attn_shared, and where they lie in its workspace: what the prefix leaves for each query and its
// counters, its partial results, and the rest's.
struct SharedPlan {
  AttnCall prefix{}, rest{};
  bool whole = false;  // `rest` alone, each sequence reading the shared keys for itself
  bool join = false;  // the rest may be split
  size_t arrived_at = 0, lead_bytes = 0, prefix_bytes = 0, bytes = 0;
};

int check_shared(const qvx_kv_cache* cache, uint32_t q_type, int q_heads, int n_seqs, int table_width, int n_groups,
                 SharedPlan& p) {
  if (int rc = check_pages(cache, q_heads, n_seqs, table_width, p.rest); rc != QVX_OK) return rc;
  if (!q_type_ok(q_type)) return QVX_E_TYPE;
  if (n_groups <= 0) return QVX_E_SHAPE;
  if (n_groups > n_seqs || (int64_t)n_seqs * p.rest.group > 0x7fffff00ll) return QVX_E_RANGE;
  p.rest.q_type = q_type;
  if (read_whole(p.rest, n_groups)) {
    p.whole = true;
    p.rest.mode = kMaskWhole;
    p.rest.n_groups = n_groups;
    p.rest.tile_rows = tile_rows(p.rest.group);
    const int64_t row_tiles = (int64_t)n_seqs * ((p.rest.group + p.rest.tile_rows - 1) / p.rest.tile_rows);
    if (!plan_split(p.rest, row_tiles, &p.join, &p.bytes)) return QVX_E_RANGE;
    p.rest.read_once = false;  // a group's sequences read the same keys
    p.bytes = std::max<size_t>(p.bytes, 16);
    return QVX_OK;
  }
  AttnCall& c = p.prefix;
  c = p.rest;
  c.mode = kMaskPrefix;
  c.n_seqs = n_groups;
  const int64_t rows = (int64_t)n_seqs * c.group;
  const int64_t mean = (rows + n_groups - 1) / n_groups;
  bool split = false;
  // Every chunk leaves its partial results: two chunks a CU, of 128 keys at least.  64 sequences of 4 heads a group behind 1000
  // keys 28.6 us, with chunks of 256 32.2, of 512 41.5; 128 behind 8192, fp16, 61.6, with a chunk a CU 66.8.
  if (many_rows(cache, mean, c)) {
    c.min_chunk = 8;
    c.target = std::max(1, kAttnWgs / c.kv_heads);
    if (!plan_items(c, rows / c.tile_rows + n_groups, &split, &p.prefix_bytes)) return QVX_E_RANGE;
  } else {
    c.tile_rows = tile_rows(mean);
    if (!plan_split(c, rows / c.tile_rows + n_groups, &split, &p.prefix_bytes)) return QVX_E_RANGE;
  }
  AttnCall& r = p.rest;
  r.mode = kMaskRest;
  r.lead_rows = c.tile_rows;
  r.lead_slots = c.slots;
  r.tile_rows = tile_rows(r.group);
  // Whole up to 512 keys: its chunks meet through memory, 4 us or so.  64 sequences of 1 to 512 own tokens behind 8192 49.9 us,
  // with chunks of 128 keys 56.9, of 1024 50.7; 5 of 1000 32.6, with 256 30.1, with 1024 35.5.
  size_t rest_bytes = 0;
  r.min_chunk = 32;
  r.target = std::max(1, kAttnWgs / r.kv_heads);
  if (!plan_items(r, (int64_t)n_seqs * ((r.group + r.tile_rows - 1) / r.tile_rows), &p.join, &rest_bytes)) return QVX_E_RANGE;
  r.rest_tiles = c.rest_tiles = (r.group + r.tile_rows - 1) / r.tile_rows;
  p.arrived_at = sizeof(AttnLead) * (size_t)n_seqs;
  p.lead_bytes = p.arrived_at + (4 * (size_t)n_seqs * r.rest_tiles * r.kv_heads + 15) / 16 * 16;
  p.bytes = p.lead_bytes + p.prefix_bytes + rest_bytes;
  return QVX_OK;
}

// wide: the call runs on the 16-bit matrix cores (qvx_attn16.hip): q and the states share a 16-bit type, the scale is
// positive (the kernel takes the largest product for the largest logit, and -inf times the scale for a masked one),
// sequences have more than 16 rows in the mean, and its tiles of 64 states stay inside 32-bit offsets.  20 heads of 64 on
// 1500 states, one sequence and eight, there against the split kernel: 16 queries 12.0 and 20.1 us against 12.9 and 19.4, 24
// 12.3 and 20.3 against 14.8 and 29.2, 128 16.2 and 31.6 against 19.3 and 59.3.
int check_cross(const qvx_kv_states* st, uint32_t q_type, int q_heads, bool ragged, int n_q, int n_seqs, float scale,
                AttnCall& c, bool* wide, bool* join, size_t* ws_bytes) {
  if (!st) return QVX_E_NULL;
  if (n_seqs <= 0) return QVX_E_NVEC;
  if ((q_type != T_F32 && q_type != T_F16 && q_type != T_BF16) ||
      (st->type != T_F32 && st->type != T_F16 && st->type != T_BF16))
    return QVX_E_TYPE;
  if (n_q < 0 || (!ragged && n_q % n_seqs) || q_heads <= 0 || st->kv_heads <= 0 || q_heads % st->kv_heads ||
      st->max_len < 0 || !head_dim_ok(st->type, st->head_dim) || st->row_stride < st->head_dim || st->batch_stride < 0 ||
      st->head_stride < 0)
    return QVX_E_SHAPE;
  const int64_t es = value_bytes(st->type, 1);
  constexpr int64_t kMost = 1ll << 56;
  if (n_seqs > kAttnMaxSeqs || st->max_len > kMaxLen || st->kv_heads > 65535 || st->batch_stride > kMost ||
      st->head_stride > kMost || st->row_stride > kMaxPitch / es || (st->row_stride * es) % 16 || (st->batch_stride * es) % 16 ||
      (st->head_stride * es) % 16)
    return QVX_E_RANGE;
  if (st->max_len && (!st->d_k || !st->d_v)) return QVX_E_NULL;
  if (!aligned(st->d_k, 16) || !aligned(st->d_v, 16)) return QVX_E_RANGE;
  c.q_type = q_type;
  c.k = static_cast<const uint8_t*>(st->d_k);
  c.v = static_cast<const uint8_t*>(st->d_v);
  c.page_stride = st->batch_stride * es;
  c.head_stride = st->head_stride * es;
  c.pitch = (int)(st->row_stride * es);
  c.key_bytes = (int)(st->head_dim * es);
  c.n_pages = n_seqs;
  c.page_tiles = std::max(1, st->max_len / kAttnTile + (st->max_len % kAttnTile != 0));
  c.page_size = std::max(1, st->max_len);
  c.max_len = st->max_len;
  c.n_seqs = n_seqs;
  c.n_q = n_q;
  c.q_each = ragged ? 0 : n_q / n_seqs;
  c.kv_heads = st->kv_heads;
  c.group = q_heads / st->kv_heads;
  c.head_dim = st->head_dim;
  const int64_t rows = (int64_t)(ragged ? n_q : n_q / n_seqs) * c.group;
  if ((int64_t)n_q * c.group > 0x7fffff00ll) return QVX_E_RANGE;
  *wide = q_type == st->type && q_type != T_F32 && scale >= kLeastScale && c.pitch <= kMaxPitch / 4 &&
          (int64_t)n_q * c.group > 16 * (int64_t)n_seqs;
  c.tile_rows = *wide ? kAttnRows16 : tile_rows(ragged ? rows / n_seqs : rows);  // ragged: of a sequence in the mean
  const int64_t row_tiles =
      ragged ? rows / c.tile_rows + n_seqs : n_seqs * ((rows + c.tile_rows - 1) / c.tile_rows);
  return (*wide ? plan16 : plan_split)(c, row_tiles, join, ws_bytes) ? QVX_OK : QVX_E_RANGE;
}

// What qvx_rope_kv and qvx_norm_rope_kv check alike.  vec: rows on 16-byte addresses (q_out's of 16 bits on 8-byte ones).
int check_rope(void* d_q_out, int64_t q_out_stride, uint32_t q_out_type, const float* d_q, int64_t q_stride, int q_heads,
               const float* d_k, int64_t k_stride, const float* d_v, int64_t v_stride, int n_tokens, int head_dim,
               const qvx_rope* rope, const int32_t* d_pos, int64_t pos_stride, const qvx_kv_cache* cache,
               const int32_t* d_slots, RopeCall& c, uint32_t* type, bool* vec) {
  if (n_tokens <= 0) return QVX_E_NVEC;
  if (!rope) return QVX_E_NULL;
  *type = T_F32;
  if (cache) {
    if (int rc = check_cache(cache, &c.page_stride); rc != QVX_OK) return rc;
    if (cache->head_dim != head_dim) return QVX_E_SHAPE;
    *type = cache->type;
    c.kv_heads = cache->kv_heads;
    c.k_pages = static_cast<uint8_t*>(cache->d_k);
    c.v_pages = static_cast<uint8_t*>(cache->d_v);
    c.scale_off = (int64_t)cache->kv_heads * cache->page_size * head_dim;
    c.page_size = cache->page_size;
    c.n_slots = (int64_t)cache->n_pages * cache->page_size;
  }
  if (rope->pairing != QVX_ROPE_HALVES && rope->pairing != QVX_ROPE_PAIRS) return QVX_E_VARIANT;
  if (q_heads < 0 || q_heads + c.kv_heads <= 0 || !head_dim_ok(T_F32, head_dim) || rope->rot_dim < 0 ||
      rope->rot_dim > head_dim || rope->rot_dim % 8 || rope->n_axes < 1 || rope->n_axes > 4)
    return QVX_E_SHAPE;
  const int64_t q_row = (int64_t)q_heads * head_dim, kv_row = (int64_t)c.kv_heads * head_dim;
  if (q_stride < 0 || q_out_stride < q_row || (cache && (k_stride < 0 || v_stride < 0)) || pos_stride < 0 ||
      (rope->n_axes > 1 && pos_stride < n_tokens))
    return QVX_E_SHAPE;
  if (q_row > 0x7fffffffll / 16 || kv_row > 0x7fffffffll / 16 || n_tokens > kRopeMaxTokens * kMostWgs)
    return QVX_E_RANGE;
  if ((q_heads && (!d_q || !d_q_out)) || (cache && (!d_k || !d_v || !d_slots)) ||
      (rope->rot_dim && (!rope->d_inv_freq || !d_pos)))
    return QVX_E_NULL;
  if (q_heads && d_q == d_q_out && (q_stride != q_out_stride || q_out_type != T_F32)) return QVX_E_RANGE;
  const uintptr_t size = q_out_type == T_F32 ? 4 : 2;
  if (q_out_type != T_F32 && !aligned(d_q_out, 2)) return QVX_E_RANGE;
  c.q_out = static_cast<float*>(d_q_out);
  c.q = d_q;
  c.q_out_stride = q_out_stride;
  c.q_stride = q_stride;
  c.q_heads = q_heads;
  c.head_dim = head_dim;
  c.n_tokens = n_tokens;
  c.inv_freq = rope->d_inv_freq;
  c.axis = rope->d_axis;
  c.rot_dim = rope->rot_dim;
  c.n_axes = rope->n_axes;
  c.halves = rope->pairing == QVX_ROPE_HALVES;
  c.scale = rope->scale;
  c.pos = d_pos;
  c.pos_stride = pos_stride;
  *vec = q_stride % 4 == 0 && q_out_stride % 4 == 0 && aligned(d_q, 16) && aligned(d_q_out, 4 * size);
  if (cache) {
    c.k = d_k;
    c.v = d_v;
    c.k_stride = k_stride;
    c.v_stride = v_stride;
    c.slots = d_slots;
    *vec = *vec && k_stride % 4 == 0 && v_stride % 4 == 0 && aligned(d_k, 16) && aligned(d_v, 16);
  }
  return QVX_OK;
}

constexpr float kLog2e = 1.4426950408889634f;

// The rows of q and out of a masked call, which may be the same ones.
int check_rows(void* d_out, int64_t out_stride, const void* d_q, int64_t q_stride, AttnCall& c) {
  const uintptr_t size = c.q_type == T_F32 ? 4 : 2;
  if (q_stride < 0 || out_stride < (int64_t)c.group * c.kv_heads * c.head_dim) return QVX_E_SHAPE;
  if (!aligned(d_out, size) || !aligned(d_q, size) || (d_out == d_q && d_q && q_stride != out_stride)) return QVX_E_RANGE;
  c.q = d_q;
  c.out = d_out;
  c.q_stride = q_stride;
  c.out_stride = out_stride;
  return QVX_OK;
}

}  // namespace

#pragma GCC visibility push(default)
extern "C" {

size_t qvx_kv_page_bytes(uint32_t type, int kv_heads, int page_size, int head_dim) {
  return (size_t)page_bytes(type, kv_heads, page_size, head_dim);
}

int qvx_kv_map(const int32_t* d_held, const int32_t* d_new, int n_seqs, int32_t* d_table, int table_width,
               int page_size, const int32_t* d_free, int n_free, const int32_t* d_taken_in, int32_t* d_taken_out,
               int32_t* d_lens, int32_t* d_offsets, int32_t* d_slots, int32_t* d_pos, int32_t* d_seq,
               int max_tokens, void* stream) {
  if (n_seqs <= 0) return QVX_E_NVEC;
  if (table_width <= 0 || page_size <= 0 || n_free < 0 || max_tokens < 0) return QVX_E_SHAPE;
  if (n_seqs > kMapMaxSeqs) return QVX_E_RANGE;
  if (!d_held || !d_new || !d_table || (!d_free && n_free) || !d_taken_in || !d_taken_out || !d_lens || !d_offsets ||
      (!d_slots && max_tokens))
    return QVX_E_NULL;
  const struct {
    const int32_t* p;
    int64_t n;
  } ins[] = {{d_held, n_seqs}, {d_new, n_seqs}, {d_taken_in, 2}},
    outs[] = {{d_lens, n_seqs}, {d_taken_out, 2}, {d_offsets, n_seqs + 1}, {d_slots, max_tokens}, {d_pos, max_tokens},
              {d_seq, max_tokens}};
  bool alias = false;
  for (const auto& i : ins)
    for (const auto& o : outs) {
      const auto a = reinterpret_cast<uintptr_t>(i.p), b = reinterpret_cast<uintptr_t>(o.p);
      if (!b || a + 4 * i.n <= b || b + 4 * o.n <= a) continue;
      if (i.p == o.p && ((i.p == d_held && o.p == d_lens) || (i.p == d_taken_in && o.p == d_taken_out)))
        alias = true;
      else
        return QVX_E_RANGE;
    }
  const MapCall c{d_held, d_new,  n_seqs,    d_table, table_width, page_size, d_free, n_free,
                  d_taken_in, d_taken_out, d_lens, d_offsets, d_slots, d_pos, d_seq, max_tokens};
  return attn_status(launch_kv_map(c, alias, static_cast<hipStream_t>(stream)));
}

int qvx_rope_kv(float* d_q_out, int64_t q_out_stride, const float* d_q, int64_t q_stride, int q_heads,
                const float* d_k, int64_t k_stride, const float* d_v, int64_t v_stride, int n_tokens, int head_dim,
                const qvx_rope* rope, const int32_t* d_pos, int64_t pos_stride, const qvx_kv_cache* cache,
                const int32_t* d_slots, void* stream) {
  RopeCall c{};
  uint32_t type = 0;
  bool vec = false;
  if (int rc = check_rope(d_q_out, q_out_stride, T_F32, d_q, q_stride, q_heads, d_k, k_stride, d_v, v_stride, n_tokens,
                          head_dim, rope, d_pos, pos_stride, cache, d_slots, c, &type, &vec);
      rc != QVX_OK)
    return rc;
  launch_rope_kv(c, type, vec, static_cast<hipStream_t>(stream));
  return attn_status(true);
}

int qvx_norm_rope_kv(void* d_q_out, int64_t q_out_stride, uint32_t q_out_type, const float* d_q, int64_t q_stride,
                     int q_heads, const float* d_k, int64_t k_stride, const float* d_v, int64_t v_stride, int n_tokens,
                     int head_dim, const qvx_qk_norm* norm, const qvx_rope* rope, const int32_t* d_pos, int64_t pos_stride,
                     const qvx_kv_cache* cache, const int32_t* d_slots, void* stream) {
  NormRopeCall c{};
  uint32_t type = 0;
  bool vec = false;
  if (!norm) return QVX_E_NULL;
  if (q_out_type != T_F32 && q_out_type != T_F16 && q_out_type != T_BF16) return QVX_E_TYPE;
  if (int rc = check_rope(d_q_out, q_out_stride, q_out_type, d_q, q_stride, q_heads, d_k, k_stride, d_v, v_stride, n_tokens,
                          head_dim, rope, d_pos, pos_stride, cache, d_slots, c, &type, &vec);
      rc != QVX_OK)
    return rc;
  if (norm->head_stride != 0 && norm->head_stride < head_dim) return QVX_E_SHAPE;
  if (!(norm->eps >= 0.0f)) return QVX_E_RANGE;
  c.q_typed = d_q_out;
  c.q_w = norm->d_q_w;
  c.k_w = norm->d_k_w;
  c.w_stride = norm->head_stride;
  c.eps = norm->eps;
  c.inv_dim = 1.0 / head_dim;
  launch_norm_rope(c, type, q_out_type, vec, static_cast<hipStream_t>(stream));
  return attn_status(true);
}

size_t qvx_attn_paged_ws(const qvx_kv_cache* cache, int q_heads, int n_seqs, int table_width) {
  AttnCall c{};
  bool join = false;
  size_t bytes = 0;
  return check_paged(cache, q_heads, n_seqs, table_width, c, &join, &bytes) == QVX_OK ? bytes : 0;
}

int qvx_attn_paged(float* d_out, int64_t out_stride, const float* d_q, int64_t q_stride, int q_heads,
                   const qvx_kv_cache* cache, const int32_t* d_table, int table_width, const int32_t* d_lens,
                   int n_seqs, float scale, void* d_ws, size_t ws_bytes, void* stream) {
  AttnCall c{};
  bool join = false;
  size_t need = 0;
  if (int rc = check_paged(cache, q_heads, n_seqs, table_width, c, &join, &need); rc != QVX_OK) return rc;
  if (q_stride < 0 || out_stride < (int64_t)q_heads * cache->head_dim) return QVX_E_SHAPE;
  if (!d_out || !d_q || !d_table || !d_lens || (need && !d_ws)) return QVX_E_NULL;
  if (ws_bytes < need || !aligned(d_ws, 16) || (d_out == d_q && q_stride != out_stride)) return QVX_E_RANGE;
  c.q = d_q;
  c.out = d_out;
  c.q_stride = q_stride;
  c.out_stride = out_stride;
  c.q_type = T_F32;
  c.table = d_table;
  c.lens = d_lens;
  c.scale2 = scale * kLog2e;
  c.ws = join ? static_cast<float*>(d_ws) : nullptr;
  return attn_status(launch_attn_split(c, cache->type, join, static_cast<hipStream_t>(stream)));
}

size_t qvx_attn_window_ws(const qvx_kv_cache* cache, uint32_t q_type, int q_heads, int n_q, int n_seqs, int table_width,
                          int window, int sinks) {
  size_t most = 0;
  for (int i = 0; i < 2; ++i) {  // ragged or equal queries
    AttnCall c{};
    bool join = false;
    size_t bytes = 0;
    if (check_window(cache, q_type, q_heads, i, n_q, n_seqs, table_width, window, sinks, c, &join, &bytes) == QVX_OK)
      most = std::max(most, bytes);
  }
  return most;
}

int qvx_attn_window(void* d_out, int64_t out_stride, const void* d_q, int64_t q_stride, uint32_t q_type, int q_heads,
                    const int32_t* d_offsets, int n_q, const qvx_kv_cache* cache, const int32_t* d_table, int table_width,
                    const int32_t* d_lens, int n_seqs, int window, int sinks, float scale, void* d_ws, size_t ws_bytes,
                    void* stream) {
  AttnCall c{};
  bool join = false;
  size_t need = 0;
  if (int rc = check_window(cache, q_type, q_heads, d_offsets != nullptr, n_q, n_seqs, table_width, window, sinks, c, &join,
                            &need);
      rc != QVX_OK)
    return rc;
  if (int rc = check_rows(d_out, out_stride, d_q, q_stride, c); rc != QVX_OK) return rc;
  if (n_q == 0) return QVX_OK;
  if (!d_out || !d_q || !d_table || !d_lens || (need && !d_ws)) return QVX_E_NULL;
  if (ws_bytes < need || !aligned(d_ws, 16)) return QVX_E_RANGE;
  c.q_offsets = d_offsets;
  c.table = d_table;
  c.lens = d_lens;
  c.scale2 = scale * kLog2e;
  c.in_order = scale >= kLeastScale;
  c.ws = join ? static_cast<float*>(d_ws) : nullptr;
  c.q_wide = aligned(d_q, 16) && q_stride % 8 == 0;
  c.out_wide = aligned(d_out, 8) && out_stride % 4 == 0;
  return attn_status(launch_attn_mask(c, cache->type, join, static_cast<hipStream_t>(stream)));
}

size_t qvx_attn_shared_ws(const qvx_kv_cache* cache, uint32_t q_type, int q_heads, int n_seqs, int table_width,
                          int n_groups) {
  SharedPlan p;
  return check_shared(cache, q_type, q_heads, n_seqs, table_width, n_groups, p) == QVX_OK ? p.bytes : 0;
}

int qvx_attn_shared(void* d_out, int64_t out_stride, const void* d_q, int64_t q_stride, uint32_t q_type, int q_heads,
                    const qvx_kv_cache* cache, const int32_t* d_table, int table_width, const int32_t* d_lens, int n_seqs,
                    const int32_t* d_groups, const int32_t* d_shared, int n_groups, float scale, void* d_ws,
                    size_t ws_bytes, void* stream) {
  SharedPlan p;
  if (int rc = check_shared(cache, q_type, q_heads, n_seqs, table_width, n_groups, p); rc != QVX_OK) return rc;
  if (int rc = check_rows(d_out, out_stride, d_q, q_stride, p.rest); rc != QVX_OK) return rc;
  if (!d_out || !d_q || !d_table || !d_lens || (!d_groups && n_groups > 1) || !d_shared || !d_ws) return QVX_E_NULL;
  if (ws_bytes < p.bytes || !aligned(d_ws, 16)) return QVX_E_RANGE;
  uint8_t* ws = static_cast<uint8_t*>(d_ws);
  for (AttnCall* c : {&p.prefix, &p.rest}) {
    c->q = d_q;
    c->out = d_out;
    c->q_stride = q_stride;
    c->out_stride = out_stride;
    c->table = d_table;
    c->lens = d_lens;
    c->scale2 = scale * kLog2e;
    c->in_order = scale >= kLeastScale;
    c->leads = reinterpret_cast<AttnLead*>(ws);
    c->arrived = reinterpret_cast<int*>(ws + p.arrived_at);
    c->q_wide = aligned(d_q, 16) && q_stride % 8 == 0;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  p.prefix.groups = p.rest.groups = d_groups;
  p.prefix.shared = p.rest.shared = d_shared;
  if (p.whole) {
    p.rest.ws = p.join ? static_cast<float*>(d_ws) : nullptr;
    return attn_status(launch_attn_mask(p.rest, cache->type, p.join, s));
  }
  p.prefix.ws = reinterpret_cast<float*>(ws + p.lead_bytes);
  p.rest.lead_ws = p.prefix.ws;
  p.rest.ws = p.join ? reinterpret_cast<float*>(ws + p.lead_bytes + p.prefix_bytes) : nullptr;
  if (!launch_attn_mask(p.prefix, cache->type, false, s)) return attn_status(false);
  return attn_status(launch_attn_mask(p.rest, cache->type, false, s));  // the rest's chunks join themselves
}

size_t qvx_attn_cross_ws(const qvx_kv_states* states, uint32_t q_type, int q_heads, int n_q, int n_seqs) {
  // Ragged and equal queries differ in their bounds, scales of either sign in their kernel: the largest need serves all.
  size_t most = 0;
  for (int i = 0; i < 4; ++i) {
    AttnCall c{};
    bool wide = false, join = false;
    size_t bytes = 0;
    if (check_cross(states, q_type, q_heads, i & 1, n_q, n_seqs, i & 2 ? 1.0f : -1.0f, c, &wide, &join, &bytes) == QVX_OK)
      most = std::max(most, bytes);
  }
  return most;
}

int qvx_attn_cross(void* d_out, int64_t out_stride, const void* d_q, int64_t q_stride, uint32_t q_type, int q_heads,
                   const int32_t* d_offsets, int n_q, const qvx_kv_states* states, const int32_t* d_lens, int n_seqs,
                   float scale, void* d_ws, size_t ws_bytes, void* stream) {
  AttnCall c{};
  bool wide = false, join = false;
  size_t need = 0;
  if (int rc = check_cross(states, q_type, q_heads, d_offsets != nullptr, n_q, n_seqs, scale, c, &wide, &join, &need);
      rc != QVX_OK)
    return rc;
  if (q_stride < 0 || out_stride < (int64_t)q_heads * states->head_dim) return QVX_E_SHAPE;
  if (n_q == 0) return QVX_OK;
  if (!d_out || !d_q || (need && !d_ws)) return QVX_E_NULL;
  if (!aligned(d_out, q_type == T_F32 ? 4 : 2) || !aligned(d_q, q_type == T_F32 ? 4 : 2) || ws_bytes < need ||
      !aligned(d_ws, 16) || (d_out == d_q && q_stride != out_stride))
    return QVX_E_RANGE;
  c.q = d_q;
  c.out = d_out;
  c.q_stride = q_stride;
  c.out_stride = out_stride;
  c.q_offsets = d_offsets;
  c.lens = d_lens;
  c.scale2 = scale * kLog2e;
  c.ws = join ? static_cast<float*>(d_ws) : nullptr;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (!wide) return attn_status(launch_attn_split(c, states->type, join, s));
  c.q_wide = aligned(d_q, 16) && q_stride % 8 == 0;
  c.out_wide = aligned(d_out, 8) && out_stride % 4 == 0;
  const bool ok = launch_attn16(c, states->type, s);
  if (ok && join) launch_attn_join(c, s);
  return attn_status(ok);
}

}  // extern "C"
#pragma GCC visibility pop
