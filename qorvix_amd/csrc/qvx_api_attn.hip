// qvx_api_attn.hip -- the extern "C" boundary of the attention calls (include/qvx.h): argument checks,
// which run before any device work, and the bounds that the kernels' partition of the work needs.
#include "qvx_attn.hpp"
#include "qvx_kv.hpp"

#include <cstdio>

namespace qvx {
bool launch_attn_split(const AttnCall& c, uint32_t type, bool join, hipStream_t s);
void launch_attn_join(const AttnCall& c, hipStream_t s);
bool launch_attn16(const AttnCall& c, uint32_t type, hipStream_t s);
bool launch_kv_map(const MapCall& c, bool alias, hipStream_t s);
void launch_rope_kv(RopeCall c, uint32_t type, bool vec, hipStream_t s);
}  // namespace qvx

using namespace qvx;

namespace {

constexpr int kAttnMaxSeqs = 65536, kMapMaxSeqs = 16384;
constexpr int kMaxLen = 0x7ffffff0;  // the kernels round lengths up to whole tiles
constexpr int kMaxTiles = 0x3fffffff;  // and add a chunk's first tile and length, each at most this
constexpr int64_t kMaxPitch = 64ll << 20;  // sixteen rows stay far inside 32-bit offsets
constexpr float kLeastScale = 1e-30f;       // far above the subnormal numbers

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int attn_status(bool launched) {
  const hipError_t e = hipGetLastError();
  if (launched && e == hipSuccess) return QVX_OK;
  std::fprintf(stderr, "qvx: HIP error %d (%s)\n", (int)e, hipGetErrorString(e));
  return QVX_E_HIP;
}

// Bytes of n values of a cache or states type; 0 for another type.
int64_t value_bytes(uint32_t type, int64_t n) {
  switch (type) {
    case T_F32: return 4 * n;
    case T_F16: case T_BF16: return 2 * n;
    case T_Q8_0: return n + n / 16;
    default: return 0;
  }
}

bool head_dim_ok(uint32_t type, int d) { return d > 0 && d <= 256 && d % (type == T_Q8_0 ? 32 : 8) == 0; }

int64_t page_bytes(uint32_t type, int kv_heads, int page_size, int head_dim) {
  if (!value_bytes(type, 1) || kv_heads <= 0 || page_size <= 0 || !head_dim_ok(type, head_dim)) return 0;
  const int64_t rows = (int64_t)kv_heads * page_size;
  if (rows > (1ll << 40)) return 0;
  return (value_bytes(type, rows * head_dim) + 15) / 16 * 16;
}

int check_cache(const qvx_kv_cache* c, int64_t* stride) {
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

// The partition of a call whose heads, pages and sequences are filled in: how many work items are
// aimed at, and the bounds that grid and workspace are sized by.  Workgroups to fill the chip: two a CU.
// A chunk has at least 8 tiles (128 keys), two a wave: 2048 tokens of 8 heads of 128 11.3 us, with 4 tiles 12.0 and with 16
// 12.3; 8192 tokens 16.2, 17.7 and 16.1.
constexpr int kAttnWgs = 512, kMinChunk = 8;

// Rows of a row tile for sequences of `rows` rows.  Up to four rows run on a matrix instruction that computes
// four, a quarter the time of sixteen; up to eight on two of those: 2048 tokens, 4 heads a group, 11.2 us against 12.7 as 16
// rows, 8 heads 12.9 against 13.3.
int tile_rows(int64_t rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : 16; }

// Tiles of the longest sequence that the call allows.
int64_t most_tiles(const AttnCall& c) {
  return (int64_t)c.max_len / c.page_size * c.page_tiles + (c.max_len % c.page_size + kAttnTile - 1) / kAttnTile;
}

// The rest of a partition whose row tiles, target and min_chunk (0: one chunk, whatever the length) are chosen.
// False: it passes what a launch or 32 bits hold.
bool plan_items(AttnCall& c, int64_t row_tiles, bool* join, size_t* ws_bytes) {
  const int64_t tiles = most_tiles(c);
  *join = c.min_chunk && tiles > c.min_chunk;
  const int64_t most = *join ? (tiles + c.min_chunk - 1) / c.min_chunk : 1;  // chunks of a row tile
  const int64_t items = std::min(row_tiles + c.target, row_tiles * most);
  if (items * c.kv_heads > kMostWgs || tiles > kMaxTiles) return false;
  if (!*join) c.min_chunk = 0x7ffffff0;
  c.items = (int)items;
  c.most_tiles = (int)tiles;
  c.by_length = items * c.kv_heads > kAttnWgs;
  const int d16 = (c.head_dim + 15) / 16 * 16;
  c.small_sum = row_tiles * tiles <= 0x7fffffffll;
  c.read_once = row_tiles <= c.n_seqs;
  c.slots = (int)std::min<int64_t>(2 * (int64_t)c.target, row_tiles * most);
  *ws_bytes = *join ? sizeof(AttnPiece) * (1 + (size_t)c.slots) +
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
bool plan16(AttnCall& c, int64_t row_tiles, bool* join, size_t* ws_bytes) {
  c.tile_rows = kAttnRows16;
  const int64_t whole = row_tiles * c.kv_heads;
  const bool split = whole < kAttnWgs / 2 && most_tiles(c) > 40 + whole / 2;
  c.min_chunk = split ? 16 : 0;
  const bool sparse = 2 * (int64_t)c.n_q * c.group <= kAttnRows16 * row_tiles;
  c.target = std::max(1, (sparse ? kAttnWgs : kAttnWgs / 2) / c.kv_heads);
  return plan_items(c, row_tiles, join, ws_bytes);
}

int check_paged(const qvx_kv_cache* cache, int q_heads, int n_seqs, int table_width, AttnCall& c, bool* join,
                size_t* ws_bytes) {
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
  c.tile_rows = tile_rows(c.group);
  const int64_t row_tiles = (int64_t)n_seqs * ((c.group + c.tile_rows - 1) / c.tile_rows);
  return plan_split(c, row_tiles, join, ws_bytes) ? QVX_OK : QVX_E_RANGE;
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

constexpr float kLog2e = 1.4426950408889634f;

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
  if (n_tokens <= 0) return QVX_E_NVEC;
  if (!rope) return QVX_E_NULL;
  RopeCall c{};
  uint32_t type = T_F32;
  if (cache) {
    if (int rc = check_cache(cache, &c.page_stride); rc != QVX_OK) return rc;
    if (cache->head_dim != head_dim) return QVX_E_SHAPE;
    type = cache->type;
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
  if (d_q == d_q_out && q_stride != q_out_stride) return QVX_E_RANGE;
  c.q_out = d_q_out;
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
  bool vec = q_stride % 4 == 0 && q_out_stride % 4 == 0 && aligned(d_q, 16) && aligned(d_q_out, 16);
  if (cache) {
    c.k = d_k;
    c.v = d_v;
    c.k_stride = k_stride;
    c.v_stride = v_stride;
    c.slots = d_slots;
    vec = vec && k_stride % 4 == 0 && v_stride % 4 == 0 && aligned(d_k, 16) && aligned(d_v, 16);
  }
  launch_rope_kv(c, type, vec, static_cast<hipStream_t>(stream));
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
