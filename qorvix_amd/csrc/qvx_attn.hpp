// qvx_attn.hpp -- what the attention kernels share: the call as the host checked it, element types,
// and the partition of the work (sequence, row tile, chunk of keys) that every workgroup derives by
// itself from the lengths on the device.
//
// A call attends rows of queries to the keys of their own sequence.  For one key / value head, the
// query heads of its group at each query of a sequence are its rows, row = query * group + head in
// the group, taken R at a time; the keys are taken in tiles of 16.
// A page of the paged cache holds whole tiles but for its last one, so tiles never cross a page.
#pragma once

#include "qvx_common.hpp"

namespace qvx {

constexpr int kAttnTile = 16;   // keys of a tile
constexpr int kAttnRows16 = 128;  // query rows of a workgroup of the 16-bit kernel
constexpr int kMostWgs = (1 << 24) - 1;  // of 256 threads: a launch holds fewer than 2^32 of them
constexpr int kAttnWaves = 4;   // waves of a workgroup of the split kernel
constexpr float kAttnLow = -3.4028235e38f;  // stands for the maximum of keys that are all at -inf; -inf: of no keys

struct AttnCall {
  const void* q;
  void* out;
  int64_t q_stride, out_stride;  // elements from one query's heads to the next query's
  uint32_t q_type;               // T_F32, T_F16 or T_BF16, the output's type too
  bool q_wide, out_wide;         // 16-bit rows of q on 16-byte, of out on 8-byte addresses
  const int32_t* q_offsets;      // [n_seqs + 1], or null: q_each queries a sequence
  int q_each, n_q;
  const uint8_t *k, *v;
  int64_t page_stride;  // bytes from a page (or a sequence's states) to the next
  int64_t head_stride;  // bytes from a head to the next within it
  int64_t scale_off;    // Q8_0: bytes from a page's quants to its scales
  int pitch;            // bytes from a token's values of one head to the next token's
  int key_bytes;        // bytes of those values
  const int32_t* table;  // paged: [n_seqs, table_width]; null: sequence b is "page" b
  int table_width, n_pages;
  int page_size;       // tokens of a page (states: the longest sequence)
  int page_tiles;      // tiles of a page
  const int32_t* lens;  // null: every sequence has max_len keys
  int max_len;
  int most_tiles;      // of a sequence of that length
  int n_seqs, kv_heads, group, head_dim;
  float scale2;     // scale * log2(e): the kernels work with powers of two
  int tile_rows;    // query rows of a row tile: 4, 8 or 16 in the split kernel, 64 or 128 of many rows, 128 in the 16-bit one
  int items;        // bound on the work items of a key / value head; the grid is items * kv_heads
  int target, min_chunk;  // work items aimed at, fewest tiles of a chunk
  int slots;              // bound on the items of split sequences: the workspace's parts
  bool read_once;         // no two row tiles read the same keys
  bool by_length;         // more items than places: the longer rests first
  bool small_sum;         // the tiles of all row tiles stay below 2^31
  float* ws;        // partial results of split sequences

  // Of masked calls alone.  Window: the queries of a sequence are its last tokens, and the one at position p sees the keys
  // j <= p that are later than p - window or before `sinks`.  Prefix and rest: qvx_attn_shared's two parts; whole: all of it at
  // once, each sequence reading the shared keys for itself.
  int mode;
  int window, sinks;
  int table_page;  // many rows: tokens of a page, page_size then standing for the longest sequence
  bool in_order;   // the scale is positive and not tiny: the largest product is the largest logit
  const int32_t *groups, *shared;  // prefix: "sequence" g is the group of queries groups[g] .. and its first shared[g] keys
  int n_groups;                    // whole
  struct AttnLead* leads;          // [queries]: what the prefix leaves the rest
  const float* lead_ws;            // rest: the prefix's workspace
  int lead_rows, lead_slots;       // its tile_rows and slots
  int* arrived;                    // [queries][rest_tiles][kv_heads]: chunks of the rest that are done, zeroed by the prefix
  int rest_tiles;                  // row tiles of a query in the rest
};
enum { kNoMask, kMaskWindow, kMaskPrefix, kMaskRest, kMaskWhole };

// Of a query behind a shared prefix: how many of the prefix's keys it sees, its first row in its group, and where the partial
// results of that group lie.
struct AttnLead {
  int32_t start, row, slot0, chunks;
};

// What k_attn_join needs to know of a split sequence's item.
struct AttnPiece {
  int32_t q0, row0, rows, chunk, chunks, pad[3];
};

// Floats of the workspace per item of a split sequence and key / value head, head_dim rounded up to a
// multiple of 16: the rows' values, maxima and sums.
__host__ __device__ inline size_t attn_part(int rows, int d16) { return (size_t)rows * (d16 + 4); }

// The partition's bounds.  A chunk has C = max(min_chunk, sum / target) tiles, so sequences give at
// most target items more than they have row tiles, and those of several chunks, each less than twice
// its share, at most 2 target in all: the workspace holds no more, however many sequences there are.
// It begins with the number of those items and a piece for each.
__host__ __device__ inline AttnPiece* attn_pieces(float* ws) { return reinterpret_cast<AttnPiece*>(ws) + 1; }
__host__ __device__ inline float* attn_parts(float* ws, int slots) {
  return reinterpret_cast<float*>(attn_pieces(ws) + slots);
}

__device__ inline int attn_tiles(const AttnCall& c, int len) {
  const int full = len / c.page_size;
  return full * c.page_tiles + (len - full * c.page_size + kAttnTile - 1) / kAttnTile;
}

// One work item: rows [row0, row0 + R) of sequence seq over tiles [tile0, tile1); `chunk` of `chunks`.
struct AttnItem {
  bool any;
  int seq, len, q0, rows, row0;  // q0: the sequence's first query; rows: of the whole sequence
  int chunk, chunks, tile0, tile1;
  int slot;  // its place in the workspace, if chunks > 1
  int lead, start;  // whole: the sequence that holds its first `start` keys, or ~ its group; prefix: that sequence
};

struct AttnSeq {
  int len, q0, nq, row_tiles, tiles;
  int lead, start;  // whole
};

// The tile that key `at` lies in.
__device__ inline int attn_tile_of(const AttnCall& c, int at) {
  const int full = at / c.page_size;
  return full * c.page_tiles + (at - full * c.page_size) / kAttnTile;
}

// Tiles that `keys` keys in a row touch at most, wherever they begin: x + y keys touch at most one tile more than x and y keys
// from a page's start (a page's last tile may be short), and the first of them may begin inside a tile.
__host__ __device__ inline long long attn_most_tiles(int page_size, int page_tiles, long long keys) {
  return keys / page_size * page_tiles + (keys % page_size + kAttnTile - 1) / kAttnTile + 2;
}
// Queries of a row tile at most.
__host__ __device__ inline int attn_span(int rows, int group) { return (rows + group - 2) / group + 1; }

// A masked call's sequences.
template <int R, int M> __device__ inline AttnSeq attn_masked_seq(const AttnCall& c, int b) {
  AttnSeq s{};
  if constexpr (M == kMaskPrefix) {
    s.q0 = b && c.groups ? min(max(c.groups[b], 0), c.n_q) : 0;
    s.nq = max((b + 1 < c.n_seqs && c.groups ? min(max(c.groups[b + 1], 0), c.n_q) : c.n_q) - s.q0, 0);
    s.len = min(max(c.shared[b], 0), c.max_len);
    s.tiles = attn_tiles(c, s.len);
  } else {
    s.len = min(max(c.lens[b], 0), c.max_len);
    if constexpr (M == kMaskWhole) {
      s.q0 = b;
      s.nq = 1;
      int g = 0, end = c.groups ? c.n_groups : 1;  // the last group that begins at b or before
      while (end - g > 1) {
        const int mid = (g + end) / 2;
        if (c.groups[mid] <= b) g = mid; else end = mid;
      }
      const int first = g ? min(max(c.groups[g], 0), c.n_seqs - 1) : 0, keys = min(max(c.shared[g], 0), c.max_len);
      s.lead = c.lens[first] >= keys ? first : ~g;
      s.start = min(keys, s.len);
      // the tile in which the shared keys end stands for both parts
      s.tiles = attn_tiles(c, s.start) + (s.len > s.start ? attn_tiles(c, s.len) - attn_tile_of(c, s.start) : 0);
    } else if constexpr (M == kMaskRest) {
      s.q0 = b;
      s.nq = 1;
      const int start = min(max(c.leads[b].start, 0), s.len);
      s.tiles = s.len > start ? attn_tiles(c, s.len) - attn_tile_of(c, start) : 0;
    } else {
      s.q0 = c.q_offsets ? min(max(c.q_offsets[b], 0), c.n_q) : b * c.q_each;
      s.nq = c.q_offsets ? max(min(max(c.q_offsets[b + 1], 0), c.n_q) - s.q0, 0) : c.q_each;
      s.tiles = attn_tiles(c, s.len);  // a row tile may see fewer: its chunks end there, or are empty
      if (c.window < s.len) {
        const long long near = (long long)c.window + min(attn_span(R, c.group), s.nq) - 1;
        const long long most =
            attn_tiles(c, min(c.sinks, s.len)) + attn_most_tiles(c.page_size, c.page_tiles, max(near, 0ll));
        s.tiles = (int)min((long long)s.tiles, most);
      }
    }
  }
  s.row_tiles = (s.nq * c.group + R - 1) / R;
  return s;
}

// R: query rows of a row tile, M: the call's mode, here and below.
template <int R, int M> __device__ inline AttnSeq attn_seq(const AttnCall& c, int b) {
  AttnSeq s{};
  if (b >= c.n_seqs) return s;
  if constexpr (M != kNoMask) return attn_masked_seq<R, M>(c, b);
  int len = c.lens ? c.lens[b] : c.max_len;
  s.len = min(max(len, 0), c.max_len);
  if (c.q_offsets) {  // clamped to the rows that the host vouches for
    s.q0 = min(max(c.q_offsets[b], 0), c.n_q);
    s.nq = max(min(max(c.q_offsets[b + 1], 0), c.n_q) - s.q0, 0);
  } else {
    s.q0 = b * c.q_each;
    s.nq = c.q_each;
  }
  s.row_tiles = (s.nq * c.group + R - 1) / R;
  s.tiles = attn_tiles(c, s.len);
  return s;
}

// Tiles of a chunk: the same for every sequence, so that no workgroup has more than its share.
__device__ inline int attn_chunk(const AttnCall& c, long long total) {
  const long long per = (total + c.target - 1) / c.target;
  return (int)min(max((long long)c.min_chunk, (per + 3) / 4 * 4), 0x7ffffff0ll);
}

// A sequence's items: row_tiles times its chunks of C tiles (kind 0), and row_tiles times one shorter rest (an empty
// sequence has one, which writes zeros).  All sequences' full chunks come first and then the rests, those of more
// than three quarters of a chunk (of the longest sequence, where that is less) before those of more than a half and
// so on (kinds 1 to 4), so that the last items to start are short: 48 sequences of 1 to 8192 tokens 47.4 us
// against 51.8 with the rests in the order of the sequences.  Where all items find a place at once that order
// stays (kind 1).  `slots` is the sequence's share of the workspace.
constexpr int kAttnKinds = 5;
// Whether every item leaves a partial result, split or not.
template <int M> __device__ constexpr bool attn_parts_always() { return M == kMaskPrefix; }
struct AttnCount {
  int full, rest, kind, slots;  // rest: row_tiles or 0, of that kind
  __device__ int items(int k) const { return k == 0 ? full : k == kind ? rest : 0; }
};
template <int M> __device__ inline AttnCount attn_count(const AttnCall& c, const AttnSeq& s, int chunk) {
  const int full = s.tiles / chunk, left = s.tiles - full * chunk, rest = left > 0 || s.tiles == 0 ? 1 : 0;
  const int quarter = min(chunk, c.most_tiles) / 4;
  const int kind = c.by_length ? 1 + (left <= 3 * quarter) + (left <= 2 * quarter) + (left <= quarter) : 1;
  return {s.row_tiles * full, s.row_tiles * rest, kind, full + rest > 1 || attn_parts_always<M>() ? s.row_tiles * (full + rest) : 0};
}

// Item i of sequence b's full (or else short) ones; slot0: its first slot.
template <int R, int M>
__device__ inline AttnItem attn_take(const AttnCall& c, const AttnSeq& s, int b, int chunk, int i, bool full, int slot0) {
  AttnItem it;
  it.seq = b;
  it.len = s.len;
  it.q0 = s.q0;
  it.chunks = max((s.tiles + chunk - 1) / chunk, 1);
  const int whole = s.tiles / chunk;
  int rt = full ? i / max(whole, 1) : i;
  it.chunk = full ? i - rt * whole : whole;
  it.rows = s.nq;
  // Later queries see more keys: their row tiles come first.
  if (M == kMaskWindow) rt = (s.nq + R - 1) / R - 1 - rt;
  it.row0 = rt * R;
  it.tile0 = it.chunk * chunk;
  it.tile1 = min(it.tile0 + chunk, s.tiles);
  it.slot = slot0 + rt * it.chunks + it.chunk;
  it.lead = s.lead;
  it.start = s.start;
  // Offsets that are no running sums can wrap the counts: nothing past the rows or the workspace then.
  it.any = i >= 0 && it.row0 >= 0 && it.row0 < it.rows && it.tile0 >= 0 &&
           ((it.chunks == 1 && !attn_parts_always<M>()) || (unsigned)it.slot < (unsigned)c.slots);
  return it;
}

// Sum over the lanes up to this one (lane 63: of all).
__device__ inline int attn_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // from 1, 2, 4, 8 lanes to the left in each sixteen
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 to the next sixteen, of each two
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
  return x;
}

// A value that is the same in all lanes, as one that the compiler knows to be.
__device__ inline long long attn_uniform(long long x) {
  return (long long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}

// Of the whole call: items of split sequences, and tiles (a row tile's each).
struct AttnSums {
  int slots;
  long long tiles;
};

// The work item of number `item`, the same in every thread of the workgroup (256 threads); `lds`:
// 48 words that the caller does not use across the call.
// Sequences that fit a wave are looked through by every wave for itself, more by the workgroup together.
template <int R, int M> __device__ inline AttnItem attn_item(const AttnCall& c, int item, int* lds, AttnSums& sums) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  AttnItem none{};
  if (c.n_seqs <= 64) {
    const AttnSeq s = attn_seq<R, M>(c, lane);
    long long total;
    if (c.small_sum) {
      total = __builtin_amdgcn_readlane(attn_scan(s.row_tiles * s.tiles), 63);
    } else {
      total = (long long)s.row_tiles * s.tiles;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
    }
    sums.tiles = attn_uniform(total);
    const int chunk = attn_chunk(c, sums.tiles);
    const AttnCount n = attn_count<M>(c, s, chunk);
    int slots = 0, i = item, kind = 1, mine, run;
    sums.slots = 0;
    if (c.ws) {  // without a workspace no sequence is split: rests alone
      kind = 0;
      slots = attn_scan(n.slots);
      sums.slots = __builtin_amdgcn_readlane(slots, 63);
    }
    unsigned long long past = 0;
#pragma unroll 1
    for (;;) {  // one kind after the other: a loop, as every workgroup begins by fetching this code
      mine = n.items(kind);
      run = attn_scan(mine);
      past = __ballot(run > i);
      const int total = __builtin_amdgcn_readlane(run, 63);
      if (past || kind == kAttnKinds - 1) break;
      i -= total;
      ++kind;
    }
    if (!past) return none;
    const int b = __builtin_ctzll(past);
    AttnSeq t;
    t.len = __builtin_amdgcn_readlane(s.len, b);
    t.q0 = __builtin_amdgcn_readlane(s.q0, b);
    t.nq = __builtin_amdgcn_readlane(s.nq, b) * c.group;
    t.tiles = __builtin_amdgcn_readlane(s.tiles, b);
    t.lead = M == kMaskWhole ? __builtin_amdgcn_readlane(s.lead, b) : 0;
    t.start = M == kMaskWhole ? __builtin_amdgcn_readlane(s.start, b) : 0;
    return attn_take<R, M>(c, t, b, chunk, i - __builtin_amdgcn_readlane(run - mine, b), kind == 0,
                        __builtin_amdgcn_readlane(slots - n.slots, b));
  }
  // Every thread takes a run of sequences; the runs' sums are scanned through LDS.
  const int per = (c.n_seqs + 255) / 256;
  const int b0 = (int)threadIdx.x * per, b1 = min(b0 + per, c.n_seqs);
  // Up to 256 sequences are looked at once, each by its thread, the item found handed on: 200 of 84 tokens 31.1
  // us, where every look loads them again 32.8.
  const AttnSeq first = attn_seq<R, M>(c, b0);
  auto of = [&](int b) { return b == b0 ? first : attn_seq<R, M>(c, b); };
  long long total = 0;
  for (int b = b0; b < b1; ++b) {
    const AttnSeq s = of(b);
    total += (long long)s.row_tiles * s.tiles;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
  long long* parts = reinterpret_cast<long long*>(lds);
  if (lane == 0) parts[wave] = total;
  __syncthreads();
  sums.tiles = attn_uniform(parts[0] + parts[1] + parts[2] + parts[3]);
  const int chunk = attn_chunk(c, sums.tiles);
  int items[kAttnKinds] = {}, own = 0;  // own: slots of this thread's sequences
  for (int b = b0; b < b1; ++b) {
    const AttnCount x = attn_count<M>(c, of(b), chunk);
#pragma unroll
    for (int k = 0; k < kAttnKinds; ++k) items[k] += x.items(k);
    own += x.slots;
  }
  int upto[kAttnKinds], slots = attn_scan(own), i = item, kind = 0;
  int* words = lds + 8;  // [kind, and slots][wave], then the item's three
#pragma unroll
  for (int k = 0; k < kAttnKinds; ++k) {
    upto[k] = attn_scan(items[k]);
    if (lane == 63) words[4 * k + wave] = upto[k];
  }
  if (lane == 63) words[4 * kAttnKinds + wave] = slots;
  int* found = words + 4 * (kAttnKinds + 1);
  if (threadIdx.x == 0) found[0] = -1;
  __syncthreads();
  int run = 0, mine = 0;
#pragma unroll
  for (int k = 0; k <= kAttnKinds; ++k) {
    int total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w == wave) before = total;
      total += words[4 * k + w];
    }
    total = __builtin_amdgcn_readfirstlane(total);
    if (k == kAttnKinds) {
      sums.slots = total;
      slots += before;
    } else if (kind == k) {
      if (k < kAttnKinds - 1 && i >= total)
        i -= total, kind = k + 1;
      else
        run = upto[k] + before, mine = items[k];
    }
  }
  if (i >= run - mine && i < run) {
    int before = run - mine, slot0 = slots - own;
    for (int b = b0; b < b1; ++b) {
      const AttnSeq s = of(b);
      const AttnCount x = attn_count<M>(c, s, chunk);
      const int here = x.items(kind);
      if (i < before + here) {
        found[0] = b;
        found[1] = i - before;
        found[2] = slot0;
        found[3] = s.len;
        found[4] = s.q0;
        found[5] = s.nq;
        found[6] = s.tiles;
        found[7] = s.lead;
        found[8] = s.start;
        break;
      }
      before += here;
      slot0 += x.slots;
    }
  }
  __syncthreads();
  auto word = [&](int i) { return __builtin_amdgcn_readfirstlane(found[i]); };
  const int b = word(0), at = word(1), slot0 = word(2);
  if (b < 0) return none;
  AttnSeq s{word(3), word(4), word(5) * c.group, 0, word(6), 0, 0};
  if constexpr (M == kMaskWhole) s.lead = word(7), s.start = word(8);
  return attn_take<R, M>(c, s, b, chunk, at, kind == 0, slot0);
}

// What a row tile of a masked call sees: tiles [0, sinks) and [first, end) of its sequence, ordinals one behind the other, and
// the keys [low, high) and [0, sink_keys) that any of its rows sees.
struct AttnView {
  int p0;  // window: the first query's position
  int sinks, first, end;
  int low, high, sink_keys;
  __device__ int tiles() const { return sinks + max(end - first, 0); }
  __device__ int tile(int t) const { return t < sinks ? t : t - sinks + first; }
};
template <int R, int M> __device__ inline AttnView attn_view(const AttnCall& c, const AttnItem& it) {
  AttnView v{0, 0, 0, 0, 0, it.len, 0};
  if constexpr (M == kMaskWhole) {  // tiles of the shared keys, then the sequence's own
    v.low = it.start;
    v.first = attn_tile_of(c, it.start);
    v.sinks = attn_tiles(c, it.start);
    v.end = it.len > it.start ? attn_tiles(c, it.len) : v.first;
    return v;
  } else if constexpr (M == kMaskRest) {
    v.low = min(max(c.leads[it.seq].start, 0), it.len);
    v.first = attn_tile_of(c, v.low);
  } else if constexpr (M == kMaskWindow) {
    const int nq = it.rows / c.group, qa = it.row0 / c.group, qb = (min(it.row0 + R, it.rows) - 1) / c.group;
    v.p0 = it.len - nq;
    v.high = max(v.p0 + qb + 1, 0);
    // from the first row's first key to the last row's last: a row's keys end where the next one's begin, or later, but for a
    // window of 0, of which no row sees any
    v.low = c.window ? (int)min(max((long long)v.p0 + qa + 1 - c.window, 0ll), (long long)v.high) : v.high;
    v.sink_keys = min(c.sinks, v.high);
    v.first = attn_tile_of(c, v.low);
    v.sinks = attn_tiles(c, v.sink_keys);
    if (v.sinks >= v.first) v.first = v.sinks = 0;
  }
  v.end = v.high > v.low || v.first == 0 ? attn_tiles(c, v.high) : v.first;
  return v;
}
// A group's shared keys are read from the pages of the first of its sequences that holds most of them, hardly ever another than
// the first of all, and end where that one does: what stands behind it is no sequence's.  Each wave looks for itself.
struct AttnHolder {
  int row, keys;
};
__device__ inline AttnHolder attn_holder(const AttnCall& c, int first, int end, int keys) {
  AttnHolder h{first, min(max(c.lens[first], 0), keys)};
  const int lane = threadIdx.x & 63;
  for (int b0 = first + 1; b0 < end && h.keys < keys; b0 += 64) {
    const int here = b0 + lane < end ? min(max(c.lens[b0 + lane], 0), keys) : 0;
    int most = here;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) most = max(most, __shfl_xor(most, x));
    most = __builtin_amdgcn_readfirstlane(most);
    if (most > h.keys) h = {b0 + (int)__builtin_ctzll(__ballot(here == most)), most};
  }
  return {__builtin_amdgcn_readfirstlane(h.row), __builtin_amdgcn_readfirstlane(h.keys)};
}
// Where the item's shared keys are.
template <int M> __device__ inline void attn_held(const AttnCall& c, AttnItem& it) {
  if constexpr (M == kMaskPrefix) {
    const AttnHolder h = attn_holder(c, it.q0, it.q0 + it.rows / c.group, it.len);
    it.lead = h.row;
    it.len = h.keys;
  } else if (it.lead < 0) {
    const int g = ~it.lead, end = g + 1 < c.n_groups && c.groups ? min(max(c.groups[g + 1], 0), c.n_seqs) : c.n_seqs;
    const int first = g ? min(max(c.groups[g], 0), c.n_seqs - 1) : 0;
    it.lead = attn_holder(c, first, end, min(max(c.shared[g], 0), c.max_len)).row;
  }
}
// The keys that one row sees: those of [low, high) and of [0, sinks).
struct AttnRange {
  int low, high, sinks;
  __device__ bool sees(int key) const { return (key >= low || key < sinks) && key < high; }
};
template <int M>
__device__ inline AttnRange attn_range(const AttnCall& c, const AttnItem& it, const AttnView& v, int row) {
  if (row >= it.rows) return {0, 0, 0};
  const int query = row / c.group;
  if constexpr (M == kMaskPrefix) return {0, min(max(c.lens[it.q0 + query], 0), it.len), 0};
  if constexpr (M == kMaskRest || M == kMaskWhole) return {v.low, it.len, 0};
  const int p = v.p0 + query;
  return {(int)max((long long)p + 1 - c.window, 0ll), max(p + 1, 0), c.sinks};
}

// Leaves the rest what it needs of the prefix, and its counters at zero: by a row tile's first chunk, for the queries whose
// first row it holds.
template <int R>
__device__ inline void attn_leads(const AttnCall& c, const AttnItem& it, int kvh) {
  if (kvh != 0 || it.chunk != 0) return;
  const int first = (it.row0 + c.group - 1) / c.group, end = (min(it.row0 + R, it.rows) + c.group - 1) / c.group;
  for (int q = first + (int)threadIdx.x; q < end; q += (int)blockDim.x)
    c.leads[it.q0 + q] = AttnLead{min(max(c.lens[it.q0 + q], 0), it.len), q * c.group,
                                  it.slot - it.row0 / R * it.chunks, it.chunks};
  const int each = c.rest_tiles * c.kv_heads;
  for (int64_t e = (int64_t)(it.q0 + first) * each + threadIdx.x; e < (int64_t)(it.q0 + end) * each; e += blockDim.x)
    c.arrived[e] = 0;
}

// Leaves the join what it needs: the number of pieces, and this item's if it is one (of one head, as all
// heads' are alike).
__device__ inline void attn_note(const AttnCall& c, const AttnItem& it, int item, int kvh, const AttnSums& sums) {
  if (!c.ws || kvh != 0 || threadIdx.x != 0) return;
  if (item == 0) *reinterpret_cast<int*>(c.ws) = min(sums.slots, c.slots);
  if (it.any && it.chunks > 1) attn_pieces(c.ws)[it.slot] = AttnPiece{it.q0, it.row0, it.rows, it.chunk, it.chunks, {}};
}

}  // namespace qvx
