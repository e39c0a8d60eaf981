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
constexpr int kAttnWaves = 4;   // waves of a workgroup of the split kernel

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
  const int32_t* table;  // paged: [n_seqs, table_width]; null: sequence b is "page" b
  int table_width, n_pages;
  int page_size;       // tokens of a page (states: the longest sequence)
  int page_tiles;      // tiles of a page
  const int32_t* lens;  // null: every sequence has max_len keys
  int max_len;
  int n_seqs, kv_heads, group, head_dim;
  float scale2;     // scale * log2(e): the kernels work with powers of two
  int tile_rows;    // query rows of a row tile of the split kernel: 4, 8 or 16
  int items;        // bound on the work items of a key / value head (grid x)
  int target, min_chunk;  // work items aimed at, fewest tiles of a chunk
  float* ws;        // partial results of split sequences
};

// Floats of the workspace per item of a split sequence and key / value head, head_dim rounded up to a
// multiple of 16: the rows' values, maxima and sums.
__host__ __device__ inline size_t attn_part(int rows, int d16) { return (size_t)rows * (d16 + 4); }

// The partition's bounds.  A chunk has C = max(min_chunk, sum / target) tiles, so sequences give at
// most target items more than they have row tiles, and those of several chunks, each less than twice
// its share, at most 2 target in all: the workspace holds no more, however many sequences there are.
inline int attn_slots(const AttnCall& c) { return 2 * c.target; }

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
};

struct AttnSeq {
  int len, q0, nq, row_tiles, tiles;
};

// R: query rows of a row tile, here and below.
template <int R> __device__ inline AttnSeq attn_seq(const AttnCall& c, int b) {
  AttnSeq s{0, 0, 0, 0, 0};
  if (b >= c.n_seqs) return s;
  int len = c.lens ? c.lens[b] : c.max_len;
  s.len = min(max(len, 0), c.max_len);
  if (c.q_offsets) {  // clamped to the rows that the host vouches for
    s.q0 = min(max(c.q_offsets[b], 0), c.n_q);
    s.nq = max(min(c.q_offsets[b + 1], c.n_q) - s.q0, 0);
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

template <int R>
__device__ inline AttnItem attn_take(const AttnCall& c, const AttnSeq& s, int b, int chunk, int i, int slot0) {
  AttnItem it;
  it.seq = b;
  it.len = s.len;
  it.q0 = s.q0;
  it.chunks = max((s.tiles + chunk - 1) / chunk, 1);
  const int rt = i / it.chunks;
  it.chunk = i - rt * it.chunks;
  it.rows = s.nq;
  it.row0 = rt * R;
  it.tile0 = it.chunk * chunk;
  it.tile1 = min(it.tile0 + chunk, s.tiles);
  it.slot = slot0 + i;
  // Offsets that are no running sums can wrap the counts: nothing past the rows or the workspace then.
  it.any = i >= 0 && it.row0 < it.rows && (it.chunks == 1 || (unsigned)it.slot < 2u * (unsigned)c.target);
  return it;
}

// The work item of number `item`, the same in every thread of the workgroup (256 threads); `lds`:
// 20 words that the caller does not use across the call.  Sequences that fit a wave are looked
// through by every wave for itself, more by the workgroup together.
template <int R> __device__ inline AttnItem attn_item(const AttnCall& c, int item, int* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (c.n_seqs <= 64) {
    const AttnSeq s = attn_seq<R>(c, lane);
    long long total = (long long)s.row_tiles * s.tiles;
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
      if (d < c.n_seqs) total += __shfl_xor(total, d);
    total = __shfl(total, 0);
    const int chunk = attn_chunk(c, total);
    const int parts = (s.tiles + chunk - 1) / chunk;
    const int mine = s.row_tiles * max(parts, 1), split = parts > 1 ? mine : 0;
    int upto = mine, slots = split;
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
      if (d < c.n_seqs) {
        const int o = __shfl_up(upto, d), p = __shfl_up(slots, d);
        if (lane >= d) upto += o, slots += p;
      }
    const unsigned long long past = __ballot(upto > item);
    AttnItem none{};
    if (!past) return none;
    const int b = __builtin_ctzll(past);
    AttnSeq t;
    t.len = __builtin_amdgcn_readlane(s.len, b);
    t.q0 = __builtin_amdgcn_readlane(s.q0, b);
    t.nq = __builtin_amdgcn_readlane(s.nq, b) * c.group;
    t.tiles = __builtin_amdgcn_readlane(s.tiles, b);
    return attn_take<R>(c, t, b, chunk, item - __builtin_amdgcn_readlane(upto - mine, b),
                     __builtin_amdgcn_readlane(slots - split, b));
  }
  // Every thread takes a run of sequences; the runs' sums are scanned through LDS.
  const int per = (c.n_seqs + 255) / 256;
  const int b0 = (int)threadIdx.x * per, b1 = min(b0 + per, c.n_seqs);
  long long total = 0;
  for (int b = b0; b < b1; ++b) {
    const AttnSeq s = attn_seq<R>(c, b);
    total += (long long)s.row_tiles * s.tiles;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
  long long* sums = reinterpret_cast<long long*>(lds);
  if (lane == 0) sums[wave] = total;
  __syncthreads();
  const int chunk = attn_chunk(c, sums[0] + sums[1] + sums[2] + sums[3]);
  int mine = 0, split = 0;
  for (int b = b0; b < b1; ++b) {
    const AttnSeq s = attn_seq<R>(c, b);
    const int parts = (s.tiles + chunk - 1) / chunk, n = s.row_tiles * max(parts, 1);
    mine += n;
    split += parts > 1 ? n : 0;
  }
  int upto = mine, slots = split;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(upto, d), p = __shfl_up(slots, d);
    if (lane >= d) upto += o, slots += p;
  }
  if (lane == 63) lds[8 + wave] = upto, lds[12 + wave] = slots;
  if (threadIdx.x == 0) lds[16] = -1;
  __syncthreads();
  for (int w = 0; w < wave; ++w) upto += lds[8 + w], slots += lds[12 + w];
  if (item >= upto - mine && item < upto) {
    int first = upto - mine, slot0 = slots - split;
    for (int b = b0; b < b1; ++b) {
      const AttnSeq s = attn_seq<R>(c, b);
      const int parts = (s.tiles + chunk - 1) / chunk, n = s.row_tiles * max(parts, 1);
      if (item < first + n) {
        lds[16] = b;
        lds[17] = item - first;
        lds[18] = slot0;
        break;
      }
      first += n;
      slot0 += parts > 1 ? n : 0;
    }
  }
  __syncthreads();
  const int b = __builtin_amdgcn_readfirstlane(lds[16]), i = __builtin_amdgcn_readfirstlane(lds[17]);
  const int slot0 = __builtin_amdgcn_readfirstlane(lds[18]);
  AttnItem none{};
  if (b < 0) return none;
  AttnSeq s = attn_seq<R>(c, b);
  s.nq *= c.group;
  return attn_take<R>(c, s, b, chunk, i, slot0);
}

}  // namespace qvx
