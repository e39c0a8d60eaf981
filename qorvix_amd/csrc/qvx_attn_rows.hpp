// qvx_attn_rows.hpp -- attention of many query rows over a paged 16-bit cache on gfx950's matrix cores, rows seeing parts of
// their sequence's keys: the kernel behind qvx_attn_window and behind qvx_attn_shared's prefixes for more than 16 rows.
//
//   out[row] = sum_j p_j v_j / sum_j p_j over the keys j that the row sees,  p_j = 2^(s_j - m),  s_j = scale log2(e) q[row] . k_j
//
// as in qvx_attn16.hip (128 rows a workgroup, 32 a wave, or 64 in two groups of waves that take other keys and join at the end;
// S^T = K Q^T and O^T = V^T P^T on the 32x32x16 instruction; K and V tiles staged in LDS, the next one in flight).  What is
// different:
//
// Pages.  The keys' offsets are looked up 1024 at a time, half a block ahead, and stand in LDS, so a page may hold any
// number of tokens.  Tiles are copied to LDS straight from the pages, NB - 1 tiles ahead.
//
// Masks.  The tiles of sixteen keys that any row of the tile sees are numbered one behind the other (AttnView), first tokens
// before the window, so a row's keys are two ranges of numbers.  Tiles that all rows of a wave see whole take the
// unmasked path, tiles that none sees are passed over, and keys that no row sees are zeros, whatever the page holds.
//
// Precision.  Queries of the cache's own type are multiplied as they are and the weights rounded to that type (PARTS
// false).  Others, fp32 above all, go in 16-bit parts (AttnQuery's: two of fp16, three of bf16, which leave 2^-23 and nothing), and
// so do the weights: two parts, which leave 2^-22 (fp16) or 2^-18 (bf16) of a weight.  The products of 16-bit values are
// exact and all sums fp32, so the matrix cores do two to three times the work, an eighth of what fp32 instructions would take.
//
// Measured, 32 query and 8 key / value heads of 128, bf16, where a large product reaches 1155 TFLOP/s: a prompt of 8192 tokens 650
// us (847 TFLOP/s; the matrix instructions busy a third of the cycles), with fp32 queries 1240; three pieces of up to 2500 tokens
// behind a window of 1024 84 us (510: 688 workgroups on 512 places, and a start of three dependent loads, lengths, table, keys,
// before the first product, some 7 us each), with fp32 queries 145; 64 fp32 queries of 4 heads a group over 8192 shared fp16 keys 35
// us, the matrix instructions busy 6.8 of them.  Few rows of many sequences are bound by memory: 64 sequences of 16000 fp16 tokens
// and 5 new ones 696 us (4.2 GB, 6.0 TB/s).
#pragma once

#include "qvx_attn_split.hpp"

#include <utility>

namespace qvx {

namespace rows {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

constexpr float kSlackRows = 8.0f;
template <uint32_t T> constexpr float kUpRows = T == T_F16 ? 15.0f : 0.0f;

typedef __attribute__((address_space(3))) uint8_t* LdsPtr;

template <uint32_t T> __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (T == T_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <uint32_t T> __device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (T == T_F16) {
    const f16x2 h = {(_Float16)x, (_Float16)y};
    return __builtin_bit_cast(uint32_t, h);
  } else {
    const bf16x2 h = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, h);
  }
}
// What is left of x and y beside their rounded values in w.
template <uint32_t T> __device__ __forceinline__ void leave(float& x, float& y, uint32_t w) {
  if constexpr (T == T_F16) {
    asm("" : "+v"(w));  // read back, in one instruction a value: left to itself the compiler rounds x and y again
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    x = __builtin_fmaf((float)h.x, -1.0f, x), y = __builtin_fmaf((float)h.y, -1.0f, y);
  } else {
    x -= __builtin_bit_cast(float, w << 16), y -= __builtin_bit_cast(float, w & 0xffff0000u);
  }
}

// DP: head_dim rounded up to a multiple of 32; KT: keys of a tile.  Swizzled as in qvx_attn16.hip.
template <int DP, int KT> struct Tile {
  static constexpr int kPitch = 2 * DP, kUnits = DP / 8, kBanks = kPitch / 4 % 64, kBytes = KT * kPitch;
  static constexpr int kLoads = (KT * kUnits + 255) / 256;  // 16-byte units a thread stages
  // The slot of row r that holds unit u, and the unit that slot u holds.
  static __device__ __forceinline__ int k_unit(int r, int u) {
    return u ^ (kBanks == 0 ? r & 15 : kBanks == 32 ? (r >> 1) & 7 : (r >> 2) & 3);
  }
  static __device__ __forceinline__ int v_unit(int r, int u) {
    return u ^ 4 * (kBanks == 0 ? r & 3 : kBanks == 32 ? (r >> 1) & 1 : 0);
  }
  static __device__ __forceinline__ int k_at(int r, int u) { return r * kPitch + 16 * k_unit(r, u); }
  static __device__ __forceinline__ int v_at(int r, int u) { return r * kPitch + 16 * v_unit(r, u); }
};

constexpr int kBlock = 1024;  // keys whose offsets are looked up together

// Waits until at most N copies to LDS are on their way.
template <int N> __device__ __forceinline__ void wait_copies() {
  static_assert(N < 64);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Everyone's LDS accesses done, and nothing moved past it.
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int N, class F> __device__ __forceinline__ void unrolled(F f) {
  [&]<int... I>(std::integer_sequence<int, I...>) __attribute__((always_inline)) {
    (f.template operator()<I>(), ...);
  }(std::make_integer_sequence<int, N>{});
}

// The second product's left operand for N x 32 values: of each two transposing reads, OFF and OFF + STEP bytes behind an LDS
// address.  Read and waited for in one piece: before a transposing read of its own the compiler would wait for every copy to
// LDS that is on its way.
template <int N, int OFF, int STEP> __device__ __forceinline__ void read_values(u32x4 (&v)[N], const uint32_t (&a)[N]) {
  static_assert(OFF + STEP < 65536);
  u32x2 l[N], h[N];
#define QVX_TR(o, at) "ds_read_b64_tr_b16 %" #o ", %" #at
#define QVX_LO(o, at, n) QVX_TR(o, at) " offset:%" #n "\n\t"
  if constexpr (N == 1)
    asm volatile(QVX_LO(0, 2, 3) QVX_LO(1, 2, 4) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(l[0]), "=&v"(h[0])
                 : "v"(a[0]), "n"(OFF), "n"(OFF + STEP)
                 : "memory");
  else if constexpr (N == 2)
    asm volatile(QVX_LO(0, 4, 6) QVX_LO(1, 4, 7) QVX_LO(2, 5, 6) QVX_LO(3, 5, 7) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(l[0]), "=&v"(h[0]), "=&v"(l[1]), "=&v"(h[1])
                 : "v"(a[0]), "v"(a[1]), "n"(OFF), "n"(OFF + STEP)
                 : "memory");
  else if constexpr (N == 3)
    asm volatile(QVX_LO(0, 6, 9) QVX_LO(1, 6, 10) QVX_LO(2, 7, 9) QVX_LO(3, 7, 10) QVX_LO(4, 8, 9) QVX_LO(5, 8, 10)
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(l[0]), "=&v"(h[0]), "=&v"(l[1]), "=&v"(h[1]), "=&v"(l[2]), "=&v"(h[2])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "n"(OFF), "n"(OFF + STEP)
                 : "memory");
  else
    asm volatile(QVX_LO(0, 8, 12) QVX_LO(1, 8, 13) QVX_LO(2, 9, 12) QVX_LO(3, 9, 13) QVX_LO(4, 10, 12) QVX_LO(5, 10, 13)
                 QVX_LO(6, 11, 12) QVX_LO(7, 11, 13) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(l[0]), "=&v"(h[0]), "=&v"(l[1]), "=&v"(h[1]), "=&v"(l[2]), "=&v"(h[2]), "=&v"(l[3]), "=&v"(h[3])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(OFF), "n"(OFF + STEP)
                 : "memory");
#undef QVX_LO
#undef QVX_TR
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = u32x4{l[j][0], l[j][1], h[j][0], h[j][1]};
}

// N 16-byte LDS reads, waited for together: one by one each of them would be waited for before the product that needs it.
template <int N> __device__ __forceinline__ void read_keys(u32x4 (&k)[N], const uint32_t (&a)[N]) {
#define QVX_RD(o, at) "ds_read_b128 %" #o ", %" #at "\n\t"
  static_assert(N == 2 || N == 4 || N == 5 || N == 6 || N == 8);
  if constexpr (N == 2)
    asm volatile(QVX_RD(0, 2) QVX_RD(1, 3) "s_waitcnt lgkmcnt(0)" : "=&v"(k[0]), "=&v"(k[1]) : "v"(a[0]), "v"(a[1]) : "memory");
  else if constexpr (N == 4)
    asm volatile(QVX_RD(0, 4) QVX_RD(1, 5) QVX_RD(2, 6) QVX_RD(3, 7) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
                 : "memory");
  else if constexpr (N == 5)
    asm volatile(QVX_RD(0, 5) QVX_RD(1, 6) QVX_RD(2, 7) QVX_RD(3, 8) QVX_RD(4, 9) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(k[4])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4])
                 : "memory");
  else if constexpr (N == 6)
    asm volatile(QVX_RD(0, 6) QVX_RD(1, 7) QVX_RD(2, 8) QVX_RD(3, 9) QVX_RD(4, 10) QVX_RD(5, 11) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(k[4]), "=&v"(k[5])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5])
                 : "memory");
  else
    asm volatile(QVX_RD(0, 8) QVX_RD(1, 9) QVX_RD(2, 10) QVX_RD(3, 11) QVX_RD(4, 12) QVX_RD(5, 13) QVX_RD(6, 14)
                 QVX_RD(7, 15) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(k[4]), "=&v"(k[5]), "=&v"(k[6]), "=&v"(k[7])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
                 : "memory");
#undef QVX_RD
}

// What keys that are not there are loaded from.
__device__ const uint32_t kZeros[4] __attribute__((aligned(16))) = {0, 0, 0, 0};

// KT: keys of a round, of G groups of waves KT / G each, in 128 / G rows; W: workgroups a CU.
template <uint32_t T, int M, int DP, int KT, int NB, bool PARTS, int W, int G>
__global__ __launch_bounds__(256, W) void k_attn_rows(AttnCall c) {
  using L = Tile<DP, KT>;
  constexpr int kRows = kAttnRows16 / G, KW = KT / G;  // keys of a wave's tile
  constexpr int KS = DP / 16, DB = DP / 32, KB = KW / 32;
  constexpr int QP = !PARTS ? 1 : T == T_F16 ? 2 : 3, PP = PARTS ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_rows[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5, my_rows = 32 * (wave % (4 / G)), my_keys = wave / (4 / G) * KW;
  const int d = c.head_dim, item = (int)blockIdx.x / c.kv_heads, kvh = (int)blockIdx.x - item * c.kv_heads;
  AttnSums sums;
  AttnItem it = attn_item<kRows, M>(c, item, reinterpret_cast<int*>(lds_rows), sums);
  if constexpr (M == kMaskWindow) attn_note(c, it, item, kvh, sums);
  if (!it.any) return;
  if constexpr (M == kMaskPrefix) {
    attn_held<M>(c, it);
    attn_leads<kRows>(c, it, kvh);
  }
  const AttnView view = attn_view<kRows, M>(c, it);
  it.tile1 = min(it.tile1, view.tiles());
  if constexpr (M == kMaskPrefix) it.seq = it.lead;  // the table's row
  __syncthreads();  // the item's words are read before tiles overwrite them
  const LdsPtr lds = (LdsPtr)lds_rows;

  const int row = it.row0 + my_rows + col, my_row = min(row, it.rows - 1);
  const bool live = row < it.rows;
  const int64_t qat = attn_row(c, it.q0, my_row, kvh, c.q_stride);
  // What this lane's row sees, in numbers of keys: [0, first_end) and [low, high); and over the wave's rows.
  const int shift = kAttnTile * (view.first - view.sinks);  // from a number to its key, behind the first tokens' tiles
  const AttnRange range = attn_range<M>(c, it, view, my_row);
  const int first_end = min(range.sinks, range.high), low = range.low - shift;
  const unsigned width = (unsigned)max(range.high - range.low, 0);
  // Over the wave's rows: least_low .. most_high and below most_first some row sees a key, wave_low .. wave_high all do.
  int wave_low = 0, wave_high = 0, most_high = 0, least_low = 0, most_first = 0;
  if constexpr (M == kMaskWindow) {  // they rise with the row
    const int row_a = min(it.row0 + my_rows, it.rows - 1), row_b = min(row_a + 31, it.rows - 1);
    const AttnRange ra = attn_range<M>(c, it, view, row_a), rb = attn_range<M>(c, it, view, row_b);
    least_low = ra.low - shift;
    wave_high = least_low + max(ra.high - ra.low, 0);
    wave_low = rb.low - shift;
    most_high = wave_low + max(rb.high - rb.low, 0);
    most_first = min(rb.sinks, rb.high);
  } else {
    wave_high = most_high = it.len;
    if (!__all(range.high == it.len)) {  // sequences that end inside their prefix
      wave_high = most_high = range.high;
#pragma unroll
      for (int x = 1; x < 32; x *= 2) {
        wave_high = min(wave_high, __shfl_xor(wave_high, x));
        most_high = max(most_high, __shfl_xor(most_high, x));
      }
      wave_high = __builtin_amdgcn_readfirstlane(wave_high);
      most_high = __builtin_amdgcn_readfirstlane(most_high);
    }
  }

  // The chunk's keys by number, in blocks of kBlock whose offsets from the cache's start (-1: no such key) stand in LDS, the
  // next block's looked up in the table while this one is in work: look asks, place leaves what came.
  const int key0 = it.tile0 * kAttnTile, key_end = it.tile1 * kAttnTile;
  const int tiles = max(key_end - key0 + KT - 1, 0) / KT;
  const int32_t* table = c.table + (int64_t)it.seq * c.table_width;
  const int64_t head_at = (int64_t)kvh * c.head_stride;
  int64_t* offsets = reinterpret_cast<int64_t*>(lds_rows + NB * 2 * L::kBytes);  // [2][kBlock]
  constexpr int kLooks = kBlock / 256;
  int page_id[kLooks], page_off[kLooks];
  auto look = [&](int block) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLooks; ++i) {
      const int number = key0 + block * kBlock + 256 * i + tid;
      const int key = number < kAttnTile * view.sinks ? number : number + shift;
      const bool there = number < key_end && key < view.high && (key >= view.low || key < view.sink_keys);
      const int column = there ? key / c.table_page : 0;
      page_off[i] = key - column * c.table_page;
      page_id[i] = there ? table[column] : -1;
    }
  };
  auto place = [&](int block) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLooks; ++i) {
      const bool there = (unsigned)page_id[i] < (unsigned)c.n_pages;
      offsets[(block & 1) * kBlock + 256 * i + tid] =
          there ? page_id[i] * c.page_stride + head_at + (int64_t)page_off[i] * c.pitch : -1;
    }
  };

  // Staging, straight to LDS: the lanes of a wave fill 64 slots of 16 bytes in a row, so the swizzle is in what each of
  // them loads.  Slot e = tid + 256 i of a tile is slot e % kUnits of its key e / kUnits.  Keys that are not there and
  // values past the head's come from the zeros.
  int slot_key[L::kLoads], koff[L::kLoads], voff[L::kLoads];
#pragma unroll
  for (int i = 0; i < L::kLoads; ++i) {
    const int e = tid + 256 * i, r = e / L::kUnits, u = e - r * L::kUnits;
    slot_key[i] = r < KT ? r : 0;
    koff[i] = L::k_unit(r, u) * 8 < d ? 16 * L::k_unit(r, u) : -1;
    voff[i] = L::v_unit(r, u) * 8 < d ? 16 * L::v_unit(r, u) : -1;
  }
  // ask: where tile t's slots come from, by the offsets in LDS, a round before they are copied: nothing waits for them then.
  int64_t from[L::kLoads];
  auto ask = [&](int t) __attribute__((always_inline)) {
    const int64_t* keys = offsets + t * KT % (2 * kBlock);
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) from[i] = keys[slot_key[i]];
  };
  auto fetch = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
      if (KT * L::kUnits % 256 != 0 && 64 * (wave + 4 * i) >= KT * L::kUnits) break;
      const uint8_t* zeros = reinterpret_cast<const uint8_t*>(kZeros);
      const uint8_t* kp = from[i] >= 0 && koff[i] >= 0 ? c.k + from[i] + koff[i] : zeros;
      const uint8_t* vp = from[i] >= 0 && voff[i] >= 0 ? c.v + from[i] + voff[i] : zeros;
      const LdsPtr to = lds + buf * 2 * L::kBytes + 1024 * (wave + 4 * i);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)kp,
                                       (__attribute__((address_space(3))) void*)to, 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)vp,
                                       (__attribute__((address_space(3))) void*)(to + L::kBytes), 16, 0, 0);
    }
  };

  const bool any_row = it.row0 + my_rows < it.rows;  // a wave past the rows only stages
  constexpr uint64_t kAll = KW == 64 ? ~0ull : (1ull << KW) - 1;
  constexpr int kTiles = kBlock / KT;  // of a block
  static_assert(kTiles - NB > kTiles / 2);  // a block is in place a tile before its first one is asked for
  // Copies a wave has on its way at least for each tile behind the next one: the next one has landed when no more are.
  constexpr int kBehind = (NB - 2) * 2 * (KT * L::kUnits / 256);
  // The queries are asked for before anything that waits for the table, and made ready while the first tiles are on their way.
  u32x4 q[QP][KS];
  float x[PARTS ? KS : 1][8];
  if constexpr (!PARTS) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int i = 16 * s + 8 * h;
      q[0][s] = u32x4{0, 0, 0, 0};
      if (live && i < d) {  // element by element where rows are not on 16-byte addresses
        const uint16_t* p = static_cast<const uint16_t*>(c.q) + qat + i;
        if (c.q_wide) {
          q[0][s] = *reinterpret_cast<const u32x4*>(p);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) q[0][s][j] = (uint32_t)p[2 * j] | (uint32_t)p[2 * j + 1] << 16;
        }
      }
    }
  } else {
    int64_t from[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) from[s] = qat + (16 * s + 8 * h < d ? 16 * s + 8 * h : 0);
    attn_load8(x, c.q, from, c.q_type);
  }
  if (tiles > 0) {
    look(0);
    place(0);
    if (tiles > kTiles) look(1);
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NB - 1; ++t)
    if (t < tiles) {
      ask(t);
      fetch(t);
    }
  float mul = c.scale2;  // of a product to a logit in powers of two
  if constexpr (PARTS) {
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[s][j] = live && 16 * s + 8 * h < d ? x[s][j] * c.scale2 : 0.0f;
        top = fmaxf(top, fabsf(x[s][j]));
      }
    top = fmaxf(top, __shfl_xor(top, 32));
    // by a power of two into the range that AttnQuery says
    const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
    const int up = e == 128 ? 0 : (T == T_BF16 ? min(max(e, -10), 60) : 14) - e;
    mul = __builtin_ldexpf(1.0f, -up);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        float a = __builtin_ldexpf(x[s][j], up), b = __builtin_ldexpf(x[s][j + 1], up);
#pragma unroll
        for (int i = 0; i < QP; ++i) {
          const uint32_t w = pack2<T>(a, b);
          q[i][s][j / 2] = w;
          leave<T>(a, b, w);
        }
      }
  }

  // Lane addresses of the transposing reads, as in qvx_attn16.hip; the swizzle of rows sixteen and eight apart is the same.
  constexpr int kV = DB % 4 == 0 ? 4 : DB % 3 == 0 ? 3 : DB % 2 == 0 ? 2 : 1;
  constexpr int kK = QP == 3 && DP >= 128 && KS * KB % 4 == 0 ? 4 : KS * KB % 8 == 0 ? 8 : KS * KB % 6 == 0 ? 6 : KS * KB % 5 == 0 ? 5 : KS * KB % 4 == 0 ? 4 : 2;
  static_assert(KS * KB % kK == 0 && DB % kV == 0);
  const uint32_t key_at = (uint32_t)(uintptr_t)lds + (uint32_t)(my_keys * L::kPitch);
  uint32_t value_at[DB];
#pragma unroll
  for (int e = 0; e < DB; ++e) {
    const int vrow = 4 * h + (lane & 15) / 4, vcol = 32 * e + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
    value_at[e] = (uint32_t)(uintptr_t)(lds + L::kBytes) + (uint32_t)(my_keys * L::kPitch) + L::v_at(vrow, vcol / 8) + 2 * (vcol & 7);
  }

  float m = -INFINITY, l = 0.0f;
  bool saw = false;
  f32x16 acc[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[b][r] = 0.0f;

  // One tile from buffer `buf`; `there`: the keys that are; masked: some row of the wave does not see all of them.
  auto tile = [&](int first, int buf, uint64_t there, bool masked) __attribute__((always_inline)) {
    f32x16 s[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
    unrolled<KS * KB / kK>([&]<int P>() __attribute__((always_inline)) {
      u32x4 k[kK];
      uint32_t from[kK];
#pragma unroll
      for (int j = 0; j < kK; ++j) {  // read (i, b), the b of a step side by side
        const int i = (P * kK + j) / KB, b = (P * kK + j) % KB;
        from[j] = key_at + (uint32_t)(buf * 2 * L::kBytes) + L::k_at(32 * b + col, 2 * i + h);
      }
      read_keys<kK>(k, from);
#pragma unroll
      for (int j = 0; j < kK; ++j) {
        const int i = (P * kK + j) / KB, b = (P * kK + j) % KB;
#pragma unroll
        for (int x = QP - 1; x >= 0; --x) s[b] = mma<T>(k[j], q[x][i], s[b]);
      }
    });
    // The mask alone stands in a branch, which changes the products in place: with two versions of the tile the sums change
    // registers between them.  The products have to be there on either way, and a branch right behind the instruction hides
    // from the compiler what it has to wait for: twenty wait states, one more than it takes.
#pragma unroll
    for (int b = 0; b < KB; ++b) asm volatile("s_nop 15\n\ts_nop 3" : "+v"(s[b]));
    if (masked) {
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const uint32_t mine = (uint32_t)(there >> (32 * b)) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = 32 * b + 8 * (r / 4) + 4 * h + r % 4 + first;
          const bool sees = (key < first_end || (unsigned)(key - low) < width) && (mine >> (8 * (r / 4) + r % 4) & 1);
          s[b][r] = sees ? s[b][r] : -INFINITY;
          saw = saw || sees;
        }
      }
    } else {
      saw = true;
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
    top *= mul;  // mul > 0: the order stays
    if (__any(top > m)) {
      const float both = fmaxf(top, __shfl_xor(top, 32)), now = both > m ? both + kSlackRows : m;
      const float f = m == now ? 1.0f : attn_pow2(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][r] *= f;
    }
    const float ref = m == -INFINITY ? 0.0f : m - kUpRows<T>;
    u32x4 p[PP][KB][2];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        float x = attn_pow2(__builtin_fmaf(s[b][r], mul, -ref));
        float y = attn_pow2(__builtin_fmaf(s[b][r + 1], mul, -ref));
        const uint32_t xy = pack2<T>(x, y);
        p[0][b][r / 8][r / 2 % 4] = xy;
        if constexpr (!PARTS && T == T_BF16) {  // the sum of the weights as rounded: see qvx_attn16.hip
          const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
          l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, xy), one, l, false);
        } else {
          l += x + y;
        }
        if constexpr (PARTS) {
          leave<T>(x, y, xy);
          p[PP - 1][b][r / 8][r / 2 % 4] = pack2<T>(x, y);
        }
      }
    unrolled<2 * KB>([&]<int S>() __attribute__((always_inline)) {  // sixteen keys a step
      constexpr int B = S / 2, N = S % 2;
      unrolled<DB / kV>([&]<int E>() __attribute__((always_inline)) {
        u32x4 v[kV];
        uint32_t from[kV];
#pragma unroll
        for (int j = 0; j < kV; ++j) from[j] = value_at[E * kV + j] + (uint32_t)(buf * 2 * L::kBytes);
        read_values<kV, 16 * S * L::kPitch, 8 * L::kPitch>(v, from);
#pragma unroll
        for (int j = 0; j < kV; ++j)
#pragma unroll
          for (int i = PP - 1; i >= 0; --i) acc[E * kV + j] = mma<T>(v[j], p[i][B][N], acc[E * kV + j]);
      });
    });
  };

  if (NB - 1 < tiles) {
    ask(NB - 1);
    wait_copies<kBehind>();
  } else {
    wait_copies<0>();
  }
  auto whole = [&](int t) __attribute__((always_inline)) {
    return (uint64_t)__ballot(offsets[t * KT % (2 * kBlock) + my_keys + (lane & (KW - 1))] >= 0) & kAll;
  };
  uint64_t there = tiles > 0 ? whole(0) : 0;
  meet();
  // Buffers by number, not by unrolling: constants of several buffers would be held in registers across the loop.
  int buf = 0;
#pragma unroll 1
  for (int t = 0; t < tiles; ++t) {
    const int ahead = t + NB - 1;
    if (ahead < tiles) {
      fetch(buf == 0 ? NB - 1 : buf - 1);  // the buffer that everyone left a barrier ago
      if (ahead + 1 < tiles) ask(ahead + 1);
    }
    const int first = key0 + t * KT + my_keys;
    const uint64_t now = there;
    if (t + 1 < tiles) there = whole(t + 1);
    const bool none =
        !any_row || now == 0 || ((first >= most_high || first + KW <= least_low) && first >= most_first);
    if (!none) tile(first, buf, now, now != kAll || first < wave_low || first + KW > wave_high);
    // In the middle of a block the one before is no longer read, and the next one takes its place.
    if (t % kTiles == kTiles / 2) {
      const int block = t / kTiles + 1;
      if (block * kTiles < tiles) place(block);
      if ((block + 1) * kTiles < tiles) look(block + 1);
    }
    if (ahead < tiles)
      wait_copies<kBehind>();
    else
      wait_copies<0>();
    meet();
    buf = buf == NB - 1 ? 0 : buf + 1;
  }

  l += __shfl_xor(l, 32);
  saw = __shfl_xor((int)saw, 32) || saw;
  if (saw) m = fmaxf(m, kAttnLow);
  if constexpr (G == 2) {  // the second group's sums go to the first one's waves, through the tiles' place
    static_assert(2 * (16 * DB + 2) * 64 * sizeof(float) <= NB * 2 * L::kBytes);
    float* other = reinterpret_cast<float*>(lds_rows) + my_rows / 32 * (16 * DB + 2) * 64 + lane;
    if (my_keys) {
#pragma unroll
      for (int e = 0; e < DB; ++e)
#pragma unroll
        for (int r = 0; r < 16; ++r) other[(16 * e + r) * 64] = acc[e][r];
      other[16 * DB * 64] = m;
      other[(16 * DB + 1) * 64] = l;
    }
    __syncthreads();
    if (my_keys) return;
    const float m1 = other[16 * DB * 64], l1 = other[(16 * DB + 1) * 64], both = fmaxf(m, m1);
    const float base = both == -INFINITY ? 0.0f : both, f0 = attn_pow2(m - base), f1 = attn_pow2(m1 - base);
    m = both;
    saw = both != -INFINITY;  // a group that saw a key stands at kAttnLow or above: the row may have seen the other's alone
    l = l * f0 + l1 * f1;
#pragma unroll
    for (int e = 0; e < DB; ++e)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[e][r] = acc[e][r] * f0 + other[(16 * e + r) * 64] * f1;
  }
  if (!live) return;
  if (it.chunks > 1 || M == kMaskPrefix) {  // a part of the keys
    const int d16 = (d + 15) & ~15, r16 = row - it.row0;
    float* part = attn_parts(c.ws, c.slots) + ((size_t)it.slot * c.kv_heads + kvh) * attn_part(kRows, d16);
    // weights as small as the split kernel's, whose results these are joined with
    const float down = __builtin_ldexpf(kWeight, -(int)kUpRows<T>);
#pragma unroll
    for (int e = 0; e < DB; ++e)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int i = 32 * e + 8 * (r / 4) + 4 * h;
        if (i < d)
          *reinterpret_cast<f32x4*>(part + r16 * d16 + i) =
              f32x4{acc[e][r] * down, acc[e][r + 1] * down, acc[e][r + 2] * down, acc[e][r + 3] * down};
      }
    if (h == 0) {
      part[kRows * d16 + r16] = m;
      part[kRows * (d16 + 1) + r16] = l * down;
    }
    return;
  }
  const float inv = saw ? 1.0f / l : 0.0f;  // no keys: zeros (acc is zero)
  const int64_t oat = attn_row(c, it.q0, row, kvh, c.out_stride);
#pragma unroll
  for (int e = 0; e < DB; ++e)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int i = 32 * e + 8 * (r / 4) + 4 * h;
      if (i >= d) continue;
      if constexpr (PARTS) {
        const float o[4] = {acc[e][r] * inv, acc[e][r + 1] * inv, acc[e][r + 2] * inv, acc[e][r + 3] * inv};
        attn_store4(c.out, oat + i, c.q_type, o);
      } else {
        uint32_t w0 = pack2<T>(acc[e][r] * inv, acc[e][r + 1] * inv), w1 = pack2<T>(acc[e][r + 2] * inv, acc[e][r + 3] * inv);
        asm("" : "+v"(w0), "+v"(w1));  // one product and rounding for both stores: a last bit could depend on the stride
        const u32x2 w = {w0, w1};
        uint16_t* o = static_cast<uint16_t*>(c.out) + oat + i;
        if (c.out_wide) {
          *reinterpret_cast<u32x2*>(o) = w;
        } else {
          o[0] = (uint16_t)w[0], o[1] = (uint16_t)(w[0] >> 16);
          o[2] = (uint16_t)w[1], o[3] = (uint16_t)(w[1] >> 16);
        }
      }
    }
}

template <uint32_t T, int M, int DP, int KT, int NB, bool PARTS, int W, int G = 1>
bool launch(const AttnCall& c, dim3 grid, hipStream_t s) {
  static LdsLimit lim;
  const auto kernel = &k_attn_rows<T, M, DP, KT, NB, PARTS, W, G>;
  constexpr size_t lds = NB * 2 * (size_t)Tile<DP, KT>::kBytes + 2 * kBlock * sizeof(int64_t);
  static_assert(W * lds <= kLdsPerCU);
  if (!lds_ready(reinterpret_cast<const void*>(kernel), lim, lds)) return false;
  kernel<<<grid, 256, lds, s>>>(c);
  return true;
}

// Row tiles of 64 rows, each wave's keys half of a round's.
template <uint32_t T, int M> bool launch_half(const AttnCall& c, bool parts, dim3 grid, hipStream_t s) {
  const int d = c.head_dim;
  if (!parts) {
    if (d <= 32) return launch<T, M, 32, 64, 2, false, 3, 2>(c, grid, s);
    if (d <= 64) return launch<T, M, 64, 64, 2, false, 3, 2>(c, grid, s);
    if (d <= 96) return launch<T, M, 96, 64, 2, false, 2, 2>(c, grid, s);
    if (d <= 128) return launch<T, M, 128, 64, 2, false, 2, 2>(c, grid, s);
    if (d <= 160) return launch<T, M, 160, 64, 2, false, 1, 2>(c, grid, s);
    return launch<T, M, 256, 64, 2, false, 1, 2>(c, grid, s);
  }
  if (d <= 32) return launch<T, M, 32, 64, 2, true, 3, 2>(c, grid, s);
  if (d <= 64) return launch<T, M, 64, 64, 2, true, 2, 2>(c, grid, s);
  if (d <= 96) return launch<T, M, 96, 64, 2, true, 2, 2>(c, grid, s);
  if (d <= 128) return launch<T, M, 128, 64, 2, true, 2, 2>(c, grid, s);
  if (d <= 160) return launch<T, M, 160, 64, 2, true, 1, 2>(c, grid, s);
  return launch<T, M, 256, 64, 2, true, 1, 2>(c, grid, s);
}

// Tiles of 64 keys where the registers reach, of 32 with more of them on their way where queries in parts take two or three
// times as many.
template <uint32_t T, int M> bool launch_dp(const AttnCall& c, bool parts, dim3 grid, hipStream_t s) {
  const int d = c.head_dim;
  if (c.tile_rows == kAttnRows16 / 2) return launch_half<T, M>(c, parts, grid, s);
  if (!parts) {
    if (d <= 32) return launch<T, M, 32, 64, 2, false, 3>(c, grid, s);
    if (d <= 64) return launch<T, M, 64, 64, 2, false, 3>(c, grid, s);
    if (d <= 96) return launch<T, M, 96, 64, 2, false, 2>(c, grid, s);
    if (d <= 128) return launch<T, M, 128, 64, 2, false, 2>(c, grid, s);
    if (d <= 160) return launch<T, M, 160, 32, 3, false, 2>(c, grid, s);
    return launch<T, M, 256, 32, 3, false, 1>(c, grid, s);
  }
  if (d <= 32) return launch<T, M, 32, 64, 2, true, 3>(c, grid, s);
  if (d <= 64) return launch<T, M, 64, 64, 2, true, 2>(c, grid, s);
  if (d <= 96) return launch<T, M, 96, 32, 4, true, 2>(c, grid, s);
  if (d <= 128) return launch<T, M, 128, 32, 4, true, 2>(c, grid, s);
  if (d <= 160) return launch<T, M, 160, 32, 3, true, 1>(c, grid, s);
  return launch<T, M, 256, 32, 3, true, 1>(c, grid, s);
}

template <uint32_t T> bool launch_mode(const AttnCall& c, bool parts, dim3 grid, hipStream_t s) {
  return c.mode == kMaskPrefix ? launch_dp<T, kMaskPrefix>(c, parts, grid, s) : launch_dp<T, kMaskWindow>(c, parts, grid, s);
}

}  // namespace rows

}  // namespace qvx
