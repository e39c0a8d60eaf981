// qvx_attn_split.hpp -- attention of few query rows over many keys on gfx950: the kernel behind
// qvx_attn_paged and behind qvx_attn_cross for single tokens and fp32 queries.
//
//   out[row] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q[row] . k_j
//
// for any m, here a running reference that follows the largest s_j seen (below).  The sum is one pass
// over the keys, so the cache is read once and that read bounds the kernel.
//
// Arithmetic: fp32 sums and weights, whatever the cache holds.  The first product takes 16-bit keys as they are
// and the queries in 16-bit parts (below); fp32 keys, and the values of
// every type widened in registers, run on the fp32 matrix instructions (16x16x4, and 4x4x1 for up to eight rows), so
// the weights are never rounded.
//
// Layout.  S^T = K Q^T puts key 4 g + r (g = lane / 16) and row lane % 16 into register r; the second
// product reads its left operand, P, with row lane % 16 and key index g.  So the weights go from one
// product to the next in place, without a lane exchange or LDS, when the values of key 4 g + r are
// loaded by the lanes of group g: 16 lanes cover a token's values in consecutive pieces.
//
// The reference m.  A row's weights may use any common m; it is the row's largest logit (in powers of two) when it is set,
// and set again only when a logit passes it by more than kSlack, which after the first tiles is rare, so a step costs
// a compare and a wave vote instead of a lane reduction and a rescale.  All weights are 2^kSlack smaller than 2^(s_j - m): never
// above 1, the row's largest never below 2^-kSlack.  So their sums stay finite for values of up to fp32's largest number over
// the number of keys, and weights of 2^-100 of the largest are still normal numbers.  The factor follows the power of
// two: taken into m it would cost the exponents near 0 their last five bits (33 keys, an error of 4.3e-7 against 2.1e-7).
//
// Split.  A work item is a chunk of a sequence's tiles (qvx_attn.hpp); its four waves take tiles in
// turn and join through LDS.  Items of a sequence that has several leave their sums, their maxima
// and values in the workspace, and k_attn_join adds them up in the order of the chunks.
//
// Measured, 32 query and 8 key / value heads of 128, where a read of 2 GiB reaches 6.8 TB/s: one sequence of 131071
// tokens in bf16 92 us (5.8 TB/s, the join's 6 in it), 64 of 4096 in Q8_0 104 us (5.5), 128 of 4096 in fp16 345 us (6.2);
// 48 of 1 to 8192 tokens in fp16 47 us (4.2: uneven chunks, and the join).  Calls that do not fill the card are
// bound by latency and by what one CU reads, about 45 GB/s, with four waves as with eight.
#pragma once

#include "qvx_attn.hpp"

#include <algorithm>

namespace qvx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr float kSlack = 20.0f, kWeight = 0x1p-20f;  // 2^-kSlack
constexpr uint32_t kPastEnd = 0x7fffff00u;  // an offset no descriptor reaches: the load gives zeros

// A descriptor of `bytes` bytes from p (the same in all lanes): loads past them give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t attn_rsrc(const uint8_t* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00020000);
}

// N consecutive values of type T, N in 4, 8, 16: the raw words as loaded, and their fp32 values.
template <uint32_t T, int N> struct AttnRaw;

// AUX: the load's cache policy, 0 or kOnce.
constexpr int kOnce = 2;  // non-temporal: will not be read again
template <int W> struct AttnWords {
  uint32_t w[W];
  template <int AUX = 0> __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    if constexpr (W == 1) {
      w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, AUX);
    } else if constexpr (W == 2) {
      const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, AUX);
      w[0] = x[0], w[1] = x[1];
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off + 4 * i, 0, AUX);
        w[i] = x[0], w[i + 1] = x[1], w[i + 2] = x[2], w[i + 3] = x[3];
      }
    }
  }
};

template <int N> struct AttnRaw<T_F32, N> : AttnWords<N> {
  static constexpr int kBytes = 4 * N;
  __device__ __forceinline__ float at(int i, float) const { return __builtin_bit_cast(float, this->w[i]); }
};
template <int N> struct AttnRaw<T_F16, N> : AttnWords<N / 2> {
  static constexpr int kBytes = 2 * N;
  __device__ __forceinline__ float at(int i, float) const {
    const f16x2 h = __builtin_bit_cast(f16x2, this->w[i / 2]);
    return i % 2 ? (float)h.y : (float)h.x;
  }
};
template <int N> struct AttnRaw<T_BF16, N> : AttnWords<N / 2> {
  static constexpr int kBytes = 2 * N;
  __device__ __forceinline__ float at(int i, float) const {
    return __builtin_bit_cast(float, i % 2 ? this->w[i / 2] & 0xffff0000u : this->w[i / 2] << 16);
  }
};
template <int N> struct AttnRaw<T_Q8_0, N> : AttnWords<N / 4> {
  static constexpr int kBytes = N;
  __device__ __forceinline__ float at(int i, float step) const {
    return (float)(int8_t)(this->w[i / 4] >> (8 * (i % 4))) * step;
  }
};

// Eight consecutive elements of a query row at each of N places, on any address of their type.  One branch
// for all of them: a branch a place would wait for each before the next.
template <int N>
__device__ __forceinline__ void attn_load8(float (&x)[N][8], const void* p, const int64_t (&at)[N], uint32_t type) {
  if (type == T_F32) {
    struct __attribute__((packed, aligned(4))) Eight {
      float v[8];
    } e[N];
#pragma unroll
    for (int s = 0; s < N; ++s) e[s] = *reinterpret_cast<const Eight*>(static_cast<const float*>(p) + at[s]);
#pragma unroll
    for (int s = 0; s < N; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] = e[s].v[i];
  } else {
    struct __attribute__((packed, aligned(2))) Eight {
      uint16_t v[8];
    } e[N];
#pragma unroll
    for (int s = 0; s < N; ++s) e[s] = *reinterpret_cast<const Eight*>(static_cast<const uint16_t*>(p) + at[s]);
#pragma unroll
    for (int s = 0; s < N; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[s][i] = type == T_F16 ? (float)__builtin_bit_cast(_Float16, e[s].v[i])
                                : __builtin_bit_cast(float, (uint32_t)e[s].v[i] << 16);
  }
}

// Four consecutive elements of an output row, on any address of their type.
__device__ __forceinline__ void attn_store4(void* p, int64_t at, uint32_t type, const float (&x)[4]) {
  if (type == T_F32) {
    struct __attribute__((packed, aligned(4))) Four {
      float v[4];
    };
    *reinterpret_cast<Four*>(static_cast<float*>(p) + at) = Four{{x[0], x[1], x[2], x[3]}};
  } else {
    struct __attribute__((packed, aligned(2))) Four {
      uint16_t v[4];
    };
    Four f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f.v[i] = type == T_F16 ? __builtin_bit_cast(uint16_t, (_Float16)x[i]) : __builtin_bit_cast(uint16_t, (__bf16)x[i]);
    *reinterpret_cast<Four*>(static_cast<uint16_t*>(p) + at) = f;
  }
}

// Lanes 4 r .. 4 r + 3 of each row of sixteen lanes: x of the lane `shift` to the left (to the right if
// negative); the other lanes keep `old`.
template <int r, int shift> __device__ __forceinline__ int attn_move(int old, float x) {
  constexpr int ctrl = shift == 0 ? 0xe4 : shift > 0 ? 0x110 + shift : 0x100 - shift;
  return __builtin_amdgcn_update_dpp(old, __builtin_bit_cast(int, x), ctrl, 0xf, 1 << r, false);
}

// x of the lane N further to the right in its sixteen, around the end.
template <int N> __device__ __forceinline__ float attn_rotate(float x) {
  const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + N, 0xf, 0xf, false);
  return __builtin_bit_cast(float, y);
}

// Rows 4 t .. 4 t + 3 of the first product, key 4 g + r in register r of lanes 4 t .. 4 t + 3 of each sixteen, to
// key 4 g + r in lanes 4 r .. 4 r + 3.
template <int t> __device__ __forceinline__ float attn_gather(const f32x4& s) {
  int z = attn_move<0, -4 * t>(0, s[0]);
  z = attn_move<1, 4 - 4 * t>(z, s[1]);
  z = attn_move<2, 8 - 4 * t>(z, s[2]);
  z = attn_move<3, 12 - 4 * t>(z, s[3]);
  return __builtin_bit_cast(float, z);
}

// a and b exchange halves between the lanes N apart and are added: the lanes with bit N clear get a + a',
// the others b + b', the stroke marking the other lane's.
template <int N> __device__ __forceinline__ float attn_swap_add(float a, float b) {
  const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
  const u32x2 s = N == 32 ? __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(x, y, false, false))
                          : __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(x, y, false, false));
  // through scalars: a bit cast of a vector's element reads element 0 whichever it names
  const uint32_t s0 = s[0], s1 = s[1];
  return __builtin_bit_cast(float, s0) + __builtin_bit_cast(float, s1);
}

// Element offset of a row's head in q (stride: q_stride) or out.
__device__ __forceinline__ int64_t attn_row(const AttnCall& c, int q0, int row, int kvh, int64_t stride) {
  const int query = row / c.group, head = row - query * c.group;
  return (int64_t)(q0 + query) * stride + (int64_t)(kvh * c.group + head) * c.head_dim;
}

__device__ __forceinline__ float attn_pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// The queries as the first product's right operand, KS pieces of 32 values.  F32: fp32 itself, eight
// values a lane for eight 16x16x4 instructions a piece.  Otherwise 16-bit parts, each multiplied by the keys in its
// own 16x16x32 instruction: bf16 three times (8 + 8 + 8 bits), which add up to the fp32 value; fp16 twice (11 + 11), which
// leave at most 2^-23 of it, as much as the products' own rounding in fp32 and the scale's before them add: a third
// instruction a piece would be a half more of them for less than either.  Products of 16-bit values are exact.  The
// row is first multiplied by a power of two, undone in the exponent.  For fp16 (and Q8_0's integers) to a largest
// magnitude of 2^14, so that no part overflows and the small part of every value that matters stays normal.  bf16
// keys reach as far as fp32: there rows below 2^-10 are brought to that, where 256 products with keys of any size stay
// below 2^127 and the small parts far above 2^-126, and rows above 2^60 to that, where no part rounds to infinity and
// products that matter to a logit stay normal; those between are as they are, and their sums as large as their logits.
template <uint32_t T, int KS> struct AttnQuery {
  typedef _Float16 Key __attribute__((ext_vector_type(8)));
  Key hi[KS], lo[KS];
  __device__ __forceinline__ void set(int s, const float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      hi[s][j] = (_Float16)x[j];
      lo[s][j] = (_Float16)(x[j] - (float)hi[s][j]);
    }
  }
  __device__ __forceinline__ f32x4 mul(int s, Key k, f32x4 c) const {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, lo[s], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(k, hi[s], c, 0, 0, 0);
  }
};
template <int KS> struct AttnQuery<T_BF16, KS> {
  typedef __bf16 Key __attribute__((ext_vector_type(8)));
  Key part[3][KS];
  __device__ __forceinline__ void set(int s, const float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float rest = x[j];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        part[i][s][j] = (__bf16)rest;
        rest -= (float)part[i][s][j];
      }
    }
  }
  __device__ __forceinline__ f32x4 mul(int s, Key k, f32x4 c) const {
#pragma unroll
    for (int i = 2; i >= 0; --i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, part[i][s], c, 0, 0, 0);
    return c;
  }
};
template <int KS> struct AttnQuery<T_F32, KS> {
  float v[KS][8];
  __device__ __forceinline__ void set(int s, const float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[s][j] = x[j];
  }
};

// A tile of 16 keys and their values as loaded: lane (col, g) holds pieces 32 s + 8 g of key col, and
// values col * VB .. of keys 4 g .. 4 g + 3; of Q8_0 also the scales of those four keys' blocks, and of
// the values' block in each of them.  FULL: head_dim is DT, so a key's scales are one load.
//
// Q8_0 for four rows or eight (kGroup): the products of each block have to be summed alone, and sixteen lanes that each
// fetch 8 bytes of another key keep the address units busier than the memory (4.4 TB/s where fp16 reaches
// 5.6).  So a lane group takes whole blocks: NP of them at a time, one for 4 / NP groups, in 16-byte
// loads, and the rows stand NP times among the sixteen columns of the product, each time with the
// values of one group's block and zeros for the others': one instruction chain sums NP blocks apart.
template <uint32_t T, int DT, bool FULL, int NS> struct AttnTile {
  static constexpr int KS = DT / 32, VB = DT / 16, VU = VB < 8 ? VB : 8, VN = VB / VU;
  static constexpr bool kQ8 = T == T_Q8_0, kGroup = kQ8 && NS <= 2;
  static constexpr int kMostNP = 4 / NS, NP = kGroup ? (KS < kMostNP ? KS : kMostNP) : 1, U = KS / NP, J = KS / U, G4 = 4 / NP;
  static constexpr int kRegs = 2 * DT * AttnRaw<T, 8>::kBytes / 32 / 4 +
                               (kGroup ? 4 * U + 4 : kQ8 ? 2 * KS + 4 : 0);  // of a lane
  AttnRaw<T, 8> k[KS];
  AttnRaw<T, VU> v[4][VN];
  // [key r][two blocks' scales a word]; kGroup: [key r][this lane's block of round u]
  uint32_t kstep[kQ8 ? 4 : 1][kGroup ? U : kQ8 ? (KS + 1) / 2 : 1];
  uint16_t vstep[kQ8 ? 4 : 1];
  int live;
};

__device__ __forceinline__ float attn_half(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }

// Values formed here, all of them, before anything that uses them.  Left to itself the compiler converts each
// value right before the matrix instruction that reads it, in one register, and every pair then waits out
// the hazard between the two: two idle slots a value.
template <int N> __device__ __forceinline__ void attn_pin(float (&v)[N]) {
  if constexpr (N == 8)
    asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(v[4]), "+v"(v[5]), "+v"(v[6]), "+v"(v[7]));
  else
    asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
}

// The second product for values 4 g + r of a tile, up to three sets of four rows: 16 blocks of 4 x 4 x 1, the four
// of a lane group all taking the weights of block 4 g + r, that is of the group's key.  Q8_0 up to 128 values:
// what the four lanes of a block hold has one scale, so that goes into the weights, which each block then
// takes for itself, and the values are the integers.
template <int r, int NT, int VN, int VU, bool Q8, class Tile, int VB>
__device__ __forceinline__ void attn_values(f32x4 (&acc)[NT][VB], const float (&p)[NT], const Tile& x) {
  constexpr bool kOwn = Q8 && VB <= 8;  // the values of a block of four lanes, 16 or 32, lie in one 32-value block
  float w[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    w[t] = p[t];
    if constexpr (kOwn)  // lanes 4 r + lane % 4 of the sixteen
      w[t] = __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, p[t]), 4 * r << 5 | 0x13)) *
             attn_half(x.vstep[r]);
  }
  const float vs = Q8 && !kOwn ? attn_half(x.vstep[Q8 ? r : 0]) : 1.0f;
#pragma unroll
  for (int u = 0; u < VN; ++u) {
    float v[VU];
#pragma unroll
    for (int j = 0; j < VU; ++j) v[j] = x.v[r][u].at(j, vs);
    attn_pin(v);
#pragma unroll
    for (int j = 0; j < VU; ++j)
#pragma unroll
      for (int t = 0; t < NT; ++t)
        acc[t][u * VU + j] =
            __builtin_amdgcn_mfma_f32_4x4x1f32(w[t], v[j], acc[t][u * VU + j], kOwn ? 0 : 2, kOwn ? 0 : r, 0);
  }
}

// Eight int8 as fp16: each byte b becomes the fp16 number 1024 + (b + 128), less 1152: exact.
__device__ __forceinline__ AttnQuery<T_F16, 1>::Key attn_bytes(const uint32_t (&w)[2]) {
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = w[i / 2] ^ 0x80808080u;
    const uint32_t h = __builtin_amdgcn_perm(0x64646464u, u, i % 2 ? 0x04030402u : 0x04010400u);
    x[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, h) - f16x2{(_Float16)1152.0f, (_Float16)1152.0f});
  }
  return __builtin_bit_cast(AttnQuery<T_F16, 1>::Key, u32x4{x[0], x[1], x[2], x[3]});
}

// DT: head_dim rounded up to 64, 128 or 256.  T: the type of the keys and values.  NS: sets of four
// rows of a row tile, 1, 2 or 4.
template <uint32_t T, int DT, bool FULL, int NS>
__global__ __launch_bounds__(64 * kAttnWaves, DT == 256 ? 1 : 2) void k_attn_split(AttnCall c) {
  using Tile = AttnTile<T, DT, FULL, NS>;
  constexpr int KS = Tile::KS, VB = Tile::VB, VU = Tile::VU, VN = Tile::VN, R = 4 * NS;
  constexpr int kKeyBytes = AttnRaw<T, 8>::kBytes, kValBytes = AttnRaw<T, VU>::kBytes / VU;
  constexpr bool kQ8 = T == T_Q8_0, kGroup = Tile::kGroup;
  constexpr int NP = Tile::NP, U = Tile::U, J = Tile::J, G4 = Tile::G4;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int d = c.head_dim, item = (int)blockIdx.x / c.kv_heads, kvh = (int)blockIdx.x - item * c.kv_heads;
  AttnSums sums;
  const AttnItem it = attn_item<R>(c, item, reinterpret_cast<int*>(lds), sums);
  attn_note(c, it, item, kvh, sums);
  if (!it.any) return;
  // A call that reads more than half the 256 MB memory-side cache finds nothing of it there again, and its
  // loads are marked so: fp16 of 131071 tokens 102 -> 90 us, 128 x 4096 tokens 377 -> 345.  Smaller calls
  // keep the ordinary policy: 47 MB of fp32 in turn with two others like it 17.5 us against 19.3 with the mark.
  const bool once = c.read_once && sums.tiles * (long long)(2 * kAttnTile) * c.key_bytes * c.kv_heads > (128ll << 20);

  // The wave takes tiles tile0 + wave, + 4, ...; lane i looks up the i-th of them, 64 at a time.
  const int tiles = (it.tile1 - it.tile0 - wave + kAttnWaves - 1) / kAttnWaves;
  const int spitch = kQ8 ? d / 16 : 0;  // bytes of a token's scales
  int64_t at = 0, sat = 0;  // of the tile's keys (and values), and of their scales, from the cache's start
  int live = 0, seen = 0;  // seen: keys that count
  auto look_up = [&](int n) __attribute__((always_inline)) {
    const int t = it.tile0 + wave + (n + lane) * kAttnWaves;
    live = 0;
    if (t < it.tile1) {
      const int p = t / c.page_tiles, tok = (t - p * c.page_tiles) * kAttnTile;
      int page = c.table ? c.table[(int64_t)it.seq * c.table_width + p] : it.seq;
      live = min(min(kAttnTile, c.page_size - tok), it.len - p * c.page_size - tok);
      if (page < 0 || page >= c.n_pages) page = 0, live = 0;  // no such page: its keys do not count
      at = page * c.page_stride + kvh * c.head_stride + (int64_t)tok * c.pitch;
      if constexpr (kQ8) sat = page * c.page_stride + c.scale_off + ((int64_t)kvh * c.page_size + tok) * spitch;
    }
  };
  // A lane's 64-bit value in all of them.
  auto of_lane = [](int64_t x, int i) __attribute__((always_inline)) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)x, i));
  };
  look_up(0);

  // The first of the eight values that this lane's piece s of a key stands for.
  auto piece = [&](int s) __attribute__((always_inline)) {
    return kGroup ? (s / J * NP + g / G4) * 32 + g % G4 * (32 / G4) + 8 * (s % J) : 32 * s + 8 * g;
  };
  uint32_t koff[KS], voff[VN], soff = 0, svoff = 0;
#pragma unroll
  for (int s = 0; s < KS; ++s)
    koff[s] = piece(s) < d ? (uint32_t)(col * c.pitch + piece(s) * kKeyBytes / 8) : kPastEnd;
#pragma unroll
  for (int u = 0; u < VN; ++u) {
    const int i = col * VB + u * VU;
    voff[u] = i < d ? (uint32_t)(4 * g * c.pitch + i * kValBytes) : kPastEnd;
  }
  if constexpr (kQ8) {
    soff = (uint32_t)(4 * g * spitch);
    svoff = col * VB < d ? (uint32_t)(4 * g * spitch + col * VB / 32 * 2) : kPastEnd;
  }
  // Tile n of the wave's, none (and no memory) past the last.
  auto load = [&]<int AUX>(Tile& x, int n) __attribute__((always_inline)) {
    if (n && (n & 63) == 0 && n < tiles) look_up(n);
    x.live = n < tiles ? __builtin_amdgcn_readlane(live, n & 63) : 0;
    seen |= x.live;
    const int64_t ta = of_lane(at, n & 63);
    const uint32_t bytes = (uint32_t)(x.live * c.pitch);
    const __amdgpu_buffer_rsrc_t kr = attn_rsrc(c.k + ta, bytes);
    const __amdgpu_buffer_rsrc_t vr = attn_rsrc(c.v + ta, bytes);
    if constexpr (kGroup) {  // a round's pieces lie side by side
#pragma unroll
      for (int u = 0; u < U; ++u) {
        AttnWords<2 * J> w;
        w.template load<AUX>(kr, koff[u * J]);
#pragma unroll
        for (int i = 0; i < 2 * J; ++i) x.k[u * J + i / 2].w[i % 2] = w.w[i];
      }
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) x.k[s].template load<AUX>(kr, koff[s]);
    }
    if constexpr (kQ8) {
      const int64_t ts = of_lane(sat, n & 63);
      const __amdgpu_buffer_rsrc_t ks = attn_rsrc(c.k + ts, (uint32_t)(x.live * spitch));
      const __amdgpu_buffer_rsrc_t vs = attn_rsrc(c.v + ts, (uint32_t)(x.live * spitch));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (kGroup) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int block = u * NP + col / R;
            x.kstep[r][u] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
                ks, col / R < NP && 32 * block < d ? soff + r * spitch + 2 * block : kPastEnd, 0, 0);
          }
        } else if constexpr (FULL) {
          AttnWords<(KS + 1) / 2> w;
          w.load(ks, soff + r * spitch);
#pragma unroll
          for (int i = 0; i < (KS + 1) / 2; ++i) x.kstep[r][i] = w.w[i];
        } else {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const uint32_t h =
                (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(ks, 32 * s < d ? soff + r * spitch + 2 * s : kPastEnd, 0, 0);
            x.kstep[r][s / 2] = s % 2 ? x.kstep[r][s / 2] | h << 16 : h;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) x.vstep[r] = __builtin_amdgcn_raw_buffer_load_b16(vs, svoff + r * spitch, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int u = 0; u < VN; ++u) x.v[r][u].template load<AUX>(vr, voff[u] + r * c.pitch);
  };
  // Tiles in registers, one in work and one on its way where they fit: 131071 tokens in bf16 103 us against 111 with one.
  // For eight rows of 128 values they do but for 1 to 22 registers (32 x 2000 tokens in bf16, 7 heads of 80 a group, 45 us
  // against 77; 64 x 4096 in Q8_0 139 against 145), but not fp32 (8 heads of 128 a group 175 against 128) or 256 values.
  constexpr int kHeld = Tile::kRegs <= 64 && !(NS == 2 && (DT == 256 || (DT == 128 && T == T_F32))) ? 2 : 1;
  Tile held[kHeld];
  AttnQuery<T, KS> q;
  float mul = 1.0f;
  // Four sets of rows: a lane's weights are row col's for keys 4 g + r in register r.  Fewer: row
  // 4 t + lane % 4's for key lane / 4 in register t.
  constexpr bool kSets = NS < 4;
  constexpr int NT = kSets ? NS : 1;
  float m[NT], l[NT], muls[NT];
  f32x4 acc[NT][VB];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.0f;
#pragma unroll
    for (int j = 0; j < VB; ++j) acc[t][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // This lane's query values: row col's pieces; rows and values that are not there are zeros.
  auto set_query = [&]() __attribute__((always_inline)) {
    const int row = it.row0 + (kGroup ? col % R : col);
    const bool mine = row < it.rows && (kGroup ? col / R == g / G4 : col < R);
    const int64_t first = attn_row(c, it.q0, min(row, it.rows - 1), kvh, c.q_stride);
    int64_t from[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) from[s] = first + (piece(s) < d ? piece(s) : 0);
    float x[KS][8];
    attn_load8(x, c.q, from, c.q_type);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[s][j] = mine && piece(s) < d ? x[s][j] * c.scale2 : 0.0f;
    if constexpr (T != T_F32) {
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[s][j]));
#pragma unroll
      for (int o = kGroup ? R : 16; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
      // 2^e <= top < 2^(e + 1) to 2^14, for bf16 into 2^-10 .. 2^60; a row with an infinite value as it is
      const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
      const int up = e == 128 ? 0 : (T == T_BF16 ? min(max(e, -10), 60) : 14) - e;
      mul = __builtin_ldexpf(1.0f, -up);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[s][j] = __builtin_ldexpf(x[s][j], up);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) q.set(s, x[s]);
#pragma unroll
    for (int t = 0; t < NT; ++t) muls[t] = kSets ? __shfl(mul, 4 * t + (lane & 3)) : mul;
  };

  auto step = [&](const Tile& x) __attribute__((always_inline)) {
    f32x4 sc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (kGroup) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        f32x4 y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < J; ++j) y = q.mul(u * J + j, attn_bytes(x.k[u * J + j].w), y);
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[r] = __builtin_fmaf(attn_half((uint16_t)x.kstep[r][u]), y[r], sc[r]);
      }
      // The blocks of a row stand in four columns, or two (zeros where there are fewer groups): their sum, in all of them.
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (NS == 1) sc[r] += attn_rotate<4>(sc[r]);
        sc[r] += attn_rotate<8>(sc[r]);
      }
    }
#pragma unroll
    for (int s = 0; s < (kGroup ? 0 : KS); ++s) {
      if constexpr (T == T_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          sc = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, x.k[s].w[j]), q.v[s][j], sc, 0, 0, 0);
      } else if constexpr (kQ8) {
        // The piece is a block: its products are summed alone and then scaled, key by key.
        const f32x4 y = q.mul(s, attn_bytes(x.k[s].w), f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f16x2 two = __builtin_bit_cast(f16x2, x.kstep[r][s / 2]);
          sc[r] = __builtin_fmaf((float)(s % 2 ? two.y : two.x), y[r], sc[r]);
        }
      } else {
        sc = q.mul(s, __builtin_bit_cast(typename AttnQuery<T, KS>::Key, x.k[s].w), sc);
      }
    }
    if constexpr (kSets) {
      float top[NT], p[NT];
      bool past = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        p[t] = t == 0 ? attn_gather<0>(sc) : attn_gather<1>(sc);
        if (lane >> 2 >= x.live) p[t] = -INFINITY;
        top[t] = p[t] * muls[t];
        past |= top[t] > m[t] + kSlack;  // m + slack is -inf at the start: any finite logit moves it
      }
      if (__any(past)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float now = top[t];
#pragma unroll
          for (int s = 4; s < 64; s *= 2) now = fmaxf(now, __shfl_xor(now, s));
          now = fmaxf(m[t], now);
          const float f = m[t] == now ? 1.0f : attn_pow2(m[t] - now);
          m[t] = now;
          l[t] *= f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float fi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i));
#pragma unroll
            for (int j = 0; j < VB; ++j) acc[t][j][i] *= fi;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        p[t] = attn_pow2(__builtin_fmaf(p[t], muls[t], m[t] == -INFINITY ? 0.0f : -m[t])) * kWeight;
        l[t] += p[t];
      }
      attn_values<0, NT, VN, VU, kQ8>(acc, p, x);
      attn_values<1, NT, VN, VU, kQ8>(acc, p, x);
      attn_values<2, NT, VN, VU, kQ8>(acc, p, x);
      attn_values<3, NT, VN, VU, kQ8>(acc, p, x);
    } else {
      // In every tile: a branch around it right behind the product would lead to reads of sc sooner than the
      // matrix instruction's results are there, and the compiler counts the wait on the other path alone.
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[r] = 4 * g + r >= x.live ? -INFINITY : sc[r];
      const float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])) * mul;
      if (__any(top > m[0] + kSlack)) {
        float t = fmaxf(top, __shfl_xor(top, 16));
        t = fmaxf(t, __shfl_xor(t, 32));
        const float now = fmaxf(m[0], t);
        const float f = m[0] == now ? 1.0f : attn_pow2(m[0] - now);
        m[0] = now;
        l[0] *= f;
        float fr[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) fr[r] = __shfl(f, 4 * g + r);
#pragma unroll
        for (int j = 0; j < VB; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[0][j][r] *= fr[r];
      }
      const float ref = m[0] == -INFINITY ? 0.0f : m[0];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = attn_pow2(__builtin_fmaf(sc[r], mul, -ref)) * kWeight;
        l[0] += p;
        const float vs = kQ8 ? attn_half(x.vstep[kQ8 ? r : 0]) : 1.0f;
#pragma unroll
        for (int u = 0; u < VN; ++u) {
          float v[VU];
#pragma unroll
          for (int j = 0; j < VU; ++j) v[j] = x.v[r][u].at(j, vs);
          attn_pin(v);
#pragma unroll
          for (int j = 0; j < VU; ++j)
            acc[0][u * VU + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(p, v[j], acc[0][u * VU + j], 0, 0, 0);
        }
      }
    }
  };
  auto run = [&]<int AUX>() __attribute__((always_inline)) {
    load.template operator()<AUX>(held[0], 0);
    set_query();
    for (int n = 0; n < tiles; n += kHeld) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if (n + i >= tiles) break;
        if constexpr (kHeld == 2) {
          load.template operator()<AUX>(held[i ^ 1], n + i + 1);
          __builtin_amdgcn_sched_barrier(0);  // the loads go out before the tile in work is waited for
        } else if (n) {
          load.template operator()<AUX>(held[0], n);
          // Both loads before the first product: the compiler would have the values' wait behind it (fp32, 32 x 2000
          // tokens, heads of 256: 405 us against 263).
          __builtin_amdgcn_sched_barrier(0);
        }
        step(held[i]);
      }
    }
  };
  // The two loops apart: loads of one kind or the other inside one loop would blur what is on its way.
  if (once)
    run.template operator()<kOnce>();
  else
    run.template operator()<0>();

  // Weightless keys, all at -inf, are keys all the same: their row is 0 / 0, a row without keys zeros.
  if (seen) {
#pragma unroll
    for (int t = 0; t < NT; ++t) m[t] = fmaxf(m[t], kAttnLow);
  }

  // Join the waves: m, l and the values of the rows, through LDS.
  const int d16 = (d + 15) & ~15, nrow = min(R, it.rows - it.row0);
  float* lm = lds;                   // [wave][R]
  float* ll = lds + kAttnWaves * R;  // [wave][R]
  float* lv = lds + 2 * kAttnWaves * R + wave * R * d16;
  __syncthreads();  // attn_item's words have been read
  if constexpr (kSets) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int s = 4; s < 64; s *= 2) l[t] += __shfl_xor(l[t], s);
      if (lane < 4) {
        lm[wave * R + 4 * t + lane] = m[t];
        ll[wave * R + 4 * t + lane] = l[t];
      }
      // The lane groups hold sums over their own keys.  Halves of the values change places between the
      // groups and are added, twice: group g ends with values VB / 4 * (2 (g / 2) + g % 2) .. of its VB.
      constexpr int H = VB / 2, Q = VB / 4;
      f32x4 half[H];
#pragma unroll
      for (int j = 0; j < H; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) half[j][i] = attn_swap_add<32>(acc[t][j][i], acc[t][j + H][i]);
#pragma unroll
      for (int j = 0; j < Q; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = attn_swap_add<16>(half[j][i], half[j + Q][i]);
          const int at = col * VB + (g >> 1) * H + (g & 1) * Q + j;
          if (at < d) lv[(4 * t + i) * d16 + at] = v;
        }
    }
  } else {
    l[0] += __shfl_xor(l[0], 16);
    l[0] += __shfl_xor(l[0], 32);
    if (lane < 16) {
      lm[wave * R + lane] = m[0];
      ll[wave * R + lane] = l[0];
    }
#pragma unroll
    for (int j = 0; j < VB; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col * VB + j < d) lv[(4 * g + r) * d16 + col * VB + j] = acc[0][j][r];
  }
  __syncthreads();
  const float* v0 = lds + 2 * kAttnWaves * R;
  float* part = it.chunks > 1 ? attn_parts(c.ws, c.slots) + ((size_t)it.slot * c.kv_heads + kvh) * attn_part(R, d16)
                              : nullptr;
  const int quads = d / 4;
  for (int e = threadIdx.x; e < nrow * quads; e += 64 * kAttnWaves) {
    const int r = e / quads, i = 4 * (e - r * quads);
    float top = lm[r];
#pragma unroll
    for (int w = 1; w < kAttnWaves; ++w) top = fmaxf(top, lm[w * R + r]);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    f32x4 val = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) {
      const float f = attn_pow2(lm[w * R + r] - ref);
      sum += ll[w * R + r] * f;
      const f32x4 x = *reinterpret_cast<const f32x4*>(v0 + (w * R + r) * d16 + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) val[k] += x[k] * f;
    }
    if (it.chunks == 1) {
      float o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = top == -INFINITY ? 0.0f : val[k] / sum;
      attn_store4(c.out, attn_row(c, it.q0, it.row0 + r, kvh, c.out_stride) + i, c.q_type, o);
    } else {
      *reinterpret_cast<f32x4*>(part + r * d16 + i) = val;
      if (i == 0) {
        part[R * d16 + r] = top;
        part[R * (d16 + 1) + r] = sum;
      }
    }
  }
}

// Rows of a row tile, 4, 8 or 16: as many as a call's row tiles hold (the launchers' and the join's R).
template <uint32_t T, int DT, bool FULL, int NS> bool attn_split(const AttnCall& c, dim3 grid, hipStream_t s) {
  static LdsLimit lim;
  const size_t lds = (size_t)kAttnWaves * 4 * NS * (2 + (c.head_dim + 15) / 16 * 16) * sizeof(float);
  if (!lds_ready(reinterpret_cast<const void*>(&k_attn_split<T, DT, FULL, NS>), lim, lds)) return false;
  k_attn_split<T, DT, FULL, NS><<<grid, 64 * kAttnWaves, lds, s>>>(c);
  return true;
}

template <uint32_t T, int DT, bool FULL> bool attn_split_rows(const AttnCall& c, dim3 grid, hipStream_t s) {
  if (c.tile_rows == 4) return attn_split<T, DT, FULL, 1>(c, grid, s);
  if (c.tile_rows == 8) return attn_split<T, DT, FULL, 2>(c, grid, s);
  return attn_split<T, DT, FULL, 4>(c, grid, s);
}

template <uint32_t T> bool attn_split_dt(const AttnCall& c, dim3 grid, hipStream_t s) {
  if constexpr (T == T_Q8_0) {
    if (c.head_dim == 64) return attn_split_rows<T, 64, true>(c, grid, s);
    if (c.head_dim == 128) return attn_split_rows<T, 128, true>(c, grid, s);
    if (c.head_dim == 256) return attn_split_rows<T, 256, true>(c, grid, s);
  }
  if (c.head_dim <= 64) return attn_split_rows<T, 64, false>(c, grid, s);
  if (c.head_dim <= 128) return attn_split_rows<T, 128, false>(c, grid, s);
  return attn_split_rows<T, 256, false>(c, grid, s);
}

}  // namespace qvx
