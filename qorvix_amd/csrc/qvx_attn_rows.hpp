// qvx_attn_rows.hpp -- attention of many query rows over a paged 16-bit cache on gfx950's matrix cores, rows seeing parts of
// their sequence's keys: the kernel behind qvx_attn_window for prompts and behind qvx_attn_shared's prefixes.
//
//   out[row] = sum_j p_j v_j / sum_j p_j over the keys j that the row sees,  p_j = 2^(s_j - m),  s_j = scale log2(e) q[row] . k_j
//
// as in qvx_attn16.hip (128 rows a workgroup, 32 a wave; S^T = K Q^T and O^T = V^T P^T on the 32x32x16 instruction; K and V
// tiles staged in LDS, the next one in flight).  What is different:
//
// Pages.  Lane i of a wave looks tile t's key i up, two tiles ahead, so a page may hold any number of tokens; the threads
// that stage a key get its address from that lane.
//
// Masks.  The tiles of sixteen keys that any row of the tile sees are numbered one behind the other (AttnView), first tokens
// before the window, so a row's keys are two ranges of numbers.  Tiles that all rows of a wave see whole take the
// unmasked path, tiles that none sees are passed over, and keys that no row sees are zeros, whatever the page holds.
//
// Precision.  Queries of the cache's own type are multiplied as they are and the weights rounded to that type (PARTS
// false).  Others, fp32 above all, go in 16-bit parts (AttnQuery's: two of fp16, three of bf16, which leave 2^-23 and nothing), and
// so do the weights: two parts, which leave 2^-22 (fp16) or 2^-18 (bf16) of a weight.  The products of 16-bit values are
// exact and all sums fp32, so the matrix cores do two to three times the work, an eighth of what fp32 instructions would take.
#pragma once

#include "qvx_attn_split.hpp"

namespace qvx {

namespace rows {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

constexpr int kRows = kAttnRows16;
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
template <uint32_t T> __device__ __forceinline__ float low2(uint32_t w) {
  if constexpr (T == T_F16) return (float)__builtin_bit_cast(f16x2, w).x;
  return __builtin_bit_cast(float, w << 16);
}
template <uint32_t T> __device__ __forceinline__ float high2(uint32_t w) {
  if constexpr (T == T_F16) return (float)__builtin_bit_cast(f16x2, w).y;
  return __builtin_bit_cast(float, w & 0xffff0000u);
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

// What keys that are not there are loaded from.
__device__ const uint32_t kZeros[4] __attribute__((aligned(16))) = {0, 0, 0, 0};

template <uint32_t T, int DP, int KT, bool PARTS, int WGS>
__global__ __launch_bounds__(256, WGS) void k_attn_rows(AttnCall c) {
  using L = Tile<DP, KT>;
  constexpr int KS = DP / 16, DB = DP / 32, KB = KT / 32;
  constexpr int QP = !PARTS ? 1 : T == T_F16 ? 2 : 3, PP = PARTS ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_rows[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int d = c.head_dim, item = (int)blockIdx.x / c.kv_heads, kvh = (int)blockIdx.x - item * c.kv_heads;
  AttnSums sums;
  AttnItem it = attn_item<kRows, true>(c, item, reinterpret_cast<int*>(lds_rows), sums);
  if (c.mode != kMaskPrefix) attn_note(c, it, item, kvh, sums);
  if (!it.any) return;
  if (c.mode == kMaskPrefix) attn_leads<kRows>(c, it, kvh);
  const AttnView view = attn_view<kRows>(c, it);
  it.tile1 = min(it.tile1, view.tiles());
  if (c.mode == kMaskPrefix) it.seq = it.q0;  // the table's row
  __syncthreads();  // the item's words are read before tiles overwrite them
  const LdsPtr lds = (LdsPtr)lds_rows;

  const int row = it.row0 + 32 * wave + col, my_row = min(row, it.rows - 1);
  const bool live = row < it.rows;
  const int64_t qat = attn_row(c, it.q0, my_row, kvh, c.q_stride);
  u32x4 q[QP][KS];
  float mul = c.scale2;  // of a product to a logit in powers of two
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
    float x[KS][8];
    attn_load8(x, c.q, from, c.q_type);
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
          a -= low2<T>(w), b -= high2<T>(w);
        }
      }
  }

  // What this lane's row sees, in numbers of keys: [0, first_end) and [low, high); and over the wave's rows.
  const int shift = kAttnTile * (view.first - view.sinks);  // from a number to its key, behind the first tokens' tiles
  const AttnRange range = attn_range(c, it, view, my_row);
  const int first_end = min(range.sinks, range.high), low = range.low - shift;
  const unsigned width = (unsigned)max(range.high - range.low, 0);
  int wave_low = low, wave_high = low + (int)width, most_high = wave_high, least_low = low, most_first = first_end;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) {
    wave_low = max(wave_low, __shfl_xor(wave_low, x));
    wave_high = min(wave_high, __shfl_xor(wave_high, x));
    most_high = max(most_high, __shfl_xor(most_high, x));
    least_low = min(least_low, __shfl_xor(least_low, x));
    most_first = max(most_first, __shfl_xor(most_first, x));
  }
  wave_low = __builtin_amdgcn_readfirstlane(wave_low);
  wave_high = __builtin_amdgcn_readfirstlane(wave_high);
  most_high = __builtin_amdgcn_readfirstlane(most_high);
  least_low = __builtin_amdgcn_readfirstlane(least_low);
  most_first = __builtin_amdgcn_readfirstlane(most_first);

  // Tile t's keys: number key0 + t KT + lane.  look: asks the table; resolve: the address that it gives, and which keys
  // are there.
  const int key0 = it.tile0 * kAttnTile, key_end = it.tile1 * kAttnTile;
  const int32_t* table = c.table + (int64_t)it.seq * c.table_width;
  const int64_t head_at = (int64_t)kvh * c.head_stride;
  int page_id = -1, page_off = 0;
  int64_t at = -1;
  auto look = [&](int t) __attribute__((always_inline)) {
    const int number = key0 + t * KT + (lane & (KT - 1));
    const int key = number < kAttnTile * view.sinks ? number : number + shift;
    const bool there = number < key_end && key < view.high && (key >= view.low || key < view.sink_keys);
    const int column = there ? key / c.table_page : 0;
    page_off = key - column * c.table_page;
    page_id = there ? table[column] : -1;
  };
  auto resolve = [&]() __attribute__((always_inline)) {
    const bool there = (unsigned)page_id < (unsigned)c.n_pages;
    at = there ? page_id * c.page_stride + head_at + (int64_t)page_off * c.pitch : -1;
    return (uint64_t)__ballot(there);
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
  auto fetch = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) {
      if (KT * L::kUnits % 256 != 0 && 64 * (wave + 4 * i) >= KT * L::kUnits) break;
      const int64_t from = (int64_t)((uint64_t)(uint32_t)__shfl((int)(at >> 32), slot_key[i]) << 32 |
                                     (uint32_t)__shfl((int)at, slot_key[i]));
      const uint8_t* zeros = reinterpret_cast<const uint8_t*>(kZeros);
      const uint8_t* kp = from >= 0 && koff[i] >= 0 ? c.k + from + koff[i] : zeros;
      const uint8_t* vp = from >= 0 && voff[i] >= 0 ? c.v + from + voff[i] : zeros;
      const LdsPtr to = lds + buf * 2 * L::kBytes + 1024 * (wave + 4 * i);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)kp,
                                       (__attribute__((address_space(3))) void*)to, 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)vp,
                                       (__attribute__((address_space(3))) void*)(to + L::kBytes), 16, 0, 0);
    }
  };

  // Lane addresses of the transposing reads, as in qvx_attn16.hip.
  const int vrow = 4 * h + (lane & 15) / 4, vcol = 16 * (lane >> 4 & 1) + 4 * (lane & 3);

  float m = -INFINITY, l = 0.0f;
  bool saw = false;
  f32x16 acc[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[b][r] = 0.0f;

  // One tile from buffer `buf`; `there`: the keys that are.
  auto tile = [&]<bool MASKED>(int first, int buf, uint64_t there) __attribute__((always_inline)) {
    const LdsPtr kb = lds + buf * 2 * L::kBytes, vb = kb + L::kBytes;
    f32x16 s[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const u32x4 a = *(__attribute__((address_space(3))) u32x4*)(kb + L::k_at(32 * b + col, 2 * i + h));
#pragma unroll
        for (int j = QP - 1; j >= 0; --j) s[b] = mma<T>(a, q[j][i], s[b]);
      }
    if constexpr (MASKED) {
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
        if constexpr (PARTS) p[PP - 1][b][r / 8][r / 2 % 4] = pack2<T>(x - low2<T>(xy), y - high2<T>(xy));
      }
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < DB; ++e) {
          const int r0 = 32 * b + 16 * n + vrow, cc = 32 * e + vcol;
          const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) i16x4*)(vb + L::v_at(r0, cc / 8) + 2 * (cc & 7)));
          const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) i16x4*)(vb + L::v_at(r0 + 8, cc / 8) + 2 * (cc & 7)));
          const i16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
          for (int j = PP - 1; j >= 0; --j) acc[e] = mma<T>(__builtin_bit_cast(u32x4, v), p[j][b][n], acc[e]);
        }
  };

  const int tiles = max(key_end - key0 + KT - 1, 0) / KT;
  const bool any_row = it.row0 + 32 * wave < it.rows;  // a wave past the rows only stages
  constexpr uint64_t kAll = KT == 64 ? ~0ull : (1ull << KT) - 1;
  uint64_t there = 0, next = 0;
  if (tiles > 0) {
    look(0);
    there = resolve() & kAll;
    fetch(0);
    look(1);
    next = resolve() & kAll;
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the tile is in LDS when everyone passes the barrier
  __syncthreads();
  for (int t0 = 0; t0 < tiles; t0 += 2) {
#pragma unroll
    for (int buf = 0; buf < 2; ++buf) {
      const int t = t0 + buf;
      if (t >= tiles) break;
      if (t + 1 < tiles) fetch(buf ^ 1);  // the buffer that everyone left a barrier ago
      if (t + 2 < tiles) look(t + 2);
      const int first = key0 + t * KT;
      const bool none = !any_row || there == 0 || ((first >= most_high || first + KT <= least_low) && first >= most_first);
      if (!none) {
        if (there == kAll && first >= wave_low && first + KT <= wave_high)
          tile.template operator()<false>(first, buf, there);
        else
          tile.template operator()<true>(first, buf, there);
      }
      there = next;
      if (t + 2 < tiles) next = resolve() & kAll;
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();
    }
  }

  l += __shfl_xor(l, 32);
  saw = __shfl_xor((int)saw, 32) || saw;
  if (!live) return;
  if (saw) m = fmaxf(m, kAttnLow);
  if (it.chunks > 1 || c.mode == kMaskPrefix) {  // a part of the keys
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
        const u32x2 w = {pack2<T>(acc[e][r] * inv, acc[e][r + 1] * inv), pack2<T>(acc[e][r + 2] * inv, acc[e][r + 3] * inv)};
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

template <uint32_t T, int DP, int KT, bool PARTS, int WGS> bool launch(const AttnCall& c, dim3 grid, hipStream_t s) {
  static LdsLimit lim;
  const size_t lds = 4 * (size_t)Tile<DP, KT>::kBytes;
  if (!lds_ready(reinterpret_cast<const void*>(&k_attn_rows<T, DP, KT, PARTS, WGS>), lim, lds)) return false;
  k_attn_rows<T, DP, KT, PARTS, WGS><<<grid, 256, lds, s>>>(c);
  return true;
}

// Registers: with parts a query row alone takes two or three times the others'.
template <uint32_t T> bool launch_dp(const AttnCall& c, bool parts, dim3 grid, hipStream_t s) {
  const int d = c.head_dim;
  if (!parts) {
    if (d <= 32) return launch<T, 32, 64, false, 3>(c, grid, s);
    if (d <= 64) return launch<T, 64, 64, false, 3>(c, grid, s);
    if (d <= 96) return launch<T, 96, 64, false, 2>(c, grid, s);
    if (d <= 128) return launch<T, 128, 64, false, 2>(c, grid, s);
    if (d <= 160) return launch<T, 160, 32, false, 2>(c, grid, s);
    return launch<T, 256, 32, false, 1>(c, grid, s);
  }
  if (d <= 32) return launch<T, 32, 64, true, 2>(c, grid, s);
  if (d <= 64) return launch<T, 64, 64, true, 2>(c, grid, s);
  if (d <= 96) return launch<T, 96, 32, true, 2>(c, grid, s);
  if (d <= 128) return launch<T, 128, 32, true, 2>(c, grid, s);
  if (d <= 160) return launch<T, 160, 32, true, 1>(c, grid, s);
  return launch<T, 256, 32, true, 1>(c, grid, s);
}

}  // namespace rows

}  // namespace qvx
