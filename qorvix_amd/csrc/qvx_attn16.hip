// qvx_attn16.hip -- cross attention of many queries in fp16 / bf16 on gfx950's 16-bit matrix cores.
//
//   out[row] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c (q[row] . k_j) - m),  c = scale log2(e)
//
// in one pass over the keys, 128 query rows a workgroup (32 a wave) against key and value tiles that
// the workgroup stages in LDS, the next tile in flight while the present one is multiplied.
//
// Arithmetic.  S^T = K Q^T and O^T = V^T P^T on the 32x32x16 instruction, fp32 sums.  The weights are
// rounded to the operands' type (to the nearest) before the second product: each by at most half a
// step; the denominator sums them in fp32.  The reference m follows the largest logit lazily, as in
// qvx_attn_split.hpp, kSlack16 above it when it is set (which moves a weight by 2^-21 of itself at most), so the largest
// bf16 weight lies at 2^-kSlack16 to 1.  In fp16 all weights are
// 2^kUp16 larger than that: up to 2^15 they stay in range, and down to 2^-21 of the largest above its smallest normal number.
//
// Layout.  In S^T a lane holds query row lane % 32 and, with h = lane / 32, the keys 8 (r / 4) + 4 h + r % 4
// in registers r = 0 .. 15.  The second product's right operand wants, for 16 keys, eight of them in
// lane half h: registers 8 n .. 8 n + 7 are such eight for one order of the keys, so the weights are
// only rounded and packed, and V^T is read with its keys in the same order: quads 4 h .. 4 h + 3 and
// 8 + 4 h .. of a 16-key step, each by one transposing LDS read.  A lane's row is the same in S^T, P^T
// and O^T, so maxima, sums and rescales need no lane exchange but that of the two halves.
//
// LDS rows are swizzled: 16-byte units of K by the row, so that sixteen rows' equal units cover the
// banks, 64-byte runs of V by the row, so that the four rows of a transposing read do.
//
// Bound by the vector instructions beside the matrix ones: per weight an fma, a power of two, half a maximum, half a
// pack and half a sum.  Measured, 2048 queries on 2048 states, 16 heads, 16 sequences, bf16: head size 64 800 TFLOP/s,
// 96 855, 128 905, 256 730, where a library product of 8192 cubed reaches 1264.  Three workgroups a CU up to a head size
// of 64 (with four, one register spills: 47.8 us against 46.4 for the ragged prompts below), two up to 160.
#include "qvx_attn_split.hpp"

namespace qvx {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

constexpr int kRows16 = kAttnRows16;
constexpr float kSlack16 = 8.0f;
template <uint32_t T> constexpr float kUp16 = T == T_F16 ? 15.0f : 0.0f;

typedef __attribute__((address_space(3))) uint8_t* LdsPtr;

template <uint32_t T> __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
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
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 h = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, h);
  }
}

// The denominator's sum with two more weights: bf16 as rounded (one instruction for both, and the rounding then
// cancels where values are alike), fp16 unrounded (its dot instruction is not promised to keep subnormal
// inputs, and many small weights may carry a row).
template <uint32_t T> __device__ __forceinline__ float sum2(float l, float x, float y, uint32_t xy) {
  if constexpr (T == T_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, xy), one, l, false);
  } else {
    return l + x + y;
  }
}

// DP: head_dim rounded up to a multiple of 32; KT: keys of a tile.
template <uint32_t T, int DP, int KT> struct Tile16 {
  static constexpr int kPitch = 2 * DP;       // bytes of a row
  static constexpr int kUnits = DP / 8;       // 16-byte units of a row
  static constexpr int kBanks = kPitch / 4 % 64;
  static constexpr int kBytes = KT * kPitch;  // of a tile of K, or of V
  static constexpr int kLoads = (KT * kUnits + 255) / 256;  // units a thread stages
  // Byte offset of unit u of row r.
  static __device__ __forceinline__ int k_at(int r, int u) {
    const int x = kBanks == 0 ? r & 15 : kBanks == 32 ? (r >> 1) & 7 : (r >> 2) & 3;
    return r * kPitch + 16 * (u ^ x);
  }
  static __device__ __forceinline__ int v_at(int r, int u) {
    const int x = kBanks == 0 ? r & 3 : kBanks == 32 ? (r >> 1) & 1 : 0;
    return r * kPitch + 16 * (u ^ (4 * x));
  }
};

template <uint32_t T, int DP, int KT>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : DP <= 160 ? 2 : 1) void k_attn16(AttnCall c) {
  using L = Tile16<T, DP, KT>;
  constexpr int KS = DP / 16, DB = DP / 32, KB = KT / 32;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds16[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int d = c.head_dim, item = (int)blockIdx.x / c.kv_heads, kvh = (int)blockIdx.x - item * c.kv_heads;
  AttnSums sums;
  const AttnItem it = attn_item<kRows16, kNoMask>(c, item, reinterpret_cast<int*>(lds16), sums);
  attn_note(c, it, item, kvh, sums);
  if (!it.any) return;
  __syncthreads();  // the item's words are read before tiles overwrite them
  const LdsPtr lds = (LdsPtr)lds16;

  const int row = it.row0 + 32 * wave + col;
  const bool live = row < it.rows;
  const int64_t qat = attn_row(c, it.q0, min(row, it.rows - 1), kvh, c.q_stride);
  u32x4 q[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int i = 16 * s + 8 * h;
    q[s] = u32x4{0, 0, 0, 0};
    if (live && i < d) {  // element by element where rows are not on 16-byte addresses
      const uint16_t* p = static_cast<const uint16_t*>(c.q) + qat + i;
      if (c.q_wide) {
        q[s] = *reinterpret_cast<const u32x4*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) q[s][j] = (uint32_t)p[2 * j] | (uint32_t)p[2 * j + 1] << 16;
      }
    }
  }

  // Staging: unit e = tid + 256 i of a tile is unit e % kUnits of its row e / kUnits.
  uint32_t goff[L::kLoads];
  int kst[L::kLoads], vst[L::kLoads];
#pragma unroll
  for (int i = 0; i < L::kLoads; ++i) {
    const int e = tid + 256 * i, r = e / L::kUnits, u = e - r * L::kUnits;
    goff[i] = 8 * u < d && r < KT ? (uint32_t)(r * c.pitch + 16 * u) : kPastEnd;
    kst[i] = L::k_at(r, u);
    vst[i] = L::v_at(r, u);
  }
  u32x4 kreg[L::kLoads], vreg[L::kLoads];
  const int key0 = it.tile0 * kAttnTile, keys = min(it.tile1 * kAttnTile, it.len) - key0;  // of this chunk
  const int64_t base = (int64_t)it.seq * c.page_stride + (int64_t)kvh * c.head_stride + (int64_t)key0 * c.pitch;
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const int n = min(KT, keys - t * KT);
    const int64_t at = base + (int64_t)t * KT * c.pitch;
    const __amdgpu_buffer_rsrc_t kr = attn_rsrc(c.k + at, (uint32_t)(n * c.pitch));
    const __amdgpu_buffer_rsrc_t vr = attn_rsrc(c.v + at, (uint32_t)(n * c.pitch));
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) kreg[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, goff[i], 0, 0);
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) vreg[i] = __builtin_amdgcn_raw_buffer_load_b128(vr, goff[i], 0, 0);
  };
  auto stage = [&](int buf) __attribute__((always_inline)) {
    const LdsPtr kb = lds + buf * 2 * L::kBytes, vb = kb + L::kBytes;
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i)
      if (KT * L::kUnits % 256 == 0 || tid + 256 * i < KT * L::kUnits) {
        *(__attribute__((address_space(3))) u32x4*)(kb + kst[i]) = kreg[i];
        *(__attribute__((address_space(3))) u32x4*)(vb + vst[i]) = vreg[i];
      }
  };

  // Lane addresses of the transposing reads: row 4 h + lane % 16 / 4 and column quad lane % 4 of the
  // sixteen columns that this group of sixteen lanes gets.
  const int vrow = 4 * h + (lane & 15) / 4, vcol = 16 * (lane >> 4 & 1) + 4 * (lane & 3);

  float m = -INFINITY, l = 0.0f;
  f32x16 acc[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[b][r] = 0.0f;

  const int tiles = (keys + KT - 1) / KT;
  if (tiles > 0) {
    fetch(0);
    stage(0);
  }
  // Nothing is on its way when the loop starts: a query register that might be makes the compiler wait, in
  // every tile, for the loads of the next one.
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
  // One tile from buffer `buf`, a constant in the unrolled loop: the LDS addresses are then lane offsets and immediates.
  // LAST: the chunk's last tile, which may end early, with its first BN blocks of 32 keys alone where the rest
  // holds none.  It stands behind the loop: as a branch inside it the values changed registers in every tile
  // (16 sequences of 448 queries on 1500 states, ragged, 52.9 -> 46.4 us).
  auto tile = [&]<int BN, bool LAST>(int t, int buf) __attribute__((always_inline)) {
    const LdsPtr kb = lds + buf * 2 * L::kBytes, vb = kb + L::kBytes;
    f32x16 s[BN];
#pragma unroll
    for (int b = 0; b < BN; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int b = 0; b < BN; ++b) {
        const u32x4 a = *(__attribute__((address_space(3))) u32x4*)(kb + L::k_at(32 * b + col, 2 * i + h));
        s[b] = mma32<T>(a, q[i], s[b]);
      }
    if constexpr (LAST) {
      const int left = keys - t * KT;
#pragma unroll
      for (int b = 0; b < BN; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = 32 * b + 8 * (r / 4) + 4 * h + r % 4 >= left ? -INFINITY : s[b][r];
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < BN; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
    top *= c.scale2;  // scale2 >= 0: the order stays
    if (__any(top > m)) {
      const float both = fmaxf(top, __shfl_xor(top, 32)), now = both > m ? both + kSlack16 : m;
      const float f = m == now ? 1.0f : attn_pow2(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][r] *= f;
    }
    const float ref = m == -INFINITY ? 0.0f : m - kUp16<T>;
    u32x4 p[BN][2];
#pragma unroll
    for (int b = 0; b < BN; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float x = attn_pow2(__builtin_fmaf(s[b][r], c.scale2, -ref));
        const float y = attn_pow2(__builtin_fmaf(s[b][r + 1], c.scale2, -ref));
        const uint32_t xy = pack2<T>(x, y);
        l = sum2<T>(l, x, y, xy);
        p[b][r / 8][r / 2 % 4] = xy;
      }
#pragma unroll
    for (int b = 0; b < BN; ++b)
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
          acc[e] = mma32<T>(__builtin_bit_cast(u32x4, v), p[b][n], acc[e]);
        }
  };
  const bool any_row = it.row0 + 32 * wave < it.rows;  // a wave past the rows only stages
  const int last = tiles - 1;
  for (int t0 = 0; t0 < last; t0 += 2) {
#pragma unroll
    for (int buf = 0; buf < 2; ++buf) {
      const int t = t0 + buf;
      if (t >= last) break;
      fetch(t + 1);
      if (any_row) tile.template operator()<KB, false>(t, buf);
      stage(buf ^ 1);  // the buffer that everyone left a barrier ago
      __syncthreads();
    }
  }
  if (any_row && tiles > 0) {
    if (KB == 1 || keys - last * KT > 32)
      tile.template operator()<KB, true>(last, last & 1);
    else
      tile.template operator()<1, true>(last, last & 1);
  }

  l += __shfl_xor(l, 32);
  if (!live) return;
  if (it.chunks > 1) {  // a part of the keys: for k_attn_join
    const int d16 = (d + 15) & ~15, r16 = row - it.row0;
    float* part = attn_parts(c.ws, c.slots) + ((size_t)it.slot * c.kv_heads + kvh) * attn_part(kRows16, d16);
#pragma unroll
    for (int e = 0; e < DB; ++e)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int i = 32 * e + 8 * (r / 4) + 4 * h;
        if (i < d)
          *reinterpret_cast<f32x4*>(part + r16 * d16 + i) = f32x4{acc[e][r], acc[e][r + 1], acc[e][r + 2], acc[e][r + 3]};
      }
    if (h == 0) {
      part[kRows16 * d16 + r16] = fmaxf(m, kAttnLow);  // a chunk has keys
      part[kRows16 * (d16 + 1) + r16] = l;
    }
    return;
  }
  const float inv = it.len ? 1.0f / l : 0.0f;  // no keys: zeros (acc is zero)
  uint16_t* o = static_cast<uint16_t*>(c.out) + attn_row(c, it.q0, row, kvh, c.out_stride);
#pragma unroll
  for (int e = 0; e < DB; ++e)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int i = 32 * e + 8 * (r / 4) + 4 * h;
      if (i >= d) continue;
      const u32x2 w = {pack2<T>(acc[e][r] * inv, acc[e][r + 1] * inv), pack2<T>(acc[e][r + 2] * inv, acc[e][r + 3] * inv)};
      if (c.out_wide) {
        *reinterpret_cast<u32x2*>(o + i) = w;
      } else {
        o[i] = (uint16_t)w[0], o[i + 1] = (uint16_t)(w[0] >> 16);
        o[i + 2] = (uint16_t)w[1], o[i + 3] = (uint16_t)(w[1] >> 16);
      }
    }
}

template <uint32_t T, int DP, int KT> bool attn16(const AttnCall& c, dim3 grid, hipStream_t s) {
  static LdsLimit lim;
  const size_t lds = 4 * (size_t)Tile16<T, DP, KT>::kBytes;
  if (!lds_ready(reinterpret_cast<const void*>(&k_attn16<T, DP, KT>), lim, lds)) return false;
  k_attn16<T, DP, KT><<<grid, 256, lds, s>>>(c);
  return true;
}

template <uint32_t T> bool attn16_dp(const AttnCall& c, dim3 grid, hipStream_t s) {
  const int d = c.head_dim;
  if (d <= 32) return attn16<T, 32, 64>(c, grid, s);
  if (d <= 64) return attn16<T, 64, 64>(c, grid, s);
  if (d <= 96) return attn16<T, 96, 64>(c, grid, s);
  if (d <= 128) return attn16<T, 128, 64>(c, grid, s);
  if (d <= 160) return attn16<T, 160, 32>(c, grid, s);
  return attn16<T, 256, 32>(c, grid, s);
}

}  // namespace

bool launch_attn16(const AttnCall& c, uint32_t type, hipStream_t s) {
  const dim3 grid((unsigned)c.items * (unsigned)c.kv_heads);
  return type == T_F16 ? attn16_dp<T_F16>(c, grid, s) : attn16_dp<T_BF16>(c, grid, s);
}

}  // namespace qvx
