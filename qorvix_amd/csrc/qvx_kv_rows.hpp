// qvx_kv_rows.hpp -- rows of q, k and v as the rotating kernels load and store them (qvx_kv.hip, qvx_norm_rope.hip).
#pragma once

#include "qvx_attn.hpp"
#include "qvx_kv.hpp"

namespace qvx {

// The cosines and sines of a workgroup's tokens t0 .. t0 + nt - 1, in LDS.  The angle's whole turns are taken off in 64 bits.
template <int THREADS> __device__ __forceinline__ void rope_table(const RopeCall& c, float* cs, int t0, int nt) {
  const int half = c.rot_dim / 2;
  for (int e = threadIdx.x; e < nt * half; e += THREADS) {
    const int t = e / half, i = e - t * half;
    const int axis = c.axis ? min((int)c.axis[i], c.n_axes - 1) : 0;
    double x = (double)c.pos[(int64_t)axis * c.pos_stride + t0 + t] * c.inv_freq[i] * 0.3183098861837906715;  // half turns
    x -= 2.0 * __builtin_rint(0.5 * x);
    float sn, cn;
    sincospif((float)x, &sn, &cn);
    cs[2 * t * half + i] = cn * c.scale;
    cs[2 * t * half + half + i] = sn * c.scale;
  }
}

struct Quad {
  float v[4];
};

template <bool VEC> __device__ __forceinline__ Quad quad_load(const float* p) {
  Quad x;
  if constexpr (VEC) {
    const float4 y = *reinterpret_cast<const float4*>(p);
    x.v[0] = y.x, x.v[1] = y.y, x.v[2] = y.z, x.v[3] = y.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[i] = p[i];
  }
  return x;
}
template <bool VEC> __device__ __forceinline__ void quad_store(float* p, const Quad& x) {
  if constexpr (VEC) {
    *reinterpret_cast<float4*>(p) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = x.v[i];
  }
}

// Eight consecutive values of a cache row, rounded to the cache's type; Q8_0 through the four lanes
// that hold a block of 32.
template <uint32_t T>
__device__ __forceinline__ void cache_store(const RopeCall& c, uint8_t* pages, int64_t pg, int head, int off, int i,
                                            const Quad& a, const Quad& b) {
  const int64_t row = (int64_t)head * c.page_size + off;
  uint8_t* page = pages + pg * c.page_stride;
  if constexpr (T == T_F32) {
    float4* p = reinterpret_cast<float4*>(page + (row * c.head_dim + i) * 4);
    p[0] = make_float4(a.v[0], a.v[1], a.v[2], a.v[3]);
    p[1] = make_float4(b.v[0], b.v[1], b.v[2], b.v[3]);
  } else if constexpr (T == T_F16 || T == T_BF16) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = j < 2 ? a.v[2 * j] : b.v[2 * j - 4], y = j < 2 ? a.v[2 * j + 1] : b.v[2 * j - 3];
      if constexpr (T == T_F16)
        w[j] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x) |
               (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)y) << 16;
      else
        w[j] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)y) << 16;
    }
    *reinterpret_cast<uint4*>(page + (row * c.head_dim + i) * 2) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    // scale = max|x| / 127 rounded to fp16, quants to the nearest (ties to even) of x / that scale, -127 to 127:
    // dividing by the rounded scale keeps each value within half a step of what is stored, but for what a scale rounded
    // down leaves of the block's largest: 127 times fp16's half step, which counts where the scale is subnormal (max|x|
    // below 2^-14 * 127; below 2^-25 * 127 the block is zeros).  Past 65504 * 127 the scale is infinite, the block NaN.
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(fabsf(a.v[j]), fabsf(b.v[j])));
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) nan |= a.v[j] != a.v[j] || b.v[j] != b.v[j];
    if (nan) top = __builtin_nanf("");
    // a NaN spreads through the maximum: the block stands for NaN, as its values do
#pragma unroll
    for (int x = 1; x < 4; x *= 2) {
      const float o = __shfl_xor(top, x);
      top = top != top || o != o ? __builtin_nanf("") : fmaxf(top, o);
    }
    const _Float16 scale = (_Float16)(top * (1.0f / 127.0f));
    const float s = (float)scale, inv = s > 0.0f ? 1.0f / s : 0.0f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = j < 4 ? a.v[j] : b.v[j - 4];
      const float r = __builtin_rintf(x * inv);
      const int q = (int)fminf(fmaxf(r, -127.0f), 127.0f);
      w[j / 4] |= (uint32_t)(q & 255) << (8 * (j % 4));
    }
    *reinterpret_cast<uint2*>(page + row * c.head_dim + i) = make_uint2(w[0], w[1]);
    if ((i & 31) == 0)
      *reinterpret_cast<_Float16*>(page + c.scale_off + (row * (c.head_dim / 32) + i / 32) * 2) = scale;
  }
}

// The launch of a call: `lanes` threads take a row.
inline dim3 rope_grid(RopeCall& c, int threads, int lanes) {
  const int rows = c.q_heads + 2 * c.kv_heads, half = c.rot_dim / 2;
  // A workgroup takes one token, or several whose rows together occupy its threads once.  (As many as their pairs
  // occupied it, four of 64 pairs: 8192 tokens 78.7 us against 71.5, 2048 29.4 against 19.2.)  Few tokens spread their
  // heads over workgroups, until there are two of them a CU: 8 tokens 4.2 us, 12.5 with each on one.
  const int least = std::max(1, threads / lanes);  // rows that occupy the threads once
  const int most = std::max(1, std::min(kRopeMaxTokens, half ? threads / half : kRopeMaxTokens));
  c.tokens_wg = std::max(1, std::min({most, threads / (rows * lanes), c.n_tokens / 512}));
  c.tokens_wg = std::max(c.tokens_wg, (c.n_tokens + kMostWgs - 1) / kMostWgs);  // at most kRopeMaxTokens: checked
  c.rows_wg = rows;
  if (c.n_tokens < 512) {
    const int parts = std::max(1, std::min((rows + least - 1) / least, 512 / c.n_tokens));
    c.rows_wg = (rows + parts - 1) / parts;
  }
  return dim3((unsigned)((c.n_tokens + c.tokens_wg - 1) / c.tokens_wg), (unsigned)((rows + c.rows_wg - 1) / c.rows_wg));
}

}  // namespace qvx
