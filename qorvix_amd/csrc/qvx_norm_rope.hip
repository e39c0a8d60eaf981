// qvx_norm_rope.hip -- norms of each query and key head, rotary positions and the append to the paged cache in one
// pass on gfx950.
//
//   y = x * w / sqrt(sum_i x_i^2 / d + eps),  then pairs of y turn as in qvx_kv.hip; q rounded to its output's type, k and
//   v to the cache's.
//
// The bytes bound it, q, k and v once in and once out, so the norm costs what it keeps the rows waiting: a row's d / 8
// lanes (rounded up to a power of two) hold it whole and add their squares by lane moves, without LDS or a barrier.
// The squares are summed in 64 bits: they do not overflow where fp32's would, from values of 1e18 on, and those
// instructions hide behind the loads.
//
// Measured, 32 query and 8 key / value heads of 128: 8192 tokens in bf16 70 us (302 MB, 4.3 TB/s, where a large copy
// reaches 4.85; the rotation alone, which writes q in fp32, 71); one token 4.1 us, the launch and four dependent loads.
#include "qvx_kv_rows.hpp"

namespace qvx {

namespace {

constexpr int kNormThreads = 256;

template <int CTRL> __device__ __forceinline__ double lane_move(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sum over 2^log lanes side by side, in all of them: neighbours, pairs, and mirrored halves of eight and of sixteen lanes.
__device__ __forceinline__ double lanes_sum(double x, int log) {
  if (log > 0) x += lane_move<0xb1>(x);
  if (log > 1) x += lane_move<0x4e>(x);
  if (log > 2) x += lane_move<0x141>(x);
  if (log > 3) x += lane_move<0x140>(x);
  if (log > 4) x += __shfl_xor(x, 16);
  return x;
}

// 1 / sqrt(mean): in fp32 where it and its root are normal numbers there.
__device__ __forceinline__ float norm_scale(double mean) {
  if (mean > 1e-30 && mean < 1e30) return 1.0f / sqrtf((float)mean);
  return (float)(1.0 / sqrt(mean));
}

template <uint32_t QT, bool VEC> __device__ __forceinline__ void q_store(void* out, int64_t at, const Quad& x) {
  if constexpr (QT == T_F32) {
    quad_store<VEC>(static_cast<float*>(out) + at, x);
  } else {
    uint16_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      h[j] = QT == T_F16 ? __builtin_bit_cast(uint16_t, (_Float16)x.v[j]) : __builtin_bit_cast(uint16_t, (__bf16)x.v[j]);
    uint16_t* p = static_cast<uint16_t*>(out) + at;
    if constexpr (VEC) {
      *reinterpret_cast<uint2*>(p) =
          make_uint2((uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = h[j];
    }
  }
}

template <uint32_t T, uint32_t QT, bool VEC>
__global__ __launch_bounds__(kNormThreads) void k_norm_rope(NormRopeCall c) {
  __shared__ float cs[2 * kRopeMaxPairs * kRopeMaxTokens];  // [token][cos, sin][pair]
  const int tid = threadIdx.x;
  const int rot = c.rot_dim, half = rot / 2, units = c.head_dim / 8, log = c.lanes_log;
  const int t0 = (int)blockIdx.x * c.tokens_wg, nt = min(c.tokens_wg, c.n_tokens - t0);
  rope_table<kNormThreads>(c, cs, t0, nt);
  __syncthreads();
  // Rows of a token: its q heads, then its k heads, then its v heads.
  const int rows = c.q_heads + 2 * c.kv_heads;
  const int r0 = (int)blockIdx.y * c.rows_wg, nr = min(c.rows_wg, rows - r0);
  const int u = tid & ((1 << log) - 1);
  const bool mine = u < units;
  for (int f = tid >> log; f < nt * nr; f += kNormThreads >> log) {
    const int t = f / nr, row = r0 + f - t * nr;  // the same in a row's lanes, and so are the branches but `mine`
    const int64_t token = t0 + t;
    const float* cn = cs + 2 * t * half;
    const float* sn = cn + half;
    const int slot = c.slots ? c.slots[token] : 0;
    if (slot < 0 || (c.k_pages && slot >= c.n_slots)) continue;  // no slot: the row is padding
    const bool is_q = row < c.q_heads, is_v = row >= c.q_heads + c.kv_heads;
    const int head = row - (is_q ? 0 : c.q_heads) - (is_v ? c.kv_heads : 0);
    const float* x = (is_q ? c.q + token * c.q_stride : is_v ? c.v + token * c.v_stride : c.k + token * c.k_stride) +
                     (int64_t)head * c.head_dim;
    const float* w = is_q ? c.q_w : is_v ? nullptr : c.k_w;
    if (w) w += (int64_t)head * c.w_stride;
    // A query's unit: two quads, a pair's halves half a rotation apart or side by side.  Of the cache's rows: eight values
    // in a row, and the quads that they turn with.
    const bool turned = !is_v && 8 * u < rot, apart = turned && c.halves;
    int ia = 8 * u, ib = 8 * u + 4;
    if (is_q && apart) ia = 4 * u, ib = 4 * u + half;
    const bool low = ia < half, high_b = ib < half;  // which half of its pair a quad of the cache's rows is
    Quad a{}, b{}, pa{}, pb{};
    double sum = 0.0;
    if (mine) {
      a = quad_load<VEC>(x + ia), b = quad_load<VEC>(x + ib);
      if (!is_q && apart) {  // quads never straddle the middle, nor the end: half is a multiple of 4
        pa = quad_load<VEC>(x + (low ? ia + half : ia - half));
        pb = quad_load<VEC>(x + (high_b ? ib + half : ib - half));
      }
    }
    if (w) {
      if (mine) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum = __builtin_fma((double)a.v[j], (double)a.v[j], sum);
          sum = __builtin_fma((double)b.v[j], (double)b.v[j], sum);
        }
      }
      sum = lanes_sum(sum, log);
      if (mine) {
        const float s = norm_scale(sum * c.inv_dim + (double)c.eps);
#pragma unroll
        for (int j = 0; j < 4; ++j) a.v[j] = a.v[j] * s * w[ia + j], b.v[j] = b.v[j] * s * w[ib + j];
        if (!is_q && apart) {
          const float *wa = w + (low ? ia + half : ia - half), *wb = w + (high_b ? ib + half : ib - half);
#pragma unroll
          for (int j = 0; j < 4; ++j) pa.v[j] = pa.v[j] * s * wa[j], pb.v[j] = pb.v[j] * s * wb[j];
        }
      }
    }
    if (!mine) continue;
    if (turned && !c.halves) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        Quad& z = j < 2 ? a : b;
        const int k = 2 * (j % 2);
        const float p = z.v[k], r = z.v[k + 1];
        z.v[k] = p * cn[4 * u + j] - r * sn[4 * u + j];
        z.v[k + 1] = p * sn[4 * u + j] + r * cn[4 * u + j];
      }
    } else if (apart && is_q) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = a.v[j], r = b.v[j];
        a.v[j] = p * cn[4 * u + j] - r * sn[4 * u + j];
        b.v[j] = p * sn[4 * u + j] + r * cn[4 * u + j];
      }
    } else if (apart) {
      const int ka = low ? ia : ia - half, kb = high_b ? ib : ib - half;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a.v[j] = low ? a.v[j] * cn[ka + j] - pa.v[j] * sn[ka + j] : pa.v[j] * sn[ka + j] + a.v[j] * cn[ka + j];
        b.v[j] = high_b ? b.v[j] * cn[kb + j] - pb.v[j] * sn[kb + j] : pb.v[j] * sn[kb + j] + b.v[j] * cn[kb + j];
      }
    }
    if (is_q) {
      const int64_t at = token * c.q_out_stride + (int64_t)row * c.head_dim;
      q_store<QT, VEC>(c.q_typed, at + ia, a);
      q_store<QT, VEC>(c.q_typed, at + ib, b);
    } else {
      const int pg = slot / c.page_size;
      cache_store<T>(c, is_v ? c.v_pages : c.k_pages, pg, head, slot - pg * c.page_size, 8 * u, a, b);
    }
  }
}

template <uint32_t T, uint32_t QT> void norm_launch(const NormRopeCall& c, bool vec, dim3 grid, hipStream_t s) {
  if (vec)
    k_norm_rope<T, QT, true><<<grid, kNormThreads, 0, s>>>(c);
  else
    k_norm_rope<T, QT, false><<<grid, kNormThreads, 0, s>>>(c);
}
template <uint32_t T> void norm_type(const NormRopeCall& c, uint32_t q_type, bool vec, dim3 grid, hipStream_t s) {
  switch (q_type) {
    case T_F16: norm_launch<T, T_F16>(c, vec, grid, s); break;
    case T_BF16: norm_launch<T, T_BF16>(c, vec, grid, s); break;
    default: norm_launch<T, T_F32>(c, vec, grid, s); break;
  }
}

}  // namespace

void launch_norm_rope(NormRopeCall c, uint32_t type, uint32_t q_type, bool vec, hipStream_t s) {
  const int units = c.head_dim / 8;
  c.lanes_log = 0;
  while ((1 << c.lanes_log) < units) ++c.lanes_log;
  const dim3 grid = rope_grid(c, kNormThreads, 1 << c.lanes_log);
  switch (type) {
    case T_F16: norm_type<T_F16>(c, q_type, vec, grid, s); break;
    case T_BF16: norm_type<T_BF16>(c, q_type, vec, grid, s); break;
    case T_Q8_0: norm_type<T_Q8_0>(c, q_type, vec, grid, s); break;
    default: norm_type<T_F32>(c, q_type, vec, grid, s); break;
  }
}

}  // namespace qvx
