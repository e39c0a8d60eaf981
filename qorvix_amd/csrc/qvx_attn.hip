// qvx_attn.hip -- the join of the split attention's partial results, and the launches of a call.
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_split_f16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_split_bf16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_split_f32(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_split_q8(const AttnCall& c, dim3 grid, hipStream_t s);

namespace {

// The chunks of a split sequence's row tile joined: out = sum_j 2^(m_j - m) v_j / sum_j 2^(m_j - m) l_j,
// m the largest m_j.  The grid is k_attn_split's; the workgroups of a row tile's chunks share its rows, one
// at a time.  A row's factors are formed first, 256 chunks at a time, so that the loads of the values
// depend on nothing and go out together: 4 values a lane, the lanes that a row leaves over on other
// chunks.  Sums are taken in the same order in every run.
template <int R> __global__ __launch_bounds__(256) void k_attn_join(AttnCall c) {
  __shared__ __attribute__((aligned(16))) float factor[256];
  __shared__ __attribute__((aligned(16))) float4 sums[256];
  __shared__ float red[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kvh = blockIdx.y;
  const AttnItem it = attn_item<R>(c, blockIdx.x, reinterpret_cast<int*>(factor));
  if (!it.any || it.chunks == 1) return;
  const int d = c.head_dim, d16 = (d + 15) & ~15, nrow = min(R, it.rows - it.row0);
  const size_t size = attn_part(R, d16), step = (size_t)c.kv_heads * size;
  const float* first = c.ws + ((size_t)(it.slot - it.chunk) * c.kv_heads + kvh) * size;
  const int quads = d / 4, groups = 256 / quads, mine = tid / quads, quad = tid - mine * quads;
  for (int r = it.chunk; r < nrow; r += it.chunks) {
    const float* ms = first + R * d16 + r;
    float top = -INFINITY;
    for (int j = tid; j < it.chunks; j += 256) top = fmaxf(top, ms[j * step]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    __syncthreads();
    if (lane == 0) red[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float ref = top == -INFINITY ? 0.0f : top;
    float l = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j0 = 0; j0 < it.chunks; j0 += 256) {
      const int n = min(256, it.chunks - j0);
      if (j0) __syncthreads();
      if (tid < n) {
        const float* p = ms + (size_t)(j0 + tid) * step;
        const float f = attn_pow2(p[0] - ref);
        factor[tid] = f;
        l += f * p[R];
      }
      __syncthreads();
      if (mine < groups) {
        const float* p = first + (size_t)j0 * step + r * d16 + 4 * quad;
#pragma unroll 8
        for (int j = mine; j < n; j += groups) {
          const float4 x = *reinterpret_cast<const float4*>(p + (size_t)j * step);
          const float f = factor[j];
          v.x += f * x.x, v.y += f * x.y, v.z += f * x.z, v.w += f * x.w;
        }
      }
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x);
    if (lane == 0) red[4 + wave] = l;
    sums[tid] = v;
    __syncthreads();
    if (mine == 0) {
      for (int i = 1; i < groups; ++i) {
        const float4 x = sums[i * quads + quad];
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      const float sum = red[4] + red[5] + red[6] + red[7];
      const int64_t at = attn_row(c, it, it.row0 + r, kvh, c.out_stride) + 4 * quad;
      const float o[4] = {v.x / sum, v.y / sum, v.z / sum, v.w / sum};
      attn_store4(c.out, at, c.q_type, o);
    }
  }
}

}  // namespace

// The split kernel and, where the host's bound on the chunks allows a split, the join.
bool launch_attn_split(const AttnCall& c, uint32_t type, bool join, hipStream_t s) {
  const dim3 grid((unsigned)c.items, (unsigned)c.kv_heads);
  bool ok = false;
  switch (type) {
    case T_F16: ok = launch_attn_split_f16(c, grid, s); break;
    case T_BF16: ok = launch_attn_split_bf16(c, grid, s); break;
    case T_F32: ok = launch_attn_split_f32(c, grid, s); break;
    case T_Q8_0: ok = launch_attn_split_q8(c, grid, s); break;
    default: break;
  }
  if (ok && join) {
    if (c.tile_rows == 4)
      k_attn_join<4><<<grid, 256, 0, s>>>(c);
    else if (c.tile_rows == 8)
      k_attn_join<8><<<grid, 256, 0, s>>>(c);
    else
      k_attn_join<16><<<grid, 256, 0, s>>>(c);
  }
  return ok;
}

}  // namespace qvx
