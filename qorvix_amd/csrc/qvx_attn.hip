// qvx_attn.hip -- the join of the split attention's partial results, and the launches of a call.
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_split_f16(const AttnCall& c, dim3 grid, size_t lds, hipStream_t s);
bool launch_attn_split_bf16(const AttnCall& c, dim3 grid, size_t lds, hipStream_t s);
bool launch_attn_split_f32(const AttnCall& c, dim3 grid, size_t lds, hipStream_t s);
bool launch_attn_split_q8(const AttnCall& c, dim3 grid, size_t lds, hipStream_t s);

namespace {

// The chunks of a split sequence's row tile joined: out = sum_j 2^(m_j - m) v_j / sum_j 2^(m_j - m) l_j,
// m the largest m_j, in the same order of chunks in every run.  The grid is k_attn_split's; the workgroups of
// a row tile's chunks share its values, 64 of them a workgroup at a time, a value a lane, every fourth
// chunk a wave.
__global__ __launch_bounds__(256) void k_attn_join(AttnCall c) {
  __shared__ __attribute__((aligned(16))) float lds[3 * 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kvh = blockIdx.y;
  const AttnItem it = attn_item<kAttnRows>(c, blockIdx.x, reinterpret_cast<int*>(lds));
  if (!it.any || it.chunks == 1) return;
  const int d = c.head_dim, d16 = (d + 15) & ~15, nrow = min(kAttnRows, it.rows - it.row0);
  const size_t size = attn_part(c.lds_rows, d16), step = (size_t)c.kv_heads * size;
  const float* first = c.ws + ((size_t)(it.slot - it.chunk) * c.kv_heads + kvh) * size;
  for (int e0 = 64 * it.chunk; e0 < nrow * d; e0 += 64 * it.chunks) {
    const int e = min(e0 + lane, nrow * d - 1), r = e / d, i = e - r * d;
    float m = -INFINITY, sum = 0.0f, val = 0.0f;
    for (int j = wave; j < it.chunks; j += 4) {
      const float* part = first + j * step;
      const float mj = part[c.lds_rows * d16 + r], lj = part[c.lds_rows * (d16 + 1) + r], vj = part[r * d16 + i];
      const float top = fmaxf(m, mj), ref = top == -INFINITY ? 0.0f : top;
      const float f = attn_pow2(m - ref), fj = attn_pow2(mj - ref);
      sum = sum * f + lj * fj;
      val = val * f + vj * fj;
      m = top;
    }
    __syncthreads();
    lds[threadIdx.x] = m;
    lds[256 + threadIdx.x] = sum;
    lds[512 + threadIdx.x] = val;
    __syncthreads();
    if (wave == 0) {
      float top = m;
      for (int w = 1; w < 4; ++w) top = fmaxf(top, lds[64 * w + lane]);
      const float ref = top == -INFINITY ? 0.0f : top;
      sum = val = 0.0f;
      for (int w = 0; w < 4; ++w) {
        const float f = attn_pow2(lds[64 * w + lane] - ref);
        sum += lds[256 + 64 * w + lane] * f;
        val += lds[512 + 64 * w + lane] * f;
      }
      if (e0 + lane < nrow * d)
        attn_store(c.out, attn_row(c, it, it.row0 + r, kvh, c.out_stride) + i, c.q_type, val / sum);
    }
  }
}

}  // namespace

// The split kernel and, where the host's bound on the chunks allows a split, the join.
bool launch_attn_split(const AttnCall& c, uint32_t type, bool join, hipStream_t s) {
  const int d16 = (c.head_dim + 15) & ~15;
  const size_t lds = (size_t)kAttnWaves * (2 * kAttnRows + (size_t)c.lds_rows * d16) * sizeof(float);
  const dim3 grid((unsigned)c.items, (unsigned)c.kv_heads);
  bool ok = false;
  switch (type) {
    case T_F16: ok = launch_attn_split_f16(c, grid, lds, s); break;
    case T_BF16: ok = launch_attn_split_bf16(c, grid, lds, s); break;
    case T_F32: ok = launch_attn_split_f32(c, grid, lds, s); break;
    case T_Q8_0: ok = launch_attn_split_q8(c, grid, lds, s); break;
    default: break;
  }
  if (ok && join) k_attn_join<<<grid, 256, 0, s>>>(c);
  return ok;
}

}  // namespace qvx
