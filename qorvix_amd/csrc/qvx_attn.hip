// qvx_attn.hip -- the join of the split attention's partial results, and the launches of a call.
#include "qvx_attn_split.hpp"

namespace qvx {

bool launch_attn_split_f16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_split_bf16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_split_f32(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_split_q8(const AttnCall& c, dim3 grid, hipStream_t s);

bool launch_attn_window_f16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_window_bf16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_window_f32(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_window_q8(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_prefix_f16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_prefix_bf16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_prefix_f32(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_prefix_q8(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_rest_f16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_rest_bf16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_rest_f32(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_rest_q8(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_whole_f16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_whole_bf16(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_whole_f32(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_whole_q8(const AttnCall& c, dim3 grid, hipStream_t s);
bool launch_attn_rows_f16(const AttnCall& c, bool parts, dim3 grid, hipStream_t s);
bool launch_attn_rows_bf16(const AttnCall& c, bool parts, dim3 grid, hipStream_t s);

void launch_attn_join(const AttnCall& c, hipStream_t s);

namespace {

// The chunks of a split sequence's row tile joined: out = sum_j 2^(m_j - m) v_j / sum_j 2^(m_j - m) l_j,
// m the largest m_j.  A workgroup a piece and key / value head; the workgroups of a row tile share its rows, as
// many at a time as fill the threads up to kFewChunks chunks, else one at a time.  Four values a
// thread; the threads that the rows leave over take other chunks, each a running maximum over its own, eight
// chunks' loads at a time; then the groups meet in LDS.  Latency bounds it: three dependent loads
// (piece, partial results, store): 4.3 us for a hundred pieces, 6.0 for 512 of one sequence, 4.8 where there are none.
// The order of the sums is the same in every run.
// One row at a time throughout took 2048 tokens from 11.3 to 12.0 us, rows together throughout 65536 from 54.4 to 58.0.
constexpr int kFewChunks = 16;
constexpr int kJoinShares = 4;  // workgroups a piece of 64 or 128 rows: of 128, with one 32 row tiles on 700 states 26.4 us
                                // against 21.1, with 8 20.0, but on 4000 then 44.3 against 35.9

template <int R> __global__ __launch_bounds__(256) void k_attn_join(AttnCall c) {
  __shared__ __attribute__((aligned(16))) float4 vals[256];
  __shared__ float2 stats[256];
  const int tid = threadIdx.x, kvh = blockIdx.y, slot = blockIdx.x;
  const AttnPiece pc = attn_pieces(c.ws)[slot];  // of the workspace: may be read before it is known to be one
  if (slot >= *reinterpret_cast<const int*>(c.ws)) return;
  // Offsets that are no running sums can name more pieces than there are workgroups to leave them: what stands there
  // instead is used only as far as it stays inside the call's rows and parts.
  if (pc.q0 < 0 || pc.row0 < 0 || pc.row0 >= pc.rows || pc.chunk < 0 || pc.chunk >= pc.chunks || pc.chunk > slot ||
      pc.chunks > c.slots - (slot - pc.chunk) || (int64_t)pc.q0 * c.group + pc.rows > (int64_t)c.n_q * c.group)
    return;
  const bool few = pc.chunks <= kFewChunks;
  const int d = c.head_dim, d16 = (d + 15) & ~15, quads = d / 4, nrow = min(R, pc.rows - pc.row0);
  const size_t size = attn_part(R, d16), step = (size_t)c.kv_heads * size;
  const float* first = attn_parts(c.ws, c.slots) + ((size_t)(slot - pc.chunk) * c.kv_heads + kvh) * size;
  const int wide = few ? min(R, 256 / quads) : 1;  // rows at a time
  const int groups = 256 / (quads * wide), mine = tid / (quads * wide), rest = tid - mine * quads * wide;
  const int row = rest / quads, quad = rest - row * quads;
  const int share = pc.chunk * (int)gridDim.z + (int)blockIdx.z, shares = pc.chunks * (int)gridDim.z;
  for (int r0 = share * wide; r0 < nrow; r0 += shares * wide) {
    const int r = r0 + row;
    float m = -INFINITY, l = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (mine < groups && r < nrow) {
      for (int j0 = mine; j0 < pc.chunks; j0 += 8 * groups) {
        float mj[8], lj[8];
        float4 vj[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = j0 + i * groups;
          const float* p = first + (size_t)min(j, pc.chunks - 1) * step;
          mj[i] = p[R * d16 + r];
          lj[i] = p[R * (d16 + 1) + r];
          vj[i] = *reinterpret_cast<const float4*>(p + r * d16 + 4 * quad);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (j0 + i * groups >= pc.chunks) mj[i] = -INFINITY, lj[i] = 0.0f, vj[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          top = fmaxf(top, mj[i]);
        }
        const float ref = top == -INFINITY ? 0.0f : top, f0 = attn_pow2(m - ref);
        m = top;
        l *= f0;
        v.x *= f0, v.y *= f0, v.z *= f0, v.w *= f0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = attn_pow2(mj[i] - ref);
          l += f * lj[i];
          v.x += f * vj[i].x, v.y += f * vj[i].y, v.z += f * vj[i].z, v.w += f * vj[i].w;
        }
      }
    }
    __syncthreads();  // the round before has been read
    vals[tid] = v;
    stats[tid] = make_float2(m, l);
    __syncthreads();
    if (mine == 0 && r < nrow) {
      float top = m;
      for (int i = 1; i < groups; ++i) top = fmaxf(top, stats[i * quads * wide + rest].x);
      const float ref = top == -INFINITY ? 0.0f : top, f0 = attn_pow2(m - ref);
      float sum = l * f0;
      float o[4] = {v.x * f0, v.y * f0, v.z * f0, v.w * f0};
      for (int i = 1; i < groups; ++i) {
        const float2 ml = stats[i * quads * wide + rest];
        const float4 x = vals[i * quads * wide + rest];
        const float f = attn_pow2(ml.x - ref);
        sum += ml.y * f;
        o[0] += x.x * f, o[1] += x.y * f, o[2] += x.z * f, o[3] += x.w * f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = top == -INFINITY ? 0.0f : o[k] / sum;
      attn_store4(c.out, attn_row(c, pc.q0, pc.row0 + r, kvh, c.out_stride) + 4 * quad, c.q_type, o);
    }
  }
}

}  // namespace

// The split kernel and, where the host's bound on the chunks allows a split, the join.
bool launch_attn_split(const AttnCall& c, uint32_t type, bool join, hipStream_t s) {
  const dim3 grid((unsigned)c.items * (unsigned)c.kv_heads);
  bool ok = false;
  switch (type) {
    case T_F16: ok = launch_attn_split_f16(c, grid, s); break;
    case T_BF16: ok = launch_attn_split_bf16(c, grid, s); break;
    case T_F32: ok = launch_attn_split_f32(c, grid, s); break;
    case T_Q8_0: ok = launch_attn_split_q8(c, grid, s); break;
    default: break;
  }
  if (ok && join) launch_attn_join(c, s);
  return ok;
}

// The same for masked calls; row tiles of 64 and 128 rows are the kernel's of many rows, with 16-bit parts where q is of another
// type than the cache or its scale does not keep the order of the products.
bool launch_attn_mask(const AttnCall& c, uint32_t type, bool join, hipStream_t s) {
  const dim3 grid((unsigned)c.items * (unsigned)c.kv_heads);
  bool ok = false;
  if (c.tile_rows >= kAttnRows16 / 2) {
    const bool parts = c.q_type != type || !c.in_order;
    ok = type == T_F16 ? launch_attn_rows_f16(c, parts, grid, s) : launch_attn_rows_bf16(c, parts, grid, s);
    if (ok && join) launch_attn_join(c, s);
    return ok;
  }
#define QVX_MODE(f)                                       \
  (c.mode == kMaskPrefix  ? launch_attn_prefix_##f        \
   : c.mode == kMaskRest  ? launch_attn_rest_##f          \
   : c.mode == kMaskWhole ? launch_attn_whole_##f         \
                          : launch_attn_window_##f)(c, grid, s)
  switch (type) {
    case T_F16: ok = QVX_MODE(f16); break;
    case T_BF16: ok = QVX_MODE(bf16); break;
    case T_F32: ok = QVX_MODE(f32); break;
    case T_Q8_0: ok = QVX_MODE(q8); break;
    default: break;
  }
#undef QVX_MODE
  if (ok && join) launch_attn_join(c, s);
  return ok;
}

void launch_attn_join(const AttnCall& c, hipStream_t s) {
  const dim3 grid((unsigned)c.slots, (unsigned)c.kv_heads);
  switch (c.tile_rows) {
    case 4: k_attn_join<4><<<grid, 256, 0, s>>>(c); break;
    case 8: k_attn_join<8><<<grid, 256, 0, s>>>(c); break;
    case 16: k_attn_join<16><<<grid, 256, 0, s>>>(c); break;
    case kAttnRows16 / 2: k_attn_join<kAttnRows16 / 2><<<dim3(grid.x, grid.y, kJoinShares), 256, 0, s>>>(c); break;
    default: k_attn_join<kAttnRows16><<<dim3(grid.x, grid.y, kJoinShares), 256, 0, s>>>(c); break;
  }
}

}  // namespace qvx
