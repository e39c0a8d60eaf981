// qvx_kv.hip -- the paged key / value cache's upkeep on gfx950: page tables and slots from request
// lengths, and rotary positions with the append.
#include "qvx_attn.hpp"
#include "qvx_kv.hpp"

namespace qvx {

namespace {

// ---- page tables ------------------------------------------------------------------------------------
//
// Sequence b holds c_b tokens and gets n_b more: its new pages are the columns ceil(c_b / P) ..
// ceil((c_b + n_b) / P) - 1 of its table row, filled from the free list in sequence order, so both the
// tokens' rows and the pages are prefix sums over the sequences.  Every workgroup forms both sums for
// itself in LDS (a few loads a thread: less than a launch of their own would take) and then looks its
// share of the tokens up by bisection.  A token at the start of a page stores the page's table entry:
// new pages all have one.  Bound by latency: for 256 sequences a few KB are touched (4.4 us captured; 1024 with
// 151640 new tokens 5.9).

constexpr int kMapThreads = 1024;

struct MapSums {
  long long tokens, pages;
};

// Sum over the wave's lanes up to this one: the halves of 16 bits each in 32 (64 of them take 22).
__device__ inline long long map_sum(long long x) {
  const int low = attn_scan((int)(x & 0xffff)), high = attn_scan((int)(x >> 16));
  return ((long long)high << 16) + low;
}

// Exclusive prefix sums over the workgroup of one value pair a thread (each below 2^32), and the totals.
__device__ inline MapSums map_scan(MapSums mine, MapSums* wave_sums, MapSums& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const MapSums x{map_sum(mine.tokens), map_sum(mine.pages)};
  __syncthreads();
  if (lane == 63) wave_sums[wave] = x;
  __syncthreads();
  MapSums before{0, 0};
  total = MapSums{0, 0};
  for (int w = 0; w < kMapThreads / 64; ++w) {
    if (w == wave) before = total;
    total.tokens += wave_sums[w].tokens;
    total.pages += wave_sums[w].pages;
  }
  return MapSums{before.tokens + x.tokens - mine.tokens, before.pages + x.pages - mine.pages};
}

// `write`: which outputs the launch stores: the tokens' (kMapTokens), the sequences' (kMapSeqs) or both.
__global__ __launch_bounds__(kMapThreads) void k_kv_map(MapCall c, int write) {
  __shared__ MapSums wave_sums[kMapThreads / 64];
  __shared__ int bad;
  extern __shared__ int32_t sums[];  // [n_seqs] rows behind each sequence, [n_seqs] its first new page
  const int tid = threadIdx.x, n = c.n_seqs, page = c.page_size;
  const int taken = c.taken_in[0];
  if (tid == 0) bad = taken < 0 ? QVX_MAP_NEGATIVE : 0;
  __syncthreads();
  MapSums all{0, 0};
  for (int b0 = 0; b0 < n; b0 += kMapThreads) {
    const int b = b0 + tid;
    MapSums mine{0, 0};
    int flags = 0;
    if (b < n) {
      const long long held = c.held[b], add = c.added[b];
      if (held < 0 || add < 0) {
        flags = QVX_MAP_NEGATIVE;
      } else {
        mine.tokens = add;
        mine.pages = (held + add + page - 1) / page - (held + page - 1) / page;
        if (held + add > (long long)c.table_width * page || held + add > 0x7fffffffll) flags = QVX_MAP_COLUMNS;
      }
    }
    if (flags) atomicOr(&bad, flags);
    MapSums total;
    const MapSums at = map_scan(mine, wave_sums, total);
    if (b < n) {  // meaningless past 32 bits, and then not used
      sums[b] = (int32_t)(all.tokens + at.tokens + mine.tokens);
      sums[n + b] = (int32_t)(all.pages + at.pages);
    }
    all.tokens += total.tokens;
    all.pages += total.pages;
  }
  __syncthreads();
  int status = bad;
  if (all.tokens > c.max_tokens) status |= QVX_MAP_ROWS;
  if (taken >= 0 && taken + all.pages > c.n_free) status |= QVX_MAP_PAGES;
  const bool ok = status == 0;

  if ((write & kMapSeqs) && blockIdx.x == 0) {
    for (int b = tid; b < n; b += kMapThreads) {
      const int held = c.held[b], add = c.added[b];
      c.lens[b] = ok ? held + add : held;
      c.offsets[b + 1] = ok ? sums[b] : 0;
    }
    if (tid == 0) {
      c.offsets[0] = 0;
      c.taken_out[0] = ok ? taken + (int)all.pages : taken;
      c.taken_out[1] = status;
    }
  }
  if (!(write & kMapTokens)) return;
  const int tokens = ok ? (int)all.tokens : 0;
  const int stride = (int)gridDim.x * kMapThreads;
  for (int t = (int)blockIdx.x * kMapThreads + tid; t < c.max_tokens; t += stride) {
    int slot = -1, pos = 0, seq = -1;
    if (t < tokens) {
      int lo = 0, hi = n - 1;  // the first sequence whose rows end past t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > t) hi = mid; else lo = mid + 1;
      }
      seq = lo;
      const int held = c.held[seq];
      pos = held + t - (seq ? sums[seq - 1] : 0);
      const int column = pos / page, off = pos - column * page, first = (int)(((long long)held + page - 1) / page);
      int32_t* entry = c.table + (int64_t)seq * c.table_width + column;
      const int id = column < first ? *entry : c.free_list[taken + sums[n + seq] + column - first];
      if (off == 0) *entry = id;  // a page starts here, so it is new (or was left empty: its own id again)
      const long long s = (long long)id * page + off;
      slot = id < 0 || s > 0x7fffffffll ? -1 : (int)s;
    }
    c.slots[t] = slot;
    if (c.pos) c.pos[t] = pos;
    if (c.seq) c.seq[t] = seq;
    if (t > 0x7fffffff - stride) break;
  }
}

// ---- rotary positions and the append -----------------------------------------------------------------
//
// Pair i of a head is turned by pos[axis[i]] * inv_freq[i]; the angle's whole turns are taken off in
// 64 bits (at position 10^6 an fp32 product is off by 0.06), the rest is an fp32 number of half turns.
// One pass over q, k and v; the bytes bound it: 8192 tokens of 32 + 2 x 8 heads of 128 into a bf16 cache 70.7 us,
// 5.2 TB/s where an elementwise pass over as many bytes reaches 5.9, into a Q8_0 one 70.3 (5.0); one token 3.5 us.  A workgroup takes `tokens_wg` tokens and a range of
// their heads: its threads first form the cosines and sines of the tokens' pairs in LDS, each once, and
// then take 8 values of a head at a time.

constexpr int kRopeThreads = 256;

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

template <uint32_t T, bool VEC>
__global__ __launch_bounds__(kRopeThreads) void k_rope_kv(RopeCall c) {
  __shared__ float cs[2 * kRopeMaxPairs * kRopeMaxTokens];  // [token][cos, sin][pair]
  const int tid = threadIdx.x;
  const int rot = c.rot_dim, half = rot / 2, units = c.head_dim / 8;
  const int t0 = (int)blockIdx.x * c.tokens_wg, nt = min(c.tokens_wg, c.n_tokens - t0);
  for (int e = tid; e < nt * half; e += kRopeThreads) {
    const int t = e / half, i = e - t * half;
    const int axis = c.axis ? min((int)c.axis[i], c.n_axes - 1) : 0;
    double x = (double)c.pos[(int64_t)axis * c.pos_stride + t0 + t] * c.inv_freq[i] * 0.3183098861837906715;  // half turns
    x -= 2.0 * __builtin_rint(0.5 * x);
    float sn, cn;
    sincospif((float)x, &sn, &cn);
    cs[2 * t * half + i] = cn * c.scale;
    cs[2 * t * half + half + i] = sn * c.scale;
  }
  __syncthreads();
  // Rows of a token: its q heads, then its k heads, then its v heads.
  const int rows = c.q_heads + 2 * c.kv_heads;
  const int r0 = (int)blockIdx.y * c.rows_wg, nr = min(c.rows_wg, rows - r0);
  const int work = nt * nr * units;
  for (int e = tid; e < work; e += kRopeThreads) {
    // A row's units lie in consecutive threads: blocks of 32 values in four of them.
    const int t = e / (nr * units), f = e - t * (nr * units), rr = f / units, u = f - rr * units;
    const int row = r0 + rr;
    const int64_t token = t0 + t;
    const float* cn = cs + 2 * t * half;
    const float* sn = cn + half;
    const int slot = c.slots ? c.slots[token] : 0;
    if (slot < 0 || (c.k_pages && slot >= c.n_slots)) continue;  // no slot: the row is padding
    if (row < c.q_heads) {
      const float* x = c.q + token * c.q_stride + (int64_t)row * c.head_dim;
      float* y = c.q_out + token * c.q_out_stride + (int64_t)row * c.head_dim;
      // The unit's two quads: a pair's halves lie half a rotation apart, or side by side.
      int ia = 8 * u, ib = 8 * u + 4;
      const bool turned = ia < rot;
      if (turned && c.halves) ia = 4 * u, ib = 4 * u + half;
      Quad a = quad_load<VEC>(x + ia), b = quad_load<VEC>(x + ib);
      if (turned) {
        if (c.halves) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = a.v[j], r = b.v[j];
            a.v[j] = p * cn[4 * u + j] - r * sn[4 * u + j];
            b.v[j] = p * sn[4 * u + j] + r * cn[4 * u + j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            Quad& z = j < 2 ? a : b;
            const int k = 2 * (j % 2);
            const float p = z.v[k], r = z.v[k + 1];
            z.v[k] = p * cn[4 * u + j] - r * sn[4 * u + j];
            z.v[k + 1] = p * sn[4 * u + j] + r * cn[4 * u + j];
          }
        }
      }
      quad_store<VEC>(y + ia, a);
      quad_store<VEC>(y + ib, b);
      continue;
    }
    const bool is_v = row >= c.q_heads + c.kv_heads;
    const int head = row - c.q_heads - (is_v ? c.kv_heads : 0);
    const float* x = (is_v ? c.v + token * c.v_stride : c.k + token * c.k_stride) + (int64_t)head * c.head_dim;
    Quad z[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = 8 * u + 4 * h;
      z[h] = quad_load<VEC>(x + i);
      if (is_v || i >= rot) continue;
      if (c.halves) {  // quads never straddle the middle: half is a multiple of 4
        const bool low = i < half;
        const Quad o = quad_load<VEC>(x + (low ? i + half : i - half));
        const int p = low ? i : i - half;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          z[h].v[j] = low ? z[h].v[j] * cn[p + j] - o.v[j] * sn[p + j] : o.v[j] * sn[p + j] + z[h].v[j] * cn[p + j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const int p = (i + j) / 2;
          const float a = z[h].v[j], b = z[h].v[j + 1];
          z[h].v[j] = a * cn[p] - b * sn[p];
          z[h].v[j + 1] = a * sn[p] + b * cn[p];
        }
      }
    }
    const int pg = slot / c.page_size;
    cache_store<T>(c, is_v ? c.v_pages : c.k_pages, pg, head, slot - pg * c.page_size, 8 * u, z[0], z[1]);
  }
}

template <uint32_t T> void rope_launch(const RopeCall& c, bool vec, dim3 grid, hipStream_t s) {
  if (vec)
    k_rope_kv<T, true><<<grid, kRopeThreads, 0, s>>>(c);
  else
    k_rope_kv<T, false><<<grid, kRopeThreads, 0, s>>>(c);
}

}  // namespace

bool launch_kv_map(const MapCall& c, bool alias, hipStream_t s) {
  static LdsLimit lim;
  const size_t lds = 2 * (size_t)c.n_seqs * sizeof(int32_t);
  if (!lds_ready(reinterpret_cast<const void*>(&k_kv_map), lim, lds)) return false;
  // A token a thread up to a workgroup a CU; more only repeat the sums (506196 rows 9.0 us, with 512 workgroups 11.2).
  // With four tokens a thread, which share a bisection and load together, 151640 rows took 8.7 us against 6.5 and 506196
  // 9.4: neighbours are then different sequences or pages.
  const int wgs = std::min(256, c.max_tokens / kMapThreads + 1);
  // Outputs that lie on inputs are stored by a launch of one workgroup, behind the one that reads them.
  k_kv_map<<<wgs, kMapThreads, lds, s>>>(c, alias ? kMapTokens : kMapTokens | kMapSeqs);
  if (alias) k_kv_map<<<1, kMapThreads, lds, s>>>(c, kMapSeqs);
  return true;
}

void launch_rope_kv(RopeCall c, uint32_t type, bool vec, hipStream_t s) {
  const int rows = c.q_heads + 2 * c.kv_heads, half = c.rot_dim / 2;
  // A workgroup takes one token, or several whose rows together occupy its threads once.  (As many as their pairs
  // occupied it, four of 64 pairs: 8192 tokens 78.7 us against 71.5, 2048 29.4 against 19.2.)  Few tokens spread their
  // heads over workgroups, until there are two of them a CU: 8 tokens 4.2 us, 12.5 with each on one.
  const int units = c.head_dim / 8, least = std::max(1, kRopeThreads / units);  // rows that occupy the threads once
  const int most = std::max(1, std::min(kRopeMaxTokens, half ? kRopeThreads / half : kRopeMaxTokens));
  c.tokens_wg = std::max(1, std::min({most, kRopeThreads / (rows * units), c.n_tokens / 512}));
  c.tokens_wg = std::max(c.tokens_wg, (c.n_tokens + kMostWgs - 1) / kMostWgs);  // at most kRopeMaxTokens: checked
  c.rows_wg = rows;
  if (c.n_tokens < 512) {
    const int parts = std::max(1, std::min((rows + least - 1) / least, 512 / c.n_tokens));
    c.rows_wg = (rows + parts - 1) / parts;
  }
  const dim3 grid((unsigned)((c.n_tokens + c.tokens_wg - 1) / c.tokens_wg), (unsigned)((rows + c.rows_wg - 1) / c.rows_wg));
  switch (type) {
    case T_F16: rope_launch<T_F16>(c, vec, grid, s); break;
    case T_BF16: rope_launch<T_BF16>(c, vec, grid, s); break;
    case T_Q8_0: rope_launch<T_Q8_0>(c, vec, grid, s); break;
    default: rope_launch<T_F32>(c, vec, grid, s); break;
  }
}

}  // namespace qvx
