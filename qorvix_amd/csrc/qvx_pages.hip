// qvx_pages.hip -- pages of a cache that several sequences hold, on gfx950: forks, copies, releases, compaction.
//
// extra[p] counts the rows that hold page p beside the first, so a page of one owner needs no upkeep.  A fork shares a
// sequence's full pages (extra + 1 each) and takes a fresh page for its last one where that is not full, which a copy then
// fills: no shared page is ever appended to.  A release takes one holder from each page; pages without any go back to the
// free list.  All results are whole numbers and the same in every run: counts meet in integer atomics, whose order does
// not matter, and pages return in the order of their ids, not of their release.
//
// Bound by latency but for the copies, which the bytes bound.  Measured: 128 forks of 256 shared pages 8.4 us, the copy of their
// last pages in 16 layers 45 (269 MB read and written, 6 TB/s, part of it in the caches; a large copy reaches 4.85), their release
// 5.8 + 4.7; the compaction of 4500 pages 9 us, its copy in 8 layers 230 (1.13 GB, 4.9 TB/s); 8 forks, copies and releases 6.3, 3.8
// and 5.8, chains of dependent loads and atomics.
#include "qvx_pages.hpp"

namespace qvx {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ bool page_ok(int id, int n_pages) { return (unsigned)id < (unsigned)n_pages; }

// Sum over the workgroup, in every thread; `part`: LDS of a word a wave, free again at return.
template <int THREADS> __device__ __forceinline__ int block_sum(int x, int* part) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) sum += part[w];
  __syncthreads();
  return sum;
}

// Sum over the threads before this one.
template <int THREADS> __device__ __forceinline__ int block_before(int x, int* part, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int upto = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
  }
  if (lane == 63) part[wave] = upto;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w == wave) before = total;
    total += part[w];
  }
  __syncthreads();
  return before + upto - x;
}

// ---- fork --------------------------------------------------------------------------------------------
//
// Every workgroup looks all forks through for itself (a few loads a thread): how many want a fresh page before its own,
// whether the free list reaches, whether any is wrong.  Then it takes kTogether forks and a column of theirs a thread:
// forks of one prompt hold the same page there, and one atomic counts all of them.  (An atomic each: 128 forks of 256 shared
// pages 14.8 us, most of it atomics on the same lines.)

constexpr int kTogether = 16;

// What a fork wants: 1 where its sequence's last page is not full; `bad` gets status bits, `len` the sequence's length.
__device__ __forceinline__ int fork_wants(const ForkCall& c, int from, int to, int& len, int& bad) {
  if ((unsigned)from >= (unsigned)c.n_rows || (unsigned)to >= (unsigned)c.n_rows || from == to) {
    bad |= QVX_MAP_SEQUENCE;
    return 0;
  }
  len = c.lens[from];
  if (len < 0) bad |= QVX_MAP_NEGATIVE;
  if (len > (long long)c.table_width * c.page_size) bad |= QVX_MAP_COLUMNS;
  return len > 0 && len % c.page_size != 0;
}

// Pages one behind the other that are counted together; `sign` 1 or -1.
struct PageRun {
  int32_t* extra;
  int n_pages, id = -1, n = 0;
  __device__ __forceinline__ void flush(int sign) {
    if (n) atomicAdd(&extra[id], sign * n);
  }
  __device__ __forceinline__ void take(int page, int sign) {
    if (!page_ok(page, n_pages)) return;
    if (page != id) {
      flush(sign);
      id = page, n = 0;
    }
    ++n;
  }
};

__global__ __launch_bounds__(kThreads) void k_kv_fork(ForkCall c, int write) {
  __shared__ int part[kThreads / 64], all_bad;
  __shared__ int from[kTogether], to[kTogether], lens[kTogether], fresh[kTogether];
  __shared__ int place[kTogether];  // of this workgroup's forks: fresh pages of those before
  const int own = (int)blockIdx.x * kTogether, n = min(kTogether, c.n - own);
  const int tid = threadIdx.x, taken = c.taken_in[0];
  if (tid < kTogether) from[tid] = 0, lens[tid] = 0;  // past the last fork: read like the others, not used
  if (tid == 0) all_bad = taken < 0 ? QVX_MAP_NEGATIVE : 0;
  int bad = 0, all = 0;
  for (int i0 = 0; i0 < c.n; i0 += kThreads) {
    const int i = i0 + tid;
    const int source = i < c.n ? c.from[i] : 0, target = i < c.n ? c.to[i] : 0;
    int total, len = 0;
    const int wants = i < c.n ? fork_wants(c, source, target, len, bad) : 0;
    const int before = block_before<kThreads>(wants, part, total);
    if (i >= own && i < own + n) from[i - own] = source, to[i - own] = target, lens[i - own] = len, place[i - own] = all + before;
    all += total;
  }
  if (bad) atomicOr(&all_bad, bad);
  __syncthreads();
  int status = all_bad;
  if (taken >= 0 && (long long)taken + all > c.n_free) status |= QVX_MAP_PAGES;
  const bool first = blockIdx.x == 0 && blockIdx.y == 0 && tid == 0;
  if ((write & kForkTotals) && first) {
    c.taken_out[0] = status ? taken : taken + all;
    c.taken_out[1] = status;
    *c.n_pairs = status ? 0 : all;
  }
  if (!(write & kForkRows) || status) return;
  // All of it is read before anything is stored: the compiler has to assume that a store changes it.
  if (tid < n) {
    const int at = taken + place[tid];
    fresh[tid] = at < c.n_free ? c.free_list[at] : -1;  // a fork that wants none, or whose length another one changes
  }
  __syncthreads();
  for (int col = (int)blockIdx.y * kThreads + tid; col < c.table_width; col += (int)gridDim.y * kThreads) {
    int ids[kTogether];
#pragma unroll
    for (int j = 0; j < kTogether; ++j) ids[j] = c.table[(int64_t)from[j] * c.table_width + col];
    PageRun run{c.extra, c.n_pages};
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      if (j >= n) continue;
      const int full = lens[j] / c.page_size;
      int id = -1;
      if (col < full) {
        id = ids[j];
        run.take(id, 1);
      } else if (col == full && lens[j] > full * c.page_size) {
        id = fresh[j];
        c.pairs[2 * place[j]] = ids[j];
        c.pairs[2 * place[j] + 1] = id;
      }
      c.table[(int64_t)to[j] * c.table_width + col] = id;
    }
    run.flush(1);
  }
  if (blockIdx.y == 0 && tid < n) c.lens[to[tid]] = lens[tid];
}

// ---- release -----------------------------------------------------------------------------------------
//
// First every entry is taken out of the table and one holder from its page, which leaves -1 in extra where there was
// none beside.  Then those are counted, range by range of ids, and stored in front of what is free.

// Column col of rows i0 .. i0 + n - 1, n up to kTogether.
__device__ __forceinline__ void free_column(const FreeCall& c, int i0, int n, int col) {
  int rows[kTogether], ids[kTogether];
#pragma unroll
  for (int j = 0; j < kTogether; ++j) {  // all read before the first exchange, which would keep them in order
    const int i = i0 + min(j, n - 1);
    rows[j] = j < n ? c.rows[i] : -1;
    if (c.begin && (col < c.begin[i] || col >= c.end[i])) rows[j] = -1;
    if ((unsigned)rows[j] >= (unsigned)c.n_rows) rows[j] = -1;
  }
#pragma unroll
  for (int j = 0; j < kTogether; ++j)  // by exchange: a row that is listed twice is released once
    ids[j] = rows[j] < 0 ? -1 : atomicExch(&c.table[(int64_t)rows[j] * c.table_width + col], -1);
  PageRun run{c.extra, c.n_pages};
#pragma unroll
  for (int j = 0; j < kTogether; ++j) run.take(ids[j], -1);
  run.flush(-1);
}
// The lengths of the rows from i0 on that are released whole, by the threads t < n.
__device__ __forceinline__ void free_lens(const FreeCall& c, int i0, int n, int t) {
  if (t < n && !c.begin && (unsigned)c.rows[i0 + t] < (unsigned)c.n_rows) c.lens[c.rows[i0 + t]] = 0;
}

__global__ __launch_bounds__(kThreads) void k_free_mark(FreeCall c) {
  const int i0 = (int)blockIdx.x * kTogether, n = min(kTogether, c.n - i0);
  for (int col = (int)blockIdx.y * kThreads + threadIdx.x; col < c.table_width; col += (int)gridDim.y * kThreads)
    free_column(c, i0, n, col);
  if (blockIdx.y == 0) free_lens(c, i0, n, threadIdx.x);
}

// Pages freed in each range of kFreePages.
__global__ __launch_bounds__(1024) void k_free_count(FreeCall c) {
  __shared__ int part[16];
  const int p0 = (int)blockIdx.x * kFreePages, n = min(kFreePages, c.n_pages - p0);  // n_pages may be 2^31 - 1: no sum past it
  int mine = 0;
  for (int i = threadIdx.x; i < n; i += 1024) mine += c.extra[p0 + i] < 0;
  mine = block_sum<1024>(mine, part);
  if (threadIdx.x == 0) c.counts[blockIdx.x] = mine;
  // the count taken so far, as the next launch's first workgroup may overwrite it before the others read it
  if (threadIdx.x == 0 && blockIdx.x == 0) c.counts[gridDim.x] = c.taken_in[0];
}

// The free list's front and the totals.  ONE: this workgroup is the only one, for up to 16384 pages; MARK: it also takes the
// entries out.
template <bool ONE, bool MARK> __global__ __launch_bounds__(1024) void k_free_store(FreeCall c) {
  __shared__ int part[16], bad_row;
  const int tid = threadIdx.x, taken = ONE ? c.taken_in[0] : c.counts[gridDim.x];
  constexpr int kEach = (ONE ? 2 : 1) * kFreePages / 1024;
  if (tid == 0) bad_row = 0;
  if constexpr (MARK) {
    const int groups = (c.n + kTogether - 1) / kTogether;
    for (int e = tid; e < groups * c.table_width; e += 1024) {
      const int g = e / c.table_width;
      free_column(c, g * kTogether, min(kTogether, c.n - g * kTogether), e - g * c.table_width);
    }
    free_lens(c, 0, c.n, tid);  // at most 1024 rows
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the counts are taken where the atomics of all waves have arrived
  }
  __syncthreads();
  // a thread takes up to kEach pages in a row: one scan for all of them; no load waits for another
  const int each = ONE ? (c.n_pages + 1023) / 1024 : kEach, p0 = (int)blockIdx.x * kFreePages + tid * each;
  int flags = 0, held[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int* p = &c.extra[min(p0 + j, c.n_pages - 1)];
    held[j] = 0;
    if (j < each) held[j] = MARK ? __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *p;
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j) flags |= (j < each && p0 + j < c.n_pages && held[j] < 0) << j;
  if (blockIdx.x == 0)
    for (int i = tid; i < c.n; i += 1024)
      if ((unsigned)c.rows[i] >= (unsigned)c.n_rows) bad_row = 1;
  int all, at = block_before<1024>(__builtin_popcount(flags), part, all);
  if constexpr (!ONE) {
    const int blocks = gridDim.x;
    int mine = 0, past = 0;
    for (int b = tid; b < blocks; b += 1024) {
      const int x = c.counts[b];
      mine += x;
      past += b < (int)blockIdx.x ? x : 0;
    }
    all = block_sum<1024>(mine, part);
    at += block_sum<1024>(past, part);
  }
  const int first = taken - all;  // negative: ids without a place are lost
  at += first;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (!(flags >> j & 1)) continue;
    c.extra[p0 + j] = 0;
    if (at >= 0 && at < c.n_free) c.free_list[at] = p0 + j;
    ++at;
  }
  if (blockIdx.x == 0 && tid == 0) {
    c.taken_out[0] = max(first, 0);
    c.taken_out[1] = (bad_row ? QVX_MAP_SEQUENCE : 0) | (taken < 0 ? QVX_MAP_NEGATIVE : 0) |
                     (first < 0 || taken > c.n_free ? QVX_MAP_PAGES : 0);
  }
}

// ---- compaction --------------------------------------------------------------------------------------
//
// Pages in use are those that the free list does not name.  With n of them, each of id n or above moves to an unused id
// below n, the r-th to the r-th in ascending order.  Every workgroup sets the free pages' bits in LDS for itself (one bit a page) and
// sums them up by words of kRun bits, so that any page's rank is a few population counts; then it takes its share of the
// outputs.  One launch; a second where the free list is rewritten in place, which the others read.

constexpr int kCompactThreads = 1024, kRun = 256;  // bits of a run

struct FreeBits {
  const uint32_t* bits;
  const int* runs;  // free pages before each run
  int n_pages;
  __device__ bool is_free(int p) const { return bits[p >> 5] >> (p & 31) & 1; }
  __device__ int free_before(int p) const {  // p up to n_pages
    int n = runs[p / kRun];
    for (int w = p / kRun * (kRun / 32); w < p >> 5; ++w) n += __builtin_popcount(bits[w]);
    return p & 31 ? n + __builtin_popcount(bits[p >> 5] & ((1u << (p & 31)) - 1)) : n;
  }
};

// The r-th free page (r below the free pages' number): bisection over the runs, then its words.
__device__ inline int free_at(const FreeBits& f, int r, int n_runs) {
  int lo = 0, hi = n_runs - 1;  // the last run with at most r free pages before it
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (f.runs[mid] <= r) lo = mid; else hi = mid - 1;
  }
  int left = r - f.runs[lo], w = lo * (kRun / 32);
  for (int n; left >= (n = __builtin_popcount(f.bits[w])); ++w) left -= n;
  uint32_t b = f.bits[w];
  for (; left; --left) b &= b - 1;
  return 32 * w + __builtin_ctz(b);
}

__global__ __launch_bounds__(kCompactThreads) void k_kv_compact(CompactCall c, bool in_place) {
  extern __shared__ uint32_t lds[];
  __shared__ int part[kCompactThreads / 64];
  const int tid = threadIdx.x, runs = c.n_pages / kRun + 1;
  const int whole = runs * (kRun / 32);  // words of whole runs
  int* sums = reinterpret_cast<int*>(lds + whole);
  for (int w = tid; w < whole; w += kCompactThreads) lds[w] = 0;
  __syncthreads();
  const int taken = min(max(c.taken[0], 0), c.n_free);
  for (int i = taken + tid; i < c.n_free; i += kCompactThreads) {
    const int id = c.free_list[i];
    if (page_ok(id, c.n_pages)) atomicOr(&lds[id >> 5], 1u << (id & 31));
  }
  __syncthreads();
  int free_pages = 0;
  for (int r0 = 0; r0 < runs; r0 += kCompactThreads) {
    const int r = r0 + tid;
    int n = 0;
    if (r < runs)
      for (int w = 0; w < kRun / 32; ++w) n += __builtin_popcount(lds[r * (kRun / 32) + w]);
    int total;
    const int before = block_before<kCompactThreads>(n, part, total);
    if (r < runs) sums[r] = free_pages + before;
    free_pages += total;
  }
  __syncthreads();
  const FreeBits f{lds, sums, c.n_pages};
  const int used = c.n_pages - free_pages;  // ids below it are in use afterwards
  const int moves = f.free_before(used);    // as many free ids below as used ones from it on
  const int used_low = used - moves;
  // Where page p, in use, lies afterwards.
  auto place = [&](int p) { return p < used ? p : free_at(f, p - f.free_before(p) - used_low, runs); };
  const int64_t step = (int64_t)gridDim.x * kCompactThreads, me = (int64_t)blockIdx.x * kCompactThreads + tid;
  for (int64_t i = me; i < c.entries; i += step) {
    const int id = c.table[i];
    c.table_out[i] = page_ok(id, c.n_pages) && !f.is_free(id) ? place(id) : id;
  }
  for (int64_t p = me; p < c.n_pages; p += step) {
    const bool gone = f.is_free((int)p);
    if (gone && p < used) continue;  // the page that moves here brings its count
    const int x = gone ? 0 : c.extra[p];
    if (!gone && p >= used) {
      const int to = place((int)p), r = (int)p - f.free_before((int)p) - used_low;
      c.extra_out[to] = x;
      c.pairs[2 * r] = (int)p;
      c.pairs[2 * r + 1] = to;
    }
    c.extra_out[p] = gone || p >= used ? 0 : x;
  }
  if (!in_place)
    for (int64_t i = me; i < c.n_free; i += step) {
      const int64_t id = used + (i - taken);
      c.free_out[i] = i < taken ? c.free_list[i] : id < c.n_pages ? (int)id : -1;
    }
  if (me == 0) {
    c.moved[0] = moves;
    c.moved[1] = used;
  }
}

__global__ __launch_bounds__(kThreads) void k_compact_list(CompactCall c) {
  const int taken = min(max(c.taken[0], 0), c.n_free), used = c.moved[1];
  for (int64_t i = taken + (int64_t)blockIdx.x * kThreads + threadIdx.x; i < c.n_free; i += (int64_t)gridDim.x * kThreads) {
    const int64_t id = used + (i - taken);
    c.free_out[i] = id < c.n_pages ? (int)id : -1;
  }
}

// ---- copies ------------------------------------------------------------------------------------------
//
// Units of 16 KB (64 bytes a thread in four loads that go out together) of a pair's page of K or V of a cache, taken in
// turn by as many workgroups as the card holds: the number of pairs is the device's.  What is stored is marked as not needed
// again: 128 pages of 16 layers 55.9 us with their forks and releases, 59.3 without the mark, 59.9 with loads marked as well;
// 1080 of 8 layers 237, 239 and 232.

constexpr int kCopyUnit = 16 << 10, kCopyWgs = 2048;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(kThreads) void k_kv_copy(CopyCall c, int parts) {
  const int each = c.n_caches * 2 * parts;
  const int count = c.count ? min(max(*c.count, 0), c.most) : c.most;
  for (int pair = blockIdx.y; pair < count; pair += (int)gridDim.y) {
    const int src = c.pairs[2 * (int64_t)pair], dst = c.pairs[2 * (int64_t)pair + 1];
    if (!page_ok(src, c.n_pages) || !page_ok(dst, c.n_pages) || src == dst) continue;
    for (int u = blockIdx.x; u < each; u += (int)gridDim.x) {
      const int plane = u / parts, part = u - plane * parts;
      const auto& x = c.cache[plane >> 1];
      uint8_t* base = plane & 1 ? x.v : x.k;
      const int64_t at = (int64_t)part * kCopyUnit + 16 * threadIdx.x;
      const uint8_t* from = base + src * x.stride;
      uint8_t* to = base + dst * x.stride;
      u32x4 w[4];  // a vector type of the compiler's: an array of structures is moved to LDS, each load waited for
#pragma unroll
      for (int j = 0; j < 4; ++j)  // past the page its last bytes again: a load in a branch would be waited for there
        w[j] = *reinterpret_cast<const u32x4*>(from + min(at + j * 16 * kThreads, c.page_bytes - 16));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (at + j * 16 * kThreads < c.page_bytes) __builtin_nontemporal_store(w[j], reinterpret_cast<u32x4*>(to + at + j * 16 * kThreads));
    }
  }
}

}  // namespace

void launch_kv_fork(const ForkCall& c, bool alias, hipStream_t s) {
  // Totals that lie on what the others read are stored by a launch behind them.
  const int groups = (c.n + kTogether - 1) / kTogether, cols = std::min((c.table_width + kThreads - 1) / kThreads, 64);
  k_kv_fork<<<dim3(groups, cols), kThreads, 0, s>>>(c, alias ? kForkRows : kForkRows | kForkTotals);
  if (alias) k_kv_fork<<<1, kThreads, 0, s>>>(c, kForkTotals);
}

void launch_kv_free(const FreeCall& c, hipStream_t s) {
  const bool one = c.n_pages <= 2 * kFreePages;
  const int groups = (c.n + kTogether - 1) / kTogether, cols = std::min((c.table_width + kThreads - 1) / kThreads, 64);
  // One workgroup for all of it up to two columns a thread; its launch alone takes less than two.
  if (one && (int64_t)groups * c.table_width <= 2048 && c.n <= 1024) {
    k_free_store<true, true><<<1, 1024, 0, s>>>(c);
    return;
  }
  k_free_mark<<<dim3(groups, cols), kThreads, 0, s>>>(c);
  if (one) {
    k_free_store<true, false><<<1, 1024, 0, s>>>(c);
    return;
  }
  const int blocks = (c.n_pages - 1) / kFreePages + 1;
  k_free_count<<<blocks, 1024, 0, s>>>(c);
  k_free_store<false, false><<<blocks, 1024, 0, s>>>(c);
}

bool launch_kv_compact(const CompactCall& c, bool in_place, hipStream_t s) {
  static LdsLimit lim;
  const int runs = c.n_pages / kRun + 1;
  const size_t lds = (size_t)runs * (kRun / 32) * 4 + (size_t)runs * 4;
  if (!lds_ready(reinterpret_cast<const void*>(&k_kv_compact), lim, lds)) return false;
  const int64_t most = std::max<int64_t>(std::max<int64_t>(c.entries, c.n_pages), c.n_free);
  const int wgs = (int)std::min<int64_t>(256, (most + kCompactThreads - 1) / kCompactThreads);
  k_kv_compact<<<wgs, kCompactThreads, lds, s>>>(c, in_place);
  if (in_place) k_compact_list<<<std::max(1, std::min(256, (c.n_free + kThreads - 1) / kThreads)), kThreads, 0, s>>>(c);
  return true;
}

void launch_kv_copy(const CopyCall& c, hipStream_t s) {
  const int parts = (int)((c.page_bytes + kCopyUnit - 1) / kCopyUnit), each = c.n_caches * 2 * parts;
  const int wide = std::min(each, kCopyWgs), high = std::min(c.most, std::max(1, kCopyWgs / wide));
  k_kv_copy<<<dim3(wide, high), kThreads, 0, s>>>(c, parts);
}

}  // namespace qvx
