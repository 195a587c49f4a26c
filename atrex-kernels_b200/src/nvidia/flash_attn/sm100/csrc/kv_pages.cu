// Page bookkeeping of paged KV caches: fork / free (reassign) and compact, declared in include/atrex_kvpages_sm100.h.
//
// The decisions (who keeps an unfinished page, which free page goes where) are prefix sums over the batch and the
// pool; they run on the device, so a serving loop never waits for a length or a count.  The work is the copies: every
// copied byte is read and written once, bound by HBM.  Destinations are pages that were free before the call and
// sources are pages that were held, so no page is both and the copies need no order.
//
// Small pools take one kernel whose CTAs each make the whole plan for themselves.  In larger ones, reassign: one CTA makes
// the list of copies (a batch has few rows; the free pages it needs are found by scanning the counts from the front until
// there are enough) while the others copy the counts; a second kernel writes tables and counts and copies the tokens.
// compact: per-chunk counts, then lists, then tables, counts and copies.
#include <algorithm>
#include <atomic>
#include <cstring>

#include "atrex_kvpages_sm100.h"
#include "fa_kernels.cuh"

namespace atrex_sm100 {
namespace {

constexpr int kThreads = 256;
constexpr int kPlanThreads = 1024;
constexpr int kChunk = 1024;               // pages per CTA of the compaction's listing kernel
constexpr int kMaxCaches = 256;            // caches per launch; their descriptions travel as kernel arguments (12 KB)
constexpr int kFewCaches = 16, kSomeCaches = 64;   // smaller argument blocks for fewer
constexpr int kSharedRows = 4096;          // rows whose parents fit the planning CTA's shared memory

// A cache as runs of bytes: a page is `outer` x (rows, unless they are part of the run) runs at the given strides.
struct CacheDesc {
  uint8_t* base;
  long long page_stride, row_stride, outer_stride;
  int outer;             // runs beside each other: heads, or 1 where a token's heads lie together
  int run_bytes;         // bytes per row of a run
  int rows_in_run;       // 1: the rows of a run follow each other without gaps
  int vec;               // bytes per access: 16, 8, 4, 2 or 1
};
template <int N>
struct Caches {
  CacheDesc c[N];
  int n;
};

struct PageParams {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* refs;
  const int32_t* parents;
  int32_t* new_table;
  int32_t* new_lens;
  int32_t* new_refs;
  int32_t* page_map;
  int32_t* count;
  long long table_stride;
  int batch, width, pages, page_size;
  // scratch
  int32_t* header;       // [0] copies, [1] pages missing / live pages
  int32_t* job_src;      // [max(batch, pages)] source page of a copy
  int32_t* job_dst;      // destination page
  int32_t* job_rows;     // [batch] tokens of a copy (reassign)
  int32_t* row_job;      // [batch] copy that a row waits for, -1
  int32_t* first;        // [batch] lowest row that continues a row's sequence (reassign)
  int32_t* rank;         // [pages] a page's place among its kind (compact)
  int32_t* chunk_live;   // [chunks]
};

__device__ __forceinline__ int pages_of(const PageParams& p, int len) {
  const int n = len <= 0 ? 0 : (int)(((long long)len + p.page_size - 1) / p.page_size);
  return n < p.width ? n : p.width;
}

// Exclusive prefix sum of one value per thread over the CTA; `total` = the sum.  `shared`: 33 words.
__device__ __forceinline__ int block_scan(int v, int* shared, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();                         // the previous round's readers are done
  if (lane == 31) shared[warp] = x;
  __syncthreads();
  if (warp == 0) {
    const int s = lane < warps ? shared[lane] : 0;
    int t = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += y;
    }
    if (lane < warps) shared[lane] = t - s;
    if (lane == 31) shared[32] = t;
  }
  __syncthreads();
  total = shared[32];
  return x - v + shared[warp];
}

// ---- reassign, first kernel: CTA 0 plans, the others copy the counts ----
__global__ void __launch_bounds__(kPlanThreads) atrex_sm100_kvpages_plan_kernel(const __grid_constant__ PageParams p) {
  if (blockIdx.x > 0) {
    const long long step = (long long)(gridDim.x - 1) * kPlanThreads;
    for (long long i = (long long)(blockIdx.x - 1) * kPlanThreads + threadIdx.x; i < p.pages; i += step)
      p.new_refs[i] = p.refs[i];
    return;
  }
  __shared__ int shared[33], s_first[kSharedRows], s_parents[kSharedRows];
  const int tid = threadIdx.x;
  const bool small = p.batch <= kSharedRows;
  int32_t* const first = small ? s_first : p.first;
  const int32_t* const parents = small ? s_parents : p.parents;
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    first[b] = 0x7fffffff;
    if (small) s_parents[b] = p.parents[b];
  }
  __syncthreads();
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    const int parent = parents[b];
    if (parent >= 0 && parent < p.batch) atomicMin(&first[parent], b);
  }
  __syncthreads();
  int needed = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int need = 0, src = 0, rows = 0;
    if (b < p.batch) {
      const int parent = parents[b];
      if (parent >= 0 && parent < p.batch) {
        const int len = max(p.lens[parent], 0), full = len / p.page_size;
        const int keeper = parents[parent] == parent ? parent : *(volatile int*)&first[parent];
        rows = len % p.page_size;
        if (rows > 0 && full < p.width && keeper != b) {
          src = p.table[(long long)parent * p.table_stride + full];
          need = src >= 0 && src < p.pages;
        }
      }
    }
    int total;
    const int at = needed + block_scan(need, shared, total);
    if (b < p.batch) p.row_job[b] = need ? at : -1;
    if (need) {
      p.job_src[at] = src;
      p.job_rows[at] = rows;
    }
    needed += total;
  }
  // the lowest free pages, four counts a thread and round
  int found = 0;
  for (long long i0 = 0; i0 < p.pages && found < needed; i0 += 4 * kPlanThreads) {
    const long long i = i0 + 4 * tid;
    int is_free[4], mine = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      is_free[u] = i + u < p.pages && p.refs[i + u] <= 0;
      mine += is_free[u];
    }
    int total;
    int at = found + block_scan(mine, shared, total);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (is_free[u]) {
        if (at < needed) p.job_dst[at] = (int)(i + u);
        ++at;
      }
    found += total;
  }
  if (tid == 0) {
    const int missing = needed > found ? needed - found : 0;
    p.header[0] = missing ? 0 : needed;
    p.header[1] = missing;
    *p.count = missing;
  }
}

// ---- the copies, shared by both operators: copy `job` of every cache, sliced ----
__device__ __forceinline__ void copy_bytes(uint8_t* dst, const uint8_t* src, int vec) {
  switch (vec) {
    case 16: *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src); break;
    case 8: *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src); break;
    case 4: *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src); break;
    case 2: *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src); break;
    default: *dst = *src;
  }
}

constexpr int kInFlight = 4;
constexpr int kSlice = kThreads * kInFlight;        // accesses per unit of work

// Accesses `at .. at + kSlice` of one page of one cache, `rows` tokens of it, by kThreads threads.
__device__ __forceinline__ void copy_slice(const CacheDesc& c, int src_page, int dst_page, int rows, long long at, int tid) {
  const uint8_t* src = c.base + src_page * c.page_stride;
  uint8_t* dst = c.base + dst_page * c.page_stride;
  const int per_run = (c.rows_in_run ? rows * c.run_bytes : c.run_bytes) / c.vec;
  const long long runs = c.rows_in_run ? c.outer : (long long)c.outer * rows;
  const long long total = runs * per_run;
  long long off[kInFlight];
#pragma unroll
  for (int u = 0; u < kInFlight; ++u) {
    const long long v = at + u * kThreads + tid;
    off[u] = -1;
    if (v >= total) continue;
    if (runs == 1) {
      off[u] = v * c.vec;
    } else {
      const int run = (int)(v / per_run);
      const int in_run = (int)(v - (long long)run * per_run);
      const int outer = c.rows_in_run ? run : run % c.outer, row = c.rows_in_run ? 0 : run / c.outer;
      off[u] = outer * c.outer_stride + row * c.row_stride + (long long)in_run * c.vec;
    }
  }
  if (c.vec == 16) {
    uint4 x[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (off[u] >= 0) x[u] = *reinterpret_cast<const uint4*>(src + off[u]);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (off[u] >= 0) *reinterpret_cast<uint4*>(dst + off[u]) = x[u];
  } else {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (off[u] >= 0) copy_bytes(dst + off[u], src + off[u], c.vec);
  }
}

// Units of work: (copy, cache, slice), slice fastest; CTA `cta` of `ctas` takes every ctas-th.
template <int N>
__device__ __forceinline__ void copy_jobs(const PageParams& p, const Caches<N>& caches, int slices, bool whole_pages,
                                          int cta, int ctas) {
  const long long units = (long long)p.header[0] * caches.n * slices;
  for (long long unit = cta; unit < units; unit += ctas) {
    const int slice = (int)(unit % slices);
    const long long rest = unit / slices;
    const CacheDesc& c = caches.c[rest % caches.n];
    const int job = (int)(rest / caches.n);
    copy_slice(c, p.job_src[job], p.job_dst[job], whole_pages ? p.page_size : p.job_rows[job], (long long)slice * kSlice, threadIdx.x);
  }
}

// ---- reassign, second kernel: tables, counts and copies ----
template <int N>
__global__ void __launch_bounds__(kThreads)
atrex_sm100_kvpages_apply_kernel(const __grid_constant__ PageParams p, const __grid_constant__ Caches<N> caches, int slices,
                                 int meta_ctas) {
  if ((int)blockIdx.x >= meta_ctas) {
    copy_jobs(p, caches, slices, false, blockIdx.x - meta_ctas, gridDim.x - meta_ctas);
    return;
  }
  const bool unchanged = p.header[1] > 0;
  const int lane = threadIdx.x & 31, warps = meta_ctas * (kThreads / 32);
  for (int b = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); b < p.batch; b += warps) {
    const int parent = unchanged ? b : p.parents[b];
    const bool alive = parent >= 0 && parent < p.batch;
    const int len = alive ? p.lens[parent] : 0, n = pages_of(p, len);
    const int job = unchanged || !alive ? -1 : p.row_job[b];
    const int own = job >= 0 ? p.job_dst[job] : -1, own_at = job >= 0 ? max(len, 0) / p.page_size : -1;
    const int old_n = parent == b ? 0 : pages_of(p, p.lens[b]);       // a row that continues itself gives nothing up
    for (int i = lane; i < p.width; i += 32) {
      int page = -1;
      if (i < n) page = i == own_at ? own : p.table[parent * p.table_stride + i];
      p.new_table[(long long)b * p.width + i] = page;
      if (parent == b) continue;
      if (page >= 0 && page < p.pages) atomicAdd(&p.new_refs[page], 1);
      if (i < old_n) {
        const int old = p.table[b * p.table_stride + i];
        if (old >= 0 && old < p.pages) atomicSub(&p.new_refs[old], 1);
      }
    }
    if (lane == 0) p.new_lens[b] = len;
  }
}

// ---- compact ----
__global__ void __launch_bounds__(kThreads) atrex_sm100_kvpages_count_kernel(const __grid_constant__ PageParams p) {
  __shared__ int shared[33];
  int live = 0;
#pragma unroll
  for (int i = 0; i < kChunk / kThreads; ++i) {
    const long long page = (long long)blockIdx.x * kChunk + i * kThreads + threadIdx.x;
    live += page < p.pages && p.refs[page] > 0;
  }
  int total;
  block_scan(live, shared, total);
  if (threadIdx.x == 0) p.chunk_live[blockIdx.x] = total;
}

// Lists of the pages that move and of where they go; rank[page] = a page's place in its list.
__global__ void __launch_bounds__(kThreads) atrex_sm100_kvpages_list_kernel(const __grid_constant__ PageParams p) {
  __shared__ int shared[33];
  const int tid = threadIdx.x, chunks = gridDim.x;
  int sum = 0, before = 0;
  for (int i = tid; i < chunks; i += kThreads) {
    const int n = p.chunk_live[i];
    sum += n;
    if (i < (int)blockIdx.x) before += n;
  }
  int live, prefix;
  block_scan(sum, shared, live);
  block_scan(before, shared, prefix);
  // live pages before page `live`: whole chunks, then part of the one it lies in
  const int edge = live / kChunk;
  int part = 0;
  for (int i = tid; i < edge; i += kThreads) part += p.chunk_live[i];
#pragma unroll 8
  for (int i = edge * kChunk + tid; i < live; i += kThreads) part += p.refs[i] > 0;
  int stay;
  block_scan(part, shared, stay);
  constexpr int kPer = kChunk / kThreads;
  const long long first = (long long)blockIdx.x * kChunk + tid * kPer;
  int flags = 0, mine = 0;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int is_live = first + u < p.pages && p.refs[first + u] > 0;
    flags |= is_live << u;
    mine += is_live;
  }
  int total;
  int at = prefix + block_scan(mine, shared, total);       // live pages before this thread's first
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const long long page = first + u;
    if (page >= p.pages) break;
    const bool is_live = (flags >> u) & 1;
    if (is_live && page >= live) {
      p.job_src[at - stay] = (int)page;
      p.rank[page] = at - stay;
    } else if (!is_live && page < live) {
      p.job_dst[page - at] = (int)page;
      p.rank[page] = (int)(page - at);
    }
    at += is_live;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.header[0] = live - stay;
    p.header[1] = live;
    *p.count = live;
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads)
atrex_sm100_kvpages_move_kernel(const __grid_constant__ PageParams p, const __grid_constant__ Caches<N> caches, int slices,
                                int meta_ctas) {
  if ((int)blockIdx.x >= meta_ctas) {
    copy_jobs(p, caches, slices, true, blockIdx.x - meta_ctas, gridDim.x - meta_ctas);
    return;
  }
  const int live = p.header[1];
  const long long step = (long long)meta_ctas * kThreads, at = (long long)blockIdx.x * kThreads + threadIdx.x;
  for (long long i = at; i < p.pages; i += step) {
    const int refs = p.refs[i];
    p.page_map[i] = refs <= 0 ? -1 : i < live ? (int)i : p.job_dst[p.rank[i]];
    p.new_refs[i] = i >= live ? 0 : refs > 0 ? refs : p.refs[p.job_src[p.rank[i]]];
  }
  for (long long i = at; i < (long long)p.batch * p.width; i += step) {
    const int b = (int)(i / p.width), col = (int)(i - (long long)b * p.width);
    int page = -1;
    if (col < pages_of(p, p.lens[b])) {
      page = p.table[b * p.table_stride + col];
      // a page that the counts call free stays where it is
      if (page >= live && page < p.pages && p.refs[page] > 0) page = p.job_dst[p.rank[page]];
    }
    p.new_table[i] = page;
  }
}

// ---- small pools: one kernel, every CTA plans for itself ----
// A second launch costs ~3 us of the host and, unless the plan is long, more of the device than a plan in every CTA.
// Microseconds a call, 20 calls in one graph, one kernel / two: forks of 16 rows in 1 024 pages 5.8 / 6.8, of 32 in 2 048
// 6.1 / 7.1, of 64 in 4 096 ~9 / 7.3 (one CTA adds up all counts); compaction of 512 pages 6.0 / 7.2, of 1 024 8.8 / 9.1, of
// 2 048 12.1 / 11.1, of 4 096 21.4 / 22.1, of 16 384 as long either way.
constexpr int kOnePages = 16384;           // compaction: page numbers fit 14 bits, and a CTA looks at 16 pages a thread
constexpr int kForkPages = 2048, kForkCells = 8192;   // reassign: pages, and entries of the table
constexpr int kOneRows = kPlanThreads;     // rows a CTA plans in one pass
constexpr int kGroups = kPlanThreads / kThreads;   // copying groups of a CTA

template <int N, typename Job>
__device__ __forceinline__ void copy_units(const PageParams& p, const Caches<N>& caches, int slices, int jobs, int worker,
                                           int workers, const Job& job) {
  const int tid = threadIdx.x % kThreads;
  const long long units = (long long)jobs * caches.n * slices;
  for (long long unit = (long long)worker * kGroups + threadIdx.x / kThreads; unit < units; unit += (long long)workers * kGroups) {
    const int slice = (int)(unit % slices);
    const long long rest = unit / slices;
    int src, dst, rows;
    job((int)(rest / caches.n), src, dst, rows);
    copy_slice(caches.c[rest % caches.n], src, dst, rows, (long long)slice * kSlice, tid);
  }
}

// CTA 0 writes the counts, the others tables, lengths and copies.
template <int N>
__global__ void __launch_bounds__(kPlanThreads)
atrex_sm100_kvpages_reassign_kernel(const __grid_constant__ PageParams p, const __grid_constant__ Caches<N> caches, int slices) {
  __shared__ int shared[33], s_first[kOneRows], s_parents[kOneRows], s_lens[kOneRows], row_job[kOneRows];
  __shared__ int job_src[kOneRows], job_dst[kOneRows], job_rows[kOneRows];
  extern __shared__ int delta[];           // CTA 0: what the call adds to each page's count
  const int tid = threadIdx.x;
  int parent = -1;
  if (tid < p.batch) {
    parent = s_parents[tid] = p.parents[tid];
    s_lens[tid] = p.lens[tid];
    s_first[tid] = 0x7fffffff;
  }
  __syncthreads();
  const bool alive = parent >= 0 && parent < p.batch;
  if (alive) atomicMin(&s_first[parent], tid);
  __syncthreads();
  int need = 0, src = 0, rows = 0;
  if (alive) {
    const int len = max(s_lens[parent], 0), full = len / p.page_size;
    const int keeper = s_parents[parent] == parent ? parent : s_first[parent];
    rows = len % p.page_size;
    if (rows > 0 && full < p.width && keeper != tid) {
      src = p.table[(long long)parent * p.table_stride + full];
      need = src >= 0 && src < p.pages;
    }
  }
  int needed;
  const int mine = block_scan(need, shared, needed);
  row_job[tid] = need ? mine : -1;
  if (need) {
    job_src[mine] = src;
    job_rows[mine] = rows;
  }
  // the lowest free pages, four counts a thread and round
  int found = 0;
  for (int i0 = 0; i0 < p.pages && found < needed; i0 += 4 * kPlanThreads) {
    const int i = i0 + 4 * tid;
    int is_free[4], free_here = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      is_free[u] = i + u < p.pages && p.refs[i + u] <= 0;
      free_here += is_free[u];
    }
    int total;
    int at = found + block_scan(free_here, shared, total);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (is_free[u]) {
        if (at < needed) job_dst[at] = i + u;
        ++at;
      }
    found += total;
  }
  __syncthreads();
  const int missing = needed > found ? needed - found : 0;
  const bool unchanged = missing > 0;
  const int cells = p.batch * p.width;
  // what row b holds in column i after the call, before the call
  auto page_after = [&](int b, int par, int i) {
    const int len = s_lens[par];
    if (i >= pages_of(p, len)) return -1;
    const int job = unchanged ? -1 : row_job[b];
    return job >= 0 && i == max(len, 0) / p.page_size ? job_dst[job] : p.table[par * p.table_stride + i];
  };
  if (blockIdx.x == 0) {
    if (tid == 0) *p.count = missing;
    for (int i = tid; i < p.pages; i += kPlanThreads) delta[i] = 0;
    __syncthreads();
    for (int at = tid; at < cells && !unchanged; at += kPlanThreads) {
      const int b = at / p.width, i = at - b * p.width, par = s_parents[b];
      if (par == b) continue;              // a row that continues itself gives nothing up and takes nothing
      const int page = par >= 0 && par < p.batch ? page_after(b, par, i) : -1;
      if (page >= 0 && page < p.pages) atomicAdd(&delta[page], 1);
      if (i < pages_of(p, s_lens[b])) {
        const int old = p.table[b * p.table_stride + i];
        if (old >= 0 && old < p.pages) atomicSub(&delta[old], 1);
      }
    }
    __syncthreads();
    for (int i = tid; i < p.pages; i += kPlanThreads) p.new_refs[i] = p.refs[i] + delta[i];
    return;
  }
  const int worker = blockIdx.x - 1, workers = gridDim.x - 1;
  for (int at = worker * kPlanThreads + tid; at < cells; at += workers * kPlanThreads) {
    const int b = at / p.width, par = unchanged ? b : s_parents[b];
    p.new_table[at] = par >= 0 && par < p.batch ? page_after(b, par, at - b * p.width) : -1;
  }
  if (worker == 0 && tid < p.batch) {
    const int par = unchanged ? tid : parent;
    p.new_lens[tid] = par >= 0 && par < p.batch ? s_lens[par] : 0;
  }
  copy_units(p, caches, slices, unchanged ? 0 : needed, worker, workers, [&](int job, int& from, int& to, int& n) {
    from = job_src[job];
    to = job_dst[job];
    n = job_rows[job];
  });
}

// The first meta_ctas CTAs write counts, page map and tables, the others copy.
template <int N>
__global__ void __launch_bounds__(kPlanThreads)
atrex_sm100_kvpages_compact_kernel(const __grid_constant__ PageParams p, const __grid_constant__ Caches<N> caches, int slices,
                                   int meta_ctas) {
  __shared__ int shared[33], s_stay;
  extern __shared__ uint16_t lists[];
  constexpr uint16_t kFree = 0x8000;
  uint16_t* const moved = lists;                            // [pages] where a live page goes; kFree | source of a page that fills
  uint16_t* const job_src = lists + p.pages;                // [pages / 2] pages that move, in order
  uint16_t* const job_dst = job_src + (p.pages + 1) / 2;    // [pages / 2] pages that they fill
  const int tid = threadIdx.x, per = (p.pages + kPlanThreads - 1) / kPlanThreads;
  const int first = tid * per, last = min(first + per, p.pages);
  int flags = 0, mine = 0;
#pragma unroll 4
  for (int i = first; i < last; ++i) {
    const int is_live = p.refs[i] > 0;
    flags |= is_live << (i - first);
    mine += is_live;
  }
  int live;
  const int before = block_scan(mine, shared, live);        // live pages before this thread's first
  // `stay`: live pages before page `live`, known to the thread that has that page; all of them when no page is free
  if (tid == 0 && live == p.pages) s_stay = live;
  if (live >= first && live < last) s_stay = before + __popc(flags & ((1 << (live - first)) - 1));
  __syncthreads();
  const int stay = s_stay;
  int at = before;
  for (int i = first; i < last; ++i) {
    const bool is_live = (flags >> (i - first)) & 1;
    if (is_live && i >= live) job_src[at - stay] = (uint16_t)i;
    else if (!is_live && i < live) job_dst[i - at] = (uint16_t)i;
    at += is_live;
  }
  __syncthreads();
  if ((int)blockIdx.x >= meta_ctas) {
    copy_units(p, caches, slices, live - stay, blockIdx.x - meta_ctas, gridDim.x - meta_ctas,
               [&](int job, int& from, int& to, int& n) {
                 from = job_src[job];
                 to = job_dst[job];
                 n = p.page_size;
               });
    return;
  }
  at = before;
  for (int i = first; i < last; ++i) {
    const bool is_live = (flags >> (i - first)) & 1;
    moved[i] = is_live ? (i < live ? (uint16_t)i : job_dst[at - stay]) : (uint16_t)(kFree | (i < live ? job_src[i - at] : 0));
    at += is_live;
  }
  __syncthreads();
  const int step = meta_ctas * kPlanThreads, start = blockIdx.x * kPlanThreads + tid;
  for (int i = start; i < p.pages; i += step) {
    const uint16_t m = moved[i];
    p.page_map[i] = m & kFree ? -1 : (int)m;
    p.new_refs[i] = i >= live ? 0 : p.refs[m & kFree ? m & ~kFree : i];
  }
  const int cells = p.batch * p.width;
  for (int c = start; c < cells; c += step) {
    const int b = c / p.width, col = c - b * p.width;
    int page = -1;
    if (col < pages_of(p, p.lens[b])) {
      page = p.table[b * p.table_stride + col];
      // a page that the counts call free stays where it is
      if (page >= live && page < p.pages && !(moved[page] & kFree)) page = moved[page];
    }
    p.new_table[c] = page;
  }
  if (start == 0) *p.count = live;
}

// ---- host ----
uint64_t align_up(uint64_t x) { return (x + 255) / 256 * 256; }
struct Scratch {
  uint64_t header, src, dst, rows, row_job, first, rank, chunks, bytes;
};
Scratch scratch_of(int64_t batch, int64_t pages) {
  Scratch s;
  const int64_t jobs = batch > pages ? batch : pages;
  uint64_t at = 0;
  auto take = [&](int64_t n) {
    const uint64_t here = at;
    at = align_up(at + 4 * (uint64_t)n);
    return here;
  };
  s.header = take(2);
  s.src = take(jobs);
  s.dst = take(jobs);
  s.rows = take(batch);
  s.row_job = take(batch);
  s.first = take(batch);
  s.rank = take(pages);
  s.chunks = take(pages / kChunk + 1);
  s.bytes = at;
  return s;
}

int check(const atrex_kvpages_sm100_params* p, bool reassign) {
  if (p == nullptr) return report_failure(ATREX_FA_INVALID_VALUE, "parameter block is NULL");
  if (p->struct_bytes != sizeof(*p) || p->abi_version != ATREX_KVPAGES_SM100_ABI_VERSION)
    return report_failure(ATREX_FA_ABI_MISMATCH, "struct_bytes / abi_version do not match this library");
  if (p->batch < 0 || p->width < 0 || p->num_pages < 0 || p->page_size <= 0 || p->num_caches < 0 || p->table_row_stride < 0)
    return report_failure(ATREX_FA_INVALID_VALUE, "negative size");
  const bool rows = p->batch > 0, cells = rows && p->width > 0, pages = p->num_pages > 0;
  if (p->count == nullptr || (cells && (p->block_table == nullptr || p->new_table == nullptr)) ||
      (rows && p->seq_lens == nullptr) || (pages && (p->ref_counts == nullptr || p->new_refs == nullptr)) ||
      (p->num_caches > 0 && (p->caches == nullptr || p->bases == nullptr)))
    return report_failure(ATREX_FA_INVALID_VALUE, "a required pointer is NULL");
  if (reassign ? rows && (p->parents == nullptr || p->new_lens == nullptr) : pages && p->page_map == nullptr)
    return report_failure(ATREX_FA_INVALID_VALUE, "parents / new_lens / page_map is NULL");
  for (int i = 0; i < p->num_caches; ++i) {
    const atrex_kvpages_sm100_cache& c = p->caches[i];
    if (c.heads <= 0 || c.row_bytes <= 0 || (pages && p->bases[i] == nullptr))
      return report_failure(ATREX_FA_INVALID_VALUE, "a cache has no base, heads or row bytes");
    if (c.page_stride < 0 || c.row_stride < 0 || c.head_stride < 0 ||
        (int64_t)c.row_bytes * c.heads * p->page_size > 0x7fffffffll)
      return report_failure(ATREX_FA_UNSUPPORTED, "a cache stride is negative or a page is 2 GB or larger");
  }
  return ATREX_FA_OK;
}

CacheDesc describe(const atrex_kvpages_sm100_cache& c, void* base, int page_size, bool whole_pages) {
  CacheDesc d;
  d.base = static_cast<uint8_t*>(base);
  d.page_stride = c.page_stride;
  d.row_stride = c.row_stride;
  d.outer_stride = c.head_stride;
  d.outer = c.heads;
  d.run_bytes = c.row_bytes;
  if (c.heads == 1 || c.head_stride == c.row_bytes) {       // a token's heads lie together
    d.run_bytes = c.row_bytes * c.heads;
    d.outer = 1;
    d.outer_stride = 0;
  }
  d.rows_in_run = page_size == 1 || c.row_stride == d.run_bytes;
  if (whole_pages && d.rows_in_run && d.outer > 1 && c.head_stride == (int64_t)d.run_bytes * page_size) {
    d.run_bytes *= d.outer;                                 // heads follow each other: the page is one run
    d.outer = 1;
    d.outer_stride = 0;
  }
  // the widest access that every address of the cache allows
  uint64_t all = reinterpret_cast<uintptr_t>(d.base) | (uint64_t)d.page_stride | (uint64_t)d.run_bytes |
                 (uint64_t)d.outer_stride | (d.rows_in_run ? 0ull : (uint64_t)d.row_stride);
  d.vec = 16;
  while (all % d.vec != 0) d.vec /= 2;
  return d;
}

// Descriptions of n caches from `done` on; returns the slices of a page.
template <int N>
int describe_caches(Caches<N>& caches, const atrex_kvpages_sm100_params* p, int done, int n, bool reassign) {
  caches.n = n;
  long long most = 0;
  for (int i = 0; i < n; ++i) {
    caches.c[i] = describe(p->caches[done + i], p->bases[done + i], p->page_size, !reassign);
    const CacheDesc& c = caches.c[i];
    most = std::max(most, (long long)c.outer * c.run_bytes * p->page_size / c.vec);
  }
  return (int)std::max<long long>(1, (most + kSlice - 1) / kSlice);
}

// The whole call in one kernel.
template <int N>
cudaError_t launch_one(const PageParams& k, const atrex_kvpages_sm100_params* p, int sms, bool reassign, cudaStream_t stream) {
  Caches<N> caches;
  const int slices = describe_caches(caches, p, 0, p->num_caches, reassign);
  const long long jobs = reassign ? p->batch : p->num_pages / 2;
  const long long cells = ((long long)p->batch * p->width + kPlanThreads - 1) / kPlanThreads;
  const long long copies = (jobs * p->num_caches * slices + kGroups - 1) / kGroups;
  // shared memory beyond the default, once per device
  static std::atomic<int> ready[64];
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(atrex_sm100_kvpages_compact_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)(sizeof(uint16_t) * (2 * kOnePages + 2)));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) ready[dev].store(1, std::memory_order_release);
  }
  if (reassign)
    return launch_kernel(atrex_sm100_kvpages_reassign_kernel<N>,
                         dim3(1 + (unsigned)std::min<long long>(std::max(std::max(copies, cells), 1ll), 2 * sms)),
                         dim3(kPlanThreads), sizeof(int) * p->num_pages, stream, k, caches, slices);
  const int meta = (int)std::min<long long>(std::max(cells, ((long long)p->num_pages + kPlanThreads - 1) / kPlanThreads) + 1, 16);
  // all of the metadata CTAs, whose stride counts on each other, and one that copies at least, however few SMs are asked for
  const long long copying = std::min<long long>(copies, std::max<long long>(1, 2ll * sms - meta));
  return launch_kernel(atrex_sm100_kvpages_compact_kernel<N>, dim3((unsigned)(meta + copying)), dim3(kPlanThreads),
                       sizeof(uint16_t) * (2ull * p->num_pages + 2), stream, k, caches, slices, meta);
}

// The second kernel over n caches from `done` on; the first such launch writes tables and counts too.
template <int N>
cudaError_t launch_copies(const PageParams& k, const atrex_kvpages_sm100_params* p, int done, int n, int sms,
                          long long meta_work, bool reassign, cudaStream_t stream) {
  Caches<N> caches;
  const int slices = describe_caches(caches, p, done, n, reassign);
  const int meta = done == 0 ? (int)std::max<long long>(1, std::min<long long>(meta_work, 4 * sms)) : 0;
  const long long jobs = reassign ? p->batch : p->num_pages;
  const long long copies = std::min<long long>(jobs * n * slices, 8ll * sms);
  const unsigned grid = (unsigned)(meta + copies);
  if (grid == 0) return cudaSuccess;
  return launch_kernel(reassign ? atrex_sm100_kvpages_apply_kernel<N> : atrex_sm100_kvpages_move_kernel<N>, dim3(grid),
                       dim3(kThreads), 0, stream, k, caches, slices, meta);
}

int run(const atrex_kvpages_sm100_params* p, void* workspace, uint64_t workspace_bytes, void* stream_ptr, bool reassign) {
  clear_failure();
  int st = check(p, reassign);
  if (st != ATREX_FA_OK) return st;
  const Scratch s = scratch_of(p->batch, p->num_pages);
  if (workspace == nullptr || workspace_bytes < s.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return report_failure(ATREX_FA_WORKSPACE_TOO_SMALL, "workspace missing, misaligned or too small");
  int sms = 0;
  st = current_sm_count(&sms);
  if (st != ATREX_FA_OK) return st;
  if (p->sm_count > 0) sms = p->sm_count;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto at = [&](uint64_t off) { return reinterpret_cast<int32_t*>(ws + off); };
  PageParams k;
  k.table = p->block_table; k.lens = p->seq_lens; k.refs = p->ref_counts; k.parents = p->parents;
  k.new_table = p->new_table; k.new_lens = p->new_lens; k.new_refs = p->new_refs; k.page_map = p->page_map;
  k.count = p->count;
  k.table_stride = p->table_row_stride;
  k.batch = p->batch; k.width = p->width; k.pages = p->num_pages; k.page_size = p->page_size;
  k.header = at(s.header); k.job_src = at(s.src); k.job_dst = at(s.dst); k.job_rows = at(s.rows);
  k.row_job = at(s.row_job); k.first = at(s.first); k.rank = at(s.rank); k.chunk_live = at(s.chunks);

  cudaError_t e;
  const long long cells = (long long)p->batch * p->width;
  const bool one = reassign ? p->num_pages <= kForkPages && p->batch <= kOneRows && cells <= kForkCells
                            : p->num_pages <= kOnePages && cells <= 0x3fffffffll;
  if (one && p->num_caches <= kSomeCaches) {
    e = p->num_caches <= kFewCaches ? launch_one<kFewCaches>(k, p, sms, reassign, stream)
                                    : launch_one<kSomeCaches>(k, p, sms, reassign, stream);
    return e == cudaSuccess ? ATREX_FA_OK : report_failure(ATREX_FA_CUDA_ERROR, "launch of the page kernel", e);
  }
  if (reassign) {
    const long long copy = std::min<long long>(((long long)p->num_pages + kPlanThreads - 1) / kPlanThreads, 2 * sms);
    e = launch_kernel(atrex_sm100_kvpages_plan_kernel, dim3((unsigned)(1 + copy)), dim3(kPlanThreads), 0, stream, k);
  } else {
    const unsigned chunks = (unsigned)(p->num_pages / kChunk + 1);
    e = launch_kernel(atrex_sm100_kvpages_count_kernel, dim3(chunks), dim3(kThreads), 0, stream, k);
    if (e == cudaSuccess)
      e = launch_kernel(atrex_sm100_kvpages_list_kernel, dim3(chunks), dim3(kThreads), 0, stream, k);
  }
  if (e != cudaSuccess) return report_failure(ATREX_FA_CUDA_ERROR, "launch of the page plan", e);

  // the first launch writes tables and counts too; caches beyond kMaxCaches take further launches
  const long long meta_work = reassign ? ((long long)p->batch + 7) / 8
                                       : (std::max<long long>(p->num_pages, (long long)p->batch * p->width) + kThreads - 1) / kThreads;
  for (int done = 0; done == 0 || done < p->num_caches; done += kMaxCaches) {
    const int n = std::min(kMaxCaches, p->num_caches - done);
    e = n <= kFewCaches    ? launch_copies<kFewCaches>(k, p, done, n, sms, meta_work, reassign, stream)
        : n <= kSomeCaches ? launch_copies<kSomeCaches>(k, p, done, n, sms, meta_work, reassign, stream)
                           : launch_copies<kMaxCaches>(k, p, done, n, sms, meta_work, reassign, stream);
    if (e != cudaSuccess) return report_failure(ATREX_FA_CUDA_ERROR, "launch of the page copies", e);
  }
  return ATREX_FA_OK;
}

}  // namespace
}  // namespace atrex_sm100

extern "C" {

int atrex_kvpages_sm100_abi_version(void) { return ATREX_KVPAGES_SM100_ABI_VERSION; }
size_t atrex_kvpages_sm100_params_bytes(void) { return sizeof(atrex_kvpages_sm100_params); }
size_t atrex_kvpages_sm100_cache_bytes(void) { return sizeof(atrex_kvpages_sm100_cache); }
uint64_t atrex_kvpages_sm100_workspace_bytes(int32_t batch, int32_t num_pages) {
  return atrex_sm100::scratch_of(batch < 0 ? 0 : batch, num_pages < 0 ? 0 : num_pages).bytes;
}
int atrex_kvpages_sm100_reassign(const atrex_kvpages_sm100_params* p, void* workspace, uint64_t workspace_bytes,
                                 void* stream) {
  return atrex_sm100::run(p, workspace, workspace_bytes, stream, true);
}
int atrex_kvpages_sm100_compact(const atrex_kvpages_sm100_params* p, void* workspace, uint64_t workspace_bytes,
                                void* stream) {
  return atrex_sm100::run(p, workspace, workspace_bytes, stream, false);
}

}  // extern "C"
