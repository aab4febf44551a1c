// page_ops.cu -- pages that follow their hypotheses (linmt_fork_pages), pools made dense (linmt_compact_pages), copies of pages (linmt_copy_pages).
//
// Both plans are a chain of small steps, each of which needs all of the one before: what rows name, which pages are left over, where those go.  One
// cluster of CTAs does the chain in one launch, its steps parted by the cluster's barrier; launches or a barrier over the whole grid in its place
// would cost 2 to 4 us a step, and what there is to read (a table, a list) is a few hundred kilobytes.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "device_ops.h"

namespace linmt {
namespace ops {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRows = 16384;
constexpr int kMaxPlaces = INT32_MAX - (1 << 17);    // columns of a table, pages: what is counted in 32 bits may run ahead of them by all threads' next four places
constexpr int kRowBytes = 3 * (int)sizeof(int) + (int)sizeof(short);
constexpr int kPortableCluster = 8, kMaxCluster = 16;

struct ForkParams {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* len;
  const int32_t* parents;
  const uint8_t* done;
  const int32_t* shares;
  const int32_t* free_pages;
  const int32_t* used;
  int32_t* out_table;
  int64_t out_table_stride;
  int32_t* out_len;
  int32_t* out_shares;
  int32_t* out_free;
  int32_t* out_used;
  int32_t* out_src;
  int32_t* out_dst;
  int32_t rows, k, width, page, n_pages, n_free;
};

// A row's length, held to what its columns have room for.
__device__ __forceinline__ int length_of(const int32_t* len, int row, int width, int page) {
  return (int)min((int64_t)max(__ldg(len + row), 0), (int64_t)width * page);
}
__device__ __forceinline__ int pages_of(int len, int page) { return (int)(((uint32_t)len + (uint32_t)page - 1) / (uint32_t)page); }

// Sum over the CTA's warps of one number each before warp `warp`, and of all; `sums` has a place for each warp.
__device__ __forceinline__ int before_warp(int mine, int* sums, int& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) sums[warp] = mine;
  __syncthreads();
  const int x = sums[lane];
  static_assert(kWarps == 32, "a lane for each warp");
  all = __reduce_add_sync(~0u, x);
  return __reduce_add_sync(~0u, lane < warp ? x : 0);
}

// The CTA's and the warp's stretch of n things, in whole 32s.
struct Stretch { int begin, end; };
__device__ __forceinline__ Stretch stretch_of(int n, int at, int of) {
  const int64_t groups = ((int64_t)n + 31) / 32;
  return {(int)min((int64_t)n, groups * at / of * 32), (int)min((int64_t)n, groups * (at + 1) / of * 32)};
}

// Every `all`-th place of a table from `at` on, kAtOnce at a time, so that as many loads are on their way: f(row, column, inside) for each.
constexpr int kAtOnce = 4;
template <class F>
__device__ __forceinline__ void for_places(int rows, int width, int at, int all, const F& f) {
  if (width == 0) return;
  const int down = all / width, right = all - down * width;
  int r = at / width, c = at - r * width;
  while (r < rows) {
    int rs[kAtOnce], cs[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      rs[i] = r;
      cs[i] = c;
      r += down;
      c += right;
      if (c >= width) { c -= width; ++r; }
    }
    f(rs, cs);
  }
}

__global__ void __launch_bounds__(kThreads) fork_kernel(const ForkParams a) {
  const cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ int fork_smem[];
  int* const children = fork_smem;              // [rows]
  int* const first = fork_smem + a.rows;        // [rows] a row's first child
  int* const lens = fork_smem + 2 * a.rows;     // [rows]
  short* const parents = reinterpret_cast<short*>(fork_smem + 3 * a.rows);      // [rows], -1: none
  __shared__ int sums[kWarps], total;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), all = ctas * kThreads, at = rank * kThreads + tid;
  auto sync = [&] {
    if (ctas > 1) cluster.sync();
    else __syncthreads();
  };

  // Who has which children: every CTA for all rows.
  for (int r = tid; r < a.rows; r += kThreads) {
    children[r] = 0;
    first[r] = 0x7fffffff;
    lens[r] = length_of(a.len, r, a.width, a.page);
    const int p = a.parents ? __ldg(a.parents + r) : r % a.k;
    parents[r] = (short)(p < 0 || p >= a.k || (a.done && __ldg(a.done + r)) ? -1 : r - r % a.k + p);
  }
  if (a.out_shares != a.shares)
#pragma unroll 4
    for (int64_t i = at; i < a.n_pages; i += all) a.out_shares[i] = __ldg(a.shares + i);
  if (a.out_free != a.free_pages)
#pragma unroll 4
    for (int64_t i = at; i < a.n_free; i += all) a.out_free[i] = __ldg(a.free_pages + i);
  __syncthreads();
  for (int r = tid; r < a.rows; r += kThreads) {
    const int p = parents[r];
    if (p < 0) continue;
    atomicAdd(children + p, 1);
    atomicMin(first + p, r);
  }
  sync();

  // What that does to the pages' shares, and the new rows but for pages that are copied.
  for_places(a.rows, a.width, at, all, [&](const int (&r)[kAtOnce], const int (&c)[kAtOnce]) {
    int by[kAtOnce], page[kAtOnce], take[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      by[i] = 0;
      take[i] = -1;
      if (r[i] >= a.rows) continue;
      const int len = lens[r[i]], have = pages_of(len, a.page), more = children[r[i]] - 1, p = parents[r[i]];
      if (c[i] < have) by[i] = len % a.page && c[i] == have - 1 ? min(more, 0) : more;
      if (by[i]) page[i] = __ldg(a.table + r[i] * a.table_stride + c[i]);
      if (p >= 0 && c[i] < pages_of(lens[p], a.page)) take[i] = __ldg(a.table + p * a.table_stride + c[i]);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (by[i] && page[i] >= 0 && page[i] < a.n_pages) atomicAdd(a.out_shares + page[i], by[i]);
      if (r[i] < a.rows) a.out_table[r[i] * a.out_table_stride + c[i]] = take[i] < a.n_pages ? max(take[i], -1) : -1;
    }
  });
  for (int r = at; r < a.rows; r += all) a.out_len[r] = parents[r] >= 0 ? lens[parents[r]] : 0;
  sync();

  // Pages that no row names any more, ascending: those before the warp's stretch of them, and of all.
  const Stretch mine = stretch_of(a.n_pages, rank * kWarps + warp, ctas * kWarps);
  uint32_t seen = 0;                            // the lane's of the warp's first 32 times 32 pages
  int gone = 0;
#pragma unroll 4
  for (int i = mine.begin + lane, j = 0; i < mine.end; i += 32, ++j) {
    const bool is = __ldcg(a.out_shares + i) < 0;
    gone += is;
    if (is && j < 32) seen |= 1u << j;
  }
  int cta;
  int before = before_warp(__reduce_add_sync(~0u, gone), sums, cta);
  if (tid == 0) total = cta;
  const int used = min(max(__ldg(a.used), 0), a.n_free);
  sync();
  int freed = 0;
  for (int i = 0; i < ctas; ++i) {
    const int x = *cluster.map_shared_rank(&total, i);
    if (i < rank) before += x;
    freed += x;
  }
  for (int i0 = mine.begin, j = 0; i0 < mine.end; i0 += 32, ++j) {
    const bool is = j < 32 ? seen >> j & 1 : i0 + lane < mine.end && __ldcg(a.out_shares + i0 + lane) < 0;
    const uint32_t which = __ballot_sync(~0u, is);
    if (is) {
      a.out_shares[i0 + lane] = 0;
      const int to = used - freed + before + __popc(which & ((1u << lane) - 1));
      if (to >= 0) a.out_free[to] = i0 + lane;           // (more given back than was taken: a fault of the caller's, and the rest is lost)
    }
    before += __popc(which);
  }
  sync();
  if (rank) return;

  // Children that need a page of their own for what their parent's last one holds, in order.
  const int begin = max(used - freed, 0);
  int copies = 0;
  for (int r0 = 0; r0 < a.rows; r0 += kThreads) {
    const int r = r0 + tid;
    int page = -1, column = 0;
    if (r < a.rows) {
      const int p = parents[r];
      if (p >= 0 && first[p] != r) {
        const int len = lens[p];
        if (len % a.page) {
          column = len / a.page;
          page = __ldg(a.table + p * a.table_stride + column);
          if (page >= a.n_pages) page = -1;
        }
      }
    }
    const uint32_t which = __ballot_sync(~0u, page >= 0);
    int some;
    const int place = copies + before_warp(__popc(which), sums, some) + __popc(which & ((1u << lane) - 1));
    if (page >= 0) {
      const int fresh = begin + place < a.n_free ? __ldcg(a.out_free + begin + place) : -1;
      a.out_table[r * a.out_table_stride + column] = fresh;
      a.out_src[place] = page;
      a.out_dst[place] = fresh;
    }
    copies += some;
  }
  for (int i = copies + tid; i < a.rows; i += kThreads) a.out_src[i] = a.out_dst[i] = -1;
  if (tid == 0) *a.out_used = (int)min((int64_t)begin + copies, (int64_t)0x7fffffff);
}

struct CompactParams {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* len;
  const int32_t* shares;
  int32_t* out_table;
  int64_t out_table_stride;
  int32_t* out_shares;
  int32_t* out_free;
  int32_t* out_used;
  int32_t* out_src;
  int32_t* out_dst;
  int32_t* to;               // [n_pages]: 1 for pages that rows name; then a page's new number, -2 - i for the i-th that moves
  int32_t rows, width, page, n_pages;
};

__global__ void __launch_bounds__(kThreads) compact_kernel(const CompactParams a) {
  const cg::cluster_group cluster = cg::this_cluster();
  __shared__ int sums[kWarps], total;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), all = ctas * kThreads, at = rank * kThreads + tid;
  auto sync = [&] {
    if (ctas > 1) cluster.sync();
    else __syncthreads();
  };
  // A row's pages, -1 where there is none: loaded side by side.
  auto named_at = [&](const int (&r)[kAtOnce], const int (&c)[kAtOnce], int (&page)[kAtOnce]) {
    int len[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      page[i] = -1;
      len[i] = 0;
      if (r[i] >= a.rows) continue;
      page[i] = a.table[r[i] * a.table_stride + c[i]];
      len[i] = length_of(a.len, r[i], a.width, a.page);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (c[i] >= pages_of(len[i], a.page) || page[i] >= a.n_pages) page[i] = -1;
  };
  for (int64_t i = at; i < a.n_pages; i += all) a.to[i] = 0;
  sync();
  for_places(a.rows, a.width, at, all, [&](const int (&r)[kAtOnce], const int (&c)[kAtOnce]) {
    int page[kAtOnce];
    named_at(r, c, page);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (page[i] >= 0) a.to[page[i]] = 1;
  });
  sync();
  // How many are named: of the CTA's stretch, before the warp's, in all, and below their number.
  const Stretch mine = stretch_of(a.n_pages, rank * kWarps + warp, ctas * kWarps);
  uint32_t seen = 0;                            // the lane's of the warp's first 32 times 32 pages
  int named = 0;
#pragma unroll 4
  for (int i = mine.begin + lane, j = 0; i < mine.end; i += 32, ++j) {
    const int is = __ldcg(a.to + i);
    named += is;
    if (is && j < 32) seen |= 1u << j;
  }
  int cta;
  int before = before_warp(__reduce_add_sync(~0u, named), sums, cta);
  if (tid == 0) total = cta;
  sync();
  int count = 0, here = 0;
  for (int i = 0; i < ctas; ++i) {
    const int x = *cluster.map_shared_rank(&total, i);
    if (i < rank) here += x;
    count += x;
  }
  before += here;
  int below = 0, first = 0, owner = 0;          // CTA `owner` has page number `count` in its stretch, or ends with the page before
  for (; owner < ctas; ++owner) {
    first = stretch_of(a.n_pages, owner * kWarps, ctas * kWarps).begin;
    const int end = stretch_of(a.n_pages, owner * kWarps + kWarps - 1, ctas * kWarps).end;
    if (count <= end) break;
    below += *cluster.map_shared_rank(&total, owner);
  }
  int more = 0;
#pragma unroll 4
  for (int i = first + tid; i < count; i += kThreads) more += __ldcg(a.to + i);
  int part;
  before_warp(__reduce_add_sync(~0u, more), sums, part);
  below += part;
  sync();                               // (all have counted before numbers take the marks' place)
  for (int i0 = mine.begin, j = 0; i0 < mine.end; i0 += 32, ++j) {
    const int i = i0 + lane;
    const bool in = i < mine.end, is = j < 32 ? seen >> j & 1 : in && __ldcg(a.to + i);
    const uint32_t which = __ballot_sync(~0u, is);
    const int n = before + __popc(which & ((1u << lane) - 1));      // named pages before this one
    if (in) {
      if (is && i >= count) {
        a.out_src[n - below] = i;
        a.to[i] = -2 - (n - below);
      } else {
        if (!is && i < count) a.out_dst[i - n] = i;
        a.to[i] = is ? i : -1;
      }
      a.out_free[i] = i;
    }
    before += __popc(which);
  }
  const int moves = count - below;
  for (int i = moves + at; i < a.n_pages / 2; i += all) a.out_src[i] = a.out_dst[i] = -1;
  if (at == 0) *a.out_used = count;
  sync();
  // The shares go along; a place that is taken is one that nothing named.
  for (int64_t i = at; i < a.n_pages; i += all) {
    const int to = __ldcg(a.to + i);
    if (to >= 0) {
      if (a.out_shares != a.shares) a.out_shares[i] = __ldg(a.shares + i);
    } else {
      if (to <= -2) a.out_shares[__ldcg(a.out_dst - 2 - to)] = a.shares[i];
      if (i >= count) a.out_shares[i] = 0;
    }
  }
  for_places(a.rows, a.width, at, all, [&](const int (&r)[kAtOnce], const int (&c)[kAtOnce]) {
    int page[kAtOnce];
    named_at(r, c, page);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (page[i] >= 0) page[i] = __ldcg(a.to + page[i]);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (page[i] <= -2) page[i] = __ldcg(a.out_dst - 2 - page[i]);
      if (r[i] < a.rows) a.out_table[r[i] * a.out_table_stride + c[i]] = page[i];
    }
  });
}

// ---- copies

constexpr int kCopyThreads = 256;
constexpr int kCopyEach = 8;           // loads of a thread on their way (with four: half of a pool of 0.8 GB made dense in 95 us, not 91)

struct CopyParams {
  const int32_t* src;
  const int32_t* dst;
  int32_t n, n_pages, n_pools, slices;
  linmt_page_pool pool[16];
  int32_t begins[17];                  // first slice of a pool's pages
};

// A CTA has every gridDim.x-th entry and every gridDim.y-th slice of its pages; 32 entries are looked at together, as most of them may copy nothing.
template <class Unit>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyParams a) {
  constexpr int kSlice = kCopyThreads * kCopyEach;
  const int tid = threadIdx.x, lane = tid & 31;
  for (int64_t e0 = blockIdx.x; e0 < a.n; e0 += 32ll * gridDim.x) {
    const int64_t e = e0 + (int64_t)lane * gridDim.x;
    const int from = e < a.n ? __ldg(a.src + e) : -1, to = e < a.n ? __ldg(a.dst + e) : -1;
    uint32_t which = __ballot_sync(~0u, from >= 0 && from < a.n_pages && to >= 0 && to < a.n_pages && from != to);
    for (; which; which &= which - 1) {
      const int64_t s = __shfl_sync(~0u, from, __ffs(which) - 1), d = __shfl_sync(~0u, to, __ffs(which) - 1);
      int p = 0;
      for (int slice = blockIdx.y; slice < a.slices; slice += gridDim.y) {
        while (slice >= a.begins[p + 1]) ++p;
        const linmt_page_pool& pool = a.pool[p];
        const int64_t units = pool.page_bytes / (int64_t)sizeof(Unit), at = (int64_t)(slice - a.begins[p]) * kSlice + tid;
        const Unit* const x = reinterpret_cast<const Unit*>(static_cast<const char*>(pool.data) + s * pool.stride_page);
        Unit* const y = reinterpret_cast<Unit*>(static_cast<char*>(pool.data) + d * pool.stride_page);
        Unit v[kCopyEach];
#pragma unroll
        for (int i = 0; i < kCopyEach; ++i)
          if (at + i * kCopyThreads < units) v[i] = x[at + i * kCopyThreads];
#pragma unroll
        for (int i = 0; i < kCopyEach; ++i)
          if (at + i * kCopyThreads < units) y[at + i * kCopyThreads] = v[i];
      }
    }
  }
}

// CTAs of a cluster for so many things to look at: up to two a thread by one, which needs no barrier of a cluster; beyond that as many as there are to have.  (Eight a thread: 768 hypotheses
// of 20 to 90 positions take 17.5 us with their copies, not 14.8; eight CTAs at most: 2048 of 100 to 1500 positions 30 us, not 25.)
int cluster_for(int64_t things) {
  int c = 1;
  while (c < kMaxCluster && (int64_t)c * kThreads * 2 < things) c *= 2;
  return c;
}
// Whether the device has room for a cluster of 16 with as much shared memory as the kernel may ask for (a part of a GPU may not): asked once for each of the first 64 devices.
template <class P>
bool has_room(void (*kernel)(P), int device, cudaLaunchConfig_t cfg, size_t most_smem) {
  static std::atomic<signed char> known[64];           // 1: yes, -1: no
  const bool keep = device >= 0 && device < 64;
  if (const int was = keep ? known[device].load(std::memory_order_relaxed) : 0) return was > 0;
  cfg.dynamicSmemBytes = most_smem;
  int clusters = 0;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most_smem);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
  if (e != cudaSuccess) cudaGetLastError();
  const bool room = e == cudaSuccess && clusters > 0;
  if (keep) known[device].store(room ? 1 : -1, std::memory_order_relaxed);
  return room;
}
template <class P>
cudaError_t launch_cluster(void (*kernel)(P), const P& p, int device, int ctas, size_t smem, size_t most_smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = ctas > kPortableCluster ? cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) : cudaSuccess;
  if (e == cudaSuccess && ctas > kPortableCluster && !has_room(kernel, device, cfg, most_smem)) {
    attr.val.clusterDim.x = kPortableCluster;
    cfg.gridDim = dim3(kPortableCluster);
  }
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

template <class... P> bool all_aligned4(P... p) { return (aligned(p, 4) && ...); }

}  // namespace
}  // namespace ops
}  // namespace linmt

extern "C" {

int linmt_fork_pages(const linmt_fork_pages_args* g) {
  using namespace linmt::ops;
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "fork_pages: not this library's argument struct");
  if (g->n < 0 || g->k < 0 || g->width < 0 || g->page < 1 || g->n_pages < 0 || g->n_free < 0)
    return op_fail(LINMT_EINVAL, "fork_pages: n = %d, k = %d, width = %d, page = %d, n_pages = %d, n_free = %d", g->n, g->k, g->width, g->page, g->n_pages, g->n_free);
  const int64_t rows = (int64_t)g->n * g->k;
  if (!g->used || !g->out_used || (rows && (!g->len || !g->out_len || !g->out_src || !g->out_dst)) || (rows && g->width && (!g->table || !g->out_table)) ||
      (g->n_pages && (!g->shares || !g->out_shares)) || (g->n_free && (!g->free_pages || !g->out_free)))
    return op_fail(LINMT_EINVAL, "fork_pages: an array is missing");
  if (!all_aligned4(g->table, g->len, g->parents, g->shares, g->free_pages, g->used, g->out_table, g->out_len, g->out_shares, g->out_free, g->out_used, g->out_src, g->out_dst))
    return op_fail(LINMT_EINVAL, "fork_pages: an array is not aligned to its type");
  if (rows > kMaxRows || rows * g->width > kMaxPlaces || g->n_pages > kMaxPlaces || g->n_free > kMaxPlaces)
    return op_fail(LINMT_ELIMIT, "fork_pages: n * k = %lld (at most %d), rows * width = %lld, n_pages = %d, n_free = %d (at most 2^31 - 2^17 - 1)", (long long)rows, kMaxRows, (long long)rows * g->width, g->n_pages, g->n_free);
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "fork_pages");
  const ForkParams p{g->table, g->table_stride, g->len, g->parents, g->done, g->shares, g->free_pages, g->used, g->out_table, g->out_table_stride, g->out_len, g->out_shares, g->out_free,
                     g->out_used, g->out_src, g->out_dst, (int)rows, g->k, g->width, g->page, g->n_pages, g->n_free};
  const size_t smem = (size_t)rows * kRowBytes;
  if (smem > 40 << 10) {
    const cudaError_t e = cudaFuncSetAttribute(fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRows * kRowBytes);
    if (e != cudaSuccess) return op_cuda(e, "fork_pages");
  }
  const cudaError_t e = launch_cluster(fork_kernel, p, g->device, cluster_for(std::max(rows * g->width, (int64_t)g->n_pages + g->n_free)), smem, (size_t)kMaxRows * kRowBytes, static_cast<cudaStream_t>(g->stream));
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "fork_pages");
}

int linmt_compact_pages(const linmt_compact_pages_args* g) {
  using namespace linmt::ops;
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "compact_pages: not this library's argument struct");
  if (g->rows < 0 || g->width < 0 || g->page < 1 || g->n_pages < 0) return op_fail(LINMT_EINVAL, "compact_pages: rows = %d, width = %d, page = %d, n_pages = %d", g->rows, g->width, g->page, g->n_pages);
  if (!g->out_used || (g->rows && (!g->len || (g->width && (!g->table || !g->out_table)))) || (g->n_pages && (!g->shares || !g->out_shares || !g->out_free || !g->workspace)) ||
      (g->n_pages > 1 && (!g->out_src || !g->out_dst)))
    return op_fail(LINMT_EINVAL, "compact_pages: an array is missing");
  if (!all_aligned4(g->table, g->len, g->shares, g->out_table, g->out_shares, g->out_free, g->out_used, g->out_src, g->out_dst, g->workspace))
    return op_fail(LINMT_EINVAL, "compact_pages: an array is not aligned to its type");
  if ((int64_t)g->rows * g->width > kMaxPlaces || g->n_pages > kMaxPlaces)
    return op_fail(LINMT_ELIMIT, "compact_pages: rows * width = %lld, n_pages = %d (at most 2^31 - 2^17 - 1)", (long long)g->rows * g->width, g->n_pages);
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "compact_pages");
  const CompactParams p{g->table, g->table_stride, g->len, g->shares, g->out_table, g->out_table_stride, g->out_shares, g->out_free, g->out_used, g->out_src, g->out_dst, g->workspace,
                        g->rows, g->width, g->page, g->n_pages};
  const cudaError_t e = launch_cluster(compact_kernel, p, g->device, cluster_for(std::max((int64_t)g->rows * g->width, (int64_t)g->n_pages)), 0, 0, static_cast<cudaStream_t>(g->stream));
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "compact_pages");
}

int linmt_copy_pages(const linmt_copy_pages_args* g) {
  using namespace linmt::ops;
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "copy_pages: not this library's argument struct");
  if (g->n < 0 || g->n_pages < 0 || g->n_pools < 0 || g->n_pools > 16) return op_fail(LINMT_EINVAL, "copy_pages: n = %d, n_pages = %d, %d pools (at most 16)", g->n, g->n_pages, g->n_pools);
  if (g->n && (!g->src || !g->dst)) return op_fail(LINMT_EINVAL, "copy_pages: an array is missing");
  if (!aligned(g->src, 4) || !aligned(g->dst, 4)) return op_fail(LINMT_EINVAL, "copy_pages: an array is not aligned to its type");
  uint64_t bits = 0;
  for (int i = 0; i < g->n_pools; ++i) {
    const linmt_page_pool& pool = g->pool[i];
    if (pool.page_bytes < 0 || (pool.page_bytes && !pool.data)) return op_fail(LINMT_EINVAL, "copy_pages: pool %d of pages of %lld bytes at %p", i, (long long)pool.page_bytes, pool.data);
    if (g->n_pages > 1 && pool.page_bytes && (pool.stride_page < 0 ? -pool.stride_page : pool.stride_page) < pool.page_bytes) return op_fail(LINMT_EINVAL, "copy_pages: the pages of pool %d overlap", i);
    if (pool.page_bytes) bits |= reinterpret_cast<uintptr_t>(pool.data) | (uint64_t)pool.stride_page | (uint64_t)pool.page_bytes;
  }
  CopyParams p{g->src, g->dst, g->n, g->n_pages, g->n_pools, 0, {}, {}};
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  int64_t slices = 0;
  for (int i = 0; i < g->n_pools; ++i) {
    p.pool[i] = g->pool[i];
    p.begins[i] = (int)slices;
    slices += (g->pool[i].page_bytes / unit + kCopyThreads * kCopyEach - 1) / (kCopyThreads * kCopyEach);
    if (slices > INT32_MAX) return op_fail(LINMT_ELIMIT, "copy_pages: pages of %lld bytes are too large", (long long)g->pool[i].page_bytes);
  }
  for (int i = g->n_pools; i < 17; ++i) p.begins[i] = (int)slices;
  p.slices = (int)slices;
  if (g->n == 0 || slices == 0) return LINMT_OK;
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "copy_pages");
  // Some 16 CTAs for each SM, as many of them side by side in a page as there are slices.
  const int64_t fit = 16 * 148, x = std::min<int64_t>(g->n, fit), y = std::min<int64_t>(std::min<int64_t>(slices, std::max<int64_t>(1, fit / x)), 65535);
  const dim3 grid((unsigned)x, (unsigned)y);
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  if (unit == 16) copy_kernel<uint4><<<grid, kCopyThreads, 0, st>>>(p);
  else if (unit == 4) copy_kernel<uint32_t><<<grid, kCopyThreads, 0, st>>>(p);
  else copy_kernel<uint8_t><<<grid, kCopyThreads, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "copy_pages");
}

}  // extern "C"
