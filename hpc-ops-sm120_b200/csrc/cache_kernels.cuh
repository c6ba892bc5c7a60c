// cache_kernels.cuh -- kernels that keep a paged K/V cache: the write of new
// tokens into their pages, page copies, and the bookkeeping of pages
// (resize, fork, compact).
//
// The bookkeeping state is device memory that a captured graph can change:
//   table  int32 [rows][max_blocks]  page j of a row's tokens, -1 where none is held
//   refs   int32 [num_blocks]        how many rows hold a page (0: free)
// and the lowest free page is always taken first, so the result of a call
// depends on its inputs alone.
//
// A bookkeeping call is a few dependent steps over little data (refs once,
// the table entries that change): it is bound by latency, not by bytes.  Each
// is therefore ONE launch of ONE cluster of 8 CTAs x 1024 threads, whose steps
// are separated by cluster barriers and whose prefix sums cross CTAs through
// distributed shared memory, instead of a chain of kernels.
#pragma once

#include "device_primitives.cuh"

namespace adb {

constexpr int kBookCtas = 8;       // portable cluster size
constexpr int kBookThreads = 1024;
constexpr int kBookWarps = kBookThreads / 32;
constexpr int kBookAllWarps = kBookCtas * kBookWarps;
constexpr int kBookChunk = 512;    // table entries of a row that one warp handles

// ------------------------------------------------------------ cluster
// Release/acquire at cluster scope: orders global and shared accesses of the
// cluster's threads before it against those after it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// The int at this CTA's shared address `p`, read in CTA `rank`.
__device__ __forceinline__ int peer_shared(const int* p, int rank) {
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// ------------------------------------------------------------ block scan
__device__ __forceinline__ int warp_inclusive(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

struct BookShared {
  int warp[kBookWarps];
  int total[2];    // of this CTA, read by its peers (one per counting pass)
  int before;      // sum of the totals of the CTAs before this one
  int all;         // sum of every CTA's total
  int flag;        // read by its peers
};

// Exclusive prefix of v over the block; *sum gets the block's total.
__device__ __forceinline__ int block_exclusive(int v, BookShared& sh, int* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int inc = warp_inclusive(v, lane);
  __syncthreads();
  if (lane == 31) sh.warp[warp] = inc;
  __syncthreads();
  if (warp == 0) sh.warp[lane] = warp_inclusive(sh.warp[lane], lane);
  __syncthreads();
  *sum = sh.warp[kBookWarps - 1];
  return inc - v + (warp > 0 ? sh.warp[warp - 1] : 0);
}

// A warp's contiguous share of the pool's pages, in multiples of 32.
struct Region {
  int lo, hi;
};
__device__ __forceinline__ Region page_region(int num_blocks) {
  const int all_warp = cluster_rank() * kBookWarps + (threadIdx.x >> 5);
  const int64_t per = (((static_cast<int64_t>(num_blocks) + kBookAllWarps - 1) / kBookAllWarps) + 31) & ~int64_t(31);
  const int64_t lo = per * all_warp, hi = lo + per;
  return {static_cast<int>(lo < num_blocks ? lo : num_blocks), static_cast<int>(hi < num_blocks ? hi : num_blocks)};
}

// Counts the pages that `pred` holds for: returns how many are in regions
// before this warp's; sh.all is the count over the pool.  Ends with a cluster
// barrier, so what was written before the call is visible to the cluster.
template <int kPass, typename Pred>
__device__ __forceinline__ int count_pages(const Region& r, BookShared& sh, Pred pred) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int mine = 0;
#pragma unroll 4
  for (int p = r.lo; p < r.hi; p += 32) {
    const bool hit = p + lane < r.hi && pred(p + lane);
    mine += __popc(__ballot_sync(0xffffffffu, hit));
  }
  __syncthreads();
  if (lane == 0) sh.warp[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const int inc = warp_inclusive(sh.warp[lane], lane);
    sh.warp[lane] = inc;
    if (lane == 31) sh.total[kPass] = inc;
  }
  cluster_sync();
  if (warp == 0) {
    const int rank = cluster_rank();
    const int t = lane < kBookCtas ? peer_shared(&sh.total[kPass], lane) : 0;
    const int inc = warp_inclusive(t, lane);
    if (lane == rank) sh.before = inc - t;
    if (lane == 31) sh.all = inc;
  }
  __syncthreads();
  return sh.before + sh.warp[warp] - mine;
}

// Whether any CTA of the cluster raised sh.flag before its last barrier.
__device__ __forceinline__ bool any_flag(BookShared& sh) {
  const int lane = threadIdx.x & 31;
  const int f = lane < kBookCtas ? peer_shared(&sh.flag, lane) : 0;
  return __any_sync(0xffffffffu, f != 0);
}

// Last index i of [0, n) with prefix[i] <= rank (prefix ascending, prefix[0] = 0).
__device__ __forceinline__ int last_at_most(const int* prefix, int n, int rank) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= rank)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int clamp_len(int n, int cap) { return n < 0 ? 0 : (n > cap ? cap : n); }

// ------------------------------------------------------------ resize
struct ResizeParams {
  int32_t* table;
  int64_t stride;
  const int32_t* lens;   // lengths before
  const int32_t* want;   // lengths asked for
  int32_t* refs;
  int32_t* lens_out;     // lengths after
  int batch, max_blocks, num_blocks, page_shift;
};

// Takes entries [from(b), to(b)) of every row out of the table and the counts.
template <typename Range>
__device__ __forceinline__ void let_go(const ResizeParams& p, Range range) {
  const int lane = threadIdx.x & 31;
  const int64_t chunks = (p.max_blocks + kBookChunk - 1) / kBookChunk;
  for (int64_t u = cluster_rank() * kBookWarps + (threadIdx.x >> 5); u < chunks * p.batch; u += kBookAllWarps) {
    const int b = static_cast<int>(u / chunks), c = static_cast<int>(u % chunks) * kBookChunk;
    int from, to;
    range(b, from, to);
    from = max(from, c);
    to = min(to, c + kBookChunk);
    int32_t* row = p.table + b * p.stride;
#pragma unroll 4
    for (int j = from + lane; j < to; j += 32) {
      const int page = row[j];
      row[j] = -1;
      if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks)) {
        if (atomicSub(&p.refs[page], 1) > 0) continue;
        atomicAdd(&p.refs[page], 1);  // nobody held it: the tables disagree
      }
      atomicOr(&g_adb_error_flag, kErrCachePage);
    }
  }
}

// Steps: rows that end let their pages go; cuts are judged (refused where the
// page that stays partly used is held by another row, whose tokens the row's
// next ones would overwrite) and then made; the free pages are counted and
// handed out, lowest first, to the growing rows in row order.
__global__ void __cluster_dims__(kBookCtas, 1, 1) __launch_bounds__(kBookThreads)
    cache_resize_kernel(const ResizeParams p) {
  extern __shared__ int prefix[];  // [batch]: pages needed by the rows before
  __shared__ BookShared sh;
  const int tid = threadIdx.x, lane = tid & 31;
  const int mask = (1 << p.page_shift) - 1;
  const int cap = p.max_blocks << p.page_shift;
  const auto pages = [&](int n) { return static_cast<int>((static_cast<unsigned>(n) + mask) >> p.page_shift); };
  if (tid == 0) sh.flag = 0;
  griddep_wait();

  let_go(p, [&](int b, int& from, int& to) {
    from = 0;
    to = p.want[b] == 0 ? pages(clamp_len(p.lens[b], cap)) : 0;
  });
  cluster_sync();

  for (int b = cluster_rank() * kBookThreads + tid; b < p.batch; b += kBookCtas * kBookThreads) {
    const int old = clamp_len(p.lens[b], cap), w = p.want[b];
    int after = old;
    bool refused = w < 0 || w > cap;
    if (w == 0) {
      after = 0;
    } else if (!refused && w < old) {
      if (w & mask) {
        const int page = p.table[b * p.stride + (w >> p.page_shift)];
        refused = static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks) && p.refs[page] > 1;
      }
      if (!refused) {
        after = w;
        sh.flag = 1;
      }
    }
    p.lens_out[b] = after;
    if (refused) atomicOr(&g_adb_error_flag, kErrCacheRefused);
  }
  // the pages that each growing row needs, and those of the rows before it
  int needed = 0;
  for (int base = 0; base < p.batch; base += kBookThreads) {
    const int b = base + tid;
    int need = 0;
    if (b < p.batch) {
      const int old = clamp_len(p.lens[b], cap), w = p.want[b];
      if (w > old && w <= cap) need = pages(w) - pages(old);
    }
    int sum;
    const int before = block_exclusive(need, sh, &sum);
    if (b < p.batch) prefix[b] = needed + before;
    needed += sum;
  }
  cluster_sync();
  if (any_flag(sh)) {
    let_go(p, [&](int b, int& from, int& to) {
      const int old = clamp_len(p.lens[b], cap), w = p.want[b];
      const bool cut = w > 0 && w < old && p.lens_out[b] == w;
      from = cut ? pages(w) : 0;
      to = cut ? pages(old) : 0;
    });
    cluster_sync();
  }

  const Region r = page_region(p.num_blocks);
  int rank = count_pages<0>(r, sh, [&](int page) { return p.refs[page] == 0; });
  const int free_pages = sh.all;
  for (int at = r.lo; at < r.hi && rank < needed; at += 32) {
    const int page = at + lane;
    const bool hit = page < r.hi && p.refs[page] == 0;
    const unsigned hits = __ballot_sync(0xffffffffu, hit);
    const int mine = rank + __popc(hits & ((1u << lane) - 1));
    if (hit && mine < needed) {
      const int b = last_at_most(prefix, p.batch, mine);
      const int first = pages(clamp_len(p.lens[b], cap)), last = pages(p.want[b]);
      if (prefix[b] + (last - first) <= free_pages) {
        p.table[b * p.stride + first + mine - prefix[b]] = page;
        p.refs[page] = 1;
      }
    }
    rank += __popc(hits);
  }
  for (int b = cluster_rank() * kBookThreads + tid; b < p.batch; b += kBookCtas * kBookThreads) {
    const int old = clamp_len(p.lens[b], cap), w = p.want[b];
    if (w <= old || w > cap) continue;
    const int need = pages(w) - pages(old);
    if (need == 0 || prefix[b] + need <= free_pages)
      p.lens_out[b] = w;
    else
      atomicOr(&g_adb_error_flag, kErrCacheFull);
  }
  griddep_launch_dependents();
  cluster_sync();  // no CTA leaves while a peer may read its shared memory
}

// ------------------------------------------------------------ fork
struct ForkParams {
  int32_t* table;
  int64_t stride;
  const int32_t* lens;
  int32_t* refs;
  const int32_t* parents;
  const int32_t* children;
  int32_t* lens_out;
  int32_t* src;  // [forks] page copies that the caller makes: a parent's partly
  int32_t* dst;  // [forks] filled last page -> the child's own; -1 where none
  int batch, forks, max_blocks, num_blocks, page_shift;
};

// A child shares its parent's full pages (they no longer change) and gets a
// page of its own for the partly filled last one.  Each CTA keeps, redundantly,
// which fork a row is the child of (the first that names it) and the prefix
// sum of the pages needed.
__global__ void __cluster_dims__(kBookCtas, 1, 1) __launch_bounds__(kBookThreads)
    cache_fork_kernel(const ForkParams p) {
  extern __shared__ int fork_smem[];
  int* prefix = fork_smem;            // [forks]
  int* claim = fork_smem + p.forks;   // [batch]: first fork that names the row as its child
  __shared__ BookShared sh;
  const int tid = threadIdx.x, lane = tid & 31;
  const int mask = (1 << p.page_shift) - 1;
  const int cap = p.max_blocks << p.page_shift;
  for (int b = tid; b < p.batch; b += kBookThreads) claim[b] = INT32_MAX;
  __syncthreads();
  griddep_wait();
  for (int i = tid; i < p.forks; i += kBookThreads) {
    const int c = p.children[i];
    if (static_cast<unsigned>(c) < static_cast<unsigned>(p.batch)) atomicMin(&claim[c], i);
  }
  __syncthreads();
  // -1: refused; otherwise the tokens that the child takes over
  const auto tokens = [&](int i) {
    const int a = p.parents[i], c = p.children[i];
    const unsigned rows = static_cast<unsigned>(p.batch);
    if (static_cast<unsigned>(a) >= rows || static_cast<unsigned>(c) >= rows) return -1;
    if (claim[c] != i || p.lens[c] != 0) return -1;
    return clamp_len(p.lens[a], cap);
  };
  int needed = 0;
  for (int base = 0; base < p.forks; base += kBookThreads) {
    const int i = base + tid;
    const int n = i < p.forks ? tokens(i) : 0;
    int sum;
    const int before = block_exclusive(n > 0 && (n & mask) != 0, sh, &sum);
    if (i < p.forks) prefix[i] = needed + before;
    needed += sum;
  }
  const Region r = page_region(p.num_blocks);
  int rank = count_pages<0>(r, sh, [&](int page) { return p.refs[page] == 0; });
  const int free_pages = sh.all;
  // every CTA has counted (the barrier in count_pages): the counts may change now
  const auto granted = [&](int i, int n) { return n >= 0 && ((n & mask) == 0 || prefix[i] < free_pages); };

  for (int at = r.lo; at < r.hi && rank < needed; at += 32) {
    const int page = at + lane;
    const bool hit = page < r.hi && p.refs[page] == 0;
    const unsigned hits = __ballot_sync(0xffffffffu, hit);
    const int mine = rank + __popc(hits & ((1u << lane) - 1));
    if (hit && mine < needed) {
      // forks without a copy repeat the next prefix: the last one at `mine` is the one that needs it
      const int i = last_at_most(prefix, p.forks, mine);
      const int a = p.parents[i], full = clamp_len(p.lens[a], cap) >> p.page_shift;
      p.src[i] = p.table[a * p.stride + full];
      p.dst[i] = page;
      p.table[p.children[i] * p.stride + full] = page;
      p.refs[page] = 1;
    }
    rank += __popc(hits);
  }

  const int all_tid = cluster_rank() * kBookThreads + tid;
  for (int i = all_tid; i < p.forks; i += kBookCtas * kBookThreads) {
    const int n = tokens(i);
    const bool copies = granted(i, n) && (n & mask) != 0;
    if (!copies) p.src[i] = p.dst[i] = -1;
    if (n < 0) atomicOr(&g_adb_error_flag, kErrCacheRefused);
    if (n >= 0 && !granted(i, n)) atomicOr(&g_adb_error_flag, kErrCacheFull);
  }
  for (int b = all_tid; b < p.batch; b += kBookCtas * kBookThreads) {
    const int i = claim[b];
    const int n = i < p.forks ? tokens(i) : -1;
    p.lens_out[b] = n >= 0 && granted(i, n) ? n : p.lens[b];
  }
  const int64_t chunks = (p.max_blocks + kBookChunk - 1) / kBookChunk;
  for (int64_t u = cluster_rank() * kBookWarps + (tid >> 5); u < chunks * p.forks; u += kBookAllWarps) {
    const int i = static_cast<int>(u / chunks), c = static_cast<int>(u % chunks) * kBookChunk;
    const int n = tokens(i);
    if (!granted(i, n)) continue;
    const int to = min(n >> p.page_shift, c + kBookChunk);
    const int32_t* from_row = p.table + p.parents[i] * p.stride;
    int32_t* to_row = p.table + p.children[i] * p.stride;
#pragma unroll 4
    for (int j = c + lane; j < to; j += 32) {
      const int page = from_row[j];
      to_row[j] = page;
      if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks))
        atomicAdd(&p.refs[page], 1);
      else
        atomicOr(&g_adb_error_flag, kErrCachePage);
    }
  }
  griddep_launch_dependents();
  cluster_sync();
}

// ------------------------------------------------------------ compact
struct CompactParams {
  int32_t* table;
  int64_t stride;
  const int32_t* lens;
  int32_t* refs;
  int32_t* src;    // [num_blocks / 2] page copies that the caller makes,
  int32_t* dst;    // then -1
  int32_t* remap;  // [num_blocks] scratch: where a page at or above the live count goes
  int batch, max_blocks, num_blocks, page_shift;
};

// With n live pages, the i-th live page at or above n moves to the i-th free
// page below n: the fewest copies that leave the live pages at the front, and
// no page is both a source and a destination.
__global__ void __cluster_dims__(kBookCtas, 1, 1) __launch_bounds__(kBookThreads)
    cache_compact_kernel(const CompactParams p) {
  __shared__ BookShared sh;
  const int tid = threadIdx.x, lane = tid & 31;
  const int mask = (1 << p.page_shift) - 1;
  const int cap = p.max_blocks << p.page_shift;
  griddep_wait();
  const Region r = page_region(p.num_blocks);
  int before = count_pages<0>(r, sh, [&](int page) { return p.refs[page] > 0; });
  const int live = sh.all;
  // live pages below `live` stay; their count ranks the others
  count_pages<1>(r, sh, [&](int page) { return page < live && p.refs[page] > 0; });
  const int stay = sh.all, moves = live - stay;
  for (int at = r.lo; at < r.hi; at += 32) {
    const int page = at + lane;
    const bool in = page < r.hi, held = in && p.refs[page] > 0;
    const unsigned hits = __ballot_sync(0xffffffffu, held);
    const int mine = before + __popc(hits & ((1u << lane) - 1));  // live pages before this one
    if (in && page < live && !held) p.dst[page - mine] = page;
    if (in && page >= live) {
      p.remap[page] = held ? mine - stay : -1;
      if (held) p.src[mine - stay] = page;
    }
    before += __popc(hits);
  }
  cluster_sync();
  const int all_tid = cluster_rank() * kBookThreads + tid;
  for (int i = all_tid; i < p.num_blocks / 2; i += kBookCtas * kBookThreads) {
    if (i < moves) {
      const int from = p.src[i], to = p.dst[i];
      p.refs[to] = p.refs[from];
      p.refs[from] = 0;
    } else {
      p.src[i] = p.dst[i] = -1;
    }
  }
  const int64_t chunks = (p.max_blocks + kBookChunk - 1) / kBookChunk;
  for (int64_t u = cluster_rank() * kBookWarps + (tid >> 5); u < chunks * p.batch; u += kBookAllWarps) {
    const int b = static_cast<int>(u / chunks), c = static_cast<int>(u % chunks) * kBookChunk;
    const int held = static_cast<int>((static_cast<unsigned>(clamp_len(p.lens[b], cap)) + mask) >> p.page_shift);
    const int to = min(held, c + kBookChunk);
    int32_t* row = p.table + b * p.stride;
#pragma unroll 4
    for (int j = c + lane; j < to; j += 32) {
      const int page = row[j];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) {
        atomicOr(&g_adb_error_flag, kErrCachePage);
      } else if (page >= live) {
        const int i = p.remap[page];
        if (i >= 0)
          row[j] = p.dst[i];
        else
          atomicOr(&g_adb_error_flag, kErrCachePage);  // a page that refs calls free
      }
    }
  }
  griddep_launch_dependents();
  cluster_sync();
}

// ------------------------------------------------------------ page copies
struct CopyParams {
  uint4* k;
  uint4* v;
  const int32_t* src;
  const int32_t* dst;
  int64_t count;       // entries of src / dst
  int64_t page_vecs;   // 16-byte vectors of a page
  int chunks;          // parts of a page, kCopyVecs each but the last
  int num_blocks;
};
constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 1024;  // of K and of V: 16 KB each per unit of work

// One unit is a part of one entry's page, of K and of V.  The lists that
// cache_compact returns are mostly -1 behind the moves, so each warp looks at
// 32 of its CTA's units at a time and the CTA copies the valid ones.
__global__ void __launch_bounds__(kCopyThreads) cache_copy_pages_kernel(const CopyParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t units = p.count * p.chunks;
  griddep_wait();
  for (int64_t base = blockIdx.x; base < units; base += 32 * static_cast<int64_t>(gridDim.x)) {
    const int64_t u = base + lane * static_cast<int64_t>(gridDim.x);
    int from = -1, to = -1;
    if (u < units) {
      from = p.src[u / p.chunks];
      to = p.dst[u / p.chunks];
    }
    const bool in = static_cast<unsigned>(from) < static_cast<unsigned>(p.num_blocks) &&
                    static_cast<unsigned>(to) < static_cast<unsigned>(p.num_blocks);
    if (!in && (from >= p.num_blocks || to >= p.num_blocks || from < -1 || to < -1))
      atomicOr(&g_adb_error_flag, kErrCachePage);
    unsigned todo = __ballot_sync(0xffffffffu, in && from != to);
    while (todo) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1;
      const int64_t a = __shfl_sync(0xffffffffu, from, l), b = __shfl_sync(0xffffffffu, to, l);
      const int64_t first = ((base + l * static_cast<int64_t>(gridDim.x)) % p.chunks) * kCopyVecs;
      const int n = static_cast<int>(min(static_cast<int64_t>(kCopyVecs), p.page_vecs - first));
      const int64_t from_at = a * p.page_vecs + first, to_at = b * p.page_vecs + first;
      uint4 x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = threadIdx.x + i * kCopyThreads;
        if (at < n) {
          x[i] = __ldcs(&p.k[from_at + at]);
          x[4 + i] = __ldcs(&p.v[from_at + at]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = threadIdx.x + i * kCopyThreads;
        if (at < n) {
          p.k[to_at + at] = x[i];
          p.v[to_at + at] = x[4 + i];
        }
      }
    }
  }
}

// ------------------------------------------------------------ write
struct WriteParams {
  const __nv_bfloat16* k;  // [total][heads][D], strides in elements
  const __nv_bfloat16* v;
  int64_t k_token, k_head, v_token, v_head;
  __nv_bfloat16* k_cache;
  __nv_bfloat16* v_cache;
  const int32_t* table;
  int64_t stride;
  const int32_t* cu;      // [batch + 1]
  const int32_t* starts;  // [batch]: tokens that a row held before
  int64_t total;
  int batch, heads, dim, max_blocks, num_blocks, page_shift, nhd;
};
constexpr int kWriteThreads = 256;

// One thread moves one 16-byte vector of K and the same one of V.  The source
// loads do not depend on the place, so they are issued first and the search
// for the token's row runs in their shadow.
__global__ void __launch_bounds__(kWriteThreads) cache_write_kernel(const WriteParams p) {
  const int head_vecs = p.dim >> 3;
  const int vecs = p.heads * head_vecs;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kWriteThreads + threadIdx.x;
  griddep_wait();
  if (i >= p.total * vecs) return;
  const int64_t t = i / vecs;
  const int x = static_cast<int>(i - t * vecs);
  const int head = x / head_vecs, e = (x - head * head_vecs) * 8;
  const uint4 kv = __ldcs(reinterpret_cast<const uint4*>(p.k + t * p.k_token + head * p.k_head + e));
  const uint4 vv = __ldcs(reinterpret_cast<const uint4*>(p.v + t * p.v_token + head * p.v_head + e));
  // last row whose tokens start at or before t
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int64_t first = p.cu[lo];
  if (t < first || t >= p.cu[lo + 1]) return;  // padding behind the last row
  const int64_t pos = p.starts[lo] + (t - first);
  const int64_t j = pos >> p.page_shift;
  int page = -1;
  if (pos >= 0 && j < p.max_blocks) page = p.table[lo * p.stride + j];
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) {
    if (x == 0) atomicOr(&g_adb_error_flag, kErrCachePage);
    return;
  }
  const int64_t slot = pos & ((int64_t(1) << p.page_shift) - 1);
  const int64_t page_size = int64_t(1) << p.page_shift;
  const int64_t row = p.nhd ? (page * page_size + slot) * p.heads + head
                            : (static_cast<int64_t>(page) * p.heads + head) * page_size + slot;
  const int64_t at = row * p.dim + e;
  *reinterpret_cast<uint4*>(p.k_cache + at) = kv;
  *reinterpret_cast<uint4*>(p.v_cache + at) = vv;
}

}  // namespace adb
