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
// distributed shared memory, instead of a chain of kernels.  What all CTAs need
// of the rows (lengths, prefix sums) each keeps in its own shared memory, read
// from global memory once, and a warp keeps the bits of the pages that it
// counted, so that a step waits for memory as seldom as possible.
//
// Every kernel lets the next one start at once: kernels of this library wait
// (griddepcontrol.wait) before they touch memory, others for the grid's end.
#pragma once

#include "device_primitives.cuh"

namespace adb {

constexpr int kBookCtas = 8;       // portable cluster size
constexpr int kBookThreads = 1024;
constexpr int kBookWarps = kBookThreads / 32;
constexpr int kBookAllWarps = kBookCtas * kBookWarps;
constexpr int kBookChunk = 128;    // table entries of a row that one warp handles

// ------------------------------------------------------------ cluster
// Release/acquire at cluster scope: orders global and shared accesses of the
// cluster's threads before it against those after it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// No CTA of the cluster leaves before all have come here; orders no memory.
__device__ __forceinline__ void cluster_leave() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
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

// The pages of a warp's region for which a predicate holds: the bits of pages
// lo + 32 n .. + 31 are in lane n of `bits`, read again where a region has more
// than 32 x 32 pages.
struct PageBits {
  Region r;
  uint32_t bits;
  int count;
};

template <typename Pred>
__device__ __forceinline__ PageBits find_pages(int num_blocks, Pred pred) {
  const int lane = threadIdx.x & 31;
  PageBits b{page_region(num_blocks), 0u, 0};
  if (b.r.hi - b.r.lo <= 32) {  // (the loop's code alone takes 1000 cycles to arrive)
    b.bits = __ballot_sync(0xffffffffu, b.r.lo + lane < b.r.hi && pred(b.r.lo + lane));
    b.count = __popc(b.bits);
    return b;  // page_bits asks lane 0
  }
  constexpr int kAtOnce = 16;  // loads in flight
  for (int p0 = b.r.lo; p0 < b.r.hi; p0 += 32 * kAtOnce) {
    bool hit[kAtOnce];
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) hit[x] = p0 + 32 * x + lane < b.r.hi && pred(p0 + 32 * x + lane);
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      if (p0 + 32 * x >= b.r.hi) break;
      const unsigned hits = __ballot_sync(0xffffffffu, hit[x]);
      if (lane == ((p0 - b.r.lo) >> 5) + x) b.bits = hits;
      b.count += __popc(hits);
    }
  }
  return b;
}

template <typename Pred>
__device__ __forceinline__ unsigned page_bits(const PageBits& b, int at, Pred pred) {
  const int n = (at - b.r.lo) >> 5, lane = threadIdx.x & 31;
  if (n < 32) return __shfl_sync(0xffffffffu, b.bits, n);
  return __ballot_sync(0xffffffffu, at + lane < b.r.hi && pred(at + lane));
}

// Sums a warp's count over the cluster: returns the sum over the warps before
// this one; sh.all is the total.  Ends with a cluster barrier, so what was
// written before the call is visible to the cluster.
template <int kPass>
__device__ __forceinline__ int cluster_prefix(int mine, BookShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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

// Last index i of [lo, hi] with prefix[i] <= rank (prefix ascending, prefix[lo] <= rank).
__device__ __forceinline__ int last_at_most(const int* prefix, int lo, int hi, int rank) {
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= rank)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Entries [from, to) of the rows in units of kBookChunk, a warp per unit: each
// lane looks whether there is work in one unit, then the warp does those units.
// range(row, from, to); work(row, from, to) with from < to inside one unit.
template <typename Range, typename Work>
__device__ __forceinline__ void each_chunk(int rows, int max_blocks, Range range, Work work) {
  const int lane = threadIdx.x & 31;
  const int chunks = (max_blocks + kBookChunk - 1) / kBookChunk, units = rows * chunks;
  for (int u0 = cluster_rank() * kBookWarps + (threadIdx.x >> 5); u0 < units; u0 += 32 * kBookAllWarps) {
    const int u = u0 + lane * kBookAllWarps;
    int row = 0, from = 0, to = 0;
    if (u < units) {
      row = u / chunks;
      const int c = (u - row * chunks) * kBookChunk;
      range(row, from, to);
      from = max(from, c);
      to = min(to, c + kBookChunk);
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, from < to); todo != 0; todo &= todo - 1) {
      const int l = __ffs(todo) - 1;
      work(__shfl_sync(0xffffffffu, row, l), __shfl_sync(0xffffffffu, from, l), __shfl_sync(0xffffffffu, to, l));
    }
  }
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
  each_chunk(p.batch, p.max_blocks, range, [&](int b, int from, int to) {
    int32_t* row = p.table + b * p.stride;
    int page[kBookChunk / 32], left[kBookChunk / 32];
#pragma unroll
    for (int x = 0; x < kBookChunk / 32; ++x) {
      const int j = from + lane + 32 * x;
      page[x] = j < to ? row[j] : -1;
    }
#pragma unroll
    for (int x = 0; x < kBookChunk / 32; ++x) {
      const int j = from + lane + 32 * x;
      left[x] = 1;
      if (j < to) {
        row[j] = -1;
        left[x] = static_cast<unsigned>(page[x]) < static_cast<unsigned>(p.num_blocks) ? atomicSub(&p.refs[page[x]], 1) : 0;
      }
    }
#pragma unroll
    for (int x = 0; x < kBookChunk / 32; ++x) {
      if (left[x] > 0) continue;  // no page, or nobody held it: the tables disagree
      if (static_cast<unsigned>(page[x]) < static_cast<unsigned>(p.num_blocks)) atomicAdd(&p.refs[page[x]], 1);
      atomicOr(&g_adb_error_flag, kErrCachePage);
    }
  });
}

// 8 us for 32 rows that grow by a token, 15 us for 256 rows of which 30 end and
// 212 grow in a pool of 66548 pages (one CTA-wide chunk per row and warp, without
// the look ahead by lanes: 33 us).  Here and below: in a graph of 20 calls, without
// the copies that bring the state back.
//
// Steps: rows that end let their pages go; cuts are judged (refused where the
// page that stays partly used is held by another row, whose tokens the row's
// next ones would overwrite) and then made; the free pages are counted and
// handed out, lowest first, to the growing rows in row order.  Steps that no
// row asks for are skipped.
__global__ void __cluster_dims__(kBookCtas, 1, 1) __launch_bounds__(kBookThreads, 1)
    cache_resize_kernel(const ResizeParams p) {
  extern __shared__ int resize_smem[];
  int* prefix = resize_smem;             // [batch]: pages needed by the rows before
  int* olds = resize_smem + p.batch;     // [batch]: lengths before
  int* wants = resize_smem + 2 * p.batch;  // [batch]: lengths asked for; refused: as before
  __shared__ BookShared sh;
  const int tid = threadIdx.x, lane = tid & 31;
  const int all_tid = cluster_rank() * kBookThreads + tid;
  const int mask = (1 << p.page_shift) - 1;
  const int cap = p.max_blocks << p.page_shift;
  const auto pages = [&](int n) { return static_cast<int>((static_cast<unsigned>(n) + mask) >> p.page_shift); };
  griddep_launch_dependents();
  griddep_wait();

  int needed = 0, drops = 0, cuts = 0;
  for (int base = 0; base < p.batch; base += kBookThreads) {
    const int b = base + tid;
    int need = 0;
    if (b < p.batch) {
      const int old = clamp_len(p.lens[b], cap);
      int w = p.want[b];
      if (w < 0 || w > cap) {
        w = old;
        if (cluster_rank() == 0) atomicOr(&g_adb_error_flag, kErrCacheRefused);
      }
      olds[b] = old;
      wants[b] = w;
      if (w > old) need = pages(w) - pages(old);
      drops |= w == 0 && old > 0;
      cuts |= w > 0 && w < old;
    }
    int sum;
    const int before = block_exclusive(need, sh, &sum);
    if (b < p.batch) prefix[b] = needed + before;
    needed += sum;
  }
  drops = __syncthreads_or(drops);
  cuts = __syncthreads_or(cuts);
  if (drops) {
    let_go(p, [&](int b, int& from, int& to) {
      from = 0;
      to = wants[b] == 0 ? pages(olds[b]) : 0;
    });
    cluster_sync();
  }
  if (cuts) {
    // every CTA judges for itself, and none changes a count until all have
    bool refused = false;
    for (int b = tid; b < p.batch; b += kBookThreads) {
      const int old = olds[b], w = wants[b];
      if (w == 0 || w >= old || (w & mask) == 0) continue;
      const int page = p.table[b * p.stride + (w >> p.page_shift)];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks) || __ldcg(&p.refs[page]) <= 1) continue;
      wants[b] = old;
      refused = true;
    }
    if (refused && cluster_rank() == 0) atomicOr(&g_adb_error_flag, kErrCacheRefused);
    cluster_sync();
    let_go(p, [&](int b, int& from, int& to) {
      const bool cut = wants[b] > 0 && wants[b] < olds[b];
      from = cut ? pages(wants[b]) : 0;
      to = cut ? pages(olds[b]) : 0;
    });
    cluster_sync();
  }

  const auto is_free = [&](int page) { return __ldcg(&p.refs[page]) == 0; };
  if (needed > 0) {  // (the same in all CTAs)
    const PageBits free = find_pages(p.num_blocks, is_free);
    int rank = cluster_prefix<0>(free.count, sh);
    // Consecutive ranks are mostly of one row: the warp keeps the row of its last
    // one, where its entries go and its last rank, and lanes search only where a
    // row ends among the 32 pages.  (Eight SMs issue this loop for the whole pool:
    // with the row's values read again for every 32 pages it took 10400 cycles for
    // 256 rows and 66548 pages, so 7300.)
    int row = rank < needed ? last_at_most(prefix, 0, p.batch - 1, rank) : 0;
    int row_end = -1;  // none kept yet
    bool granted = false;
    int32_t* entries = nullptr;  // of rank 0, if the row had it
    for (int at = free.r.lo; at < free.r.hi && rank < needed; at += 32) {
      const unsigned hits = page_bits(free, at, is_free);
      const int mine = rank + __popc(hits & ((1u << lane) - 1));
      rank += __popc(hits);
      if (rank <= row_end) {
        if ((hits >> lane & 1) && granted) {
          entries[mine] = at + lane;
          p.refs[at + lane] = 1;
        }
        continue;
      }
      if (hits == 0) continue;
      const int row0 = row;
      row = last_at_most(prefix, row0, p.batch - 1, rank - 1);
      if ((hits >> lane & 1) && mine < needed) {
        const int b = last_at_most(prefix, row0, row, mine);
        const int first = pages(olds[b]), last = pages(wants[b]);
        if (prefix[b] + (last - first) <= sh.all) {
          p.table[b * p.stride + first + mine - prefix[b]] = at + lane;
          p.refs[at + lane] = 1;
        }
      }
      const int first = pages(olds[row]);
      row_end = prefix[row] + pages(wants[row]) - first;
      granted = row_end <= sh.all;
      entries = p.table + row * p.stride + (first - prefix[row]);
    }
  }
  for (int b = all_tid; b < p.batch; b += kBookCtas * kBookThreads) {
    const int old = olds[b];
    int after = wants[b];
    if (after > old) {
      const int need = pages(after) - pages(old);
      if (need > 0 && prefix[b] + need > sh.all) {
        after = old;
        atomicOr(&g_adb_error_flag, kErrCacheFull);
      }
    }
    p.lens_out[b] = after;
  }
  cluster_leave();  // a peer may still read this CTA's shared memory
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

// 6 us for 12 forks, 7 us for 248.
//
// A child shares its parent's full pages (they no longer change) and gets a
// page of its own for the partly filled last one.  Each CTA keeps, redundantly,
// which fork a row is the child of (the first that names it), the tokens that
// each fork takes over and the prefix sum of the pages needed.
__global__ void __cluster_dims__(kBookCtas, 1, 1) __launch_bounds__(kBookThreads, 1)
    cache_fork_kernel(const ForkParams p) {
  extern __shared__ int fork_smem[];
  int* prefix = fork_smem;               // [forks]
  int* tokens = fork_smem + p.forks;     // [forks]: -1 where refused
  int* claim = fork_smem + 2 * p.forks;  // [batch]: first fork that names the row as its child
  __shared__ BookShared sh;
  const int tid = threadIdx.x, lane = tid & 31;
  const int all_tid = cluster_rank() * kBookThreads + tid;
  const int mask = (1 << p.page_shift) - 1;
  const int cap = p.max_blocks << p.page_shift;
  const unsigned rows = static_cast<unsigned>(p.batch);
  for (int b = tid; b < p.batch; b += kBookThreads) claim[b] = INT32_MAX;
  __syncthreads();
  griddep_launch_dependents();
  griddep_wait();
  // the pages' loads do not depend on the forks': issued first
  const auto is_free = [&](int page) { return __ldcg(&p.refs[page]) == 0; };
  const PageBits free = find_pages(p.num_blocks, is_free);
  for (int i = tid; i < p.forks; i += kBookThreads) {
    const int c = p.children[i];
    if (static_cast<unsigned>(c) < rows) atomicMin(&claim[c], i);
  }
  __syncthreads();
  int needed = 0;
  for (int base = 0; base < p.forks; base += kBookThreads) {
    const int i = base + tid;
    int n = -1;
    if (i < p.forks) {
      const int a = p.parents[i], c = p.children[i];
      if (static_cast<unsigned>(a) < rows && static_cast<unsigned>(c) < rows && claim[c] == i && p.lens[c] == 0)
        n = clamp_len(p.lens[a], cap);
      tokens[i] = n;
      if (n < 0 && cluster_rank() == 0) atomicOr(&g_adb_error_flag, kErrCacheRefused);
    }
    int sum;
    const int before = block_exclusive(n > 0 && (n & mask) != 0, sh, &sum);
    if (i < p.forks) prefix[i] = needed + before;
    needed += sum;
  }
  int rank = cluster_prefix<0>(free.count, sh);
  const int free_pages = sh.all;
  // every CTA has counted (the barrier in cluster_prefix): the counts may change now
  const auto granted = [&](int i, int n) { return n >= 0 && ((n & mask) == 0 || prefix[i] < free_pages); };

  // (a region of more pages than its bits hold is read again: only pages that were live change their count)
  for (int at = free.r.lo; at < free.r.hi && rank < needed; at += 32) {
    const unsigned hits = page_bits(free, at, is_free);
    const int mine = rank + __popc(hits & ((1u << lane) - 1));
    if ((hits >> lane & 1) && mine < needed) {
      // forks without a copy repeat the next prefix: the last one at `mine` is the one that needs it
      const int i = last_at_most(prefix, 0, p.forks - 1, mine);
      const int full = tokens[i] >> p.page_shift;
      const int page = p.table[p.parents[i] * p.stride + full];
      const bool in = static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks);
      if (!in) atomicOr(&g_adb_error_flag, kErrCachePage);
      p.src[i] = in ? page : -1;
      p.dst[i] = in ? at + lane : -1;
      p.table[p.children[i] * p.stride + full] = at + lane;
      p.refs[at + lane] = 1;
    }
    rank += __popc(hits);
  }

  for (int i = all_tid; i < p.forks; i += kBookCtas * kBookThreads) {
    const int n = tokens[i];
    if (!granted(i, n) || (n & mask) == 0) p.src[i] = p.dst[i] = -1;
    if (n >= 0 && !granted(i, n)) atomicOr(&g_adb_error_flag, kErrCacheFull);
  }
  for (int b = all_tid; b < p.batch; b += kBookCtas * kBookThreads) {
    const int i = claim[b];
    const int n = i < p.forks ? tokens[i] : -1;
    p.lens_out[b] = n >= 0 && granted(i, n) ? n : p.lens[b];
  }
  each_chunk(
      p.forks, p.max_blocks,
      [&](int i, int& from, int& to) {
        const int n = tokens[i];
        from = 0;
        to = granted(i, n) ? n >> p.page_shift : 0;
      },
      [&](int i, int from, int to) {
        const int32_t* from_row = p.table + p.parents[i] * p.stride;
        int32_t* to_row = p.table + p.children[i] * p.stride;
#pragma unroll
        for (int x = 0; x < kBookChunk / 32; ++x) {
          const int j = from + lane + 32 * x;
          if (j >= to) continue;
          const int page = from_row[j];
          to_row[j] = page;
          if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks))
            atomicAdd(&p.refs[page], 1);
          else
            atomicOr(&g_adb_error_flag, kErrCachePage);
        }
      });
  cluster_leave();
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

// 6 us for 224 pages, 7 us for 6681 of which 1600 move.
//
// With n live pages, the i-th live page at or above n moves to the i-th free
// page below n: the fewest copies that leave the live pages at the front, and
// no page is both a source and a destination.
__global__ void __cluster_dims__(kBookCtas, 1, 1) __launch_bounds__(kBookThreads, 1)
    cache_compact_kernel(const CompactParams p) {
  __shared__ BookShared sh;
  const int tid = threadIdx.x, lane = tid & 31;
  const int mask = (1 << p.page_shift) - 1;
  const int cap = p.max_blocks << p.page_shift;
  griddep_launch_dependents();
  griddep_wait();
  const auto is_live = [&](int page) { return __ldcg(&p.refs[page]) > 0; };
  const PageBits held = find_pages(p.num_blocks, is_live);
  int before = cluster_prefix<0>(held.count, sh);
  const int live = sh.all;
  // live pages below `live` stay; their count ranks the others
  int below = 0;
  for (int at = held.r.lo; at < held.r.hi && at < live; at += 32) {
    const unsigned bits = page_bits(held, at, is_live);
    below += __popc(live - at >= 32 ? bits : bits & ((1u << (live - at)) - 1));
  }
  cluster_prefix<1>(below, sh);
  const int stay = sh.all, moves = live - stay;
  for (int at = held.r.lo; at < held.r.hi; at += 32) {
    const int page = at + lane;
    const unsigned bits = page_bits(held, at, is_live);
    const bool mine_held = bits >> lane & 1;
    const int mine = before + __popc(bits & ((1u << lane) - 1));  // live pages before this one
    if (page < held.r.hi) {
      if (page >= live) {
        p.remap[page] = mine_held ? mine - stay : -1;
        if (mine_held) p.src[mine - stay] = page;
      } else if (!mine_held) {
        p.dst[page - mine] = page;
      }
    }
    before += __popc(bits);
  }
  cluster_sync();
  const int all_tid = cluster_rank() * kBookThreads + tid;
  for (int i = all_tid; i < p.num_blocks / 2; i += kBookCtas * kBookThreads) {
    if (i < moves) {
      const int from = __ldcg(&p.src[i]), to = __ldcg(&p.dst[i]);
      p.refs[to] = __ldcg(&p.refs[from]);
      p.refs[from] = 0;
    } else {
      p.src[i] = p.dst[i] = -1;
    }
  }
  each_chunk(
      p.batch, p.max_blocks,
      [&](int b, int& from, int& to) {
        from = 0;
        to = static_cast<int>((static_cast<unsigned>(clamp_len(p.lens[b], cap)) + mask) >> p.page_shift);
      },
      [&](int b, int from, int to) {
        int32_t* row = p.table + b * p.stride;
        int page[kBookChunk / 32], move[kBookChunk / 32];
#pragma unroll
        for (int x = 0; x < kBookChunk / 32; ++x) page[x] = from + lane + 32 * x < to ? row[from + lane + 32 * x] : 0;
#pragma unroll
        for (int x = 0; x < kBookChunk / 32; ++x) {
          const bool in = static_cast<unsigned>(page[x]) < static_cast<unsigned>(p.num_blocks);
          move[x] = -2;  // stays
          if (!in)
            move[x] = -1;
          else if (page[x] >= live)
            move[x] = __ldcg(&p.remap[page[x]]);  // -1: a page that refs calls free
        }
#pragma unroll
        for (int x = 0; x < kBookChunk / 32; ++x) {
          const int j = from + lane + 32 * x;
          if (j >= to || move[x] == -2) continue;
          if (move[x] >= 0)
            row[j] = __ldcg(&p.dst[move[x]]);
          else
            atomicOr(&g_adb_error_flag, kErrCachePage);
        }
      });
  cluster_leave();
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

// Bound by HBM: 1607 pages of 32 KB in each pool take 35 us, 105 MB read and as
// much written (6.0 TB/s).
//
// One unit is a part of one entry's page, of K and of V.  The lists that
// cache_compact returns are mostly -1 behind the moves, so each warp looks at
// 32 of its CTA's units at a time and the CTA copies the valid ones.
__global__ void __launch_bounds__(kCopyThreads) cache_copy_pages_kernel(const CopyParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t units = p.count * p.chunks;
  griddep_launch_dependents();
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
constexpr int kWriteVecs = 2;         // of K and of V per thread
constexpr int kWriteRows = 2048;      // rows whose offsets a block keeps in shared memory

// Bound by HBM for prompts (6204 tokens, 50.7 MB moved: 9.6 us; 134 MB: 23.7 us,
// 5.7 TB/s; 1 / 4 vectors per thread: 24.8 / 24.1 us), by latency for a step (32
// tokens: 2.6 us behind another).
//
// A block takes `tokens` tokens.  The source loads do not depend on the places,
// so they are issued first; meanwhile a thread per token finds its row, in
// offsets that the block has read at once, and its page.
__global__ void __launch_bounds__(kWriteThreads) cache_write_kernel(const WriteParams p, const int tokens) {
  __shared__ int cu[kWriteRows + 1], starts[kWriteRows];
  __shared__ int64_t place[kWriteThreads];  // element offset of head 0's row; -1: not written
  const int tid = threadIdx.x;
  const int head_vecs = p.dim >> 3, vecs = p.heads * head_vecs;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(tokens), p.total - first));
  const int64_t page_size = int64_t(1) << p.page_shift;
  const int64_t head_step = p.nhd ? p.dim : page_size * p.dim;
  griddep_launch_dependents();
  griddep_wait();
  const bool local = p.batch <= kWriteRows;
  if (local)
    for (int b = tid; b <= p.batch; b += kWriteThreads) {
      cu[b] = p.cu[b];
      if (b < p.batch) starts[b] = p.starts[b];
    }
  for (int base = 0; base < n * vecs; base += kWriteThreads * kWriteVecs) {
    uint4 k[kWriteVecs], v[kWriteVecs];
#pragma unroll
    for (int x = 0; x < kWriteVecs; ++x) {
      const int i = base + tid + x * kWriteThreads;
      if (i >= n * vecs) continue;
      const int t = i / vecs, r = i - t * vecs, head = r / head_vecs, e = (r - head * head_vecs) * 8;
      k[x] = __ldcs(reinterpret_cast<const uint4*>(p.k + (first + t) * p.k_token + head * p.k_head + e));
      v[x] = __ldcs(reinterpret_cast<const uint4*>(p.v + (first + t) * p.v_token + head * p.v_head + e));
    }
    if (base == 0) {
      __syncthreads();
      if (tid < n) {
        const int64_t t = first + tid;
        const int* offsets = local ? cu : p.cu;
        // last row whose tokens start at or before t
        int lo = 0, hi = p.batch - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (offsets[mid] <= t)
            lo = mid;
          else
            hi = mid - 1;
        }
        int64_t at = -1;
        if (t >= offsets[lo] && t < offsets[lo + 1]) {  // otherwise padding behind the last row
          const int64_t pos = static_cast<int64_t>(local ? starts[lo] : p.starts[lo]) + (t - offsets[lo]), j = pos >> p.page_shift;
          int page = -1;
          if (pos >= 0 && j < p.max_blocks) page = p.table[lo * p.stride + j];
          if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks)) {
            const int64_t slot = pos & (page_size - 1);
            at = p.nhd ? (page * page_size + slot) * p.heads * p.dim
                       : (static_cast<int64_t>(page) * p.heads * page_size + slot) * p.dim;
          } else {
            atomicOr(&g_adb_error_flag, kErrCachePage);
          }
        }
        place[tid] = at;
      }
      __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < kWriteVecs; ++x) {
      const int i = base + tid + x * kWriteThreads;
      if (i >= n * vecs) continue;
      const int t = i / vecs, r = i - t * vecs, head = r / head_vecs, e = (r - head * head_vecs) * 8;
      if (place[t] < 0) continue;
      const int64_t at = place[t] + head * head_step + e;
      *reinterpret_cast<uint4*>(p.k_cache + at) = k[x];
      *reinterpret_cast<uint4*>(p.v_cache + at) = v[x];
    }
  }
}

}  // namespace adb
