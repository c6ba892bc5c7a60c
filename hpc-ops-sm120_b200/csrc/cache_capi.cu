// cache_capi.cu -- host side of the paged-cache operators: argument checks and
// launches of the kernels in cache_kernels.cuh.  Every check is made on the
// host before the device is touched; a captured call reads its lengths,
// tables and lists from device memory when it runs.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "attention_decode_b200.h"
#include "cache_kernels.cuh"
#include "host_common.h"

namespace adb_host {

cudaError_t cache_error_word(int* word, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(word, adb::g_adb_error_flag, sizeof(int));
  const int zero = 0;
  if (e == cudaSuccess && reset) e = cudaMemcpyToSymbol(adb::g_adb_error_flag, &zero, sizeof(int));
  return e;
}

}  // namespace adb_host

namespace {

using adb_host::cuda_fail;
using adb_host::DeviceGuard;
using adb_host::fail;
using adb_host::is_aligned;

constexpr int64_t kMaxRows = 16384;  // rows or forks of one bookkeeping call: three ints each in shared memory
constexpr int kMaxBookSmem = 3 * kMaxRows * sizeof(int);

int check_pages(int64_t page_size, int64_t num_blocks, int64_t max_blocks, int* shift) {
  if (page_size < 8 || page_size > (1 << 20) || (page_size & (page_size - 1)) != 0)
    return fail(ADB_ERR_UNSUPPORTED, "page size must be a power of two from 8 to 2^20 (got %lld)",
                (long long)page_size);
  if (num_blocks <= 0 || max_blocks <= 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "num_blocks and max_blocks_per_seq must be positive");
  if (num_blocks > (1 << 30) || max_blocks > INT32_MAX / page_size)
    return fail(ADB_ERR_INVALID_ARGUMENT, "num_blocks must be at most 2^30 and max_blocks_per_seq * page_size below 2^31");
  *shift = 0;
  while ((int64_t(1) << *shift) < page_size) ++*shift;
  return ADB_OK;
}

int check_rows(const void* table, int64_t stride, const void* lens, int64_t batch, int64_t max_blocks) {
  if (table == nullptr || lens == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "block table and sequence lengths must be non-null");
  if (batch <= 0) return fail(ADB_ERR_INVALID_ARGUMENT, "batch must be positive");
  if (batch > kMaxRows)
    return fail(ADB_ERR_UNSUPPORTED, "at most %lld rows per call (got %lld)", (long long)kMaxRows, (long long)batch);
  if (stride < max_blocks)
    return fail(ADB_ERR_INVALID_ARGUMENT, "block table row stride %lld is below max_blocks_per_seq %lld",
                (long long)stride, (long long)max_blocks);
  if (batch * max_blocks > INT32_MAX)
    return fail(ADB_ERR_INVALID_ARGUMENT, "the block table must have fewer than 2^31 entries");
  return ADB_OK;
}

// Once per device: the shared memory that the rows of a resize or fork may take.
// Whatever this call's size: beyond 48 KB in all a kernel needs the permission,
// and beside its dynamic part it has a static one.
int prepare(int device) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = uint64_t(1) << device;
  if (done.load(std::memory_order_acquire) & bit) return ADB_OK;
  for (const void* kernel : {reinterpret_cast<const void*>(&adb::cache_resize_kernel),
                             reinterpret_cast<const void*>(&adb::cache_fork_kernel)}) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBookSmem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(max dynamic smem)");
  }
  done.fetch_or(bit, std::memory_order_release);
  return ADB_OK;
}

// Launches `kernel` with programmatic stream serialisation (it waits for the
// kernels before it itself).
template <typename... Args>
int launch(void (*kernel)(Args...), int64_t grid, int threads, size_t smem, int device, void* stream,
           const char* what, Args... args) {
  DeviceGuard guard(device);
  if (guard.error != cudaSuccess) return cuda_fail(guard.error, "cudaSetDevice");
  int sms = 0;
  int rc = adb_host::sm_count(device, &sms);  // refuses other devices
  if (rc == ADB_OK && smem > 0) rc = prepare(device);
  if (rc != ADB_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return cuda_fail(e, what);
  adb_host::count_launch();
  return ADB_OK;
}

}  // namespace

extern "C" {

int adb_cache_write(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                    int64_t v_token_stride, int64_t v_head_stride, void* k_cache, void* v_cache,
                    const int32_t* block_table, int64_t block_table_stride, const int32_t* cu_seqlens,
                    const int32_t* starts, int64_t total, int64_t batch, int64_t kv_heads, int64_t head_dim,
                    int64_t num_blocks, int64_t page_size, int64_t max_blocks_per_seq, int layout, int device,
                    void* stream) {
  if (k == nullptr || v == nullptr || k_cache == nullptr || v_cache == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "K, V and cache pointers must be non-null");
  if (block_table == nullptr || cu_seqlens == nullptr || starts == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "cache write needs a block table, cu_seqlens and starts");
  if (layout != ADB_PAGED_HND && layout != ADB_PAGED_NHD)
    return fail(ADB_ERR_INVALID_ARGUMENT, "unknown paged layout %d (ADB_PAGED_HND or ADB_PAGED_NHD)", layout);
  if (total <= 0 || batch <= 0 || kv_heads <= 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "tokens, batch and KV heads must be positive");
  if (batch >= INT32_MAX || total > INT32_MAX)
    return fail(ADB_ERR_INVALID_ARGUMENT, "tokens and batch must be below 2^31");
  if (kv_heads > (1 << 16))
    return fail(ADB_ERR_UNSUPPORTED, "at most 65536 KV heads are supported (got %lld)", (long long)kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return fail(ADB_ERR_UNSUPPORTED, "head dimension must be 64 or 128 (got %lld)", (long long)head_dim);
  int shift = 0;
  const int rc = check_pages(page_size, num_blocks, max_blocks_per_seq, &shift);
  if (rc != ADB_OK) return rc;
  if (num_blocks * kv_heads > INT32_MAX)
    return fail(ADB_ERR_INVALID_ARGUMENT, "num_blocks * kv_heads exceeds 2^31-1");
  if (block_table_stride < max_blocks_per_seq)
    return fail(ADB_ERR_INVALID_ARGUMENT, "block table row stride %lld is below max_blocks_per_seq %lld",
                (long long)block_table_stride, (long long)max_blocks_per_seq);
  if (!is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(k_cache, 16) || !is_aligned(v_cache, 16) ||
      ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) != 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "K, V and caches must be 16-byte aligned, strides multiples of 8 elements");
  int sms = 0;
  const int status = adb_host::sm_count(device, &sms);
  if (status != ADB_OK) return status;
  // tokens per block: as many as fill its threads' loads, fewer where the GPU would not be filled
  const int64_t vecs = kv_heads * (head_dim / 8);
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(adb::kWriteThreads, adb::kWriteThreads * adb::kWriteVecs / vecs));
  const int64_t tokens = std::max<int64_t>(1, std::min<int64_t>(most, total / (2 * sms)));
  const int64_t blocks = (total + tokens - 1) / tokens;
  adb::WriteParams p;
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.k_token = k_token_stride;
  p.k_head = k_head_stride;
  p.v_token = v_token_stride;
  p.v_head = v_head_stride;
  p.k_cache = static_cast<__nv_bfloat16*>(k_cache);
  p.v_cache = static_cast<__nv_bfloat16*>(v_cache);
  p.table = block_table;
  p.stride = block_table_stride;
  p.cu = cu_seqlens;
  p.starts = starts;
  p.total = total;
  p.batch = static_cast<int>(batch);
  p.heads = static_cast<int>(kv_heads);
  p.dim = static_cast<int>(head_dim);
  p.max_blocks = static_cast<int>(max_blocks_per_seq);
  p.num_blocks = static_cast<int>(num_blocks);
  p.page_shift = shift;
  p.nhd = layout == ADB_PAGED_NHD;
  return launch(&adb::cache_write_kernel, blocks, adb::kWriteThreads, 0, device, stream, "cache write launch", p,
                static_cast<int>(tokens));
}

int adb_cache_copy_pages(void* k_cache, void* v_cache, const int32_t* src, const int32_t* dst, int64_t count,
                         int64_t num_blocks, int64_t page_bytes, int device, void* stream) {
  if (k_cache == nullptr || v_cache == nullptr || src == nullptr || dst == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "cache and page list pointers must be non-null");
  if (count <= 0 || num_blocks <= 0 || num_blocks > (1 << 30) || page_bytes <= 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "count, num_blocks and page_bytes must be positive");
  if (!is_aligned(k_cache, 16) || !is_aligned(v_cache, 16) || (page_bytes & 15) != 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "caches must be 16-byte aligned, pages a multiple of 16 bytes");
  adb::CopyParams p;
  p.k = static_cast<uint4*>(k_cache);
  p.v = static_cast<uint4*>(v_cache);
  p.src = src;
  p.dst = dst;
  p.count = count;
  p.page_vecs = page_bytes / 16;
  const int64_t chunks = (p.page_vecs + adb::kCopyVecs - 1) / adb::kCopyVecs;
  if (chunks > INT32_MAX) return fail(ADB_ERR_INVALID_ARGUMENT, "page too large");
  p.chunks = static_cast<int>(chunks);
  p.num_blocks = static_cast<int>(num_blocks);
  int sms = 0;
  const int rc = adb_host::sm_count(device, &sms);
  if (rc != ADB_OK) return rc;
  const int64_t grid = std::min<int64_t>(count * chunks, 8 * sms);
  return launch(&adb::cache_copy_pages_kernel, grid, adb::kCopyThreads, 0, device, stream, "page copy launch", p);
}

int adb_cache_resize(int32_t* block_table, int64_t block_table_stride, const int32_t* seqlens,
                     const int32_t* new_lens, int32_t* page_refs, int32_t* lens_out, int64_t batch,
                     int64_t num_blocks, int64_t page_size, int64_t max_blocks_per_seq, int device, void* stream) {
  int rc = check_rows(block_table, block_table_stride, seqlens, batch, max_blocks_per_seq);
  if (rc != ADB_OK) return rc;
  if (new_lens == nullptr || page_refs == nullptr || lens_out == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "resize needs the new lengths, page_refs and an output");
  adb::ResizeParams p;
  rc = check_pages(page_size, num_blocks, max_blocks_per_seq, &p.page_shift);
  if (rc != ADB_OK) return rc;
  p.table = block_table;
  p.stride = block_table_stride;
  p.lens = seqlens;
  p.want = new_lens;
  p.refs = page_refs;
  p.lens_out = lens_out;
  p.batch = static_cast<int>(batch);
  p.max_blocks = static_cast<int>(max_blocks_per_seq);
  p.num_blocks = static_cast<int>(num_blocks);
  return launch(&adb::cache_resize_kernel, adb::kBookCtas, adb::kBookThreads, 3 * batch * sizeof(int), device, stream,
                "cache resize launch", p);
}

int adb_cache_fork(int32_t* block_table, int64_t block_table_stride, const int32_t* seqlens, int32_t* page_refs,
                   const int32_t* parents, const int32_t* children, int64_t forks, int32_t* lens_out, int32_t* src,
                   int32_t* dst, int64_t batch, int64_t num_blocks, int64_t page_size, int64_t max_blocks_per_seq,
                   int device, void* stream) {
  int rc = check_rows(block_table, block_table_stride, seqlens, batch, max_blocks_per_seq);
  if (rc != ADB_OK) return rc;
  if (page_refs == nullptr || parents == nullptr || children == nullptr || lens_out == nullptr || src == nullptr ||
      dst == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "fork needs page_refs, parents, children and its outputs");
  if (forks <= 0 || forks > kMaxRows)
    return fail(ADB_ERR_UNSUPPORTED, "1 to %lld forks per call (got %lld)", (long long)kMaxRows, (long long)forks);
  if (forks * max_blocks_per_seq > INT32_MAX)
    return fail(ADB_ERR_INVALID_ARGUMENT, "forks * max_blocks_per_seq must be below 2^31");
  adb::ForkParams p;
  rc = check_pages(page_size, num_blocks, max_blocks_per_seq, &p.page_shift);
  if (rc != ADB_OK) return rc;
  p.table = block_table;
  p.stride = block_table_stride;
  p.lens = seqlens;
  p.refs = page_refs;
  p.parents = parents;
  p.children = children;
  p.lens_out = lens_out;
  p.src = src;
  p.dst = dst;
  p.batch = static_cast<int>(batch);
  p.forks = static_cast<int>(forks);
  p.max_blocks = static_cast<int>(max_blocks_per_seq);
  p.num_blocks = static_cast<int>(num_blocks);
  return launch(&adb::cache_fork_kernel, adb::kBookCtas, adb::kBookThreads, (batch + 2 * forks) * sizeof(int), device,
                stream, "cache fork launch", p);
}

int adb_cache_compact(int32_t* block_table, int64_t block_table_stride, const int32_t* seqlens, int32_t* page_refs,
                      int32_t* src, int32_t* dst, int32_t* remap, int64_t batch, int64_t num_blocks,
                      int64_t page_size, int64_t max_blocks_per_seq, int device, void* stream) {
  int rc = check_rows(block_table, block_table_stride, seqlens, batch, max_blocks_per_seq);
  if (rc != ADB_OK) return rc;
  if (page_refs == nullptr || remap == nullptr || (num_blocks > 1 && (src == nullptr || dst == nullptr)))
    return fail(ADB_ERR_INVALID_ARGUMENT, "compact needs page_refs, its outputs and a scratch of num_blocks");
  adb::CompactParams p;
  rc = check_pages(page_size, num_blocks, max_blocks_per_seq, &p.page_shift);
  if (rc != ADB_OK) return rc;
  p.table = block_table;
  p.stride = block_table_stride;
  p.lens = seqlens;
  p.refs = page_refs;
  p.src = src;
  p.dst = dst;
  p.remap = remap;
  p.batch = static_cast<int>(batch);
  p.max_blocks = static_cast<int>(max_blocks_per_seq);
  p.num_blocks = static_cast<int>(num_blocks);
  return launch(&adb::cache_compact_kernel, adb::kBookCtas, adb::kBookThreads, 0, device, stream,
                "cache compact launch", p);
}

}  // extern "C"
