// prefill_capi.cu -- host side of prompt attention: argument checks and
// launches of the kernels in prefill_kernels.cuh.
#include <cuda_runtime.h>

#include <cmath>

#include "attention_decode_b200.h"
#include "host_common.h"
#include "prefill_kernels.cuh"

namespace adb_host {

cudaError_t prefill_error_word(int* word, bool reset) {
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

int check_heads(int64_t total, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
  if (total <= 0 || batch <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0)
    return fail(ADB_ERR_INVALID_ARGUMENT,
                "all dimensions must be positive: tokens=%lld batch=%lld q_heads=%lld kv_heads=%lld head_dim=%lld",
                (long long)total, (long long)batch, (long long)q_heads, (long long)kv_heads, (long long)head_dim);
  if (q_heads % kv_heads != 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "query heads (%lld) must be divisible by KV heads (%lld)",
                (long long)q_heads, (long long)kv_heads);
  if (q_heads / kv_heads > 64)
    return fail(ADB_ERR_UNSUPPORTED, "GQA groups up to 64 are supported (got %lld)", (long long)(q_heads / kv_heads));
  if (head_dim != 64 && head_dim != 128)
    return fail(ADB_ERR_UNSUPPORTED, "head dimension must be 64 or 128 (got %lld)", (long long)head_dim);
  if (total > (1 << 30) || batch > (1 << 30) || q_heads > (1 << 16) || total * q_heads > INT32_MAX)
    return fail(ADB_ERR_INVALID_ARGUMENT, "tokens * query heads must be below 2^31");
  return ADB_OK;
}

int launch(adb::PrefillParams& p, int64_t head_dim, int device, void* stream) {
  DeviceGuard guard(device);
  if (guard.error != cudaSuccess) return cuda_fail(guard.error, "cudaSetDevice");
  int sms = 0;
  const int rc = adb_host::sm_count(device, &sms);
  if (rc != ADB_OK) return rc;
  p.scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(head_dim)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(p.total) * p.q_heads + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(
      &cfg, head_dim == 128 ? adb::prefill_rows_kernel<128> : adb::prefill_rows_kernel<64>, p);
  if (e != cudaSuccess) return cuda_fail(e, "prefill kernel launch");
  adb_host::count_launch();
  return ADB_OK;
}

}  // namespace

extern "C" {

int adb_prefill_workspace_size(int64_t total, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                               int device, size_t* bytes, size_t* header_bytes) {
  if (bytes == nullptr) return fail(ADB_ERR_INVALID_ARGUMENT, "bytes pointer is null");
  const int rc = check_heads(total, batch, q_heads, kv_heads, head_dim);
  if (rc != ADB_OK) return rc;
  (void)device;
  *bytes = 256;
  if (header_bytes != nullptr) *header_bytes = 0;
  return ADB_OK;
}

int adb_prefill(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                const int32_t* cu_seqlens, void* out, int64_t total, int64_t batch, int64_t q_heads,
                int64_t kv_heads, int64_t head_dim, void* workspace, size_t workspace_bytes, unsigned flags,
                int device, void* stream) {
  const int rc = check_heads(total, batch, q_heads, kv_heads, head_dim);
  if (rc != ADB_OK) return rc;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || cu_seqlens == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "Q, K, V, cu_seqlens and output pointers must be non-null");
  if (!is_aligned(q, 16) || !is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(out, 16) ||
      ((q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) != 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "Q, K and V must be 16-byte aligned, their strides multiples of 8 elements");
  adb::PrefillParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.k_token = k_token_stride;
  p.k_head = k_head_stride;
  p.v_token = v_token_stride;
  p.v_head = v_head_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.cu = cu_seqlens;
  p.total = static_cast<int>(total);
  p.batch = static_cast<int>(batch);
  p.q_heads = static_cast<int>(q_heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = static_cast<int>(q_heads / kv_heads);
  return launch(p, head_dim, device, stream);
}

int adb_prefill_paged(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k_cache,
                      const void* v_cache, const int32_t* block_table, int64_t block_table_stride,
                      const int32_t* cu_seqlens, const int32_t* seqlens, void* out, int64_t total, int64_t batch,
                      int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t page_size,
                      int64_t max_blocks_per_seq, int layout, void* workspace, size_t workspace_bytes,
                      unsigned flags, int device, void* stream) {
  const int rc = check_heads(total, batch, q_heads, kv_heads, head_dim);
  if (rc != ADB_OK) return rc;
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || out == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "Q, cache and output pointers must be non-null");
  if (block_table == nullptr || cu_seqlens == nullptr || seqlens == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "paged prefill needs a block table, cu_seqlens and sequence lengths");
  if (layout != ADB_PAGED_HND && layout != ADB_PAGED_NHD)
    return fail(ADB_ERR_INVALID_ARGUMENT, "unknown paged layout %d (ADB_PAGED_HND or ADB_PAGED_NHD)", layout);
  if (page_size < 8 || page_size > (1 << 20) || (page_size & (page_size - 1)) != 0)
    return fail(ADB_ERR_UNSUPPORTED, "page size must be a power of two from 8 to 2^20 (got %lld)",
                (long long)page_size);
  if (num_blocks <= 0 || max_blocks_per_seq <= 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "num_blocks and max_blocks_per_seq must be positive");
  if (num_blocks > INT32_MAX / kv_heads || max_blocks_per_seq > INT32_MAX / page_size)
    return fail(ADB_ERR_INVALID_ARGUMENT,
                "num_blocks * kv_heads and max_blocks_per_seq * page_size must be below 2^31");
  if (block_table_stride < max_blocks_per_seq)
    return fail(ADB_ERR_INVALID_ARGUMENT, "block table row stride %lld is below max_blocks_per_seq %lld",
                (long long)block_table_stride, (long long)max_blocks_per_seq);
  if (!is_aligned(q, 16) || !is_aligned(k_cache, 16) || !is_aligned(v_cache, 16) || !is_aligned(out, 16) ||
      ((q_token_stride | q_head_stride) & 7) != 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "Q and caches must be 16-byte aligned, Q's strides multiples of 8 elements");
  adb::PrefillParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k_cache);
  p.v = static_cast<const __nv_bfloat16*>(v_cache);
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.cu = cu_seqlens;
  p.lens = seqlens;
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.total = static_cast<int>(total);
  p.batch = static_cast<int>(batch);
  p.q_heads = static_cast<int>(q_heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = static_cast<int>(q_heads / kv_heads);
  p.paged = layout == ADB_PAGED_HND ? 1 : 2;
  p.max_blocks = static_cast<int>(max_blocks_per_seq);
  p.num_blocks = static_cast<int>(num_blocks);
  while ((int64_t(1) << p.page_shift) < page_size) ++p.page_shift;
  return launch(p, head_dim, device, stream);
}

}  // extern "C"
