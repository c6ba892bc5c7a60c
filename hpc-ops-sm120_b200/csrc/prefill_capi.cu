// prefill_capi.cu -- host side of prompt attention: argument checks and
// launches of the kernels in prefill_kernels.cuh.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
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

constexpr int64_t kL2Bytes = 96 << 20;  // of 126 MB, with room for Q and O

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

// Tensor map over bf16 with a 128-byte swizzle; dims and strides (elements)
// innermost first, the innermost box always 64 columns.
int encode(CUtensorMap* map, const void* base, int rank, const int64_t* dims, const int64_t* strides, const int* box) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  const int rc = adb_host::get_encoder(&fn);
  if (rc != ADB_OK) return rc;
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], one[5] = {1u, 1u, 1u, 1u, 1u};
  for (int i = 0; i < rank; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i]);
    b[i] = static_cast<cuuint32_t>(box[i]);
    if (i > 0) s[i - 1] = static_cast<cuuint64_t>(strides[i] * 2);
  }
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), d, s, b, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ADB_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", int(r));
  return ADB_OK;
}

// [tokens][heads][D] with a box of `rows` tokens x `heads_box` heads.
int encode_packed(CUtensorMap* map, const void* base, int64_t tokens, int64_t heads, int64_t dim, int64_t token_stride,
                  int64_t head_stride, int heads_box, int rows) {
  const int64_t dims[3] = {dim, heads, tokens}, strides[3] = {1, head_stride, token_stride};
  const int box[3] = {64, heads_box, rows};
  return encode(map, base, 3, dims, strides, box);
}

// Pages of either layout as [blocks][heads][64-column blocks][tokens][64].
int encode_pages(CUtensorMap* map, const void* base, const adb::PrefillParams& p, int64_t dim, bool pair) {
  const int64_t page = int64_t(1) << p.page_shift, heads = p.kv_heads;
  const int rows = static_cast<int>(page < adb::kTile ? page : adb::kTile);
  const bool hnd = p.paged == 1;
  const int64_t dims[5] = {64, page, dim / 64, heads, p.num_blocks};
  const int64_t strides[5] = {1, hnd ? dim : heads * dim, 64, hnd ? page * dim : dim, heads * page * dim};
  const int box[5] = {64, rows, pair ? 2 : 1, 1, 1};
  return encode(map, base, 5, dims, strides, box);
}

struct Kernel {
  void (*run)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const adb::PrefillParams);
  int smem;
};
const Kernel kKernels[] = {{adb::prefill_kernel<64, false>, adb::PrefillCfg<64>::kSmemBytes},
                           {adb::prefill_kernel<128, false>, adb::PrefillCfg<128>::kSmemBytes},
                           {adb::prefill_kernel<128, true>, adb::PrefillCfg<128>::kSmemBytes}};

// Once per device: the kernels' shared-memory limit, and that they were
// compiled to the registers that the split between their warps counts on.
int prepare(int device) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = uint64_t(1) << device;
  if (done.load(std::memory_order_acquire) & bit) return ADB_OK;
  for (const Kernel& k : kKernels) {
    const void* fn = reinterpret_cast<const void*>(k.run);
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(max dynamic smem)");
    cudaFuncAttributes a;
    e = cudaFuncGetAttributes(&a, fn);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes");
    if (a.numRegs * 3 < 2 * adb::kSoftmaxRegs + adb::kOtherRegs)
      return fail(ADB_ERR_CUDA, "the prefill kernel was compiled to %d registers, too few for its split", a.numRegs);
  }
  done.fetch_or(bit, std::memory_order_release);
  return ADB_OK;
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Workspace, of nothing but parts: O, (maximum, total), the list of what to
// join.  The kernel makes at most as many more units by cutting as there are
// SMs, so that at most twice as many are parts (a cut pair has two or more).
struct Workspace {
  int64_t slots, rows;  // no slots: nothing can be cut into parts
  size_t off_ml, off_joins, off_count, bytes;
};

// `max_keys`: of a sequence in the cache, or 0 for packed prompts.
Workspace plan_workspace(int64_t total, int64_t kv_heads, int64_t group, int64_t dim, int64_t max_keys, int64_t sms) {
  // A cut needs a sequence of one and a half of the smallest parts.  The pairs
  // of a prompt of n tokens have n / 256 tiles on average, so that only short
  // prompts of few KV heads are longer than their even share.
  const int64_t longest =
      max_keys > 0 ? max_keys : std::min<int64_t>(total, 2 * (adb::kTile / group) * sms * 4 / (3 * kv_heads));
  Workspace w = {};
  if (longest <= (max_keys > 0 ? 3 * adb::kMinPart / 2 - 1 : 2 * adb::kMinPart) * adb::kTile) return w;
  w.slots = 2 * sms;
  w.rows = std::min<int64_t>(2 * (adb::kTile / group), total) * group;
  w.off_ml = align256(static_cast<size_t>(w.slots * w.rows * dim) * sizeof(float));
  w.off_joins = w.off_ml + align256(static_cast<size_t>(w.slots * w.rows) * sizeof(float2));
  w.off_count = w.off_joins + align256(static_cast<size_t>(w.slots / 2) * sizeof(adb::PrefillJoin));
  w.bytes = w.off_count + 256;
  return w;
}

// `k`, the K tensor; p holds everything else.
int launch(adb::PrefillParams& p, const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
           int64_t k_head, int64_t dim, void* workspace, size_t workspace_bytes, int device, void* stream) {
  DeviceGuard guard(device);
  if (guard.error != cudaSuccess) return cuda_fail(guard.error, "cudaSetDevice");
  int sms = 0;
  int rc = adb_host::sm_count(device, &sms);
  if (rc == ADB_OK) rc = prepare(device);
  if (rc != ADB_OK) return rc;
  p.scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(dim)));
  p.tile_tokens = adb::kTile / p.group;
  p.group_magic = (65536 + p.group - 1) / p.group;
  // one box of both 64-column blocks where a page is too small to pay for two
  // (one token over 131072, pages of 8 / 16 / 64 tokens: 180 / 119 / 105 us with
  // two, 118 / 110 us with one)
  const bool pair = p.paged && dim == 128 && p.page_shift <= 4;
  CUtensorMap q_map, k_map, v_map;
  rc = encode_packed(&q_map, q, p.total, p.q_heads, dim, q_token, q_head, p.group, p.tile_tokens);
  if (rc != ADB_OK) return rc;
  if (p.paged) {
    rc = encode_pages(&k_map, k, p, dim, pair);
    if (rc == ADB_OK) rc = encode_pages(&v_map, p.v, p, dim, pair);
  } else {
    rc = encode_packed(&k_map, k, p.total, p.kv_heads, dim, k_token, k_head, 1, adb::kTile);
    if (rc == ADB_OK) rc = encode_packed(&v_map, p.v, p.total, p.kv_heads, dim, p.v_token, p.v_head, 1, adb::kTile);
  }
  if (rc != ADB_OK) return rc;
  // every sequence with a token may end in a partly filled pair of tiles
  const int64_t per = 2 * p.tile_tokens;
  const int64_t pairs = p.total / per + std::min(p.batch, p.total);
  const int64_t max_keys = p.paged ? int64_t(p.max_blocks) << p.page_shift : 0;
  const Workspace ws = plan_workspace(p.total, p.kv_heads, p.group, dim, max_keys, sms);
  if (ws.slots > 0 && (workspace == nullptr || !is_aligned(workspace, 256)))
    return fail(ADB_ERR_WORKSPACE, "workspace must be a non-null 256-byte aligned device buffer");
  if (workspace_bytes < ws.bytes)
    return fail(ADB_ERR_WORKSPACE, "workspace too small: %zu bytes given, %zu needed", workspace_bytes, ws.bytes);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  p.sms = sms;
  p.slot_rows = static_cast<int>(ws.rows);
  p.part_o = reinterpret_cast<float*>(base);
  p.part_ml = reinterpret_cast<float2*>(base + ws.off_ml);
  p.joins = reinterpret_cast<adb::PrefillJoin*>(base + ws.off_joins);
  p.join_count = reinterpret_cast<int*>(base + ws.off_count);
  p.max_slots = static_cast<int>(ws.slots);
  // KV heads worked on at a time: even groups that keep the longest possible
  // sequence's K and V in L2
  const int64_t keys = p.paged ? max_keys : p.total;
  const int64_t groups = std::min<int64_t>(p.kv_heads, (p.kv_heads * keys * dim * 4 + kL2Bytes - 1) / kL2Bytes);
  p.head_group = static_cast<int>((p.kv_heads + groups - 1) / groups);
  const int64_t grid = pairs * p.kv_heads + (ws.slots > 0 ? sms : 0);
  if (grid > INT32_MAX) return fail(ADB_ERR_INVALID_ARGUMENT, "too many tiles for one call");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(adb::kPrefillThreads);
  const Kernel& kernel = kKernels[dim == 64 ? 0 : pair ? 2 : 1];
  cfg.dynamicSmemBytes = static_cast<size_t>(kernel.smem);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel.run, q_map, k_map, v_map, p);
  if (e != cudaSuccess) return cuda_fail(e, "prefill kernel launch");
  adb_host::count_launch();
  if (ws.slots == 0) return ADB_OK;
  const int64_t join_rows = ws.slots / 2 * ws.rows;
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(2 * sms, (join_rows + 7) / 8)));
  cfg.blockDim = dim3(adb::kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, dim == 128 ? adb::prefill_join_kernel<128> : adb::prefill_join_kernel<64>, p);
  if (e != cudaSuccess) return cuda_fail(e, "prefill join kernel launch");
  adb_host::count_launch();
  return ADB_OK;
}

}  // namespace

extern "C" {

int adb_prefill_workspace_size(int64_t total, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                               int64_t max_keys, int device, size_t* bytes) {
  if (bytes == nullptr) return fail(ADB_ERR_INVALID_ARGUMENT, "bytes pointer is null");
  const int rc = check_heads(total, batch, q_heads, kv_heads, head_dim);
  if (rc != ADB_OK) return rc;
  if (max_keys < 0) return fail(ADB_ERR_INVALID_ARGUMENT, "max_keys must not be negative");
  int sms = 0;
  const int status = adb_host::sm_count(device, &sms);
  if (status != ADB_OK) return status;
  *bytes = plan_workspace(total, kv_heads, q_heads / kv_heads, head_dim, max_keys, sms).bytes;
  return ADB_OK;
}

int adb_prefill(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                const int32_t* cu_seqlens, void* out, int64_t total, int64_t batch, int64_t q_heads,
                int64_t kv_heads, int64_t head_dim, void* workspace, size_t workspace_bytes, int device,
                void* stream) {
  const int rc = check_heads(total, batch, q_heads, kv_heads, head_dim);
  if (rc != ADB_OK) return rc;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || cu_seqlens == nullptr)
    return fail(ADB_ERR_INVALID_ARGUMENT, "Q, K, V, cu_seqlens and output pointers must be non-null");
  if (!is_aligned(q, 16) || !is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(out, 16) ||
      ((q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) != 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "Q, K and V must be 16-byte aligned, their strides multiples of 8 elements");
  adb::PrefillParams p = {};
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.v_token = v_token_stride;
  p.v_head = v_head_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.cu = cu_seqlens;
  p.total = static_cast<int>(total);
  p.batch = static_cast<int>(batch);
  p.q_heads = static_cast<int>(q_heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = static_cast<int>(q_heads / kv_heads);
  return launch(p, q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, head_dim, workspace,
                workspace_bytes, device, stream);
}

int adb_prefill_paged(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k_cache,
                      const void* v_cache, const int32_t* block_table, int64_t block_table_stride,
                      const int32_t* cu_seqlens, const int32_t* seqlens, void* out, int64_t total, int64_t batch,
                      int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t page_size,
                      int64_t max_blocks_per_seq, int layout, void* workspace, size_t workspace_bytes, int device,
                      void* stream) {
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
  if (num_blocks > INT32_MAX / kv_heads || max_blocks_per_seq > (1 << 30) / page_size)
    return fail(ADB_ERR_INVALID_ARGUMENT,
                "num_blocks * kv_heads must be below 2^31, max_blocks_per_seq * page_size at most 2^30");
  if (block_table_stride < max_blocks_per_seq)
    return fail(ADB_ERR_INVALID_ARGUMENT, "block table row stride %lld is below max_blocks_per_seq %lld",
                (long long)block_table_stride, (long long)max_blocks_per_seq);
  if (!is_aligned(q, 16) || !is_aligned(k_cache, 16) || !is_aligned(v_cache, 16) || !is_aligned(out, 16) ||
      ((q_token_stride | q_head_stride) & 7) != 0)
    return fail(ADB_ERR_INVALID_ARGUMENT, "Q and caches must be 16-byte aligned, Q's strides multiples of 8 elements");
  adb::PrefillParams p = {};
  p.v = static_cast<const __nv_bfloat16*>(v_cache);
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
  return launch(p, q, q_token_stride, q_head_stride, k_cache, 0, 0, head_dim, workspace, workspace_bytes, device,
                stream);
}

}  // extern "C"
