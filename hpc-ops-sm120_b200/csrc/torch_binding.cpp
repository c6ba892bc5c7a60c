// torch_binding.cpp -- the PyTorch C++ extension of this library.
//
// Replaces the reference's pybind module (csrc/binding.cpp:3-8), whose
// `forward(q, k, v)` is attention_decode_cuda (csrc/decode.cu:223-258): the
// same name, argument meaning, checks and error messages (TORCH_CHECK ->
// RuntimeError), the output a fresh tensor like q, every launch on the
// current CUDA stream with no host synchronisation.  The kernels are not
// compiled here: this module calls the C ABI of libattention_decode_b200.so
// (include/attention_decode_b200.h), which it links against and finds next
// to itself.
//
// Additions, all compatible with the 3-argument call: an optional int32
// `seqlens` [B] on forward, forward_partial (unnormalised (acc, m, l) states
// for sequence sharding) and combine (merge of R such states); prompt attention
// (prefill, prefill_paged) and the upkeep of a paged cache (cache_*).
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime_api.h>

#include <map>
#include <mutex>
#include <string>
#include <utility>

#include "attention_decode_b200.h"

namespace {

void check_status(int status) {
  TORCH_CHECK(status == ADB_OK, "attention_decode: ", adb_last_error());
}

// The reference's input contract (csrc/decode.cu:225-241 and
// attention_decode/__init__.py:35-38), with the INT_MAX element limit
// dropped (64-bit indexing) and a GQA group of 8 accepted.
void check_inputs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                  const c10::optional<at::Tensor>& seqlens) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "Q, K, and V must be CUDA tensors");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 &&
                  v.scalar_type() == at::kBFloat16,
              "Q/K/V dtype must be BF16 (bfloat16)");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "Q/K/V must have rank four");
  TORCH_CHECK(q.is_contiguous() && k.is_contiguous() && v.is_contiguous(), "Q/K/V must be contiguous");
  TORCH_CHECK(!q.requires_grad() && !k.requires_grad() && !v.requires_grad(),
              "attention_decode is forward inference only; no backward/grad support");
  TORCH_CHECK(q.numel() > 0 && k.numel() > 0 && v.numel() > 0, "empty tensors are unsupported");
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "Q/K/V device must match");
  TORCH_CHECK(k.sizes() == v.sizes(), "K/V shape must match");
  TORCH_CHECK(q.size(2) == 1, "query length must be 1");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(3) == k.size(3), "Q/K/V batch and head dimension must match");
  TORCH_CHECK(q.size(1) % k.size(1) == 0, "query heads must be divisible by KV heads");
  const int64_t group = q.size(1) / k.size(1);
  TORCH_CHECK(group == 1 || group == 4 || group == 8, "supported GQA group sizes are 1, 4 and 8");
  TORCH_CHECK(q.size(3) == 64 || q.size(3) == 128, "head dimension must be 64 or 128");
  if (seqlens.has_value()) {
    const at::Tensor& s = *seqlens;
    TORCH_CHECK(s.device() == q.device(), "seqlens must be on the same CUDA device as Q/K/V");
    TORCH_CHECK(s.scalar_type() == at::kInt, "seqlens dtype must be int32");
    TORCH_CHECK(s.dim() == 1 && s.size(0) == q.size(0) && s.is_contiguous(),
                "seqlens must be a contiguous [batch] tensor");
  }
}

// One workspace per (device, stream), as the Python layer keeps: calls on one
// stream are ordered and every completed call leaves its scheduler header
// zero, so the header is cleared only when a larger problem's header reaches
// past the prefix known to be zero.  A call being captured into a CUDA graph
// gets its own buffer (from the graph's pool) with the header memset captured.
struct StreamWorkspace {
  at::Tensor buffer;
  size_t clean = 0;  // leading bytes known to be zero
};
std::mutex g_mutex;
std::map<std::pair<int, cudaStream_t>, StreamWorkspace> g_workspaces;
constexpr size_t kMaxWorkspaces = 64;

struct Workspace {
  at::Tensor buffer;
  unsigned flags;
};

Workspace workspace_for(const at::Tensor& q, int device, cudaStream_t stream, size_t bytes,
                        size_t header) {
  bytes = bytes < 256 ? 256 : bytes;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  TORCH_CHECK(cudaStreamIsCapturing(stream, &capture) == cudaSuccess, "cudaStreamIsCapturing failed");
  if (capture != cudaStreamCaptureStatusNone)
    return {at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte)), 0u};
  std::lock_guard<std::mutex> lock(g_mutex);
  const auto key = std::make_pair(device, stream);
  auto it = g_workspaces.find(key);
  if (it == g_workspaces.end() || static_cast<size_t>(it->second.buffer.numel()) < bytes) {
    if (it == g_workspaces.end() && g_workspaces.size() >= kMaxWorkspaces)
      g_workspaces.erase(g_workspaces.begin());  // freed stream-ordered by the caching allocator
    StreamWorkspace ws;
    ws.buffer = at::zeros({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    ws.clean = bytes;
    it = g_workspaces.insert_or_assign(key, std::move(ws)).first;
  }
  const unsigned flags = header <= it->second.clean ? ADB_FLAG_HEADER_ZEROED : 0u;
  it->second.clean = header;  // after the call only its own header is known to be zero
  return {it->second.buffer, flags};
}

struct Call {
  int device;
  cudaStream_t stream;
  Workspace ws;
};

Call prepare(const at::Tensor& q, const at::Tensor& k, const c10::optional<at::Tensor>& seqlens) {
  const int device = q.get_device();
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(device).stream();
  size_t total = 0, header = 0;
  check_status(adb_decode_workspace_size(q.size(0), q.size(1), k.size(1), k.size(2), q.size(3),
                                         seqlens.has_value() ? 1 : 0, device, &total, &header));
  return {device, stream, workspace_for(q, device, stream, total, header)};
}

// forward(q, k, v, seqlens=None) -> O [B, Hq, 1, D] BF16.
at::Tensor forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                   const c10::optional<at::Tensor>& seqlens) {
  check_inputs(q, k, v, seqlens);
  const c10::cuda::CUDAGuard guard(q.device());
  Call call = prepare(q, k, seqlens);
  at::Tensor out = at::empty_like(q);
  check_status(adb_decode(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                          seqlens.has_value() ? seqlens->data_ptr<int32_t>() : nullptr, out.data_ptr(),
                          q.size(0), q.size(1), k.size(1), k.size(2), q.size(3), call.ws.buffer.data_ptr(),
                          static_cast<size_t>(call.ws.buffer.numel()), call.ws.flags, call.device, call.stream));
  return out;
}

// forward_partial(q, k, v, seqlens=None) -> (acc FP32 [B, Hq, D], ml FP32 [B, Hq, 2]).
std::tuple<at::Tensor, at::Tensor> forward_partial(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                   const c10::optional<at::Tensor>& seqlens) {
  check_inputs(q, k, v, seqlens);
  const c10::cuda::CUDAGuard guard(q.device());
  Call call = prepare(q, k, seqlens);
  auto f32 = q.options().dtype(at::kFloat);
  at::Tensor acc = at::empty({q.size(0), q.size(1), q.size(3)}, f32);
  at::Tensor ml = at::empty({q.size(0), q.size(1), 2}, f32);
  check_status(adb_decode_partial(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                  seqlens.has_value() ? seqlens->data_ptr<int32_t>() : nullptr,
                                  acc.data_ptr<float>(), ml.data_ptr<float>(), q.size(0), q.size(1), k.size(1),
                                  k.size(2), q.size(3), call.ws.buffer.data_ptr(),
                                  static_cast<size_t>(call.ws.buffer.numel()), call.ws.flags, call.device,
                                  call.stream));
  return {acc, ml};
}

// combine(acc FP32 [R, B, Hq, D], ml FP32 [R, B, Hq, 2]) -> O BF16 [B, Hq, 1, D].
at::Tensor combine(const at::Tensor& acc, const at::Tensor& ml) {
  TORCH_CHECK(acc.is_cuda() && ml.is_cuda(), "partial states must be CUDA tensors");
  TORCH_CHECK(acc.scalar_type() == at::kFloat && ml.scalar_type() == at::kFloat, "partial states must be float32");
  TORCH_CHECK(acc.dim() == 4 && ml.dim() == 4, "acc must be [R, B, Hq, D] and ml [R, B, Hq, 2]");
  TORCH_CHECK(acc.is_contiguous() && ml.is_contiguous(), "partial states must be contiguous");
  TORCH_CHECK(ml.size(0) == acc.size(0) && ml.size(1) == acc.size(1) && ml.size(2) == acc.size(2) && ml.size(3) == 2,
              "ml must have shape [R, B, Hq, 2]");
  const c10::cuda::CUDAGuard guard(acc.device());
  const int device = acc.get_device();
  const int64_t parts = acc.size(0), rows = acc.size(1) * acc.size(2), dim = acc.size(3);
  at::Tensor out = at::empty({acc.size(1), acc.size(2), 1, dim}, acc.options().dtype(at::kBFloat16));
  check_status(adb_combine(acc.data_ptr<float>(), rows * dim, ml.data_ptr<float>(), rows * 2, parts, rows, dim,
                           out.data_ptr(), device, at::cuda::getCurrentCUDAStream(device).stream()));
  return out;
}

// ---- Prompt attention and paged-cache upkeep.  The checks that need no
// device come first, that the tensors are on one comes last.

void check_bf16(const at::Tensor& t, const char* name, int64_t rank) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " dtype must be BF16 (bfloat16)");
  TORCH_CHECK(t.dim() == rank, name, " must have rank ", std::to_string(rank).c_str());
  TORCH_CHECK(!t.requires_grad(), name, ": forward inference only; no backward/grad support");
}

void check_int32(const at::Tensor& t, const char* name, int64_t rank) {
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " dtype must be int32");
  TORCH_CHECK(t.dim() == rank, name, " must have rank ", std::to_string(rank).c_str());
  if (rank == 1) {
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  } else {
    TORCH_CHECK(t.size(0) > 0 && t.size(1) > 0 && t.stride(1) == 1 && (t.size(0) == 1 || t.stride(0) >= t.size(1)),
                name, " must have contiguous, distinct rows");
  }
}

// A packed [tokens, heads, D] tensor: any token and head stride that keeps
// 16-byte vectors aligned (views of a fused projection qualify).
void check_packed(const at::Tensor& t, const char* name) {
  check_bf16(t, name, 3);
  TORCH_CHECK(t.size(2) == 64 || t.size(2) == 128, "head dimension must be 64 or 128");
  TORCH_CHECK(t.size(1) > 0, name, " must have heads");
  TORCH_CHECK(t.stride(2) == 1, name, " must be contiguous in the head dimension");
  TORCH_CHECK((t.size(0) <= 1 || t.stride(0) % 8 == 0) && (t.size(1) <= 1 || t.stride(1) % 8 == 0) &&
                  t.storage_offset() % 8 == 0,
              name, " must start at, and have token and head strides of, a multiple of 8 elements");
  TORCH_CHECK((t.size(0) <= 1 || t.stride(0) > 0) && (t.size(1) <= 1 || t.stride(1) > 0), name,
              " must not be expanded");
}

// Strides as the C ABI takes them (a stride of a dimension of size 1 may be anything).
int64_t token_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2); }
int64_t head_stride(const at::Tensor& t) { return t.size(1) > 1 ? t.stride(1) : t.size(2); }

int64_t row_stride(const at::Tensor& table) { return table.size(0) > 1 ? table.stride(0) : table.size(1); }

struct Pages {
  int64_t blocks, heads, page, dim;
  int layout;
};

Pages check_caches(const at::Tensor& k_cache, const at::Tensor& v_cache, bool nhd) {
  check_bf16(k_cache, "k_cache", 4);
  check_bf16(v_cache, "v_cache", 4);
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "K/V cache shapes must match");
  TORCH_CHECK(k_cache.is_contiguous() && v_cache.is_contiguous(), "K/V caches must be contiguous");
  TORCH_CHECK(k_cache.numel() > 0, "empty caches are unsupported");
  return {k_cache.size(0), k_cache.size(nhd ? 2 : 1), k_cache.size(nhd ? 1 : 2), k_cache.size(3),
          nhd ? ADB_PAGED_NHD : ADB_PAGED_HND};
}

void check_batch(const at::Tensor& t, const char* name, int64_t batch) {
  check_int32(t, name, 1);
  TORCH_CHECK(t.size(0) == batch, name, " must have ", std::to_string(batch).c_str(), " entries");
}

// All on the CUDA device of the first (ValueError, as for Q, K and V elsewhere).
void check_devices(std::initializer_list<std::pair<const char*, const at::Tensor*>> tensors) {
  const at::Tensor* first = tensors.begin()->second;
  for (const auto& t : tensors) {
    TORCH_CHECK_VALUE(t.second->is_cuda(), t.first, " must be a CUDA tensor");
    TORCH_CHECK(t.second->device() == first->device(), t.first, " must be on the same CUDA device as ",
                tensors.begin()->first);
  }
}

// An uninitialised tensor of t's type on its device; past the dispatcher, whose
// share of a short call counts.
at::Tensor empty_for(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, t.device(), c10::nullopt));
}
at::Tensor empty_for(const at::Tensor& t, at::IntArrayRef sizes) { return empty_for(t, sizes, t.scalar_type()); }

// Scratch from the caching allocator (it is given back in the stream's order;
// a captured call's belongs to the graph's pool).
at::Tensor prefill_workspace(const at::Tensor& q, int64_t batch, int64_t kv_heads, int64_t max_keys) {
  size_t bytes = 0;
  check_status(adb_prefill_workspace_size(q.size(0), batch, q.size(1), kv_heads, q.size(2), max_keys, q.get_device(),
                                          &bytes));
  return bytes > 0 ? empty_for(q, {static_cast<int64_t>(bytes)}, at::kByte) : at::Tensor();
}

size_t bytes_of(const at::Tensor& workspace) {
  return workspace.defined() ? static_cast<size_t>(workspace.numel()) : 0;
}
void* data_of(const at::Tensor& workspace) { return workspace.defined() ? workspace.data_ptr() : nullptr; }

at::Tensor prefill(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu_seqlens) {
  check_packed(q, "Q");
  check_packed(k, "K");
  check_packed(v, "V");
  check_int32(cu_seqlens, "cu_seqlens", 1);
  TORCH_CHECK(cu_seqlens.size(0) >= 1, "cu_seqlens must have batch + 1 entries");
  TORCH_CHECK(k.sizes() == v.sizes(), "K/V shape must match");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(2) == k.size(2), "Q/K/V tokens and head dimension must match");
  TORCH_CHECK(q.size(1) % k.size(1) == 0, "query heads must be divisible by KV heads");
  check_devices({{"Q", &q}, {"K", &k}, {"V", &v}, {"cu_seqlens", &cu_seqlens}});
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t batch = cu_seqlens.size(0) - 1;
  if (q.size(0) == 0 || batch == 0) return at::zeros({q.size(0), q.size(1), q.size(2)}, q.options());
  at::Tensor out = empty_for(q, {q.size(0), q.size(1), q.size(2)});
  const int device = q.get_device();
  const at::Tensor ws = prefill_workspace(q, batch, k.size(1), 0);
  check_status(adb_prefill(q.data_ptr(), token_stride(q), head_stride(q), k.data_ptr(), token_stride(k),
                           head_stride(k), v.data_ptr(), token_stride(v), head_stride(v),
                           cu_seqlens.data_ptr<int32_t>(), out.data_ptr(), q.size(0), batch, q.size(1), k.size(1),
                           q.size(2), data_of(ws), bytes_of(ws), device,
                           at::cuda::getCurrentCUDAStream(device).stream()));
  return out;
}

at::Tensor prefill_paged(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                         const at::Tensor& block_table, const at::Tensor& cu_seqlens, const at::Tensor& seqlens,
                         bool nhd) {
  check_packed(q, "Q");
  const Pages pages = check_caches(k_cache, v_cache, nhd);
  check_int32(block_table, "block_table", 2);
  const int64_t batch = block_table.size(0);
  check_batch(cu_seqlens, "cu_seqlens", batch + 1);
  check_batch(seqlens, "seqlens", batch);
  TORCH_CHECK(q.size(2) == pages.dim, "Q and cache head dimension must match");
  TORCH_CHECK(q.size(1) % pages.heads == 0, "query heads must be divisible by KV heads");
  check_devices({{"Q", &q}, {"k_cache", &k_cache}, {"v_cache", &v_cache}, {"block_table", &block_table},
                 {"cu_seqlens", &cu_seqlens}, {"seqlens", &seqlens}});
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = empty_for(q, {q.size(0), q.size(1), q.size(2)});
  if (q.size(0) == 0) return out;
  const int device = q.get_device();
  const at::Tensor ws = prefill_workspace(q, batch, pages.heads, block_table.size(1) * pages.page);
  check_status(adb_prefill_paged(
      q.data_ptr(), token_stride(q), head_stride(q), k_cache.data_ptr(), v_cache.data_ptr(),
      block_table.data_ptr<int32_t>(), row_stride(block_table),
      cu_seqlens.data_ptr<int32_t>(), seqlens.data_ptr<int32_t>(), out.data_ptr(), q.size(0), batch, q.size(1),
      pages.heads, pages.dim, pages.blocks, pages.page, block_table.size(1), pages.layout,
      data_of(ws), bytes_of(ws), device, at::cuda::getCurrentCUDAStream(device).stream()));
  return out;
}

void cache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
                 const at::Tensor& block_table, const at::Tensor& cu_seqlens, const at::Tensor& starts, bool nhd) {
  check_packed(k, "K");
  check_packed(v, "V");
  const Pages pages = check_caches(k_cache, v_cache, nhd);
  TORCH_CHECK(k.sizes() == v.sizes(), "K/V shape must match");
  TORCH_CHECK(k.size(1) == pages.heads && k.size(2) == pages.dim, "K/V heads and head dimension must match the caches");
  check_int32(block_table, "block_table", 2);
  const int64_t batch = block_table.size(0);
  check_batch(cu_seqlens, "cu_seqlens", batch + 1);
  check_batch(starts, "starts", batch);
  check_devices({{"K", &k}, {"V", &v}, {"k_cache", &k_cache}, {"v_cache", &v_cache}, {"block_table", &block_table},
                 {"cu_seqlens", &cu_seqlens}, {"starts", &starts}});
  if (k.size(0) == 0) return;
  const c10::cuda::CUDAGuard guard(k.device());
  const int device = k.get_device();
  check_status(adb_cache_write(
      k.data_ptr(), token_stride(k), head_stride(k), v.data_ptr(), token_stride(v), head_stride(v),
      k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr<int32_t>(),
      row_stride(block_table), cu_seqlens.data_ptr<int32_t>(),
      starts.data_ptr<int32_t>(), k.size(0), batch, pages.heads, pages.dim, pages.blocks, pages.page,
      block_table.size(1), pages.layout, device, at::cuda::getCurrentCUDAStream(device).stream()));
}

void cache_copy_pages(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& src,
                      const at::Tensor& dst) {
  const Pages pages = check_caches(k_cache, v_cache, false);
  check_int32(src, "src", 1);
  check_batch(dst, "dst", src.size(0));
  check_devices({{"k_cache", &k_cache}, {"v_cache", &v_cache}, {"src", &src}, {"dst", &dst}});
  if (src.size(0) == 0) return;
  const c10::cuda::CUDAGuard guard(k_cache.device());
  const int device = k_cache.get_device();
  check_status(adb_cache_copy_pages(k_cache.data_ptr(), v_cache.data_ptr(), src.data_ptr<int32_t>(),
                                    dst.data_ptr<int32_t>(), src.size(0), pages.blocks,
                                    pages.heads * pages.page * pages.dim * 2, device,
                                    at::cuda::getCurrentCUDAStream(device).stream()));
}

void check_book(const at::Tensor& block_table, const at::Tensor& seqlens, const at::Tensor& page_refs) {
  check_int32(block_table, "block_table", 2);
  check_batch(seqlens, "seqlens", block_table.size(0));
  check_int32(page_refs, "page_refs", 1);
  TORCH_CHECK(page_refs.size(0) > 0, "page_refs must have an entry per page");
}

at::Tensor cache_resize(const at::Tensor& block_table, const at::Tensor& seqlens, const at::Tensor& new_lens,
                        const at::Tensor& page_refs, int64_t page_size) {
  check_book(block_table, seqlens, page_refs);
  check_batch(new_lens, "new_lens", block_table.size(0));
  check_devices({{"block_table", &block_table}, {"seqlens", &seqlens}, {"new_lens", &new_lens},
                 {"page_refs", &page_refs}});
  const c10::cuda::CUDAGuard guard(block_table.device());
  const int device = block_table.get_device();
  at::Tensor lens = empty_for(seqlens, {seqlens.size(0)});
  check_status(adb_cache_resize(block_table.data_ptr<int32_t>(), row_stride(block_table), seqlens.data_ptr<int32_t>(),
                                new_lens.data_ptr<int32_t>(), page_refs.data_ptr<int32_t>(), lens.data_ptr<int32_t>(),
                                block_table.size(0), page_refs.size(0), page_size, block_table.size(1), device,
                                at::cuda::getCurrentCUDAStream(device).stream()));
  return lens;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> cache_fork(const at::Tensor& block_table, const at::Tensor& seqlens,
                                                          const at::Tensor& page_refs, const at::Tensor& parents,
                                                          const at::Tensor& children, int64_t page_size) {
  check_book(block_table, seqlens, page_refs);
  check_int32(parents, "parents", 1);
  check_batch(children, "children", parents.size(0));
  check_devices({{"block_table", &block_table}, {"seqlens", &seqlens}, {"page_refs", &page_refs},
                 {"parents", &parents}, {"children", &children}});
  const c10::cuda::CUDAGuard guard(block_table.device());
  const int device = block_table.get_device();
  at::Tensor src = empty_for(parents, {parents.size(0)}), dst = empty_for(parents, {parents.size(0)});
  if (parents.size(0) == 0) return {seqlens.clone(), src, dst};
  at::Tensor lens = empty_for(seqlens, {seqlens.size(0)});
  check_status(adb_cache_fork(block_table.data_ptr<int32_t>(), row_stride(block_table), seqlens.data_ptr<int32_t>(),
                              page_refs.data_ptr<int32_t>(), parents.data_ptr<int32_t>(),
                              children.data_ptr<int32_t>(), parents.size(0), lens.data_ptr<int32_t>(),
                              src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(), block_table.size(0),
                              page_refs.size(0), page_size, block_table.size(1), device,
                              at::cuda::getCurrentCUDAStream(device).stream()));
  return {lens, src, dst};
}

std::tuple<at::Tensor, at::Tensor> cache_compact(const at::Tensor& block_table, const at::Tensor& seqlens,
                                                 const at::Tensor& page_refs, int64_t page_size) {
  check_book(block_table, seqlens, page_refs);
  check_devices({{"block_table", &block_table}, {"seqlens", &seqlens}, {"page_refs", &page_refs}});
  const c10::cuda::CUDAGuard guard(block_table.device());
  const int device = block_table.get_device();
  const int64_t blocks = page_refs.size(0);
  at::Tensor src = empty_for(page_refs, {blocks / 2}), dst = empty_for(page_refs, {blocks / 2});
  at::Tensor remap = empty_for(page_refs, {blocks});
  check_status(adb_cache_compact(block_table.data_ptr<int32_t>(), row_stride(block_table),
                                 seqlens.data_ptr<int32_t>(), page_refs.data_ptr<int32_t>(),
                                 src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(), remap.data_ptr<int32_t>(),
                                 block_table.size(0), blocks, page_size, block_table.size(1), device,
                                 at::cuda::getCurrentCUDAStream(device).stream()));
  return {src, dst};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "BF16 split-K attention decode for B200 (sm_100a): the reference extension's forward(q, k, v)";
  m.def("forward", &forward, "O = softmax(Q K^T / sqrt(D)) V for one query token per sequence",
        pybind11::arg("q"), pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("seqlens") = pybind11::none());
  m.def("forward_partial", &forward_partial, "unnormalised (acc, (m, l)) states of this call's KV",
        pybind11::arg("q"), pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("seqlens") = pybind11::none());
  m.def("combine", &combine, "merge R partial states into the BF16 output", pybind11::arg("acc"),
        pybind11::arg("ml"));
  m.def("prefill", &prefill, "causal attention of packed prompts");
  m.def("prefill_paged", &prefill_paged, "causal attention of new tokens over a paged cache");
  m.def("cache_write", &cache_write, "new tokens' K and V into their pages");
  m.def("cache_copy_pages", &cache_copy_pages, "copies of pages inside both pools");
  m.def("cache_resize", &cache_resize, "pages for new lengths");
  m.def("cache_fork", &cache_fork, "rows that share their parents' pages");
  m.def("cache_compact", &cache_compact, "live pages to the front of the pool");
}
