// prefill_kernels.cuh -- causal attention of whole prompts (packed sequences)
// and of new tokens over a paged K/V cache.
//
// Row (token i of sequence b, head h) stands at position p = c_b + i, where
// c_b = L_b - n_b tokens come before the n_b new ones (0 for packed prompts):
//     o = sum_{j <= p} softmax_j(q . k_j / sqrt(D)) v_j,   h_kv = h / G
// with an FP32 online softmax.  A row that sees no key is zero.
#pragma once

#include "device_primitives.cuh"

namespace adb {

struct PrefillParams {
  const __nv_bfloat16* q;  // [total][q_heads][D], strides in elements
  const __nv_bfloat16* k;  // [total][kv_heads][D], or the pool of pages
  const __nv_bfloat16* v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  __nv_bfloat16* out;      // [total][q_heads][D], contiguous
  const int32_t* cu;       // [batch + 1]
  const int32_t* lens;     // [batch] tokens in the cache, new ones included (paged)
  const int32_t* table;    // paged: [batch][max_blocks]
  int64_t table_stride;
  int total, batch, q_heads, kv_heads, group;
  int paged;               // 0 packed K/V, 1 HND pages, 2 NHD pages
  int max_blocks, num_blocks, page_shift;
  float scale_log2;        // log2(e) / sqrt(D)
};

// One warp per row: the lanes share the head dimension.
template <int D>
__global__ void __launch_bounds__(128) prefill_rows_kernel(const PrefillParams p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  griddep_wait();
  if (row >= static_cast<int64_t>(p.total) * p.q_heads) return;
  const int t = static_cast<int>(row / p.q_heads), h = static_cast<int>(row % p.q_heads), hkv = h / p.group;
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int first = p.cu[lo], last = min(p.cu[lo + 1], p.total);
  int keys = 0;
  if (t >= first && t < last) {
    const int cap = p.paged ? p.max_blocks << p.page_shift : 0;
    const int len = p.paged ? min(max(p.lens[lo], 0), cap) : last - first;
    keys = max(0, len - (last - first) + (t - first) + 1);
  }
  float q[E], acc[E] = {};
  for (int e = 0; e < E; ++e)
    q[e] = __bfloat162float(p.q[t * p.q_token + h * p.q_head + lane * E + e]) * p.scale_log2;
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < keys; ++j) {
    int64_t ka, va;
    if (p.paged) {
      const int page = p.table[lo * p.table_stride + (j >> p.page_shift)];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) {  // counts as zeros
        if (lane == 0) atomicOr(&g_adb_error_flag, kErrCachePage);
        const float top = fmaxf(m, 0.f), keep = m == top ? 1.f : exp2f(m - top);
        m = top;
        l = l * keep + exp2f(-top);
        for (int e = 0; e < E; ++e) acc[e] *= keep;
        continue;
      }
      const int64_t size = int64_t(1) << p.page_shift, slot = j & (size - 1);
      ka = (p.paged == 1 ? (static_cast<int64_t>(page) * p.kv_heads + hkv) * size + slot
                         : (page * size + slot) * p.kv_heads + hkv) * D;
      va = ka;
    } else {
      ka = static_cast<int64_t>(first + j) * p.k_token + hkv * p.k_head;
      va = static_cast<int64_t>(first + j) * p.v_token + hkv * p.v_head;
    }
    float s = 0.f;
    for (int e = 0; e < E; ++e) s += q[e] * __bfloat162float(p.k[ka + lane * E + e]);
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float top = fmaxf(m, s);
    const float keep = m == top ? 1.f : exp2f(m - top), w = exp2f(s - top);
    m = top;
    l = l * keep + w;
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * keep + w * __bfloat162float(p.v[va + lane * E + e]);
  }
  for (int e = 0; e < E; ++e)
    p.out[row * D + lane * E + e] = __float2bfloat16(keys > 0 ? acc[e] / l : 0.f);
}

}  // namespace adb
