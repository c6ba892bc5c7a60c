// prefill_kernels.cuh -- causal attention of whole prompts (packed sequences)
// and of new tokens over a paged K/V cache.
//
// Row (token i of sequence b, head h) stands at position p = c_b + i, where
// c_b = L_b - n_b tokens come before the n_b new ones (0 for packed prompts):
//     o = sum_{j <= p} softmax_j(q . k_j / sqrt(D)) v_j,   h_kv = h / G
// with an FP32 online softmax.  A row that sees no key is zero.
//
// Rows.  The G query heads that share a KV head are packed into the 128 rows
// of a tensor-core tile beside 128 / G consecutive tokens (row = token * G +
// head), so that every K/V tile serves all of them and short chunks still
// fill tiles; any G up to 64 works.  A CTA owns two such tiles of one
// (sequence, KV head) and streams the K/V tiles (128 keys) that they see.
//
// Work.  A unit is a pair of tiles of one (sequence, KV head), or a part of
// its K/V tiles (below).  The grid has a CTA for every unit there can be; a
// running CTA takes over units whose CTA has not started (cluster launch
// control), so that one CTA's loads and first products overlap the end of its
// unit before.  Units that see the most keys come first.
//
// Splits.  In batches of up to 256 sequences, where a sequence's K/V tiles are
// one and a half times an SM's even share of all tiles or more (few rows over a
// long cache), its pairs are cut into parts of about that share.  A part leaves its unnormalised O and
// (maximum, total) in the workspace, and a second kernel joins them, a warp per
// row.  (Joined in the CTA of the part that finishes last, 256 rows of 16 parts
// took 45 us.)
//
// Small pages.  The TMA unit takes about 70 cycles per box, whatever it holds,
// so pages of 8 and 16 tokens come as one box of both 64-column blocks (D 128).
// A page's rows of a block then lie behind its rows of the other, and the rows
// 8 r .. 8 r + 7 of all pages are one operand (pages are its stride): the keys
// of a tile are taken in the order r, page, row (tile_key), in S, P and V alike.
//
// What bounds it: for long prompts the chain S -> softmax -> P V of a tile (3100
// cycles per K/V tile for both tiles, 2048 of them tensor work) and the power
// cap: 8192 tokens, 32/8 heads, D 128 take 415 us (1320 TFLOP/s) in 20 calls, 475
// us in 1000; D 64 345 us.  For a few rows over a long cache the chain of one tile
// (1.6 us) against 1.5 us of HBM time: one token over 131072, group 8, takes 103
// us (5.2 TB/s).  A unit costs about 3 us outside its tile loop.
//
// Pipeline of a CTA (384 threads):
//   warps 0-3, 4-7   softmax of tile 0, 1: one thread per row
//   warp 8           finds the units; TMA loads: Q, then K_0 V_0 K_1 V_1 ...
//                    into a ring that runs on over the units
//   warp 9           issues the tensor-core products
//   warps 10, 11     clear masked V rows of border tiles (below)
// S_i = Q_i K_j^T (FP32) and O_i live in tensor memory; the softmax thread
// reads its row of S_i, writes the weights P_i (BF16) over it, and the product
// O_i += P_i V_j takes P_i from tensor memory.  While one tile's softmax runs
// the tensor cores work on the other tile.
//
// P_i takes the first half of S_i's columns.  Where a unit has one tile only
// (and always with D 64 and pages of 16) the next S's other half is computed as
// soon as the first weights are handed over, and its keys' maximum is found
// while the rest follows.  A product of 64 columns has the shared memory's rate
// (three quarters of the time of 128), so with two tiles, which keep the tensor
// cores busier, S comes at once.  Split / at once: 103 / 109 us for one token
// over 131072, 226 / 243 for 256 rows of 1000, 445 / 427 for 8192 tokens and
// 849 / 808 for 16384 tokens of 16/2 heads (20 calls after a pause; 496 / 475
// and 958 / 913 in 1000).
//
// The weights are rounded to BF16 for the product (half a step is 2^-8 of a
// weight): A and B of a product have one type, and V is BF16.  The total sums
// the unrounded weights; it, the maximum and O are FP32 throughout, parts too.
//
// The running maximum is raised (and O rescaled) only when it grows by more
// than 2^8: until then weights up to 2^8 are exact enough in FP32 sums and in
// BF16's relative rounding, and the factor cancels in O / l.
//
// Masked keys have weight 0, and 0 * NaN is NaN: rows of V behind the sequence
// (recycled pages, the next sequence) are therefore cleared in shared memory,
// and non-finite values of V that only some rows of the tiles may see are
// cleared there and added to those rows at the end.
#pragma once

#include "tcgen05_primitives.cuh"

namespace adb {

constexpr int kPrefillThreads = 384;
constexpr int kTile = 128;  // rows of a Q tile, keys of a K/V tile
// Keys whose weights are handed to the tensor cores before the others are
// computed (32 / 64 / 96: 450 / 438 / 436 us on 8192 tokens, 32/8 heads, D 128,
// and 396 / 368 / 381 us with D 64).
constexpr int kFirstPart = 64;
constexpr float kRescaleLog2 = 8.f;
// K/V tiles of a part, at least (4 / 8: 71 / 63 us for 64 tokens over 16384,
// 61 / 62 us for 8 sequences of up to 16384 with 1 to 5 new tokens).
constexpr int kMinPart = 8;
// Registers: 12 warps x 168 at launch; the loading and issuing warps give theirs to the softmax.
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * 168, "more registers than the block is launched with");

struct PrefillParams {
  const __nv_bfloat16* v;  // [total][kv_heads][D] or the pool of pages (non-finite values only)
  int64_t v_token, v_head;
  __nv_bfloat16* out;      // [total][q_heads][D], contiguous
  const int32_t* cu;       // [batch + 1]
  const int32_t* lens;     // [batch] tokens in the cache, new ones included (paged)
  const int32_t* table;    // paged: [batch][max_blocks]
  int64_t table_stride;
  int total, batch, q_heads, kv_heads, group;
  int tile_tokens;         // tokens of a Q tile: 128 / group
  int head_group;          // KV heads that are worked on at a time
  int group_magic;         // ceil(2^16 / group): row / group = row * magic >> 16 for rows below 128
  int paged;               // 0 packed K/V, 1 HND pages, 2 NHD pages
  int max_blocks, num_blocks, page_shift;
  float scale_log2;        // log2(e) / sqrt(D)
  int sms;
  int max_slots;           // parts that the workspace holds (0: no splits)
  int slot_rows;           // rows of a part: group times the tokens of a pair, or of all sequences
  float* part_o;           // [max_slots][slot_rows][D]
  float2* part_ml;         // [max_slots][slot_rows] maximum (of q . k), total
  struct PrefillJoin* joins;  // [max_slots / 2] pairs cut into parts
  int* join_count;
};

// A pair of tiles whose parts are to be joined.
struct PrefillJoin {
  int row;     // of its first token in out
  int rows;    // of both tiles
  int head;    // KV head
  int slot, parts;
};

template <int D>
struct PrefillCfg {
  static constexpr int kHalves = D / 64;                     // 128-byte column blocks of a row
  static constexpr int kHalfBytes = kTile * 128;             // one column block of a tile
  static constexpr int kTileBytes = kHalves * kHalfBytes;
  static constexpr int kStages = D == 128 ? 4 : 8;           // K and V tiles in flight (5 or 9: no faster)
  static constexpr int kSmemBytes = (2 + kStages) * kTileBytes + 2 * kHalfBytes + 1024;
};

// What a CTA works on.
struct PrefillWork {
  int seq, head;     // sequence, KV head; seq -1: only padding, -2: no more work
  int index;         // of the unit (its share of the padding)
  int row0;          // first row of the sequence in q / out
  int token0;        // first token of tile 0, within the sequence's new ones
  int before;        // keys before the sequence's token 0 (may be negative)
  int keys;          // keys of the sequence
  int valid[2];      // tokens of the tiles
  int first;         // K/V tiles first .. first + steps[i] - 1 are tile i's
  int steps[2];
  int open_keys;     // keys from here on are hidden from some row of the tiles
  int parts, part;   // of the pair's K/V tiles
  int slot;          // of the pair's part 0 in the workspace
  int join;          // its place among the pairs cut into parts
  int pad_head, pad_tail;  // rows before the first / from the end of the last sequence
};

// Key of a tile in column c of S, for pages of 16 tokens that come as one box.
__host__ __device__ constexpr int tile_key16(int c) { return ((c & 63) >> 3) * 16 + (c >> 6) * 8 + (c & 7); }

template <int D>
struct PrefillShared {
  alignas(16) uint4 next;  // cluster launch control's answer
  uint64_t next_full;
  uint64_t work_full[2], work_empty[2];
  uint64_t q_full, q_empty;
  uint64_t kv_full[PrefillCfg<D>::kStages], kv_empty[PrefillCfg<D>::kStages];
  uint64_t s_high[2], s_full[2], p_part[2], p_full[2], o_full[2];
  uint64_t v_turn[PrefillCfg<D>::kStages];   // a border tile of V is on its way
  uint64_t v_clean[PrefillCfg<D>::kStages];  // and cleared
  uint64_t fix_done[2];
  uint32_t tmem;
  int abort;
  int fix[2];        // number of the unit of which a non-finite value of V was cleared
  PrefillWork work[2];
};

__device__ __forceinline__ int clamp_to(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// First row, row count and keys of sequence b, whatever cu and lens hold.
struct Sequence {
  int first, count, keys;
};
__device__ __forceinline__ Sequence load_sequence(const PrefillParams& p, int b) {
  const int from = p.cu[b], to = p.cu[b + 1], len = p.paged ? p.lens[b] : 0;
  const int first = clamp_to(from, 0, p.total), count = clamp_to(to, first, p.total) - first;
  return {first, count, p.paged ? clamp_to(len, 0, p.max_blocks << p.page_shift) : count};
}

// The units of all sequences, held by one warp: lane l has sequences l, l + 32,
// ...  Pair i of a sequence is on level base + i + 1, the keys that it sees in
// units of a pair's tokens, and higher levels come first: with counts F(l) of
// the pairs above a level, a pair is found by bisection and no list is needed.
// Larger batches are walked in their order and nothing is cut, so that one CTA
// per KV head streams a long cache among them: 300 single tokens, one over 131072
// and the others over 500, 64/8 heads, D 128, take 1503 us, 250 take 245.  (300
// prompts, 299 of 100 tokens and then one of 8192: 588 us, 250 of them 578.)
constexpr int kPlanRows = 8;
struct PrefillPlan {
  int pairs[kPlanRows], base[kPlanRows];
  int parts[kPlanRows];            // of each of a sequence's pairs
  int units;                       // parts of all pairs of all sequences
  int joins;                       // pairs cut into parts
  int top;                         // highest level
  int scan_base, scan_before;      // where the walk stands
  Sequence own;                    // sequence `lane`
};

__device__ __forceinline__ bool plan_is_sorted(const PrefillParams& p) { return p.batch <= 32 * kPlanRows; }

__device__ __forceinline__ int pairs_of(const PrefillParams& p, int count) {
  return static_cast<int>(static_cast<unsigned>(count + 2 * p.tile_tokens - 1) / static_cast<unsigned>(2 * p.tile_tokens));
}

__device__ __forceinline__ void make_plan(const PrefillParams& p, PrefillPlan& plan) {
  const int lane = threadIdx.x & 31;
  plan.scan_base = plan.scan_before = plan.joins = 0;
  int units = 0, top = 0;
  float tiles = 0.f;  // K/V tiles of all pairs
  plan.own = {0, 0, 0};
#pragma unroll
  for (int r = 0; r < kPlanRows; ++r) plan.pairs[r] = plan.base[r] = 0, plan.parts[r] = 1;
  if (plan_is_sorted(p)) {
#pragma unroll
    for (int r = 0; r < kPlanRows; ++r) {
      if (32 * r >= p.batch) break;
      const int b = 32 * r + lane;
      if (b < p.batch) {
        const Sequence s = load_sequence(p, b);
        if (r == 0) plan.own = s;
        const int before = max(s.keys - s.count, 0);
        plan.pairs[r] = pairs_of(p, s.count);
        if (before > 0)
          plan.base[r] = static_cast<int>(static_cast<unsigned>(before) / static_cast<unsigned>(2 * p.tile_tokens));
        units += plan.pairs[r];
        top = max(top, plan.base[r] + plan.pairs[r]);
        // for now the tiles of the sequence's last pair, its longest
        plan.parts[r] = (s.keys + kTile - 1) / kTile;
        tiles += 0.5f * plan.pairs[r] * (plan.parts[r] + (before + kTile) / kTile);
      }
    }
    if (p.max_slots > 0) {
      // parts of an SM's even share
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, d);
      // ... or more, until the parts of more than half a share get an SM each (if
      // there are no more pairs than SMs) and there are no more of them than the
      // workspace and the grid have room for
      const bool few = __reduce_add_sync(0xffffffffu, units) * p.kv_heads <= p.sms;
      int share = max(kMinPart, static_cast<int>(fminf(ceilf(__fdividef(tiles * p.kv_heads, p.sms)), 1e8f)));
      for (;; share += share / 8 + 1) {
        int more = 0, large = 0;  // units that the cuts add, those of half a share or more
        units = 0;
#pragma unroll
        for (int r = 0; r < kPlanRows; ++r) {
          if (32 * r >= p.batch) break;
          const int parts = max(1, (2 * plan.parts[r] + share) / (2 * share));
          units += plan.pairs[r] * parts;
          more += plan.pairs[r] * (parts - 1);
          if (2 * plan.parts[r] > share) large += plan.pairs[r] * parts;
        }
        more = __reduce_add_sync(0xffffffffu, more);
        large = __reduce_add_sync(0xffffffffu, large);
        if (more == 0 || (more <= p.sms / p.kv_heads && !(few && large * p.kv_heads > p.sms))) break;
      }
#pragma unroll
      for (int r = 0; r < kPlanRows; ++r) {
        if (32 * r >= p.batch) break;
        plan.parts[r] = max(1, (2 * plan.parts[r] + share) / (2 * share));
        if (plan.parts[r] > 1) {
          plan.joins += plan.pairs[r];
          plan.base[r] /= plan.parts[r];  // the order goes by a part's length
          // (the highest level stays an upper bound)
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < kPlanRows; ++r) plan.parts[r] = 1;
    }
  } else {
    for (int b = lane; b < p.batch; b += 32) units += pairs_of(p, load_sequence(p, b).count);
  }
  plan.units = __reduce_add_sync(0xffffffffu, units);
  plan.top = __reduce_max_sync(0xffffffffu, top);
  plan.joins = __reduce_add_sync(0xffffffffu, plan.joins);
}

// Inclusive prefix of v over the warp.
__device__ __forceinline__ int warp_prefix(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// Sequence, pair and part of the r-th unit of the plan (r < units).
__device__ __forceinline__ void find_pair(const PrefillParams& p, PrefillPlan& plan, int r, PrefillWork& w, int& pair) {
  const int lane = threadIdx.x & 31;
  int& seq = w.seq;
  w.parts = 1;
  w.part = 0;
  if (p.batch == 1) {
    w.parts = __shfl_sync(0xffffffffu, plan.parts[0], 0);
    const int i = w.parts == 1 ? r : r / w.parts;
    seq = 0;
    w.part = r - i * w.parts;
    pair = __shfl_sync(0xffffffffu, plan.pairs[0], 0) - 1 - i;
    return;
  }
  if (plan_is_sorted(p)) {
    // lowest level with at most r pairs above it
    int lo = 0, hi = plan.top, above = 0;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      int n = 0;
#pragma unroll
      for (int s = 0; s < kPlanRows; ++s) {
        if (32 * s >= p.batch) break;
        n += clamp_to(plan.base[s] + plan.pairs[s] - mid, 0, plan.pairs[s]) * plan.parts[s];
      }
      n = __reduce_add_sync(0xffffffffu, n);
      if (n <= r)
        hi = mid, above = n;
      else
        lo = mid;
    }
    int k = r - above;
    seq = pair = 0;
#pragma unroll
    for (int s = 0; s < kPlanRows; ++s) {
      const int here = plan.base[s] < hi && hi <= plan.base[s] + plan.pairs[s] ? plan.parts[s] : 0;
      const int inc = warp_prefix(here);
      const int n = __shfl_sync(0xffffffffu, inc, 31);
      if (k < n) {
        const int l = __ffs(__ballot_sync(0xffffffffu, inc > k)) - 1;
        seq = 32 * s + l;
        pair = hi - __shfl_sync(0xffffffffu, plan.base[s], l) - 1;
        w.parts = __shfl_sync(0xffffffffu, here, l);
        w.part = k - (__shfl_sync(0xffffffffu, inc, l) - w.parts);
        break;
      }
      k -= n;
    }
    return;
  }
  if (r < plan.scan_before) plan.scan_base = plan.scan_before = 0;
  for (;;) {
    const int b = plan.scan_base + lane;
    const int mine = b < p.batch ? pairs_of(p, load_sequence(p, b).count) : 0;
    const int inc = warp_prefix(mine);
    const unsigned hit = __ballot_sync(0xffffffffu, r < plan.scan_before + inc);
    if (hit) {
      const int l = __ffs(hit) - 1;
      seq = plan.scan_base + l;
      const int pairs = __shfl_sync(0xffffffffu, mine, l);
      const int at = r - plan.scan_before - (__shfl_sync(0xffffffffu, inc, l) - pairs);
      pair = pairs - 1 - at;  // the one that sees the most keys first
      return;
    }
    plan.scan_before += __shfl_sync(0xffffffffu, inc, 31);
    plan.scan_base += 32;
    if (plan.scan_base >= p.batch) {  // not reached while r < units
      seq = -1;
      pair = 0;
      return;
    }
  }
}

// Keys that token t of the unit's sequence sees (0 or less: none).
__device__ __forceinline__ int keys_of(const PrefillWork& w, int t) { return w.before + t + 1; }

// The index-th unit.  Heads are the fastest index within a group of heads whose
// K and V stay in L2 together.
__device__ __forceinline__ void find_work(const PrefillParams& p, PrefillPlan& plan, int index, PrefillWork& w) {
  w.index = index;
  w.seq = -1;
  w.first = w.steps[0] = w.steps[1] = w.valid[0] = w.valid[1] = 0;
  w.head = w.row0 = w.token0 = w.before = w.keys = w.open_keys = 0;
  w.parts = 1;
  w.part = w.slot = w.join = 0;
  if (index >= plan.units * p.kv_heads) return;
  // (a group has to fill the GPU several times over: its last units leave SMs idle)
  int heads0 = 0;
  if (p.head_group < p.kv_heads && plan.units * p.head_group >= 4 * p.sms)
    heads0 = index / (plan.units * p.head_group) * p.head_group;
  const int heads = plan.units * p.head_group >= 4 * p.sms ? min(p.head_group, p.kv_heads - heads0) : p.kv_heads;
  const int at = index - heads0 * plan.units, r = static_cast<int>(static_cast<unsigned>(at) / static_cast<unsigned>(heads));
  w.head = heads0 + at - r * heads;
  int pair;
  find_pair(p, plan, r, w, pair);
  if (w.seq < 0) return;
  if (w.parts > 1) {
    // places in the workspace: those of the sequences before, then pair by pair
    int slots = 0, pairs = 0;
#pragma unroll
    for (int s = 0; s < kPlanRows; ++s) {
      if (32 * s + (threadIdx.x & 31) < w.seq && plan.parts[s] > 1) {
        slots += plan.pairs[s] * plan.parts[s];
        pairs += plan.pairs[s];
      }
    }
    slots = __reduce_add_sync(0xffffffffu, slots);
    pairs = __reduce_add_sync(0xffffffffu, pairs);
    w.slot = (slots + pair * w.parts) * p.kv_heads + w.head * w.parts;
    w.join = (pairs + pair) * p.kv_heads + w.head;
  }
  Sequence s;
  if (p.batch <= 32) {
    s.first = __shfl_sync(0xffffffffu, plan.own.first, w.seq);
    s.count = __shfl_sync(0xffffffffu, plan.own.count, w.seq);
    s.keys = __shfl_sync(0xffffffffu, plan.own.keys, w.seq);
  } else {
    s = load_sequence(p, w.seq);
  }
  w.row0 = s.first;
  w.keys = s.keys;
  w.before = s.keys - s.count;
  w.token0 = pair * 2 * p.tile_tokens;
  w.open_keys = max(keys_of(w, w.token0), 0);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = w.token0 + i * p.tile_tokens;
    w.valid[i] = clamp_to(s.count - t, 0, p.tile_tokens);
    const int last = keys_of(w, t + w.valid[i] - 1);
    w.steps[i] = w.valid[i] > 0 && last > 0 ? (last + kTile - 1) / kTile : 0;
  }
  if (w.parts > 1) {
    const int length = (max(w.steps[0], w.steps[1]) + w.parts - 1) / w.parts;
    w.first = w.part * length;
    w.steps[0] = clamp_to(w.steps[0] - w.first, 0, length);
    w.steps[1] = clamp_to(w.steps[1] - w.first, 0, length);
  }
}

// A wait that goes on in any case: when it runs out (mbar_wait) the abort flag
// is set, every later wait ends at once, no more loads are started and nothing
// is written.
__device__ __forceinline__ void wait_or_abort(const uint64_t* bar, uint32_t parity, volatile int* abort) {
  mbar_wait(smem_u32(bar), parity, abort);
  __syncwarp();
}

// Two bf16 values: a bit of either half is set if that value's exponent is all
// ones (infinite or not a number).
__device__ __forceinline__ uint32_t non_finite_bits(uint32_t x) { return ((x & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t x) {
  const uint32_t bad = non_finite_bits(x);
  return x & ~((bad & 0x8000u ? 0xFFFFu : 0u) | (bad & 0x80000000u ? 0xFFFF0000u : 0u));
}

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

// Adds the non-finite values of V[key][d], key in [lo, hi), that were cleared
// for the tile to the row `out` that sees them.
// It is in `out`, or in a part's O (`part`).
__device__ __noinline__ void add_non_finite(const PrefillParams& p, int seq, int head, int row0, int dim, int lo,
                                            int hi, __nv_bfloat16* out, float* part) {
  for (int key = max(lo, 0); key < hi; ++key) {
    int64_t at;
    if (p.paged) {
      const int page = p.table[seq * p.table_stride + (key >> p.page_shift)];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) continue;
      const int64_t size = int64_t(1) << p.page_shift, slot = key & (size - 1);
      at = (p.paged == 1 ? (static_cast<int64_t>(page) * p.kv_heads + head) * size + slot
                         : (page * size + slot) * p.kv_heads + head) * dim;
    } else {
      at = static_cast<int64_t>(row0 + key) * p.v_token + head * p.v_head;
    }
    for (int d = 0; d < dim; ++d) {
      const float x = __bfloat162float(p.v[at + d]);
      if (fabsf(x) <= 3.4e38f) continue;
      if (part != nullptr)
        part[d] += x;
      else
        out[d] = __float2bfloat16(__bfloat162float(out[d]) + x);
    }
  }
}

// kPair: pages come as one box of both column blocks (small pages, D 128).
template <int D, bool kPair>
__global__ void __launch_bounds__(kPrefillThreads, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                   const __grid_constant__ CUtensorMap v_map, const __grid_constant__ PrefillParams p) {
  using C = PrefillCfg<D>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t raw[];
  __shared__ PrefillShared<D> sh;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t tiles = (smem_u32(raw) + 1023u) & ~1023u;  // Q_0 Q_1, then the K/V ring
  const uint32_t ring = tiles + 2 * C::kTileBytes;
  const uint32_t staging = ring + S * C::kTileBytes;  // 64 columns of each output tile
  volatile int* abort = &sh.abort;

  if (tid == 0) {
    const auto init = [](uint64_t& bar, int count) { mbar_init(smem_u32(&bar), count); };
    init(sh.next_full, 1);
    init(sh.q_full, 1);
    init(sh.q_empty, 1);
    for (int s = 0; s < S; ++s) {
      init(sh.kv_full[s], 1);
      init(sh.kv_empty[s], 1);
      init(sh.v_turn[s], 1);
      init(sh.v_clean[s], 2);
    }
    for (int i = 0; i < 2; ++i) {
      init(sh.work_full[i], 1);
      init(sh.work_empty[i], 11);
      init(sh.s_high[i], 1);
      init(sh.s_full[i], 1);
      init(sh.p_part[i], 4);
      init(sh.p_full[i], 4);
      init(sh.o_full[i], 1);
      init(sh.fix_done[i], 2);
    }
    sh.abort = 0;
    sh.fix[0] = sh.fix[1] = 0;
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(smem_u32(&sh.tmem), 512);
  if (warp == 8 && lane == 0) {
    prefetch_tensormap(&q_map);
    prefetch_tensormap(&k_map);
    prefetch_tensormap(&v_map);
  }
  tcgen05_before_sync();
  __syncthreads();
  tcgen05_after_sync();
  const uint32_t tmem = sh.tmem;
  griddep_wait();

  // Whether there is a unit of turn n (0, 1, ...), in sh.work[n & 1] until
  // work_done(n); for every warp but the loading one.
  const auto next_work = [&](int n) {
    wait_or_abort(&sh.work_full[n & 1], (n >> 1) & 1, abort);
    return !__any_sync(0xffffffffu, *abort != 0 || sh.work[n & 1].seq == -2);
  };
  const auto work_done = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh.work_empty[n & 1]));
  };

  if (warp >= 8) {
    regs_dec<kOtherRegs>();
    if (warp == 8) {
      // ------------------------------------------------------------ loads
      const int pad_tail = clamp_to(p.cu[p.batch], 0, p.total), pad_head = clamp_to(p.cu[0], 0, p.total);
      PrefillPlan plan;
      make_plan(p, plan);
      const bool pads = pad_tail < p.total || pad_head > 0;
      const int boxes = p.paged ? max(1, kTile >> p.page_shift) : 1;
      const int box_rows = kTile / boxes;
      // Page of the box-th box of a sequence; -1 (reads as zeros) if it has none there.
      const auto page_of = [&](const PrefillWork& w, int box) {
        const int key = box * box_rows;
        if (!p.paged || w.seq < 0 || key >= w.keys) return -1;
        const int page = p.table[w.seq * p.table_stride + (key >> p.page_shift)];
        if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks)) return page;
        atomicOr(&g_adb_error_flag, kErrCachePage);
        return -1;
      };
      int stage = 0, phase = 0;    // ring position of the next tile
      int loaded = 0, q_loads = 0;  // tiles, Q pairs so far
      int turn = 0;                // units handed to the other warps
      int index = blockIdx.x;
      bool go = true;
      for (int asked = 0; go; ++asked) {
        if (p.max_slots > 0 && index == 0 && lane == 0) *p.join_count = plan.joins * p.kv_heads;
        PrefillWork w;
        find_work(p, plan, index, w);
        w.pad_head = pad_head;
        w.pad_tail = pad_tail;
        if (w.seq >= 0 || pads) {
          if (turn >= 2) wait_or_abort(&sh.work_empty[turn & 1], ((turn >> 1) - 1) & 1, abort);
          if (lane == 0) {
            sh.work[turn & 1] = w;
            mbar_arrive(smem_u32(&sh.work_full[turn & 1]));
          }
          __syncwarp();
          ++turn;
        }
        const int steps = max(w.steps[0], w.steps[1]);
        if (steps > 0) {
          if (q_loads > 0) wait_or_abort(&sh.q_empty, (q_loads - 1) & 1, abort);
          ++q_loads;
          if (__any_sync(0xffffffffu, *abort)) break;
          if (lane == 0) {
            const uint32_t bar = smem_u32(&sh.q_full);
            const int n = (w.steps[0] > 0) + (w.steps[1] > 0);
            mbar_arrive_expect_tx(bar, n * C::kHalves * p.tile_tokens * p.group * 128);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              for (int h = 0; h < C::kHalves && w.steps[i] > 0; ++h)
                tma_load_tile_3d(tiles + i * C::kTileBytes + h * C::kHalfBytes, &q_map, h * 64, w.head * p.group,
                                 w.row0 + w.token0 + i * p.tile_tokens, bar);
          }
          __syncwarp();
        }
        // page numbers of 32 / boxes tiles in the lanes, and those of the next ones on their way
        const int ahead = 32 / boxes;
        int pages = page_of(w, w.first * boxes + lane), next_pages = page_of(w, (w.first + ahead) * boxes + lane);
        int tiles_left = ahead;
        // The next unit is asked for late: one taken over at the start would wait for
        // the end of a long one while other CTAs run out of work.
        if (steps < 2 && lane == 0) ask_next(smem_u32(&sh.next), smem_u32(&sh.next_full));
        for (int t = 0; t < 2 * steps; ++t) {
          if (t == 2 * steps - 4 && lane == 0) ask_next(smem_u32(&sh.next), smem_u32(&sh.next_full));
          if (loaded >= S) {
            wait_or_abort(&sh.kv_empty[stage], phase ^ 1, abort);
            if (__any_sync(0xffffffffu, *abort)) break;
          }
          const int tile = w.first + (t >> 1);
          const uint32_t bar = smem_u32(&sh.kv_full[stage]);
          const CUtensorMap* map = (t & 1) ? &v_map : &k_map;
          if (lane == 0) {
            mbar_arrive_expect_tx(bar, C::kTileBytes);
            if ((t & 1) && tile >= w.open_keys / kTile) mbar_arrive(smem_u32(&sh.v_turn[stage]));
          }
          __syncwarp();
          const int page = __shfl_sync(0xffffffffu, pages, (ahead - tiles_left) * boxes + lane % boxes);
          if (lane < boxes) {
            const int key = tile * kTile + lane * box_rows;
            const uint32_t dst = ring + stage * C::kTileBytes;
            const int slot = key & ((1 << p.page_shift) - 1);
            if (kPair) {
              tma_load_tile_5d(dst + lane * box_rows * C::kHalves * 128, map, 0, slot, 0, w.head, page, bar);
            } else {
#pragma unroll
              for (int h = 0; h < C::kHalves; ++h) {
                const uint32_t at = dst + h * C::kHalfBytes + lane * box_rows * 128;
                if (p.paged)
                  tma_load_tile_5d(at, map, 0, slot, h, w.head, page, bar);
                else
                  tma_load_tile_3d(at, map, h * 64, w.head, w.row0 + key, bar);
              }
            }
          }
          if ((t & 1) && --tiles_left == 0) {
            tiles_left = ahead;
            pages = next_pages;
            next_pages = page_of(w, (tile + 1 + ahead) * boxes + lane);
          }
          __syncwarp();
          ++loaded;
          if (++stage == S) stage = 0, phase ^= 1;
        }
        wait_or_abort(&sh.next_full, asked & 1, abort);
        if (__any_sync(0xffffffffu, *abort)) break;
        go = answer_next(smem_u32(&sh.next), index);
        __syncwarp();
      }
      if (turn >= 2) wait_or_abort(&sh.work_empty[turn & 1], ((turn >> 1) - 1) & 1, abort);
      if (lane == 0) {
        sh.work[turn & 1].seq = -2;
        mbar_arrive(smem_u32(&sh.work_full[turn & 1]));
      }
      __syncwarp();
      // every arrival on this CTA's barriers has to come before it is gone
      for (int s = 0; s < S && s < loaded; ++s) {
        if (stage == 0) stage = S, phase ^= 1;
        --stage;
        wait_or_abort(&sh.kv_empty[stage], phase, abort);
      }
      if (q_loads > 0) wait_or_abort(&sh.q_empty, (q_loads - 1) & 1, abort);
    } else if (warp == 9) {
      // ------------------------------------------------------------ products
      // The whole warp runs the loop, so that the compiler sees uniform values
      // (descriptors in uniform registers); one lane issues.  With the loop in
      // one lane's branch an MMA took 65 cycles to issue, and the issue was
      // what bounded the kernel (567 us for 8192 tokens, 32/8 heads, D 128).
      constexpr uint64_t k_major = smem_desc_base(16, 1024);
      const bool pair16 = kPair && p.page_shift == 4;
      const uint32_t page_bytes = 256u << p.page_shift;  // of both column blocks
      const uint64_t k_ring = kPair ? smem_desc_base(16, page_bytes) : k_major;
      const uint64_t v_ring = kPair ? smem_desc_base(page_bytes / 2, page_bytes) : smem_desc_base(C::kHalfBytes, 1024);
      const uint32_t k_half = (kPair ? page_bytes / 2 : C::kHalfBytes) >> 4;
      constexpr uint32_t qk_idesc = mma_idesc(kTile, kTile, false), half_idesc = mma_idesc(kTile, kTile / 2, false);
      constexpr uint32_t pv_idesc = mma_idesc(kTile, D, true);
      // from a tile's first 64 columns of S to its others: the second 8 rows of all pages, half of the pages, 64 keys
      const uint32_t high = (pair16 ? 1024 : kPair ? (kTile / 2) * 256 : (kTile / 2) * 128) >> 4;
      const auto qk_columns = [&](int i, int stage, int half, uint32_t idesc) {
        const uint64_t a = smem_desc(k_major, tiles + i * C::kTileBytes);
        const uint64_t b = smem_desc(k_ring, ring + stage * C::kTileBytes) + (half ? high : 0);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ss(tmem + i * kTile + half * (kTile / 2), a + ((k >> 2) * (C::kHalfBytes >> 4) + (k & 3) * 2),
                 b + ((k >> 2) * k_half + (k & 3) * 2), idesc, k > 0);
      };
      const auto qk_high = [&](int i, int stage) {
        if (elect_one()) {
          qk_columns(i, stage, 1, half_idesc);
          mma_commit(smem_u32(&sh.s_high[i]));
        }
        __syncwarp();
      };
      // the first columns where qk_high has done the others, else all
      const auto qk_rest = [&](int i, int stage, bool split) {
        if (elect_one()) {
          if (pair16 && !split) qk_columns(i, stage, 1, half_idesc);
          qk_columns(i, stage, 0, split || pair16 ? half_idesc : qk_idesc);
          if (!split) mma_commit(smem_u32(&sh.s_high[i]));
          mma_commit(smem_u32(&sh.s_full[i]));
        }
        __syncwarp();
      };
      const auto pv = [&](int i, int stage, int first, int last, bool accumulate) {
        const uint64_t v = smem_desc(v_ring, ring + stage * C::kTileBytes);
        // from one 16 keys to the next: two pages of 8 rows, or half of all pages' rows and then the other
        const uint32_t step = (kPair ? 2 * page_bytes : 2048) >> 4;
        if (elect_one()) {
#pragma unroll
          for (int k = first; k < last; ++k)
            mma_ts(tmem + 2 * kTile + i * kTile, tmem + i * kTile + k * 8,
                   v + (pair16 ? (k & 3) * step + (k >> 2) * (1024 >> 4) : k * step), pv_idesc, accumulate || k > 0);
        }
        __syncwarp();
      };
      const auto commit = [&](uint64_t* bar) {
        if (elect_one()) mma_commit(smem_u32(bar));
        __syncwarp();
      };
      int stage = 0, phase = 0, q_phase = 0, p_phase0 = 0, p_phase1 = 0;
      uint32_t clean_phases = 0;  // bit s: parity of v_clean[s]
      const auto advance = [&] {
        if (++stage == S) stage = 0, phase ^= 1;
      };
      for (int n = 0;; ++n) {
        if (!next_work(n)) break;
        const int steps0 = sh.work[n & 1].steps[0], steps1 = sh.work[n & 1].steps[1], steps = max(steps0, steps1);
        if (steps > 0) {
          const int first_open = sh.work[n & 1].open_keys / kTile - sh.work[n & 1].first;
          const bool split = D == 64 || pair16 || steps0 == 0 || steps1 == 0;
          wait_or_abort(&sh.q_full, q_phase, abort);
          q_phase ^= 1;
          wait_or_abort(&sh.kv_full[stage], phase, abort);
          tcgen05_after_sync();
#pragma unroll 1  // less code: with both calls inlined 4 x 2048 tokens took 170 us, 165 so
          for (int i = 0; i < 2; ++i)
            if ((i ? steps1 : steps0) > 0) qk_rest(i, stage, false);
          commit(&sh.kv_empty[stage]);
          if (steps == 1) commit(&sh.q_empty);
          advance();
          for (int j = 0; j < steps; ++j) {
            const int v_stage = stage;
            wait_or_abort(&sh.kv_full[stage], phase, abort);
            if (j >= first_open) {
              wait_or_abort(&sh.v_clean[stage], (clean_phases >> stage) & 1, abort);
              clean_phases ^= 1u << stage;
            }
            advance();
            const int k_stage = stage;
            if (j + 1 < steps) {
              wait_or_abort(&sh.kv_full[stage], phase, abort);
              advance();
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int mine = i ? steps1 : steps0;
              if (j >= mine) continue;
              int& p_phase = i ? p_phase1 : p_phase0;
              wait_or_abort(&sh.p_part[i], p_phase, abort);
              tcgen05_after_sync();
              if (split && j + 1 < mine) qk_high(i, k_stage);
              pv(i, v_stage, 0, kFirstPart / 16, j > 0);
              wait_or_abort(&sh.p_full[i], p_phase, abort);
              tcgen05_after_sync();
              p_phase ^= 1;
              pv(i, v_stage, kFirstPart / 16, kTile / 16, true);
              if (j + 1 < mine)
                qk_rest(i, k_stage, split);
              else
                commit(&sh.o_full[i]);
            }
            commit(&sh.kv_empty[v_stage]);
            if (j + 1 < steps) commit(&sh.kv_empty[k_stage]);
            if (j + 2 == steps) commit(&sh.q_empty);
          }
        }
        work_done(n);
      }
    } else {
      // ------------------------------------------------------------ masked V
      // Warps 10 and 11 take every other 128 vectors of 16 bytes.
      uint32_t turn_phases = 0;
      int stage = 0, phase = 0;
      for (int n = 0;; ++n) {
        if (!next_work(n)) break;
        const int steps = max(sh.work[n & 1].steps[0], sh.work[n & 1].steps[1]);
        const int first_tile = sh.work[n & 1].first, open_keys = sh.work[n & 1].open_keys, keys = sh.work[n & 1].keys;
        bool fix = false;
        for (int j = 0; j < steps; ++j) {
          const int tile = first_tile + j;
          // past K to V
          if (++stage == S) stage = 0, phase ^= 1;
          if (tile >= open_keys / kTile) {
            // the loads' word that the stage has come to this tile, whose parity then is unmistakable
            wait_or_abort(&sh.v_turn[stage], (turn_phases >> stage) & 1, abort);
            turn_phases ^= 1u << stage;
            wait_or_abort(&sh.kv_full[stage], phase, abort);
            const int first = 8 * max(open_keys - tile * kTile, 0);           // first vector that some row may not see
            const int behind = 8 * clamp_to(keys - tile * kTile, 0, kTile);  // first vector behind the sequence
            for (int h = 0; h < C::kHalves; ++h) {
              const uint32_t tile_at = ring + stage * C::kTileBytes;
              const auto vector_at = [&](int x) {  // x-th vector of the column block, 8 per key
                if (!kPair) return tile_at + h * C::kHalfBytes + x * 16;
                const int shift = p.page_shift + 3;
                return tile_at + (((x >> shift) * C::kHalves + h) << (shift + 4)) + (x & ((1 << shift) - 1)) * 16;
              };
              for (int x0 = (warp - 10) * 128 + lane; x0 < kTile * 8; x0 += 256) {
                uint4 v[4];
                uint32_t bad = 0;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                  const int x = x0 + 32 * u;
                  v[u] = make_uint4(0, 0, 0, 0);
                  if (x >= first && x < behind) v[u] = ld_shared_v4(vector_at(x));
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                  bad |= non_finite_bits(v[u].x) | non_finite_bits(v[u].y) | non_finite_bits(v[u].z) |
                         non_finite_bits(v[u].w);
                if (bad != 0) {
                  fix = true;
#pragma unroll
                  for (int u = 0; u < 4; ++u) {
                    const int x = x0 + 32 * u;
                    if (x >= first && x < behind)
                      st_shared_v4(vector_at(x), make_uint4(finite_or_zero(v[u].x), finite_or_zero(v[u].y),
                                                            finite_or_zero(v[u].z), finite_or_zero(v[u].w)));
                  }
                }
                if (x0 + 96 >= behind) {
#pragma unroll
                  for (int u = 0; u < 4; ++u)
                    if (x0 + 32 * u >= behind) st_shared_v4(vector_at(x0 + 32 * u), make_uint4(0, 0, 0, 0));
                }
              }
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.v_clean[stage]));
          }
          if (++stage == S) stage = 0, phase ^= 1;
        }
        if (fix) *reinterpret_cast<volatile int*>(&sh.fix[n & 1]) = n + 1;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.fix_done[n & 1]));
        work_done(n);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    regs_inc<kSoftmaxRegs>();
    const int i = warp >> 2;
    const int row = tid & (kTile - 1);
    const int token = row * p.group_magic >> 16;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + i * kTile + lanes, o_at = tmem + 2 * kTile + i * kTile + lanes;
    const float scale = p.scale_log2;
    int s_phase = 0, o_phase = 0;
    for (int n = 0;; ++n) {
      if (!next_work(n)) break;
      const PrefillWork& w = sh.work[n & 1];
      if (w.pad_tail < p.total || w.pad_head > 0) {
        const int64_t vecs = static_cast<int64_t>(p.q_heads) * (D / 8);
        uint4* o = reinterpret_cast<uint4*>(p.out);
        const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
        const int64_t at = static_cast<int64_t>(w.index) * 256 + tid;
        for (int64_t x = w.pad_tail * vecs + at; x < p.total * vecs; x += step) o[x] = make_uint4(0, 0, 0, 0);
        for (int64_t x = at; x < w.pad_head * vecs; x += step) o[x] = make_uint4(0, 0, 0, 0);
      }
      const int steps = i ? w.steps[1] : w.steps[0], valid = i ? w.valid[1] : w.valid[0];
      const bool live = token < valid;
      // keys that the row sees, and that every row of the tile sees, from the unit's first on
      const int all_see = keys_of(w, w.token0 + i * p.tile_tokens) - w.first * kTile;
      const int sees = live ? all_see + token : 0;
      float top = -INFINITY, total = 0.f;
      for (int j = 0; j < steps; ++j) {
        float s[kTile];
        float m0 = -INFINITY, m1 = m0, m2 = m0, m3 = m0;
#pragma unroll
        for (int c0 = kTile / 2; c0 >= 0; c0 -= kTile / 2) {
          wait_or_abort(c0 > 0 ? &sh.s_high[i] : &sh.s_full[i], s_phase, abort);
          tcgen05_after_sync();
          tmem_ld32(s_at + c0, s + c0);
          tmem_ld32(s_at + c0 + 32, s + c0 + 32);
          tmem_wait_ld();
          if ((j + 1) * kTile > all_see) {
            const int limit = sees - j * kTile;
            if (kPair && p.page_shift == 4) {
#pragma unroll
              for (int c = c0; c < c0 + kTile / 2; ++c) s[c] = tile_key16(c) < limit ? s[c] : -INFINITY;
            } else {
#pragma unroll
              for (int c = c0; c < c0 + kTile / 2; ++c) s[c] = c < limit ? s[c] : -INFINITY;
            }
          }
#pragma unroll
          for (int c = c0; c < c0 + kTile / 2; c += 8) {
            m0 = max3(m0, s[c], s[c + 1]);
            m1 = max3(m1, s[c + 2], s[c + 3]);
            m2 = max3(m2, s[c + 4], s[c + 5]);
            m3 = max3(m3, s[c + 6], s[c + 7]);
          }
        }
        s_phase ^= 1;
        const float high = fmaxf(max3(m0, m1, m2), m3);
        if (j == 0) {
          top = high;
        } else if (__any_sync(0xffffffffu, live && (high - top) * scale > kRescaleLog2)) {
          // O_i holds the sum up to tile j - 1: S_i was issued after that product.  Rows outside the
          // sequence have no say: the result would depend on what lies there.
          const float next = fmaxf(top, high);
          const float keep = next == top ? 1.f : fast_exp2((top - next) * scale);
          top = next;
          total *= keep;
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {  // few registers: S is still in hand
            uint32_t o[16];
            tmem_ld16(o_at + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tmem_st16(o_at + c, o);
          }
        }
        const float shift = top == -INFINITY ? 0.f : -top * scale;
        const uint64_t scale2 = pack2(scale, scale), shift2 = pack2(shift, shift);
        uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
        for (int c = 0; c < kTile; c += 32) {
          uint32_t w16[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float a, b;
            unpack2(fma2(pack2(s[c + 2 * e], s[c + 2 * e + 1]), scale2, shift2), a, b);
            a = fast_exp2(a);
            b = fast_exp2(b);
            if (e & 1)
              sum1 = add2(sum1, pack2(a, b));
            else
              sum0 = add2(sum0, pack2(a, b));
            w16[e] = pack_bf16x2(a, b);
          }
          tmem_st16(s_at + c / 2, w16);
          if (c + 32 == kFirstPart) {
            tmem_wait_st();
            tcgen05_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.p_part[i]));
          }
        }
        tmem_wait_st();
        tcgen05_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[i]));
        float a, b;
        unpack2(add2(sum0, sum1), a, b);
        total += a + b;
      }
      wait_or_abort(&sh.fix_done[n & 1], (n >> 1) & 1, abort);
      if (steps > 0) {
        wait_or_abort(&sh.o_full[i], o_phase, abort);
        o_phase ^= 1;
        tcgen05_after_sync();
      }
      if (__any_sync(0xffffffffu, *abort)) break;
      // A warp's 32 rows go through shared memory, 64 columns at a time, so that a
      // store covers whole lines (16 bytes of 32 rows each took 2.5 us per unit).
      const float inv = total == 0.f ? 0.f : 1.f / total;
      __nv_bfloat16* out = p.out + (static_cast<int64_t>(w.row0 + w.token0 + i * p.tile_tokens) * p.q_heads +
                                    w.head * p.group) * D;
      const int gap = (p.q_heads - p.group) * D;  // between the rows of two tokens (a tile's offsets fit 32 bits)
      const int rows = valid * p.group;
      const uint32_t mine = staging + i * C::kHalfBytes + (warp & 3) * 4096;
      if (w.parts > 1) {
        const int64_t first_row = static_cast<int64_t>(w.slot + w.part) * p.slot_rows + i * p.tile_tokens * p.group;
        if ((warp & 3) * 32 < rows) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float o[32] = {};
            if (steps > 0) {
              tmem_ld32(o_at + c, o);
              tmem_wait_ld();
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
              st_shared_v4(mine + lane * 128 + (e ^ (lane & 7)) * 16,
                           make_uint4(__float_as_uint(o[4 * e]), __float_as_uint(o[4 * e + 1]),
                                      __float_as_uint(o[4 * e + 2]), __float_as_uint(o[4 * e + 3])));
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int l = 4 * k + (lane >> 3), x = lane & 7, r = (warp & 3) * 32 + l;
              const uint4 v = ld_shared_v4(mine + l * 128 + (x ^ (l & 7)) * 16);
              if (r < rows) *reinterpret_cast<uint4*>(p.part_o + (first_row + r) * D + c + x * 4) = v;
            }
            __syncwarp();
          }
          if (live) {
            p.part_ml[first_row + row] = make_float2(top, total);
            // Only those of the part's own keys: the join multiplies by 0 what a row has
            // of a part that it sees nothing of, and 0 * infinity is NaN.
            if (*reinterpret_cast<volatile int*>(&sh.fix[n & 1]) == n + 1)
              add_non_finite(p, w.seq, w.head, w.row0, D, max(w.open_keys, w.first * kTile),
                             w.first * kTile + min(sees, steps * kTile), out, p.part_o + (first_row + row) * D);
          }
        }
        if (tid == 0 && w.part == 0)
          p.joins[w.join] = {w.row0 + w.token0, (w.valid[0] + w.valid[1]) * p.group, w.head, w.slot, w.parts};
      } else if ((warp & 3) * 32 < rows) {
        int offset[8];  // of this lane's 16 bytes in eight stores, 4 rows each
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = (warp & 3) * 32 + 4 * k + (lane >> 3);
          offset[k] = r < rows ? (r * p.group_magic >> 16) * gap + r * D + (lane & 7) * 8 : -1;
        }
#pragma unroll 1
        for (int c = 0; c < D; c += 64) {
#pragma unroll
          for (int h = 0; h < 64; h += 32) {
            float o[32];
            if (steps > 0) {
              tmem_ld32(o_at + c + h, o);
              tmem_wait_ld();
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = inv == 0.f ? 0.f : o[e] * inv;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              st_shared_v4(mine + lane * 128 + (((h >> 3) + e) ^ (lane & 7)) * 16,
                           make_uint4(pack_bf16x2(o[8 * e], o[8 * e + 1]), pack_bf16x2(o[8 * e + 2], o[8 * e + 3]),
                                      pack_bf16x2(o[8 * e + 4], o[8 * e + 5]), pack_bf16x2(o[8 * e + 6], o[8 * e + 7])));
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int l = 4 * k + (lane >> 3), x = lane & 7;
            const uint4 v = ld_shared_v4(mine + l * 128 + (x ^ (l & 7)) * 16);
            if (offset[k] >= 0) *reinterpret_cast<uint4*>(out + offset[k] + c) = v;
          }
          __syncwarp();
        }
        if (live && *reinterpret_cast<volatile int*>(&sh.fix[n & 1]) == n + 1)
          add_non_finite(p, w.seq, w.head, w.row0, D, w.open_keys, w.first * kTile + sees,
                         out + token * gap + row * D, nullptr);
      }
      tcgen05_before_sync();
      work_done(n);
    }
  }
  __syncthreads();
  griddep_launch_dependents();
  if (*abort != 0) {
    // after a wait that ran out: parts are missing, so none are joined (the count
    // was written at the start, long ago); and what was still in flight
    if (tid == 0 && p.max_slots > 0) *p.join_count = 0;
    __nanosleep(1000000);
  }
  if (warp == 9) {
    tcgen05_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts, a warp per row:
//   M = max m, o = sum e^(m - M) O / sum e^(m - M) l.
// Bound by latency (a few KB per row), so a row's loads go out together, the
// first parts of O beside the maxima. Two blocks per SM: 5.4 us for
// 1 to 5 new tokens of 8 sequences (4 query heads per key head), 8.9 us for
// up to 1021 of 4 (8 query heads); a load per part in turn with every row of a
// slot dealt out one by one took 7.0 and 11.5, four blocks per SM 6.2 and 8.7.
constexpr int kJoinThreads = 256;
constexpr int kJoinAhead = 8;  // loads of O in flight per lane
template <int D>
__global__ void __launch_bounds__(kJoinThreads) prefill_join_kernel(const __grid_constant__ PrefillParams p) {
  constexpr int kLanes = D / 4;              // of a row of O, 16 bytes each
  constexpr int kAtOnce = 32 / kLanes;       // parts that a load of the warp covers
  constexpr int kChunk = kJoinAhead * kAtOnce;
  constexpr int kWarps = kJoinThreads / 32;
  const int lane = threadIdx.x & 31;
  griddep_wait();
  const int count = __ldcg(p.join_count);
  if (count == 0) return;
  // Blocks to an entry: all of them at once where the entries are few, else
  // four rounds, so that entries of many rows are shared out evenly.
  const int grid = gridDim.x;
  const int share = count <= grid / 4 ? grid / count : max(4 * grid / count, 1);
  for (int x = blockIdx.x; x < count * share; x += grid) {
    const int* words = reinterpret_cast<const int*>(p.joins + x / share);
    const PrefillJoin j = {__ldcg(words), __ldcg(words + 1), __ldcg(words + 2), __ldcg(words + 3), __ldcg(words + 4)};
    for (int r = x % share * kWarps + (threadIdx.x >> 5); r < j.rows; r += share * kWarps) {
      const float2* ml = p.part_ml + static_cast<int64_t>(j.slot) * p.slot_rows + r;
      const float* o = p.part_o + (static_cast<int64_t>(j.slot) * p.slot_rows + r) * D + (lane % kLanes) * 4;
      const auto state = [&](int k) {
        return k < j.parts ? __ldcg(&ml[static_cast<int64_t>(k) * p.slot_rows]) : make_float2(-INFINITY, 0.f);
      };
      float4 a[kJoinAhead];
      const auto load = [&](int k0) {
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
          const int k = k0 + u * kAtOnce + lane / kLanes;
          a[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (k < j.parts) a[u] = __ldcg(reinterpret_cast<const float4*>(o + static_cast<int64_t>(k) * p.slot_rows * D));
        }
      };
      float2 mine = state(lane);
      load(0);
      float top = mine.x;
      for (int k = 32 + lane; k < j.parts; k += 32) top = fmaxf(top, state(k).x);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      float total = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int b = 0; b < j.parts; b += 32) {
        if (b > 0) mine = state(b + lane);
        const float f = mine.x == top ? 1.f : fast_exp2((mine.x - top) * p.scale_log2);
        if (b + lane < j.parts) total += f * mine.y;
        for (int k0 = b; k0 < min(b + 32, j.parts); k0 += kChunk) {
          if (k0 > 0) load(k0);
#pragma unroll
          for (int u = 0; u < kJoinAhead; ++u) {
            const int k = k0 + u * kAtOnce + lane / kLanes;
            const float g = __shfl_sync(0xffffffffu, f, k & 31);
            if (k < j.parts) {
              sum.x += g * a[u].x;
              sum.y += g * a[u].y;
              sum.z += g * a[u].z;
              sum.w += g * a[u].w;
            }
          }
        }
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
#pragma unroll
      for (int d = 16; d >= kLanes; d >>= 1) {
        sum.x += __shfl_xor_sync(0xffffffffu, sum.x, d);
        sum.y += __shfl_xor_sync(0xffffffffu, sum.y, d);
        sum.z += __shfl_xor_sync(0xffffffffu, sum.z, d);
        sum.w += __shfl_xor_sync(0xffffffffu, sum.w, d);
      }
      const float inv = total == 0.f ? 0.f : 1.f / total;
      if (lane < kLanes) {
        const int64_t row = static_cast<int64_t>(j.row + r / p.group) * p.q_heads + j.head * p.group + r % p.group;
        *reinterpret_cast<uint2*>(p.out + row * D + lane * 4) =
            make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
      }
    }
  }
}

}  // namespace adb
