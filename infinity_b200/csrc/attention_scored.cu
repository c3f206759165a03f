// Attention with modified scores over a packed batch, and the same over a paged key / value cache, on the 5th-generation
// tensor cores.
//
// Rows. The G query heads that share a key head are packed into one 128-row tile: row r of a tile is token r / G, head
// r % G, so a single new token of a grouped model fills G rows of one tile instead of one row of G tiles, and its keys are read
// once. An item is a query tile of one key head with the key tiles (64 keys) its masks can reach: at most two runs of
// tiles, the prefix and the window (a document mask cuts both to the tiles whose documents meet the query tile's).
//
// Split. A planning kernel (one block) lists the items and cuts the row of all (item, key tile) steps into equal parts, one
// per stream of the grid, wherever the cuts fall: few rows over long caches and many short sequences are balanced by the same
// rule. An item that a cut divides leaves partial results (fp32 numerators, maximum, denominator) in the workspace; the
// stream that finishes last joins them in the order of the parts, so the result depends on the lengths and not on timing.
//
// A CTA (one per SM) runs two streams, A and B, each with its own 128-row tile, softmax warpgroup and tensor-memory
// accumulators, so that one stream's exponentials run under the other's matrix products. Each walks its own part. (Streams on
// neighbouring tiles of one item row that share every key and value tile read half as much, but what bounds the kernel is the softmax:
// 4 sequences of 4000 tokens, 28/4 heads of 128, 1058 us so and 993 us apart; 16 heads of 64 513 and 517.)
// Per step of a stream, 64 keys:
//   S = Q K^T     tcgen05.mma 128 x N x 16 (N = valid keys rounded up to 16), fp32 in tensor memory
//   softmax       128 threads, one row each, in one pass over the row: a score becomes its exponential against the row's reference
//                 at once. The reference is a guess (from the first 32 scores of the row's first step) and is only replaced, by the
//                 exact maximum and a second pass, when the sum leaves 2^-60 .. 2^48: numerators and denominator share its
//                 scale, and fp32 sums and bf16 probabilities keep their relative precision anywhere in between; the numerators of values
//                 up to 2^79 stay finite. Capped scores lie within +-cap and need no reference at all (caps up to 55: 2^+-80).
//   O += P V      P rounded to bf16 (the tensor core's operand type; half a step of 2^-8 per probability) in tensor memory, V as an MN-major
//                 shared-memory operand
// What bounds it: a softmax warp's chain of dependent instructions, two such warps on each scheduler; the special-function unit is
// busy 15 to 47 % of the time, the tensor cores 10 to 46 %, the issue slots 38 to 51 % (single tokens over a cache: 8, 27 and 19 %, they wait
// for memory). 8 sequences of 2048 tokens, 28/4 heads of 128, normal inputs: 541 us (890 TFLOP/s; 580 with slopes, 668 capped, 373 causal,
// 709 with a bias table of radius 128); 16 heads of 64: 266 us (517 TFLOP/s; 281 with slopes, 334 capped, 177 causal). One new token of 64
// sequences over 64 to 8192 keys, 28/4 heads of 128: 66 us, 3.5 TB/s, 6 of them the plan.
// Warps: 0-3 softmax A, 4-7 softmax B, 8 loads Q and K, 9 loads V, 10 and 11 issue the matrix instructions of A and B.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "kernels.h"
// waits here are short and on the chain softmax -> MMA -> softmax: plain polling, as in attention_tc2.cu
#define B2_MBAR_SUSPEND_NS 0
#include "ptx.cuh"

namespace b2 {

static constexpr int AS_MAX_RADIUS = 1023;
static constexpr int AS_MAX_GROUP = 128;
static constexpr int AS_MAX_POSITIONS = 1 << 30;   // a tile's end stays inside 32 bits
static constexpr int64_t AS_ALIGN = 256;
static constexpr int AS_MAX_CTAS = 160;
static constexpr int AS_MAX_SLOTS = 2 * AS_MAX_CTAS;
static constexpr int AS_SOFTMAX_WARPS = 8, AS_K_WARP = 8, AS_V_WARP = 9, AS_MMA_WARP = 10;  // and 11: one a stream
static constexpr int AS_THREADS = 12 * 32;
static constexpr int AS_PLAN_THREADS = 1024, AS_PLAN_CACHE = 1024;  // entries whose prefix sums the planner keeps in shared memory
// What an item costs beside its steps, in steps (its loads, first scores, output): measured on 16 sequences of causal attention,
// where slots of short items took 2.7 us an item longer than equal slots of long ones at 1.45 us a step;
// 1, 3, 4 and 6 in its place were no faster for any of short, long, causal, cached and single-token batches.
static constexpr int AS_ITEM_STEPS = 2;
static constexpr int AS_STAGE = 16 * 64;           // output staging of a warp: 16 rows of 64 bytes
static constexpr uint32_t AS_TMEM_COLS = 512;
static constexpr int AS_COLD = 12;                 // words of a softmax warp's values that only an item's ends need
static constexpr int AS_PACKED_BOX = 32;           // rows of one copy of a packed key tile: short sequences copy few rows
static constexpr int AS_TABLE = 1024;              // floats of a stream's staged bias tables
static constexpr float AS_LOG2E = 1.4426950408889634f;
static constexpr float AS_SUM_LOW = 0x1p-60f, AS_SUM_HIGH = 0x1p48f;  // sums that keep the reference, see above
static constexpr float AS_CAP_LOW = 0x1p-7f, AS_CAP_HIGH = 80.f;      // cap * log2(e) that AS_CAP serves: 2^+-80 keeps fp32 sums in range

struct AttnMod {
  float scale, cap;
  int left, right, radius;
  const float* slopes;
  const float* bias;
  const int32_t* prefix;
  const int32_t* docs;
};

// One query tile of one sequence; the same for every key head.
struct __align__(16) AttnEntry {
  int32_t seq, tok0, n_tok, pos0;     // first row of q and out, tokens, position of the first
  int32_t kv_len, kv_row0, prefix, n; // keys; packed: first row of k and v; visible prefix; key tiles visited
  int32_t a0, n0, a1, near;           // visited tiles: a0 .. a0 + n0 - 1, then the run from a1, tile a1 + near first, down, then up
  int64_t before;                     // key tiles of the entries in front (per key head)
  int64_t cost;                       // the same with AS_ITEM_STEPS more for each entry
};
static_assert(sizeof(AttnEntry) == 64, "entry layout");

struct AttnSlot {  // where a stream starts, and its steps
  int32_t e, h, k, count;
};

struct AttnPlan {  // views into the workspace
  int32_t* status;
  int64_t* bound;        // [slots + 1] first step of each slot
  AttnSlot* slot;        // [slots]
  int32_t* counter;      // [slots] finished parts of the item that starts in a slot
  int32_t* seq_first;    // [n_seqs + 1] first entry of a sequence
  int2* doc_range;       // [n_tokens / keys of a tile + n_seqs + 1] smallest and largest document of a key tile
  AttnEntry* entry;
  float2* part_ml;       // [2 * slots][rows] maximum (log2 units) and denominator
  float* part_o;         // [...][rows][Dp]
  int32_t max_entries, rows;
};

struct AttnJob {
  __nv_bfloat16* out;
  int64_t out_stride;
  const int32_t* cu;
  const int32_t* kv_lens;
  const int32_t* page_table;
  int n_seqs, n_tokens, n_heads, n_kv_heads, head_dim, group, group_inv, tile_tokens;  // r / group = r * group_inv >> 16 for r, group <= 128
  int n_pages, page_size, table_stride, box_rows, head_first;
};

__device__ __forceinline__ float as_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float as_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float as_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float as_max3_abs(float a, float b, float c) {  // max(|a|, |b|, |c|)
  float d;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 1 - 2 / (1 + e^2x), off by about 2^-22 of one
__device__ __forceinline__ float as_tanh(float x) { return fmaf(-2.f, as_rcp(1.f + as_ex2(x * (2.f * AS_LOG2E))), 1.f); }
// 32-bit mask of the x lowest bits, x clamped to 0 .. 32
__device__ __forceinline__ uint32_t as_below(int x) {
  uint32_t m;
  asm("bmsk.clamp.b32 %0, 0, %1;" : "=r"(m) : "r"(max(x, 0)));
  return m;
}

// ---- planning -------------------------------------------------------------------------

// Tokens of sequence s, cut to the buffer.
__device__ __forceinline__ int2 as_rows_of(const AttnJob& j, int s) {
  const int first = min(max(j.cu[s], 0), j.n_tokens);
  return make_int2(first, min(max(j.cu[s + 1], first), j.n_tokens));
}

// Exclusive sum over the block of v, plus *carry, which then grows by the block's total.
__device__ int64_t as_block_sum(int64_t v, int64_t* carry, int64_t* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int64_t w = lane < (blockDim.x >> 5) ? scratch[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += y;
    }
    scratch[lane] = w;
  }
  __syncthreads();
  const int64_t base = *carry + (warp ? scratch[warp - 1] : 0);
  const int64_t total = scratch[31];
  __syncthreads();
  if (threadIdx.x == 0) *carry += total;
  __syncthreads();
  return base + x - v;
}

// First key tile record of sequence s: (first token / kv) + s never runs into the next sequence's.
__device__ __forceinline__ int as_doc_base(int first, int s, int kv) { return first / kv + s; }

__global__ void __launch_bounds__(AS_PLAN_THREADS, 1)
attn_plan_kernel(const AttnJob j, const AttnMod mod, const AttnPlan p, int tokens_per_entry, int max_slots, int kv) {
  __shared__ int64_t scratch[32];
  __shared__ int64_t carry;
  __shared__ int64_t steps_of[AS_PLAN_CACHE];  // AttnEntry::before
  __shared__ int64_t cuts[AS_MAX_SLOTS + 1];
  __shared__ int2 rows_s[AS_PLAN_CACHE];        // as_rows_of, for so many sequences
  __shared__ int first_s[AS_PLAN_CACHE];        // AttnPlan::seq_first
  __shared__ int2 docs_s[AS_PLAN_CACHE];        // AttnPlan::doc_range
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    *p.status = 0;
    carry = 0;
  }
  for (int i = tid; i < max_slots; i += static_cast<int>(blockDim.x)) p.counter[i] = 0;
  for (int i = tid; i < max_slots; i += static_cast<int>(blockDim.x)) p.slot[i] = AttnSlot{0, 0, 0, 0};
  __syncthreads();
  // the device copies of the lengths, read once
  const bool few = j.n_seqs <= AS_PLAN_CACHE;
  if (few)
    for (int s = tid; s < j.n_seqs; s += static_cast<int>(blockDim.x)) rows_s[s] = as_rows_of(j, s);
  __syncthreads();
  auto rows_of = [&](int s) { return few ? rows_s[s] : as_rows_of(j, s); };
  auto first_of = [&](int s) { return few ? first_s[s] : p.seq_first[s]; };
  // entries of each sequence
  for (int base = 0; base < j.n_seqs; base += static_cast<int>(blockDim.x)) {
    const int s = base + tid;
    int count = 0;
    if (s < j.n_seqs) {
      const int2 r = rows_of(s);
      count = (r.y - r.x + tokens_per_entry - 1) / tokens_per_entry;
    }
    const int64_t at = as_block_sum(count, &carry, scratch);
    if (s < j.n_seqs) {
      const int e0 = static_cast<int>(min(at, static_cast<int64_t>(p.max_entries)));
      p.seq_first[s] = e0;
      if (few) first_s[s] = e0;
    }
  }
  const int n_entries = static_cast<int>(min(carry, static_cast<int64_t>(p.max_entries)));
  if (tid == 0) p.seq_first[j.n_seqs] = n_entries;
  __syncthreads();
  auto sequence_of_entry = [&](int e) {  // the last sequence whose first entry is <= e: empty ones in front share it
    int lo = 0, hi = j.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_of(mid) <= e) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  if (mod.docs != nullptr) {
    // documents of every key tile (tokens of no document left out), a warp a tile
    const int records = j.n_tokens / kv + j.n_seqs;
    for (int i = warp; i < records; i += static_cast<int>(blockDim.x) >> 5) {
      int lo = 0, hi = j.n_seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (as_doc_base(rows_of(mid).x, mid, kv) <= i) lo = mid;
        else hi = mid;
      }
      const int2 r = rows_of(lo);
      const int t0 = r.x + (i - as_doc_base(r.x, lo, kv)) * kv;
      if (t0 < r.x) continue;  // only where cu_seqlens is not sorted
      int dmin = INT_MAX, dmax = -1;
      for (int t = t0 + lane; t < min(t0 + kv, r.y); t += 32) {
        const int d = mod.docs[t];
        if (d >= 0) {
          dmin = min(dmin, d);
          dmax = max(dmax, d);
        }
      }
      dmin = __reduce_min_sync(0xffffffffu, dmin);
      dmax = __reduce_max_sync(0xffffffffu, dmax);
      if (lane == 0 && t0 < r.y) {
        p.doc_range[i] = make_int2(dmin, dmax);
        if (i < AS_PLAN_CACHE) docs_s[i] = make_int2(dmin, dmax);
      }
    }
    __syncthreads();
    // first and past-the-last key tile whose documents meet an entry's (kept in its record), a warp an entry, 32 key tiles at a time
    for (int e = warp; e < n_entries; e += static_cast<int>(blockDim.x) >> 5) {
      const int s = sequence_of_entry(e);
      const int2 r = rows_of(s);
      const int q0 = (e - first_of(s)) * tokens_per_entry, tiles = (r.y - r.x + kv - 1) / kv;
      const int base = as_doc_base(r.x, s, kv);
      auto range = [&](int t) { return base + t < AS_PLAN_CACHE ? docs_s[base + t] : p.doc_range[base + t]; };
      int dmin = INT_MAX, dmax = -1;
      for (int t = q0 / kv + lane; t <= min(q0 + tokens_per_entry, r.y - r.x) / kv && t < tiles; t += 32) {
        const int2 d = range(t);
        dmin = min(dmin, d.x);
        dmax = max(dmax, d.y);
      }
      dmin = __reduce_min_sync(0xffffffffu, dmin);
      dmax = __reduce_max_sync(0xffffffffu, dmax);
      int first = INT_MAX, last = -1;
      for (int t0 = 0; t0 < tiles; t0 += 32) {
        bool meets = false;
        if (t0 + lane < tiles) {
          const int2 d = range(t0 + lane);
          meets = d.x <= dmax && d.y >= dmin;
        }
        const uint32_t m = __ballot_sync(0xffffffffu, meets);
        if (m) {
          first = min(first, t0 + __ffs(m) - 1);
          last = t0 + 31 - __clz(m);
        }
      }
      if (lane == 0) {
        p.entry[e].a0 = last < 0 ? 0 : first;
        p.entry[e].n0 = last + 1;
      }
    }
    __syncthreads();
  }
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int base = 0; base < n_entries; base += static_cast<int>(blockDim.x)) {
    const int e = base + tid;
    AttnEntry x = {};
    int doc_lo = 0, doc_hi = INT_MAX;
    if (e < n_entries) {
      const int lo = sequence_of_entry(e);
      const int2 r = rows_of(lo);
      const int q0 = (e - first_of(lo)) * tokens_per_entry;
      x.seq = lo;
      x.tok0 = r.x + q0;
      x.n_tok = min(tokens_per_entry, r.y - r.x - q0);
      x.kv_row0 = r.x;
      x.kv_len = j.kv_lens == nullptr ? r.y - r.x : min(max(j.kv_lens[lo], 0), j.table_stride * j.page_size);
      x.pos0 = x.kv_len - (r.y - r.x) + q0;
      x.prefix = mod.prefix == nullptr ? 0 : min(max(mod.prefix[lo], 0), x.kv_len);
      if (mod.docs != nullptr) {
        doc_lo = p.entry[e].a0;
        doc_hi = p.entry[e].n0;
      }
    }
    if (e < n_entries) {
      // keys that the window of some token reaches, then the tiles of the prefix in front of them
      const int p1 = x.pos0 + x.n_tok - 1;
      const int key_lo = static_cast<int>(max(static_cast<int64_t>(x.pos0) - mod.left, int64_t(0)));
      const int key_hi = static_cast<int>(min(static_cast<int64_t>(p1) + mod.right + 1, static_cast<int64_t>(x.kv_len)));
      int b0 = 0, b1 = 0, f1 = min((x.prefix + kv - 1) / kv, doc_hi);
      if (key_hi > key_lo) {
        b0 = max(key_lo / kv, doc_lo);
        b1 = max(min((key_hi + kv - 1) / kv, doc_hi), b0);
      }
      const int f0 = min(doc_lo, f1);
      if (b1 == b0) b0 = b1 = f1;  // no window: the prefix alone
      if (f1 >= b0) {              // the two runs meet
        b0 = min(b0, f0);
        b1 = max(b1, f1);
        f1 = f0;
      }
      x.a0 = f0;
      x.n0 = f1 - f0;
      x.a1 = b0;
      x.n = x.n0 + (b1 - b0);
      if (mod.slopes != nullptr) x.near = min(max(p1 / kv - b0, 0), max(b1 - b0 - 1, 0));
      if (x.n == 0) {  // nothing visible: one step whose keys are all masked writes the zeros
        x.a0 = x.a1 = 0;
        x.n0 = 0;
        x.n = 1;
      }
    }
    x.before = as_block_sum(x.n, &carry, scratch);
    x.cost = x.before + static_cast<int64_t>(AS_ITEM_STEPS) * e;
    if (e < n_entries) {
      p.entry[e] = x;
      if (e < AS_PLAN_CACHE) steps_of[e] = x.before;
    }
  }
  // Parts of equal cost; a cut moves to an item's edge that is nearer than 1/16 of a part.
  const int heads = j.n_kv_heads;
  const int64_t total = carry * heads, total_cost = (carry + static_cast<int64_t>(AS_ITEM_STEPS) * n_entries) * heads;
  // parts have two steps or more on average, since what a part costs to join is more than a step (a cut by cost may still leave one)
  const int64_t most = max(min(total, static_cast<int64_t>(n_entries) * heads), (total + 1) / 2);
  const int slots = static_cast<int>(min(most, static_cast<int64_t>(max_slots)));
  __syncthreads();
  if (slots == 0) return;
  auto before_of = [&](int e) { return e < AS_PLAN_CACHE ? steps_of[e] : p.entry[e].before; };
  auto last_entry = [&](int64_t at, int extra) {  // the last entry that starts at or before `at`, with `extra` steps for each in front
    int lo = 0, hi = n_entries;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((before_of(mid) + static_cast<int64_t>(extra) * mid) * heads <= at) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  auto tiles_of = [&](int e) { return static_cast<int>((e + 1 < n_entries ? before_of(e + 1) : carry) - before_of(e)); };
  const int64_t slack = total_cost / (16 * static_cast<int64_t>(slots));
  for (int s = tid; s <= slots; s += static_cast<int>(blockDim.x)) {
    int64_t cut = total;
    if (s < slots) {
      const int64_t at = total_cost / slots * s + total_cost % slots * s / slots;
      const int e = last_entry(at, AS_ITEM_STEPS), n = tiles_of(e);
      const int64_t in = at - (before_of(e) + static_cast<int64_t>(AS_ITEM_STEPS) * e) * heads;
      const int h = static_cast<int>(in / (n + AS_ITEM_STEPS));
      int k = min(max(static_cast<int>(in - static_cast<int64_t>(h) * (n + AS_ITEM_STEPS)) - AS_ITEM_STEPS / 2, 0), n);
      if (k <= slack && k <= n - k) k = 0;
      else if (n - k <= slack) k = n;
      cut = before_of(e) * heads + static_cast<int64_t>(h) * n + k;
    }
    cuts[s] = cut - s;
  }
  __syncthreads();
  // every part has a step: the running maximum of (cut - number) makes the cuts strictly ascending, the end bounds them
  if (warp == 0) {
    const int per = (slots + 32) / 32;
    int64_t top = INT64_MIN;
    for (int i = 0; i < per; ++i)
      if (lane * per + i <= slots) top = max(top, cuts[lane * per + i]);
    int64_t front = top;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, front, d);
      if (lane >= d) front = max(front, y);
    }
    front = __shfl_up_sync(0xffffffffu, front, 1);
    if (lane == 0) front = INT64_MIN;
    for (int i = 0; i < per; ++i) {
      const int s = lane * per + i;
      if (s <= slots) {
        front = max(front, cuts[s]);
        cuts[s] = min(front + s, total - (slots - s));
      }
    }
  }
  __syncthreads();
  for (int s = tid; s <= slots; s += static_cast<int>(blockDim.x)) {
    const int64_t cut = cuts[s];
    p.bound[s] = cut;
    if (s < slots) {
      const int e = last_entry(cut, 0), n = tiles_of(e);
      const int64_t in = cut - before_of(e) * heads;
      p.slot[s] = AttnSlot{e, static_cast<int>(in / n), static_cast<int>(in % n), static_cast<int>(cuts[s + 1] - cut)};
    }
  }
}

// ---- the attention kernel -----------------------------------------------------------------

template <int D>
struct AsCfg {
  static constexpr int BLOCKS = D / 64;
  // Keys of a step. Steps of 64 leave room in tensor memory for two score buffers a stream, so that the next scores are there
  // before the softmax has finished these.
  static constexpr int KV = 64;
  static constexpr int Q_BLOCK = 128 * 128, Q_TILE = BLOCKS * Q_BLOCK;     // rows of 64 columns, 128-byte swizzle
  static constexpr int KV_BLOCK = KV * 128, KV_TILE = BLOCKS * KV_BLOCK;
  static constexpr int RING = D == 64 ? 8 : 4;  // key (and value) tiles in flight: 64 KB of each
  static constexpr int Q_BUFS = D == 64 ? 2 : 1;  // query tiles of a stream
  static constexpr int STAGE_BYTES = AS_SOFTMAX_WARPS * AS_STAGE;
  static constexpr int TABLE_BYTES = 2 * AS_TABLE * 4;
  static constexpr int BAR_BYTES = 512;
  static constexpr int COLD_BYTES = AS_SOFTMAX_WARPS * AS_COLD * 4;
  static constexpr int SMEM_BYTES = 2 * Q_BUFS * Q_TILE + 2 * RING * KV_TILE + STAGE_BYTES + TABLE_BYTES + BAR_BYTES + COLD_BYTES + 1024;
  static constexpr int N_BARS = 4 * RING + 4 * 2 + 2 * 7;
  static_assert(N_BARS * 8 + 16 <= BAR_BYTES, "barrier area");
  static_assert(SMEM_BYTES <= 232448, "shared memory");
  // Tensor memory of stream t: two score buffers of 64 columns, the accumulators, and P of a buffer's chunk of 32 keys in the first 16
  // of the chunk's own 32 columns.
  static __host__ __device__ constexpr uint32_t S(int t, int b) { return t * 128 + b * 64; }
  static __host__ __device__ constexpr uint32_t O(int t) { return 256 + t * D; }
};

// The steps of a stream, in order. Every role of the stream walks the same ones.
template <int KV>
struct AsWalk {
  int left, e, h, k;  // steps left (this one included); entry, key head, key tile of the item
  bool first;         // first step of a segment (an item, or this stream's part of one)
  int4 f0, f1, f2;    // the entry
  __device__ void load(const AttnEntry* entry) {
    const int4* p = reinterpret_cast<const int4*>(entry + e);
    f0 = p[0];
    f1 = p[1];
    f2 = p[2];
  }
  __device__ void start(const AttnPlan& p, int slot) {
    const int4 s = *reinterpret_cast<const int4*>(p.slot + slot);
    e = s.x;
    h = s.y;
    k = s.z;
    left = s.w;
    first = true;
    if (left > 0) load(p.entry);
  }
  __device__ bool last() const { return left == 1 || k == f1.w - 1; }
  // With a bias that falls with the distance the run starts at the queries' own tile and moves away from it, so that the first
  // reference of a row serves all steps; otherwise near is 0 and the run is taken in order.
  __device__ int key0() const {
    const int i = k - f2.y;
    return (i < 0 ? f2.x + k : f2.z + (i <= f2.w ? f2.w - i : i)) * KV;
  }
  __device__ int n_valid() const { return min(max(f1.x - key0(), 0), KV); }
  __device__ void next(const AttnPlan& p, int n_kv_heads) {
    first = false;
    if (++k == f1.w) {
      k = 0;
      first = true;
      if (++h == n_kv_heads) {
        h = 0;
        ++e;
        if (left > 1) load(p.entry);
      }
    }
    --left;
  }
};

__device__ __forceinline__ int as_round16(int n) { return max((n + 15) & ~15, 16); }

__device__ __forceinline__ void as_tma_3d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                   smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void as_tma_4d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
                   smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}

// Bounded wait of a whole warp. Every lane has its own clock, and a phase may end while they run out: the warp takes one answer, since
// lanes that went on would wait in a vote for lanes that have left. (The vote of the first look spares the loop: capped batches 3 % and
// documents 0.5 % faster so, plain scores at head_dim 128 1 % slower.)
__device__ __forceinline__ bool as_wait(uint64_t* bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// One look at a barrier: whether the phase of this parity is over.
__device__ __forceinline__ bool as_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bound of a loop that looks at several barriers in turn: false when nothing has moved for WAIT_LIMIT_NS. Every lane asks; the
// warp gives up together.
struct AsPatience {
  uint32_t idle = 0;
  unsigned long long since = 0;
  __device__ bool go_on(bool moved) {
    if (moved) {
      idle = 0;
      return true;
    }
    __nanosleep(40);  // leaves the issue slots to the warps that have work
    if ((++idle & 0xffu) != 0u) return true;
    const unsigned long long now = globaltimer_ns();
    if (idle == 0x100u) since = now;
    return __all_sync(0xffffffffu, now - since <= WAIT_LIMIT_NS) != 0;
  }
};

// After a failed wait: lets the copies still in flight land before shared memory is released (bounded).
__device__ __forceinline__ void as_drain(uint64_t* full, uint32_t fills, uint32_t slots) {
  for (uint32_t i = 0; i < (fills < slots ? fills : slots); ++i) {
    const uint32_t idx = fills - 1 - i;
    as_wait(&full[idx % slots], (idx / slots) & 1u);
  }
}

// Copies the valid rows of a step's key (or value) tile: lane l takes rows (l % 16) * box_rows .. of the 64-column block l / 16.
template <int D, bool PAGED>
__device__ __forceinline__ void as_load_tile(const AttnJob& j, const AsWalk<AsCfg<D>::KV>& w, const CUtensorMap* tmap, uint8_t* dst,
                                             uint64_t* full, int lane) {
  const int n_valid = w.n_valid();
  const int boxes = (n_valid + j.box_rows - 1) / j.box_rows;
  const int r = lane & 15, cb = lane >> 4;
  const bool mine = r < boxes && cb < AsCfg<D>::BLOCKS;
  int page = 0, off = 0;
  const int key = w.key0() + r * j.box_rows;
  if (PAGED && mine) {
    const int at = key / j.page_size;
    off = key - at * j.page_size;
    page = __ldg(j.page_table + static_cast<int64_t>(w.f0.x) * j.table_stride + at);
    if (page < 0 || page >= j.n_pages) page = j.n_pages;  // outside the tensor: zeros
  }
  if (lane == 0) mbar_arrive_expect_tx(full, boxes * j.box_rows * 128 * AsCfg<D>::BLOCKS);
  __syncwarp();
  if (mine) {
    uint8_t* to = dst + cb * AsCfg<D>::KV_BLOCK + r * j.box_rows * 128;
    if (PAGED) {
      if (j.head_first) as_tma_4d(to, tmap, full, cb * 64, w.h, off, page);
      else as_tma_4d(to, tmap, full, cb * 64, off, w.h, page);
    } else {
      as_tma_3d(to, tmap, full, cb * 64, w.h, w.f1.y + key);
    }
  }
}

// What happens to a score before it is masked. The kernel is built for each: a row of scores is worked on in straight-line
// code, and one body with every branch in it is 120 KB of instructions, which the instruction caches do not hold (7 us a step).
enum { AS_PLAIN = 0, AS_SLOPES = 1, AS_CAP = 2, AS_BIAS = 3, AS_DOCS = 4, AS_ANY = 5 };
// (AS_BIAS: a bias table alone; AS_DOCS: documents, with or without one)

// tanh(x) = x (c0 + c1 u + ... + c5 u^5), u = x^2, within 2.5e-7 on [-1, 1]: the odd polynomial with the smallest largest error there
// (fitted to tanh in 64 bits by reweighted least squares). It spares the two special-function instructions of
// 1 - 2 / (1 + e^2x) on top of the exponential's own; scores within the cap never leave its range. Two values at a time;
// c tanh(v / c) is formed with c^-2k folded into the coefficients (AS_CAP_LOW .. AS_CAP_HIGH keeps them in fp32's range).
struct AsTanh {
  float2 c[6];
  __device__ explicit AsTanh(float cap) {
    const float f = 1.f / (cap * cap);
    const float c0[6] = {0.9999968409538269f, -0.3332400321960449f, 0.13253524899482727f, -0.05097285658121109f, 0.01611417345702648f, -0.0028394628316164017f};
    float g = 1.f;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      c[i] = make_float2(c0[i] * g, c0[i] * g);
      g *= f;
    }
  }
  __device__ float2 operator()(float2 v, float2 w) const {
    float2 y = __ffma2_rn(w, c[5], c[4]);
    y = __ffma2_rn(w, y, c[3]);
    y = __ffma2_rn(w, y, c[2]);
    y = __ffma2_rn(w, y, c[1]);
    y = __ffma2_rn(w, y, c[0]);
    return __fmul2_rn(v, y);
  }
};

template <int D, bool PAGED, int MODE>
__global__ void __launch_bounds__(AS_THREADS, 1)
attn_scored_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ AttnJob j, const __grid_constant__ AttnMod mod,
                   const __grid_constant__ AttnPlan plan) {
  using Cfg = AsCfg<D>;
  constexpr int RING = Cfg::RING, KV = Cfg::KV;
  constexpr uint32_t Q_BUFS = Cfg::Q_BUFS;
  // Whether a segment's first step may go the straight way, us with it and without. Caps (they need no reference): 96 sequences of 300 tokens,
  // 16 heads of 64, 174 and 194; 64 of 300, 28/4 heads of 128, 186 and 204; 8 of 2048 334 and 343, 670 and 690. Bias tables: the same short
  // batches 205 and 225, 214 and 231, long ones equal. Plain scores at head_dim 128: short 153 and 156, causal 131 and 133, long 543 and 536; at 64 long
  // ones lose more (283 and 265; short 144 and 147, causal 121 and 126). Slopes: their first step holds the queries' own positions.
  constexpr bool FIRST = MODE == AS_CAP || MODE == AS_BIAS || (MODE == AS_PLAIN && D == 128);
  constexpr bool DOCS = MODE == AS_DOCS || MODE == AS_ANY, TABLES = DOCS || MODE == AS_BIAS;
  // A stream's own tiles in flight, so that neither stream waits for the other's.
  constexpr uint32_t SLOTS = RING / 2;
  extern __shared__ uint8_t as_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(as_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;
  uint8_t* k_s = q_s + 2 * Cfg::Q_BUFS * Cfg::Q_TILE;
  uint8_t* v_s = k_s + RING * Cfg::KV_TILE;
  uint8_t* stage_s = v_s + RING * Cfg::KV_TILE;
  float* table_s = reinterpret_cast<float*>(stage_s + Cfg::STAGE_BYTES);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(stage_s + Cfg::STAGE_BYTES + Cfg::TABLE_BYTES);
  uint64_t* k_empty = k_full + RING;
  uint64_t* v_full = k_empty + RING;
  uint64_t* v_empty = v_full + RING;
  uint64_t* q_full = v_empty + RING;  // the following ones per stream: [stream][buffer]
  uint64_t* q_empty = q_full + 4;
  uint64_t* s_full = q_empty + 4;     // [stream][buffer] S of a step is in tensor memory
  uint64_t* p_full = s_full + 4;      // [stream][buffer] P of a step is in tensor memory, O may be added to
  uint64_t* pv_done = p_full + 4;     // [stream][buffer] P V of a step has finished
  uint64_t* group_bar = pv_done + 4;  // the softmax warps of a stream meet
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(group_bar + 2);
  uint32_t* joins = tmem_slot + 1;                                          // per stream: these warps join the parts of the item

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < RING; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&q_full[2 * t + b], 1);
        mbar_init(&q_empty[2 * t + b], 1);
        mbar_init(&s_full[2 * t + b], 1);
        mbar_init(&p_full[2 * t + b], AS_SOFTMAX_WARPS / 2);
        mbar_init(&pv_done[2 * t + b], 1);
      }
      mbar_init(&group_bar[t], AS_SOFTMAX_WARPS / 2);
    }
    fence_mbar_init();
  }
  if (warp == AS_MMA_WARP) {
    tmem_alloc(tmem_slot, AS_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();  // the plan, and whatever wrote q, k and v

  if (warp == AS_K_WARP || warp == AS_V_WARP) {
    // ---------------- loads: Q and K, V ----------------
    const bool is_k = warp == AS_K_WARP;
    const CUtensorMap* tmap = is_k ? &tmap_k : &tmap_v;
    uint8_t* ring = is_k ? k_s : v_s;
    uint64_t* full = is_k ? k_full : v_full;
    uint64_t* empty = is_k ? k_empty : v_empty;
    if (lane == 0) {
      tma_prefetch_desc(tmap);
      if (is_k) tma_prefetch_desc(&tmap_q);
    }
    AsWalk<KV> w[2];
    w[0].start(plan, blockIdx.x);
    w[1].start(plan, blockIdx.x + gridDim.x);
    uint32_t fills[2] = {0, 0}, q_fills[2] = {0, 0};
    AsPatience patience;
    bool ok = true;
    // whichever stream has room takes its next step
    while (ok && (w[0].left > 0 || w[1].left > 0)) {
      bool moved = false;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (w[t].left <= 0) continue;
        const uint32_t slot = t * SLOTS + fills[t] % SLOTS;
        bool ready = as_test(&empty[slot], ((fills[t] / SLOTS) & 1u) ^ 1u);
        if (is_k && w[t].first) ready = ready && as_test(&q_empty[2 * t + q_fills[t] % Q_BUFS], ((q_fills[t] / Q_BUFS) & 1u) ^ 1u);
        if (!__all_sync(0xffffffffu, ready)) continue;
        moved = true;
        if (is_k && w[t].first) {
          if (lane == 0) {
            const uint32_t qb = q_fills[t] % Q_BUFS;
            mbar_arrive_expect_tx(&q_full[2 * t + qb], j.group * j.tile_tokens * 128 * Cfg::BLOCKS);
#pragma unroll
            for (int b = 0; b < Cfg::BLOCKS; ++b)
              as_tma_3d(q_s + (t * Q_BUFS + qb) * Cfg::Q_TILE + b * Cfg::Q_BLOCK, &tmap_q, &q_full[2 * t + qb], b * 64, w[t].h * j.group,
                        w[t].f0.y);
          }
          ++q_fills[t];
        }
        as_load_tile<D, PAGED>(j, w[t], tmap, ring + slot * Cfg::KV_TILE, &full[slot], lane);
        ++fills[t];
        w[t].next(plan, j.n_kv_heads);
      }
      ok = patience.go_on(moved);
    }
    if (is_k) pdl_launch_dependents();
    if (!ok) {
      if (lane == 0) atomicExch(plan.status, is_k ? 5 : 8);
      for (int t = 0; t < 2; ++t) as_drain(&full[t * SLOTS], fills[t], SLOTS);
      if (is_k)
        for (int u = 0; u < 2; ++u) as_drain(&q_full[2 * u], q_fills[u], Q_BUFS);
    }
  } else if (warp >= AS_MMA_WARP) {
    // ---------------- matrix instructions of stream t: all lanes walk, one elected lane issues ----------------
    // (a warp for each stream: one warp that looks at both streams' barriers in turn answers each some hundred cycles later)
    const int t = warp - AS_MMA_WARP;
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0);
    const uint32_t q_addr = smem_u32(q_s) + t * Q_BUFS * Cfg::Q_TILE, k_addr = smem_u32(k_s), v_addr = smem_u32(v_s);
    const uint32_t ring0 = t * SLOTS;
    AsWalk<KV> sw, pw;  // the next S, and the next P V
    sw.start(plan, blockIdx.x + t * gridDim.x);
    pw = sw;
    uint32_t q_uses = 0, n_s = 0, n_pv = 0;
    const uint32_t idesc_pv = make_idesc_bf16_f32_b_mn(128, D);
    auto issue_s = [&]() -> bool {
      const uint32_t slot = ring0 + n_s % SLOTS, buf = n_s % 2;
      if (sw.first) {
        if (!as_wait(&q_full[2 * t + q_uses % Q_BUFS], (q_uses / Q_BUFS) & 1u)) return false;
        ++q_uses;
      }
      const uint32_t qb = (q_uses - 1) % Q_BUFS;
      if (!as_wait(&k_full[slot], (n_s / SLOTS) & 1u)) return false;
      tc_fence_after_sync();
      const uint32_t idesc = make_idesc_bf16_f32(128, as_round16(sw.n_valid()));
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint64_t a = make_kmajor_sw128_desc(q_addr + qb * Cfg::Q_TILE + (k / 4) * Cfg::Q_BLOCK) + 2 * (k % 4);
        const uint64_t b = make_kmajor_sw128_desc(k_addr + slot * Cfg::KV_TILE + (k / 4) * Cfg::KV_BLOCK) + 2 * (k % 4);
        if (elect_one()) tc_mma_f16(tmem_u + t * Cfg::S(1, 0) + buf * Cfg::S(0, 1), a, b, idesc, k != 0);
      }
      if (elect_one()) {
        tc_commit(&s_full[2 * t + buf]);
        tc_commit(&k_empty[slot]);
        if (sw.last()) tc_commit(&q_empty[2 * t + qb]);
      }
      ++n_s;
      sw.next(plan, j.n_kv_heads);
      return true;
    };
    auto issue_pv = [&]() -> bool {
      const uint32_t slot = ring0 + n_pv % SLOTS, buf = n_pv % 2;
      if (!as_wait(&v_full[slot], (n_pv / SLOTS) & 1u)) return false;
      const int n_valid = pw.n_valid(), n_eff = as_round16(n_valid);
      if (n_valid < n_eff) {
        // value rows behind the last key: whatever lies there must not meet a zero probability (0 * NaN)
        uint8_t* tile = v_s + slot * Cfg::KV_TILE;
        for (int i = lane; i < (n_eff - n_valid) * 8 * Cfg::BLOCKS; i += 32) {
          const int b = i / ((n_eff - n_valid) * 8), at = i - b * ((n_eff - n_valid) * 8);
          *reinterpret_cast<uint4*>(tile + b * Cfg::KV_BLOCK + n_valid * 128 + at * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (!as_wait(&p_full[2 * t + buf], (n_pv / 2) & 1u)) return false;
      tc_fence_after_sync();
      const uint64_t v_desc = make_mnmajor_sw128_desc(v_addr + slot * Cfg::KV_TILE, Cfg::KV_BLOCK);
      const uint32_t p_at = tmem_u + t * Cfg::S(1, 0) + buf * Cfg::S(0, 1);
#pragma unroll
      for (int k = 0; k < KV / 16; ++k)
        if (k * 16 < n_eff && elect_one())
          tc_mma_f16_tmem_a(tmem_u + Cfg::O(0) + t * (Cfg::O(1) - Cfg::O(0)), p_at + (k / 2) * 32 + (k % 2) * 8, v_desc + k * 128,
                            idesc_pv, !pw.first || k != 0);
      if (elect_one()) {
        tc_commit(&pv_done[2 * t + buf]);
        tc_commit(&v_empty[slot]);
      }
      ++n_pv;
      pw.next(plan, j.n_kv_heads);
      return true;
    };
    bool ok = true;
    for (int i = 0; i < 2; ++i)
      if (ok && sw.left > 0) ok = issue_s();
    while (ok && pw.left > 0) {
      // P V reads the P that took the place of its scores, then the scores of the step after the next may go there
      ok = issue_pv();
      if (ok && sw.left > 0) ok = as_wait(&pv_done[2 * t + (n_pv - 1) % 2], ((n_pv - 1) / 2) & 1u) && issue_s();
    }
    if (!ok && lane == 0) atomicExch(plan.status, 7);
  } else {
    // ---------------- softmax: stream t, one row per thread ----------------
    // Registers are what limits this role: what only the ends of a segment need lies in shared memory in between.
    const int t = warp >> 2, wq = warp & 3, row = wq * 32 + lane;
    const uint32_t lanes = tmem_base + (static_cast<uint32_t>(wq * 32) << 16);
    enum { C_LEFT, C_E, C_H, C_K, C_TOK0, C_NTOK, C_KVROW0, C_PREFIX, C_N };
    volatile int* cold = reinterpret_cast<volatile int*>(smem + Cfg::SMEM_BYTES - 1024 - Cfg::COLD_BYTES) + warp * AS_COLD;
    float* table = table_s + t * AS_TABLE;
    const int row_tok = (row * j.group_inv) >> 16, g = row - row_tok * j.group;
    const int my_slot = blockIdx.x + t * gridDim.x;
    const float scale_log2 = mod.scale * AS_LOG2E, cap_out = mod.cap * AS_LOG2E;
    // held finite: a score of zero stays zero under the smallest caps
    const float cap_in = mod.cap > 0.f ? fminf(fmaxf(mod.scale / mod.cap, -FLT_MAX), FLT_MAX) : 0.f;
    const float cap_far = mod.cap > 0.f ? fabsf(mod.cap / mod.scale) : 0.f;
    const float2 scale2 = make_float2(scale_log2, scale_log2);
    // exponent of a capped score v = scale_log2 * s: cap_out tanh(v / cap_out), see AsTanh
    const AsTanh tanh_near(MODE == AS_CAP ? cap_out : 1.f);
    if (lane == 0) {
      const int4 s = *reinterpret_cast<const int4*>(plan.slot + my_slot);
      cold[C_E] = s.x;
      cold[C_H] = s.y;
      cold[C_K] = s.z;
      cold[C_LEFT] = s.w;
    }
    __syncwarp();
    uint32_t step = 0, meetings = 0;
    bool failed = false;  // the same in all lanes: see as_wait
    // Bounded barrier of the stream's softmax warps: one that gave up elsewhere makes the others give up here.
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&group_bar[t]);
      if (!as_wait(&group_bar[t], meetings++ & 1u)) failed = true;
    };
    // P V of step s, one of the last two. A barrier is told by its parity alone, so each of two score buffers has its own: of the P V
    // of two steps before, the scores of step s + 1 have already told.
    auto pv_wait = [&](uint32_t s) { return as_wait(&pv_done[2 * t + s % 2], (s / 2) & 1u); };
    auto part_of = [&](int slot, bool tail) -> int64_t { return 2 * slot + (tail ? 1 : 0); };
    float slope = 0.f;
    const float* tab = nullptr;
    float tab_unit = 1.f;
    // every head's slope, for the whole launch (the tables of a bias are not in use then)
    const bool slopes_here = MODE == AS_SLOPES && j.n_heads <= 2 * AS_TABLE;
    if (slopes_here) {
      for (int i = row; i < j.n_heads; i += 128) table_s[i] = __ldg(mod.slopes + i) * AS_LOG2E;  // both streams write the same
      meet();
    }
    while (cold[C_LEFT] > 0 && !failed) {
      // ---- one segment: an item, or this stream's part of one ----
      int i_k, i_end, run0, run_n0, run1, run_near, kv_len, pos, n_rows;
      {
        const int h = cold[C_H];
        const int4* entry = reinterpret_cast<const int4*>(plan.entry + cold[C_E]);
        const int4 f0 = entry[0], f1 = entry[1], f2 = entry[2];
        const int n_tok = f0.z;
        i_k = cold[C_K];
        i_end = min(f1.w, i_k + cold[C_LEFT]);
        run0 = f2.x;
        run_n0 = f2.y;
        run1 = f2.z;
        run_near = f2.w;
        kv_len = f1.x;
        pos = f0.w + row_tok;
        n_rows = n_tok * j.group;
        __syncwarp();
        if (lane == 0) {
          cold[C_TOK0] = f0.y;
          cold[C_NTOK] = n_tok;
          cold[C_KVROW0] = f1.y;
          cold[C_PREFIX] = f1.z;
          cold[C_N] = f1.w;
        }
        __syncwarp();
        if ((MODE == AS_SLOPES || MODE == AS_ANY) && mod.slopes != nullptr)
          slope = slopes_here ? table_s[h * j.group + g] : __ldg(mod.slopes + h * j.group + g) * AS_LOG2E;
        if (TABLES && mod.bias != nullptr) {
          const int width = 2 * mod.radius + 1, n = j.group * width;
          if (n <= AS_TABLE) {
            meet();  // the previous item's reads are over
            if (failed) break;
            for (int i = row; i < n; i += 128) table[i] = __ldg(mod.bias + static_cast<int64_t>(h) * n + i) * AS_LOG2E;
            meet();
            if (failed) break;
            tab = table + g * width + mod.radius;
          } else {
            tab = mod.bias + static_cast<int64_t>(h * j.group + g) * width + mod.radius;
            tab_unit = AS_LOG2E;
          }
        }
      }
      const bool active = wq * 32 < n_rows, real = row < n_rows;
      const int doc = DOCS && mod.docs != nullptr && real ? __ldg(mod.docs + cold[C_TOK0] + row_tok) : -1;
      // first and past-the-last visible key of the window of this row
      auto key_lo = [&]() { return mod.left >= pos ? 0 : pos - mod.left; };
      auto key_hi = [&]() { return mod.right >= kv_len - pos ? kv_len : pos + mod.right + 1; };
      // what holds for all rows of the warp (rows of no token do not count)
      const uint32_t real_rows = __ballot_sync(0xffffffffu, real);
      const int all_lo = __reduce_max_sync(0xffffffffu, real ? key_lo() : INT_MIN), all_hi = __reduce_min_sync(0xffffffffu, real ? key_hi() : INT_MAX);
      const int pos_first = __reduce_min_sync(0xffffffffu, real ? pos : INT_MAX), pos_last = __reduce_max_sync(0xffffffffu, real ? pos : INT_MIN);
      int one_doc = -1;  // the document of all rows, or -1
      if (DOCS && mod.docs != nullptr) {
        const int least = __reduce_min_sync(0xffffffffu, real ? doc : INT_MAX), most = __reduce_max_sync(0xffffffffu, real ? doc : -1);
        one_doc = least == most ? most : -1;
      }
      auto key0_of = [&](int k) {  // as AsWalk::key0
        const int i = k - run_n0;
        return (i < 0 ? run0 + k : run1 + (i <= run_near ? run_near - i : i)) * KV;
      };
      float ref = 0.f, l_run = 0.f;  // reference (log2 units), and the sum of the exponentials against it
      bool first = true;
      int kv0 = key0_of(i_k);
      int next_docs[2] = {-1, -1};  // documents of a step's keys, lane l's of l and 32 + l: asked for a step ahead
      auto docs_of = [&](int key) {
#pragma unroll
        for (int q = 0; q < 2; ++q) next_docs[q] = key + q * 32 + lane < kv_len ? __ldg(mod.docs + cold[C_KVROW0] + key + q * 32 + lane) : -1;
      };
      if (DOCS && mod.docs != nullptr) docs_of(kv0);
      for (; i_k < i_end; ++i_k) {
        const int buf = step % 2, n_valid = min(max(kv_len - kv0, 0), KV), n_rem = as_round16(n_valid);
        const int next_kv0 = i_k + 1 < i_end ? key0_of(i_k + 1) : 0;
        int key_docs[2] = {next_docs[0], next_docs[1]};
        if (DOCS && mod.docs != nullptr) docs_of(next_kv0);
        if (!as_wait(&s_full[2 * t + buf], (step / 2) & 1u)) failed = true;
        if (failed) break;
        tc_fence_after_sync();
        if (active) {
          const uint32_t s_at = lanes + t * Cfg::S(1, 0) + buf * Cfg::S(0, 1);
          bool whole = all_lo <= kv0 && all_hi >= kv0 + KV;  // no masks
          if (DOCS && mod.docs != nullptr && whole)
            whole = one_doc >= 0 && __all_sync(0xffffffffu, key_docs[0] == one_doc && key_docs[1] == one_doc);
          auto seen_of = [&](int q) -> uint32_t {
            const int key = kv0 + q * 32;
            uint32_t seen = (as_below(key_hi() - key) & ~as_below(key_lo() - key)) | as_below(cold[C_PREFIX] - key);
            if (DOCS && mod.docs != nullptr) {
              const int key_doc = q == 0 ? key_docs[0] : key_docs[1];
              uint32_t same = 0;
              if (one_doc >= 0) {
                same = __ballot_sync(0xffffffffu, key_doc == one_doc);
              } else {  // the keys of each document that some row of the warp belongs to
                uint32_t todo = __ballot_sync(0xffffffffu, doc >= 0);
                while (todo) {
                  const int d = __shfl_sync(0xffffffffu, doc, __ffs(todo) - 1);
                  const uint32_t keys = __ballot_sync(0xffffffffu, key_doc == d);
                  if (doc == d) same = keys;
                  todo &= ~__ballot_sync(0xffffffffu, doc == d);
                }
              }
              seen &= same;
            }
            return seen;
          };
          // O, and P of the first 32 keys when the second are at work, follow a reference that has moved (by a whole power of two: nothing
          // is rounded)
          auto rescale = [&](float alpha, bool p_too) {
            if (!__any_sync(0xffffffffu, alpha != 1.f)) return;
            if (!first) {
              if (!pv_wait(step - 1)) failed = true;
              tc_fence_after_sync();
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                tmem_ld_32x32b_x16(lanes + Cfg::O(t) + c, o);
                tmem_ld_wait_for16(o);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                tmem_st_32x32b_x16(lanes + Cfg::O(t) + c, o);
              }
            }
            tmem_st_wait();
            if (p_too) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(s_at, o);
              tmem_ld_wait_for16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&o[i]));
                const __nv_bfloat162 h2 = __floats2bfloat162_rn(x.x * alpha, x.y * alpha);
                o[i] = *reinterpret_cast<const uint32_t*>(&h2);
              }
              tmem_st_32x32b_x16(s_at, o);
              tmem_st_wait();
            }
          };
          // probabilities of 32 keys, two to a register, and the sum of what the rounding left of them: the weights that reach O then add
          // up to one, and the rounding of a key that dominates its row cancels (error against 64 bits 0.0024 -> 0.0020 on an
          // indexing batch, 0.0017 of it the rounding of the output, for 3 % of the time)
          auto exponentials = [&](const float2 (&e2)[16], uint32_t (&pk)[16]) -> float {
            float2 sum = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const __nv_bfloat162 a = __floats2bfloat162_rn(as_ex2(e2[i].x), as_ex2(e2[i].y));
              const __nv_bfloat162 b = __floats2bfloat162_rn(as_ex2(e2[i + 1].x), as_ex2(e2[i + 1].y));
              pk[i] = *reinterpret_cast<const uint32_t*>(&a);
              pk[i + 1] = *reinterpret_cast<const uint32_t*>(&b);
              sum = __fadd2_rn(sum, make_float2(__uint_as_float(pk[i] << 16), __uint_as_float(pk[i] & 0xffff0000u)));
              sum1 = __fadd2_rn(sum1, make_float2(__uint_as_float(pk[i + 1] << 16), __uint_as_float(pk[i + 1] & 0xffff0000u)));
            }
            return (sum.x + sum1.x) + (sum.y + sum1.y);
          };
          // AS_BIAS, AS_DOCS, AS_ANY: 32 scores into exponents against the reference
          auto any_scores = [&](const uint32_t (&z)[32], int key32, float2 (&e2)[16]) {
            float y[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(z[i]);
            if (MODE == AS_ANY && cap_out > AS_CAP_HIGH) {
              // the cap multiplies the error: 2^-22 of one is 2^-16 of a score's unit at a cap of 55, and 0.24 of it at 1e6
#pragma unroll
              for (int i = 0; i < 32; ++i) y[i] = fmaf(cap_out, tanhf(y[i] * cap_in), -ref);
            } else if (MODE == AS_ANY && mod.cap > 0.f) {
#pragma unroll
              for (int i = 0; i < 32; ++i) y[i] = fmaf(cap_out, as_tanh(y[i] * cap_in), -ref);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) y[i] = fmaf(y[i], scale_log2, -ref);
            }
            const int d0 = key32 - pos;
            if (MODE == AS_ANY && mod.slopes != nullptr) {
              const float f = static_cast<float>(d0);
#pragma unroll
              for (int i = 0; i < 32; ++i) y[i] = fmaf(-slope, fabsf(f + static_cast<float>(i)), y[i]);
            }
            if (MODE == AS_BIAS || mod.bias != nullptr) {
              if (key32 + 31 - pos_first <= -mod.radius || key32 - pos_last >= mod.radius) {  // beyond the table for all rows
                const float b = tab[key32 < pos_last ? -mod.radius : mod.radius] * tab_unit;
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] += b;
              } else if (key32 - pos_last >= -mod.radius && key32 + 31 - pos_first <= mod.radius && real) {  // inside for all rows
                const float* from = tab + d0;
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = fmaf(from[i], tab_unit, y[i]);
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = fmaf(tab[min(max(d0 + i, -mod.radius), mod.radius)], tab_unit, y[i]);
              }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) e2[i] = make_float2(y[2 * i], y[2 * i + 1]);
          };
          // Most steps: every row sees all 64 keys, the reference stands, nothing is asked of a score one by one. What does not fit
          // (a sum out of range, a score beyond the cap) is taken again below, from the same scores. Steps within a bias
          // table's reach, documents and modifications together are left to the code below altogether: here they cost more in instructions
          // fetched than they save (documents with a table, 4 sequences of 2500 to 4096, 12 heads of 32: 171 us and 142; beyond the table
          // it pays: 8 of 2048, 28/4 heads of 128, radius 128: 1009 us without and 725).
          bool done = false;
          const bool left_of = kv0 + KV - 1 - pos_first <= -mod.radius, right_of = kv0 - pos_last >= mod.radius;  // AS_BIAS: beyond the table
          if (!DOCS && whole && (FIRST || !first) && (MODE != AS_SLOPES || kv0 + KV <= pos_first || kv0 > pos_last) &&
              (MODE != AS_BIAS || left_of || right_of)) {
            uint32_t z[2][32];
            tmem_ld_32x32b_x32(s_at, z[0]);
            tmem_ld_32x32b_x32(s_at + 32, z[1]);
            tmem_ld_wait_for(z[0]);
            tmem_ld_wait_for(z[1]);
            float2 e2[2][16];
            auto two = [&](int g2, int i) { return make_float2(__uint_as_float(z[g2][2 * i]), __uint_as_float(z[g2][2 * i + 1])); };
            bool odd = false;
            if (MODE == AS_PLAIN || MODE == AS_BIAS) {
              float base = -ref;
              if (MODE == AS_BIAS) base = fmaf(tab[left_of ? -mod.radius : mod.radius], tab_unit, base);
              const float2 base2 = make_float2(base, base);
#pragma unroll
              for (int i = 0; i < 32; ++i) e2[i >> 4][i & 15] = __ffma2_rn(two(i >> 4, i & 15), scale2, base2);
            } else if (MODE == AS_SLOPES) {
              const float f = static_cast<float>(kv0 - pos), rise = kv0 < pos_first ? slope : -slope;
              const float2 rise2 = make_float2(2.f * rise, 2.f * rise);
              float2 bias2 = make_float2(fmaf(rise, f, -ref), fmaf(rise, f + 1.f, -ref));
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                e2[i >> 4][i & 15] = __ffma2_rn(two(i >> 4, i & 15), scale2, bias2);
                bias2 = __fadd2_rn(bias2, rise2);
              }
            } else {
              float top = 0.f;
#pragma unroll
              for (int i = 0; i < 64; i += 2) top = as_max3_abs(top, __uint_as_float(z[i >> 5][i & 31]), __uint_as_float(z[i >> 5][(i & 31) + 1]));
              odd = odd || top > cap_far;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float2 v = __fmul2_rn(two(i >> 4, i & 15), scale2);
                e2[i >> 4][i & 15] = tanh_near(v, __fmul2_rn(v, v));
              }
            }
            if (FIRST && MODE != AS_CAP && first) {  // the reference, from these scores (nothing is summed yet)
              float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                m0 = as_max3(m0, e2[0][i].x, e2[0][i].y);
                m1 = as_max3(m1, e2[1][i].x, e2[1][i].y);
              }
              float by = ceilf(fmaxf(m0, m1));
              if (by == -INFINITY) by = 0.f;
              ref += by;
#pragma unroll
              for (int i = 0; i < 32; ++i) e2[i >> 4][i & 15] = __fadd2_rn(e2[i >> 4][i & 15], make_float2(-by, -by));
            }
            uint32_t pk[2][16];
            float total = exponentials(e2[0], pk[0]);
            total += exponentials(e2[1], pk[1]);
            const float sum_now = l_run + total;
            if (MODE != AS_CAP) odd = odd || !(sum_now >= AS_SUM_LOW && sum_now <= AS_SUM_HIGH);
            done = (__ballot_sync(0xffffffffu, odd) & real_rows) == 0u;
            if (done) {
              l_run = sum_now;
              tmem_st_32x32b_x16(s_at, pk[0]);
              tmem_st_32x32b_x16(s_at + 32, pk[1]);
            }
          }
          // 32 keys at a time: masks, the segment's first scores, references that move. (Kept small in registers: what spills from here is
          // a trip to L2 each, shared memory has taken all of L1.)
#pragma unroll 1
          for (int q = 0; !done && q * 32 < n_rem; ++q) {
            const int key32 = kv0 + q * 32;
            uint32_t seen = 0xffffffffu;
            if (!whole) seen = seen_of(q);
            if ((__ballot_sync(0xffffffffu, seen != 0u) & real_rows) == 0u && !(first && q == 0)) {  // no row of the warp sees one of them
              uint32_t none[16] = {};
              tmem_st_32x32b_x16(s_at + q * 32, none);
              continue;
            }
            bool moves = MODE != AS_CAP && first && q == 0 && real;  // the segment's first scores set the reference
            bool again = false;
            float total;
            uint32_t pk[16];
#pragma unroll 1
            while (true) {
              uint32_t z[32];
              tmem_ld_32x32b_x32(s_at + q * 32, z);
              tmem_ld_wait_for(z);
              const bool guess = MODE != AS_CAP && first && q == 0 && !again;
              float2 e2[16];  // exponents against the reference
              float mx = -INFINITY;
              auto two = [&](int i) { return make_float2(__uint_as_float(z[2 * i]), __uint_as_float(z[2 * i + 1])); };
              if (MODE == AS_SLOPES && guess) {
                // the first guess takes the bias of the step's nearest key, which later scores will not exceed by much
#pragma unroll
                for (int i = 0; i < 32; ++i) mx = fmaxf(mx, (seen >> i) & 1u ? __uint_as_float(z[i]) * scale_log2 : -INFINITY);
                mx -= slope * static_cast<float>(max(max(kv0 - pos, pos - (kv0 + n_valid - 1)), 0));
              }
              if (MODE == AS_PLAIN) {
                const float2 base2 = make_float2(-ref, -ref);
#pragma unroll
                for (int i = 0; i < 16; ++i) e2[i] = __ffma2_rn(two(i), scale2, base2);
              } else if (MODE == AS_SLOPES) {
                const float f = static_cast<float>(key32 - pos);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  e2[i] = __ffma2_rn(two(i), scale2, make_float2(fmaf(-slope, fabsf(f + static_cast<float>(2 * i)), -ref),
                                                                 fmaf(-slope, fabsf(f + static_cast<float>(2 * i + 1)), -ref)));
              } else if (MODE == AS_CAP) {
                // good for every score; the polynomial beside it for those within the cap costs more to fetch than it saves (8 sequences of 600
                // to 2048, 28/4 heads of 128, causal, window 1023: 209 us, 221 with both)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float2 v = two(i);
                  e2[i] = make_float2(cap_out * as_tanh(v.x * cap_in), cap_out * as_tanh(v.y * cap_in));
                }
              } else {
                any_scores(z, key32, e2);
              }
              if (!whole) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  if (!((seen >> (2 * i)) & 1u)) e2[i].x = -INFINITY;
                  if (!((seen >> (2 * i + 1)) & 1u)) e2[i].y = -INFINITY;
                }
              }
              if (MODE != AS_CAP && (guess || again)) {
                // The reference moves to the larger of these scores and the logarithm of the sum so far (which lies far below it where the
                // reference was a bad guess), by a whole number.
                if (MODE != AS_SLOPES || again) {
#pragma unroll
                  for (int i = 0; i < 16; ++i) mx = as_max3(mx, e2[i].x, e2[i].y);
                }
                float by = ceilf(fmaxf(mx, l_run > 0.f ? __log2f(l_run) : -INFINITY));
                if (!moves || by == -INFINITY) by = 0.f;
                const float alpha = l_run > 0.f ? as_ex2(-by) : by != 0.f ? l_run : 1.f;  // nothing summed: 0, and NaN stays NaN
                l_run *= alpha;
                ref += by;
#pragma unroll
                for (int i = 0; i < 16; ++i) e2[i] = __fadd2_rn(e2[i], make_float2(-by, -by));
                if (again) rescale(alpha, q != 0);
              }
              total = exponentials(e2, pk);
              if (again) break;
              // sums out of range
              const float sum_now = l_run + total;
              const bool bad = MODE != AS_CAP && seen != 0u && !(sum_now >= AS_SUM_LOW && sum_now <= AS_SUM_HIGH);
              if ((__ballot_sync(0xffffffffu, bad) & real_rows) == 0u) break;
              moves = bad && real;
              again = true;
            }
            if (failed) break;
            l_run += total;
            tmem_st_32x32b_x16(s_at + q * 32, pk);
          }
          if (failed) break;
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * t + buf]);
        } else {
          // nothing to compute: arrive in step with the warps that do
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * t + buf]);
        }
        first = false;
        ++step;
        kv0 = next_kv0;
      }
      if (failed) break;
      // ---- the segment's rows ----
      if (!pv_wait(step - 1)) failed = true;
      if (failed) break;
      tc_fence_after_sync();
      const int k_first = cold[C_K], n_tiles = cold[C_N], seg_h = cold[C_H], seg_e = cold[C_E], tok0 = cold[C_TOK0];
      if (k_first == 0 && i_end == n_tiles) {
        uint8_t* stage = stage_s + warp * AS_STAGE;
        if (active) {
          const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
#pragma unroll 1
          for (int c = 0; c < D && c < j.head_dim; c += 32) {
            uint32_t ra[32];
            tmem_ld_32x32b_x32(lanes + Cfg::O(t) + c, ra);
            tmem_ld_wait_for(ra);
            // 32 columns (64 bytes) of 16 rows at a time through shared memory, 16-byte pieces swizzled by row
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if ((lane >> 4) == half) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  uint4 x;
                  __nv_bfloat162 p0 = __floats2bfloat162_rn(__uint_as_float(ra[8 * i]) * inv, __uint_as_float(ra[8 * i + 1]) * inv);
                  __nv_bfloat162 p1 = __floats2bfloat162_rn(__uint_as_float(ra[8 * i + 2]) * inv, __uint_as_float(ra[8 * i + 3]) * inv);
                  __nv_bfloat162 p2 = __floats2bfloat162_rn(__uint_as_float(ra[8 * i + 4]) * inv, __uint_as_float(ra[8 * i + 5]) * inv);
                  __nv_bfloat162 p3 = __floats2bfloat162_rn(__uint_as_float(ra[8 * i + 6]) * inv, __uint_as_float(ra[8 * i + 7]) * inv);
                  x.x = *reinterpret_cast<uint32_t*>(&p0);
                  x.y = *reinterpret_cast<uint32_t*>(&p1);
                  x.z = *reinterpret_cast<uint32_t*>(&p2);
                  x.w = *reinterpret_cast<uint32_t*>(&p3);
                  if (inv == 0.f) x = make_uint4(0, 0, 0, 0);  // no key seen (the accumulator may hold 0 * NaN)
                  *reinterpret_cast<uint4*>(stage + (lane & 15) * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = x;
                }
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int rl = i * 8 + (lane >> 2), cc = lane & 3, r = wq * 32 + half * 16 + rl;
                const int col = c + cc * 8;
                if (r < n_rows && col < j.head_dim) {
                  const uint4 x = *reinterpret_cast<const uint4*>(stage + rl * 64 + ((cc ^ ((rl >> 1) & 3)) << 4));
                  const int tk = (r * j.group_inv) >> 16;
                  *reinterpret_cast<uint4*>(j.out + static_cast<int64_t>(tok0 + tk) * j.out_stride +
                                            static_cast<int64_t>(seg_h * j.group + r - tk * j.group) * j.head_dim + col) = x;
                }
              }
              __syncwarp();
            }
          }
        }
      } else {
        // A part: numerators, reference and denominator go to the workspace. Parts of an item: the one that starts it is the tail of
        // its slot (odd index), the others are the head of theirs (even).
        const int64_t id = part_of(my_slot, k_first == 0);
        if (real) plan.part_ml[id * plan.rows + row] = make_float2(ref, l_run);
        if (active) {
          // four columns of all rows lie together: neighbouring lanes write neighbouring 16 bytes
          float* dst = plan.part_o + (id * (D / 4) * plan.rows + row) * 4;
#pragma unroll 1
          for (int c = 0; c < D && c < j.head_dim; c += 32) {
            uint32_t ra[32];
            tmem_ld_32x32b_x32(lanes + Cfg::O(t) + c, ra);
            tmem_ld_wait_for(ra);
            if (real) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<uint4*>(dst + static_cast<int64_t>((c + i) / 4) * plan.rows * 4) = make_uint4(ra[i], ra[i + 1], ra[i + 2], ra[i + 3]);
            }
          }
        }
        // the item's steps, and the slots they lie in
        const int64_t before = plan.entry[seg_e].before;
        const int64_t from = before * j.n_kv_heads + static_cast<int64_t>(seg_h) * n_tiles, to = from + n_tiles;
        int s0 = my_slot, s1 = my_slot;
        while (plan.bound[s0] > from) --s0;
        while (plan.bound[s1 + 1] < to) ++s1;
        meet();  // the part is written; one fence publishes what the barrier has gathered
        if (failed) break;
        if (row == 0) {
          __threadfence();
          const int old = atomicAdd(&plan.counter[s0], 1);
          __threadfence();
          joins[t] = old == s1 - s0;
        }
        meet();
        if (failed) break;
        const bool join = joins[t] != 0;
        if (join) {
          const int pieces = j.head_dim >> 3;
          for (int i = row; i < n_rows * pieces; i += 128) {
            const int piece = i / n_rows, r = i - piece * n_rows, col = piece * 8;
            float top = -INFINITY, l = 0.f, o[8] = {};
            // four parts' reads at a time
#pragma unroll 4
            for (int s = s0; s <= s1; ++s) {
              const float2 ml = __ldcg(&plan.part_ml[part_of(s, s == s0) * plan.rows + r]);
              top = fmaxf(top, ml.y > 0.f ? ml.x + __log2f(ml.y) : -INFINITY);  // a reference alone may be far from its sum
            }
#pragma unroll 4
            for (int s = s0; s <= s1; ++s) {
              const int64_t id2 = part_of(s, s == s0);
              const float2 ml = __ldcg(&plan.part_ml[id2 * plan.rows + r]);
              const float* src = plan.part_o + ((id2 * (D / 4) + 2 * piece) * plan.rows + r) * 4;
              const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
              const float4 y = __ldcg(reinterpret_cast<const float4*>(src + static_cast<int64_t>(plan.rows) * 4));
              const float f = ml.y > 0.f ? as_ex2(ml.x - top) : ml.y;  // nothing seen: 0, and NaN stays NaN
              l = fmaf(f, ml.y, l);
              o[0] = fmaf(f, x.x, o[0]);
              o[1] = fmaf(f, x.y, o[1]);
              o[2] = fmaf(f, x.z, o[2]);
              o[3] = fmaf(f, x.w, o[3]);
              o[4] = fmaf(f, y.x, o[4]);
              o[5] = fmaf(f, y.y, o[5]);
              o[6] = fmaf(f, y.z, o[6]);
              o[7] = fmaf(f, y.w, o[7]);
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            uint4 x;
            __nv_bfloat162 p0 = __floats2bfloat162_rn(o[0] * inv, o[1] * inv), p1 = __floats2bfloat162_rn(o[2] * inv, o[3] * inv);
            __nv_bfloat162 p2 = __floats2bfloat162_rn(o[4] * inv, o[5] * inv), p3 = __floats2bfloat162_rn(o[6] * inv, o[7] * inv);
            x.x = *reinterpret_cast<uint32_t*>(&p0);
            x.y = *reinterpret_cast<uint32_t*>(&p1);
            x.z = *reinterpret_cast<uint32_t*>(&p2);
            x.w = *reinterpret_cast<uint32_t*>(&p3);
            if (inv == 0.f) x = make_uint4(0, 0, 0, 0);
            const int tk = (r * j.group_inv) >> 16;
            *reinterpret_cast<uint4*>(j.out + static_cast<int64_t>(tok0 + tk) * j.out_stride +
                                      static_cast<int64_t>(seg_h * j.group + r - tk * j.group) * j.head_dim + col) = x;
          }
        }
        meet();  // joins[t] may be written again
      }
      tc_fence_before_sync();  // O has been read: the next segment's first P V may overwrite it
      __syncwarp();
      if (lane == 0) {
        cold[C_LEFT] -= i_end - k_first;
        const bool over = i_end == n_tiles, head_over = over && seg_h + 1 == j.n_kv_heads;
        cold[C_K] = over ? 0 : i_end;
        cold[C_H] = head_over ? 0 : seg_h + (over ? 1 : 0);
        cold[C_E] = seg_e + (head_over ? 1 : 0);
      }
      __syncwarp();
    }
    if (failed && lane == 0) atomicExch(plan.status, 4);
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == AS_MMA_WARP) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, AS_TMEM_COLS);
  }
}

// ---- host side ----------------------------------------------------------------------

static int check_shape(int n_seqs, int n_tokens, int n_heads, int n_kv_heads, int head_dim, const char* who) {
  if (n_seqs < 0 || n_tokens < 0 || n_heads <= 0 || n_kv_heads <= 0)
    return set_error(B200EMB_ERR_INVALID, "%s: bad sizes", who);
  if (n_tokens > AS_MAX_POSITIONS) return set_error(B200EMB_ERR_UNSUPPORTED, "%s: more than %d tokens", who, AS_MAX_POSITIONS);
  if (n_heads % n_kv_heads != 0)
    return set_error(B200EMB_ERR_INVALID, "%s: %d query heads are no multiple of %d key heads", who, n_heads, n_kv_heads);
  if (n_heads / n_kv_heads > AS_MAX_GROUP)
    return set_error(B200EMB_ERR_UNSUPPORTED, "%s: more than %d query heads per key head", who, AS_MAX_GROUP);
  if (head_dim < 8 || head_dim > 128 || head_dim % 8 != 0)
    return set_error(B200EMB_ERR_UNSUPPORTED, "%s: head_dim %d is no multiple of 8 from 8 to 128", who, head_dim);
  return B200EMB_OK;
}

// Device form of the options (null: none, `causal` as given by the entry point).
static int make_mod(const b200emb_attn_opts* o, int head_dim, bool paged, const char* who, AttnMod* m) {
  *m = AttnMod{1.f / sqrtf(static_cast<float>(head_dim)), 0.f, INT_MAX, paged ? 0 : INT_MAX, 0, nullptr, nullptr, nullptr, nullptr};
  if (o == nullptr) return B200EMB_OK;
  if (!isfinite(o->scale * AS_LOG2E) || !isfinite(o->cap * AS_LOG2E) || o->cap < 0.f)  // both in the units of the exponent
    return set_error(B200EMB_ERR_INVALID, "%s: scale and cap must be finite and at most 2e38, cap not negative", who);
  if (o->causal != 0 && o->causal != 1) return set_error(B200EMB_ERR_INVALID, "%s: causal must be 0 or 1", who);
  if (o->causal == 1 && o->window_right > 0)
    return set_error(B200EMB_ERR_INVALID, "%s: causal together with window_right %d", who, o->window_right);
  if (o->slopes != nullptr && o->bias != nullptr)
    return set_error(B200EMB_ERR_INVALID, "%s: slopes together with a bias table", who);
  if (o->bias_radius < 0 || o->bias_radius > AS_MAX_RADIUS)
    return set_error(B200EMB_ERR_UNSUPPORTED, "%s: bias_radius %d outside 0 .. %d", who, o->bias_radius, AS_MAX_RADIUS);
  if (paged && o->doc_ids != nullptr) return set_error(B200EMB_ERR_INVALID, "%s: doc_ids need the packed call", who);
  for (int i = 0; i < 4; ++i)
    if (o->reserved[i] != 0) return set_error(B200EMB_ERR_INVALID, "%s: reserved fields must be zero", who);
  if (o->scale != 0.f) m->scale = o->scale;
  m->cap = o->cap;
  if (o->window_left >= 0) m->left = o->window_left;
  m->right = o->causal == 1 ? 0 : o->window_right >= 0 ? o->window_right : INT_MAX;
  m->radius = o->bias_radius;
  m->slopes = o->slopes;
  m->bias = o->bias;
  m->prefix = o->prefix_lens;
  m->docs = o->doc_ids;
  return B200EMB_OK;
}

static int check_rows(const void* p, int64_t stride, int64_t width, const char* name, const char* who) {
  if (p == nullptr) return set_error(B200EMB_ERR_INVALID, "%s: null pointer %s", who, name);
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || stride % 8 != 0)
    return set_error(B200EMB_ERR_INVALID, "%s: %s must be 16-byte aligned with a row stride that is a multiple of 8", who, name);
  if (stride < width) return set_error(B200EMB_ERR_INVALID, "%s: the row stride of %s is smaller than its heads", who, name);
  return B200EMB_OK;
}

static int check_workspace(const void* ws, int64_t have, int64_t want, const char* who) {
  if (ws == nullptr || reinterpret_cast<uintptr_t>(ws) % AS_ALIGN != 0)
    return set_error(B200EMB_ERR_INVALID, "%s: the workspace must be 256-byte aligned device memory", who);
  if (have < want)
    return set_error(B200EMB_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", who, static_cast<long long>(have),
                     static_cast<long long>(want));
  return B200EMB_OK;
}

// A call without rows launches nothing: it clears what an earlier call, or whatever used the memory before, left in the status word at
// the start of the workspace. A workspace that is not device memory is left alone, as such a call leaves all its pointers.
static int as_clear_status(void* workspace, int64_t bytes, cudaStream_t s) {
  if (workspace == nullptr || bytes < static_cast<int64_t>(sizeof(int32_t))) return B200EMB_OK;
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, workspace) != cudaSuccess) {
    cudaGetLastError();  // not a pointer of this process's devices, or no device at all: nobody's error
    return B200EMB_OK;
  }
  if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) return B200EMB_OK;
  B2_CUDA_CHECK(cudaMemsetAsync(workspace, 0, sizeof(int32_t), s));
  return B200EMB_OK;
}

static int as_tile_tokens(int n_heads, int n_kv_heads) { return 128 / (n_heads / n_kv_heads); }

// Carves the workspace (null: only measures it); returns its size.
static int64_t as_layout(void* workspace, int n_seqs, int n_tokens, int n_heads, int n_kv_heads, int head_dim, AttnPlan* p) {
  const int64_t seqs = n_seqs, tokens = n_tokens;
  const int group = n_heads / n_kv_heads, tile = as_tile_tokens(n_heads, n_kv_heads);
  const int64_t entries = tokens / tile + seqs + 1;
  const int64_t rows = (tokens < tile ? (tokens > 0 ? tokens : 1) : tile) * group;
  const int64_t parts = 2 * AS_MAX_SLOTS, dp = head_dim <= 64 ? 64 : 128;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t mine = at;
    at += (bytes + AS_ALIGN - 1) / AS_ALIGN * AS_ALIGN;
    return static_cast<char*>(workspace) + mine;
  };
  AttnPlan q = {};
  q.status = reinterpret_cast<int32_t*>(take(sizeof(int32_t)));
  q.bound = reinterpret_cast<int64_t*>(take((AS_MAX_SLOTS + 1) * sizeof(int64_t)));
  q.slot = reinterpret_cast<AttnSlot*>(take(AS_MAX_SLOTS * sizeof(AttnSlot)));
  q.counter = reinterpret_cast<int32_t*>(take(AS_MAX_SLOTS * sizeof(int32_t)));
  q.seq_first = reinterpret_cast<int32_t*>(take((seqs + 1) * sizeof(int32_t)));
  q.doc_range = reinterpret_cast<int2*>(take((tokens / 64 + seqs + 1) * sizeof(int2)));
  q.entry = reinterpret_cast<AttnEntry*>(take(entries * sizeof(AttnEntry)));
  q.part_ml = reinterpret_cast<float2*>(take(parts * rows * sizeof(float2)));
  q.part_o = reinterpret_cast<float*>(take(parts * rows * dp * sizeof(float)));
  q.max_entries = static_cast<int32_t>(entries < INT_MAX ? entries : INT_MAX);
  q.rows = static_cast<int32_t>(rows);
  if (p != nullptr) *p = q;
  return at;
}

struct AsMaps {
  CUtensorMap q, k, v;
};

struct AsDevice {
  int id, sms;
};

// Opt-in shared memory of one kernel, at its first launch on a device: setting it loads the kernel, and who never launches one of the 22 is
// not to wait for it (all of them at the library's first call: see kernels_init_device, which leaves them out).
template <int D, bool PAGED, int MODE>
static int as_init_kernel(int device) {
  static std::atomic<uint64_t> ready{0};
  const uint64_t bit = device >= 0 && device < 64 ? uint64_t(1) << device : 0;
  if (ready.load(std::memory_order_acquire) & bit) return B200EMB_OK;
  B2_CUDA_CHECK(cudaFuncSetAttribute(attn_scored_kernel<D, PAGED, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, AsCfg<D>::SMEM_BYTES));
  ready.fetch_or(bit, std::memory_order_release);
  return B200EMB_OK;
}

template <int D, bool PAGED, int MODE>
static int as_launch(const AsMaps& m, const AttnJob& j, const AttnMod& mod, const AttnPlan& plan, const AsDevice& dev, cudaStream_t s) {
  const int rc = as_init_kernel<D, PAGED, MODE>(dev.id);
  if (rc) return rc;
  int64_t grid = dev.sms < AS_MAX_CTAS ? dev.sms : AS_MAX_CTAS;
  if (!PAGED) {  // no more CTAs than steps there can be
    const int64_t steps = static_cast<int64_t>(plan.max_entries) * j.n_kv_heads * ((j.n_tokens + AsCfg<D>::KV - 1) / AsCfg<D>::KV);
    if (steps < grid) grid = steps;
  }
  const int slots = static_cast<int>(2 * grid);
  // few entries are planned by fewer threads: their barriers are what it takes
  const int threads = plan.max_entries <= 256 && j.n_seqs <= 256 && mod.docs == nullptr ? 256 : AS_PLAN_THREADS;
  cudaError_t e = launch_pdl(attn_plan_kernel, dim3(1), dim3(threads), 0, s, j, mod, plan, j.tile_tokens, slots, AsCfg<D>::KV);
  if (e == cudaSuccess)
    e = launch_pdl(attn_scored_kernel<D, PAGED, MODE>, dim3(static_cast<unsigned>(grid)), dim3(AS_THREADS), AsCfg<D>::SMEM_BYTES, s, m.q, m.k,
                   m.v, j, mod, plan);
  if (e != cudaSuccess) return set_error(B200EMB_ERR_CUDA, "attention launch: %s", cudaGetErrorString(e));
  return B200EMB_OK;
}

// rows of n heads: [tokens, heads, head_dim] with a row stride
static int as_map_rows(CUtensorMap* m, const void* base, int n_tokens, int heads, int head_dim, int64_t stride, int box_heads, int box_tokens) {
  const uint64_t dims[3] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(heads), static_cast<uint64_t>(n_tokens)};
  const uint64_t strides[2] = {static_cast<uint64_t>(head_dim) * 2, static_cast<uint64_t>(stride) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(box_heads), static_cast<uint32_t>(box_tokens)};
  return encode_tmap_bf16(m, base, 3, dims, strides, box);
}

static int as_map_pages(CUtensorMap* m, const void* base, const b200emb_kv_cache& c, bool head_first, int box_rows) {
  // a dimension of one element may have any stride: give it one the encoder takes
  const uint64_t ts = static_cast<uint64_t>(c.token_stride) * 2, hs = static_cast<uint64_t>(c.n_kv_heads > 1 ? c.head_stride : c.token_stride) * 2;
  const uint64_t ps = c.n_pages > 1 ? static_cast<uint64_t>(c.page_stride) * 2 : ts * c.page_size;
  const uint64_t heads = c.n_kv_heads, page = c.page_size;
  const uint64_t dims[4] = {static_cast<uint64_t>(c.head_dim), head_first ? heads : page, head_first ? page : heads, static_cast<uint64_t>(c.n_pages)};
  const uint64_t strides[3] = {head_first ? hs : ts, head_first ? ts : hs, ps};
  const uint32_t rows = box_rows, box[4] = {64, head_first ? 1u : rows, head_first ? rows : 1u, 1};
  return encode_tmap_bf16(m, base, 4, dims, strides, box);
}

template <int D, bool PAGED>
static int as_launch_mode(const AsMaps& m, const AttnJob& j, const AttnMod& mod, const AttnPlan& plan, const AsDevice& dev, cudaStream_t s) {
  if constexpr (!PAGED)
    if (mod.docs != nullptr)
      return mod.cap == 0.f && mod.slopes == nullptr ? as_launch<D, PAGED, AS_DOCS>(m, j, mod, plan, dev, s)
                                                     : as_launch<D, PAGED, AS_ANY>(m, j, mod, plan, dev, s);
  if (mod.cap == 0.f) {
    if (mod.slopes != nullptr) return as_launch<D, PAGED, AS_SLOPES>(m, j, mod, plan, dev, s);
    return mod.bias != nullptr ? as_launch<D, PAGED, AS_BIAS>(m, j, mod, plan, dev, s) : as_launch<D, PAGED, AS_PLAIN>(m, j, mod, plan, dev, s);
  }
  const float cap = mod.cap * AS_LOG2E;
  if (cap >= AS_CAP_LOW && cap <= AS_CAP_HIGH && mod.slopes == nullptr && mod.bias == nullptr)
    return as_launch<D, PAGED, AS_CAP>(m, j, mod, plan, dev, s);
  return as_launch<D, PAGED, AS_ANY>(m, j, mod, plan, dev, s);
}

template <bool PAGED>
static int as_dispatch(const AsMaps& m, const AttnJob& j, const AttnMod& mod, void* workspace, cudaStream_t s) {
  AsDevice dev = {};
  B2_CUDA_CHECK(cudaGetDevice(&dev.id));
  B2_CUDA_CHECK(cudaDeviceGetAttribute(&dev.sms, cudaDevAttrMultiProcessorCount, dev.id));
  AttnPlan plan;
  as_layout(workspace, j.n_seqs, j.n_tokens, j.n_heads, j.n_kv_heads, j.head_dim, &plan);
  return j.head_dim <= 64 ? as_launch_mode<64, PAGED>(m, j, mod, plan, dev, s) : as_launch_mode<128, PAGED>(m, j, mod, plan, dev, s);
}

}  // namespace b2

using namespace b2;

extern "C" int64_t b200emb_attention_workspace_bytes(int32_t n_seqs, int32_t n_tokens, int32_t n_heads, int32_t n_kv_heads,
                                                     int32_t head_dim) {
  const int rc = check_shape(n_seqs, n_tokens, n_heads, n_kv_heads, head_dim, "attention_workspace_bytes");
  return rc ? rc : as_layout(nullptr, n_seqs, n_tokens, n_heads, n_kv_heads, head_dim, nullptr);
}

extern "C" int b200emb_op_workspace_status(const void* workspace, void* stream) {
  if (workspace == nullptr) return set_error(B200EMB_ERR_INVALID, "workspace_status: null pointer");
  int herr = 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  B2_CUDA_CHECK(cudaMemcpyAsync(&herr, workspace, sizeof(int), cudaMemcpyDeviceToHost, s));
  B2_CUDA_CHECK(cudaStreamSynchronize(s));
  if (herr != 0) return set_error(B200EMB_ERR_DEVICE_WAIT, "attention: a device-side wait gave up (role %d)", herr);
  return B200EMB_OK;
}

extern "C" int b200emb_op_attention_scored(const void* q, int64_t q_row_stride, const void* k, int64_t k_row_stride, const void* v,
                                           int64_t v_row_stride, void* out, int64_t out_row_stride, const int32_t* d_cu_seqlens,
                                           int32_t n_seqs, int32_t n_tokens, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                           const b200emb_attn_opts* opts, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "attention_scored";
  int rc = check_shape(n_seqs, n_tokens, n_heads, n_kv_heads, head_dim, who);
  AttnMod mod;
  if (!rc) rc = make_mod(opts, head_dim, false, who, &mod);
  if (rc) return rc;
  if (n_tokens == 0 || n_seqs == 0) return as_clear_status(workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
  const int64_t wq = static_cast<int64_t>(n_heads) * head_dim, wk = static_cast<int64_t>(n_kv_heads) * head_dim;
  rc = check_rows(q, q_row_stride, wq, "q", who);
  if (!rc) rc = check_rows(k, k_row_stride, wk, "k", who);
  if (!rc) rc = check_rows(v, v_row_stride, wk, "v", who);
  if (!rc) rc = check_rows(out, out_row_stride, wq, "out", who);
  if (!rc && d_cu_seqlens == nullptr) rc = set_error(B200EMB_ERR_INVALID, "%s: null pointer cu_seqlens", who);
  if (!rc) rc = check_workspace(workspace, workspace_bytes, b200emb_attention_workspace_bytes(n_seqs, n_tokens, n_heads, n_kv_heads, head_dim), who);
  if (rc) return rc;
  AttnJob j = {};
  j.out = static_cast<__nv_bfloat16*>(out);
  j.out_stride = out_row_stride;
  j.cu = d_cu_seqlens;
  j.n_seqs = n_seqs;
  j.n_tokens = n_tokens;
  j.n_heads = n_heads;
  j.n_kv_heads = n_kv_heads;
  j.head_dim = head_dim;
  j.group = n_heads / n_kv_heads;
  j.group_inv = (65536 + j.group - 1) / j.group;
  j.tile_tokens = as_tile_tokens(n_heads, n_kv_heads);
  j.box_rows = AS_PACKED_BOX;
  AsMaps m;
  rc = as_map_rows(&m.q, q, n_tokens, n_heads, head_dim, q_row_stride, j.group, j.tile_tokens);
  if (!rc) rc = as_map_rows(&m.k, k, n_tokens, n_kv_heads, head_dim, k_row_stride, 1, AS_PACKED_BOX);
  if (!rc) rc = as_map_rows(&m.v, v, n_tokens, n_kv_heads, head_dim, v_row_stride, 1, AS_PACKED_BOX);
  return rc ? rc : as_dispatch<false>(m, j, mod, workspace, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int b200emb_op_attention_paged(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride,
                                          const int32_t* d_cu_seqlens, const int32_t* d_kv_lens, int32_t n_seqs, int32_t n_tokens,
                                          int32_t n_heads, const b200emb_kv_cache* cache, const b200emb_attn_opts* opts,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "attention_paged";
  int rc = check_kv_cache(cache, who);
  if (!rc) rc = check_shape(n_seqs, n_tokens, n_heads, cache->n_kv_heads, cache->head_dim, who);
  AttnMod mod;
  if (!rc) rc = make_mod(opts, cache->head_dim, true, who, &mod);
  if (rc) return rc;
  if (static_cast<int64_t>(cache->table_stride) * cache->page_size > AS_MAX_POSITIONS)
    return set_error(B200EMB_ERR_UNSUPPORTED, "%s: a page table of more than %d positions", who, AS_MAX_POSITIONS);
  if (cache->page_size % 8 != 0)
    return set_error(B200EMB_ERR_UNSUPPORTED, "%s: page_size %d is no multiple of 8", who, cache->page_size);
  if (cache->page_stride % 8 != 0 || cache->token_stride % 8 != 0 || cache->head_stride % 8 != 0 ||
      reinterpret_cast<uintptr_t>(cache->k) % 16 != 0 || reinterpret_cast<uintptr_t>(cache->v) % 16 != 0)
    return set_error(B200EMB_ERR_INVALID, "%s: the cache must be 16-byte aligned with strides that are multiples of 8", who);
  if (n_tokens == 0 || n_seqs == 0) return as_clear_status(workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
  const int64_t wq = static_cast<int64_t>(n_heads) * cache->head_dim;
  rc = check_rows(q, q_row_stride, wq, "q", who);
  if (!rc) rc = check_rows(out, out_row_stride, wq, "out", who);
  if (!rc && (d_cu_seqlens == nullptr || d_kv_lens == nullptr))
    rc = set_error(B200EMB_ERR_INVALID, "%s: null pointer cu_seqlens or kv_lens", who);
  if (!rc)
    rc = check_workspace(workspace, workspace_bytes,
                         b200emb_attention_workspace_bytes(n_seqs, n_tokens, n_heads, cache->n_kv_heads, cache->head_dim), who);
  if (rc) return rc;
  AttnJob j = {};
  j.out = static_cast<__nv_bfloat16*>(out);
  j.out_stride = out_row_stride;
  j.cu = d_cu_seqlens;
  j.kv_lens = d_kv_lens;
  j.page_table = cache->page_table;
  j.n_seqs = n_seqs;
  j.n_tokens = n_tokens;
  j.n_heads = n_heads;
  j.n_kv_heads = cache->n_kv_heads;
  j.head_dim = cache->head_dim;
  j.group = n_heads / cache->n_kv_heads;
  j.group_inv = (65536 + j.group - 1) / j.group;
  j.tile_tokens = as_tile_tokens(n_heads, cache->n_kv_heads);
  j.n_pages = cache->n_pages;
  j.page_size = cache->page_size;
  j.table_stride = cache->table_stride;
  j.head_first = cache->head_stride <= cache->token_stride;
  // rows of one copy: as many as divide both a page and a key tile
  j.box_rows = AsCfg<128>::KV;
  while (cache->page_size % j.box_rows != 0) j.box_rows >>= 1;
  AsMaps m;
  rc = as_map_rows(&m.q, q, n_tokens, n_heads, cache->head_dim, q_row_stride, j.group, j.tile_tokens);
  if (!rc) rc = as_map_pages(&m.k, cache->k, *cache, j.head_first != 0, j.box_rows);
  if (!rc) rc = as_map_pages(&m.v, cache->v, *cache, j.head_first != 0, j.box_rows);
  return rc ? rc : as_dispatch<true>(m, j, mod, workspace, reinterpret_cast<cudaStream_t>(stream));
}
