// Rotary positions as an operator, and the paged-cache append that rotates on the way.
//
// Pair (u, v) of a head turns by a = position * w_i: (u cos a - v sin a, v cos a + u sin a). The host turns the descriptor
// into one fp64 angle per position for each pair (at most 128) and passes them by value; a block forms the angles of
// its token in fp64, reduces them to [-pi, pi] there (a position of 1e6 times w_0 = 1 has lost 4 digits in fp32 before the
// cosine is taken), and keeps cos and sin in shared memory for all heads of the token.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kernels.h"

namespace b2 {

static constexpr int ROPE_MAX_PAIRS = 128;
static constexpr int ROPE_MAX_THREADS = 128;

struct RopeParams {
  double w[ROPE_MAX_PAIRS];  // angle per position of pair i
  float magnitude;           // factor on cos and sin
  float sign;                // -1: rotate back
  int n_pairs;               // 0: nothing is rotated
  int interleaved;
};

// Where the rotated (and, for the append, the copied) heads of a token go.
struct RopeJob {
  const __nv_bfloat16* x;
  int64_t x_stride;
  __nv_bfloat16* q_out;  // heads [0, n_out_heads) of a row; null: these heads are skipped
  int64_t q_stride;
  const int32_t* positions;
  const int32_t* cu;
  const int32_t* pos_start;  // rope: position of the first token (nullable); append: keys including the new tokens
  int n_seqs, n_tokens, n_out_heads, head_dim;
  // append only
  __nv_bfloat16* k;
  __nv_bfloat16* v;
  const int32_t* page_table;
  int64_t page_stride, token_stride, head_stride;
  int n_pages, page_size, n_kv_heads, table_stride;
  // set at launch, for the chosen V
  int n_rot_heads, first_head, rot_items, per_head, turned, items;
};

// Sequence of token t: the last s with cu[s] <= t (empty sequences share a start; the last of them owns the token). The warp looks
// at 32 starts at a time: two dependent reads for up to 1024 sequences.
__device__ __forceinline__ int sequence_of(const int32_t* __restrict__ cu, int n_seqs, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = n_seqs;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const bool in = lane * step < n;
    const int below = __popc(__ballot_sync(0xffffffffu, in && __ldg(cu + lo + lane * step) <= t));
    const int at = max(below - 1, 0) * step;
    lo += at;
    n = min(step, n - at);
  }
  return lo;
}

template <int V>
struct Vec;
template <>
struct Vec<8> {
  using T = uint4;
};
template <>
struct Vec<4> {
  using T = uint2;
};
template <>
struct Vec<2> {
  using T = uint32_t;
};
template <>
struct Vec<1> {
  using T = uint16_t;
};

template <int V>
union Pack {
  typename Vec<V>::T raw;
  __nv_bfloat16 e[V];
  __device__ Pack() {}
};

// One block per token. An item is V elements of the interleaved layout or of a part that passes through, or V elements of the
// first half together with the V they pair with. A thread asks for its item before the block works out its position and angles, so that
// the row is on its way meanwhile. Reading and writing the row once is all the kernel cannot do without; what bounds it is instructions
// (76 % of the issue slots with 512 threads a block), so a block is small: the search, the angles and the barrier are paid by every
// warp of it. 19 506 tokens of 32 heads of 128, half of each turned (320 MB, 49 us at the copy rate): 62 us with 64 or 128 threads, 66 with
// 256, 80 with 512; 94 us where 256 threads read after the angles; 111 us and more with blocks that stay and ask a token ahead. Keys and
// values of 8 483 tokens into their pages (156 MB, 24 us): 37 us.
template <int V, bool APPEND>
__global__ void __launch_bounds__(ROPE_MAX_THREADS) rope_kernel_op(const __grid_constant__ RopeParams p, const __grid_constant__ RopeJob j) {
  __shared__ float2 cs[ROPE_MAX_PAIRS];
  using T = typename Vec<V>::T;
  const int t = blockIdx.x;
  const int hd = j.head_dim;
  const int turned = j.turned, items = j.items;  // items of heads that turn, and with those of the values
  const __nv_bfloat16* row = j.x + static_cast<int64_t>(t) * j.x_stride;
  Pack<V> a, b;
  int head = 0, e = 0, kind = 0;  // head of the row, first element of it, and 0 copied, 1 interleaved, 2 halves
  auto fetch = [&](int w) {
    if (APPEND && w >= turned) {
      const int vecs = hd / V;
      head = (w - turned) / vecs;
      e = (w - turned - head * vecs) * V;
      head += j.n_rot_heads;
      kind = 0;
    } else {
      head = w / j.per_head;
      const int g = w - head * j.per_head;
      head += j.first_head;
      const bool turns = g < j.rot_items;
      e = turns ? g * V : 2 * p.n_pairs + (g - j.rot_items) * V;
      kind = !turns ? 0 : p.interleaved ? 1 : 2;
    }
    const __nv_bfloat16* src = row + static_cast<int64_t>(head) * hd + e;
    a.raw = *reinterpret_cast<const T*>(src);
    if (kind == 2) b.raw = *reinterpret_cast<const T*>(src + p.n_pairs);
    if (V == 1 && kind == 1 && (e & 1) == 0) b.raw = *reinterpret_cast<const T*>(src + 1);
  };
  if (threadIdx.x < items) fetch(threadIdx.x);

  int pos, seq = 0;
  if (!APPEND && j.positions != nullptr) {
    pos = __ldg(j.positions + t);
  } else {
    seq = sequence_of(j.cu, j.n_seqs, t);
    const int first = __ldg(j.cu + seq), end = __ldg(j.cu + seq + 1);
    if (t < first || t >= end) return;  // a row that belongs to no sequence
    if (APPEND) pos = __ldg(j.pos_start + seq) - (end - first) + (t - first);
    else pos = (j.pos_start != nullptr ? __ldg(j.pos_start + seq) : 0) + (t - first);
  }
  // the page slot of this token; a slot that does not exist is not written
  int64_t slot = -1;
  if (APPEND && pos >= 0 && pos / j.page_size < j.table_stride) {
    const int page = __ldg(j.page_table + static_cast<int64_t>(seq) * j.table_stride + pos / j.page_size);
    if (page >= 0 && page < j.n_pages)
      slot = static_cast<int64_t>(page) * j.page_stride + static_cast<int64_t>(pos % j.page_size) * j.token_stride;
  }
  for (int i = threadIdx.x; i < p.n_pairs; i += blockDim.x) {
    const double angle = static_cast<double>(pos) * p.w[i];
    const double turns = rint(angle * 0.15915494309189535);      // 1 / (2 pi)
    double r = fma(-turns, 6.283185307179586, angle);            // 2 pi, high part
    r = fma(-turns, 2.4492935982947064e-16, r);                  // and what the high part leaves
    float s, c;
    sincosf(static_cast<float>(r), &s, &c);
    cs[i] = make_float2(c * p.magnitude, s * p.magnitude * p.sign);
  }
  __syncthreads();

  for (int w = threadIdx.x; w < items; w += blockDim.x) {
    if (w != threadIdx.x) fetch(w);
    __nv_bfloat16* dst;
    if (!APPEND || head < j.n_out_heads) dst = j.q_out + static_cast<int64_t>(t) * j.q_stride + static_cast<int64_t>(head) * hd + e;
    else if (slot < 0) continue;
    else if (head < j.n_rot_heads) dst = j.k + slot + (head - j.n_out_heads) * j.head_stride + e;
    else dst = j.v + slot + (head - j.n_rot_heads) * j.head_stride + e;
    if (kind == 2) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 c = cs[e + k];
        const float u = __bfloat162float(a.e[k]), v = __bfloat162float(b.e[k]);
        a.e[k] = __float2bfloat16_rn(u * c.x - v * c.y);
        b.e[k] = __float2bfloat16_rn(v * c.x + u * c.y);
      }
      *reinterpret_cast<T*>(dst + p.n_pairs) = b.raw;
    } else if (kind == 1) {
      if constexpr (V > 1) {
#pragma unroll
        for (int k = 0; k < V; k += 2) {
          const float2 c = cs[(e + k) >> 1];
          const float u = __bfloat162float(a.e[k]), v = __bfloat162float(a.e[k + 1]);
          a.e[k] = __float2bfloat16_rn(u * c.x - v * c.y);
          a.e[k + 1] = __float2bfloat16_rn(v * c.x + u * c.y);
        }
      } else {  // the even element's thread turns the pair
        if (e & 1) continue;
        const float2 c = cs[e >> 1];
        const float u = __bfloat162float(a.e[0]), v = __bfloat162float(b.e[0]);
        a.e[0] = __float2bfloat16_rn(u * c.x - v * c.y);
        b.e[0] = __float2bfloat16_rn(v * c.x + u * c.y);
        *reinterpret_cast<T*>(dst + 1) = b.raw;
      }
    }
    *reinterpret_cast<T*>(dst) = a.raw;
  }
}

// Fills the per-pair angles from the descriptor (null: nothing rotates).
static int rope_params(const b200emb_rope_desc* d, int head_dim, RopeParams* p) {
  p->magnitude = 1.f;
  p->sign = 1.f;
  p->n_pairs = 0;
  p->interleaved = 0;
  if (d == nullptr) return B200EMB_OK;
  if (d->rot_dim < 2 || d->rot_dim % 2 || d->rot_dim > 2 * ROPE_MAX_PAIRS || d->rot_dim > head_dim)
    return set_error(B200EMB_ERR_INVALID, "rope: rot_dim %d must be even, 2 .. %d and at most head_dim %d", d->rot_dim,
                     2 * ROPE_MAX_PAIRS, head_dim);
  if (d->layout != B200EMB_ROPE_HALF && d->layout != B200EMB_ROPE_INTERLEAVED)
    return set_error(B200EMB_ERR_INVALID, "rope: unknown layout %d", d->layout);
  if (d->scaling < B200EMB_ROPE_SCALE_NONE || d->scaling > B200EMB_ROPE_SCALE_YARN)
    return set_error(B200EMB_ERR_INVALID, "rope: unknown scaling %d", d->scaling);
  if (!(d->theta > 0.f) || !isfinite(d->theta)) return set_error(B200EMB_ERR_INVALID, "rope: theta must be positive and finite");
  if (d->scaling != B200EMB_ROPE_SCALE_NONE && (!(d->factor > 0.f) || !isfinite(d->factor)))
    return set_error(B200EMB_ERR_INVALID, "rope: factor must be positive and finite");
  if (d->inverse != 0 && d->inverse != 1) return set_error(B200EMB_ERR_INVALID, "rope: inverse must be 0 or 1");
  if (!isfinite(d->magnitude) || d->magnitude < 0.f) return set_error(B200EMB_ERR_INVALID, "rope: magnitude must be finite and not negative");
  for (int i = 0; i < 6; ++i)
    if (d->reserved[i] != 0) return set_error(B200EMB_ERR_INVALID, "rope: reserved fields must be zero");
  const int r = d->rot_dim;
  const double f = d->factor, low = d->low, high = d->high, trained = d->original_max_pos;
  double theta = d->theta;
  double from = 0.0, to = 0.0;  // YaRN ramp
  const double two_pi = 6.283185307179586;
  if (d->scaling == B200EMB_ROPE_SCALE_NTK) {
    if (r <= 2) return set_error(B200EMB_ERR_INVALID, "rope: NTK scaling needs rot_dim > 2");
    theta *= pow(f, r / (r - 2.0));
  } else if (d->scaling == B200EMB_ROPE_SCALE_BANDS) {
    if (d->original_max_pos <= 0 || !(low >= 0.0) || !(high > low) || !isfinite(high))
      return set_error(B200EMB_ERR_INVALID, "rope: bands need original_max_pos > 0 and 0 <= low < high");
  } else if (d->scaling == B200EMB_ROPE_SCALE_YARN) {
    if (d->original_max_pos <= 0 || !(high > 0.0) || !(low >= high) || !isfinite(low) || theta == 1.0)
      return set_error(B200EMB_ERR_INVALID, "rope: YaRN needs original_max_pos > 0, 0 < high <= low and theta != 1");
    const double per = r / (2.0 * log(theta));
    from = fmax(0.0, floor(per * log(trained / (two_pi * low))));
    to = fmin(r - 1.0, ceil(per * log(trained / (two_pi * high))));
  }
  const double step = -2.0 * log(theta) / r;
  for (int i = 0; i < r / 2; ++i) {
    double w = exp(step * i);
    if (d->scaling == B200EMB_ROPE_SCALE_LINEAR) {
      w /= f;
    } else if (d->scaling == B200EMB_ROPE_SCALE_BANDS) {
      const double k = fmin(1.0, fmax(0.0, (trained * w / two_pi - low) / (high - low)));
      w = w * k + w / f * (1.0 - k);
    } else if (d->scaling == B200EMB_ROPE_SCALE_YARN) {
      const double k = fmin(1.0, fmax(0.0, (i - from) / fmax(to - from, 1e-3)));
      w = w * (1.0 - k) + w / f * k;
    }
    p->w[i] = w;
  }
  p->n_pairs = r / 2;
  p->interleaved = d->layout == B200EMB_ROPE_INTERLEAVED;
  p->sign = d->inverse ? -1.f : 1.f;
  if (d->magnitude > 0.f) p->magnitude = d->magnitude;
  else if (d->scaling == B200EMB_ROPE_SCALE_YARN) p->magnitude = static_cast<float>(0.1 * log(fmax(f, 1.0)) + 1.0);
  return B200EMB_OK;
}

// Elements per access: the widest that every row, head and half starts on.
static int rope_vector(const RopeParams& p, const RopeJob& j, bool append) {
  uint64_t elems = static_cast<uint64_t>(j.head_dim) | static_cast<uint64_t>(j.x_stride) |
                   static_cast<uint64_t>(p.interleaved ? 2 * p.n_pairs : p.n_pairs);
  uint64_t bytes = reinterpret_cast<uintptr_t>(j.x);
  if (j.q_out != nullptr) {
    elems |= static_cast<uint64_t>(j.q_stride);
    bytes |= reinterpret_cast<uintptr_t>(j.q_out);
  }
  if (append) {
    elems |= static_cast<uint64_t>(j.page_stride) | static_cast<uint64_t>(j.token_stride) | static_cast<uint64_t>(j.head_stride);
    bytes |= reinterpret_cast<uintptr_t>(j.k) | reinterpret_cast<uintptr_t>(j.v);
  }
  for (int v = 8; v > 1; v >>= 1)
    if (elems % v == 0 && bytes % (2 * v) == 0) return v;
  return 1;
}

template <int V, bool APPEND>
static int rope_launch_v(const RopeParams& p, RopeJob j, cudaStream_t s) {
  j.n_rot_heads = j.n_out_heads + (APPEND ? j.n_kv_heads : 0);
  j.first_head = (APPEND && j.q_out == nullptr) ? j.n_out_heads : 0;
  j.rot_items = (p.interleaved ? 2 * p.n_pairs : p.n_pairs) / V;
  j.per_head = j.rot_items + (j.head_dim - 2 * p.n_pairs) / V;
  const int64_t turned = static_cast<int64_t>(j.n_rot_heads - j.first_head) * j.per_head;
  const int64_t items = turned + (APPEND ? static_cast<int64_t>(j.n_kv_heads) * (j.head_dim / V) : 0);
  if (items > 0x3fffffff) return set_error(B200EMB_ERR_UNSUPPORTED, "rope: rows too wide");
  j.turned = static_cast<int>(turned);
  j.items = static_cast<int>(items);
  const int threads = static_cast<int>(items < 64 ? 64 : items < ROPE_MAX_THREADS ? (items + 31) / 32 * 32 : ROPE_MAX_THREADS);
  cudaLaunchConfig_t cfg = {};  // returns this launch's own error: what an earlier call left behind is not this one's
  cfg.gridDim = dim3(static_cast<unsigned>(j.n_tokens));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = s;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, rope_kernel_op<V, APPEND>, p, j);
  if (e != cudaSuccess) return set_error(B200EMB_ERR_CUDA, "rope launch: %s", cudaGetErrorString(e));
  return B200EMB_OK;
}

template <bool APPEND>
static int rope_launch(const RopeParams& p, const RopeJob& j, cudaStream_t s) {
  switch (rope_vector(p, j, APPEND)) {
    case 8: return rope_launch_v<8, APPEND>(p, j, s);
    case 4: return rope_launch_v<4, APPEND>(p, j, s);
    case 2: return rope_launch_v<2, APPEND>(p, j, s);
    default: return rope_launch_v<1, APPEND>(p, j, s);
  }
}

int check_kv_cache(const b200emb_kv_cache* c, const char* who) {
  if (c == nullptr) return set_error(B200EMB_ERR_INVALID, "%s: null cache", who);
  if (c->k == nullptr || c->v == nullptr || c->page_table == nullptr)
    return set_error(B200EMB_ERR_INVALID, "%s: null pointer in the cache", who);
  if (c->n_pages <= 0 || c->page_size <= 0 || c->n_kv_heads <= 0 || c->head_dim <= 0 || c->table_stride <= 0)
    return set_error(B200EMB_ERR_INVALID, "%s: cache sizes must be positive", who);
  if (c->reserved != 0) return set_error(B200EMB_ERR_INVALID, "%s: reserved fields must be zero", who);
  if (static_cast<int64_t>(c->table_stride) * c->page_size > 0x7fffffffLL)
    return set_error(B200EMB_ERR_UNSUPPORTED, "%s: a page table of more than 2^31 - 1 positions", who);
  if (c->page_stride < 0 || c->token_stride < c->head_dim || c->head_stride < 0 ||
      (c->n_kv_heads > 1 && c->head_stride < c->head_dim) || (c->n_pages > 1 && c->page_stride < c->head_dim))
    return set_error(B200EMB_ERR_INVALID, "%s: a cache stride is smaller than head_dim", who);
  return B200EMB_OK;
}

}  // namespace b2

using namespace b2;

extern "C" int b200emb_op_rope(const void* x, int64_t x_row_stride, void* out, int64_t out_row_stride, const int32_t* positions,
                               const int32_t* d_cu_seqlens, const int32_t* d_pos_start, int32_t n_seqs, int32_t n_tokens,
                               int32_t n_heads, int32_t head_dim, const b200emb_rope_desc* rope, void* stream) {
  if (n_tokens < 0 || (positions == nullptr && n_seqs < 0) || n_heads <= 0 || head_dim <= 0)
    return set_error(B200EMB_ERR_INVALID, "rope: bad sizes");
  if (rope == nullptr) return set_error(B200EMB_ERR_INVALID, "rope: null descriptor");
  RopeParams p;
  int rc = rope_params(rope, head_dim, &p);
  if (rc) return rc;
  const int64_t width = static_cast<int64_t>(n_heads) * head_dim;
  if (x_row_stride < width || out_row_stride < width)
    return set_error(B200EMB_ERR_INVALID, "rope: a row stride is smaller than n_heads * head_dim = %lld", static_cast<long long>(width));
  if (n_tokens == 0 || (positions == nullptr && n_seqs == 0)) return B200EMB_OK;
  if (x == nullptr || out == nullptr || (positions == nullptr && d_cu_seqlens == nullptr))
    return set_error(B200EMB_ERR_INVALID, "rope: null pointer");
  if (x == out && x_row_stride != out_row_stride)
    return set_error(B200EMB_ERR_INVALID, "rope: in place needs equal row strides");
  RopeJob j = {};
  j.x = static_cast<const __nv_bfloat16*>(x);
  j.x_stride = x_row_stride;
  j.q_out = static_cast<__nv_bfloat16*>(out);
  j.q_stride = out_row_stride;
  j.positions = positions;
  j.cu = d_cu_seqlens;
  j.pos_start = d_pos_start;
  j.n_seqs = n_seqs;
  j.n_tokens = n_tokens;
  j.n_out_heads = n_heads;
  j.head_dim = head_dim;
  return rope_launch<false>(p, j, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int b200emb_op_kv_append(const void* qkv, int64_t qkv_row_stride, const int32_t* d_cu_seqlens, const int32_t* d_kv_lens,
                                    int32_t n_seqs, int32_t n_tokens, int32_t n_heads, const b200emb_rope_desc* rope, void* q_out,
                                    int64_t q_out_row_stride, const b200emb_kv_cache* cache, void* stream) {
  int rc = check_kv_cache(cache, "kv_append");
  if (rc) return rc;
  if (n_tokens < 0 || n_seqs < 0 || n_heads <= 0) return set_error(B200EMB_ERR_INVALID, "kv_append: bad sizes");
  RopeParams p;
  rc = rope_params(rope, cache->head_dim, &p);
  if (rc) return rc;
  const int64_t hd = cache->head_dim;
  if (qkv_row_stride < (n_heads + 2ll * cache->n_kv_heads) * hd || (q_out != nullptr && q_out_row_stride < n_heads * hd))
    return set_error(B200EMB_ERR_INVALID, "kv_append: a row stride is smaller than its heads");
  if (n_tokens == 0 || n_seqs == 0) return B200EMB_OK;
  if (qkv == nullptr || d_cu_seqlens == nullptr || d_kv_lens == nullptr)
    return set_error(B200EMB_ERR_INVALID, "kv_append: null pointer");
  if (q_out == qkv && q_out_row_stride != qkv_row_stride)
    return set_error(B200EMB_ERR_INVALID, "kv_append: queries in place need equal row strides");
  RopeJob j = {};
  j.x = static_cast<const __nv_bfloat16*>(qkv);
  j.x_stride = qkv_row_stride;
  j.q_out = static_cast<__nv_bfloat16*>(q_out);
  j.q_stride = q_out_row_stride;
  j.cu = d_cu_seqlens;
  j.pos_start = d_kv_lens;
  j.n_seqs = n_seqs;
  j.n_tokens = n_tokens;
  j.n_out_heads = n_heads;
  j.head_dim = cache->head_dim;
  j.k = static_cast<__nv_bfloat16*>(cache->k);
  j.v = static_cast<__nv_bfloat16*>(cache->v);
  j.page_table = cache->page_table;
  j.page_stride = cache->page_stride;
  j.token_stride = cache->token_stride;
  j.head_stride = cache->head_stride;
  j.n_pages = cache->n_pages;
  j.page_size = cache->page_size;
  j.n_kv_heads = cache->n_kv_heads;
  j.table_stride = cache->table_stride;
  return rope_launch<true>(p, j, reinterpret_cast<cudaStream_t>(stream));
}
