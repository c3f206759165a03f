// Attention with modified scores over a packed batch, and the same over a paged key / value cache.
//
// One warp per (query token, head): the lanes share the head dimension, the keys are walked once with a running
// maximum and sum (m, l, o) <- (m', l e^(m - m') + e^(s - m'), o e^(m - m') + e^(s - m') v).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "kernels.h"

namespace b2 {

static constexpr int AS_MAX_RADIUS = 1023;
static constexpr int AS_MAX_GROUP = 128;
static constexpr int64_t AS_ALIGN = 256;

struct AttnMod {
  float scale, cap;
  int left, right, radius;
  const float* slopes;
  const float* bias;
  const int32_t* prefix;
  const int32_t* docs;
};

struct AttnIo {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  __nv_bfloat16* out;
  int64_t q_stride, k_stride, v_stride, out_stride;
  const int32_t* cu;
  const int32_t* kv_lens;
  const int32_t* page_table;
  int64_t page_stride, token_stride, head_stride;
  int n_seqs, n_tokens, n_heads, n_kv_heads, head_dim;
  int n_pages, page_size, table_stride;
};

__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&x)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  x[0] = a.x;
  x[1] = a.y;
  x[2] = b.x;
  x[3] = b.y;
}

template <bool PAGED>
__global__ void __launch_bounds__(256) attn_rows_kernel(const AttnIo io, const AttnMod mod, int* __restrict__ status) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *status = 0;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= static_cast<int64_t>(io.n_tokens) * io.n_heads) return;
  const int t = static_cast<int>(row / io.n_heads), h = static_cast<int>(row % io.n_heads);
  const int hk = h / (io.n_heads / io.n_kv_heads);
  int lo = 0, hi = io.n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (io.cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int first = max(io.cu[lo], 0), end = min(io.cu[lo + 1], io.n_tokens);
  if (t < first || t >= end) return;
  int kv_len = end - first;
  if (PAGED) kv_len = min(max(io.kv_lens[lo], 0), io.table_stride * io.page_size);
  const int pos = kv_len - (end - first) + (t - first);
  const int prefix = mod.prefix != nullptr ? mod.prefix[lo] : 0;
  const int doc = mod.docs != nullptr ? mod.docs[t] : 0;
  const bool on = lane * 4 < io.head_dim;
  float q[4] = {}, o[4] = {}, k[4] = {}, v[4] = {};
  if (on) load4(io.q + t * io.q_stride + static_cast<int64_t>(h) * io.head_dim + lane * 4, q);
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < kv_len; ++j) {
    const int d = j - pos;
    bool seen = (d <= mod.right && d >= -mod.left) || j < prefix;
    if (mod.docs != nullptr) seen = seen && doc >= 0 && mod.docs[first + j] == doc;
    if (!seen) continue;
    const __nv_bfloat16* kp = nullptr;
    const __nv_bfloat16* vp = nullptr;
    if (PAGED) {
      const int page = io.page_table[static_cast<int64_t>(lo) * io.table_stride + j / io.page_size];
      if (page >= 0 && page < io.n_pages) {
        const int64_t at = page * io.page_stride + (j % io.page_size) * io.token_stride + hk * io.head_stride;
        kp = io.k + at;
        vp = io.v + at;
      }
    } else {
      kp = io.k + (first + j) * io.k_stride + static_cast<int64_t>(hk) * io.head_dim;
      vp = io.v + (first + j) * io.v_stride + static_cast<int64_t>(hk) * io.head_dim;
    }
    if (on && kp != nullptr) {
      load4(kp + lane * 4, k);
      load4(vp + lane * 4, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) k[e] = v[e] = 0.f;
    }
    float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= mod.scale;
    if (mod.cap > 0.f) s = mod.cap * tanhf(s / mod.cap);
    if (mod.slopes != nullptr) s -= mod.slopes[h] * fabsf(static_cast<float>(d));
    if (mod.bias != nullptr)
      s += mod.bias[static_cast<int64_t>(h) * (2 * mod.radius + 1) + min(max(d, -mod.radius), mod.radius) + mod.radius];
    const float m_new = fmaxf(m, s);
    if (m_new == -INFINITY && s == s) continue;  // nothing seen yet (a NaN score goes on and makes the row NaN)
    const float keep = expf(m - m_new), p = expf(s - m_new);
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * keep + p * v[e];
    m = m_new;
  }
  if (on) {
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    __nv_bfloat162 a = __floats2bfloat162_rn(o[0] * inv, o[1] * inv), b = __floats2bfloat162_rn(o[2] * inv, o[3] * inv);
    uint2 u;
    u.x = *reinterpret_cast<uint32_t*>(&a);
    u.y = *reinterpret_cast<uint32_t*>(&b);
    *reinterpret_cast<uint2*>(io.out + t * io.out_stride + static_cast<int64_t>(h) * io.head_dim + lane * 4) = u;
  }
}

// ---- host side ----------------------------------------------------------------------

static int check_shape(int n_seqs, int n_tokens, int n_heads, int n_kv_heads, int head_dim, const char* who) {
  if (n_seqs < 0 || n_tokens < 0 || n_heads <= 0 || n_kv_heads <= 0)
    return set_error(B200EMB_ERR_INVALID, "%s: bad sizes", who);
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
  if (!isfinite(o->scale) || !isfinite(o->cap) || o->cap < 0.f)
    return set_error(B200EMB_ERR_INVALID, "%s: scale must be finite and cap finite and not negative", who);
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

template <bool PAGED>
static int launch_rows(const AttnIo& io, const AttnMod& mod, void* workspace, cudaStream_t s) {
  const int64_t blocks = (static_cast<int64_t>(io.n_tokens) * io.n_heads + 7) / 8;
  if (blocks > INT_MAX) return set_error(B200EMB_ERR_UNSUPPORTED, "attention: too many rows");
  attn_rows_kernel<PAGED><<<static_cast<unsigned>(blocks), 256, 0, s>>>(io, mod, static_cast<int*>(workspace));
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(B200EMB_ERR_CUDA, "attention launch: %s", cudaGetErrorString(e));
  return B200EMB_OK;
}

}  // namespace b2

using namespace b2;

extern "C" int64_t b200emb_attention_workspace_bytes(int32_t n_seqs, int32_t n_tokens, int32_t n_heads, int32_t n_kv_heads,
                                                     int32_t head_dim) {
  const int rc = check_shape(n_seqs, n_tokens, n_heads, n_kv_heads, head_dim, "attention_workspace_bytes");
  return rc ? (rc < 0 ? rc : -rc) : AS_ALIGN;
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
  if (n_tokens == 0 || n_seqs == 0) return B200EMB_OK;
  const int64_t wq = static_cast<int64_t>(n_heads) * head_dim, wk = static_cast<int64_t>(n_kv_heads) * head_dim;
  rc = check_rows(q, q_row_stride, wq, "q", who);
  if (!rc) rc = check_rows(k, k_row_stride, wk, "k", who);
  if (!rc) rc = check_rows(v, v_row_stride, wk, "v", who);
  if (!rc) rc = check_rows(out, out_row_stride, wq, "out", who);
  if (!rc && d_cu_seqlens == nullptr) rc = set_error(B200EMB_ERR_INVALID, "%s: null pointer cu_seqlens", who);
  if (!rc) rc = check_workspace(workspace, workspace_bytes, b200emb_attention_workspace_bytes(n_seqs, n_tokens, n_heads, n_kv_heads, head_dim), who);
  if (rc) return rc;
  AttnIo io = {};
  io.q = static_cast<const __nv_bfloat16*>(q);
  io.k = static_cast<const __nv_bfloat16*>(k);
  io.v = static_cast<const __nv_bfloat16*>(v);
  io.out = static_cast<__nv_bfloat16*>(out);
  io.q_stride = q_row_stride;
  io.k_stride = k_row_stride;
  io.v_stride = v_row_stride;
  io.out_stride = out_row_stride;
  io.cu = d_cu_seqlens;
  io.n_seqs = n_seqs;
  io.n_tokens = n_tokens;
  io.n_heads = n_heads;
  io.n_kv_heads = n_kv_heads;
  io.head_dim = head_dim;
  return launch_rows<false>(io, mod, workspace, reinterpret_cast<cudaStream_t>(stream));
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
  if (cache->page_size % 8 != 0)
    return set_error(B200EMB_ERR_UNSUPPORTED, "%s: page_size %d is no multiple of 8", who, cache->page_size);
  if (cache->page_stride % 8 != 0 || cache->token_stride % 8 != 0 || cache->head_stride % 8 != 0 ||
      reinterpret_cast<uintptr_t>(cache->k) % 16 != 0 || reinterpret_cast<uintptr_t>(cache->v) % 16 != 0)
    return set_error(B200EMB_ERR_INVALID, "%s: the cache must be 16-byte aligned with strides that are multiples of 8", who);
  if (n_tokens == 0 || n_seqs == 0) return B200EMB_OK;
  const int64_t wq = static_cast<int64_t>(n_heads) * cache->head_dim;
  rc = check_rows(q, q_row_stride, wq, "q", who);
  if (!rc) rc = check_rows(out, out_row_stride, wq, "out", who);
  if (!rc && (d_cu_seqlens == nullptr || d_kv_lens == nullptr))
    rc = set_error(B200EMB_ERR_INVALID, "%s: null pointer cu_seqlens or kv_lens", who);
  if (!rc)
    rc = check_workspace(workspace, workspace_bytes,
                         b200emb_attention_workspace_bytes(n_seqs, n_tokens, n_heads, cache->n_kv_heads, cache->head_dim), who);
  if (rc) return rc;
  AttnIo io = {};
  io.q = static_cast<const __nv_bfloat16*>(q);
  io.k = static_cast<const __nv_bfloat16*>(cache->k);
  io.v = static_cast<const __nv_bfloat16*>(cache->v);
  io.out = static_cast<__nv_bfloat16*>(out);
  io.q_stride = q_row_stride;
  io.out_stride = out_row_stride;
  io.cu = d_cu_seqlens;
  io.kv_lens = d_kv_lens;
  io.page_table = cache->page_table;
  io.page_stride = cache->page_stride;
  io.token_stride = cache->token_stride;
  io.head_stride = cache->head_stride;
  io.n_seqs = n_seqs;
  io.n_tokens = n_tokens;
  io.n_heads = n_heads;
  io.n_kv_heads = cache->n_kv_heads;
  io.head_dim = cache->head_dim;
  io.n_pages = cache->n_pages;
  io.page_size = cache->page_size;
  io.table_stride = cache->table_stride;
  return launch_rows<true>(io, mod, workspace, reinterpret_cast<cudaStream_t>(stream));
}
