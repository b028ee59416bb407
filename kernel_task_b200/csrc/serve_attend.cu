// tr_paged_attention: attention of each request's last tokens over its paged cache.
#include <algorithm>
#include <cmath>

#include "serve_attend.cuh"

namespace trr {

// Any head_dim and type: one warp per token and query head, lane l holding elements
// l, l + 32, ... of q and of the running output, one pass over the keys with the running maximum
// and sum.  Bound by the five-step reduction of every key's product, one key after the other: 16
// requests of 4096, one new token each, 32 heads over 8, take 4.5 ms with a head_dim of 80 or 96
// in bf16 and of 128 in fp32, 5.6 ms with 256 in bf16 (their bytes: 26 to 83 us; the kernel of
// serve_attend_rows.cu does 128 in bf16 in 53 us).  It is the form for what the tensor-core kernels
// do not take, not a fast one.
template <typename E, int N>
__global__ void __launch_bounds__(128) attend_generic_kernel(const tr_attention a) {
  const int lane = threadIdx.x & 31;
  const int64_t w = blockIdx.x * 4ll + (threadIdx.x >> 5);
  if (w >= a.tokens * a.heads) return;
  const int64_t t = w / a.heads;
  const int h = (int)(w - t * a.heads), kvh = h / (a.heads / a.kv_heads);
  const int r = owner_of(a.starts, (int)a.requests, t);
  int64_t keys = 0;
  if (r >= 0) {
    const int64_t len = min((int64_t)a.lens[r], (int64_t)a.columns * a.page_size);
    keys = min(len, (int64_t)a.lens[r] - (a.starts[r + 1] - a.starts[r]) + (t - a.starts[r]) + 1);
  }
  const E* q = static_cast<const E*>(a.q) + t * a.q_token_stride + h * a.q_head_stride;
  float qf[N], o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = i * 32 + lane;
    qf[i] = d < a.head_dim ? to_f32<E>(q[d]) * a.scale : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < keys; ++j) {
    const int id = a.tables[r * a.table_stride + j / a.page_size];
    const bool held = id >= 0 && id < a.pages;
    const int64_t at =
        (((int64_t)id * a.kv_heads + kvh) * a.page_size + j % a.page_size) * a.head_dim;
    const E* k = static_cast<const E*>(a.k_pages) + at;
    const E* v = static_cast<const E*>(a.v_pages) + at;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = i * 32 + lane;
      if (held && d < a.head_dim) s = fmaf(qf[i], to_f32<E>(k[d]), s);
    }
    s = warp_sum(s);
    // scores may be -inf (a product that passes fp32): no difference of infinities
    const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
    const float keep = __expf(m - base), p = __expf(s - base);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = i * 32 + lane;
      o[i] = o[i] * keep + (held && d < a.head_dim ? p * to_f32<E>(v[d]) : 0.f);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no key, or scores of nothing but -inf
  E* out = static_cast<E*>(a.out) + (t * a.heads + h) * a.head_dim;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = i * 32 + lane;
    if (d < a.head_dim) out[d] = from_f32<E>(o[i] * inv);
  }
  if (a.lse && lane == 0) a.lse[t * a.heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

template <typename E>
static int launch_generic_attention(const tr_attention& a, void* stream) {
  const int64_t blocks = (a.tokens * a.heads + 3) / 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.head_dim <= 64) attend_generic_kernel<E, 2><<<(unsigned)blocks, 128, 0, s>>>(a);
  else if (a.head_dim <= 128) attend_generic_kernel<E, 4><<<(unsigned)blocks, 128, 0, s>>>(a);
  else attend_generic_kernel<E, 8><<<(unsigned)blocks, 128, 0, s>>>(a);
  return serve_launched("tr_paged_attention");
}

static bool on_tensor_cores(const tr_attention& a) {
  return a.dtype != TR_F32 && (a.head_dim == 64 || a.head_dim == 128);
}

// The chunk kernel above 32 query rows a request and kv head on average, of which its tiles hold
// 256; the rows kernel up to that, where reading the keys is the bound.  us of the rows kernel /
// the chunk kernel, 32 heads over 8 of 128 in bf16, with 16, 32 and 64 rows: 8 requests of 8192
// 54 / 79, 91 / 68, 164 / 71; 32 of 2048 53 / 80, 91 / 68, 140 / 73; one of 8192 25 / 56, 27 / 50,
// 31 / 50; 4 of 500 14 / 25, 18 / 27, 19 / 29.  The average is the step's: a long prompt takes the
// requests that decode beside it to the chunk kernel.
static bool in_chunks(const tr_attention& a) {
  return a.tokens * (a.heads / a.kv_heads) > 32 * a.requests;
}

static int check_attention(const tr_attention* a) {
  if (!a) {
    set_error("tr_paged_attention: null argument");
    return TR_ERR_INVALID;
  }
  if (!known_dtype(a->dtype)) {
    set_error("tr_paged_attention: unknown dtype %d", (int)a->dtype);
    return TR_ERR_INVALID;
  }
  if (a->tokens < 0 || a->requests < 0 || a->pages < 0 || a->columns < 0 || a->kv_heads < 1 ||
      a->heads < 1 || a->heads % a->kv_heads) {
    set_error("tr_paged_attention: bad shape (%d query heads over %d)", (int)a->heads,
              (int)a->kv_heads);
    return TR_ERR_INVALID;
  }
  if (a->requests > 1 && a->table_stride < a->columns) {
    set_error("tr_paged_attention: table stride %lld below its %d columns",
              (long long)a->table_stride, (int)a->columns);
    return TR_ERR_INVALID;
  }
  if (!(a->scale > 0.f) || std::isinf(a->scale)) {
    set_error("tr_paged_attention: scale must be positive and finite");
    return TR_ERR_INVALID;
  }
  if (a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8) {
    set_error("tr_paged_attention: head_dim %d (a multiple of 8 up to 256)", (int)a->head_dim);
    return TR_ERR_UNSUPPORTED;
  }
  if (a->page_size < 1 || a->page_size > 1024 || (a->page_size & (a->page_size - 1))) {
    set_error("tr_paged_attention: page_size %d (a power of two up to 1024)", (int)a->page_size);
    return TR_ERR_UNSUPPORTED;
  }
  if ((int64_t)a->columns * a->page_size > (int64_t)1 << 30 ||
      a->tokens > INT32_MAX || a->tokens * a->heads > (int64_t)1 << 31 || a->requests > (int64_t)1 << 20 ||
      a->pages > INT32_MAX ||
      (double)a->pages * a->kv_heads * a->page_size >= 4294967295.) {
    set_error("tr_paged_attention: too large (a request's cache up to 2^30 tokens, tokens x heads "
              "up to 2^31, 2^20 requests, pools below 2^32 rows)");
    return TR_ERR_UNSUPPORTED;
  }
  if (a->tokens == 0) return TR_OK;
  if (!a->q || !a->out ||
      (a->requests > 0 && (!a->lens || !a->starts || (a->columns > 0 && !a->tables))) ||
      (a->pages > 0 && (!a->k_pages || !a->v_pages))) {
    set_error("tr_paged_attention: null pointer");
    return TR_ERR_INVALID;
  }
  if (((uintptr_t)a->tables | (uintptr_t)a->lens | (uintptr_t)a->starts | (uintptr_t)a->lse) & 3) {
    set_error("tr_paged_attention: a pointer is not aligned to its elements");
    return TR_ERR_ALIGN;
  }
  const int eb = element_bytes(a->dtype);
  if ((((uintptr_t)a->q | (uintptr_t)a->k_pages | (uintptr_t)a->v_pages | (uintptr_t)a->out) & 15) ||
      ((a->q_token_stride * eb | a->q_head_stride * eb) & 15)) {
    set_error("tr_paged_attention: q (base and strides), pools and out must be 16-byte aligned");
    return TR_ERR_ALIGN;
  }
  return TR_OK;
}

static int workspace_need(const tr_attention& a, size_t* bytes) {
  const bool chunks = in_chunks(a);
  if ((chunks ? attend_chunk_items(a) : attend_rows_items(a)) > kAttendCounters) {
    set_error("tr_paged_attention: over %lld tiles of query rows", (long long)kAttendCounters);
    return TR_ERR_UNSUPPORTED;
  }
  *bytes = TR_ATTENTION_STATE_BYTES + (chunks ? attend_chunk_partials(a) : attend_rows_partials(a));
  return TR_OK;
}

}  // namespace trr

using namespace trr;

extern "C" int tr_attention_workspace_bytes(const tr_attention* a, size_t* bytes) {
  const int st = check_attention(a);
  if (st != TR_OK) return st;
  if (!bytes) {
    set_error("tr_attention_workspace_bytes: null pointer");
    return TR_ERR_INVALID;
  }
  *bytes = 0;
  return a->tokens > 0 && on_tensor_cores(*a) ? workspace_need(*a, bytes) : TR_OK;
}

extern "C" int tr_paged_attention(const tr_attention* a, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  const int st = check_attention(a);
  if (st != TR_OK || a->tokens == 0) return st;
  if (on_tensor_cores(*a)) {
    size_t need = 0;
    const int short_of = workspace_need(*a, &need);
    if (short_of != TR_OK) return short_of;
    if (!workspace || workspace_bytes < need) {
      set_error("tr_paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
      return TR_ERR_WORKSPACE;
    }
    if ((uintptr_t)workspace & 15) {
      set_error("tr_paged_attention: the workspace must be 16-byte aligned");
      return TR_ERR_ALIGN;
    }
    char* w = static_cast<char*>(workspace);
    const AttendWorkspace ws = {reinterpret_cast<int*>(w), reinterpret_cast<int*>(w + 256),
                                reinterpret_cast<float*>(w + TR_ATTENTION_STATE_BYTES)};
    return in_chunks(*a) ? launch_attend_chunk(*a, ws, stream) : launch_attend_rows(*a, ws, stream);
  }
  if (a->dtype == TR_F32) return launch_generic_attention<float>(*a, stream);
  if (a->dtype == TR_F16) return launch_generic_attention<__half>(*a, stream);
  return launch_generic_attention<__nv_bfloat16>(*a, stream);
}
