// tr_residual_norm: the norm after a block, its gate, the scaled residual add and the norm
// before the next block, in one pass over the row.
#include <algorithm>

#include "serve_util.cuh"

namespace trr {

struct NormArgs {
  const void* y;
  const void* h;
  const void* gate;
  const void* post;
  const void* post_bias;
  const void* pre;
  const void* pre_bias;
  void* h_out;
  void* x_out;
  int64_t tokens, y_stride, h_stride, gate_stride;
  int width;
  float eps, residual_scale, branch_scale;
};

// Sum over the G threads of a row.  Rows of more than a warp go through shared memory, with one
// barrier a call: successive calls alternate between the two buffers, so a thread may write the
// next sums while others still read these.
template <int G>
__device__ __forceinline__ float row_sum(float v, float (*part)[32], int& turn) {
  v = warp_sum(v);
  if constexpr (G > 32) {
    const int lane = threadIdx.x & 31;
    float* p = part[turn & 1];
    ++turn;
    if (lane == 0) p[threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_sum(lane < G / 32 ? p[lane] : 0.f);
  }
  return v;
}

// f <- N(f) * weight + bias over one row; entries past the width hold zeros and stay out of the
// sums.  The mean is taken out before the squares are summed: sums of squares about zero would
// cancel where the mean is large against the spread.  What the first mean is off by (fp32: up to
// 2^-24 of it and the sum's error) is the mean of the differences, summed next to their squares.
template <typename E, bool LAYER, int G, int N, int V>
__device__ __forceinline__ void norm_row(float (&f)[N * V], const E* weight, const E* bias,
                                         int width, float eps, float (*part)[32], int& turn) {
  const int t = G > 32 ? threadIdx.x : threadIdx.x & 31;
  const float inv_width = 1.f / (float)width;
  float mean = 0.f;
  if constexpr (LAYER) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N * V; ++i) s += f[i];
    mean = row_sum<G>(s, part, turn) * inv_width;
  }
  float s = 0.f, d = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if ((i * G + t) * V < width) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[i * V + j] -= mean;
        if constexpr (LAYER) d += f[i * V + j];
        s = fmaf(f[i * V + j], f[i * V + j], s);
      }
    }
  }
  s = row_sum<G>(s, part, turn) * inv_width;
  if constexpr (LAYER) {
    d = row_sum<G>(d, part, turn) * inv_width;
    s = fmaf(-d, d, s);
  }
  const float r = rsqrtf(s + eps);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * G + t) * V;
    if (c >= width) continue;
    if constexpr (V == 8) {
      float w[8];
      load8<E>(weight + c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i * 8 + j] = (f[i * 8 + j] - d) * (r * w[j]);
      if (bias) {
        load8<E>(bias + c, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i * 8 + j] += w[j];
      }
    } else {
      f[i] = (f[i] - d) * (r * to_f32<E>(weight[c])) + (bias ? to_f32<E>(bias[c]) : 0.f);
    }
  }
}

template <typename T, int G, int N, int V>
__device__ __forceinline__ void load_row(const T* p, int width, float (&f)[N * V]) {
  const int t = G > 32 ? threadIdx.x : threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * G + t) * V;
    if constexpr (V == 8) {
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (c < width) load8<T>(p + c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i * 8 + j] = v[j];
    } else {
      f[i] = c < width ? to_f32<T>(p[c]) : 0.f;
    }
  }
}
template <typename E, int G, int N, int V>
__device__ __forceinline__ void store_row(E* p, int width, const float (&f)[N * V]) {
  const int t = G > 32 ? threadIdx.x : threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * G + t) * V;
    if (c >= width) continue;
    if constexpr (V == 8) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = f[i * 8 + j];
      store8<E>(p + c, v);
    } else {
      p[c] = from_f32<E>(f[i]);
    }
  }
}

// G threads hold a row in registers as N vectors of V elements each (G = 32: a warp per row, 8
// rows a block; else a block per row), so y and h are read once and both outputs written once
// whatever the norms need.
template <typename E, typename Y, bool LAYER, int G, int N, int V>
__global__ void __launch_bounds__(G > 32 ? G : 256) residual_norm_kernel(const NormArgs a) {
  __shared__ float part[2][32];
  int turn = 0;
  const int64_t rows_per_block = G > 32 ? 1 : 8;
  for (int64_t row = blockIdx.x * rows_per_block + (G > 32 ? 0 : threadIdx.x >> 5); row < a.tokens;
       row += gridDim.x * rows_per_block) {
    float f[N * V], g[N * V];
    load_row<E, G, N, V>(static_cast<const E*>(a.h) + row * a.h_stride, a.width, g);
    if (a.y) {
      load_row<Y, G, N, V>(static_cast<const Y*>(a.y) + row * a.y_stride, a.width, f);
      if (a.post)
        norm_row<E, LAYER, G, N, V>(f, static_cast<const E*>(a.post),
                                    static_cast<const E*>(a.post_bias), a.width, a.eps, part, turn);
#pragma unroll
      for (int i = 0; i < N * V; ++i) g[i] *= a.residual_scale;
      if (a.gate) {
        float w[N * V];
        load_row<E, G, N, V>(static_cast<const E*>(a.gate) + row * a.gate_stride, a.width, w);
#pragma unroll
        for (int i = 0; i < N * V; ++i) f[i] *= w[i];
      }
#pragma unroll
      for (int i = 0; i < N * V; ++i) g[i] = fmaf(a.branch_scale, f[i], g[i]);
      store_row<E, G, N, V>(static_cast<E*>(a.h_out) + row * a.width, a.width, g);
    }
    if (a.pre) {
      norm_row<E, LAYER, G, N, V>(g, static_cast<const E*>(a.pre),
                                  static_cast<const E*>(a.pre_bias), a.width, a.eps, part, turn);
      store_row<E, G, N, V>(static_cast<E*>(a.x_out) + row * a.width, a.width, g);
    }
  }
}

template <typename E, typename Y, bool LAYER, int G, int N, int V>
static int launch_norm(const NormArgs& a, void* stream) {
  const int64_t rows_per_block = G > 32 ? 1 : 8;
  const int64_t blocks = (a.tokens + rows_per_block - 1) / rows_per_block;
  const int threads = G > 32 ? G : 256;
  const int64_t most = (int64_t)serve_sms() * (2048 / threads);
  residual_norm_kernel<E, Y, LAYER, G, N, V>
      <<<(unsigned)std::min(blocks, most), threads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return serve_launched("tr_residual_norm");
}

template <typename E, typename Y, bool LAYER>
static int pick_norm(const NormArgs& a, bool wide, void* stream) {
  if (wide) {
    const int vectors = a.width / 8;
    if (vectors <= 64) return launch_norm<E, Y, LAYER, 32, 2, 8>(a, stream);
    if (vectors <= 128) return launch_norm<E, Y, LAYER, 128, 1, 8>(a, stream);
    if (vectors <= 256) return launch_norm<E, Y, LAYER, 256, 1, 8>(a, stream);
    if (vectors <= 512) return launch_norm<E, Y, LAYER, 512, 1, 8>(a, stream);
    if (vectors <= 1024) return launch_norm<E, Y, LAYER, 512, 2, 8>(a, stream);
    return launch_norm<E, Y, LAYER, 1024, 4, 8>(a, stream);
  }
  if (a.width <= 256) return launch_norm<E, Y, LAYER, 32, 8, 1>(a, stream);
  if (a.width <= 2048) return launch_norm<E, Y, LAYER, 256, 8, 1>(a, stream);
  if (a.width <= 8192) return launch_norm<E, Y, LAYER, 1024, 8, 1>(a, stream);
  return launch_norm<E, Y, LAYER, 1024, 32, 1>(a, stream);
}

template <typename E, typename Y>
static int pick_kind(const NormArgs& a, int kind, bool wide, void* stream) {
  return kind == TR_NORM_LAYER ? pick_norm<E, Y, true>(a, wide, stream)
                               : pick_norm<E, Y, false>(a, wide, stream);
}

}  // namespace trr

using namespace trr;

extern "C" int tr_residual_norm(const tr_norm* n, void* stream) {
  if (!n) {
    set_error("tr_residual_norm: null argument");
    return TR_ERR_INVALID;
  }
  if (!known_dtype(n->dtype) || (n->y && n->y_dtype != n->dtype && n->y_dtype != TR_F32)) {
    set_error("tr_residual_norm: dtype %d with y in dtype %d", (int)n->dtype, (int)n->y_dtype);
    return TR_ERR_INVALID;
  }
  if (n->kind != TR_NORM_RMS && n->kind != TR_NORM_LAYER) {
    set_error("tr_residual_norm: unknown kind %d", (int)n->kind);
    return TR_ERR_INVALID;
  }
  if (n->tokens < 0 || n->width < 1) {
    set_error("tr_residual_norm: bad shape");
    return TR_ERR_INVALID;
  }
  if (n->width > 32768) {
    set_error("tr_residual_norm: width %lld (at most 32768)", (long long)n->width);
    return TR_ERR_UNSUPPORTED;
  }
  if ((!n->y && !n->pre) || (!n->post && n->post_bias) || (!n->pre && n->pre_bias) ||
      (!n->y && (n->post || n->gate)) || !(n->eps >= 0.f)) {
    set_error("tr_residual_norm: neither y nor pre, a bias without its weight, a gate or post "
              "weight without y, or a negative eps");
    return TR_ERR_INVALID;
  }
  if (n->tokens == 0) return TR_OK;
  if (!n->h || (n->y && !n->h_out) || (n->pre && !n->x_out)) {
    set_error("tr_residual_norm: null pointer");
    return TR_ERR_INVALID;
  }
  NormArgs a = {n->y,     n->h,        n->gate,        n->post,   n->post_bias, n->pre,
                n->pre_bias, n->h_out, n->x_out,       n->tokens, n->y_stride,  n->h_stride,
                n->gate_stride, (int)n->width, n->eps, n->residual_scale, n->branch_scale};
  const int eb = element_bytes(n->dtype), yb = n->y ? element_bytes(n->y_dtype) : eb;
  const uintptr_t all = (uintptr_t)n->h | (uintptr_t)n->gate | (uintptr_t)n->post |
                        (uintptr_t)n->post_bias | (uintptr_t)n->pre | (uintptr_t)n->pre_bias |
                        (uintptr_t)n->h_out | (uintptr_t)n->x_out;
  if ((all & (eb - 1)) || ((uintptr_t)n->y & (yb - 1))) {
    set_error("tr_residual_norm: a pointer is not aligned to its elements");
    return TR_ERR_ALIGN;
  }
  // 16-byte vectors where every row starts on one, else single elements
  const bool wide = n->width % 8 == 0 && !((all | (uintptr_t)n->y) & 15) &&
                    !((n->h_stride * eb | n->gate_stride * eb | n->y_stride * yb) & 15);
  const bool y32 = n->y && n->y_dtype == TR_F32;
  if (n->dtype == TR_F32) return pick_kind<float, float>(a, n->kind, wide, stream);
  if (n->dtype == TR_F16)
    return y32 ? pick_kind<__half, float>(a, n->kind, wide, stream)
               : pick_kind<__half, __half>(a, n->kind, wide, stream);
  return y32 ? pick_kind<__nv_bfloat16, float>(a, n->kind, wide, stream)
             : pick_kind<__nv_bfloat16, __nv_bfloat16>(a, n->kind, wide, stream);
}
