// tr_residual_norm: the norm after a block, its gate, the scaled residual add and the norm
// before the next block, in one pass over the row.
#include <algorithm>
#include <type_traits>

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

// Sums of x and y over the threads of a row: a warp (ROW_WARP) or the block.  Rows of more than
// a warp go through shared memory, with one barrier a call: successive calls alternate between
// the two buffers, so a thread may write the next sums while others still read these.
template <bool ROW_WARP>
__device__ __forceinline__ float2 row_sum(float x, float y, float2 (*part)[32], int& turn) {
  x = warp_sum(x);
  y = warp_sum(y);
  if constexpr (!ROW_WARP) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    float2* p = part[turn & 1];
    ++turn;
    if (lane == 0) p[threadIdx.x >> 5] = make_float2(x, y);
    __syncthreads();
    const float2 v = lane < warps ? p[lane] : make_float2(0.f, 0.f);
    x = warp_sum(v.x);
    y = warp_sum(v.y);
  }
  return make_float2(x, y);
}

// N vectors of V elements as they lie in memory; elements past the width are zeros
template <typename T, int N, int V>
struct Row {
  static constexpr int WORDS = V * sizeof(T) >= 16 ? V * sizeof(T) / 16 : 1;
  using Word = typename std::conditional<V == 8, uint4, T>::type;
  Word w[N][WORDS];

  __device__ __forceinline__ void load(const T* p, int t, int threads, int width, bool held) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * threads + t) * V;
      const bool in = held && c < width;
#pragma unroll
      for (int j = 0; j < WORDS; ++j) {
        if constexpr (V == 8)
          w[i][j] = in ? reinterpret_cast<const uint4*>(p + c)[j] : make_uint4(0, 0, 0, 0);
        else
          w[i][j] = in ? p[c] : from_f32<T>(0.f);
      }
    }
  }
  __device__ __forceinline__ void get(int i, float (&f)[V]) const {
    if constexpr (V == 1) f[0] = to_f32<T>(w[i][0]);
    else load8<T>(reinterpret_cast<const T*>(w[i]), f);
  }
};

template <typename T, int V>
__device__ __forceinline__ void get_vector(const T* p, float (&f)[V]) {
  if constexpr (V == 1) f[0] = to_f32<T>(p[0]);
  else load8<T>(p, f);
}

// f <- N(f) * weight + bias over one row; entries past the width hold zeros and stay out of the
// sums.  The mean is taken out before the squares are summed: sums of squares about zero would
// cancel where the mean is large against the spread.  What the first mean is off by (fp32: up to
// 2^-24 of it and the sum's error) is the mean of the differences, summed next to their squares.
template <typename E, bool LAYER, bool ROW_WARP, int N, int V>
__device__ __forceinline__ void norm_row(float (&f)[N][V], const E* weight, const E* bias, int t,
                                         int threads, int width, float inv_width, float eps,
                                         float2 (*part)[32], int& turn) {
  float mean = 0.f;
  if constexpr (LAYER) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s += f[i][j];
    mean = row_sum<ROW_WARP>(s, 0.f, part, turn).x * inv_width;
  }
  float s = 0.f, d = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float m = (i * threads + t) * V < width ? mean : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (LAYER) {
        f[i][j] -= m;
        d += f[i][j];
      }
      s = fmaf(f[i][j], f[i][j], s);
    }
  }
  const float2 sums = row_sum<ROW_WARP>(s, d, part, turn);
  s = sums.x * inv_width;
  if constexpr (LAYER) {
    d = sums.y * inv_width;
    s = fmaf(-d, d, s);
    // of a row of one value what is left is rounding, of either sign: below 0 it may pass a small
    // eps (a NaN stays)
    s = s < 0.f ? 0.f : s;
  }
  const float r = rsqrtf(s + eps);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * threads + t) * V;
    if (c >= width) continue;
    float w[V];
    get_vector<E, V>(weight + c, w);
#pragma unroll
    for (int j = 0; j < V; ++j) f[i][j] = (LAYER ? f[i][j] - d : f[i][j]) * (r * w[j]);
    if (bias) {
      get_vector<E, V>(bias + c, w);
#pragma unroll
      for (int j = 0; j < V; ++j) f[i][j] += w[j];
    }
  }
}

template <typename E, int N, int V>
__device__ __forceinline__ void store_row(E* p, int t, int threads, int width,
                                          const float (&f)[N][V]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * threads + t) * V;
    if (c >= width) continue;
    if constexpr (V == 8) store8<E>(p + c, f[i]);
    else p[c] = from_f32<E>(f[i][0]);
  }
}

// A row lies in the registers of its threads (a warp, 8 rows a block; or the block) as N vectors
// of V elements each, so y and h are read once and both outputs written once whatever the
// norms need.  A block takes every gridDim.x-th row.  Up to 8 elements a thread (widths to 256, and
// to 4096 where rows are not vectors) it loads the next row before it works on this one; above, two
// vectors a thread and more, other blocks of the SM cover the barrier that each sum costs.  The
// weights come from L1.  Bound by memory: 16384 rows of 4096 from fp32 with a gate per channel
// take 113 us (6.0 TB/s); 16391 of 2880 with the mean removed and a gate per token 110 us
// (4.3 TB/s), where the four sums a row are felt (a warp per row of 2880 has no barrier, but
// 184 us: too few rows in flight); one row 3.8 us.
// Rows that are not 16-byte vectors are read by elements: 16391 of 2881 from fp16 take 357 us where
// 2880 take 78 (rms, gate per channel), 8192 of 5001 from fp32 460 us (0.9 TB/s).  Widths above
// 16384 take 1024 threads of 64 registers and spill (110 to 840 bytes a thread by vectors, 260 to
// 670 by elements): 1024 rows of 32768 from fp32 83 us (4.0 TB/s), of 32767 405 us.
template <typename E, typename Y, bool LAYER, bool ROW_WARP, int N, int V, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) residual_norm_kernel(const NormArgs a) {
  constexpr bool AHEAD = N * V <= 8;
  __shared__ float2 part[2][32];
  int turn = 0;
  const int t = ROW_WARP ? threadIdx.x & 31 : threadIdx.x, threads = ROW_WARP ? 32 : blockDim.x;
  const int rows_at_once = ROW_WARP ? THREADS / 32 : 1;
  const int64_t first = (int64_t)blockIdx.x * rows_at_once + (ROW_WARP ? threadIdx.x >> 5 : 0);
  const int64_t stride = (int64_t)gridDim.x * rows_at_once;
  const float inv_width = 1.f / (float)a.width;
  const E *h = static_cast<const E*>(a.h), *gate = static_cast<const E*>(a.gate);
  const Y* y = static_cast<const Y*>(a.y);
  Row<E, N, V> next_h, next_gate;
  Row<Y, N, V> next_y;
  const auto fetch = [&](int64_t row) {
    const bool held = row < a.tokens;
    next_h.load(h + row * a.h_stride, t, threads, a.width, held);
    next_y.load(y + row * a.y_stride, t, threads, a.width, held && y);
    next_gate.load(gate + row * a.gate_stride, t, threads, a.width, held && gate);
  };
  if constexpr (AHEAD) fetch(first);
  for (int64_t row = first; row < a.tokens; row += stride) {
    if constexpr (!AHEAD) fetch(row);
    const Row<E, N, V> row_h = next_h, row_gate = next_gate;
    const Row<Y, N, V> row_y = next_y;
    if constexpr (AHEAD) fetch(row + stride);
    float f[N][V], g[V];
    if (y) {
#pragma unroll
      for (int i = 0; i < N; ++i) row_y.get(i, f[i]);
      if (a.post)
        norm_row<E, LAYER, ROW_WARP, N, V>(f, static_cast<const E*>(a.post),
                                          static_cast<const E*>(a.post_bias), t, threads, a.width,
                                          inv_width, a.eps, part, turn);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (gate) {
          row_gate.get(i, g);
#pragma unroll
          for (int j = 0; j < V; ++j) f[i][j] *= g[j];
        }
        row_h.get(i, g);
#pragma unroll
        for (int j = 0; j < V; ++j)
          f[i][j] = fmaf(a.branch_scale, f[i][j], a.residual_scale * g[j]);
      }
      store_row<E, N, V>(static_cast<E*>(a.h_out) + row * a.width, t, threads, a.width, f);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) row_h.get(i, f[i]);
    }
    if (a.pre) {
      norm_row<E, LAYER, ROW_WARP, N, V>(f, static_cast<const E*>(a.pre),
                                        static_cast<const E*>(a.pre_bias), t, threads, a.width,
                                        inv_width, a.eps, part, turn);
      store_row<E, N, V>(static_cast<E*>(a.x_out) + row * a.width, t, threads, a.width, f);
    }
  }
}

// THREADS: the most a block has; BLOCKS: the blocks of that size that an SM holds
template <typename E, typename Y, bool LAYER, bool ROW_WARP, int N, int V, int THREADS, int BLOCKS>
static int launch_norm(const NormArgs& a, void* stream) {
  const int vectors = (a.width + V - 1) / V;
  const int threads = ROW_WARP ? THREADS : ((vectors + N - 1) / N + 31) / 32 * 32;
  const int64_t rows_at_once = ROW_WARP ? THREADS / 32 : 1;
  const int64_t blocks = (a.tokens + rows_at_once - 1) / rows_at_once;
  const int64_t most = (int64_t)serve_sms() * (THREADS * BLOCKS / threads);
  residual_norm_kernel<E, Y, LAYER, ROW_WARP, N, V, THREADS, BLOCKS>
      <<<(unsigned)std::min(blocks, most), threads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return serve_launched("tr_residual_norm");
}

template <typename E, typename Y, bool LAYER>
static int pick_norm(const NormArgs& a, bool wide, void* stream) {
  if (wide) {  // widths to 512 a warp a row; then vectors a thread by what a block holds
    if (a.width <= 256) return launch_norm<E, Y, LAYER, true, 1, 8, 256, 4>(a, stream);
    if (a.width <= 512) return launch_norm<E, Y, LAYER, true, 2, 8, 256, 3>(a, stream);
    if (a.width <= 1024) return launch_norm<E, Y, LAYER, true, 4, 8, 256, 2>(a, stream);
    if (a.width <= 4096) return launch_norm<E, Y, LAYER, false, 2, 8, 256, 4>(a, stream);
    if (a.width <= 8192) return launch_norm<E, Y, LAYER, false, 2, 8, 512, 2>(a, stream);
    if (a.width <= 16384) return launch_norm<E, Y, LAYER, false, 4, 8, 512, 1>(a, stream);
    return launch_norm<E, Y, LAYER, false, 4, 8, 1024, 1>(a, stream);
  }
  if (a.width <= 256) return launch_norm<E, Y, LAYER, true, 8, 1, 256, 4>(a, stream);
  if (a.width <= 4096) return launch_norm<E, Y, LAYER, false, 8, 1, 512, 2>(a, stream);
  return launch_norm<E, Y, LAYER, false, 32, 1, 1024, 1>(a, stream);
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
