// Shared by the paged-attention kernels (serve_attend.cu, serve_attend_rows.cu,
// serve_attend_chunk.cu).
#pragma once

#include "serve_util.cuh"

namespace trr {

// The request of token t: the last one that starts at or before it, or -1 outside all of them.
__device__ __forceinline__ int owner_of(const int32_t* starts, int requests, int64_t t) {
  if (requests == 0 || t < starts[0] || t >= starts[requests]) return -1;
  int lo = 0, hi = requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Tokens a request brings and keys it has, kept inside the arrays whatever starts and lens hold.
__device__ __forceinline__ int brought(const tr_attention& a, int r) {
  const int64_t first = max((int64_t)a.starts[r], (int64_t)0);
  return (int)min(max((int64_t)a.starts[r + 1] - first, (int64_t)0), max(a.tokens - first, (int64_t)0));
}
__device__ __forceinline__ int cached(const tr_attention& a, int r) {
  return (int)min((int64_t)max(a.lens[r], 0), (int64_t)a.columns * a.page_size);
}
// Keys that token i of request r's n sees: lens[r] - n + i + 1, at most those cached.
__device__ __forceinline__ int visible(const tr_attention& a, int r, int n, int i) {
  return (int)min((int64_t)a.lens[r] - n + i + 1, (int64_t)cached(a, r));
}

// 16 bytes global -> shared, asynchronously; zeros when !held (src is then not read)
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, bool held) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src),
               "r"(held ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

// Zeros and -inf for the tokens outside [starts[0], starts[requests]); `thread` of `threads`.
template <typename E>
__device__ void clear_outside(const tr_attention& a, int64_t thread, int64_t threads) {
  const int64_t first = a.requests ? min(max((int64_t)a.starts[0], (int64_t)0), a.tokens) : a.tokens;
  const int64_t end = a.requests ? min(max((int64_t)a.starts[a.requests], first), a.tokens) : a.tokens;
  const int64_t outside = first + (a.tokens - end);
  const int64_t per = (int64_t)a.heads * a.head_dim / 8;
  for (int64_t i = thread; i < outside * per; i += threads) {
    const int64_t n = i / per, t = n < first ? n : end + (n - first);
    reinterpret_cast<uint4*>(a.out)[t * per + (i - n * per)] = make_uint4(0, 0, 0, 0);
  }
  if (a.lse)
    for (int64_t i = thread; i < outside * a.heads; i += threads) {
      const int64_t n = i / a.heads, t = n < first ? n : end + (n - first);
      a.lse[t * a.heads + (i - n * a.heads)] = -INFINITY;
    }
}

// NaN for `rows` rows from row `row0` of kv head kvh of a request (16-bit types; 0x7fff is NaN in
// both).  A call that timed out leaves arrival counters behind that are not zero, so neither what it
// did not finish nor what later calls would join by them may pass for a result: those items are
// spoiled, by the block whose run they are in, until the workspace's state is zeroed.
__device__ __forceinline__ void spoil_rows(const tr_attention& a, int64_t token0, int kvh, int g,
                                           int row0, int rows) {
  const int per = a.head_dim / 8;
#pragma unroll 1
  for (int j = threadIdx.x; j < rows * per; j += blockDim.x) {
    const int row = row0 + j / per, i = row / g, h = kvh * g + (row - i * g);
    const int64_t at = (token0 + i) * a.heads + h;
    reinterpret_cast<uint4*>(a.out)[at * per + j % per] =
        make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
    if (a.lse && j % per == 0) a.lse[at] = __int_as_float(0x7fffffff);
  }
}

// The workspace: the status word (tr_workspace_status), the arrival counters of the items, which
// are zero between calls, and the partial results, which need not be.  The first two have a size
// of their own, so that calls of any shapes can follow one another.
constexpr int64_t kAttendCounters = (TR_ATTENTION_STATE_BYTES - 256) / sizeof(int);
struct AttendWorkspace {
  int* status;
  int* counters;
  float* partials;
};

// serve_attend_rows.cu, serve_attend_chunk.cu: counters and bytes of partial results of a call
int64_t attend_rows_items(const tr_attention& a);
size_t attend_rows_partials(const tr_attention& a);
int launch_attend_rows(const tr_attention& a, const AttendWorkspace& ws, void* stream);
int64_t attend_chunk_items(const tr_attention& a);
size_t attend_chunk_partials(const tr_attention& a);
int launch_attend_chunk(const tr_attention& a, const AttendWorkspace& ws, void* stream);

}  // namespace trr
