// The paged cache's bookkeeping and writes: block tables and slot maps of a step
// (tr_plan_step), pages given back (tr_release_pages), keys and values written to their slots
// (tr_append_kv).
#include <cooperative_groups.h>

#include <algorithm>

#include "serve_util.cuh"
#include "tc_util.cuh"

namespace cg = cooperative_groups;

namespace trr {

struct StepArgs {
  const int32_t* lens;
  const int32_t* brings;
  int32_t* tables;
  int64_t table_stride;
  const int32_t* free_pages;
  const int32_t* free_count;
  int64_t* slots;
  int32_t* positions;
  int32_t* starts;
  int32_t* lens_out;
  int32_t* granted;
  int32_t* free_count_out;
  int64_t pool, tokens;
  int requests, columns, page;
};

constexpr int kStepThreads = 1024;

__device__ __forceinline__ int64_t pages_of(int64_t n, int page) { return (n + page - 1) / page; }

// What a block keeps of every request, in shared memory.
struct StepRequest {
  int32_t* start;  // [requests + 1] first token
  int32_t* base;   // [requests] pages given before this request's; -1 refused
  int32_t* len;    // [requests] tokens cached
};

// Every block of the one cluster runs the same two prefix sums over the requests (tokens, then
// pages needed), which costs less than a second launch or a barrier to share them, and then
// takes its share of the tables' new entries and of the step's tokens, four a thread: the
// first one's request by bisection of the starts in shared memory, the others from there.  A
// token's page is read from the table when the request held it before, else from the free
// stack, so no block waits for the entries another writes.  What the caller may ask for in
// place (lens, free_count) is written once every block has read it: the arrival at the cluster
// barrier stands behind the last read, the wait before the write.  Lengths are below 2^31, so
// length + tokens and its pages are exact in 32 unsigned bits.
// Bound by latency: launch, lengths, two scans, a dependent page, the stores.  256 requests with
// a token each: 6 us of the device's time, of which an empty kernel takes 2; 500 prompts of 53687
// tokens: 12 us.
__global__ void __launch_bounds__(kStepThreads, 1) plan_step_kernel(const StepArgs a) {
  extern __shared__ int32_t step_smem[];
  const StepRequest q = {step_smem, step_smem + a.requests + 1, step_smem + 2 * a.requests + 1};
  __shared__ int64_t part[32];
  __shared__ int used;
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int tid = threadIdx.x, threads = blockDim.x;
  const uint32_t page = a.page;
  const auto pages = [&](uint32_t n) { return n / page + (n % page != 0); };
  if (tid == 0) used = 0;
  const int64_t fc = min(max((int64_t)*a.free_count, (int64_t)0), a.pool);
  int64_t tokens_before = 0, need_before = 0;
  for (int r0 = 0; r0 < a.requests; r0 += threads) {
    const int r = r0 + tid;
    const bool live = r < a.requests;
    const uint32_t len = live ? max(a.lens[r], 0) : 0, n = live ? max(a.brings[r], 0) : 0;
    int64_t total;
    const int64_t through = block_scan_inclusive((int64_t)n, part, total) + tokens_before;
    tokens_before += total;
    const uint32_t held = pages(len), wants = pages(len + n);
    const bool fits = live && wants <= (uint32_t)a.columns && through <= a.tokens;
    const int64_t need = fits ? wants - held : 0;
    const int64_t taken = block_scan_inclusive(need, part, total) + need_before;
    need_before += total;
    const bool ok = fits && (need == 0 || taken <= fc);
    if (live) {
      q.start[r] = (int32_t)min(through - n, (int64_t)INT32_MAX);
      q.base[r] = ok ? (int32_t)(taken - need) : -1;
      q.len[r] = (int32_t)len;
      if (ok && need > 0) atomicMax(&used, (int)taken);
    }
  }
  if (tid == 0) q.start[a.requests] = (int32_t)min(tokens_before, (int64_t)INT32_MAX);
  __syncthreads();
  cluster_arrive_release();

  // new table entries: a thread per request where no block has more than one each, else a warp
  const bool short_ones = a.requests <= threads;
  const int lane = short_ones ? 0 : tid & 31, lanes = short_ones ? 1 : 32;
  const int groups = threads / lanes;
  for (int r = rank * groups + (short_ones ? tid : tid >> 5); r < a.requests; r += ranks * groups) {
    const int b = q.base[r];
    if (b < 0) continue;
    const uint32_t len = q.len[r];
    const int held = (int)pages(len), wants = (int)pages(len + (uint32_t)(q.start[r + 1] - q.start[r]));
    for (int c = held + lane; c < wants; c += lanes)
      a.tables[r * a.table_stride + c] = a.free_pages[fc - 1 - (b + c - held)];
  }
  const int tokens_end = q.start[a.requests];
  for (int64_t i0 = 4 * ((int64_t)rank * threads + tid); i0 < a.tokens;
       i0 += 4 * (int64_t)ranks * threads) {
    int64_t slot[4];
    int32_t position[4];
    int r = 0;
    if (i0 < tokens_end) {  // the last request that starts at or before i0
      int hi = a.requests;
      while (hi - r > 1) {
        const int mid = (r + hi) >> 1;
        if (q.start[mid] <= i0) r = mid;
        else hi = mid;
      }
    }
    int at_request = -1;
    uint32_t at_page = 0;
    int64_t id = -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = i0 + j;
      slot[j] = -1;
      position[j] = -1;
      if (i >= tokens_end) continue;
      while (q.start[r + 1] <= i) ++r;
      if (q.base[r] < 0) continue;
      const uint32_t len = q.len[r], p = len + (uint32_t)(i - q.start[r]), c = p / page;
      if (r != at_request || c != at_page) {
        const uint32_t held = pages(len);
        id = c < held ? a.tables[r * a.table_stride + c]
                      : a.free_pages[fc - 1 - (int64_t)(q.base[r] + c - held)];
        at_request = r;
        at_page = c;
      }
      slot[j] = id * page + (p - c * page);
      position[j] = (int32_t)p;
    }
    if (i0 + 4 <= a.tokens && (((uintptr_t)a.slots | (uintptr_t)a.positions) & 15) == 0) {
      reinterpret_cast<longlong2*>(a.slots + i0)[0] = make_longlong2(slot[0], slot[1]);
      reinterpret_cast<longlong2*>(a.slots + i0)[1] = make_longlong2(slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.positions + i0) =
          make_int4(position[0], position[1], position[2], position[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j < a.tokens) {
          a.slots[i0 + j] = slot[j];
          a.positions[i0 + j] = position[j];
        }
    }
  }
  cluster_wait_acquire();
  for (int r = rank * threads + tid; r < a.requests; r += ranks * threads) {
    const int n = q.start[r + 1] - q.start[r], len = a.lens[r];
    a.starts[r] = q.start[r];
    a.granted[r] = q.base[r] >= 0;
    a.lens_out[r] = q.base[r] >= 0 ? q.len[r] + n : len;
  }
  if (rank == 0 && tid == 0) {
    a.starts[a.requests] = q.start[a.requests];
    *a.free_count_out = (int32_t)(fc - used);
  }
}

struct ReleaseArgs {
  int32_t* lens;
  const int32_t* finished;
  int32_t* tables;
  int64_t table_stride;
  int32_t* free_pages;
  int32_t* free_count;
  int64_t pool;
  int requests, columns, page;
};

// As plan_step_kernel: the prefix sum of the pages given back in every block, then a warp per
// request moves them.
__global__ void __launch_bounds__(kStepThreads, 1) release_pages_kernel(const ReleaseArgs a) {
  extern __shared__ int32_t step_smem[];  // [requests] pages given back before this request's
  __shared__ int64_t part[32];
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int tid = threadIdx.x;
  const int64_t fc = min(max((int64_t)*a.free_count, (int64_t)0), a.pool);
  const auto held = [&](int r) {
    return a.finished[r] ? min(pages_of(max(a.lens[r], 0), a.page), (int64_t)a.columns)
                         : (int64_t)0;
  };
  int64_t before = 0;
  for (int r0 = 0; r0 < a.requests; r0 += kStepThreads) {
    const int r = r0 + tid;
    const int64_t n = r < a.requests ? held(r) : 0;
    int64_t total;
    const int64_t through = block_scan_inclusive(n, part, total) + before;
    before += total;
    if (r < a.requests) step_smem[r] = (int32_t)min(through - n, a.pool);
  }
  __syncthreads();
  const int warps = kStepThreads / 32, lane = tid & 31;
  for (int r = rank * warps + (tid >> 5); r < a.requests; r += ranks * warps) {
    const int n = (int)held(r);
    for (int c = lane; c < n; c += 32) {
      const int64_t at = fc + step_smem[r] + c;
      int32_t* entry = a.tables + r * a.table_stride + c;
      if (at < a.pool) a.free_pages[at] = *entry;
      *entry = -1;
    }
  }
  cluster.sync();
  if (rank == 0) {
    for (int r = tid; r < a.requests; r += kStepThreads)
      if (a.finished[r]) a.lens[r] = 0;
    if (tid == 0) *a.free_count = (int32_t)min(fc + before, a.pool);
  }
}

// One launch of a single cluster of `blocks`, with ints_per_request of shared memory a request and
// one more.  The default limit of 48 KB is for the kernel's own variables and these together; past
// 40 KB it is raised, to the same size whatever the call, so that calls of several threads do not
// lower it under one another.
template <typename Args>
static int launch_cluster(void (*kernel)(Args), const Args& args, int blocks, int threads,
                          int ints_per_request, void* stream, const char* what) {
  const size_t smem = (ints_per_request * (size_t)args.requests + 1) * sizeof(int32_t);
  if (smem > 40 * 1024) {
    const int most = (ints_per_request * TR_STEP_MAX_REQUESTS + 1) * (int)sizeof(int32_t);
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) {
      set_error("%s: %d bytes of shared memory: %s", what, most, cudaGetErrorString(e));
      return TR_ERR_CUDA;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = blocks > 1 ? 1 : 0;  // a single block is a cluster of its own
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  if (e != cudaSuccess) {
    set_error("%s launch: %s", what, cudaGetErrorString(e));
    (void)cudaGetLastError();
    return TR_ERR_CUDA;
  }
  return TR_OK;
}

// ---- tr_append_kv
struct AppendArgs {
  const void* k;
  const void* v;
  void* k_pages;
  void* v_pages;
  int64_t k_token, k_head, v_token, v_head;  // source strides
  const int64_t* slots;
  int64_t tokens, slots_end;
  int heads, dim, page;
  int page_shift;              // of a page size that is a power of two, else -1
  int step_tokens, step_rest;  // what a grid's stride of vectors is in tokens and the rest
};

// One thread per 8 elements (V = 8, 16-byte stores) or per element (V = 1, when a source row is
// not 16-byte aligned) of both keys and values; four of them at a time, so that their slots,
// then their sources, are in flight together.  The token and head of a vector are divided out
// once and carried on.  Bound by memory at large sizes, by the launch at small ones: 32771 tokens
// of 8 heads of 128 from fp32 take 66 us (6.1 TB/s; 84 us with one vector at a time), 128 from
// bf16 2.2 us.  A source of the pools' own 16 bits passes through fp32 registers too and so has
// half as many bytes in flight: 32768 tokens from bf16 66 us (4.1 TB/s).
template <typename S, typename E, int V>
__global__ void __launch_bounds__(256) append_kv_kernel(const AppendArgs a) {
  constexpr int U = 4;
  const int per_head = a.dim / V, per_token = a.heads * per_head;
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  int64_t t = i / per_token;
  int rest = (int)(i - t * per_token);
  while (t < a.tokens) {
    int64_t token[U], slot[U];
    int in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      token[u] = t;
      in[u] = rest;
      slot[u] = t < a.tokens ? a.slots[t] : -1;
      t += a.step_tokens;
      rest += a.step_rest;
      if (rest >= per_token) rest -= per_token, ++t;
    }
    float f[U][2][V];
    int64_t to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      to[u] = -1;
      if (slot[u] < 0 || slot[u] >= a.slots_end) continue;
      const int h = in[u] / per_head, d = (in[u] - h * per_head) * V;
      const int64_t page = a.page_shift >= 0 ? slot[u] >> a.page_shift : slot[u] / a.page;
      to[u] = ((page * a.heads + h) * a.page + (slot[u] - page * a.page)) * a.dim + d;
      const S* k = static_cast<const S*>(a.k) + token[u] * a.k_token + h * a.k_head + d;
      const S* v = static_cast<const S*>(a.v) + token[u] * a.v_token + h * a.v_head + d;
      if constexpr (V == 8) {
        load8<S>(k, f[u][0]);
        load8<S>(v, f[u][1]);
      } else {
        f[u][0][0] = to_f32<S>(*k);
        f[u][1][0] = to_f32<S>(*v);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (to[u] < 0) continue;
      E* k = static_cast<E*>(a.k_pages) + to[u];
      E* v = static_cast<E*>(a.v_pages) + to[u];
      if constexpr (V == 8) {
        store8<E>(k, f[u][0]);
        store8<E>(v, f[u][1]);
      } else {
        *k = from_f32<E>(f[u][0][0]);
        *v = from_f32<E>(f[u][1][0]);
      }
    }
  }
}

template <typename S, typename E>
static int launch_append(AppendArgs a, bool wide, void* stream) {
  const int64_t per_token = (int64_t)a.heads * (a.dim / (wide ? 8 : 1));
  const int64_t n = a.tokens * per_token;
  const int64_t blocks = std::min<int64_t>((n + 255) / 256, (int64_t)serve_sms() * 8);
  a.step_tokens = (int)(blocks * 256 / per_token);
  a.step_rest = (int)(blocks * 256 % per_token);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (wide) append_kv_kernel<S, E, 8><<<(unsigned)blocks, 256, 0, s>>>(a);
  else append_kv_kernel<S, E, 1><<<(unsigned)blocks, 256, 0, s>>>(a);
  return serve_launched("tr_append_kv");
}

}  // namespace trr

using namespace trr;

static int check_step(const char* what, int64_t requests, const void* a, const void* b,
                      const void* tables, int64_t table_stride, int32_t columns,
                      const void* free_pages, int64_t pool, const void* free_count,
                      int32_t page_size) {
  if (requests < 0 || columns < 0 || pool < 0 || page_size < 1) {
    set_error("%s: negative size, or page_size %d below 1", what, (int)page_size);
    return TR_ERR_INVALID;
  }
  if (requests > 1 && table_stride < columns) {
    set_error("%s: table stride %lld below its %d columns", what, (long long)table_stride,
              (int)columns);
    return TR_ERR_INVALID;
  }
  if (pool > INT32_MAX) {
    set_error("%s: pool of %lld pages (at most 2^31 - 1)", what, (long long)pool);
    return TR_ERR_INVALID;
  }
  if (requests > TR_STEP_MAX_REQUESTS) {
    set_error("%s: %lld requests (at most %d)", what, (long long)requests, TR_STEP_MAX_REQUESTS);
    return TR_ERR_UNSUPPORTED;
  }
  if ((requests > 0 && (!a || !b || (columns > 0 && !tables))) || (pool > 0 && !free_pages) ||
      !free_count) {
    set_error("%s: null pointer", what);
    return TR_ERR_INVALID;
  }
  if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)tables | (uintptr_t)free_pages |
       (uintptr_t)free_count) & 3) {
    set_error("%s: a pointer is not aligned to its elements", what);
    return TR_ERR_ALIGN;
  }
  return TR_OK;
}

extern "C" int tr_plan_step(const int32_t* lens, const int32_t* new_tokens, int64_t requests,
                            int32_t* tables, int64_t table_stride, int32_t columns,
                            const int32_t* free_pages, int64_t pool, const int32_t* free_count,
                            int32_t page_size, int64_t tokens, int64_t* slots, int32_t* positions,
                            int32_t* starts, int32_t* lens_out, int32_t* granted,
                            int32_t* free_count_out, void* stream) {
  const int st = check_step("tr_plan_step", requests, lens, new_tokens, tables, table_stride,
                            columns, free_pages, pool, free_count, page_size);
  if (st != TR_OK) return st;
  if (tokens < 0 || tokens > INT32_MAX) {
    set_error("tr_plan_step: %lld tokens (0 to 2^31 - 1)", (long long)tokens);
    return TR_ERR_INVALID;
  }
  if (!starts || !free_count_out || (requests > 0 && (!lens_out || !granted)) ||
      (tokens > 0 && (!slots || !positions))) {
    set_error("tr_plan_step: null output");
    return TR_ERR_INVALID;
  }
  if ((((uintptr_t)positions | (uintptr_t)starts | (uintptr_t)lens_out | (uintptr_t)granted |
        (uintptr_t)free_count_out) & 3) || ((uintptr_t)slots & 7)) {
    set_error("tr_plan_step: an output is not aligned to its elements");
    return TR_ERR_ALIGN;
  }
  StepArgs a = {lens, new_tokens, tables, table_stride, free_pages, free_count, slots, positions,
                starts, lens_out, granted, free_count_out, pool, tokens, (int)requests, columns,
                page_size};
  // One block serves a decode step, of as many threads as it has requests or groups of four tokens
  // (barriers of fewer warps are cheaper); the cluster of 8 pays its barrier back from a few tokens
  // per thread on.  256 requests, us a call with one block / eight: 256 tokens 7.3 / 8.3, 4096
  // 8.3 / 8.3, 8192 10.6 / 8.3, 16384 16.1 / 8.3; 8 requests: 8192 14.4 / 12.4, 16384 22.5 / 16.5;
  // 500 requests of 53687 tokens 45.2 / 13.4.
  const int64_t work = std::max(requests, tokens / 4);
  const int blocks = tokens > 8 * kStepThreads ? 8 : 1;
  const int threads = blocks > 1 || work > 512 ? kStepThreads : work > 256 ? 512 : 256;
  return launch_cluster(plan_step_kernel, a, blocks, threads, 3, stream, "tr_plan_step");
}

extern "C" int tr_release_pages(int32_t* lens, const int32_t* finished, int64_t requests,
                                int32_t* tables, int64_t table_stride, int32_t columns,
                                int32_t* free_pages, int64_t pool, int32_t* free_count,
                                int32_t page_size, void* stream) {
  const int st = check_step("tr_release_pages", requests, lens, finished, tables, table_stride,
                            columns, free_pages, pool, free_count, page_size);
  if (st != TR_OK || requests == 0) return st;
  ReleaseArgs a = {lens, finished, tables, table_stride, free_pages, free_count, pool,
                   (int)requests, columns, page_size};
  // us a call with one block / eight, all requests finished: 64 of 8 columns 4.2 / 3.9, of 64
  // 4.7 / 5.0, 256 of 16 7.9 / 4.3, of 64 9.0 / 4.6, of 512 30.7 / 7.4
  const int blocks = requests * columns > 4 * kStepThreads ? 8 : 1;
  return launch_cluster(release_pages_kernel, a, blocks, kStepThreads, 1, stream,
                        "tr_release_pages");
}

extern "C" int tr_append_kv(const void* k, int64_t k_token_stride, int64_t k_head_stride,
                            const void* v, int64_t v_token_stride, int64_t v_head_stride,
                            int32_t src_dtype, void* k_pages, void* v_pages, int32_t dtype,
                            const int64_t* slots, int64_t tokens, int32_t kv_heads,
                            int32_t head_dim, int64_t pages, int32_t page_size, void* stream) {
  if (!known_dtype(dtype) || (src_dtype != dtype && src_dtype != TR_F32)) {
    set_error("tr_append_kv: source dtype %d into dtype %d", (int)src_dtype, (int)dtype);
    return TR_ERR_INVALID;
  }
  if (tokens < 0 || kv_heads < 1 || head_dim < 1 || pages < 0 || page_size < 1 ||
      (int64_t)kv_heads * head_dim > INT32_MAX) {
    set_error("tr_append_kv: bad shape");
    return TR_ERR_INVALID;
  }
  if (tokens == 0 || pages == 0) return TR_OK;
  if (!k || !v || !k_pages || !v_pages || !slots) {
    set_error("tr_append_kv: null pointer");
    return TR_ERR_INVALID;
  }
  const int sb = element_bytes(src_dtype);
  if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) {
    set_error("tr_append_kv: the pools must be 16-byte aligned");
    return TR_ERR_ALIGN;
  }
  if ((((uintptr_t)k | (uintptr_t)v) & (sb - 1)) || ((uintptr_t)slots & 7)) {
    set_error("tr_append_kv: a pointer is not aligned to its elements");
    return TR_ERR_ALIGN;
  }
  AppendArgs a = {k, v, k_pages, v_pages, k_token_stride, k_head_stride, v_token_stride,
                  v_head_stride, slots, tokens, pages * page_size, kv_heads, head_dim, page_size,
                  page_size & (page_size - 1) ? -1 : __builtin_ctz(page_size), 0, 0};
  const bool wide = head_dim % 8 == 0 && !(((uintptr_t)k | (uintptr_t)v) & 15) &&
                    !((k_token_stride * sb | k_head_stride * sb | v_token_stride * sb |
                       v_head_stride * sb) & 15);
  if (src_dtype == TR_F32) {
    if (dtype == TR_F32) return launch_append<float, float>(a, wide, stream);
    if (dtype == TR_F16) return launch_append<float, __half>(a, wide, stream);
    return launch_append<float, __nv_bfloat16>(a, wide, stream);
  }
  if (dtype == TR_F16) return launch_append<__half, __half>(a, wide, stream);
  return launch_append<__nv_bfloat16, __nv_bfloat16>(a, wide, stream);
}
