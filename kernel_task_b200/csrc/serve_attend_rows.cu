// Paged attention for few query rows per request and kv head: decoding, and short chunks.
// 61 requests with contexts of up to 16384 tokens, 32 heads over 8 of 128: 243 us, 6.25 TB/s of the
// 6.45 that a copy has; one of 777 tokens: 13 us, the latency of some ten dependent steps.
//
// The keys and values of a request are read once for all the query heads that share them, and
// that reading is the bound (two operations a byte and row).  A row is one token and query head;
// the rows of a request over one kv head are cut into tiles of 8 or 16.
//
// Products.  S^T = K Q^T and O^T += V^T P^T, so that keys (then head_dim) lie along the 16 rows
// of mma.sync m16n8k16 and the query rows along its 8 columns: with 4 to 8 query heads per kv
// head a tile of 8 is mostly full, where Q K^T would fill 16 rows with them.  Each warp takes
// its own 16 or 32 keys of a block, with its own running maximum, sum and output, so the loop
// has no block barrier; the four warps' results are joined at the end of the item.
//
// Split.  An item is (request, row tile, kv head), a unit one block of keys of an item.  The
// blocks of the grid take equal contiguous runs of all units, found by one prefix sum over the
// requests, so ragged lengths balance to within a block of keys without the host knowing them.
// Each warp's loads run two blocks ahead along the run, over the ends of items too: with short
// contexts an item is over in the time of one memory access.
// An item that several blocks share leaves fp32 partial results in the workspace; the last block
// to arrive joins them in unit order, so the result does not depend on the order of arrival.
#include <algorithm>

#include "serve_attend.cuh"
#include "tc_util.cuh"

namespace trr {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = 32 * kRowsWarps;
// stages of a warp: three, or two for tiles of 16 rows, whose exchange buffer takes the third's room
template <int NT>
__host__ __device__ constexpr int rows_stages() {
  return NT == 1 ? 3 : 2;
}

// 16 keys of 128 elements or 32 of 64: 8 KB of keys and values a warp and stage
template <int D>
__host__ __device__ constexpr int warp_keys() {
  return D == 128 ? 16 : 32;
}
template <int D>
__host__ __device__ constexpr int block_keys() {
  return kRowsWarps * warp_keys<D>();
}

__host__ __device__ constexpr int partial_floats(int rows, int D) { return rows * (D + 2); }

__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_addr(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}

// Walks the items of a contiguous run of units.
struct RowsItem {
  int request, rows, tiles, tile, kvh;
  int blocks;      // units of the item: blocks of keys, at least one (rows without keys are written too)
  int see0, cap;   // token i of the request sees min(see0 + i, cap) keys (none if negative)
  int64_t token0;  // the request's first token
  int64_t u0;      // first unit of the item
  int64_t index;   // item number
};
template <int ROWS, int BK>
__device__ __forceinline__ void open_request(const tr_attention& a, int g, RowsItem& it, int r) {
  const int n = brought(a, r);
  it.request = r;
  it.rows = n * g;
  it.tiles = (it.rows + ROWS - 1) / ROWS;
  it.tile = it.kvh = 0;
  it.cap = cached(a, r);
  it.blocks = max((it.cap + BK - 1) / BK, 1);
  it.see0 = (int)max((int64_t)a.lens[r] - n + 1, -(int64_t)(1 << 30));
  it.token0 = max((int64_t)a.starts[r], (int64_t)0);
}
template <int ROWS, int BK>
__device__ __forceinline__ void next_item(const tr_attention& a, int g, RowsItem& it) {
  it.u0 += it.blocks;
  ++it.index;
  if (++it.kvh < a.kv_heads) return;
  it.kvh = 0;
  if (++it.tile < it.tiles) return;
  while (it.request + 1 < (int)a.requests) {
    open_request<ROWS, BK>(a, g, it, it.request + 1);
    if (it.tiles) return;
  }
}
__device__ __forceinline__ int keys_of_row(const RowsItem& it, int g, int row) {
  return max(min(it.see0 + row / g, it.cap), 0);
}

// The run of units of this block, and the item it starts in; false when there is none.  Up to 32
// requests every warp sums them by itself, else thread i takes requests [i per, (i + 1) per).
template <int ROWS, int BK>
__device__ __forceinline__ bool find_run(const tr_attention& a, int g, int64_t max_items,
                                         int64_t (&part)[2][32], RowsItem& first, int64_t& U,
                                         int64_t& G, int64_t& u_begin, int64_t& u_end) {
  const int R = (int)a.requests, lane = threadIdx.x & 31;
  const bool few = R <= 32;
  const int workers = few ? 32 : (int)blockDim.x, me = few ? lane : (int)threadIdx.x;
  const int per = (R + workers - 1) / workers;
  const int r_lo = min(me * per, R), r_hi = min(r_lo + per, R);
  RowsItem it;
  int64_t my_units = 0, my_items = 0;
  for (int r = r_lo; r < r_hi; ++r) {
    open_request<ROWS, BK>(a, g, it, r);
    my_items += (int64_t)it.tiles * a.kv_heads;
    my_units += (int64_t)it.tiles * a.kv_heads * it.blocks;
  }
  int64_t through, items_through, items;
  if (few) {
    through = warp_scan_inclusive(my_units);
    items_through = warp_scan_inclusive(my_items);
    U = __shfl_sync(0xffffffffu, through, 31);
    items = __shfl_sync(0xffffffffu, items_through, 31);
  } else {
    through = block_scan_inclusive(my_units, part[0], U);
    items_through = block_scan_inclusive(my_items, part[1], items);
  }
  if (U == 0 || items > max_items) return false;
  // Blocks to share the units: a part of an item costs the block that joins it about a third of
  // a block of keys, so an item of b blocks is best cut into sqrt(3 b) parts (one request of
  // 32768 keys over one kv head: 60 us, 77 us on all blocks of the grid)
  G = min(min((int64_t)gridDim.x, U), (int64_t)ceilf(sqrtf(3.f * (float)U * (float)items)));
  if (blockIdx.x >= G) return false;
  u_begin = U * blockIdx.x / G;
  u_end = U * (blockIdx.x + 1) / G;
  const bool mine = through - my_units <= u_begin && u_begin < through;
  int64_t u0 = through - my_units, index = items_through - my_items;
  int request = r_lo;
  if (mine) {
    for (; request < r_hi; ++request) {
      open_request<ROWS, BK>(a, g, it, request);
      const int64_t units = (int64_t)it.tiles * a.kv_heads * it.blocks;
      if (u_begin < u0 + units) break;
      u0 += units;
      index += (int64_t)it.tiles * a.kv_heads;
    }
  }
  if (few) {
    const int who = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
    request = __shfl_sync(0xffffffffu, request, who);
    u0 = __shfl_sync(0xffffffffu, u0, who);
    index = __shfl_sync(0xffffffffu, index, who);
  } else {
    if (mine) part[0][0] = u0, part[0][1] = index, part[0][2] = request;
    __syncthreads();
    u0 = part[0][0], index = part[0][1], request = (int)part[0][2];
  }
  open_request<ROWS, BK>(a, g, first, request);
  const int item = (int)((u_begin - u0) / first.blocks);
  first.u0 = u0 + (int64_t)item * first.blocks;
  first.index = index + item;
  first.tile = item / a.kv_heads;
  first.kvh = item - first.tile * a.kv_heads;
  return true;
}

template <typename E, int D, int NT>
__global__ void __launch_bounds__(kRowsThreads, 2) attend_rows_kernel(const tr_attention a,
                                                                     const int* status,
                                                                     int* counters,
                                                                     int64_t max_items,
                                                                     float* partials) {
  constexpr int ROWS = 8 * NT, WK = warp_keys<D>(), MT = WK / 16, BK = block_keys<D>();
  constexpr int STAGES = rows_stages<NT>();
  constexpr int CPR = D / 8;                // 16-byte chunks of a row
  constexpr int STAGE = 2 * WK * D * 2;     // bytes of a warp's stage: keys, then values
  constexpr int F = D / 16 / kRowsWarps;    // 16-element slices of the output that a warp ends with
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int64_t part[2][32];
  __shared__ float sh_m[kRowsWarps][ROWS], sh_l[kRowsWarps][ROWS];
  __shared__ int sh_last;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = a.heads / a.kv_heads;
  const int timed_out = __ldcg(status);  // of an earlier call; on its way while the run is found
  clear_outside<E>(a, (int64_t)blockIdx.x * kRowsThreads + tid, (int64_t)gridDim.x * kRowsThreads);
  if (a.requests == 0) return;
  RowsItem it;
  int64_t U, G, u_begin, u_end;
  if (!find_run<ROWS, BK>(a, g, max_items, part, it, U, G, u_begin, u_end)) return;
  if (timed_out) {
    for (; it.u0 < u_end; next_item<ROWS, BK>(a, g, it))
      spoil_rows(a, it.token0, it.kvh, g, it.tile * ROWS, min(ROWS, it.rows - it.tile * ROWS));
    return;
  }

  const uint32_t stage0 = smem_u32(smem) + warp * STAGES * STAGE;
  float4* exchange = reinterpret_cast<float4*>(smem + kRowsWarps * STAGES * STAGE);
  const uint4* kp = static_cast<const uint4*>(a.k_pages);
  const uint4* vp = static_cast<const uint4*>(a.v_pages);
  const float scale2 = a.scale * kLog2e;
  const int page_shift = 31 - __clz(a.page_size);

  // ---- loads.  `ahead` is the item of unit `lu`, the next to load; `rows_next` the pool rows of
  // its keys (lane i < WK: the warp's key i), ~0u past the keys and for bad pages
  RowsItem ahead = it;
  int64_t lu = u_begin;
  uint32_t rows_next = ~0u;
  int keys_ahead = 0;
  const auto open_ahead = [&] {
    keys_ahead = keys_of_row(ahead, g, min((ahead.tile + 1) * ROWS, ahead.rows) - 1);
  };
  const auto find_rows = [&] {
    const int key = (int)(lu - ahead.u0) * BK + warp * WK + lane;
    rows_next = ~0u;
    if (lu < u_end && lane < WK && key < keys_ahead) {
      const int id = a.tables[ahead.request * a.table_stride + (key >> page_shift)];
      if (id >= 0 && id < a.pages)
        rows_next = (uint32_t)((id * (int64_t)a.kv_heads + ahead.kvh) * a.page_size +
                               (key & (a.page_size - 1)));
    }
  };
  const auto load = [&] {  // one commit group, empty past the run
    if (lu < u_end) {
      const uint32_t base = stage0 + (uint32_t)(lu - u_begin) % STAGES * STAGE;
#pragma unroll
      for (int i = 0; i < WK * CPR / 32; ++i) {
        const int row = i * (32 / CPR) + lane / CPR, c = lane % CPR;
        const uint32_t r = __shfl_sync(0xffffffffu, rows_next, row);
        const bool held = r != ~0u;
        const uint64_t at = (uint64_t)(held ? r : 0u) * CPR + c;
        const uint32_t dst = base + row * (D * 2) + ((c ^ (row & 7)) << 4);
        copy16_async(dst, kp + at, held);
        copy16_async(dst + WK * D * 2, vp + at, held);
      }
      if (++lu == ahead.u0 + ahead.blocks && lu < u_end) {
        next_item<ROWS, BK>(a, g, ahead);
        open_ahead();
      }
      find_rows();
    }
    copies_commit();
  };
  open_ahead();
  find_rows();
#pragma unroll 1
  for (int s = 0; s < STAGES - 1; ++s) load();

  for (int64_t u = u_begin; u < u_end; next_item<ROWS, BK>(a, g, it)) {
    const int b_first = (int)(u - it.u0);
    const int b_last = (int)min((int64_t)it.blocks, b_first + (u_end - u));  // one past
    const int rows_here = min(ROWS, it.rows - it.tile * ROWS);

    // the two query rows of this lane's columns, per n-tile: how many keys they see
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nt * 8 + (lane & 3) * 2 + e;
        limit[nt][e] = row < rows_here ? keys_of_row(it, g, it.tile * ROWS + row) : 0;
      }

    // Q^T fragments: row lane / 4, elements ks * 16 + (lane & 3) * 2 (+1, +8, +9)
    uint32_t qf[NT][D / 16][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = nt * 8 + (lane >> 2), at = it.tile * ROWS + row;
      const int i = at / g, h = it.kvh * g + (at - i * g);
      const E* q = static_cast<const E*>(a.q) + (it.token0 + i) * a.q_token_stride +
                   h * a.q_head_stride + (lane & 3) * 2;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[nt][ks][0] = row < rows_here ? *reinterpret_cast<const uint32_t*>(q + ks * 16) : 0u;
        qf[nt][ks][1] = row < rows_here ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + 8) : 0u;
      }
    }

    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) m[nt][e] = -INFINITY, l[nt][e] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
    }

    for (int b = b_first; b < b_last; ++b, ++u) {
      load();
      copies_wait<STAGES - 1>();
      __syncwarp();
      const uint32_t ks0 = stage0 + (uint32_t)(u - u_begin) % STAGES * STAGE, vs0 = ks0 + WK * D * 2;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
        const int krow = mt * 16 + (lane & 15);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t kf[4];
          ldsm_x4_addr(kf, ks0 + krow * (D * 2) + (((ks * 2 + (lane >> 4)) ^ (krow & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt], kf, qf[nt][ks][0], qf[nt][ks][1], E());
        }
        const int key = b * BK + warp * WK + mt * 16 + (lane >> 2);
        uint32_t pf[NT][2];
        bool moved = false;
        float keep[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& s0 = s[nt][e];
            float& s1 = s[nt][e + 2];
            s0 = key < limit[nt][e] ? s0 * scale2 : -INFINITY;
            s1 = key + 8 < limit[nt][e] ? s1 * scale2 : -INFINITY;
            float top = fmaxf(s0, s1);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(top, m[nt][e]);
            const float base = top == -INFINITY ? 0.f : top;
            keep[nt][e] = exp2_approx(m[nt][e] - base);
            moved |= top != m[nt][e];
            m[nt][e] = top;
            s0 = exp2_approx(s0 - base);
            s1 = exp2_approx(s1 - base);
            l[nt][e] = l[nt][e] * keep[nt][e] + s0 + s1;
          }
          // probabilities are rounded to the values' type for the product; the sum l is not
          pf[nt][0] = transpose8x8(pack2<E>(s[nt][0], s[nt][1]));
          pf[nt][1] = transpose8x8(pack2<E>(s[nt][2], s[nt][3]));
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][i][e] *= keep[nt][e & 1];
        }
        // V^T fragments: 8x8 blocks of V read transposed: (d 0-7, d 8-15) x (keys 0-7, 8-15)
        const int vrow = mt * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t vf[4];
          ldsm_x4_trans(vf, vs0 + vrow * (D * 2) + (((i * 2 + ((lane >> 3) & 1)) ^ (vrow & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(o[nt][i], vf, pf[nt][0], pf[nt][1], E());
        }
      }
      __syncwarp();  // the stage is read before a later load overwrites it
    }

    // ---- join the four warps: warp w ends with slices w F .. w F + F - 1 of the output, as
    // fragments of 16 elements by 8 rows; the other slices go to their warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float& v = l[nt][e];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        const int row = nt * 8 + (lane & 3) * 2 + e;
        if (lane < 4) sh_m[warp][row] = m[nt][e], sh_l[warp][row] = v;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const int to = i / F, from = (warp - to - 1) & 3;  // 0 .. 2 among the others
        if (to != warp)
          exchange[(((to * 3 + from) * NT + nt) * F + i % F) * 32 + lane] =
              make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]);
      }
    }
    __syncthreads();
    float top[NT][2], sum[NT][2];
    float4 acc[NT][F];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float f[kRowsWarps][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nt * 8 + (lane & 3) * 2 + e;
        float t = sh_m[0][row];
#pragma unroll
        for (int w = 1; w < kRowsWarps; ++w) t = fmaxf(t, sh_m[w][row]);
        const float base = t == -INFINITY ? 0.f : t;
        top[nt][e] = t;
        sum[nt][e] = 0.f;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {
          f[w][e] = exp2_approx(sh_m[w][row] - base);
          sum[nt][e] += f[w][e] * sh_l[w][row];
        }
      }
#pragma unroll
      for (int k = 0; k < F; ++k) {
        acc[nt][k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {  // in warp order, whoever adds
          float4 v;
          if (w == warp) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
              if (i == warp * F + k) v = make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]);
          } else {
            v = exchange[(((warp * 3 + ((w - warp - 1) & 3)) * NT + nt) * F + k) * 32 + lane];
          }
          acc[nt][k].x += f[w][0] * v.x, acc[nt][k].y += f[w][1] * v.y;
          acc[nt][k].z += f[w][0] * v.z, acc[nt][k].w += f[w][1] * v.w;
        }
      }
    }

    bool writes = true;
    if (b_last - b_first < it.blocks) {
      // shared with other blocks: leave the partial result, and the last to arrive joins all
      const int64_t first_block = ((it.u0 + 1) * G - 1) / U;
      const int64_t last_block = ((it.u0 + it.blocks) * G - 1) / U;
      const auto slot = [&](int64_t c) {  // a block's first segment, else its last
        return partials + (2 * c + (U * c / G < it.u0 ? 1 : 0)) * partial_floats(ROWS, D);
      };
      const auto place = [&](int nt, int k) { return ((warp * NT + nt) * F + k) * 32 + lane; };
      float* mine = slot(blockIdx.x);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int k = 0; k < F; ++k) __stcg(reinterpret_cast<float4*>(mine) + place(nt, k), acc[nt][k]);
        if (warp == 0 && lane < 4) {
          float2* ml = reinterpret_cast<float2*>(mine + ROWS * D) + nt * 4 + lane;
          __stcg(ml, make_float2(top[nt][0], top[nt][1]));
          __stcg(ml + ROWS / 2, make_float2(sum[nt][0], sum[nt][1]));
        }
      }
      __syncthreads();
      if (tid == 0) {
        const int arrived = atom_add_acq_rel_gpu(counters + it.index, 1);
        sh_last = arrived == (int)(last_block - first_block);
        if (sh_last) counters[it.index] = 0;
      }
      __syncthreads();
      writes = sh_last;
      if (writes) {
        constexpr int AT_ONCE = NT == 1 ? 8 : 4;  // partial results whose loads are in flight together
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) top[nt][e] = -INFINITY, sum[nt][e] = 0.f;
#pragma unroll
          for (int k = 0; k < F; ++k) acc[nt][k] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        for (int64_t c0 = first_block; c0 <= last_block; c0 += AT_ONCE) {
          float2 pm[AT_ONCE][NT], pl[AT_ONCE][NT];
          float4 pv[AT_ONCE][NT][F];
#pragma unroll
          for (int j = 0; j < AT_ONCE; ++j) {
            const float* p = slot(min(c0 + j, last_block));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float2* ml = reinterpret_cast<const float2*>(p + ROWS * D) + nt * 4 + (lane & 3);
              pm[j][nt] = c0 + j <= last_block ? __ldcg(ml) : make_float2(-INFINITY, -INFINITY);
              pl[j][nt] = __ldcg(ml + ROWS / 2);
#pragma unroll
              for (int k = 0; k < F; ++k)
                pv[j][nt][k] = __ldcg(reinterpret_cast<const float4*>(p) + place(nt, k));
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float base[2], keep[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float t = top[nt][e];
#pragma unroll
              for (int j = 0; j < AT_ONCE; ++j) t = fmaxf(t, e ? pm[j][nt].y : pm[j][nt].x);
              base[e] = t == -INFINITY ? 0.f : t;
              keep[e] = exp2_approx(top[nt][e] - base[e]);
              top[nt][e] = t;
              sum[nt][e] *= keep[e];
            }
#pragma unroll
            for (int k = 0; k < F; ++k) {
              acc[nt][k].x *= keep[0], acc[nt][k].y *= keep[1];
              acc[nt][k].z *= keep[0], acc[nt][k].w *= keep[1];
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
              const float f0 = exp2_approx(pm[j][nt].x - base[0]), f1 = exp2_approx(pm[j][nt].y - base[1]);
              sum[nt][0] += f0 * pl[j][nt].x;
              sum[nt][1] += f1 * pl[j][nt].y;
#pragma unroll
              for (int k = 0; k < F; ++k) {
                acc[nt][k].x += f0 * pv[j][nt][k].x, acc[nt][k].y += f1 * pv[j][nt][k].y;
                acc[nt][k].z += f0 * pv[j][nt][k].z, acc[nt][k].w += f1 * pv[j][nt][k].w;
              }
            }
          }
        }
      }
    }
    if (writes) {
      // a fragment transposed: row lane / 4, elements (lane & 3) * 2 and the next, then 8 further
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float i0 = sum[nt][0] > 0.f ? 1.f / sum[nt][0] : 0.f;
        const float i1 = sum[nt][1] > 0.f ? 1.f / sum[nt][1] : 0.f;
        const int row = nt * 8 + (lane >> 2), at = it.tile * ROWS + row;
        const int i = at / g, h = it.kvh * g + (at - i * g);
        E* out = static_cast<E*>(a.out) + ((it.token0 + i) * a.heads + h) * D + (lane & 3) * 2;
#pragma unroll
        for (int k = 0; k < F; ++k) {
          const float4 v = acc[nt][k];
          const uint32_t lo = transpose8x8(pack2<E>(v.x * i0, v.y * i1));
          const uint32_t hi = transpose8x8(pack2<E>(v.z * i0, v.w * i1));
          if (row < rows_here) {
            *reinterpret_cast<uint32_t*>(out + (warp * F + k) * 16) = lo;
            *reinterpret_cast<uint32_t*>(out + (warp * F + k) * 16 + 8) = hi;
          }
        }
        if (a.lse && warp == 0 && lane < 4) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + lane * 2 + e, x = it.tile * ROWS + r;
            if (r < rows_here)
              a.lse[(it.token0 + x / g) * a.heads + it.kvh * g + x % g] =
                  sum[nt][e] == 0.f ? -INFINITY : (top[nt][e] + log2f(sum[nt][e])) * kLn2;
          }
        }
      }
    }
    __syncthreads();  // the exchange is read before the next item's
  }
  copies_wait<0>();
}

// ---- host
static int rows_of_tile(const tr_attention& a) {
  // 16 rows where the requests bring more than 8 on average: one reading of the keys for twice
  // the rows; 8 else, whose products cost half as much.  us with tiles of 8 / 16: 61 requests of
  // 8192 with 4 rows over 8 kv heads 317 / 309, 8 rows over 4 168 / 162, 12 rows 320 / 161; 8
  // requests of 8192 57 / 56, 37 / 37, 53 / 37; one of 2048 18.5 / 20.6, 12.4 / 14.4, 18.5 / 14.4.
  const int64_t rows = a.tokens * (a.heads / a.kv_heads);
  return rows > 8 * a.requests ? 16 : 8;
}
static int64_t rows_max_items(const tr_attention& a, int rows) {
  return (a.tokens * (a.heads / a.kv_heads) / rows + a.requests) * a.kv_heads;
}
static int rows_grid() { return serve_sms() * 2; }

int64_t attend_rows_items(const tr_attention& a) { return rows_max_items(a, rows_of_tile(a)); }
size_t attend_rows_partials(const tr_attention& a) {
  return (size_t)rows_grid() * 2 * partial_floats(rows_of_tile(a), a.head_dim) * sizeof(float);
}

template <typename E, int D, int NT>
static int launch_rows(const tr_attention& a, const AttendWorkspace& ws, void* stream) {
  constexpr int smem = kRowsWarps * rows_stages<NT>() * 2 * warp_keys<D>() * D * 2 +  // stages
                       kRowsWarps * 3 * NT * (D / 64) * 512;                          // exchange
  auto kernel = attend_rows_kernel<E, D, NT>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_error("tr_paged_attention: %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
    return TR_ERR_CUDA;
  }
  kernel<<<rows_grid(), kRowsThreads, smem, static_cast<cudaStream_t>(stream)>>>(
      a, ws.status, ws.counters, rows_max_items(a, 8 * NT), ws.partials);
  return serve_launched("tr_paged_attention");
}

template <typename E>
static int launch_rows_type(const tr_attention& a, const AttendWorkspace& ws, void* stream) {
  const bool wide = rows_of_tile(a) == 16;
  if (a.head_dim == 128)
    return wide ? launch_rows<E, 128, 2>(a, ws, stream)
                : launch_rows<E, 128, 1>(a, ws, stream);
  return wide ? launch_rows<E, 64, 2>(a, ws, stream)
              : launch_rows<E, 64, 1>(a, ws, stream);
}

int launch_attend_rows(const tr_attention& a, const AttendWorkspace& ws, void* stream) {
  return a.dtype == TR_F16 ? launch_rows_type<__half>(a, ws, stream)
                           : launch_rows_type<__nv_bfloat16>(a, ws, stream);
}

}  // namespace trr
