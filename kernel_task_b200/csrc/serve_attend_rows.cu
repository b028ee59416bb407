// Paged attention for few query rows per request and kv head: decoding, and short chunks.
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
// An item that several blocks share leaves fp32 partial results in the workspace; the last block
// to arrive joins them in unit order, so the result does not depend on the order of arrival.
#include <algorithm>

#include "serve_attend.cuh"
#include "tc_util.cuh"

namespace trr {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = 32 * kRowsWarps;
constexpr int kRowsStages = 3;
constexpr int kMinBlocks = 2;  // blocks of keys a grid block takes at least

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

struct RowsWork {
  int64_t units;       // of all requests
  int64_t request_u0;  // first unit of `request`
  int64_t request_i0;  // first item of `request`
  int request;         // the request of this block's first unit
};

struct RequestShape {
  int n, tiles, blocks;
  int64_t items, units;
};
template <int ROWS, int BK>
__device__ __forceinline__ RequestShape shape_of(const tr_attention& a, int r) {
  RequestShape s;
  s.n = brought(a, r);
  s.tiles = (int)(((int64_t)s.n * (a.heads / a.kv_heads) + ROWS - 1) / ROWS);
  s.blocks = max((cached(a, r) + BK - 1) / BK, 1);  // at least one: rows without keys are written too
  s.items = (int64_t)s.tiles * a.kv_heads;
  s.units = s.items * s.blocks;
  return s;
}

template <typename E, int D, int NT>
__global__ void __launch_bounds__(kRowsThreads) attend_rows_kernel(const tr_attention a, int* counters,
                                                                  int64_t max_items,
                                                                  float* partials) {
  constexpr int ROWS = 8 * NT, WK = warp_keys<D>(), MT = WK / 16, BK = block_keys<D>();
  constexpr int CPR = D / 8;                      // 16-byte chunks of a row
  constexpr int STAGE = 2 * WK * D * 2;           // bytes of a warp's stage: keys, then values
  constexpr int PAD = D + 4;                      // row stride of the joined outputs
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int64_t scan_part[32], scan_items[32];
  __shared__ RowsWork work;
  __shared__ float sh_m[kRowsWarps][ROWS], sh_l[kRowsWarps][ROWS];
  __shared__ int sh_last;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = a.heads / a.kv_heads;
  const int R = (int)a.requests;
  clear_outside<E>(a, (int64_t)blockIdx.x * kRowsThreads + tid, (int64_t)gridDim.x * kRowsThreads);
  if (R == 0) return;

  // ---- this block's run of units: thread i sums requests [i per, (i + 1) per)
  const int per = (R + kRowsThreads - 1) / kRowsThreads;
  const int r_lo = min(tid * per, R), r_hi = min(r_lo + per, R);
  int64_t my_units = 0, my_items = 0;
  for (int r = r_lo; r < r_hi; ++r) {
    const RequestShape s = shape_of<ROWS, BK>(a, r);
    my_units += s.units;
    my_items += s.items;
  }
  int64_t U, all_items;
  const int64_t through = block_scan_inclusive(my_units, scan_part, U);
  const int64_t items_through = block_scan_inclusive(my_items, scan_items, all_items);
  if (U == 0 || all_items > max_items) return;
  const int64_t G = min((int64_t)gridDim.x, (U + kMinBlocks - 1) / kMinBlocks);
  if (blockIdx.x >= G) return;
  const int64_t u_begin = U * blockIdx.x / G, u_end = U * (blockIdx.x + 1) / G;
  if (through - my_units <= u_begin && u_begin < through) {
    int64_t u = through - my_units, it = items_through - my_items;
    int r = r_lo;
    for (; r < r_hi; ++r) {
      const RequestShape s = shape_of<ROWS, BK>(a, r);
      if (u_begin < u + s.units) break;
      u += s.units;
      it += s.items;
    }
    work.request = r;
    work.request_u0 = u;
    work.request_i0 = it;
  }
  __syncthreads();
  int request = work.request;
  int64_t request_u0 = work.request_u0, request_i0 = work.request_i0;
  RequestShape shape = shape_of<ROWS, BK>(a, request);

  const uint32_t stage0 = smem_u32(smem) + warp * kRowsStages * STAGE;
  const E* kp = static_cast<const E*>(a.k_pages);
  const E* vp = static_cast<const E*>(a.v_pages);
  const float scale2 = a.scale * kLog2e;
  const int page_shift = 31 - __clz(a.page_size);

  for (int64_t u = u_begin; u < u_end;) {
    while (u >= request_u0 + shape.units) {
      request_u0 += shape.units;
      request_i0 += shape.items;
      shape = shape_of<ROWS, BK>(a, ++request);
    }
    const int64_t in_request = u - request_u0;
    const int item = (int)(in_request / shape.blocks);
    const int b_first = (int)(in_request - (int64_t)item * shape.blocks);
    const int b_last = (int)min((int64_t)shape.blocks, b_first + (u_end - u));  // one past
    const int64_t item_u0 = request_u0 + (int64_t)item * shape.blocks;
    const int tile = item / a.kv_heads, kvh = item - tile * a.kv_heads;
    const int rows_here = min((int64_t)ROWS, (int64_t)shape.n * g - (int64_t)tile * ROWS);
    const int64_t token0 = max(a.starts[request], 0);

    // the two query rows of this lane's columns, per n-tile: how many keys they see
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nt * 8 + (lane & 3) * 2 + e;
        limit[nt][e] =
            row < rows_here ? visible(a, request, shape.n, (tile * ROWS + row) / g) : 0;
      }
    const int keys_end =
        max(visible(a, request, shape.n, (tile * ROWS + rows_here - 1) / g), 0);
    const int b_stop = min(b_last, (keys_end + BK - 1) / BK);

    // Q^T fragments: row lane / 4, elements ks * 16 + (lane & 3) * 2 (+1, +8, +9)
    uint32_t qf[NT][D / 16][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = nt * 8 + (lane >> 2), at = tile * ROWS + row;
      const int i = at / g, h = kvh * g + (at - i * g);
      const E* q = static_cast<const E*>(a.q) + (token0 + i) * a.q_token_stride +
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

    const int32_t* table = a.tables + request * a.table_stride;
    // lane i < WK: page of key i of the warp's share of block b (-1 past the end)
    const auto page_id = [&](int b) {
      const int key = b * BK + warp * WK + lane;
      return lane < WK && b < b_stop && key < keys_end ? table[key >> page_shift] : -1;
    };
    const auto load = [&](int b, int id) {  // one commit group, empty past the end
      if (b < b_stop) {
        const uint32_t base = stage0 + (b - b_first) % kRowsStages * STAGE;
        const int key0 = b * BK + warp * WK;
#pragma unroll
        for (int i = 0; i < WK * CPR / 32; ++i) {
          const int row = i * (32 / CPR) + lane / CPR, c = lane % CPR, key = key0 + row;
          const int pid = __shfl_sync(0xffffffffu, id, row);
          const bool held = pid >= 0 && pid < a.pages && key < keys_end;
          const int64_t at =
              held ? (((int64_t)pid * a.kv_heads + kvh) * a.page_size + (key & (a.page_size - 1))) *
                             D + c * 8
                   : 0;
          const uint32_t dst = base + row * (D * 2) + ((c ^ (row & 7)) << 4);
          copy16_async(dst, kp + at, held);
          copy16_async(dst + WK * D * 2, vp + at, held);
        }
      }
      copies_commit();
    };
    int ids = page_id(b_first);
    for (int s = 0; s < kRowsStages - 1; ++s) {
      const int next = page_id(b_first + s + 1);
      load(b_first + s, ids);
      ids = next;
    }

    for (int b = b_first; b < b_stop; ++b) {
      const int next = page_id(b + kRowsStages);
      load(b + kRowsStages - 1, ids);
      ids = next;
      copies_wait<kRowsStages - 1>();
      __syncwarp();
      const uint32_t ks0 = stage0 + (b - b_first) % kRowsStages * STAGE, vs0 = ks0 + WK * D * 2;
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
      __syncwarp();  // the stage is read before the next load overwrites it
    }
    copies_wait<0>();
    __syncthreads();

    // ---- join the four warps
    float* so = reinterpret_cast<float*>(smem);  // [warp][row][PAD]
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
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          so[(warp * ROWS + row) * PAD + i * 16 + (lane >> 2)] = o[nt][i][e];
          so[(warp * ROWS + row) * PAD + i * 16 + (lane >> 2) + 8] = o[nt][i][e + 2];
        }
      }
    }
    __syncthreads();
    constexpr int COLS = ROWS * D / kRowsThreads;  // consecutive outputs of a thread
    const int orow = tid * COLS / D, ocol = tid * COLS % D;
    float top = -INFINITY, sum = 0.f, acc[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, sh_m[w][orow]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
      const float f = exp2_approx(sh_m[w][orow] - base);
      sum += f * sh_l[w][orow];
#pragma unroll
      for (int c = 0; c < COLS; ++c) acc[c] += f * so[(w * ROWS + orow) * PAD + ocol + c];
    }

    bool writes = true;
    if (b_last - b_first < shape.blocks) {
      // shared with other blocks: leave the partial result, and the last to arrive joins all
      const int64_t first_block = ((item_u0 + 1) * G - 1) / U;
      const int64_t last_block = ((item_u0 + shape.blocks) * G - 1) / U;
      const auto slot = [&](int64_t c) {  // a block's first segment, else its last
        return partials + (2 * c + (U * c / G < item_u0 ? 1 : 0)) * partial_floats(ROWS, D);
      };
      float* mine = slot(blockIdx.x);
#pragma unroll
      for (int c = 0; c < COLS; c += 4)
        __stcg(reinterpret_cast<float4*>(mine + orow * D + ocol + c),
               make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]));
      if (ocol == 0) {
        __stcg(mine + ROWS * D + orow, top);
        __stcg(mine + ROWS * D + ROWS + orow, sum);
      }
      __syncthreads();
      const int64_t counter = request_i0 + item;
      if (tid == 0) {
        const int arrived = atom_add_acq_rel_gpu(counters + counter, 1);
        sh_last = arrived == (int)(last_block - first_block);
        if (sh_last) counters[counter] = 0;
      }
      __syncthreads();
      writes = sh_last;
      if (writes) {
        // eight partial results at a time: their loads are in flight together
        top = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
        for (int64_t c0 = first_block; c0 <= last_block; c0 += 8) {
          float pm[8], pl[8];
          float4 pv[8][COLS / 4];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float* p = slot(min(c0 + j, last_block));
            pm[j] = c0 + j <= last_block ? __ldcg(p + ROWS * D + orow) : -INFINITY;
            pl[j] = __ldcg(p + ROWS * D + ROWS + orow);
#pragma unroll
            for (int k = 0; k < COLS / 4; ++k)
              pv[j][k] = __ldcg(reinterpret_cast<const float4*>(p + orow * D + ocol) + k);
          }
          float all = top;
#pragma unroll
          for (int j = 0; j < 8; ++j) all = fmaxf(all, pm[j]);
          const float base = all == -INFINITY ? 0.f : all;
          const float keep = exp2_approx(top - base);
          top = all;
          sum *= keep;
#pragma unroll
          for (int c = 0; c < COLS; ++c) acc[c] *= keep;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float f = exp2_approx(pm[j] - base);
            sum += f * pl[j];
#pragma unroll
            for (int k = 0; k < COLS / 4; ++k) {
              acc[4 * k] += f * pv[j][k].x, acc[4 * k + 1] += f * pv[j][k].y;
              acc[4 * k + 2] += f * pv[j][k].z, acc[4 * k + 3] += f * pv[j][k].w;
            }
          }
        }
      }
    }
    if (writes && orow < rows_here) {
      const int at = tile * ROWS + orow, i = at / g, h = kvh * g + (at - i * g);
      const int64_t out_row = (token0 + i) * a.heads + h;
      const float inv = sum > 0.f ? 1.f / sum : 0.f;
      E* out = static_cast<E*>(a.out) + out_row * D + ocol;
#pragma unroll
      for (int c = 0; c < COLS; c += 4)
        *reinterpret_cast<uint2*>(out + c) = make_uint2(pack2<E>(acc[c] * inv, acc[c + 1] * inv),
                                                        pack2<E>(acc[c + 2] * inv, acc[c + 3] * inv));
      if (a.lse && ocol == 0)
        a.lse[out_row] = top == -INFINITY ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
    u += b_last - b_first;
    __syncthreads();  // shared memory is free for the next item
  }
}

// ---- host
static int rows_of_tile(const tr_attention& a) {
  // 16 rows where the requests bring more than 8 on average: one reading of the keys for twice
  // the rows; 8 else, whose products cost half as much
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
  constexpr int pipeline = kRowsWarps * kRowsStages * 2 * warp_keys<D>() * D * 2;
  constexpr int joined = kRowsWarps * 8 * NT * (D + 4) * 4;
  constexpr int smem = pipeline > joined ? pipeline : joined;
  auto kernel = attend_rows_kernel<E, D, NT>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_error("tr_paged_attention: %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
    return TR_ERR_CUDA;
  }
  kernel<<<rows_grid(), kRowsThreads, smem, static_cast<cudaStream_t>(stream)>>>(
      a, ws.counters, rows_max_items(a, 8 * NT), ws.partials);
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
