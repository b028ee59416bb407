// Paged attention for many query rows per request and kv head: prompts and chunks of them, on
// the 5th-generation tensor cores.  8192 prompt tokens, 32 heads over 8 of 128: 515 us, 1067 TFLOP/s
// of the 1686 of a large product; 440 us with a head_dim of 64.  The products alone need 2478
// cycles for 256 rows by 128 keys (2048 but for the scores' width, see below); the chain scores -
// softmax - product through four buffers makes it 3900: the tensor pipe is active 45 % of the
// time, the exponentials' unit 45 %, the issue slots 39 %.
//
// A row is one token and query head; the rows of a request over one kv head, token-major, are
// cut into tiles of 256, so all the heads that share keys share their loads.  A tile is two
// subtiles of 128 rows, each with its own scores S and output O in tensor memory:
//     S = Q K^T   (128 x 64 keys, K-major operands in shared memory, 128-byte swizzle)
//     O += P V    (P from tensor memory, where it takes the place of S; V is read with its
//                  head_dim contiguous, the MN-major form of the same layout)
// Each subtile has two buffers of S, so the next 64 keys' scores are made while the softmax works
// on these (one buffer of 128 keys: a prompt of 8192 in 585 us then, 540 with two of 64).  64 wide
// is what two subtiles with a head_dim of 128 leave of 512 columns; it costs a quarter more
// shared-memory reading of Q.
// Warps 0-3 and 4-7 each hold a subtile's softmax, a thread per row: running maximum and sum in
// registers, P rounded to the values' type.  O is rescaled only when a row's maximum grew by
// more than 2^8 since the last time; P is then at most 256 and the fp32 sums keep their bits.
// Warp 8 issues the scores, warp 11 the products with V; warps 9 and 10 bring queries, keys and
// values, 128 rows at a time, through a ring of shared-memory slots with cp.async (zeros past
// the keys: a page's unused rows may hold anything, and 0 * NaN would reach O).
//
// Split.  An item is (request, row tile, kv head), a unit one block of 128 keys that the tile
// sees; kItemUnits more stand in front of them for what an item costs besides (queries, the
// first scores, the outputs: as long as about 3 blocks).  The grid is one block per SM (all of
// tensor memory), and each takes an equal contiguous
// run of all units, as in serve_attend_rows.cu; partial results of shared items are joined by
// the last block to arrive, in unit order.
//
// Every wait is bounded: when one runs out the block raises its abort flag, all roles leave
// their loops, tensor memory is freed, the rows of its run become NaN and the workspace's status
// word says TR_ERR_TIMEOUT; while it does, later calls give NaN too.
#include <algorithm>

#include "serve_attend.cuh"
#include "tc_util.cuh"

namespace trr {

constexpr int kBlockKeys = 128;
constexpr int kSubRows = 128, kTileRows = 2 * kSubRows;
constexpr int kChunkThreads = 12 * 32;
constexpr int kMinChunkUnits = 6;  // units a grid block takes at least
constexpr int kItemUnits = 3;
constexpr unsigned kChunkWaitPolls = 1u << 19;  // of 2638 cycles each: about 0.7 s

template <int D>
__host__ __device__ constexpr int ring_slots() {
  return D == 128 ? 5 : 8;
}
template <int D>
__host__ __device__ constexpr int slot_bytes() {
  return kBlockKeys * D * 2;
}
template <int D>
__host__ __device__ constexpr int chunk_smem() {
  return 1024 + 2 * kSubRows * D * 2 + ring_slots<D>() * slot_bytes<D>();
}

template <>
__device__ __forceinline__ void tmem_ld<32>(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}

// One try_wait without a time limit of its own: the warp is suspended for up to 2638 cycles
// (measured; with a limit of 20 us given, 7814, and 3 % slower here).
__device__ __forceinline__ bool mbar_try_once(uint32_t mbar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(mbar), "r"(parity)
      : "memory");
  return done != 0;
}

// tcgen05.mma with A in tensor memory, issued by one elected lane of a converged warp
__device__ __forceinline__ void umma_ts_one(uint32_t dtmem, uint32_t atmem, uint64_t db,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(
          dtmem),
      "r"(atmem), "l"(db), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0));
}

// ---- pairs of fp32
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// P of 32 keys from their scores: 2^(s scale - base), rounded in pairs to E; their sums added to
// `sum`.
template <typename E>
__device__ __forceinline__ void probabilities(const uint32_t* s, uint64_t scale, uint64_t minus_base,
                                              uint64_t (&sum)[2], uint32_t (&p)[16]) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float2 x = unpair(fma2(pair(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])),
                                 scale, minus_base));
    const float e0 = exp2_approx(x.x), e1 = exp2_approx(x.y);
    sum[k & 1] = add2(sum[k & 1], pair(e0, e1));
    p[k] = pack2<E>(e0, e1);
  }
}

// Four 16-byte chunks of this lane's row become chunk lane & 3 of the four rows of its quad, so
// that a warp's store covers 64 contiguous bytes of 8 rows instead of 16 bytes of 32.
__device__ __forceinline__ uint4 swap4(uint4 v, int x) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, x), __shfl_xor_sync(0xffffffffu, v.y, x),
                    __shfl_xor_sync(0xffffffffu, v.z, x), __shfl_xor_sync(0xffffffffu, v.w, x));
}
__device__ __forceinline__ void quad_transpose(uint4 (&c)[4]) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint4 got = swap4(odd ? c[i] : c[i + 1], 1);
    if (odd) c[i] = got;
    else c[i + 1] = got;
  }
  // now c[0], c[1]: chunk `odd` of the quad's even and odd row of this half; c[2], c[3]: 2 + odd
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 got = swap4(high ? c[i] : c[i + 2], 2);
    if (high) c[i] = got;
    else c[i + 2] = got;
  }
}

// Keys and values of a slot: [head_dim / 64][128 rows][128 bytes], 16-byte chunks swizzled by
// row & 7.  Values as the MN-major operand: 64-element column groups 16 KB apart, groups of 8
// keys 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_values(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(kBlockKeys * 128 >> 4) << 16 |
         (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// Walks the items of a contiguous run of units.
struct ChunkItem {
  int request, rows, tiles, tile, kvh;
  int units;       // of the item: kItemUnits, then its blocks of keys
  int see0, cap;   // token i of the request sees min(see0 + i, cap) keys (none if negative)
  int64_t token0;  // the request's first token
  int64_t u0;      // first unit of the item
  int64_t index;   // item number
};
__device__ __forceinline__ int keys_of_token(const ChunkItem& it, int i) {
  return max(min(it.see0 + i, it.cap), 0);
}
// keys that the last row of the tile sees
__device__ __forceinline__ int keys_of_tile(const ChunkItem& it, int g, int tile) {
  return keys_of_token(it, (min((tile + 1) * kTileRows, it.rows) - 1) / g);
}
__device__ __forceinline__ int tile_units(const ChunkItem& it, int g, int tile) {
  return max((keys_of_tile(it, g, tile) + kBlockKeys - 1) / kBlockKeys, 1) + kItemUnits;
}
__device__ __forceinline__ void open_request(const tr_attention& a, int g, ChunkItem& it, int r) {
  const int n = brought(a, r);
  it.request = r;
  it.rows = n * g;
  it.tiles = (it.rows + kTileRows - 1) / kTileRows;
  it.tile = it.kvh = 0;
  it.cap = cached(a, r);
  it.see0 = (int)max((int64_t)a.lens[r] - n + 1, -(int64_t)(1 << 30));
  it.token0 = max((int64_t)a.starts[r], (int64_t)0);
  it.units = it.tiles ? tile_units(it, g, 0) : 0;
}
__device__ __forceinline__ void next_item(const tr_attention& a, int g, ChunkItem& it) {
  it.u0 += it.units;
  ++it.index;
  if (++it.kvh < a.kv_heads) return;
  it.kvh = 0;
  if (++it.tile < it.tiles) {
    it.units = tile_units(it, g, it.tile);
    return;
  }
  while (it.request + 1 < (int)a.requests) {
    open_request(a, g, it, it.request + 1);
    if (it.tiles) return;
  }
}
// The blocks of keys of `it` inside [u, u_end), and u past them.
struct Segment {
  int first, last;  // last: one past
};
__device__ __forceinline__ Segment take(const ChunkItem& it, int64_t& u, int64_t u_end) {
  const int lo = (int)(u - it.u0), hi = (int)min((int64_t)it.units, u_end - it.u0);
  u = it.u0 + hi;
  return {max(lo - kItemUnits, 0), max(hi - kItemUnits, 0)};
}

enum {
  B_FULL = 0,    // [8] a slot's rows have arrived (the copies arrive by themselves)
  B_EMPTY = 8,   // [8] the products have read a slot
  B_QUERY = 16,  // the tile's queries are in shared memory
  B_QFREE = 17,  // the item's last scores are made: the queries' place is free
  B_SCORES = 18, // [2][2] a subtile's S of the first or last 64 keys is in tensor memory
  B_PROBS = 22,  // [2][2] P has taken its place, O is rescaled
  B_PRODUCT = 26, // [2][2] their P V is added to the subtile's O
  B_LEFT = 30,   // [2] a subtile's partial result is written
  B_JOIN = 32,   // [2] whether this block joins the item is known
  B_DRAIN = 34,  // [2] an issuing warp's last products
  B_COUNT = 36
};

template <typename E, int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
    attend_chunk_kernel(const tr_attention a, int* status, int* counters, int64_t max_items,
                        float* partials, unsigned last_poll) {
  constexpr int NS = ring_slots<D>();
  constexpr int QBYTES = kSubRows * D * 2, SLOT = slot_bytes<D>(), CPR = D / 8;
  constexpr int64_t PARTIAL = (int64_t)kTileRows * (D + 2);
  extern __shared__ uint8_t smem_raw[];
  __shared__ int64_t scan_part[32], scan_items[32];
  __shared__ uint64_t bars[B_COUNT];
  __shared__ ChunkItem first_item;
  __shared__ uint32_t tmem_slot;
  __shared__ int sh_abort, sh_join[2];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = a.heads / a.kv_heads, R = (int)a.requests;
  // Whether an earlier call timed out: read by one thread, since a block of this call may set the
  // word at any time, and on its way while the run is found.  All threads see it after the scans.
  if (tid == 0) sh_abort = __ldcg(status);
  clear_outside<E>(a, (int64_t)blockIdx.x * kChunkThreads + tid, (int64_t)gridDim.x * kChunkThreads);
  if (R == 0) return;

  // ---- this block's run of units
  const int per = (R + kChunkThreads - 1) / kChunkThreads;
  const int r_lo = min(tid * per, R), r_hi = min(r_lo + per, R);
  int64_t my_units = 0, my_items = 0;
  for (int r = r_lo; r < r_hi; ++r) {
    ChunkItem it;
    open_request(a, g, it, r);
    my_items += (int64_t)it.tiles * a.kv_heads;
    for (int t = 0; t < it.tiles; ++t)
      my_units += (int64_t)tile_units(it, g, t) * a.kv_heads;
  }
  int64_t U, all_items;
  const int64_t through = block_scan_inclusive(my_units, scan_part, U);
  const int64_t items_through = block_scan_inclusive(my_items, scan_items, all_items);
  if (U == 0 || all_items > max_items) return;
  const int64_t G = min((int64_t)gridDim.x, (U + kMinChunkUnits - 1) / kMinChunkUnits);
  if (blockIdx.x >= G) return;
  const int64_t u_begin = U * blockIdx.x / G, u_end = U * (blockIdx.x + 1) / G;
  if (through - my_units <= u_begin && u_begin < through) {
    ChunkItem it;
    it.u0 = through - my_units;
    it.index = items_through - my_items;
    for (int r = r_lo; r < r_hi; ++r) {
      open_request(a, g, it, r);
      int64_t units = 0;
      for (; it.tile < it.tiles; ++it.tile) {
        it.units = tile_units(it, g, it.tile);
        units = (int64_t)it.units * a.kv_heads;
        if (u_begin < it.u0 + units) break;
        it.u0 += units;
        it.index += a.kv_heads;
      }
      if (it.tile < it.tiles) break;
    }
    it.kvh = (int)((u_begin - it.u0) / it.units);
    it.u0 += (int64_t)it.kvh * it.units;
    it.index += it.kvh;
    first_item = it;
  }

  const auto spoil_run = [&] {
    ChunkItem it = first_item;
    for (; it.u0 < u_end; next_item(a, g, it))
      spoil_rows(a, it.token0, it.kvh, g, it.tile * kTileRows,
                 min(kTileRows, it.rows - it.tile * kTileRows));
  };
  if (sh_abort) {
    __syncthreads();
    spoil_run();
    return;
  }

  // ---- set-up
  const auto bar = [&](int i) { return smem_u32(&bars[i]); };
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (warp == 9) {
    for (int i = lane; i < B_COUNT; i += 32) {
      int count = 1;
      if (i < B_EMPTY || i == B_QUERY) count = 64;  // the threads of the two loading warps
      if ((i >= B_PROBS && i < B_PRODUCT) || i == B_LEFT || i == B_LEFT + 1)
        count = 4;  // the subtile's four warps
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar(i)), "r"(count)
                   : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t qbase = (smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t ring = qbase + 2 * QBYTES;
  volatile int* abort = &sh_abort;
  // Bounded wait of a whole warp.  try_wait suspends the warp, which leaves the issue slots to the
  // softmax (polling with test_wait: 4 % faster over long contexts with a head_dim of 128, 15 %
  // slower with 64 and over short prompts).  The loop is as plain as can be: a first try ahead
  // of it, or a clock in it, cost the same 15 %.
  const auto wait = [&](int b, uint32_t parity) {
    bool ok = true;
    for (unsigned i = 0; ok && !mbar_try_once(bar(b), parity); ++i) {
      if (*abort) ok = false;
      if (i >= last_poll) {
        *abort = 1;
        ok = false;
      }
    }
    return (bool)__all_sync(0xffffffffu, ok);
  };
  ChunkItem it = first_item;
  const int page_shift = 31 - __clz(a.page_size);

  if (warp < 8) {
    // ---- softmax: subtile t, row `row` of it
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + t * 128 + lanes, o_tmem = tmem + 256 + t * D + lanes;
    const float scale2 = a.scale * kLog2e;
    // phases so far: blocks of keys (B_SCORES, B_PROBS, B_PRODUCT), partial results
    uint32_t blocks = 0, lefts = 0;
    for (int64_t u = u_begin; u < u_end; next_item(a, g, it)) {
      const Segment seg = take(it, u, u_end);
      const int b_first = seg.first, b_last = seg.last;
      if (b_first == b_last) continue;  // only the units in front
      const int row0 = it.tile * kTileRows + t * kSubRows;
      const int rows_here = min(it.rows - row0, kSubRows);
      if (rows_here <= 0) continue;  // the item has one subtile
      const bool live = row < rows_here;
      const int i = (row0 + row) / g, h = it.kvh * g + (row0 + row - i * g);
      const int limit = live ? keys_of_token(it, i) : 0;
      const bool warp_live = (warp & 3) * 32 < rows_here;

      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int n = 2 * b_first; n < 2 * b_last; ++n) {  // 64 keys at a time
        const int half = n & 1;
        const uint32_t s_half = s_tmem + half * 64;
        if (!(ok = wait(B_SCORES + 2 * t + half, blocks & 1))) break;
        tc_fence_after();
        if (warp_live) {
          uint32_t s[64];
          tmem_ld<32>(s_half, reinterpret_cast<uint32_t(&)[32]>(s[0]));
          tmem_ld<32>(s_half + 32, reinterpret_cast<uint32_t(&)[32]>(s[32]));
          tmem_wait_ld();
          const int seen = limit - n * 64;
          if (__any_sync(0xffffffffu, seen < 64)) {
#pragma unroll
            for (int k = 0; k < 64; ++k) s[k] = k < seen ? s[k] : __float_as_uint(-INFINITY);
          }
          float tops[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) tops[k] = __uint_as_float(s[k]);
#pragma unroll
          for (int k = 4; k < 60; k += 8)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              tops[j] = fmaxf(fmaxf(tops[j], __uint_as_float(s[k + j])), __uint_as_float(s[k + 4 + j]));
#pragma unroll
          for (int j = 0; j < 4; ++j) tops[j] = fmaxf(tops[j], __uint_as_float(s[60 + j]));
          const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * scale2;
          // a new base where the old one would let P pass 2^8
          const bool rise = top > m + 8.f || (m == -INFINITY && top > -INFINITY);
          if (__any_sync(0xffffffffu, rise)) {
            const float keep = !rise ? 1.f : m == -INFINITY ? 0.f : exp2_approx(m - top);
            if (rise) m = top;
            l *= keep;
            if (n > 2 * b_first) {
              // O holds still once the last 64 keys' product is added; the one before is
              // already, since these scores came after it
              if (!(ok = wait(B_PRODUCT + 2 * t + 1 - half, (blocks + half - 1) & 1))) break;
              tc_fence_after();
#pragma unroll
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                tmem_ld<16>(o_tmem + c * 16, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                tmem_st16(o_tmem + c * 16, o);
              }
            }
          }
          const float base = m == -INFINITY ? 0.f : m;
          const uint64_t scales = pair(scale2, scale2), minus_base = pair(-base, -base);
          uint64_t sum[2] = {0, 0};  // pairs of zeros
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t p[16];
            probabilities<E>(s + c * 32, scales, minus_base, sum, p);
            tmem_st16(s_half + c * 16, p);
          }
          const float2 all = unpair(add2(sum[0], sum[1]));
          l += all.x + all.y;
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_PROBS + 2 * t + half));
        blocks += half;
      }
      if (!ok || !wait(B_PRODUCT + 2 * t, (blocks - 1) & 1) ||
          !wait(B_PRODUCT + 2 * t + 1, (blocks - 1) & 1))
        break;
      tc_fence_after();

      const bool shared_item = b_last - b_first < it.units - kItemUnits;
      // the grid blocks with the item's first and last block of keys
      const int64_t first_block = ((it.u0 + kItemUnits + 1) * G - 1) / U;
      const int64_t last_block = ((it.u0 + it.units) * G - 1) / U;
      const auto slot = [&](int64_t c) {
        return partials + (2 * c + (U * c / G < it.u0 ? 1 : 0)) * PARTIAL;
      };
      // the quad's four rows: element offset of each in out, or -1
      const int64_t out_row = ((it.token0 + i) * a.heads + h);
      int64_t quad_row[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        quad_row[k] = __shfl_sync(0xffffffffu, live ? out_row : -1, (lane & ~3) + k);
      const auto store4 = [&](int col, uint4 (&c)[4]) {  // 32 columns from col
        quad_transpose(c);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (quad_row[k] >= 0)
            *reinterpret_cast<uint4*>(static_cast<E*>(a.out) + quad_row[k] * D + col +
                                      (lane & 3) * 8) = c[k];
      };
      bool writes = true;
      if (shared_item) {
        // partial result: [D / 4][256 rows] float4, then maxima and sums
        float* mine = slot(blockIdx.x);
        const int at = t * kSubRows + row;
        if (warp_live) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld<16>(o_tmem + c * 16, o);
            tmem_wait_ld();
            if (live) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                __stcg(reinterpret_cast<float4*>(mine) + (c * 4 + k) * kTileRows + at,
                       make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                   __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3])));
            }
          }
          if (live) {
            __stcg(mine + (int64_t)kTileRows * D + at, m);
            __stcg(mine + (int64_t)kTileRows * (D + 1) + at, l);
          }
        }
        __syncwarp();
        if (lane == 0) {
          __threadfence();
          mbar_arrive(bar(B_LEFT + t));
        }
        __syncwarp();
        if ((warp & 3) == 0) {
          ok = wait(B_LEFT + t, lefts & 1);
          if (lane == 0) {
            int* counter = counters + it.index * 2 + t;
            const int last = ok ? atom_add_acq_rel_gpu(counter, 1) : -1;
            sh_join[t] = last == (int)(last_block - first_block);
            if (sh_join[t]) *counter = 0;
            mbar_arrive(bar(B_JOIN + t));
          }
          __syncwarp();
        }
        if (!wait(B_JOIN + t, lefts & 1)) break;
        ++lefts;
        writes = sh_join[t];
        __threadfence();
        if (writes && warp_live) {
          // half the columns at a time: 16 loads of a part in flight (rows past the tile's
          // read what the slot holds and store nothing)
          const float* maxima = partials + (int64_t)kTileRows * D + at;
          const float* sums = maxima + kTileRows;
          const auto part = [&](int64_t c) { return slot(c) - partials; };
          float top = -INFINITY;
#pragma unroll 4
          for (int64_t c = first_block; c <= last_block; ++c)
            top = fmaxf(top, __ldcg(maxima + part(c)));
          const float base = top == -INFINITY ? 0.f : top;
          float sum = 0.f;
#pragma unroll 4
          for (int64_t c = first_block; c <= last_block; ++c)
            sum += exp2_approx(__ldcg(maxima + part(c)) - base) * __ldcg(sums + part(c));
          m = top;
          l = sum;
          const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 64) {
            float acc[64];
#pragma unroll
            for (int k = 0; k < 64; ++k) acc[k] = 0.f;
#pragma unroll 1
            for (int64_t c = first_block; c <= last_block; ++c) {
              const float f = exp2_approx(__ldcg(maxima + part(c)) - base);
              float4 v[16];
#pragma unroll
              for (int k = 0; k < 16; ++k)
                v[k] = __ldcg(reinterpret_cast<const float4*>(slot(c)) + (c0 / 4 + k) * kTileRows + at);
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                acc[4 * k] += f * v[k].x, acc[4 * k + 1] += f * v[k].y;
                acc[4 * k + 2] += f * v[k].z, acc[4 * k + 3] += f * v[k].w;
              }
            }
#pragma unroll
            for (int k = 0; k < 64; k += 32) {
              uint4 c[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                c[j] = make_uint4(pack2<E>(acc[k + 8 * j] * inv, acc[k + 8 * j + 1] * inv),
                                  pack2<E>(acc[k + 8 * j + 2] * inv, acc[k + 8 * j + 3] * inv),
                                  pack2<E>(acc[k + 8 * j + 4] * inv, acc[k + 8 * j + 5] * inv),
                                  pack2<E>(acc[k + 8 * j + 6] * inv, acc[k + 8 * j + 7] * inv));
              store4(c0 + k, c);
            }
          }
        }
      } else if (warp_live) {
        const float inv = m > -INFINITY ? 1.f / l : 0.f;
#pragma unroll
        for (int k = 0; k < D; k += 32) {
          uint32_t o[32];
          tmem_ld<32>(o_tmem + k, o);
          tmem_wait_ld();
          uint4 c[4];
          const auto two = [&](int n) {
            return pack2<E>(__uint_as_float(o[n]) * inv, __uint_as_float(o[n + 1]) * inv);
          };
#pragma unroll
          for (int j = 0; j < 4; ++j)
            c[j] = make_uint4(two(8 * j), two(8 * j + 2), two(8 * j + 4), two(8 * j + 6));
          store4(k, c);
        }
      }
      if (writes && live && a.lse)
        a.lse[out_row] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
      tc_fence_before();  // O is free for the next item once its B_PROBS arrive
    }
  } else if (warp == 8) {
    // ---- scores.  Each kind of product has a warp of its own: a wait takes some 200 cycles even
    // when it is over, and the queue of products is shorter than that
    constexpr uint32_t idesc_s = umma_idesc<E>(kSubRows, 64);
    uint32_t items_done = 0, x = 0, blocks[2] = {0, 0};  // slots taken; blocks of a subtile
    bool ok = true;
    for (int64_t u = u_begin; ok && u < u_end; next_item(a, g, it)) {
      const Segment seg = take(it, u, u_end);
      const int b_first = seg.first, b_last = seg.last;
      if (b_first == b_last) continue;  // only the units in front
      const int subs = it.rows - it.tile * kTileRows > kSubRows ? 2 : 1;
      if (!(ok = wait(B_QUERY, items_done & 1))) break;
      ++items_done;
      for (int b = b_first; ok && b < b_last; ++b) {
        const uint32_t slot = x % NS, keys = ring + slot * SLOT;
        if (!(ok = wait(B_FULL + slot, (x / NS) & 1))) break;
        fence_async_smem();  // the copies were ordinary writes; the products read by the async proxy
        tc_fence_after();
        for (int half = 0; ok && half < 2; ++half) {
          for (int t = 0; t < subs; ++t) {
            // P of the block before has been read from this half
            if (blocks[t] && !(ok = wait(B_PRODUCT + 2 * t + half, (blocks[t] - 1) & 1))) break;
            tc_fence_after();
            // descriptors by adding to one: no address field overflows, and the sums of constants
            // stay in uniform registers (8192 prompt tokens: 539 us without, 523 with)
            const uint64_t queries = desc_sw128(qbase + t * QBYTES);
            const uint64_t block = desc_sw128(keys + half * (64 * 128));
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const int in = (ks >> 2) * (128 * 128) + (ks & 3) * 32;
              umma_one(tmem + t * 128 + half * 64, queries + in / 16, block + in / 16, idesc_s,
                       ks > 0);
            }
            commit_one(bar(B_SCORES + 2 * t + half));
          }
        }
        if (!ok) break;
        for (int t = 0; t < subs; ++t) ++blocks[t];
        commit_one(bar(B_EMPTY + slot));
        if (b + 1 == b_last) commit_one(bar(B_QFREE));
        x += 2;
      }
    }
    commit_one(bar(B_DRAIN));  // whatever was issued has to end before tensor memory is freed
    mbar_drain_spin(bar(B_DRAIN), 0);
  } else if (warp == 11) {
    // ---- products with the values
    constexpr uint32_t idesc_o = umma_idesc<E>(kSubRows, D) | 1u << 16;  // values: MN-major
    uint32_t x = 1, blocks[2] = {0, 0};
    bool ok = true;
    for (int64_t u = u_begin; ok && u < u_end; next_item(a, g, it)) {
      const Segment seg = take(it, u, u_end);
      const int b_first = seg.first, b_last = seg.last;
      if (b_first == b_last) continue;
      const int subs = it.rows - it.tile * kTileRows > kSubRows ? 2 : 1;
      for (int b = b_first; ok && b < b_last; ++b) {
        const uint32_t slot = x % NS, values = ring + slot * SLOT;
        if (!(ok = wait(B_FULL + slot, (x / NS) & 1))) break;
        fence_async_smem();
        for (int half = 0; ok && half < 2; ++half) {
          for (int t = 0; t < subs; ++t) {
            if (!(ok = wait(B_PROBS + 2 * t + half, blocks[t] & 1))) break;
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              umma_ts_one(tmem + 256 + t * D, tmem + t * 128 + half * 64 + ks * 8,
                          desc_values(values + (half * 4 + ks) * 2048), idesc_o,
                          b > b_first || half > 0 || ks > 0);
            commit_one(bar(B_PRODUCT + 2 * t + half));
          }
        }
        if (!ok) break;
        for (int t = 0; t < subs; ++t) ++blocks[t];
        commit_one(bar(B_EMPTY + slot));
        x += 2;
      }
    }
    commit_one(bar(B_DRAIN + 1));
    mbar_drain_spin(bar(B_DRAIN + 1), 0);
  } else {
    // ---- loads: warp w brings rows 64 w .. 64 w + 63 of every block of keys and of values, and
    // of both subtiles' queries
    const int w = warp - 9;
    uint32_t x = 0, items_done = 0;
    bool ok = true;
    // a lane's part: chunk c of row `sub` and of every RPI-th row after it
    const int c = lane % CPR, sub = lane / CPR;
    constexpr int RPI = 32 / CPR;
    const auto at_row = [&](int rr) {  // offset of the chunk in a [head_dim / 64][rows][128 B] array
      return rr * 128 + (((c & 7) ^ (rr & 7)) << 4) + (c >> 3) * (128 * 128);
    };
    // arrives on `b` when this thread's copies so far are in shared memory
    const auto hand_over = [&](int b) {
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar(b)) : "memory");
    };
    for (int64_t u = u_begin; ok && u < u_end; next_item(a, g, it)) {
      const Segment seg = take(it, u, u_end);
      const int b_first = seg.first, b_last = seg.last;
      if (b_first == b_last) continue;
      const int keys_end = keys_of_tile(it, g, it.tile);
      const int32_t* table = a.tables + it.request * a.table_stride;
      // pool rows of keys 64 w + lane and + 32 of block b; ~0u past the keys and for bad pages
      uint32_t rows[2], next[2];
      const auto find = [&](int b, uint32_t (&r)[2]) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = b * kBlockKeys + w * 64 + j * 32 + lane;
          const int id = b < b_last && key < keys_end ? table[key >> page_shift] : -1;
          r[j] = id >= 0 && id < a.pages
                     ? (uint32_t)((id * (int64_t)a.kv_heads + it.kvh) * a.page_size +
                                  (key & (a.page_size - 1)))
                     : ~0u;
        }
      };
      const auto load_rows = [&](const uint4* pool) {
        const uint32_t slot = x % NS;
        if (x >= NS && !(ok = wait(B_EMPTY + slot, (x / NS - 1) & 1))) return;
        const uint32_t dst = ring + slot * SLOT + w * 64 * 128;
#pragma unroll
        for (int i = 0; i < 64 / RPI; ++i) {
          const int rr = i * RPI + sub;
          const uint32_t r = __shfl_sync(0xffffffffu, rows[i * RPI / 32], rr & 31);
          const bool held = r != ~0u;
          copy16_async(dst + at_row(rr), pool + (uint64_t)(held ? r : 0u) * CPR + c, held);
        }
        hand_over(B_FULL + slot);
        ++x;
      };
      find(b_first, rows);
      for (int b = b_first; ok && b < b_last; ++b) {
        load_rows(static_cast<const uint4*>(a.k_pages));
        if (!ok) break;
        if (b == b_first) {
          // the queries, once the last item's are read
          if (items_done && !(ok = wait(B_QFREE, (items_done - 1) & 1))) break;
#pragma unroll 1
          for (int t = 0; t < 2; ++t) {
            // element offsets of rows 64 w + lane and + 32 of the subtile; -1 past the rows
            int64_t from[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int row = it.tile * kTileRows + t * kSubRows + w * 64 + j * 32 + lane;
              const int i = row / g;
              from[j] = row < it.rows ? (it.token0 + i) * a.q_token_stride +
                                            (it.kvh * g + row - i * g) * a.q_head_stride
                                      : -1;
            }
            const uint32_t dst = qbase + t * QBYTES + w * 64 * 128;
#pragma unroll
            for (int i = 0; i < 64 / RPI; ++i) {
              const int rr = i * RPI + sub;
              const int64_t f = __shfl_sync(0xffffffffu, from[i * RPI / 32], rr & 31);
              copy16_async(dst + at_row(rr), static_cast<const E*>(a.q) + (f < 0 ? 0 : f) + c * 8,
                           f >= 0);
            }
          }
          hand_over(B_QUERY);
          ++items_done;
        }
        find(b + 1, next);
        load_rows(static_cast<const uint4*>(a.v_pages));
        rows[0] = next[0];
        rows[1] = next[1];
      }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512)
                 : "memory");
  }
  if (sh_abort) {
    if (tid == 0) atomicExch(status, (int)TR_ERR_TIMEOUT);
    spoil_run();
  }
}

// ---- host
int64_t attend_chunk_items(const tr_attention& a) {
  return 2 * (a.tokens * (a.heads / a.kv_heads) / kTileRows + a.requests) * a.kv_heads;
}
size_t attend_chunk_partials(const tr_attention& a) {
  return (size_t)serve_sms() * 2 * kTileRows * (a.head_dim + 2) * sizeof(float);
}

template <typename E, int D>
static int launch_chunk(const tr_attention& a, const AttendWorkspace& ws, void* stream) {
  auto kernel = attend_chunk_kernel<E, D>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, chunk_smem<D>());
  if (e != cudaSuccess) {
    set_error("tr_paged_attention: %d bytes of shared memory: %s", chunk_smem<D>(),
              cudaGetErrorString(e));
    return TR_ERR_CUDA;
  }
  kernel<<<serve_sms(), kChunkThreads, chunk_smem<D>(), static_cast<cudaStream_t>(stream)>>>(
      a, ws.status, ws.counters, attend_chunk_items(a) / 2, ws.partials,
      (a.wait_polls ? a.wait_polls : kChunkWaitPolls) - 1);
  return serve_launched("tr_paged_attention");
}

int launch_attend_chunk(const tr_attention& a, const AttendWorkspace& ws, void* stream) {
  if (a.dtype == TR_F16)
    return a.head_dim == 128 ? launch_chunk<__half, 128>(a, ws, stream)
                             : launch_chunk<__half, 64>(a, ws, stream);
  return a.head_dim == 128 ? launch_chunk<__nv_bfloat16, 128>(a, ws, stream)
                           : launch_chunk<__nv_bfloat16, 64>(a, ws, stream);
}

}  // namespace trr
