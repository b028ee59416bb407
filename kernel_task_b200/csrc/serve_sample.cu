// tr_sample: the next token of every row from logits, temperature, top-k, top-p, min-p and given
// random numbers.
#include <cooperative_groups.h>

#include <algorithm>

#include "serve_util.cuh"

namespace cg = cooperative_groups;

namespace trr {

struct SampleArgs {
  const void* logits;
  const float* noise;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* tokens;
  float* logprobs;
  int64_t logits_stride, noise_stride;
  int vocab;
};

constexpr int kSampleThreads = 1024;

// Unsigned integers in the order of the floats (-0 and +0 made equal first).
__device__ __forceinline__ uint32_t order_key(float t) {
  const uint32_t u = __float_as_uint(t + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// Masses are summed as whole numbers of 2^-40 of the greatest token's, so that the sums do not
// depend on the order of the atomics.
constexpr float kMassUnit = 1099511627776.f;  // 2^40
__device__ __forceinline__ float weight_of(float t, float top) {
  return t == top ? 1.f : expf(t - top);
}
__device__ __forceinline__ unsigned long long mass_of(float w) {
  return (unsigned long long)llrintf(w * kMassUnit);
}

struct Best {
  float value;
  int index;
};
__device__ __forceinline__ Best better(Best a, Best b) {
  return b.value > a.value || (b.value == a.value && b.index < a.index) ? b : a;
}
__device__ __forceinline__ Best block_best(Best v, Best* part) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v = better(v, {__shfl_xor_sync(0xffffffffu, v.value, o), __shfl_xor_sync(0xffffffffu, v.index, o)});
  const int lane = threadIdx.x & 31;
  if (lane == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < (int)blockDim.x / 32 ? part[lane] : Best{-INFINITY, INT32_MAX};
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v = better(v, {__shfl_xor_sync(0xffffffffu, v.value, o), __shfl_xor_sync(0xffffffffu, v.index, o)});
  __syncthreads();
  return v;
}

// One block per row.  The cut of top-k and then of top-p is found by radix selection over the
// ordered keys, 8 bits a pass, counts for the first and masses for the second; ties at the cut
// are kept in index order.
template <typename L>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
  __shared__ Best part[32];
  __shared__ unsigned long long hist[256];
  __shared__ double dpart[32];
  __shared__ unsigned long long sh_left;
  __shared__ uint32_t sh_bin;
  __shared__ int sh_cut;
  __shared__ int ipart[32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, V = a.vocab;
  const L* logits = static_cast<const L*>(a.logits) + row * a.logits_stride;
  const float* noise = a.noise + row * a.noise_stride;
  const float heat = a.temperature[row];
  const bool hot = heat > 0.f;
  const float div = hot ? heat : 1.f;
  const auto value = [&](int i) {
    const float t = to_f32<L>(logits[i]) / div;
    return isnan(t) ? -INFINITY : t;
  };
  Best best = {-INFINITY, INT32_MAX};
  for (int i = tid; i < V; i += kSampleThreads) best = better(best, {value(i), i});
  best = block_best(best, part);
  const float top = best.value;
  if (top == -INFINITY) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  double z = 0.;
  for (int i = tid; i < V; i += kSampleThreads) z += weight_of(value(i), top);
  z = warp_sum(z);
  if ((tid & 31) == 0) dpart[tid >> 5] = z;
  __syncthreads();
  z = warp_sum(dpart[tid & 31]);

  if (hot) {
    const int k = a.top_k && a.top_k[row] > 0 ? min(a.top_k[row], V) : V;
    const float p = a.top_p ? a.top_p[row] : 1.f;
    uint32_t cut = 0;  // the least key kept, of which the first `ties` by index
    unsigned long long ties = V;
    if (k < V) {
      unsigned long long left = k;  // still to be kept at or below the prefix
      for (int shift = 24; shift >= 0; shift -= 8) {
        for (int b = tid; b < 256; b += kSampleThreads) hist[b] = 0;
        __syncthreads();
        for (int i = tid; i < V; i += kSampleThreads) {
          const uint32_t key = order_key(value(i));
          if (shift == 24 || (key >> (shift + 8)) == (cut >> (shift + 8)))
            atomicAdd(&hist[(key >> shift) & 255], 1ull);
        }
        __syncthreads();
        if (tid == 0) {
          int b = 255;
          while (b > 0 && hist[b] < left) left -= hist[b--];
          sh_bin = b;
          sh_left = left;
        }
        __syncthreads();
        cut |= sh_bin << shift;
        left = sh_left;
        __syncthreads();
      }
      ties = left;
    }
    if (p < 1.f) {
      const uint32_t least = cut;
      const unsigned long long least_ties = ties;
      // mass of what top-k keeps
      if (tid == 0) hist[0] = k < V ? least_ties * mass_of(weight_of(key_value(least), top)) : 0;
      __syncthreads();
      unsigned long long mine = 0;
      for (int i = tid; i < V; i += kSampleThreads) {
        const float t = value(i);
        if (k == V || order_key(t) > least) mine += mass_of(weight_of(t, top));
      }
      mine = warp_sum(mine);
      if ((tid & 31) == 0) atomicAdd(&hist[0], mine);
      __syncthreads();
      const double target = (double)p * (double)hist[0];
      unsigned long long above = 0;  // mass of the keys above the prefix
      uint32_t chosen = 0;
      __syncthreads();
      for (int shift = 24; shift >= 0; shift -= 8) {
        for (int b = tid; b < 256; b += kSampleThreads) hist[b] = 0;
        __syncthreads();
        for (int i = tid; i < V; i += kSampleThreads) {
          const float t = value(i);
          const uint32_t key = order_key(t);
          if ((k == V || key > least) &&
              (shift == 24 || (key >> (shift + 8)) == (chosen >> (shift + 8))))
            atomicAdd(&hist[(key >> shift) & 255], mass_of(weight_of(t, top)));
        }
        if (tid == 0 && k < V && (shift == 24 || (least >> (shift + 8)) == (chosen >> (shift + 8))))
          atomicAdd(&hist[(least >> shift) & 255],
                    least_ties * mass_of(weight_of(key_value(least), top)));
        __syncthreads();
        if (tid == 0) {
          int b = 255, last = -1;
          unsigned long long sum = above, at_last = above;
          for (; b >= 0 && ((double)sum < target || last < 0); --b) {
            if (hist[b] == 0) continue;
            last = b;
            at_last = sum;
            sum += hist[b];
          }
          sh_bin = last < 0 ? 0 : last;
          sh_left = at_last;
        }
        __syncthreads();
        chosen |= sh_bin << shift;
        above = sh_left;
        __syncthreads();
      }
      const double w = (double)mass_of(weight_of(key_value(chosen), top));
      const double want = w > 0. ? ceil((target - (double)above) / w) : 1.;
      const unsigned long long most = chosen == least && k < V ? least_ties : (unsigned long long)V;
      cut = chosen;
      ties = min(most, (unsigned long long)fmax(want, 1.));
    }
    // index of the last tie kept
    int cut_index = V;
    if (k < V || p < 1.f) {
      if (tid == 0) sh_cut = V;
      int before = 0;
      for (int i0 = 0; i0 < V && before < (long long)ties; i0 += kSampleThreads) {
        const int i = i0 + tid;
        const int is = i < V && order_key(value(i)) == cut;
        int total;
        const int through = block_scan_inclusive(is, ipart, total) + before;
        if (is && (unsigned long long)through == ties) sh_cut = i;
        before += total;
        __syncthreads();
      }
      __syncthreads();
      cut_index = sh_cut;
    }
    const float least_weight = a.min_p ? fminf(a.min_p[row], 1.f) : 0.f;
    best = {-INFINITY, INT32_MAX};
    for (int i = tid; i < V; i += kSampleThreads) {
      const float t = value(i);
      if (t == -INFINITY) continue;
      const uint32_t key = order_key(t);
      if (key < cut || (key == cut && i > cut_index)) continue;
      if (!(weight_of(t, top) >= least_weight) && t != top) continue;
      float s = t - logf(noise[i]);
      if (isnan(s)) s = -INFINITY;
      best = better(best, {s, i});
    }
    best = block_best(best, part);
  }
  if (tid == 0) {
    a.tokens[row] = best.index;
    const float t = value(best.index);
    if (a.logprobs) a.logprobs[row] = (t == top ? 0.f : t - top) - logf((float)z);
  }
}

// ---- one cluster per row, the row's t in shared memory ------------------------------------
//
// Every block of the cluster holds a contiguous slice of t, so the logits are read once.  A
// histogram of (greatest - t) in 1024 steps of 1/32, summed over the cluster, says down to which
// step the limits reach.  Where that leaves at most kCandidates tokens (a top_k of some hundred, or
// a top_p that the likeliest tokens reach) these are gathered, ranked, and all limits applied
// to the ranked list; noise is then read for them alone.  Else each limit's cut is narrowed down by
// further histograms over the steps that can hold it (for a mass: between the bounds that the
// steps' edges give, with the exact mass above them) until few enough tokens or a single value is
// left, and what is below the cut is struck out of the slices.
// All sums run in an order fixed by the row alone.
constexpr int kSliceThreads = 512;
constexpr int kBins = 1024;
constexpr float kBinsPerUnit = 32.f;
constexpr int kCandidates = 512;
constexpr int kMaxSlice = 52000;  // fp32 values of a block: 208 KB

struct RowSums {  // one value or two per block of the cluster, in every block
  double v[2][8][2];
};

template <typename L>
__global__ void __launch_bounds__(kSliceThreads, 2) sample_cluster_kernel(const SampleArgs a,
                                                                     int slice_size) {
  extern __shared__ float t_s[];
  __shared__ uint32_t hist[kBins];   // this block's, then the cluster's
  __shared__ uint32_t total[kBins];  // of block 0: the cluster's
  __shared__ RowSums sums;
  __shared__ float cand_t[kCandidates], rank_t[kCandidates];
  __shared__ int cand_i[kCandidates], rank_i[kCandidates];
  __shared__ Best part[32], cluster_best[8];
  __shared__ double dpart[32];
  __shared__ float fpart[32], cluster_t[8];
  __shared__ int ipart[32];
  __shared__ int sh_count, sh_bin[2], sh_ties;
  __shared__ float sh_cut;

  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / ranks;
  const int V = a.vocab;
  const int first = min((int64_t)rank * slice_size, (int64_t)V);
  const int n = min(slice_size, V - first);
  const L* logits = static_cast<const L*>(a.logits) + row * a.logits_stride + first;
  const float* noise = a.noise + row * a.noise_stride + first;
  const float heat = a.temperature[row];
  const bool hot = heat > 0.f;
  const float div = hot ? heat : 1.f;
  const int k = a.top_k && a.top_k[row] > 0 ? min(a.top_k[row], V) : V;
  const float p = a.top_p ? a.top_p[row] : 1.f;
  const float least_weight = a.min_p ? fminf(a.min_p[row], 1.f) : 0.f;

  int turn = 0;
  // Combines x (and y) over the cluster with `op`, in rank order; also a cluster barrier.
  const auto over_cluster = [&](double x, double y, auto op) {
    double(*box)[2] = sums.v[turn & 1];
    if (tid < ranks) {
      double(*there)[2] = cluster.map_shared_rank(&sums, tid)->v[turn & 1];
      there[rank][0] = x;
      there[rank][1] = y;
    }
    ++turn;
    cluster.sync();
    double2 r = make_double2(box[0][0], box[0][1]);
    for (int i = 1; i < ranks; ++i) {
      r.x = op(r.x, box[i][0]);
      r.y = op(r.y, box[i][1]);
    }
    return r;
  };
  const auto add = [](double u, double v) { return u + v; };
  const auto most = [](double u, double v) { return fmax(u, v); };
  const auto block_sum = [&](double v) {
    v = warp_sum(v);
    if (lane == 0) dpart[warp] = v;
    __syncthreads();
    v = warp_sum(lane < kSliceThreads / 32 ? dpart[lane] : 0.);
    __syncthreads();
    return v;
  };
  const auto block_max = [&](float v) {
    v = warp_max(v);
    if (lane == 0) fpart[warp] = v;
    __syncthreads();
    v = warp_max(lane < kSliceThreads / 32 ? fpart[lane] : -INFINITY);
    __syncthreads();
    return v;
  };

  // ---- the slice: t, with NaN as -inf and -0 as 0; the greatest
  for (int b = tid; b < kBins; b += kSliceThreads) hist[b] = total[b] = 0;
  if (tid == 0) sh_count = 0;
  float top = -INFINITY;
  const auto put = [&](int i, L x) {
    float t = to_f32<L>(x) / div + 0.f;
    t = isnan(t) ? -INFINITY : t;
    t_s[i] = t;
    top = fmaxf(top, t);
  };
  {
    constexpr int W = 16 / sizeof(L);  // elements of a 16-byte load
    const int head = min(n, (int)((16 - ((uintptr_t)logits & 15)) & 15) / (int)sizeof(L));
    const int vectors = (n - head) / W, tail = head + vectors * W;
    if (tid < head) put(tid, logits[tid]);
    const uint4* from = reinterpret_cast<const uint4*>(logits + head);
    for (int v = tid; v < vectors; v += kSliceThreads) {
      const uint4 x = __ldcs(from + v);
      const L* e = reinterpret_cast<const L*>(&x);
#pragma unroll
      for (int j = 0; j < W; ++j) put(head + v * W + j, e[j]);
    }
    if (tail + tid < n) put(tail + tid, logits[tail + tid]);
  }
  top = (float)over_cluster(block_max(top), 0., most).x;
  if (top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  if (top == INFINITY) {  // infinite logits share all the probability
    for (int i = tid; i < n; i += kSliceThreads) t_s[i] = t_s[i] == INFINITY ? 0.f : -INFINITY;
    top = 0.f;
    __syncthreads();
  }

  // ---- sum of the weights; histogram of the steps below the greatest
  const bool limited = hot && (k < V || p < 1.f);
  const auto weight = [&](float t) { return __expf(t - top); };
  // Bins of the values up to hi: at first by value, 1/32 each and the last one open; when a cut is
  // narrowed down, by ordered key between the least and the greatest key in reach, which puts
  // those two in different bins however near they are.
  float hi = top;
  uint64_t key_scale = 0;  // bins per key, times 2^32
  const auto bin_of = [&](float t) {
    if (key_scale) return (int)((uint64_t)(order_key(hi) - order_key(t)) * key_scale >> 32);
    return min((int)((hi - t) * kBinsPerUnit), kBins - 1);
  };
  // log-weights that the elements of bin b lie between
  const auto upper_edge = [&](int b) {
    if (!key_scale) return hi - top - b / kBinsPerUnit;
    const uint64_t off = (((uint64_t)b << 32) + key_scale - 1) / key_scale;
    return key_value((uint32_t)max((int64_t)order_key(hi) - (int64_t)off, (int64_t)0x00800000)) - top;
  };
  {
    float z = 0.f;
    int finite = 0;
    for (int i = tid; i < n; i += kSliceThreads) {
      const float t = t_s[i];
      z += weight(t);
      if (limited && t > -INFINITY) {
        atomicAdd(&hist[bin_of(t)], 1u);
        ++finite;
      }
    }
    dpart[0] = 0.;
    __syncthreads();
    const double zs = block_sum(z), fs = block_sum(finite);
    const auto pool_hist = [&] {
      uint32_t* all = cluster.map_shared_rank(total, 0);
      for (int b = tid; b < kBins; b += kSliceThreads)
        if (hist[b]) atomicAdd(all + b, hist[b]);
    };
    if (limited) pool_hist();
    const double2 both = over_cluster(zs, fs, add);
    const double Z = both.x;
    const int usable = (int)both.y;
    const float log_z = logf((float)Z);
    const auto answer = [&](int index, float t) {
      a.tokens[row] = index;
      if (a.logprobs) a.logprobs[row] = (t - top) - log_z;
    };

    // t - log(noise) of the slice's element i against the best so far, the logarithm in full only
    // where its approximation comes within 1e-3
    const auto consider = [&](Best& best, int i, float t, float e) {
      if (!(t - __logf(e) < best.value - 1e-3f)) {
        float s = t - logf(e);
        if (isnan(s)) s = -INFINITY;
        best = better(best, {s, first + i});
      }
    };
    const auto heavy_enough = [&](float t) {
      return t == top || expf(t - top) >= least_weight;
    };

    if (limited) {
      uint32_t* all = cluster.map_shared_rank(total, 0);
      // exclusive prefix of counts over the bins, two bins a thread
      const auto fetch = [&] {
        for (int b = tid; b < kBins; b += kSliceThreads) hist[b] = all[b];
        __syncthreads();
      };
      fetch();
      // Bins that hold a cut: by count the one where `want` is reached, by mass those where
      // `target` may be, given `above` (count or mass) over bin 0.  In sh_bin, last bin inclusive;
      // returns the counts up to the first of them (exclusive) and the last (inclusive).
      const auto find_bins = [&](bool by_mass, double want, double above, bool open_end) {
        if (tid == 0) sh_bin[0] = sh_bin[1] = kBins;
        const uint32_t c0 = hist[2 * tid], c1 = hist[2 * tid + 1];
        double lo0 = c0, lo1 = c1, up0 = c0, up1 = c1;
        if (by_mass) {
          const auto edge = [&](int b) { return (double)__expf(upper_edge(b)); };
          lo0 *= edge(2 * tid + 1) * (1. - 1e-4);
          lo1 *= open_end && 2 * tid + 1 == kBins - 1 ? 0. : edge(2 * tid + 2) * (1. - 1e-4);
          up0 *= edge(2 * tid) * (1. + 1e-4);
          up1 *= edge(2 * tid + 1) * (1. + 1e-4);
        }
        double all_lo, all_up;
        __syncthreads();
        const double through_lo = block_scan_inclusive(lo0 + lo1, dpart, all_lo) + above;
        const double through_up = block_scan_inclusive(up0 + up1, dpart, all_up) + above;
        if (c0 && through_up - up1 >= want) atomicMin(&sh_bin[0], 2 * tid);
        if (c1 && through_up >= want) atomicMin(&sh_bin[0], 2 * tid + 1);
        if (c0 && through_lo - lo1 >= want) atomicMin(&sh_bin[1], 2 * tid);
        if (c1 && through_lo >= want) atomicMin(&sh_bin[1], 2 * tid + 1);
        __syncthreads();
        // not reached: the last bins that hold anything
        int last = c1 ? 2 * tid + 1 : c0 ? 2 * tid : -1;
        last = (int)block_max((float)last);
        const int b1 = min(sh_bin[0], last), b2 = min(sh_bin[1], last);
        int sum;
        const int through = block_scan_inclusive((int)(c0 + c1), ipart, sum);
        __syncthreads();
        if (2 * tid == (b1 & ~1)) sh_bin[0] = through - (int)(c0 + c1) + (b1 & 1 ? (int)c0 : 0);
        if (2 * tid == (b2 & ~1)) sh_bin[1] = through - (b2 & 1 ? 0 : (int)c1);
        __syncthreads();
        const int4 r = make_int4(b1, b2, sh_bin[0], sh_bin[1]);
        __syncthreads();
        return r;
      };
      // Gathers the elements from `least` to hi with bins b1 .. b2, at most kCandidates, in block
      // 0 and ranks them there; a cluster barrier.
      const auto gather = [&](float least, int b1, int b2) {
        int* count = cluster.map_shared_rank(&sh_count, 0);
        float* ct = cluster.map_shared_rank(cand_t, 0);
        int* ci = cluster.map_shared_rank(cand_i, 0);
        for (int i = tid; i < n; i += kSliceThreads) {
          const float t = t_s[i];
          if (!(t > -INFINITY) || t < least || t > hi) continue;
          const int b = bin_of(t);
          if (b < b1 || b > b2) continue;
          const int at = atomicAdd(count, 1);
          if (at < kCandidates) {
            ct[at] = t;
            ci[at] = first + i;
          }
        }
        cluster.sync();
        if (rank == 0) {
          const int m = min(sh_count, kCandidates);
          if (tid < m) {
            const float t = cand_t[tid];
            const int i = cand_i[tid];
            int r = 0;
            for (int j = 0; j < m; ++j)
              r += cand_t[j] > t || (cand_t[j] == t && cand_i[j] < i);
            rank_t[r] = t;
            rank_i[r] = i;
          }
          __syncthreads();
          return m;
        }
        return 0;
      };

      const bool by_count = k < usable;
      int4 bins = by_count ? find_bins(false, k, 0., true) : find_bins(true, p * Z, 0., true);
      if ((by_count || p < 1.f) && bins.w <= kCandidates) {
        // ---- few enough: all limits on the ranked list
        const int m = gather(-INFINITY, 0, bins.y);
        if (rank != 0) return;
        const bool in = tid < m && (!by_count || tid < k);
        const float t = in ? rank_t[tid] : -INFINITY;
        const double w = in ? (double)weight(t) : 0.;
        double kept_mass;
        const double before = block_scan_inclusive(w, dpart, kept_mass) - w;
        const double target = p < 1.f ? p * (by_count ? kept_mass : Z) : INFINITY;
        Best best = {-INFINITY, INT32_MAX};
        if (in && (tid == 0 || before < target) && heavy_enough(t)) {
          float s = t - logf(a.noise[row * a.noise_stride + rank_i[tid]]);
          if (isnan(s)) s = -INFINITY;
          best = {s, rank_i[tid]};
          cand_t[tid] = t;
        }
        const Best won = block_best(best, part);
        if (in && best.index == won.index) answer(won.index, t);
        return;
      }

      // ---- cuts by narrowing
      for (int limit = 0; limit < 2; ++limit) {  // top_k, then top_p
        const bool by_mass = limit == 1;
        if (by_mass ? !(p < 1.f) : !by_count) continue;
        double want = k, above = 0., mass = 0.;
        if (by_mass) {
          mass = Z;
          if (by_count) {  // what top_k left
            float z = 0.f;
            for (int i = tid; i < n; i += kSliceThreads) z += weight(t_s[i]);
            mass = over_cluster(block_sum(z), 0., add).x;
          }
          want = p * mass;
        }
        bool open_end = true;
        int above_count = 0;
        for (int level = 0;; ++level) {
          if (level > 0 || (by_mass && by_count)) {  // histogram of the elements in reach
            if (level == 0) hi = top, key_scale = 0;
            for (int b = tid; b < kBins; b += kSliceThreads) hist[b] = total[b] = 0;
            cluster.sync();
            for (int i = tid; i < n; i += kSliceThreads) {
              const float t = t_s[i];
              if (!(t > -INFINITY) || t > hi) continue;
              if (level > 0 && t < sh_cut) continue;
              atomicAdd(&hist[bin_of(t)], 1u);
            }
            __syncthreads();
            for (int b = tid; b < kBins; b += kSliceThreads)
              if (hist[b]) atomicAdd(all + b, hist[b]);
            cluster.sync();
            fetch();
          }
          bins = find_bins(by_mass, by_mass ? want : want - above_count, by_mass ? above : 0.,
                           open_end);
          if (by_mass && level > 0 && bins.x == 0 && bins.y == bin_of(sh_cut)) {
            // the bounds leave every bin (coarse ones, or few values many times): the exact mass
            // of the upper half of the bins decides between the halves, and neither is empty,
            // since hi is in the first bin and the least value in the last
            const int half = bins.y / 2;
            float z = 0.f;
            int count = 0;
            for (int i = tid; i < n; i += kSliceThreads) {
              const float t = t_s[i];
              if (!(t > -INFINITY) || t < sh_cut || t > hi || bin_of(t) > half) continue;
              z += weight(t);
              ++count;
            }
            const double2 upper = over_cluster(block_sum(z), block_sum(count), add);
            if (above + upper.x >= want) bins.y = half, bins.w = (int)upper.y;
            else bins.x = half + 1, bins.z = (int)upper.y;
          }
          // mass (or count) above the bins; range of the values in them
          float z = 0.f, low = INFINITY, high = -INFINITY;
          for (int i = tid; i < n; i += kSliceThreads) {
            const float t = t_s[i];
            if (!(t > -INFINITY) || t > hi) continue;
            if (level > 0 && t < sh_cut) continue;
            const int b = bin_of(t);
            if (b < bins.x) z += weight(t);
            else if (b <= bins.y) low = fminf(low, t), high = fmaxf(high, t);
          }
          above += over_cluster(block_sum(z), 0., add).x;
          const double2 range = over_cluster(block_max(-low), block_max(high), most);
          low = -(float)range.x;
          high = (float)range.y;
          const int members = bins.w - bins.z;
          above_count += bins.z;
          __syncthreads();
          if (low == high || level >= 64) {  // ties: as many as the limit still takes
            if (tid == 0) {
              const double w = weight(low);
              const double takes = !by_mass ? want - above_count
                                   : w > 0. ? ceil((want - above) / w) : 1.;
              sh_cut = low;
              sh_ties = (int)fmin(fmax(takes, above_count ? 0. : 1.), (double)members);
            }
            __syncthreads();
            break;
          }
          if (members <= kCandidates) {
            const int m = gather(level > 0 ? sh_cut : -INFINITY, bins.x, bins.y);
            if (rank == 0) {
              const float t = tid < m ? rank_t[tid] : -INFINITY;
              const double w = tid < m ? (double)weight(t) : 0.;
              double unused;
              const double before = above + block_scan_inclusive(w, dpart, unused) - w;
              const bool in = tid < m && (by_mass ? before < want || (above_count == 0 && tid == 0)
                                                  : above_count + tid < want);
              const int kept = max((int)block_sum(in ? 1. : 0.), 1);
              const float cut = rank_t[kept - 1];
              const int ties = (int)block_sum(tid < kept && t == cut ? 1. : 0.);
              if (tid < ranks) {
                *cluster.map_shared_rank(&sh_cut, tid) = cut;
                *cluster.map_shared_rank(&sh_ties, tid) = ties;
              }
              if (tid == 0) sh_count = 0;
            }
            cluster.sync();
            break;
          }
          // narrower: the values between low and high
          if (tid == 0) sh_cut = low;
          hi = high;
          key_scale = ((uint64_t)kBins << 32) / ((uint64_t)order_key(high) - order_key(low) + 1);
          open_end = false;
          __syncthreads();
        }
        // strike out what is below the cut, and the ties past the last one kept
        const float cut = sh_cut;
        const int ties = sh_ties;
        int mine = 0;
        for (int i = tid; i < n; i += kSliceThreads) mine += t_s[i] == cut;
        mine = (int)block_sum(mine);
        double(*box)[2] = sums.v[turn & 1];
        over_cluster(mine, 0., add);
        int before = 0;
        for (int r = 0; r < rank; ++r) before += (int)box[r][0];
        const int keeps = min(max(ties - before, 0), mine);
        int seen = 0;
        for (int i0 = 0; i0 < n; i0 += kSliceThreads) {
          const int i = i0 + tid;
          const float t = i < n ? t_s[i] : INFINITY;
          if (keeps == 0 || keeps == mine) {
            if (t < cut || (t == cut && keeps == 0)) t_s[i] = -INFINITY;
            continue;
          }
          int count;
          const int through = seen + block_scan_inclusive((int)(t == cut), ipart, count);
          if (t < cut || (t == cut && through > keeps)) t_s[i] = -INFINITY;
          seen += count;
        }
        __syncthreads();
      }
    }

    // ---- the best of what is left
    Best best = {-INFINITY, INT32_MAX};
    if (!hot) {
      for (int i = tid; i < n; i += kSliceThreads) best = better(best, {t_s[i], first + i});
    } else if (least_weight > 0.f) {
      const float sure = top + logf(least_weight);
      for (int i = tid; i < n; i += kSliceThreads) {
        const float t = t_s[i];
        if (!(t > -INFINITY) || t < sure - 1e-3f || !heavy_enough(t)) continue;
        consider(best, i, t, noise[i]);
      }
    } else {
      for (int i0 = tid; i0 < n; i0 += 4 * kSliceThreads) {
        float e[4], t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = i0 + j * kSliceThreads;
          t[j] = i < n ? t_s[i] : -INFINITY;
          e[j] = t[j] > -INFINITY ? __ldcs(noise + i) : 1.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (t[j] > -INFINITY) consider(best, i0 + j * kSliceThreads, t[j], e[j]);
      }
    }
    best = block_best(best, part);
    if (tid == 0) {
      cluster.map_shared_rank(cluster_best, 0)[rank] = best;
      // the value of the block's best, for the logprob
      cluster.map_shared_rank(cluster_t, 0)[rank] = best.index < V ? t_s[best.index - first] : 0.f;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      int who = 0;
      for (int r = 1; r < ranks; ++r)
        if (cluster_best[r].value > cluster_best[who].value ||
            (cluster_best[r].value == cluster_best[who].value &&
             cluster_best[r].index < cluster_best[who].index))
          who = r;
      answer(cluster_best[who].index, cluster_t[who]);
    }
  }
}

template <typename L>
static int launch_sample(const SampleArgs& a, int64_t rows, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.vocab > 8 * kMaxSlice) {  // does not fit the cluster's shared memory
    sample_kernel<L><<<(unsigned)rows, kSampleThreads, 0, s>>>(a);
    return serve_launched("tr_sample");
  }
  // blocks per row: slices of 16384 where the rows fill the GPU, 8 blocks where they do not
  int blocks = 1;
  while (blocks < 8 && (a.vocab > blocks * 16384 ||
                        (a.vocab > blocks * 2048 && rows * blocks * 2 <= serve_sms())))
    blocks *= 2;
  const int slice = (a.vocab + blocks - 1) / blocks;
  const size_t smem = (size_t)slice * sizeof(float);
  auto kernel = sample_cluster_kernel<L>;
  if (smem > 30 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSlice * (int)sizeof(float));
    if (e != cudaSuccess) {
      set_error("tr_sample: %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
      return TR_ERR_CUDA;
    }
  }
  if (rows * blocks > INT32_MAX) {
    set_error("tr_sample: %lld rows", (long long)rows);
    return TR_ERR_UNSUPPORTED;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * blocks));
  cfg.blockDim = dim3(kSliceThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, slice);
  if (e != cudaSuccess) {
    set_error("tr_sample launch: %s", cudaGetErrorString(e));
    (void)cudaGetLastError();
    return TR_ERR_CUDA;
  }
  return TR_OK;
}

}  // namespace trr

using namespace trr;

extern "C" int tr_sample(const void* logits, int32_t dtype, int64_t logits_stride,
                         const float* noise, int64_t noise_stride, const float* temperature,
                         const int32_t* top_k, const float* top_p, const float* min_p, int64_t rows,
                         int64_t vocab, int64_t* tokens, float* logprobs, void* stream) {
  if (!known_dtype(dtype)) {
    set_error("tr_sample: unknown dtype %d", (int)dtype);
    return TR_ERR_INVALID;
  }
  if (rows < 0 || vocab < 1) {
    set_error("tr_sample: bad shape");
    return TR_ERR_INVALID;
  }
  if (vocab > 1 << 22 || rows > INT32_MAX) {
    set_error("tr_sample: vocabulary of %lld (at most 2^22)", (long long)vocab);
    return TR_ERR_UNSUPPORTED;
  }
  if (rows == 0) return TR_OK;
  if (!logits || !noise || !temperature || !tokens) {
    set_error("tr_sample: null pointer");
    return TR_ERR_INVALID;
  }
  if (((uintptr_t)logits & (element_bytes(dtype) - 1)) ||
      (((uintptr_t)noise | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p |
        (uintptr_t)min_p | (uintptr_t)logprobs) & 3) || ((uintptr_t)tokens & 7)) {
    set_error("tr_sample: a pointer is not aligned to its elements");
    return TR_ERR_ALIGN;
  }
  SampleArgs a = {logits, noise, temperature, top_k, top_p, min_p, tokens, logprobs, logits_stride,
                  noise_stride, (int)vocab};
  if (dtype == TR_F32) return launch_sample<float>(a, rows, stream);
  if (dtype == TR_F16) return launch_sample<__half>(a, rows, stream);
  return launch_sample<__nv_bfloat16>(a, rows, stream);
}
