// tr_sample: the next token of every row from logits, temperature, top-k, top-p, min-p and given
// random numbers.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

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

// For rows that a cluster's shared memory does not hold (over 800000 logits of 16 bits): one block
// per row, which reads it again for every pass.  Two rows of 900001: about 2 ms.  The cut of
// top-k and then of top-p is found by radix selection over the ordered keys, 8 bits a pass, counts
// for the first and masses for the second; ties at the cut are kept in index order.
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
  bool infinite = false;  // infinite logits share all the probability
  const auto value = [&](int i) {
    const float l = to_f32<L>(logits[i]);
    if (infinite) return l == INFINITY ? 0.f : -INFINITY;
    return isnan(l) ? -INFINITY : l;
  };
  Best best = {-INFINITY, INT32_MAX};
  for (int i = tid; i < V; i += kSampleThreads) best = better(best, {value(i), i});
  best = block_best(best, part);
  if (best.value == INFINITY) {
    infinite = true;
    best.value = 0.f;
  }
  const float top = best.value;
  if (top == -INFINITY) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  // t less the greatest t, which stays finite at the top where t itself would pass fp32; -inf
  // stays so under an infinite temperature
  const auto below_top = [&](float l) { return l == -INFINITY ? l : (l - top) / div; };
  const auto weight = [&](float l) { return expf(below_top(l)); };
  double z = 0.;
  for (int i = tid; i < V; i += kSampleThreads) z += weight(value(i));
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
      if (tid == 0) hist[0] = k < V ? least_ties * mass_of(weight(key_value(least))) : 0;
      __syncthreads();
      unsigned long long mine = 0;
      for (int i = tid; i < V; i += kSampleThreads) {
        const float l = value(i);
        if (k == V || order_key(l) > least) mine += mass_of(weight(l));
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
          const float l = value(i);
          const uint32_t key = order_key(l);
          if ((k == V || key > least) &&
              (shift == 24 || (key >> (shift + 8)) == (chosen >> (shift + 8))))
            atomicAdd(&hist[(key >> shift) & 255], mass_of(weight(l)));
        }
        if (tid == 0 && k < V && (shift == 24 || (least >> (shift + 8)) == (chosen >> (shift + 8))))
          atomicAdd(&hist[(least >> shift) & 255],
                    least_ties * mass_of(weight(key_value(least))));
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
      const double w = (double)mass_of(weight(key_value(chosen)));
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
      const float l = value(i);
      if (l == -INFINITY) continue;
      const uint32_t key = order_key(l);
      if (key < cut || (key == cut && i > cut_index)) continue;
      if (!(weight(l) >= least_weight) && l != top) continue;
      float s = below_top(l) - logf(noise[i]);
      if (isnan(s)) s = -INFINITY;
      best = better(best, {s, i});
    }
    best = block_best(best, part);
  }
  if (tid == 0) {
    a.tokens[row] = best.index;
    if (a.logprobs) a.logprobs[row] = below_top(value(best.index)) - logf((float)z);
  }
}

// ---- one cluster per row, the row in shared memory -----------------------------------------
//
// Every block of the cluster holds a contiguous slice of the logits, so they are read once.  The
// order of t = logit / temperature is the logits' own, so maxima, histograms and cuts work on
// the logits; t itself (an exact division, of the logit less the greatest) is made for the tokens
// that reach the final choice.  The weights, which every sum of mass is made of (the logprob's
// normaliser, what top-p cuts by), are one approximate power of two each, off by at most 2^-22 and
// 2^-23 of the exponent: a cut that two tokens' masses miss by less than that may fall either way.
//
// The limits mostly leave few tokens.  Each thread's greatest logit goes into a histogram of 1024
// steps below the greatest (1/32 of t each), summed over the cluster: these are some of the
// tokens, so where they alone reach top_k, or top_p of the mass, all tokens kept lie in the steps
// down to there.  They are gathered, ranked, and all limits applied to the ranked list; noise is
// read for them alone.
//
// Where that does not do, one limit needs no cut: the token drawn from all, if the limit keeps
// it (its rank, or the mass above it, is one pass), is the token drawn from the kept; if not, the
// kept are among those ranked above it, and one of these is drawn.  The first draw is kept with
// the kept tokens' probability, and every other draw halves what is left or so.  After
// kDraws, and for top_k where the mass of what it keeps is asked for, the cut is searched by
// halving the ordered keys until few enough tokens for a ranked list lie between.
// Every sum's order is fixed by the row and by the blocks it is cut over, which the vocabulary and
// the number of rows decide: the same call gives the same bits, a row sampled alone and in a batch
// may differ in the last bits of its masses.
//
// Bound by instructions and barriers rather than memory: 256 rows of 131072 in bf16 (67 MB, 10.4 us
// of memory; 134 MB of noise where it is read) take 44 us greedy, 57 us with min_p 0.05, 70 us
// with top_k 50, 83 us drawn from all tokens (2.4 TB/s), 131 us with top_p 0.9 alone and 209 us
// with top_k 2000, whose limits need draws and cuts of their own; a single row 10 to 25 us, of
// which five cluster barriers and the launch are most.
constexpr int kSliceThreads = 512;
constexpr int kBins = 1024;
constexpr float kBinsPerUnit = 32.f;
constexpr int kCandidates = 512;
constexpr int kDraws = 12;
constexpr int kSliceBytes = 65536;     // of a block where the rows fill the GPU: two blocks an SM
constexpr int kMaxSliceBytes = 200000;

struct RowSums {  // one value or two per block of the cluster, in every block
  double v[2][8][2];
};

// The greatest of the logits in a 16-byte vector without NaN.
template <typename L>
__device__ __forceinline__ float greatest_of(const uint4& x) {
  using P = typename std::conditional<std::is_same<L, __half>::value, __half2, __nv_bfloat162>::type;
  const P* w = reinterpret_cast<const P*>(&x);
  const P m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
  return fmaxf(to_f32<L>(m.x), to_f32<L>(m.y));
}
template <>
__device__ __forceinline__ float greatest_of<float>(const uint4& x) {
  return fmaxf(fmaxf(__uint_as_float(x.x), __uint_as_float(x.y)),
               fmaxf(__uint_as_float(x.z), __uint_as_float(x.w)));
}
// The same, and NaN made -inf in it.
template <typename L>
__device__ __forceinline__ float settle(uint4& x) {
  using P = typename std::conditional<std::is_same<L, __half>::value, __half2, __nv_bfloat162>::type;
  P* w = reinterpret_cast<P*>(&x);
  const bool clean = __hbeq2(w[0], w[0]) && __hbeq2(w[1], w[1]) && __hbeq2(w[2], w[2]) &&
                     __hbeq2(w[3], w[3]);
  if (!clean) {
    L* e = reinterpret_cast<L*>(&x);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (__hisnan(e[j])) e[j] = from_f32<L>(-INFINITY);
  }
  return greatest_of<L>(x);
}
template <>
__device__ __forceinline__ float settle<float>(uint4& x) {
  float* e = reinterpret_cast<float*>(&x);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (isnan(e[j])) e[j] = -INFINITY;
  return greatest_of<float>(x);
}

template <typename L>
__global__ void __launch_bounds__(kSliceThreads, 2) sample_cluster_kernel(const SampleArgs a,
                                                                        int slice_size) {
  constexpr int W = 16 / sizeof(L);  // elements of a 16-byte load
  extern __shared__ uint4 slice_raw[];
  __shared__ uint32_t hist[kBins];   // this block's, then the cluster's
  __shared__ uint32_t total[kBins];  // of block 0: the cluster's
  __shared__ RowSums sums;
  __shared__ float own_l[kCandidates], cand_l[kCandidates];  // this block's; block 0: all
  __shared__ int own_i[kCandidates], cand_i[kCandidates];
  __shared__ Best part[32], cluster_best[8];
  __shared__ double dpart[32];
  __shared__ float fpart[32];
  __shared__ int ipart[32];
  __shared__ int sh_count, sh_bin, sh_ties;
  __shared__ float sh_cut;

  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  // announce that this block runs; the wait stands before the first store into another's memory
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
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
  // Combines x and y over the cluster with `op`, in rank order; also a cluster barrier.
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

  // ---- the slice, NaN as -inf, in 16-byte groups from its first element on.  Where the row does
  // not start on 16 bytes a group is cut out of two aligned vectors, so that a thread's elements,
  // and with them the order of every sum, do not depend on where the row lies.
  const int shift = (int)((uintptr_t)logits & 15);  // in bytes
  L* slice = reinterpret_cast<L*>(slice_raw);
  const int vectors = (n + W - 1) / W;
  for (int b = tid; b < kBins; b += kSliceThreads) hist[b] = total[b] = 0;
  float greatest = -INFINITY;  // of this thread's
  {
    const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(logits) - shift);
    const int ahead = shift ? W : 0;
#pragma unroll 4
    for (int v = tid; v < vectors; v += kSliceThreads) {
      uint4 x;
      L* e = reinterpret_cast<L*>(&x);
      if ((shift == 0 || v > 0) && (v + 1) * W + ahead <= n) {
        x = from[v];
        if (shift) {
          const uint4 y = from[v + 1];
          const uint32_t bits = (shift & 3) * 8;
          uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          if (shift & 8) {
#pragma unroll
            for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
          }
          if (shift & 4) {
#pragma unroll
            for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
          }
          x = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                         __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
        }
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
          e[j] = v * W + j < n ? logits[v * W + j] : from_f32<L>(-INFINITY);
      }
      greatest = fmaxf(greatest, settle<L>(x));
      slice_raw[v] = x;
    }
  }
  const float block_top = block_max(greatest);
  asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");  // every block has started
  float top = (float)over_cluster(block_top, 0., most).x;
  if (top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  if (top == INFINITY) {  // infinite logits share all the probability
    for (int i = tid; i < n; i += kSliceThreads)
      slice[i] = from_f32<L>(to_f32<L>(slice[i]) == INFINITY ? 0.f : -INFINITY);
    greatest = greatest == INFINITY ? 0.f : -INFINITY;
    top = 0.f;
    __syncthreads();
  }
  // f(value, index in the slice) for every finite logit; a thread's come in rising order
  const auto each = [&](auto f) {
    for (int v = tid; v < vectors; v += kSliceThreads) {
      const uint4 x = slice_raw[v];
      const L* e = reinterpret_cast<const L*>(&x);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float l = to_f32<L>(e[j]);
        if (l > -INFINITY) f(l, v * W + j);
      }
    }
  };
  // the same for the finite logits from `least` on, of which there are few: a vector's greatest first
  const auto each_from = [&](float least, auto f) {
    for (int v = tid; v < vectors; v += kSliceThreads) {
      const uint4 x = slice_raw[v];
      if (greatest_of<L>(x) < least) continue;
      const L* e = reinterpret_cast<const L*>(&x);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float l = to_f32<L>(e[j]);
        if (l >= least && l > -INFINITY) f(l, v * W + j);
      }
    }
  };
  // above 0 under an infinite temperature too, so that the weight of -inf stays 0 and no NaN
  const float per_unit = fmaxf(fminf(kLog2e / div, FLT_MAX), FLT_TRUE_MIN);
  const auto weight = [&](float l) { return exp2_approx((l - top) * per_unit); };
  // t less the greatest t (of a finite logit): the logits are subtracted first, so that it is exact
  // near the top and finite there, where t itself passes fp32 at the smallest temperatures
  const auto below_top = [&](float l) { return (l - top) / div; };

  // ---- sum of the weights, and the threads' greatest in steps below the greatest
  const bool limited = hot && (k < V || p < 1.f);
  const float bins_per_logit = fminf(kBinsPerUnit / div, FLT_MAX);
  const auto bin_of = [&](float l) { return min((int)((top - l) * bins_per_logit), kBins - 1); };

  float z = 0.f;
  int finite = 0;
#pragma unroll 2
  for (int v = tid; v < vectors; v += kSliceThreads) {
    const uint4 x = slice_raw[v];
    const L* e = reinterpret_cast<const L*>(&x);
    float w[W];
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = weight(to_f32<L>(e[j]));
#pragma unroll
    for (int d = W / 2; d; d /= 2)
#pragma unroll
      for (int j = 0; j < d; ++j) w[j] += w[j + d];
    z += w[0];
    if (k < V) {
#pragma unroll
      for (int j = 0; j < W; ++j) finite += to_f32<L>(e[j]) > -INFINITY;
    }
  }
  if (limited && greatest > -INFINITY) atomicAdd(&hist[bin_of(greatest)], 1u);
  const double zs = block_sum(z), fs = block_sum(finite);
  if (limited) {  // this block's histogram added to block 0's
    uint32_t* all = cluster.map_shared_rank(total, 0);
    __syncthreads();
    for (int b = tid; b < kBins; b += kSliceThreads)
      if (hist[b]) atomicAdd(all + b, hist[b]);
  }
  const double2 both = over_cluster(zs, fs, add);
  const double Z = both.x;
  const int usable = k < V ? (int)both.y : V;  // where top_k is off, not asked for
  const float log_z = logf((float)Z);
  const auto answer = [&](int index, float l) {
    a.tokens[row] = index;
    if (a.logprobs) a.logprobs[row] = below_top(l) - log_z;
  };
  const auto heavy_enough = [&](float l) { return l == top || expf(below_top(l)) >= least_weight; };
  // t - log(noise) less the greatest t, a NaN last
  const auto key_of = [&](float l, float e) {
    const float s = below_top(l) - logf(e);
    return isnan(s) ? -INFINITY : s;
  };

  // ---- the best t - log(noise) among the tokens ranked above (bound_l, bound_i); all above -inf
  __shared__ float best_l_of[8];
  const auto draw = [&](float bound_l, int bound_i, float& won_l) {
    Best best = {-INFINITY, INT32_MAX};
    float best_l = 0.f;
    const auto ranked_above = [&](float l, int i) {
      return l > bound_l || (l == bound_l && first + i < bound_i);
    };
    const auto consider = [&](float l, int i, float e) {
      const Best b = {key_of(l, e), first + i};
      if (b.value > best.value || (b.value == best.value && b.index < best.index))
        best = b, best_l = l;
    };
    if (!hot) {
      each_from(top, [&](float l, int i) {
        if (first + i < best.index) best = {l, first + i}, best_l = l;
      });
    } else if (least_weight > 0.f) {
      // those that may be heavy enough, a little below the least weight's logit (roundings: 2^-22
      // of t's distance from the top, 2^-24 each of the two logits)
      const float t = logf(least_weight);
      float least = top + (t - 1e-3f - fabsf(t) * 5e-7f) * div;
      least -= (fabsf(least) + fabsf(top)) * 2e-7f;
      each_from(least, [&](float l, int i) {
        if (ranked_above(l, i) && heavy_enough(l)) consider(l, i, noise[i]);
      });
    } else {
      // The approximate keys of all, t log2(e) - log2(noise), the thread's greatest two kept: an
      // exact key costs four times as much, and in a warp of 32 some lane has a new greatest at
      // most steps.  Exact then are those within the approximation's reach of the block's
      // greatest (errors: 2^-23 of t log2(e), 2^-21 of the logarithm).
      float first_a = -INFINITY, second_a = -INFINITY;
      int first_i = 0;
      const auto approx = [&](float l, float e) { return l * per_unit - __log2f(e); };
      for (int i0 = tid; i0 < n; i0 += 8 * kSliceThreads) {
        float e[8], l[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = i0 + j * kSliceThreads;
          l[j] = i < n ? to_f32<L>(slice[i]) : -INFINITY;
          if (!ranked_above(l[j], i)) l[j] = -INFINITY;
          e[j] = l[j] > -INFINITY ? __ldcs(noise + i) : 1.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = approx(l[j], e[j]);
          second_a = fmaxf(second_a, fminf(first_a, x));
          if (x > first_a) first_a = x, first_i = i0 + j * kSliceThreads;
        }
      }
      const float most_a = block_max(first_a);
      const float within = most_a - 2e-3f - 1e-6f * fabsf(most_a);
      if (!(first_a < within)) {
        if (second_a < within) {
          consider(to_f32<L>(slice[first_i]), first_i, noise[first_i]);
        } else {
          for (int i = tid; i < n; i += kSliceThreads) {
            const float l = to_f32<L>(slice[i]);
            if (!(l > -INFINITY) || !ranked_above(l, i)) continue;
            const float e = noise[i];
            if (!(approx(l, e) < within)) consider(l, i, e);
          }
        }
      }
    }
    // over the block, then over the cluster: every block learns the winner
    const Best own = best;
    best = block_best(best, part);
    if (tid == 0) fpart[0] = 0.f;
    __syncthreads();
    if (own.index == best.index && best.index < V) fpart[0] = best_l;
    __syncthreads();
    if (tid < ranks) {
      cluster.map_shared_rank(cluster_best, tid)[rank] = best;
      cluster.map_shared_rank(best_l_of, tid)[rank] = fpart[0];
    }
    cluster.sync();
    Best won = cluster_best[0];
    won_l = best_l_of[0];
    for (int r = 1; r < ranks; ++r) {
      const Best b = cluster_best[r];
      if (b.value > won.value || (b.value == won.value && b.index < won.index))
        won = b, won_l = best_l_of[r];
    }
    return won;
  };

  if (limited) {
    uint32_t* all = cluster.map_shared_rank(total, 0);
    // Gathers the tokens from `least` on that `takes(l)` in block 0, if at most kCandidates, and
    // ranks them in its own_l, own_i; cluster barriers.  Returns their number.
    const auto gather = [&](float least, auto takes) {
      if (tid == 0) sh_count = 0;
      __syncthreads();
      each_from(least, [&](float l, int i) {
        if (!takes(l)) return;
        const int at = atomicAdd(&sh_count, 1);
        if (at < kCandidates) own_l[at] = l, own_i[at] = first + i;
      });
      __syncthreads();
      const int mine = sh_count;
      double(*box)[2] = sums.v[turn & 1];
      const int m = (int)over_cluster(mine, 0., add).x;
      if (m > kCandidates) return m;
      int before = 0;
      for (int r = 0; r < rank; ++r) before += (int)box[r][0];
      float* to_l = cluster.map_shared_rank(cand_l, 0);
      int* to_i = cluster.map_shared_rank(cand_i, 0);
      for (int j = tid; j < mine; j += kSliceThreads) {
        to_l[before + j] = own_l[j];
        to_i[before + j] = own_i[j];
      }
      cluster.sync();
      if (rank == 0) {
        if (tid < m) {
          const float l = cand_l[tid];
          const int i = cand_i[tid];
          int r = 0;
          for (int j = 0; j < m; ++j) r += cand_l[j] > l || (cand_l[j] == l && cand_i[j] < i);
          own_l[r] = l;
          own_i[r] = i;
        }
        __syncthreads();
      }
      return m;
    };
    const bool by_count = k < usable, by_mass = p < 1.f;

    // ---- how far down the threads' greatest reach the limit, if they do
    int reach;
    {
      if (tid == 0) sh_bin = kBins;
      const uint32_t c0 = all[2 * tid], c1 = all[2 * tid + 1];
      double v0 = c0, v1 = c1;
      if (!by_count) {  // the least mass they can have (nothing for the last, open bin)
        const auto edge = [&](int b) { return (double)weight(top - b / bins_per_logit) * (1. - 1e-4); };
        v0 *= edge(2 * tid + 1);
        v1 *= 2 * tid + 1 == kBins - 1 ? 0. : edge(2 * tid + 2);
      }
      const double want = by_count ? (double)k : (double)p * Z;
      double sum;
      const double through = block_scan_inclusive(v0 + v1, dpart, sum);
      if (through - v1 >= want) atomicMin(&sh_bin, 2 * tid);
      if (through >= want) atomicMin(&sh_bin, 2 * tid + 1);
      __syncthreads();
      reach = sh_bin;
    }
    if ((by_count || by_mass) && reach < kBins - 1) {
      // a compare first, one step too low, and the bins' exact test for what passes
      const float edge = top - (reach + 2) / bins_per_logit;
      const int m = gather(edge, [&](float l) { return bin_of(l) <= reach; });
      if (m <= kCandidates) {
        if (rank != 0) return;
        // ---- all limits on the ranked list
        const bool in = tid < m && (!by_count || tid < k);
        const float l = in ? own_l[tid] : -INFINITY;
        const double w = in ? (double)weight(l) : 0.;
        double kept_mass;
        const double before = block_scan_inclusive(w, dpart, kept_mass) - w;
        const double target = by_mass ? p * (by_count ? kept_mass : Z) : INFINITY;
        Best best = {-INFINITY, INT32_MAX};
        if (in && (tid == 0 || before < target) && heavy_enough(l))
          best = {key_of(l, a.noise[row * a.noise_stride + own_i[tid]]), own_i[tid]};
        const Best won = block_best(best, part);
        if (in && best.index == won.index) answer(won.index, l);
        return;
      }
    }

    // Count and mass of the tokens that `takes(l, i)`.
    const auto measure = [&](auto takes) {
      float m = 0.f;
      int c = 0;
      each([&](float l, int i) {
        if (takes(l, i)) m += weight(l), ++c;
      });
      return over_cluster(block_sum(m), block_sum(c), add);
    };
    // Strikes out what a limit does not keep: top_k (mass = false) or top_p with `want` of the mass
    const auto strike = [&](bool mass, double want) {
      // the least key that is kept, if only in part, is in (below, at]
      uint32_t at = order_key(top), below = order_key(-FLT_MAX) - 1;
      double above = 0.;                    // count or mass over `at`
      int over_at = 0, over_below = usable; // counts over `at` and over `below`
      while (at - below > 1 && over_below - over_at > kCandidates) {
        const uint32_t mid = below + (at - below) / 2;
        const double2 over = measure([&](float l, int) { return order_key(l) > mid; });
        const double v = mass ? over.x : over.y;
        if (v < want) at = mid, above = v, over_at = (int)over.y;
        else below = mid, over_below = (int)over.y;
      }
      if (at - below > 1) {
        const int m = gather(-INFINITY, [&](float l) {
          const uint32_t key = order_key(l);
          return key > below && key <= at;
        });
        if (rank == 0) {
          const float l = tid < m ? own_l[tid] : -INFINITY;
          const double w = tid >= m ? 0. : mass ? (double)weight(l) : 1.;
          double unused;
          const double before = above + block_scan_inclusive(w, dpart, unused) - w;
          const int kept = max((int)block_sum(tid < m && before < want ? 1. : 0.), 1);
          const float cut = own_l[kept - 1];
          const int ties = (int)block_sum(tid < kept && l == cut ? 1. : 0.);
          if (tid < ranks) {
            *cluster.map_shared_rank(&sh_cut, tid) = cut;
            *cluster.map_shared_rank(&sh_ties, tid) = ties;
          }
        }
        cluster.sync();
      } else {  // ties of one key: as many as the limit still takes
        const float cut = key_value(at);
        if (tid == 0) {
          const double w = mass ? weight(cut) : 1.;
          sh_cut = cut;
          sh_ties = w > 0. ? (int)fmin(ceil((want - above) / w), 2147483647.) : 1;
        }
        __syncthreads();
      }
      const float cut = sh_cut;
      const int ties = sh_ties;
      int mine = 0;
      each([&](float l, int) { mine += l == cut; });
      mine = (int)block_sum(mine);
      double(*box)[2] = sums.v[turn & 1];
      over_cluster(mine, 0., add);
      int before = 0;
      for (int r = 0; r < rank; ++r) before += (int)box[r][0];
      const int keeps = min(max(ties - before, 0), mine);
      int seen = 0;
      for (int i0 = 0; i0 < n; i0 += kSliceThreads) {
        const int i = i0 + tid;
        const float l = i < n ? to_f32<L>(slice[i]) : INFINITY;
        bool out = l < cut;
        if (keeps == 0) {
          out |= l == cut;
        } else if (keeps < mine) {
          int count;
          const int through = seen + block_scan_inclusive((int)(l == cut), ipart, count);
          out |= l == cut && through > keeps;
          seen += count;
        }
        if (out) slice[i] = from_f32<L>(-INFINITY);
      }
      __syncthreads();
    };

    double want = k;  // of the one limit left: a rank, or a mass
    bool left = by_count || by_mass;
    if (by_mass) {
      double mass = Z;
      if (by_count) {
        strike(false, k);
        mass = measure([](float, int) { return true; }).x;
      }
      want = fmax(p * mass, 1e-30);  // the greatest is always kept
    }
    if (left) {
      float bound_l = -INFINITY, l;
      int bound_i = 0;
      for (int turns = 0; turns < kDraws; ++turns) {
        const Best won = draw(bound_l, bound_i, l);
        const double2 over = measure([&](float x, int i) {
          return x > l || (x == l && first + i < won.index);
        });
        if ((by_mass ? over.x : over.y) < want) {
          if (rank == 0 && tid == 0) answer(won.index, l);
          return;
        }
        bound_l = l;
        bound_i = won.index;
      }
      strike(by_mass, want);
    }
  }

  float l;
  const Best won = draw(-INFINITY, 0, l);
  if (rank == 0 && tid == 0) answer(won.index, l);
}

template <typename L>
static int launch_sample(const SampleArgs& a, int64_t rows, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((int64_t)a.vocab * (int)sizeof(L) > 8 * kMaxSliceBytes) {  // more than a cluster holds
    sample_kernel<L><<<(unsigned)rows, kSampleThreads, 0, s>>>(a);
    return serve_launched("tr_sample");
  }
  // Blocks per row: as many as hold it in 64 KB each, more where the rows leave SMs idle.  Drawn
  // from all tokens (with top_k 50 and top_p 0.95), us with 2 / 4 / 8 blocks: one row of 50021 in
  // fp32 14.4 / 12.4 / 10.9 (18.4 / 16.5 / 16.5), 16 rows of 131072 in bf16 24.7 / 16.5 / 15.0
  // (22.6 / 18.5 / 19.8), 37 rows 26.8 / 21.3 / 26.2 (22.6 / 20.6 / 28.7), 256 rows 122 / 90 / 120
  // (100 / 79 / 125); 256 rows of 32000 with 1 / 2 / 4 blocks 22 / 29 / 39 (21 / 33 / 51).
  int blocks = 1;
  while (blocks < 8 && (a.vocab * (int)sizeof(L) > blocks * kSliceBytes ||
                        (a.vocab > blocks * 2048 && rows * blocks * 2 <= serve_sms())))
    blocks *= 2;
  const int slice = (a.vocab + blocks - 1) / blocks;
  const size_t smem = ((size_t)slice * sizeof(L) + 15) / 16 * 16;
  auto kernel = sample_cluster_kernel<L>;
  if (smem > 24 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSliceBytes + 64);
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
