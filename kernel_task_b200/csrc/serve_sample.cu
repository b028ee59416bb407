// tr_sample: the next token of every row from logits, temperature, top-k, top-p, min-p and given
// random numbers.
#include <algorithm>

#include "serve_util.cuh"

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

template <typename L>
static int launch_sample(const SampleArgs& a, int64_t rows, void* stream) {
  sample_kernel<L><<<(unsigned)rows, kSampleThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return serve_launched("tr_sample");
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
