// Helpers shared by the serving operators (serve_*.cu): 16-byte vectors of elements, warp and
// block reductions, host-side launch checks.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <cstdint>

#include "device_util.cuh"
#include "plan.h"

namespace trr {

// 8 consecutive elements as floats; p is aligned to 8 elements
template <typename E>
__device__ __forceinline__ void load8(const E* p, float (&f)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const float2 a = unpack2<E>(w.x), b = unpack2<E>(w.y), c = unpack2<E>(w.z),
               d = unpack2<E>(w.w);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = c.x, f[5] = c.y, f[6] = d.x, f[7] = d.y;
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&f)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
template <typename E>
__device__ __forceinline__ void store8(E* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2<E>(f[0], f[1]), pack2<E>(f[2], f[3]),
                                            pack2<E>(f[4], f[5]), pack2<E>(f[6], f[7]));
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename T>
__device__ __forceinline__ T warp_scan_inclusive(T v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// Inclusive scan over the block in thread order; `part` holds one value per warp (at most 32).
// Every thread calls it; `total` is the sum over the block.
template <typename T>
__device__ __forceinline__ T block_scan_inclusive(T v, T* part, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  v = warp_scan_inclusive(v);
  if (lane == 31) part[warp] = v;
  __syncthreads();
  T before = 0, all = 0;
  const T mine = lane < warps ? part[lane] : T(0);
  const T run = warp_scan_inclusive(mine);
  all = __shfl_sync(0xffffffffu, run, warps - 1);
  before = __shfl_sync(0xffffffffu, run - mine, warp);
  __syncthreads();
  total = all;
  return v + before;
}

// ---- host side
inline int serve_launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("%s launch: %s", what, cudaGetErrorString(e));
    return TR_ERR_CUDA;
  }
  return TR_OK;
}

// SMs of the current device (looked up once per device)
inline int serve_sms() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) n = 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

inline int element_bytes(int dtype) { return dtype == TR_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) {
  return dtype == TR_F32 || dtype == TR_F16 || dtype == TR_BF16;
}

}  // namespace trr
