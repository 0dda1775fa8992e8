// What the row operators' kernels share: element types, reductions, a launch that reports its own error.
#pragma once
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"
#include "rowops.h"

namespace eg {

using bf16_t = __bf16;
using f16_t = _Float16;

// one launch; hipLaunchKernel returns this launch's error (hipGetLastError could hand over an older one of the caller's)
template <typename... P, typename... A>
inline void row_launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t s, A... args) {
  std::tuple<P...> held{static_cast<P>(args)...};
  std::apply([&](P&... p) {
    void* ptrs[] = {const_cast<void*>(static_cast<const void*>(&p))...};
    EG_HIP(hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, ptrs, 0, s));
  }, held);
}

template <typename F>
void by_type(int type, F f) {
  if (type == ROW_F32) f(float{});
  else if (type == ROW_BF16) f(bf16_t{});
  else f(f16_t{});
}

__device__ __forceinline__ float row_act(float z, int act) {
  return act == ACT_NONE ? z : z > 0.f ? z : act == ACT_LRELU ? 0.2f * z : (z != z ? z : 0.f);
}
// derivative of row_act at the pre-activation z
__device__ __forceinline__ float row_act_grad(float z, int act) { return act == ACT_NONE || z > 0.f ? 1.f : act == ACT_LRELU ? 0.2f : 0.f; }

// Sums over the LANES (a power of two) neighbouring lanes of a wave.  Every lane gets the result.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    const float u = __shfl_xor(v, o, 64);
    v = (u > v || u != u) ? u : v;   // a NaN stays
  }
  return v;
}

// Sums of NV values over the block's NT threads (NT a multiple of 64), in one pass through `red`[NV * NT / 64].  The caller may
// use the same `red` again only behind a barrier of its own.
template <int NT, int NV>
__device__ __forceinline__ void block_sum(float (&v)[NV], float* red) {
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = lanes_sum<64>(v[i]);
  if constexpr (NT > 64) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    constexpr int NW = NT / 64;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < NV; ++i) red[i * NW + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float t = red[i * NW];
#pragma unroll
      for (int w = 1; w < NW; ++w) t += red[i * NW + w];
      v[i] = t;
    }
  }
}
template <int NT>
__device__ __forceinline__ float block_max(float v, float* red) {
  v = lanes_max<64>(v);
  if constexpr (NT > 64) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    constexpr int NW = NT / 64;
    if (lane == 0) red[wave] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      const float u = red[w];
      v = (u > v || u != u) ? u : v;
    }
  }
  return v;
}

}  // namespace eg
