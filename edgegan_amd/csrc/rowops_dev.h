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

// A product that no following sum is contracted with into an fma: it is rounded by itself, wherever it is inlined.
__device__ __forceinline__ float rounded_mul(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}
template <int ACT>
__device__ __forceinline__ float row_act(float z) {   // a NaN stays
  if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;
  else if constexpr (ACT == ACT_LRELU) return fmaxf(z, 0.2f * z);
  else return z;
}
// derivative of row_act at the pre-activation z; at zero ReLU's is 0 and LeakyReLU's `at_zero`
__device__ __forceinline__ float row_act_grad(float z, int act, float at_zero) { return act == ACT_NONE || z > 0.f ? 1.f : act == ACT_LRELU ? (z < 0.f ? 0.2f : at_zero) : 0.f; }
// f(the activation as a type)
template <typename F>
__device__ __forceinline__ void by_act(int act, F f) {
  if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>{});
  else if (act == ACT_LRELU) f(std::integral_constant<int, ACT_LRELU>{});
  else f(std::integral_constant<int, ACT_NONE>{});
}

// One step of a butterfly over a wave, by data-parallel primitives (a few cycles; a shuffle goes through LDS): (a, b) are the values of the
// two lanes whose numbers differ in X, the same pair in the same order or the other way round in both.  For X = 4, 8 the mirrored lane stands in, which holds the
// same value once the smaller steps are done.
template <int X>
__device__ __forceinline__ void lane_pair(int v, int& a, int& b) {
  a = v;
  if constexpr (X == 1) b = __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);         // quad_perm [1,0,3,2]
  else if constexpr (X == 2) b = __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);    // quad_perm [2,3,0,1]
  else if constexpr (X == 4) b = __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true);   // row_half_mirror
  else if constexpr (X == 8) b = __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, true);   // row_mirror
  else if constexpr (X == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    a = (int)r[0];
    b = (int)r[1];
  } else {
    static_assert(X == 32, "a wave has 64 lanes");
    const auto r = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    a = (int)r[0];
    b = (int)r[1];
  }
}
template <int X>
__device__ __forceinline__ void lane_pair(float v, float& a, float& b) {
  int x, y;
  lane_pair<X>(__float_as_int(v), x, y);
  a = __int_as_float(x);
  b = __int_as_float(y);
}
template <int X>
__device__ __forceinline__ void lane_pair(double v, double& a, double& b) {
  int h0, h1, l0, l1;
  lane_pair<X>(__double2hiint(v), h0, h1);
  lane_pair<X>(__double2loint(v), l0, l1);
  a = __hiloint2double(h0, l0);
  b = __hiloint2double(h1, l1);
}
__device__ __forceinline__ float max_nan(float a, float b) { return (b > a || b != b) ? b : a; }   // a NaN stays
// Sum / maximum over LANES (a power of two) neighbouring lanes; every lane gets the result.
template <int LANES, int X = 1, typename V>
__device__ __forceinline__ V lanes_sum(V v) {
  if constexpr (X < LANES) {
    V a, b;
    lane_pair<X>(v, a, b);
    return lanes_sum<LANES, 2 * X>(a + b);
  } else
    return v;
}
template <int LANES, int X = 1>
__device__ __forceinline__ float lanes_max(float v) {
  if constexpr (X < LANES) {
    float a, b;
    lane_pair<X>(v, a, b);
    return lanes_max<LANES, 2 * X>(max_nan(a, b));
  } else
    return v;
}

// Sum / maximum over the NT threads that share a row: neighbouring lanes, or (NT > 64) waves through red[NT / 64]: every
// thread of the block has to come by, and teams of the same block have a `red` each.  Calls that follow one
// another use other memory, or a barrier lies between them.
template <int NT, typename V, int N>
__device__ __forceinline__ void team_sum(V (&v)[N], V* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<(NT < 64 ? NT : 64)>(v[i]);
  if constexpr (NT > 64) {
    constexpr int NW = NT / 64;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[i * NW + (threadIdx.x >> 6) % NW] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      V t = red[i * NW];
#pragma unroll
      for (int w = 1; w < NW; ++w) t += red[i * NW + w];
      v[i] = t;
    }
  }
}
template <int NT>
__device__ __forceinline__ float team_max(float v, float* red) {
  v = lanes_max<(NT < 64 ? NT : 64)>(v);
  if constexpr (NT > 64) {
    constexpr int NW = NT / 64;
    if ((threadIdx.x & 63) == 0) red[(threadIdx.x >> 6) % NW] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) v = max_nan(v, red[w]);
  }
  return v;
}

// V consecutive elements: one aligned load / store of V sizeof(T) bytes
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T e[V];
};
// A row as a buffer of its own: a load past its end gives zero and a store there is dropped, and an element's address is one register. The row
// has to be the same one for the whole wave.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const void* p, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> buffer_load(__amdgpu_buffer_rsrc_t b, unsigned offset) {
  static_assert(sizeof(Pack<T, V>) == 2 || sizeof(Pack<T, V>) == 4 || sizeof(Pack<T, V>) == 16, "");
  if constexpr (sizeof(Pack<T, V>) == 2) return __builtin_bit_cast(Pack<T, V>, __builtin_amdgcn_raw_buffer_load_b16(b, offset, 0, 0));
  else if constexpr (sizeof(Pack<T, V>) == 4) return __builtin_bit_cast(Pack<T, V>, __builtin_amdgcn_raw_buffer_load_b32(b, offset, 0, 0));
  else return __builtin_bit_cast(Pack<T, V>, __builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, 0));
}
template <typename T, int V>
__device__ __forceinline__ void buffer_store(__amdgpu_buffer_rsrc_t b, unsigned offset, const float (&v)[V]) {
  Pack<T, V> k;
#pragma unroll
  for (int i = 0; i < V; ++i) k.e[i] = (T)v[i];
  using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
  if constexpr (sizeof(k) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, k), b, offset, 0, 0);
  else if constexpr (sizeof(k) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, k), b, offset, 0, 0);
  else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, k), b, offset, 0, 0);
}
// A value that the compiler forms anew in each turn of a loop instead of keeping everything that depends on it in registers from turn to turn.
__device__ __forceinline__ int fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// ---- what the layer norm, the quantisation and the 8-bit layer for few rows share -----------------------------------------------------
template <typename W>
__device__ __forceinline__ float affine(float xh, const W* gamma, const W* beta, int c) {
  const float z = gamma ? rounded_mul(xh, (float)gamma[c]) : xh;
  return beta ? z + (float)beta[c] : z;
}

// A row of `cols` elements over NT threads, each NV packs of V consecutive elements: pack i of thread t begins at column (i NT + t) V.  A pack is one load or store at
// any address of the element type (the hardware takes unaligned ones).  TAIL: cols need not be a multiple of V; the last pack then
// goes element by element.  cols >= V.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) LoosePack {
  T e[V];
};
template <typename T, int NT, int NV, int V>
__device__ __forceinline__ void request_row(const T* p, int cols, int t, LoosePack<T, V> (&k)[NV]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) k[i] = *reinterpret_cast<const LoosePack<T, V>*>(p + min((i * NT + t) * V, cols - V));   // (no branch: all of a thread's loads in flight at once)
}
// the cut pack: what was loaded are the row's last V elements, of which its first cols % V are the last ones; `fill` behind them
template <typename T, int NT, int NV, int V, bool TAIL>
__device__ __forceinline__ void settle_row(int cols, int t, LoosePack<T, V> (&k)[NV], T fill = (T)0.f) {
  if constexpr (TAIL) {
    const int at = cols / V / NT, shift = V - cols % V;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i == at && (i * NT + t) * V + V > cols)
#pragma unroll
        for (int by = 1; by < V; by *= 2)
          if (shift & by)
#pragma unroll
            for (int j = 0; j < V; ++j) k[i].e[j] = j + by < V ? k[i].e[j + by] : fill;
  }
}
// A whole row as f32, zeros past its end
template <typename T, int NT, int NV, int V, bool TAIL>
__device__ __forceinline__ void load_row(const T* p, int cols, int t, float (&v)[NV][V]) {
  LoosePack<T, V> k[NV];
  request_row<T, NT, NV, V>(p, cols, t, k);
  settle_row<T, NT, NV, V, TAIL>(cols, t, k);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = (i * NT + t) * V < cols ? (float)k[i].e[j] : 0.f;
}
// f(i, column) for a thread's packs that begin inside the row (what the others hold is of no use)
template <int NT, int NV, int V, typename F>
__device__ __forceinline__ void each_pack(int cols, int t, F f) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * NT + t) * V;
    if (c < cols) f(i, c);
  }
}
template <typename T, int V, bool TAIL>
__device__ __forceinline__ void store_row_pack(T* p, int c, int cols, const float (&v)[V]) {
  LoosePack<T, V> k;
#pragma unroll
  for (int j = 0; j < V; ++j) k.e[j] = (T)v[j];
  if (!TAIL || c + V <= cols) *reinterpret_cast<LoosePack<T, V>*>(p + c) = k;
  else
#pragma unroll
    for (int j = 0; j < V - 1; ++j)
      if (j < cols % V) p[c + j] = k.e[j];
}
// a vector of parameters in a row's order: its packs, if it is there
template <typename W, int NT, int NV, int V, bool TAIL>
struct Parameter {
  LoosePack<W, V> k[NV];
  __device__ __forceinline__ void load(const W* p, int cols, int t) {
    if (!p) return;
    request_row<W, NT, NV, V>(p, cols, t, k);
    settle_row<W, NT, NV, V, TAIL>(cols, t, k);
  }
};
// pairwise: of equal values exactly
template <int V>
__device__ __forceinline__ float tree_sum(const float (&v)[V]) {
  if constexpr (V == 1) return v[0];
  else {
    float h[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) h[i] = v[2 * i] + v[2 * i + 1];
    return tree_sum(h);
  }
}
// (var + eps)^-1/2.  A variance of more than 2^127 (numbers above 10^19, masks of the type's lowest value) is brought into f32's range and the root taken back by an
// exact power of two.
__device__ __forceinline__ float row_rstd(double var, float eps) {
  if (var > 0x1p127) return 1.f / (sqrtf((float)(var * 0x1p-128)) * 0x1p64f);
  return 1.f / sqrtf((float)var + eps);
}
template <int NT, int NV, int V, bool TAIL>
__device__ __forceinline__ void subtract_mean(float (&v)[NV][V], int cols, int t, float m) {
  each_pack<NT, NV, V>(cols, t, [&](int i, int c) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] -= m;
    if (TAIL && i == cols / V / NT)
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = c + j < cols ? v[i][j] : 0.f;
  });
}
template <typename T>
constexpr bool may_run_over = !std::is_same_v<T, f16_t>;   // (the sums of f32 below: 65,504^2 is far from its end)
__device__ __forceinline__ bool finite(double v) { return fabs(v) <= 1.7976931348623157e308; }
// mean and rstd of a row in registers, packs summed in f32 and their sums in f64; the row becomes x - mean (zeros past the end of a cut pack).
// A pack's sum may run over in f32 (four of the type's lowest value, squares of numbers above 10^19): true then, and centre_row_again has to follow on the row as it was.
template <int NT, int NV, int V, bool TAIL>
__device__ __forceinline__ bool centre_row(float (&v)[NV][V], int cols, int t, float eps, double* red, float& mean, float& rstd) {
  double s[1] = {0.};
  each_pack<NT, NV, V>(cols, t, [&](int i, int) { s[0] += (double)tree_sum(v[i]); });
  team_sum<NT>(s, red);
  mean = (float)(s[0] / cols);
  subtract_mean<NT, NV, V, TAIL>(v, cols, t, mean);
  s[0] = 0.;
  each_pack<NT, NV, V>(cols, t, [&](int i, int) {
    float sq[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sq[j] = rounded_mul(v[i][j], v[i][j]);   // (the same wherever it is inlined)
    s[0] += (double)tree_sum(sq);
  });
  team_sum<NT>(s, red + NT / 64);
  rstd = 1.f / sqrtf((float)(s[0] / cols) + eps);
  return !finite(s[0]);   // (a finite sum is of f32 numbers, and so is their mean one)
}
// The same with every element summed in f64, for the teams whose row ran over (the others only come by); a row that holds a NaN or an infinity stays what it is.
template <int NT, int NV, int V, bool TAIL>
__device__ __forceinline__ void centre_row_again(float (&v)[NV][V], int cols, int t, float eps, double* red, bool over, float& mean, float& rstd) {
  double s[1] = {0.};
  each_pack<NT, NV, V>(cols, t, [&](int i, int c) {
#pragma unroll
    for (int j = 0; j < V; ++j) s[0] += c + j < cols ? (double)v[i][j] : 0.;
  });
  team_sum<NT>(s, red);
  mean = over ? (float)(s[0] / cols) : mean;
  subtract_mean<NT, NV, V, TAIL>(v, cols, t, mean);
  s[0] = 0.;
  each_pack<NT, NV, V>(cols, t, [&](int i, int) {
#pragma unroll
    for (int j = 0; j < V; ++j) s[0] += (double)v[i][j] * (double)v[i][j];
  });
  team_sum<NT>(s, red + NT / 64);
  rstd = over ? row_rstd(s[0] / cols, eps) : rstd;
}
// The rows r, r + step, ... of a team that ran over: the row v without its mean goes to finish(row, v, mean, rstd).  A pass of its own behind the others, which a kernel
// enters if centre_row has said so of any of its rows (of a block of one team: a whole block then).  In the loop over the rows a branch to it would cost every row: 8,192 x
// 2,048 bf16 18.2 us against 17.4.
template <typename T, int NT, int NV, int V, bool TAIL, typename F>
__device__ __forceinline__ void rows_that_ran_over(const T* x, long long ldx, long long r, long long rows, long long step, int cols, int t, float eps, double (&red)[2][NT > 64 ? 2 * NT / 64 : 1], F finish) {
  for (; r < rows; r += step) {
    float v[NV][V], mean, rstd;
    if constexpr (NT > 64) __syncthreads();   // (whatever was read from red and what finish shares)
    load_row<T, NT, NV, V, TAIL>(x + r * ldx, cols, t, v);
    if (!centre_row<NT, NV, V, TAIL>(v, cols, t, eps, red[0], mean, rstd)) continue;   // (the team is of one mind)
    load_row<T, NT, NV, V, TAIL>(x + r * ldx, cols, t, v);
    centre_row_again<NT, NV, V, TAIL>(v, cols, t, eps, red[1], true, mean, rstd);
    finish(r, v, mean, rstd);
  }
}
constexpr int centre_lds(int nt) { return nt > 64 ? 2 * nt / 64 : 1; }   // doubles

// The whole number nearest to 127 v / amax, exactly: inv = 127 / amax in 64 bits; v inv + 98304 is rounded once (fma) to a multiple of
// 2^-36, where a true tie lands on the tie (the product is off by under 2^-45) and nothing else does (127 v / amax is at least 2^-33 from a
// border that it is not on: with x's last bit u >= 2^-32 amax, 254 v - odd amax is a multiple of u).  Adding 1.5 2^52 then rounds to whole numbers, ties to even, and the
// sum's low byte is the signed 8-bit result (98304 = 0x18000).
__device__ __forceinline__ unsigned quantize1(float v, double inv) {
  const double t = __builtin_fma((double)v, inv, 98304.0) + 6755399441055744.0;
  return (unsigned)__double2loint(t) & 0xffu;
}
// false for infinity and NaN: such a row's scale is NaN, its values zero
__device__ __forceinline__ bool quantizable(float amax) { return amax <= 3.4028235e38f; }
__device__ __forceinline__ double quantize_factor(float amax) { return quantizable(amax) && amax > 0.f ? 127.0 / (double)amax : 0.0; }
__device__ __forceinline__ float quantize_scale(float amax) { return quantizable(amax) ? amax / 127.f : __builtin_nanf(""); }

}  // namespace eg
