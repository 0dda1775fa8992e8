// Product of 8-bit integer matrices with a scale for each row of either:
//   out[i][j] = (sum_k a[i][k] b[j][k]) a_scale[i] b_scale[j] + bias[j],  sums in 32-bit integers (exact: k <= 131,071)
// a is [m][k] (rows: tokens, positions), b is [n][k] (rows: output channels); both with k consecutive, which is the operand order of
// v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive k of row l & 15, group l >> 4.
#include <tuple>

#include "rowops_dev.h"

namespace eg {

using i32x4 = __attribute__((ext_vector_type(4))) int;

// 16 bytes of a row that may end or be unaligned anywhere: one load where it is aligned and whole, else byte by byte
__device__ __forceinline__ i32x4 load16(const signed char* row, int k, int k_end, bool aligned) {
  i32x4 v = {0, 0, 0, 0};
  if (k >= k_end) return v;
  if (aligned && k + 16 <= k_end) return *reinterpret_cast<const i32x4*>(row + k);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < k_end) v[i >> 2] |= (int)(unsigned char)row[k + i] << (8 * (i & 3));
  return v;
}

template <typename T>
__device__ __forceinline__ void store_out(const Int8Args& a, long long i, int j, int sum) {
  float v = __fmul_rn((float)sum * a.a_scale[i], a.b_scale[j]);
  if (a.bias) v += a.bias[j];
  ((T*)a.out)[i * a.ldo + j] = (T)v;
}

// Any sizes, strides and alignment: 64 x 64 outputs a block, a wave 32 x 32 of them, operands straight from memory.
template <typename T>
__global__ __launch_bounds__(256) void int8_any(Int8Args a, int tiles_n, int aligned_a, int aligned_b) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long i0 = (long long)(blockIdx.x / tiles_n) * 64 + (wave >> 1) * 32;
  const int j0 = (blockIdx.x % tiles_n) * 64 + (wave & 1) * 32;
  const int l15 = lane & 15, lk = (lane >> 4) * 16;
  i32x4 acc[2][2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) acc[x][y] = i32x4{0, 0, 0, 0};
  for (int k = 0; k < a.k; k += 64) {
    i32x4 fa[2], fb[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const long long i = i0 + x * 16 + l15;
      const int j = j0 + x * 16 + l15;
      fa[x] = i < a.m ? load16(a.a + i * a.lda, k + lk, a.k, aligned_a) : i32x4{0, 0, 0, 0};
      fb[x] = j < a.n ? load16(a.b + (long long)j * a.ldb, k + lk, a.k, aligned_b) : i32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[x], fb[y], acc[x][y], 0, 0, 0);
  }
  // result layout: lane l, register v: row 4 (l >> 4) + v, column l & 15
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const long long i = i0 + x * 16 + (lane >> 4) * 4 + v;
        const int j = j0 + y * 16 + l15;
        if (i < a.m && j < a.n) store_out<T>(a, i, j, acc[x][y][v]);
      }
}

size_t int8_partial_floats(long long m, int n, int k) { return 0; }

void launch_int8_matmul(const Int8Args& a, int out_type, float* partial, hipStream_t s) {
  if (a.m == 0 || a.n == 0) return;
  const int al_a = ((uintptr_t)a.a | (uintptr_t)a.lda) % 16 == 0, al_b = ((uintptr_t)a.b | (uintptr_t)a.ldb) % 16 == 0;
  const long long tiles_m = (a.m + 63) / 64, tiles_n = (a.n + 63) / 64;
  EG_CHECK(tiles_m * tiles_n < (1ll << 24), "int8 product: too many outputs (%lld x %d)", a.m, a.n);
  by_type(out_type, [&](auto t) {
    row_launch(int8_any<decltype(t)>, dim3((unsigned)(tiles_m * tiles_n)), dim3(256), s, a, (int)tiles_n, al_a, al_b);
  });
}

}  // namespace eg
