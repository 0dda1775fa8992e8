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

// the same operations in every kernel, so that a result does not depend on the variant
__device__ __forceinline__ float int8_result(int sum, float sa, float sb, float bias) { return rounded_mul(rounded_mul((float)sum, sa), sb) + bias; }

// Any sizes, strides and alignment: 64 x 64 outputs a block, a wave 32 x 32 of them, operands straight from memory, byte by byte where they are not aligned: 23 x 8190 x 2050 204 us
// (rows at a pitch of 16 bytes take the tiles below: 6.4), 1024 x 1024 x 1001 95.
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
        if (i < a.m && j < a.n) ((T*)a.out)[i * a.ldo + j] = (T)int8_result(acc[x][y][v], a.a_scale[i], a.b_scale[j], a.bias ? a.bias[j] : 0.f);
      }
}

// ---- tiles in LDS ------------------------------------------------------------------------------------------------------------------
// BM x BN outputs a block by KS parts of WM x WN waves; a part takes every KS-th 64 bytes of k, and the parts' sums are joined through LDS at the end. A ring of
// RING buffers a part: while a step's 32x32x32 products run, the tiles of the next RING - 1 are on their way from memory straight to LDS.
// Bound by the matrix cores where there are tiles for every CU (8192 x 8192 x 4096, random values: 270 - 310 us, 1,770 - 2,030 TOPS, and 220 us with zeros: the clock
// gives way to power; the library's product takes 292), by a step's latency where there are few (a step is about 400 cycles of LDS, products and
// barrier whatever the tile), so that small products have small tiles and KS parts: 128 x 4096 x 4096 took 22 us in tiles of 128 x 128 with one part and takes 8.1.
// A deeper ring gained nothing (8 buffers: 22.4); 128 bytes a step with two buffers nothing at large k and lost 6 % at k = 64; 128 x 256 tiles two a CU
// were 10 % faster at k = 256 and 11 % slower at 4096; rows gathered in LDS for 16-byte stores 5 - 50 % slower than the stores here.
// A tile row is four 16-byte groups; group s of row r holds the row's group s ^ (r / 4 & 3), so that sixteen rows of a
// fragment lie in all 64 banks (the write is a wave's 1,024 consecutive bytes: the permutation is in the source addresses).
// Rows past the end repeat the last one (their results are not stored); groups past k read as zeros; the bytes past k in its last group are cleared
// in a's fragments, which is enough.
using i32x16 = __attribute__((ext_vector_type(16))) int;
constexpr int kStep = 64;

template <int BM, int BN, int WM, int WN, int RING_>
struct TileShape {
  static constexpr int RING = RING_, NW = WM * WN, MI = BM / WM / 32, NI = BN / WN / 32, JA = BM / 16 / NW, JB = BN / 16 / NW, BYTES = (BM + BN) * kStep, B_AT = BM * kStep;
  static_assert(JA * 16 * NW == BM && JB * 16 * NW == BN, "whole rows of 16 for every wave");
};
// A wave's part of a tile: N times 16 rows, straight into LDS
template <int N>
__device__ __forceinline__ void request_tile(__amdgpu_buffer_rsrc_t from, const unsigned (&voff)[N], bool in, int k, signed char* to, int waves, int wave) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const unsigned v = in ? voff[j] : 0x80000000u;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(to + (j * waves + wave) * 16 * kStep), 16, v, k, 0, 0);
  }
}
// One step: the tiles of three steps on requested (into `next`), the current ones multiplied.  The buffers are different memory and said to be (restrict): the compiler
// would otherwise wait for the requests before it reads the current tiles.  LAST: nothing to request, and a's bytes past k are cleared.
template <typename S, int TURN, bool LAST>
__device__ __forceinline__ void int8_step(const signed char* __restrict__ cur, signed char* __restrict__ next, __amdgpu_buffer_rsrc_t ab, __amdgpu_buffer_rsrc_t bb,
                                          const unsigned (&va)[S::JA], const unsigned (&vb)[S::JB], int koff, int k_all, int k, int wave, int lane, int arow, int brow,
                                          i32x16 (&acc)[S::MI][S::NI]) {
  if constexpr (!LAST) {
    const int ahead = k + (S::RING - 1) * TURN;
    const bool in = ahead + koff < k_all;   // (past k: zeros, from no memory)
    request_tile<S::JA>(ab, va, in, ahead, next, S::NW, wave);
    request_tile<S::JB>(bb, vb, in, ahead, next + S::B_AT, S::NW, wave);
    __builtin_amdgcn_sched_barrier(0);   // (the requests first: the scheduler would put them behind the products)
  }
  const int l31 = lane & 31, lh = lane >> 5;
#pragma unroll
  for (int ks = 0; ks < kStep / 32; ++ks) {
    const int slot = ((ks * 2 + lh) ^ ((l31 >> 2) & 3)) * 16;
    i32x4 fa[S::MI], fb[S::NI];
#pragma unroll
    for (int x = 0; x < S::MI; ++x) fa[x] = *reinterpret_cast<const i32x4*>(cur + (arow + x * 32) * kStep + slot);
#pragma unroll
    for (int y = 0; y < S::NI; ++y) fb[y] = *reinterpret_cast<const i32x4*>(cur + S::B_AT + (brow + y * 32) * kStep + slot);
    if constexpr (LAST) {
      const int ends = k_all - k - (ks * 2 + lh) * 16;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int keep = min(max(ends - 4 * d, 0), 4), mask = keep == 4 ? -1 : (1 << (8 * keep)) - 1;
#pragma unroll
        for (int x = 0; x < S::MI; ++x) fa[x][d] &= mask;
      }
    }
#pragma unroll
    for (int x = 0; x < S::MI; ++x)
#pragma unroll
      for (int y = 0; y < S::NI; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[x], fb[y], acc[x][y], 0, 0, 0);
  }
}

// Every wave's requests but those of the last RING - 2 steps have arrived, and every wave's reads of the buffer before are done.  (__syncthreads would wait for
// all requests.)
template <typename S>
__device__ __forceinline__ void tiles_ready() {
  static_assert((S::RING - 2) * (S::JA + S::JB) < 64, "what vmcnt can count");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S::RING - 2) * (S::JA + S::JB)) : "memory");
}

template <typename T, int BM, int BN, int WM, int WN, int KS, int RING>
__global__ __launch_bounds__(KS * WM * WN * 64) void int8_tiles(Int8Args a, int tiles_n) {
  using S = TileShape<BM, BN, WM, WN, RING>;
  constexpr int TURN = KS * kStep;   // bytes of k a step of the block takes
  constexpr int TILES = RING * S::BYTES, SUMS = KS > 1 ? KS * BM * BN * 4 : 0;   // a part's ring (of a's tile, b's tile); later the parts' sums
  __shared__ __attribute__((aligned(16))) signed char lds[std::max(KS * TILES, SUMS + BM * 4)];
  const int lane = threadIdx.x & 63, all_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = KS > 1 ? all_wave / S::NW : 0, wave = all_wave - part * S::NW;
  signed char* const ring = lds + part * TILES;
  const int wm = wave / WN, wn = wave % WN;
  const int tile = blockIdx.x;
  const int tm = __builtin_amdgcn_readfirstlane(tile / tiles_n), tn = tile - tm * tiles_n;
  const long long i0 = (long long)tm * BM;
  const int j0 = tn * BN;

  const __amdgpu_buffer_rsrc_t ab = row_buffer(a.a + i0 * a.lda, 0x7ffffff0u), bb = row_buffer(a.b + (long long)j0 * a.ldb, 0x7ffffff0u);
  const int koff = ((lane & 3) ^ ((lane >> 4) & 3)) * 16;   // this lane's group of its rows (16 (j NW + wave) + lane / 4) in k
  const int rows_a = (int)min((long long)BM, a.m - i0) - 1, rows_b = min(BN, a.n - j0) - 1;
  unsigned va[S::JA], vb[S::JB];
#pragma unroll
  for (int j = 0; j < S::JA; ++j) va[j] = (unsigned)min((j * S::NW + wave) * 16 + (lane >> 2), rows_a) * (unsigned)a.lda + koff;
#pragma unroll
  for (int j = 0; j < S::JB; ++j) vb[j] = (unsigned)min((j * S::NW + wave) * 16 + (lane >> 2), rows_b) * (unsigned)a.ldb + koff;
  i32x16 acc[S::MI][S::NI];
#pragma unroll
  for (int x = 0; x < S::MI; ++x)
#pragma unroll
    for (int y = 0; y < S::NI; ++y)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[x][y][v] = 0;
  const int l31 = lane & 31, lh = lane >> 5;
  const int arow = wm * (BM / WM) + l31, brow = wn * (BN / WN) + l31;
  int k = part * kStep, cur = 0;
#pragma unroll
  for (int p = 0; p < RING - 1; ++p) {
    request_tile<S::JA>(ab, va, p * TURN + k + koff < a.k, p * TURN + k, ring + p * S::BYTES, S::NW, wave);
    request_tile<S::JB>(bb, vb, p * TURN + k + koff < a.k, p * TURN + k, ring + p * S::BYTES + S::B_AT, S::NW, wave);
  }
  for (int left = a.k; left > TURN; left -= TURN, k += TURN, cur = (cur + 1) % RING) {
    tiles_ready<S>();
    int8_step<S, TURN, false>(ring + cur * S::BYTES, ring + (cur + RING - 1) % RING * S::BYTES, ab, bb, va, vb, koff, a.k, k, wave, lane, arow, brow, acc);
  }
  // the scales and the bias on their way before the last step
  static_assert(BM <= KS * S::NW * 64, "a thread for each row's scale");
  const int jw = wn * (BN / WN) + l31, iw = wm * (BM / WM) + lh * 4;
  const float sa_mine = a.a_scale[i0 + min((int)threadIdx.x, rows_a)];
  float sb[S::NI], bias[S::NI];
#pragma unroll
  for (int y = 0; y < S::NI; ++y) {
    const int j = j0 + min(jw + y * 32, rows_b);
    sb[y] = a.b_scale[j];
    bias[y] = a.bias ? a.bias[j] : 0.f;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (the last step; and no request is left that would write where the scales go)
  __syncthreads();
  int8_step<S, TURN, true>(ring + cur * S::BYTES, nullptr, ab, bb, va, vb, koff, a.k, k, wave, lane, arow, brow, acc);
  // The products behind here, then 16 idle cycles before anything reads the sums: the compiler's own count of them was seen to miss reads behind a
  // branch (a single product a wave: sums of rows 27 and 31 came out wrong).
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  // result layout: lane l, register v: row 8 (v / 4) + 4 (l >> 5) + v % 4, column l & 31
  int* sums = reinterpret_cast<int*>(lds) + wave * 64 + lane;   // of one register of one part: all its waves' lanes in a row
  float* scales = reinterpret_cast<float*>(lds + SUMS);         // the rows' scales
  constexpr int NEXT = S::NW * 64;
  __syncthreads();
  if (threadIdx.x < BM) scales[threadIdx.x] = sa_mine;
  if constexpr (KS > 1) {
#pragma unroll
    for (int x = 0; x < S::MI; ++x)
#pragma unroll
      for (int y = 0; y < S::NI; ++y)
#pragma unroll
        for (int v = 0; v < 16; ++v) sums[(((part * S::MI + x) * S::NI + y) * 16 + v) * NEXT] = acc[x][y][v];
  }
  __syncthreads();
  // (a row or column past the end has an offset past the buffer's: its store is dropped)
  const __amdgpu_buffer_rsrc_t ob = row_buffer((T*)a.out + i0 * a.ldo + j0, 0x7ffffff0u);
#pragma unroll
  for (int x = 0; x < S::MI; ++x)
#pragma unroll
    for (int u = 0; u < 16 / KS; ++u) {
      const int v = KS > 1 ? part * (16 / KS) + u : u;   // each part finishes its share of the registers
      const int i = iw + x * 32 + (v >> 2) * 8 + (v & 3);
      const float sa = scales[i];
      const unsigned at = i <= rows_a ? (unsigned)(i * (int)a.ldo + jw) * (unsigned)sizeof(T) : 0x80000000u;
#pragma unroll
      for (int y = 0; y < S::NI; ++y) {
        int sum;
        if constexpr (KS > 1) {
          sum = 0;
#pragma unroll
          for (int p = 0; p < KS; ++p) sum += sums[(((p * S::MI + x) * S::NI + y) * 16 + v) * NEXT];
        } else {
          sum = acc[x][y][u];
        }
        const float o[1] = {int8_result(sum, sa, sb[y], bias[y])};
        buffer_store<T, 1>(ob, jw + y * 32 <= rows_b ? at + y * 32 * (unsigned)sizeof(T) : 0x80000000u, o);
      }
      if (u % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
}

// ---- few rows of a ----------------------------------------------------------------------------------------------------------------
// Up to 16 rows: bound by the bytes of b and by the time a load takes (1 x 4096 x 4096: 4.4 us, 3.8 TB/s; with the quantisation and a layer norm in it 7.5). A block takes 16 rows of b, its eight waves k by turns of 128 bytes, eight loads of b a
// lane in flight; a comes from the caches or, where it is quantised in the same launch, from LDS.  The waves' sums are joined through LDS.
constexpr int kFewWaves = 8, kFewTurn = kFewWaves * 128, kFewAhead = 4;   // kFewAhead: turns at once
using FewOperand = i32x4[kFewAhead][2];

__device__ __forceinline__ void few_request(__amdgpu_buffer_rsrc_t from, unsigned row, int k0, int lk, int k_all, FewOperand& f) {
#pragma unroll
  for (int u = 0; u < kFewAhead; ++u)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + u * kFewTurn + h * 64;
      const unsigned off = k + lk < k_all ? row + k : 0x80000000u;   // (groups past k read as zeros)
      f[u][h] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(from, off, 0, 0));
    }
}
__device__ __forceinline__ void few_products(const FewOperand& fa, const FewOperand& fb, i32x4& acc) {
#pragma unroll
  for (int u = 0; u < kFewAhead; ++u)
#pragma unroll
    for (int h = 0; h < 2; ++h) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[u][h], fb[u][h], acc, 0, 0, 0);
}
// joins the waves' sums and writes the block's outputs; a_scale of row i
template <typename T, typename S>
__device__ __forceinline__ void few_finish(const Int8Args& a, int (&sums)[kFewWaves][4][64], const i32x4& acc, int j0, int lane, int wave, S a_scale) {
#pragma unroll
  for (int v = 0; v < 4; ++v) sums[wave][v][lane] = acc[v];
  __syncthreads();
  // result layout: lane l, register v: row 4 (l >> 4) + v, column l & 15
  if (wave >= 4) return;
  const int i = (lane >> 4) * 4 + wave, j = j0 + (lane & 15);
  if (i >= a.m || j >= a.n) return;
  int sum = 0;
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) sum += sums[w][wave][lane];
  ((T*)a.out)[i * a.ldo + j] = (T)int8_result(sum, a_scale(i), a.b_scale[j], a.bias ? a.bias[j] : 0.f);
}

template <typename T>
__global__ __launch_bounds__(kFewWaves * 64) void int8_few(Int8Args a) {
  __shared__ int sums[kFewWaves][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l15 = lane & 15, lk = (lane >> 4) * 16;
  const int j0 = blockIdx.x * 16;
  const __amdgpu_buffer_rsrc_t ab = row_buffer(a.a, 0x7ffffff0u), bb = row_buffer(a.b + (long long)j0 * a.ldb, 0x7ffffff0u);
  const unsigned va = (unsigned)min(l15, (int)a.m - 1) * (unsigned)a.lda + lk, vb = (unsigned)min(l15, a.n - 1 - j0) * (unsigned)a.ldb + lk;
  i32x4 acc = {0, 0, 0, 0};
  for (int k0 = wave * 128; k0 < a.k; k0 += kFewAhead * kFewTurn) {
    FewOperand fa, fb;
    few_request(bb, vb, k0, lk, a.k, fb);
    few_request(ab, va, k0, lk, a.k, fa);
    if ((a.k & 15) && k0 + (kFewAhead - 1) * kFewTurn + 128 > a.k - 16) {   // this wave may hold the group that k ends in: a's bytes past it
#pragma unroll
      for (int u = 0; u < kFewAhead; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int ends = a.k - (k0 + u * kFewTurn + h * 64 + lk);
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const int keep = min(max(ends - 4 * d, 0), 4);
            fa[u][h][d] &= keep == 4 ? -1 : (1 << (8 * keep)) - 1;
          }
        }
    }
    few_products(fa, fb, acc);
  }
  few_finish<T>(a, sums, acc, j0, lane, wave, [&](int i) { return a.a_scale[i]; });
}

// The same for up to ROWS rows that are quantised here (behind their layer norm, if there is one): every block forms them for itself while its first loads of b are
// in flight, which costs less than a launch in front.  A row is two halves of the block's work at a time: 256 threads with NV packs, as in
// quantize_rows.
template <typename T, int ROWS, int NV>
__global__ __launch_bounds__(kFewWaves * 64) void int8_few_linear(Int8Args a, QuantizeArgs q) {
  constexpr int V = 16 / sizeof(T), NT = 256, TURNS = (ROWS + 1) / 2, PITCH = NT * NV * V + 16;
  __shared__ int sums[kFewWaves][4][64];
  __shared__ __attribute__((aligned(16))) unsigned char rows[ROWS][PITCH];
  __shared__ double red[2][TURNS][centre_lds(NT)];
  __shared__ float red_max[2][TURNS][NT / 64], scales[ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l15 = lane & 15, lk = (lane >> 4) * 16;
  const int j0 = blockIdx.x * 16;
  const __amdgpu_buffer_rsrc_t bb = row_buffer(a.b + (long long)j0 * a.ldb, 0x7ffffff0u);
  const unsigned vb = (unsigned)min(l15, a.n - 1 - j0) * (unsigned)a.ldb + lk;
  i32x4 acc = {0, 0, 0, 0};
  FewOperand fa, fb;

  // the rows and the norm's parameters before b: loads arrive in order, and they are what the next lines wait for
  const int t = threadIdx.x & (NT - 1), side = wave >> 2;
  Parameter<float, NT, NV, V, false> gamma, beta;
  if (q.norm) {
    gamma.load(q.gamma, a.k, t);
    beta.load(q.beta, a.k, t);
  }
  float v[TURNS][NV][V], mean[TURNS], rstd[TURNS];
  auto load = [&](int n) {
    const long long r = min((long long)(2 * n + side), a.m - 1);
    const __amdgpu_buffer_rsrc_t xb = row_buffer((const T*)q.x + r * q.ldx, (unsigned)a.k * sizeof(T));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Pack<T, V> k = buffer_load<T, V>(xb, (i * NT + t) * V * sizeof(T));
#pragma unroll
      for (int j = 0; j < V; ++j) v[n][i][j] = (float)k.e[j];
    }
  };
#pragma unroll
  for (int n = 0; n < TURNS; ++n) load(n);
  few_request(bb, vb, wave * 128, lk, a.k, fb);
  __builtin_amdgcn_sched_barrier(0);
  if (q.norm) {
    bool over[TURNS], any_over = false;   // this side's rows whose sums ran over; any row of the block
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      over[n] = centre_row<NT, NV, V, false>(v[n], a.k, t, q.eps, red[side][n], mean[n], rstd[n]);
      double other = red[side ^ 1][n][NT / 64];   // the other side's sum, as its threads formed it
#pragma unroll
      for (int w = 1; w < NT / 64; ++w) other += red[side ^ 1][n][NT / 64 + w];
      any_over |= over[n] | !finite(other);
    }
    if (may_run_over<T> && __builtin_expect(any_over, 0)) {   // (both sides come by its barriers)
#pragma unroll
      for (int n = 0; n < TURNS; ++n) load(n);
      __syncthreads();
#pragma unroll
      for (int n = 0; n < TURNS; ++n) centre_row_again<NT, NV, V, false>(v[n], a.k, t, q.eps, red[side][n], over[n], mean[n], rstd[n]);
    }
  }
#pragma unroll
  for (int n = 0; n < TURNS; ++n) {
    if (q.norm)
      each_pack<NT, NV, V>(a.k, t, [&](int i, int) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[n][i][j] = rounded_mul(v[n][i][j], rstd[n]);
          if (q.gamma) v[n][i][j] = rounded_mul(v[n][i][j], gamma.k[i].e[j]);
          if (q.beta) v[n][i][j] += beta.k[i].e[j];
        }
      });
    float m = 0.f;
    each_pack<NT, NV, V>(a.k, t, [&](int i, int) {
#pragma unroll
      for (int j = 0; j < V; ++j) m = max_nan(m, fabsf(v[n][i][j]));
    });
    m = team_max<NT>(m, red_max[side][n]);
    const double inv = quantize_factor(m);
    const bool fine = quantizable(m);
    const int r = 2 * n + side;
    if (r < ROWS) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * NT + t) * V;
        Pack<unsigned char, V> k;
#pragma unroll
        for (int j = 0; j < V; ++j) k.e[j] = (unsigned char)(fine && c < a.k ? quantize1(v[n][i][j], inv) : 0u);
        *reinterpret_cast<Pack<unsigned char, V>*>(&rows[r][c]) = k;
      }
      if (t == 0) scales[r] = quantize_scale(m);
    }
  }
  __syncthreads();
  const unsigned char* mine = rows[min(l15, ROWS - 1)];
  for (int k0 = wave * 128; k0 < a.k; k0 += kFewAhead * kFewTurn) {
    if (k0 != wave * 128) few_request(bb, vb, k0, lk, a.k, fb);
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + u * kFewTurn + h * 64 + lk;
        fa[u][h] = *reinterpret_cast<const i32x4*>(mine + (k < a.k ? k : 0));   // (past k: anything, b's are zeros)
      }
    few_products(fa, fb, acc);
  }
  few_finish<T>(a, sums, acc, j0, lane, wave, [&](int i) { return scales[i]; });
}

// ---- short rows -------------------------------------------------------------------------------------------------------------------
// Rows of up to 32 KS values, quantised in the registers of the waves that multiply them: a wave takes 32 rows and up to 128 columns, lane l the groups of 16
// consecutive k of row l & 31 that the products take from it, so that x is read once from memory (by other columns' blocks from the caches) and no
// quantised copy is written.  Bound by the bytes of x and of the output: 65536 x 64 f32 by 128 columns 10.6 us, 4.7 TB/s.
template <typename T, int KS>
__global__ __launch_bounds__(256) void int8_short_linear(Int8Args a, QuantizeArgs q) {
  constexpr int V = 16 / sizeof(T), P = 16 / V, NY = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l31 = lane & 31, lh = lane >> 5;
  const long long i0 = (long long)blockIdx.x * 128 + wave * 32;
  if (i0 >= a.m) return;
  const int j0 = blockIdx.y * 32 * NY, rows = (int)min(32ll, a.m - i0), cols = min(32 * NY, a.n - j0);
  const __amdgpu_buffer_rsrc_t xb = row_buffer((const T*)q.x + i0 * q.ldx, 0x7ffffff0u), bb = row_buffer(a.b + (long long)j0 * a.ldb, 0x7ffffff0u);
  const unsigned xrow = (unsigned)min(l31, rows - 1) * (unsigned)(q.ldx * sizeof(T));
  Pack<T, V> x[KS][P];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int k = s * 32 + lh * 16 + p * V;
      x[s][p] = buffer_load<T, V>(xb, k < a.k ? xrow + k * sizeof(T) : 0x80000000u);   // (past k: zeros)
    }
  i32x4 fb[NY][KS];
  float sb[NY], bias[NY];
#pragma unroll
  for (int y = 0; y < NY; ++y) {
    const int j = min(y * 32 + l31, cols - 1);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int k = s * 32 + lh * 16;
      fb[y][s] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(bb, k < a.k ? (unsigned)j * (unsigned)a.ldb + k : 0x80000000u, 0, 0));
    }
    sb[y] = a.b_scale[j0 + j];
    bias[y] = a.bias ? a.bias[j0 + j] : 0.f;
  }
  __builtin_amdgcn_sched_barrier(0);
  float m = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int j = 0; j < V; ++j) m = max_nan(m, fabsf((float)x[s][p].e[j]));
  m = max_nan(m, __shfl_xor(m, 32));
  const double inv = quantize_factor(m);
  const bool fine = quantizable(m);
  i32x4 fa[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      unsigned four = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) four |= quantize1((float)x[s][(d * 4 + j) / V].e[(d * 4 + j) % V], inv) << (8 * j);
      fa[s][d] = fine ? (int)four : 0;
    }
  const float mine = quantize_scale(m);
  float sa[16];   // of the rows of this lane's results: 8 (v / 4) + 4 (l >> 5) + v % 4, column l & 31
#pragma unroll
  for (int v = 0; v < 16; ++v) sa[v] = __shfl(mine, (v >> 2) * 8 + lh * 4 + (v & 3));
  // (a row or column past the end has an offset past the buffer's: its store is dropped)
  const __amdgpu_buffer_rsrc_t ob = row_buffer((T*)a.out + i0 * a.ldo + j0, 0x7ffffff0u);
#pragma unroll
  for (int y = 0; y < NY; ++y) {
    i32x16 acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[s], fb[y][s], acc, 0, 0, 0);
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int i = (v >> 2) * 8 + lh * 4 + (v & 3), j = y * 32 + l31;
      const float o[1] = {int8_result(acc[v], sa[v], sb[y], bias[y])};
      buffer_store<T, 1>(ob, i < rows && j < cols ? (unsigned)(i * (int)a.ldo + j) * (unsigned)sizeof(T) : 0x80000000u, o);
    }
  }
}

template <int I>
using N = std::integral_constant<int, I>;
constexpr int kCUs = 256;

void launch_int8_matmul(const Int8Args& given, int out_type, hipStream_t s) {
  Int8Args a = given;
  if (a.m == 0 || a.n == 0) return;
  if (a.m == 1) a.lda = (a.k + 15) & ~15;   // (a single row's distance to the next says nothing)
  if (a.n == 1) a.ldb = (a.k + 15) & ~15;
  const int al_a = ((uintptr_t)a.a | (uintptr_t)a.lda) % 16 == 0, al_b = ((uintptr_t)a.b | (uintptr_t)a.ldb) % 16 == 0;
  auto grid = [&](int bm, int bn, int& tm, int& tn) {
    const long long m = (a.m + bm - 1) / bm, n = (a.n + bn - 1) / bn;
    EG_CHECK(m * n < (1ll << 22), "int8 product: too many outputs (%lld x %d)", a.m, a.n);
    tm = (int)m;
    tn = (int)n;
    return dim3((unsigned)(m * n));
  };
  by_type(out_type, [&](auto t) {
    using T = decltype(t);
    int tm, tn;
    if (al_a && al_b && a.lda <= 1 << 22 && a.ldb <= 1 << 22 && a.ldo <= 1 << 20 && a.k >= 16) {
      // Up to 16 rows: 16 columns a block while that is at most one block a CU (n = k = 4096: 5.8 us for 16 rows, 4.4 for one, with tiles 6.3; n = 8192, k = 1024:
      // 5.1 against 3.7).
      if (a.m <= 16 && a.n <= 16 * kCUs) return row_launch(int8_few<T>, dim3((a.n + 15) / 16), dim3(kFewWaves * 64), s, a);
      // The smallest tiles that are at most one a CU; no larger ones than the rows or columns fill.  us, of the same product with each tile:
      //   m x n x k           32x64  64x64  64x128  128x128  256x128  256x256
      //   64 x 4096 x 4096      6.5    8.1    11.9     18        -        -
      //   256 x 4096 x 4096      13     11    12.8     18        -        -
      //   512 x 4096 x 4096      23     20    15.7     20        -        -
      //   1024 x 4096 x 4096     41     38    27.6     23        -       25
      //   2048 x 4096 x 4096     77     72      51     45       42       53
      //   4096 x 4096 x 4096    148    140     103     88       81       69
      //   65536 x 128 x 1024      -      -      21      -     17.5       23
      auto few_enough = [&](int bm, int bn) { return ((a.m + bm - 1) / bm) * ((a.n + bn - 1) / bn) <= kCUs; };
      auto tiles = [&](auto bm, auto bn, auto wm, auto wn, auto ks, auto ring) {
        constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value, KS = decltype(ks)::value;
        const dim3 g = grid(BM, BN, tm, tn);
        row_launch(int8_tiles<T, BM, BN, WM, WN, KS, decltype(ring)::value>, g, dim3(KS * WM * WN * 64), s, a, tn);
      };
      if (a.m <= 32 || few_enough(32, 64)) tiles(N<32>(), N<64>(), N<1>(), N<2>(), N<4>(), N<3>());
      else if (few_enough(64, 64)) tiles(N<64>(), N<64>(), N<2>(), N<2>(), N<4>(), N<3>());
      else if (a.m <= 64 || few_enough(64, 128)) tiles(N<64>(), N<128>(), N<2>(), N<2>(), N<2>(), N<3>());
      else if (a.m <= 128 || few_enough(128, 128)) tiles(N<128>(), N<128>(), N<2>(), N<2>(), N<2>(), N<3>());
      else if (a.n <= 128 || few_enough(256, 128)) tiles(N<256>(), N<128>(), N<4>(), N<2>(), N<1>(), N<4>());
      else tiles(N<256>(), N<256>(), N<2>(), N<4>(), N<1>(), N<4>());
      return;
    }
    const dim3 g = grid(64, 64, tm, tn);
    row_launch(int8_any<T>, g, dim3(256), s, a, tn, al_a, al_b);
  });
}

static long long few_rows(int type, int k) {   // rows that int8_few_linear takes
  const int packs = (k + 256 * (type == ROW_F32 ? 4 : 8) - 1) / (256 * (type == ROW_F32 ? 4 : 8));
  return packs <= 2 ? 4 : packs <= 4 ? 2 : 0;
}
static long long linear_pitch(int k) { return (k + 15) & ~15; }
size_t int8_linear_bytes(long long m, int k) { return ((size_t)m * linear_pitch(k) + 15) / 16 * 16 + (size_t)m * 4; }

// The forms that quantise and multiply in one launch, where x and the weights are aligned and x's type is the output's.
//   few rows (int8_few_linear): up to 32 columns for each CU, us against two launches: 1 x 4096 x 4096 4.5 / 7.6, 4 x 4096 x 4096 6.5 / 8.0, 4 x 8192 x 2048 7.4 / 8.3;
//   of 16384 columns 12.8 / 11.2
//   short rows (int8_short_linear): 65536 rows of 64 values by 128 columns, f32: 10.6 / 16.5; 256 by 256: 4.7 / 5.3; of 128 values 15.6 / 20.4, but 6.9 / 5.4 for
//   256 by 256 and 50 / 39 for 512 columns (every 128 columns quantise again)
enum LinearForm { TWO_LAUNCHES, FEW_ROWS, SHORT_ROWS };
static LinearForm linear_form(const QuantizeArgs& q, const Int8Args& a, int type, int out_type) {
  const int elem = type == ROW_F32 ? 4 : 2;
  if (type != out_type || (uintptr_t)q.x % 16 || (a.m > 1 && q.ldx * elem % 16) || a.k % (16 / elem) || (uintptr_t)q.gamma % 16 || (uintptr_t)q.beta % 16 || (uintptr_t)a.b % 16 ||
      (a.n > 1 && a.ldb % 16) || a.ldb > 1 << 22)
    return TWO_LAUNCHES;
  if (a.m <= few_rows(type, a.k) && a.n <= 32 * kCUs) return FEW_ROWS;
  const bool is_short = a.k <= 64 || (a.k <= 128 && a.n <= 128 && a.m >= 64 * kCUs);
  return !q.norm && is_short && q.ldx <= 1 << 20 && a.ldo <= 1 << 20 && a.n < 1 << 22 && a.m < 1 << 30 ? SHORT_ROWS : TWO_LAUNCHES;
}
bool int8_linear_in_one(const QuantizeArgs& q, const Int8Args& a, int type, int out_type) { return linear_form(q, a, type, out_type) != TWO_LAUNCHES; }

void launch_int8_linear(const QuantizeArgs& given, const Int8Args& product, int type, int out_type, void* workspace, hipStream_t s) {
  QuantizeArgs q = given;
  Int8Args a = product;
  if (a.m == 0 || a.n == 0) return;
  const LinearForm form = linear_form(q, a, type, out_type);
  if (form != TWO_LAUNCHES) {
    by_type(type, [&](auto t) {
      using T = decltype(t);
      constexpr int V = 16 / sizeof(T);
      if (form == FEW_ROWS) {
        const dim3 grid((a.n + 15) / 16), block(kFewWaves * 64);
        if (a.m == 1 && a.k <= 256 * V * 2) row_launch(int8_few_linear<T, 1, 2>, grid, block, s, a, q);
        else if (a.m <= 2 && a.k > 256 * V * 2) row_launch(int8_few_linear<T, 2, 4>, grid, block, s, a, q);
        else row_launch(int8_few_linear<T, 4, 2>, grid, block, s, a, q);
      } else {
        const dim3 grid((unsigned)((a.m + 127) / 128), (a.n + 127) / 128), block(256);
        if (a.k <= 32) row_launch(int8_short_linear<T, 1>, grid, block, s, a, q);
        else if (a.k <= 64) row_launch(int8_short_linear<T, 2>, grid, block, s, a, q);
        else row_launch(int8_short_linear<T, 4>, grid, block, s, a, q);
      }
    });
    return;
  }
  q.q = (signed char*)workspace;
  q.ldq = linear_pitch(a.k);
  q.scale = (float*)((char*)workspace + ((size_t)a.m * q.ldq + 15) / 16 * 16);
  launch_quantize_rows(q, type, s);
  a.a = q.q;
  a.lda = q.ldq;
  a.a_scale = q.scale;
  launch_int8_matmul(a, out_type, s);
}

}  // namespace eg
