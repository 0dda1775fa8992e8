// Layer norm over rows: forward, gradient, tangent and its reverse; the row quantisation to 8 bits, with or without a layer
// norm in front.
//
//   xh = (x - m) r,  m = mean x,  r = (mean (x - m)^2 + eps)^-1/2,  y = act(xh gamma + beta)
//   gradient:  g = dy act'(xh gamma + beta),  dx = r (g gamma - mean(g gamma) - xh mean(g gamma xh)),
//              dgamma = sum over rows of g xh,  dbeta = sum over rows of g
//   quantised: q = the whole number nearest to 127 x / max |x| (a tie to the even one), scale = max |x| / 127
//
// All of it is bound by HBM, so a row is read once: it stays in the registers of the team of threads that owns it (8 to 64 lanes of a
// wave, 256 or 1,024 threads: row_team) between the statistics and the result.  A team of a wave needs no LDS and no barrier; a wider one joins its
// waves' sums through LDS.  The mean and the variance are summed in 64 bits, packs of a thread pairwise in 32: the
// mean decides every x - m, and the statistics hardly ever depend on the team.  A row of one value has xh = 0 exactly (its sums are exact; the rounded sum of a
// last pack of three is off by less than what rounding the mean of seven or more takes back).  Where a pack's sum runs over in 32 bits, the row is
// summed again in 64 (rows_that_ran_over).  The gradient's sums are in 32.  xh gamma + beta is formed by the same three rounded operations in the forward and the gradient (no
// contraction into an fma), so the gradient's sign of it is the forward's.
// Measured: forward 65,536 x 128 f32 12.9 - 15.1 us (up to 5.2 TB/s; a copy of these bytes 6.5), 8,192 x 4,096 bf16 25 us; gradient 16,384 x 4,096 bf16 79 + 5 us
// (4.8 TB/s with three tensors); quantisation 8,192 x 4,096 bf16 24 - 27 us (3.9 TB/s).  Rows that do not end with a pack: 1,023 x 5,001 f16 12.2 us, 5,000 8.6 (the cut
// pack's shift takes registers, 208 a thread, and its tail goes element by element).
#include <tuple>

#include "rowops_dev.h"

namespace eg {

// ---- rows in registers -------------------------------------------------------------------------------------------------------
template <typename T, typename W, int NT, int NV, int V, bool TAIL>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void ln_fwd(LayerNormArgs a) {
  constexpr int NB = NT > 256 ? NT : 256, TEAMS = NB / NT;
  __shared__ double red[2][centre_lds(NT)];
  const int t = TEAMS > 1 ? threadIdx.x % NT : threadIdx.x, team = TEAMS > 1 ? threadIdx.x / NT : 0;
  Parameter<W, NT, NV, V, TAIL> gamma, beta;
  auto parameters = [&] {
    gamma.load((const W*)a.gamma, a.cols, t);
    beta.load((const W*)a.beta, a.cols, t);
  };
  constexpr bool HELD = NT <= 64;   // over the rows; a wider team sees few rows and reads them again, from the caches
  if constexpr (HELD) parameters();
  auto finish = [&](long long row, float(&v)[NV][V], float mean, float rstd, bool store) {
    T* y = (T*)a.y + row * a.ldy;
    const int end = store ? a.cols : 0;
    by_act(a.act, [&](auto act) {
      each_pack<NT, NV, V>(end, t, [&](int i, int c) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = rounded_mul(v[i][j], rstd);
        if (a.gamma)
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] = rounded_mul(v[i][j], (float)gamma.k[i].e[j]);
        if (a.beta)
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] += (float)beta.k[i].e[j];
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = row_act<decltype(act)::value>(v[i][j]);
        store_row_pack<T, V, TAIL>(y, c, a.cols, v[i]);
      });
    });
    if (t == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  };
  int turn = 0;
  const long long step = (long long)gridDim.x * TEAMS, first = (long long)blockIdx.x * TEAMS + team;
  long long r = first;
  bool any_over = false;
  LoosePack<T, V> next[NV];
  if (r < a.rows) request_row<T, NT, NV, V>((const T*)a.x + r * a.ldx, a.cols, t, next);
  for (; r < a.rows; r += step, turn ^= 1) {
    float v[NV][V], mean, rstd;
    settle_row<T, NT, NV, V, TAIL>(a.cols, t, next);
    each_pack<NT, NV, V>(a.cols, t, [&](int i, int) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = (float)next[i].e[j];
    });
    if (r + step < a.rows) request_row<T, NT, NV, V>((const T*)a.x + (r + step) * a.ldx, a.cols, t, next);
    if constexpr (!HELD) parameters();
    const bool over = centre_row<NT, NV, V, TAIL>(v, a.cols, t, a.eps, red[turn], mean, rstd) && may_run_over<T>;
    any_over |= over;
    finish(r, v, mean, rstd, !over);   // (such a row is left: y may be x)
  }
  if (any_over) {
    if constexpr (!HELD) parameters();
    rows_that_ran_over<T, NT, NV, V, TAIL>((const T*)a.x, a.ldx, first, a.rows, step, a.cols, t, a.eps, red,
                                           [&](long long row, float(&v)[NV][V], float mean, float rstd) { finish(row, v, mean, rstd, true); });
  }
}

// A block's sums of the parameter gradients: put(column, sum of g xh, sum of g); several teams of a block add up in their order.
template <int NT, int NV, int V, int TEAMS, typename F>
__device__ __forceinline__ void block_sums(int cols, int t, int team, const float (&sx)[NV][V], const float (&sg)[NV][V], F put) {
  if constexpr (TEAMS > 1) {
    __shared__ float sum[2][NT * NV * V];
    for (int k = 0; k < TEAMS; ++k) {
      if (team == k)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int c = (i * NT + t) * V + j;
            sum[0][c] = (k ? sum[0][c] : 0.f) + sx[i][j];
            sum[1][c] = (k ? sum[1][c] : 0.f) + sg[i][j];
          }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += NT * TEAMS) put(c, sum[0][c], sum[1][c]);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * NT + t) * V;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < cols) put(c + j, sx[i][j], sg[i][j]);
    }
  }
}
// ... to the block's row of partial [blocks][2][cols]
template <int NT, int NV, int V, int TEAMS>
__device__ __forceinline__ void leave_partial(float* partial, int cols, int t, int team, const float (&sx)[NV][V], const float (&sg)[NV][V]) {
  float* out = partial + (size_t)blockIdx.x * 2 * cols;
  block_sums<NT, NV, V, TEAMS>(cols, t, team, sx, sg, [&](int c, float x, float g) {
    out[c] = x;
    out[cols + c] = g;
  });
}

template <typename T, typename W, int NT, int NV, int V, bool TAIL>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void ln_bwd(LayerNormGradArgs a) {
  constexpr int NB = NT > 256 ? NT : 256, TEAMS = NB / NT;
  __shared__ float red[2][NT > 64 ? 2 * NT / 64 : 1];
  const int t = TEAMS > 1 ? threadIdx.x % NT : threadIdx.x, team = TEAMS > 1 ? threadIdx.x / NT : 0;
  Parameter<W, NT, NV, V, TAIL> gamma;
  gamma.load((const W*)a.gamma, a.cols, t);
  float sx[NV][V], sg[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) sx[i][j] = sg[i][j] = 0.f;
  const float n = 1.f / a.cols;
  int turn = 0;
  const long long step = (long long)gridDim.x * TEAMS;
  long long r = (long long)blockIdx.x * TEAMS + team;
  LoosePack<T, V> next_x[NV], next_d[NV];
  float next_mean = 0.f, next_rstd = 0.f;
  auto request = [&](long long row) {
    request_row<T, NT, NV, V>((const T*)a.x + row * a.ldx, a.cols, t, next_x);
    request_row<T, NT, NV, V>((const T*)a.dy + row * a.lddy, a.cols, t, next_d);
    next_mean = a.mean[row];
    next_rstd = a.rstd[row];
  };
  auto all_packs = [&](auto f) {   // (those past the end too: d = 0 there, and a branch for each would part the loads from their use)
#pragma unroll
    for (int i = 0; i < NV; ++i) f(i);
  };
  if (r < a.rows) request(r);
  for (; r < a.rows; r += step, turn ^= 1) {
    float x[NV][V], d[NV][V];
    settle_row<T, NT, NV, V, TAIL>(a.cols, t, next_x);
    settle_row<T, NT, NV, V, TAIL>(a.cols, t, next_d);   // (d = 0 past the end: reaches no sum)
    const float mean = next_mean, rstd = next_rstd;
    all_packs([&](int i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[i][j] = rounded_mul((float)next_x[i].e[j] - mean, rstd);
        d[i][j] = (i * NT + t) * V < a.cols ? (float)next_d[i].e[j] : 0.f;
      }
    });
    if (r + step < a.rows) request(r + step);   // (in flight while this row is summed and stored)
    if (a.act != ACT_NONE) {
      Parameter<W, NT, NV, V, TAIL> beta;
      beta.load((const W*)a.beta, a.cols, t);
      all_packs([&](int i) {
        float z[V];
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = a.gamma ? rounded_mul(x[i][j], (float)gamma.k[i].e[j]) : x[i][j];
        if (a.beta)
#pragma unroll
          for (int j = 0; j < V; ++j) z[j] += (float)beta.k[i].e[j];
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] *= row_act_grad(z[j], a.act, a.at_zero);
      });
    }
    float s[2] = {0.f, 0.f};
    all_packs([&](int i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        sg[i][j] += d[i][j];
        sx[i][j] += d[i][j] * x[i][j];
        if (a.gamma) d[i][j] *= (float)gamma.k[i].e[j];
        s[0] += d[i][j];
        s[1] += d[i][j] * x[i][j];
      }
    });
    if (!a.dx) continue;
    team_sum<NT>(s, red[turn]);
    const float m0 = s[0] * n, m1 = s[1] * n;
    T* dx = (T*)a.dx + r * a.lddx;
    each_pack<NT, NV, V>(a.cols, t, [&](int i, int c) {
#pragma unroll
      for (int j = 0; j < V; ++j) d[i][j] = (d[i][j] - m0 - x[i][j] * m1) * rstd;
      if (a.acc_x) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + j < a.cols) d[i][j] += (float)dx[c + j];
      }
      store_row_pack<T, V, TAIL>(dx, c, a.cols, d[i]);
    });
  }
  if (a.partial) leave_partial<NT, NV, V, TEAMS>(a.partial, a.cols, t, team, sx, sg);
  else if (a.dgamma || a.dbeta)   // the only block
    block_sums<NT, NV, V, TEAMS>(a.cols, t, team, sx, sg, [&](int c, float x, float g) {
      W *dgamma = (W*)a.dgamma, *dbeta = (W*)a.dbeta;
      if (dgamma) dgamma[c] = (W)((a.acc_w & 1 ? (float)dgamma[c] : 0.f) + x);
      if (dbeta) dbeta[c] = (W)((a.acc_w & 2 ? (float)dbeta[c] : 0.f) + g);
    });
}

// partial [groups][2][cols] -> dgamma, dbeta: a block adds 32 of the 2 cols sums, 32 threads each every 32nd group
template <typename W>
__global__ __launch_bounds__(1024) void ln_bwd_finish(const float* partial, int groups, int cols, W* dgamma, W* dbeta, int acc) {
  __shared__ float red[16][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < 2 * cols) {
    const float* p = partial + i;
#pragma unroll 8
    for (int g = part; g < groups; g += 32) s += p[(size_t)g * 2 * cols];
  }
  s = lanes_sum<64, 32>(s);   // the wave's two groups
  if ((threadIdx.x & 32) == 0) red[threadIdx.x >> 6][lane] = s;
  __syncthreads();
  if (threadIdx.x >= 32 || i >= 2 * cols) return;
  W* out = i < cols ? dgamma : dbeta;
  if (!out) return;
  out += i < cols ? i : i - cols;
  s = acc & (i < cols ? 1 : 2) ? (float)*out : 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) s += red[k][lane];
  *out = (W)s;
}

// Bytes of a row to write: the whole row, and zeros up to the end of its last 16-byte group as far as ldq leaves room (a single row may come with any ldq,
// less than its length too).
__device__ __forceinline__ int quantized_width(const QuantizeArgs& a) { return max(a.cols, (int)min((long long)((a.cols + 15) & ~15), a.ldq)); }

template <typename T, int NT, int NV, int V, bool TAIL>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void quantize_rows(QuantizeArgs a) {
  constexpr int NB = NT > 256 ? NT : 256, TEAMS = NB / NT;
  __shared__ double red[2][centre_lds(NT)];
  __shared__ float red_max[2][NT > 64 ? NT / 64 : 1];
  const int t = TEAMS > 1 ? threadIdx.x % NT : threadIdx.x, team = TEAMS > 1 ? threadIdx.x / NT : 0;
  const int width = quantized_width(a);
  // a row without its mean, or as it is, to its 8-bit form
  auto finish = [&](long long r, float(&v)[NV][V], float rstd, float* red) {
    if (a.norm) {
      Parameter<float, NT, NV, V, TAIL> gamma, beta;
      gamma.load(a.gamma, a.cols, t);
      beta.load(a.beta, a.cols, t);
      each_pack<NT, NV, V>(a.cols, t, [&](int i, int) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[i][j] = rounded_mul(v[i][j], rstd);
          if (a.gamma) v[i][j] = rounded_mul(v[i][j], gamma.k[i].e[j]);
          if (a.beta) v[i][j] += beta.k[i].e[j];   // (zeros past the end)
        }
      });
    }
    float m = 0.f;
    each_pack<NT, NV, V>(a.cols, t, [&](int i, int) {
#pragma unroll
      for (int j = 0; j < V; ++j) m = max_nan(m, fabsf(v[i][j]));
    });
    m = team_max<NT>(m, red);
    const double inv = quantize_factor(m);
    const bool fine = quantizable(m);
    unsigned char* q = (unsigned char*)a.q + r * a.ldq;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * NT + t) * V;
      if (c >= width) continue;
      LoosePack<unsigned char, V> k;
#pragma unroll
      for (int j = 0; j < V; ++j) k.e[j] = (unsigned char)(fine && c < a.cols ? quantize1(v[i][j], inv) : 0u);   // (zeros past the end give 0)
      if (c + V <= width) *reinterpret_cast<LoosePack<unsigned char, V>*>(q + c) = k;
      else
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + j < width) q[c + j] = k.e[j];
    }
    if (t == 0) a.scale[r] = quantize_scale(m);
  };
  int turn = 0;
  const long long step = (long long)gridDim.x * TEAMS, first = (long long)blockIdx.x * TEAMS + team;
  bool any_over = false;
  for (long long r = first; r < a.rows; r += step, turn ^= 1) {
    LoosePack<T, V> k[NV];
    request_row<T, NT, NV, V>((const T*)a.x + r * a.ldx, a.cols, t, k);
    settle_row<T, NT, NV, V, TAIL>(a.cols, t, k);
    float v[NV][V], mean, rstd = 1.f;
    each_pack<NT, NV, V>(a.cols, t, [&](int i, int) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = (float)k[i].e[j];
    });
    if (a.norm) any_over |= centre_row<NT, NV, V, TAIL>(v, a.cols, t, a.eps, red[turn], mean, rstd);
    finish(r, v, rstd, red_max[turn]);
  }
  if (may_run_over<T> && any_over)
    rows_that_ran_over<T, NT, NV, V, TAIL>((const T*)a.x, a.ldx, first, a.rows, step, a.cols, t, a.eps, red,
                                           [&](long long row, float(&v)[NV][V], float, float rstd) { finish(row, v, rstd, red_max[0]); });
}

// ---- rows of any length: three passes by 256 threads, element by element -------------------------------------------------------
constexpr int kRowThreads = 256;
template <typename T>
__device__ __forceinline__ void row_statistics(const T* x, int cols, float eps, double* red, float& mean, float& rstd) {
  double s[1] = {0.};
  for (int c = threadIdx.x; c < cols; c += kRowThreads) s[0] += (double)(float)x[c];
  team_sum<kRowThreads>(s, red);
  mean = (float)(s[0] / cols);
  s[0] = 0.;
  for (int c = threadIdx.x; c < cols; c += kRowThreads) {
    const float u = (float)x[c] - mean;
    s[0] += (double)u * u;
  }
  team_sum<kRowThreads>(s, red + kRowThreads / 64);
  rstd = row_rstd(s[0] / cols, eps);
}

template <typename T, typename W>
__global__ __launch_bounds__(kRowThreads) void ln_fwd_rows(LayerNormArgs a) {
  __shared__ double red[2 * kRowThreads / 64];
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = (const T*)a.x + r * a.ldx;
    T* y = (T*)a.y + r * a.ldy;
    float mean, rstd;
    row_statistics<T>(x, a.cols, a.eps, red, mean, rstd);
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads)
      {
      const float z = affine(rounded_mul((float)x[c] - mean, rstd), (const W*)a.gamma, (const W*)a.beta, c);
      by_act(a.act, [&](auto act) { y[c] = (T)row_act<decltype(act)::value>(z); });
    }
    if (threadIdx.x == 0 && a.mean) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
    __syncthreads();
  }
}

// g = dy act'(z) and xh of one element
template <typename T, typename W>
__device__ __forceinline__ void grad_terms(const LayerNormGradArgs& a, const T* x, const T* dy, float mean, float rstd, int c, float& g, float& xh) {
  xh = rounded_mul((float)x[c] - mean, rstd);
  g = (float)dy[c];
  if (a.act != ACT_NONE) g *= row_act_grad(affine(xh, (const W*)a.gamma, (const W*)a.beta, c), a.act, a.at_zero);
}

template <typename T, typename W>
__global__ __launch_bounds__(kRowThreads) void ln_bwd_rows(LayerNormGradArgs a) {
  __shared__ float red[2 * kRowThreads / 64];
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *x = (const T*)a.x + r * a.ldx, *dy = (const T*)a.dy + r * a.lddy;
    T* dx = (T*)a.dx + r * a.lddx;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
      float g, xh;
      grad_terms<T, W>(a, x, dy, mean, rstd, c, g, xh);
      if (a.gamma) g *= (float)((const W*)a.gamma)[c];
      s[0] += g;
      s[1] += g * xh;
    }
    team_sum<kRowThreads>(s, red);
    const float m0 = s[0] / a.cols, m1 = s[1] / a.cols;
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
      float g, xh;
      grad_terms<T, W>(a, x, dy, mean, rstd, c, g, xh);
      if (a.gamma) g *= (float)((const W*)a.gamma)[c];
      float v = (g - m0 - xh * m1) * rstd;
      if (a.acc_x) v += (float)dx[c];
      dx[c] = (T)v;
    }
    __syncthreads();
  }
}

// The parameter gradients: a block takes 64 columns and a share of the rows, four of them at a time.
constexpr int kPartBlocks = 64;   // row groups
template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_bwd_columns(LayerNormGradArgs a) {
  __shared__ float red[2][4][64];
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float sg = 0.f, sx = 0.f;
  if (c < a.cols)
    for (long long r = blockIdx.y * 4 + part; r < a.rows; r += gridDim.y * 4) {
      float g, xh;
      grad_terms<T, W>(a, (const T*)a.x + r * a.ldx, (const T*)a.dy + r * a.lddy, a.mean[r], a.rstd[r], c, g, xh);
      sg += g;
      sx += g * xh;
    }
  red[0][part][lane] = sx;
  red[1][part][lane] = sg;
  __syncthreads();
  if (part < 2 && c < a.cols)
    a.partial[((size_t)blockIdx.y * 2 + part) * a.cols + c] = red[part][0][lane] + red[part][1][lane] + red[part][2][lane] + red[part][3][lane];
}
static dim3 row_grid(long long rows) { return dim3((unsigned)std::min<long long>(rows, 1 << 20)); }
static int part_groups(long long rows) { return (int)std::min<long long>(kPartBlocks, (rows + 3) / 4); }

// Calls f(threads of a row, packs of a thread, elements of a pack, whether the last pack may be cut) for the smallest team whose registers hold a row of `cols`;
// false: none does. A thread keeps at most WAVE elements where the team is a wave or less, BLOCK of 256 threads, 16 of 1,024 (which have 128 registers a thread).
// The smallest team has the fewest joins and the most rows in flight; too small a one has too few waves on a CU or runs out of registers. us, with at
// most 16 / 32 elements a thread, rows x columns: forward bf16 8192 x 2048 (256 threads or a wave) 21.4 / 16.6, 4096 x 8192 (1,024 or 256) 55 / 30.4, f32 4096 x 6000
// 45 / 34.6, but 64 x 6000 4.0 / 4.6; quantisation of the same 16.0 / 12.8, 40.8 / 21.7, 37 / 28.7, 3.6 / 4.2.  Gradient: bf16 8192 x 2048 29.2 / 35.7, so 16 in a wave;
// 4096 x 8192 124 / 59.5, so 32 in a block of 256; f32 4096 x 6000 64.0 / 64.6, 64 x 6000 10.4 / 11.0, so 16 there.  With at most 8, bf16 8192 x 4096
// takes 97 (forward) and 148 (gradient), against 26 and 45.  The gradient spills with 1,024 threads (40 to 100 registers a thread, in every type; its tangent's reverse 63
// to 71): bf16 2,048 x 10,000 72 us, 2,048 x 16,384 104, for 123 and 201 MB.  512 threads lie between and have not been tried.
template <typename T, int WAVE, int BLOCK, typename F>
static bool row_team(int cols, F f) {
  constexpr int V = 16 / sizeof(T);
  using std::integral_constant;
  auto pick = [&](auto tail) {
#define EG_TEAM(NT, NV) \
  if constexpr ((NV) * V <= ((NT) > 256 ? 16 : (NT) == 256 ? BLOCK : WAVE)) \
    if (cols <= (NT) * (NV) * V) return f(integral_constant<int, NT>{}, integral_constant<int, NV>{}, integral_constant<int, V>{}, tail), true;
    EG_TEAM(8, 1) EG_TEAM(16, 1) EG_TEAM(32, 1) EG_TEAM(64, 1) EG_TEAM(64, 2) EG_TEAM(64, 4) EG_TEAM(256, 2) EG_TEAM(256, 4) EG_TEAM(256, 8) EG_TEAM(1024, 2) EG_TEAM(1024, 4)
#undef EG_TEAM
    return false;
  };
  if (cols < V) return f(integral_constant<int, 8>{}, integral_constant<int, 1>{}, integral_constant<int, 1>{}, std::false_type{}), true;   // (shorter than a pack)
  return cols % V ? pick(std::true_type{}) : pick(std::false_type{});
}
static dim3 team_grid(long long rows, int nt, int most) {
  const int teams = nt > 256 ? 1 : 256 / nt;
  return dim3((unsigned)std::min<long long>((rows + teams - 1) / teams, most));
}
static dim3 team_block(int nt) { return dim3(nt > 256 ? nt : 256); }

// Blocks of the gradient: each leaves one row of partial parameter gradients.  With a row ahead in flight, 16,384 x 4,096 bf16 (a row a block): 512
// blocks 80 + 5 us (gradient + join), 256 83 + 5, 1,024 98 + 7; 65,536 x 128 f32 (8 rows a block): 1,024 blocks 19 + 5 us, 512 22 + 4, 256 31 + 4.
constexpr int kGradBlocks = 1024;   // half of them where the block is one row's team
static dim3 gradient_grid(long long rows, int nt) { return team_grid(rows, nt, nt > 64 ? kGradBlocks / 2 : kGradBlocks); }
// f(team) for the gradient's form of rows of type T in registers
template <typename T, typename F>
static bool gradient_team(int cols, F f) { return row_team<T, 16, sizeof(T) == 2 ? 32 : 16>(cols, f); }
// Blocks that leave a row of partial sums
template <typename T>
static int gradient_groups(long long rows, int cols) {
  int groups = 0;
  if (!gradient_team<T>(cols, [&](auto nt, auto, auto, auto) { groups = (int)gradient_grid(rows, nt).x; })) groups = part_groups(rows);
  return groups;
}
// (enough for rows of any type)
size_t layer_norm_partial_floats(long long rows, int cols) {
  if (rows == 0 || cols == 0) return 0;
  return (size_t)std::max(gradient_groups<float>(rows, cols), gradient_groups<bf16_t>(rows, cols)) * 2 * cols;
}

// Few rows by one block, which then has the whole sums: no second launch, no workspace. 4 rows for each of its teams (as many teams as f32 rows have), 2 where
// the block is one team.  us of a call / of its kernels, against two launches: 16 x 1000 bf16 11.6 / 6.7 (15.7 / 6.0), 32 x 128 11.3 / 5.1 (15.6 / 6.5), 2 x 4096 11.1 / 9.0
// (15.6 / 8.6); with 8 rows a team 32 x 1000 11.4 / 9.7 (15.7 / 6.0), and 4 x 12000, in 1,024 threads, 26.5 / 26.9 (21.0 / 21.2).
bool layer_norm_gradient_in_one(long long rows, int cols) {
  return rows > 0 && rows <= (cols <= 32 ? 128 : cols <= 64 ? 64 : cols <= 128 ? 32 : cols <= 1024 ? 16 : cols <= 8192 ? 2 : 0);
}

void launch_layer_norm(const LayerNormArgs& a, int type, int wtype, hipStream_t s) {
  if (a.rows == 0 || a.cols == 0) return;
  by_type(type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto w) {
      using W = decltype(w);
      if (!row_team<T, 32, 32>(a.cols, [&](auto nt, auto nv, auto v, auto tail) {
            row_launch(ln_fwd<T, W, nt, nv, v, tail>, team_grid(a.rows, nt, 8192), team_block(nt), s, a);
          }))
        row_launch(ln_fwd_rows<T, W>, row_grid(a.rows), dim3(kRowThreads), s, a);
    };
    if (wtype == type) go(t);
    else go(float{});
  });
}

void launch_layer_norm_backward(const LayerNormGradArgs& given, int type, int wtype, hipStream_t s) {
  LayerNormGradArgs a = given;
  if (a.cols == 0) return;
  const bool params = a.dgamma || a.dbeta, one = layer_norm_gradient_in_one(a.rows, a.cols);
  if (!params || one) a.partial = nullptr;
  by_type(type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto w) {
      using W = decltype(w);
      int groups = 0;
      if (a.rows) {
        groups = gradient_groups<T>(a.rows, a.cols);
        const bool held = gradient_team<T>(a.cols, [&](auto nt, auto nv, auto v, auto tail) {
          const dim3 grid = params && one ? dim3(1) : gradient_grid(a.rows, nt);
          row_launch(ln_bwd<T, W, nt, nv, v, tail>, grid, team_block(nt), s, a);
        });
        if (!held) {
          if (params) row_launch(ln_bwd_columns<T, W>, dim3((a.cols + 63) / 64, groups), dim3(256), s, a);   // (first: dx may be dy)
          if (a.dx) row_launch(ln_bwd_rows<T, W>, row_grid(a.rows), dim3(kRowThreads), s, a);
        }
      }
      if (params && !one)
        row_launch(ln_bwd_finish<W>, dim3((2 * a.cols + 31) / 32), dim3(1024), s, a.partial, groups, a.cols, (W*)a.dgamma, (W*)a.dbeta, a.acc_w);
    };
    if (wtype == type) go(t);
    else go(float{});
  });
}

// ---- tangent ---------------------------------------------------------------------------------------------------------------
// P = r (I - 1 1^T / C - xh xh^T / C) is the (symmetric) Jacobian of xh.  Forward: ty = act' gamma P t.  Reverse with u = d/d(ty),
// k = act' gamma u:  d/dt = P k,  dgamma = sum of act' u P t, and through P's own dependence on x
//   d/dx = -r^2 (q - W b) xh - r (b P k + W P t),   b = mean(t xh), W = mean(k xh), q = mean(k (t - mean t))
// (from <k, P t> = C r (q - W b) and dr = -r^2 mean(xh dx), d xh = P dx).
// f32 rows without gaps, in registers like the others; gamma and beta are there.
template <int NT, int NV, int V, bool TAIL>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void ln_tangent(LayerNormTangentArgs a) {
  constexpr int NB = NT > 256 ? NT : 256, TEAMS = NB / NT;
  __shared__ float red[2][NT > 64 ? 2 * NT / 64 : 1];
  const int t = TEAMS > 1 ? threadIdx.x % NT : threadIdx.x, team = TEAMS > 1 ? threadIdx.x / NT : 0;
  const float n = 1.f / a.cols;
  int turn = 0;
  for (long long r = (long long)blockIdx.x * TEAMS + team; r < a.rows; r += (long long)gridDim.x * TEAMS, turn ^= 1) {
    const size_t o = (size_t)r * a.cols;
    float x[NV][V], v[NV][V], g[NV][V], b[NV][V];
    load_row<float, NT, NV, V, TAIL>(a.x + o, a.cols, t, x);
    load_row<float, NT, NV, V, TAIL>(a.tx + o, a.cols, t, v);
    load_row<float, NT, NV, V, TAIL>(a.gamma, a.cols, t, g);
    load_row<float, NT, NV, V, TAIL>(a.beta, a.cols, t, b);
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {   // (past the end v = 0)
        x[i][j] = rounded_mul(x[i][j] - mean, rstd);
        s[0] += v[i][j];
        s[1] += v[i][j] * x[i][j];
      }
    team_sum<NT>(s, red[turn]);
    const float mt = s[0] * n, bt = s[1] * n;
    each_pack<NT, NV, V>(a.cols, t, [&](int i, int c) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        v[i][j] = row_act_grad(rounded_mul(x[i][j], g[i][j]) + b[i][j], a.act, kEngineLreluAtZero) * g[i][j] * (rstd * (v[i][j] - mt - x[i][j] * bt));
      store_row_pack<float, V, TAIL>(a.ty + o, c, a.cols, v[i]);
    });
  }
}
template <int NT, int NV, int V, bool TAIL>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void ln_tangent_bwd(LayerNormTangentArgs a) {
  constexpr int NB = NT > 256 ? NT : 256, TEAMS = NB / NT;
  __shared__ float red[2][NT > 64 ? 5 * NT / 64 : 1];
  const int t = TEAMS > 1 ? threadIdx.x % NT : threadIdx.x, team = TEAMS > 1 ? threadIdx.x / NT : 0;
  const float n = 1.f / a.cols;
  float sx[NV][V], sg[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) sx[i][j] = sg[i][j] = 0.f;
  int turn = 0;
  for (long long r = (long long)blockIdx.x * TEAMS + team; r < a.rows; r += (long long)gridDim.x * TEAMS, turn ^= 1) {
    const size_t o = (size_t)r * a.cols;
    float x[NV][V], v[NV][V], k[NV][V], g[NV][V], b[NV][V];
    load_row<float, NT, NV, V, TAIL>(a.x + o, a.cols, t, x);
    load_row<float, NT, NV, V, TAIL>(a.tx + o, a.cols, t, v);
    load_row<float, NT, NV, V, TAIL>(a.dty + o, a.cols, t, k);
    load_row<float, NT, NV, V, TAIL>(a.gamma, a.cols, t, g);
    load_row<float, NT, NV, V, TAIL>(a.beta, a.cols, t, b);
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {   // (past the end v = k = 0)
        x[i][j] = rounded_mul(x[i][j] - mean, rstd);
        k[i][j] *= row_act_grad(rounded_mul(x[i][j], g[i][j]) + b[i][j], a.act, kEngineLreluAtZero);
        b[i][j] = k[i][j];            // act' dty: dgamma's
        k[i][j] *= g[i][j];
        s[0] += v[i][j];
        s[1] += v[i][j] * x[i][j];
        s[2] += k[i][j];
        s[3] += k[i][j] * x[i][j];
        s[4] += k[i][j] * v[i][j];
      }
    team_sum<NT>(s, red[turn]);
    const float mt = s[0] * n, bt = s[1] * n, mk = s[2] * n, w = s[3] * n, q = s[4] * n - mk * mt;
    each_pack<NT, NV, V>(a.cols, t, [&](int i, int c) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float pk = rstd * (k[i][j] - mk - x[i][j] * w), pt = rstd * (v[i][j] - mt - x[i][j] * bt);
        sx[i][j] += b[i][j] * pt;
        k[i][j] = pk;
        v[i][j] = -rstd * (rstd * (q - w * bt) * x[i][j] + bt * pk + w * pt);
      }
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < a.cols) {
          if (a.acc_t) k[i][j] += a.dtx[o + c + j];
          if (a.acc_x) v[i][j] += a.dx[o + c + j];
        }
      store_row_pack<float, V, TAIL>(a.dtx + o, c, a.cols, k[i]);
      store_row_pack<float, V, TAIL>(a.dx + o, c, a.cols, v[i]);
    });
  }
  if (a.dgamma) leave_partial<NT, NV, V, TEAMS>(a.partial, a.cols, t, team, sx, sg);
}

void launch_layer_norm_tangent(const LayerNormTangentArgs& a, hipStream_t s) {
  if (!a.rows || !a.cols) return;
  const bool held = gradient_team<float>(a.cols, [&](auto nt, auto nv, auto v, auto tail) {
    row_launch(ln_tangent<nt, nv, v, tail>, team_grid(a.rows, nt, 8192), team_block(nt), s, a);
  });
  EG_CHECK(held, "layer norm tangent: %d channels", a.cols);
}
void launch_layer_norm_tangent_backward(const LayerNormTangentArgs& a, hipStream_t s) {
  if (!a.rows || !a.cols) return;
  const bool held = gradient_team<float>(a.cols, [&](auto nt, auto nv, auto v, auto tail) {
    const dim3 grid = gradient_grid(a.rows, nt);
    row_launch(ln_tangent_bwd<nt, nv, v, tail>, grid, team_block(nt), s, a);
    if (a.dgamma)
      row_launch(ln_bwd_finish<float>, dim3((2 * a.cols + 31) / 32), dim3(1024), s, a.partial, (int)grid.x, a.cols, a.dgamma, (float*)nullptr, a.acc_w);
  });
  EG_CHECK(held, "layer norm tangent: %d channels", a.cols);
}

// ---- quantisation of rows of any length -----------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kRowThreads) void quantize_kernel(QuantizeArgs a) {
  __shared__ double red[2 * kRowThreads / 64];
  __shared__ float red_max[kRowThreads / 64];
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = (const T*)a.x + r * a.ldx;
    unsigned char* q = (unsigned char*)a.q + r * a.ldq;
    float mean = 0.f, rstd = 1.f;
    if (a.norm) row_statistics<T>(x, a.cols, a.eps, red, mean, rstd);
    auto value = [&](int c) {
      float v = (float)x[c];
      if (a.norm) v = affine(rounded_mul(v - mean, rstd), a.gamma, a.beta, c);
      return v;
    };
    float m = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
      const float v = fabsf(value(c));
      m = max_nan(m, v);
    }
    m = team_max<kRowThreads>(m, red_max);
    const bool fine = quantizable(m);
    const double inv = quantize_factor(m);
    const int width = quantized_width(a);
    for (int c = threadIdx.x; c < width; c += kRowThreads) q[c] = (unsigned char)(fine && c < a.cols ? quantize1(value(c), inv) : 0u);
    if (threadIdx.x == 0) a.scale[r] = quantize_scale(m);
    __syncthreads();
  }
}

void launch_quantize_rows(const QuantizeArgs& a, int type, hipStream_t s) {
  if (!a.rows) return;
  by_type(type, [&](auto t) {
    using T = decltype(t);
    // (a row shorter than a pack: its team would not reach the end of its 16 bytes)
    if (a.cols < (int)(16 / sizeof(T)) || !row_team<T, 32, 32>(a.cols, [&](auto nt, auto nv, auto v, auto tail) {
          row_launch(quantize_rows<T, nt, nv, v, tail>, team_grid(a.rows, nt, 8192), team_block(nt), s, a);
        }))
      row_launch(quantize_kernel<T>, row_grid(a.rows), dim3(kRowThreads), s, a);
  });
}

}  // namespace eg
