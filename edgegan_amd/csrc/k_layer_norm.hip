// Layer norm over rows: forward, gradient, tangent and its reverse; the row quantisation to 8 bits, with or without a layer
// norm in front.  Bound by HBM: every pass below reads each row once from memory (further passes over a row hit the caches).
//
//   xh = (x - m) r,  m = mean x,  r = (mean (x - m)^2 + eps)^-1/2,  y = act(xh gamma + beta)
//   gradient:  g = dy act'(xh gamma + beta),  dx = r (g gamma - mean(g gamma) - xh mean(g gamma xh)),
//              dgamma = sum over rows of g xh,  dbeta = sum over rows of g
//   quantised: q = the whole number nearest to 127 x / max |x| (a tie to the even one), scale = max |x| / 127
//
// Sums are in 32 bits.  xh gamma + beta is formed by the same three rounded operations in the forward and the gradient (no
// contraction into an fma), so the gradient's sign of it is the forward's.
#include <tuple>

#include "rowops_dev.h"

namespace eg {

template <typename T>
__device__ __forceinline__ float ld1(const T* p) { return (float)*p; }

template <typename W>
__device__ __forceinline__ float affine(float xh, const W* gamma, const W* beta, int c) {
  const float z = gamma ? __fmul_rn(xh, (float)gamma[c]) : xh;
  return beta ? __fadd_rn(z, (float)beta[c]) : z;
}

// mean and 1 / sqrt(var + eps) of a row, by the whole block
template <typename T, int NT>
__device__ __forceinline__ void row_statistics(const T* x, int cols, float eps, float* red, float& mean, float& rstd) {
  float s[1] = {0.f};
  for (int c = threadIdx.x; c < cols; c += NT) s[0] += ld1(x + c);
  block_sum<NT>(s, red);
  const float m0 = s[0] / cols;
  __syncthreads();
  // the second pass also sums x - m0: what the first sum lost by rounding
  float d[2] = {0.f, 0.f};
  for (int c = threadIdx.x; c < cols; c += NT) {
    const float u = ld1(x + c) - m0;
    d[0] += u;
    d[1] += u * u;
  }
  block_sum<NT>(d, red);
  const float e = d[0] / cols;
  mean = m0 + e;
  rstd = 1.f / sqrtf(fmaxf(d[1] / cols - e * e, 0.f) + eps);
  if (d[1] != d[1]) rstd = d[1];   // (fmaxf drops a NaN)
  __syncthreads();
}

constexpr int kRowThreads = 256;

template <typename T, typename W>
__global__ __launch_bounds__(kRowThreads) void ln_fwd_rows(LayerNormArgs a) {
  __shared__ float red[2 * kRowThreads / 64];
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = (const T*)a.x + r * a.ldx;
    T* y = (T*)a.y + r * a.ldy;
    float mean, rstd;
    row_statistics<T, kRowThreads>(x, a.cols, a.eps, red, mean, rstd);
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads)
      y[c] = (T)row_act(affine(__fmul_rn(ld1(x + c) - mean, rstd), (const W*)a.gamma, (const W*)a.beta, c), a.act);
    if (threadIdx.x == 0 && a.mean) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
  }
}

// g = dy act'(z) and xh of one element
template <typename T, typename W>
__device__ __forceinline__ void grad_terms(const LayerNormGradArgs& a, const T* x, const T* dy, float mean, float rstd, int c, float& g, float& xh) {
  xh = __fmul_rn(ld1(x + c) - mean, rstd);
  g = ld1(dy + c);
  if (a.act != ACT_NONE) g *= row_act_grad(affine(xh, (const W*)a.gamma, (const W*)a.beta, c), a.act);
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
    block_sum<kRowThreads>(s, red);
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

// The parameter gradients: a block takes 64 columns and every kPartRows-th group of rows; four row lanes a block.
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
// partial [groups][2][cols] -> dgamma, dbeta
template <typename W>
__global__ __launch_bounds__(256) void ln_bwd_finish(const float* partial, int groups, int cols, W* dgamma, W* dbeta, int acc) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * cols) return;
  const int which = i / cols, c = i - which * cols;
  W* out = which ? dbeta : dgamma;
  if (!out) return;
  float s = 0.f;
  for (int p = 0; p < groups; ++p) s += partial[((size_t)p * 2 + which) * cols + c];
  if (acc) s += (float)out[c];
  out[c] = (W)s;
}

static dim3 row_grid(long long rows) { return dim3((unsigned)std::min<long long>(rows, 1 << 20)); }
static int part_groups(long long rows) { return (int)std::min<long long>(kPartBlocks, (rows + 3) / 4); }

size_t layer_norm_partial_floats(long long rows, int cols) { return (size_t)part_groups(rows) * 2 * cols; }

void launch_layer_norm(const LayerNormArgs& a, int type, int wtype, hipStream_t s) {
  if (a.rows == 0 || a.cols == 0) return;
  by_type(type, [&](auto t) {
    by_type(wtype, [&](auto w) { row_launch(ln_fwd_rows<decltype(t), decltype(w)>, row_grid(a.rows), dim3(kRowThreads), s, a); });
  });
}

void launch_layer_norm_backward(const LayerNormGradArgs& a, int type, int wtype, hipStream_t s) {
  if (a.cols == 0) return;
  by_type(type, [&](auto t) {
    by_type(wtype, [&](auto w) {
      using T = decltype(t);
      using W = decltype(w);
      auto rows = [&] { if (a.dx && a.rows) row_launch(ln_bwd_rows<T, W>, row_grid(a.rows), dim3(kRowThreads), s, a); };
      if (!a.dgamma && !a.dbeta) return rows();
      const int groups = part_groups(a.rows);
      if (groups) row_launch(ln_bwd_columns<T, W>, dim3((a.cols + 63) / 64, groups), dim3(256), s, a);
      row_launch(ln_bwd_finish<W>, dim3((2 * a.cols + 255) / 256), dim3(256), s, a.partial, groups, a.cols, (W*)a.dgamma, (W*)a.dbeta, a.acc_w);
      rows();   // (last: dx may be dy)
    });
  });
}

// ---- tangent ---------------------------------------------------------------------------------------------------------------
// P = r (I - 1 1^T / C - xh xh^T / C) is the (symmetric) Jacobian of xh.  Forward: ty = act' gamma P t.  Reverse with u = d/d(ty),
// k = act' gamma u:  d/dt = P k,  dgamma = sum of act' u P t, and through P's own dependence on x
//   d/dx = -r^2 (q - W b) xh - r (b P k + W P t),   b = mean(t xh), W = mean(k xh), q = mean(k (t - mean t))
// (from <k, P t> = C r (q - W b) and dr = -r^2 mean(xh dx), d xh = P dx).
__global__ __launch_bounds__(kRowThreads) void ln_tangent_rows(LayerNormTangentArgs a) {
  __shared__ float red[2 * kRowThreads / 64];
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const size_t o = (size_t)r * a.cols;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
      const float t = a.tx[o + c];
      s[0] += t;
      s[1] += t * __fmul_rn(a.x[o + c] - mean, rstd);
    }
    block_sum<kRowThreads>(s, red);
    const float mt = s[0] / a.cols, b = s[1] / a.cols;
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
      const float xh = __fmul_rn(a.x[o + c] - mean, rstd);
      const float d = row_act_grad(affine(xh, a.gamma, a.beta, c), a.act);
      a.ty[o + c] = d * a.gamma[c] * (rstd * (a.tx[o + c] - mt - xh * b));
    }
    __syncthreads();
  }
}
__global__ __launch_bounds__(kRowThreads) void ln_tangent_bwd_rows(LayerNormTangentArgs a) {
  __shared__ float red[5 * kRowThreads / 64];
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const size_t o = (size_t)r * a.cols;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
      const float xh = __fmul_rn(a.x[o + c] - mean, rstd), t = a.tx[o + c];
      const float k = row_act_grad(affine(xh, a.gamma, a.beta, c), a.act) * a.gamma[c] * a.dty[o + c];
      s[0] += t;
      s[1] += t * xh;
      s[2] += k;
      s[3] += k * xh;
      s[4] += k * t;
    }
    block_sum<kRowThreads>(s, red);
    const float n = 1.f / a.cols;
    const float mt = s[0] * n, b = s[1] * n, mk = s[2] * n, w = s[3] * n, q = s[4] * n - mk * mt;
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
      const float xh = __fmul_rn(a.x[o + c] - mean, rstd);
      const float k = row_act_grad(affine(xh, a.gamma, a.beta, c), a.act) * a.gamma[c] * a.dty[o + c];
      const float pk = rstd * (k - mk - xh * w), pt = rstd * (a.tx[o + c] - mt - xh * b);
      a.dtx[o + c] = (a.acc_t ? a.dtx[o + c] : 0.f) + pk;
      a.dx[o + c] = (a.acc_x ? a.dx[o + c] : 0.f) - rstd * (rstd * (q - w * b) * xh + b * pk + w * pt);
    }
    __syncthreads();
  }
}
// columns of dgamma = sum over rows of act' dty P t; the row means of t and t xh are formed again from x and tx
__global__ __launch_bounds__(256) void ln_tangent_bwd_columns(LayerNormTangentArgs a) {
  __shared__ float red[2 * 4];
  __shared__ float means[2];
  const int tid = threadIdx.x;
  // one block walks rows blockIdx.x, + gridDim.x, ...; its sums stay in memory of its own
  float* out = a.partial + (size_t)blockIdx.x * 2 * a.cols;
  bool first = true;
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const size_t o = (size_t)r * a.cols;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s[2] = {0.f, 0.f};
    for (int c = tid; c < a.cols; c += 256) {
      const float t = a.tx[o + c];
      s[0] += t;
      s[1] += t * __fmul_rn(a.x[o + c] - mean, rstd);
    }
    block_sum<256>(s, red);
    if (tid < 2) means[tid] = s[tid] / a.cols;
    __syncthreads();
    const float mt = means[0], b = means[1];
    for (int c = tid; c < a.cols; c += 256) {
      const float xh = __fmul_rn(a.x[o + c] - mean, rstd);
      const float v = row_act_grad(affine(xh, a.gamma, a.beta, c), a.act) * a.dty[o + c] * (rstd * (a.tx[o + c] - mt - xh * b));
      out[c] = (first ? 0.f : out[c]) + v;
    }
    first = false;
    __syncthreads();
  }
  for (int c = tid; c < a.cols; c += 256) out[a.cols + c] = 0.f;
}

void launch_layer_norm_tangent(const LayerNormTangentArgs& a, hipStream_t s) {
  if (a.rows && a.cols) row_launch(ln_tangent_rows, row_grid(a.rows), dim3(kRowThreads), s, a);
}
void launch_layer_norm_tangent_backward(const LayerNormTangentArgs& a, hipStream_t s) {
  if (!a.rows || !a.cols) return;
  row_launch(ln_tangent_bwd_rows, row_grid(a.rows), dim3(kRowThreads), s, a);
  if (!a.dgamma) return;
  const int groups = part_groups(a.rows);
  row_launch(ln_tangent_bwd_columns, dim3(groups), dim3(256), s, a);
  row_launch(ln_bwd_finish<float>, dim3((2 * a.cols + 255) / 256), dim3(256), s, a.partial, groups, a.cols, a.dgamma, nullptr, a.acc_w);
}

// ---- quantisation ----------------------------------------------------------------------------------------------------------
// The whole number nearest to 127 v / amax, exactly: inv = 127 / amax in 64 bits; v inv + 98304 is rounded once (fma) to a multiple of
// 2^-36, where a true tie lands on the tie (the product is off by under 2^-45) and nothing else does (127 v / amax is at least 2^-33 from a
// border that it is not on: with x's last bit u >= 2^-32 amax, 254 v - odd amax is a multiple of u).  Adding 1.5 2^52 then rounds to whole numbers, ties to even, and the
// sum's low byte is the signed 8-bit result (98304 = 0x18000).
__device__ __forceinline__ unsigned quantize1(float v, double inv) {
  const double t = __builtin_fma((double)v, inv, 98304.0) + 6755399441055744.0;
  return (unsigned)__double2loint(t) & 0xffu;
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void quantize_kernel(QuantizeArgs a) {
  __shared__ float red[2 * kRowThreads / 64];
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = (const T*)a.x + r * a.ldx;
    unsigned char* q = (unsigned char*)a.q + r * a.ldq;
    float mean = 0.f, rstd = 1.f;
    if (a.norm) row_statistics<T, kRowThreads>(x, a.cols, a.eps, red, mean, rstd);
    auto value = [&](int c) {
      float v = ld1(x + c);
      if (a.norm) v = affine(__fmul_rn(v - mean, rstd), a.gamma, a.beta, c);
      return v;
    };
    float m = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
      const float v = fabsf(value(c));
      m = (v > m || v != v) ? v : m;
    }
    m = block_max<kRowThreads>(m, red);
    const bool fine = m <= 3.4028235e38f;   // false for infinity and NaN: such a row's scale is NaN, its values zero
    const double inv = fine && m > 0.f ? 127.0 / (double)m : 0.0;
    const int width = (int)min((long long)((a.cols + 15) & ~15), a.ldq);   // the row's last 16-byte group is filled up with zeros
    for (int c = threadIdx.x; c < width; c += kRowThreads) q[c] = (unsigned char)(fine && c < a.cols ? quantize1(value(c), inv) : 0u);
    if (threadIdx.x == 0) a.scale[r] = fine ? m / 127.f : __builtin_nanf("");
    __syncthreads();
  }
}

void launch_quantize_rows(const QuantizeArgs& a, int type, hipStream_t s) {
  if (!a.rows) return;
  by_type(type, [&](auto t) { row_launch(quantize_kernel<decltype(t)>, row_grid(a.rows), dim3(kRowThreads), s, a); });
}

}  // namespace eg
