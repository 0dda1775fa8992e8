// Distillation from a teacher's top logits, loss and gradient in one launch.  For each row, with T the temperature and w the row's weight:
//   p = softmax(u / T) over the teacher's kept logits u,  q = softmax(z / T) over all of the student's logits z
//   loss = w T^2 sum_k p_k (log p_k - log q_i(k)),   dz_j = w T (q_j - sum of the p_k whose index is j)
// An index outside [0, cols) is padding: its logit is left out of p.  A row without a kept logit (none left, or all of them -inf) and a row
// of weight 0 have loss 0 and gradient 0, whatever the student's logits are.  Bound by HBM: one read and one write of the logits.
#include <tuple>

#include "rowops_dev.h"

namespace eg {

constexpr int kDistillThreads = 256;
constexpr int kDistillTop = 1024;   // most teacher logits a row (they are held in LDS)

__device__ __forceinline__ long long teacher_index(const DistillArgs& a, long long r, int k) {
  const long long i = a.index64 ? ((const long long*)a.index)[r * a.ld_index + k] : (long long)((const int*)a.index)[r * a.ld_index + k];
  return i >= 0 && i < a.cols ? i : -1;
}

template <typename T>
__global__ __launch_bounds__(kDistillThreads) void distill_rows(DistillArgs a) {
  __shared__ float red[kDistillThreads / 64];
  __shared__ float p[kDistillTop];
  __shared__ int idx[kDistillTop];
  const int tid = threadIdx.x;
  const float it = 1.f / a.temperature;
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* z = (const T*)a.logits + r * a.ld;
    T* g = a.grad ? (T*)a.grad + r * a.ldg : nullptr;
    const float w = (a.row_weight ? a.row_weight[r] : 1.f) * a.weight;
    // the teacher
    float m = -INFINITY;
    for (int k = tid; k < a.top; k += kDistillThreads) {
      idx[k] = (int)teacher_index(a, r, k);
      p[k] = idx[k] >= 0 ? a.teacher[r * a.ld_teacher + k] * it : -INFINITY;
      m = (p[k] > m || p[k] != p[k]) ? p[k] : m;
    }
    m = team_max<kDistillThreads>(m, red);
    __syncthreads();
    if (w == 0.f || m == -INFINITY) {
      if (g && !a.acc)
        for (int c = tid; c < a.cols; c += kDistillThreads) g[c] = (T)0.f;
      if (tid == 0) a.loss[r] = 0.f;
      continue;
    }
    float s[1] = {0.f};
    for (int k = tid; k < a.top; k += kDistillThreads) s[0] += expf(p[k] - m);
    team_sum<kDistillThreads>(s, red);
    const float lse_t = m + logf(s[0]);
    __syncthreads();
    // the student
    float zm = -INFINITY;
    for (int c = tid; c < a.cols; c += kDistillThreads) {
      const float v = (float)z[c] * it;
      zm = (v > zm || v != v) ? v : zm;
    }
    zm = team_max<kDistillThreads>(zm, red);
    __syncthreads();
    float e[1] = {0.f};
    for (int c = tid; c < a.cols; c += kDistillThreads) e[0] += expf((float)z[c] * it - zm);
    team_sum<kDistillThreads>(e, red);
    const float lse = zm + logf(e[0]);
    __syncthreads();
    // the loss; p becomes a probability
    float l[1] = {0.f};
    for (int k = tid; k < a.top; k += kDistillThreads) {
      const float lp = p[k] - lse_t, pk = expf(lp);
      if (idx[k] >= 0 && pk != 0.f) l[0] += pk * (lp - ((float)z[idx[k]] * it - lse));
      p[k] = pk;
    }
    team_sum<kDistillThreads>(l, red);
    if (tid == 0) a.loss[r] = w * a.temperature * a.temperature * l[0];
    if (g) {
      // the kept indexes first, from the old gradient where it is added to; then every other column by its own thread
      const float f = w * a.temperature;
      __syncthreads();
      for (int c = tid; c < a.cols; c += kDistillThreads) {
        float v = expf((float)z[c] * it - lse);
        for (int k = 0; k < a.top; ++k) v -= idx[k] == c ? p[k] : 0.f;
        v *= f;
        if (a.acc) v += (float)g[c];
        g[c] = (T)v;
      }
    }
    __syncthreads();
  }
}

size_t distill_partial_floats(long long rows, int cols) { return 0; }

void launch_distill(const DistillArgs& a, int type, hipStream_t s) {
  if (!a.rows) return;
  EG_CHECK(a.top <= kDistillTop, "distillation: at most %d teacher logits a row", kDistillTop);
  by_type(type, [&](auto t) {
    row_launch(distill_rows<decltype(t)>, dim3((unsigned)std::min<long long>(a.rows, 1 << 20)), dim3(kDistillThreads), s, a);
  });
}

}  // namespace eg
