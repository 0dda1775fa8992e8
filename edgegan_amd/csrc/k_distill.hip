// Distillation from a teacher's top logits, loss and gradient in one launch.  For each row, with T the temperature and w the row's weight:
//   p = softmax(u / T) over the teacher's kept logits u,  q = softmax(z / T) over all of the student's logits z
//   loss = w T^2 sum_k p_k (log p_k - log q_i(k)),   dz_j = w T (q_j - sum of the p_k whose index is j)
// An index outside [0, cols) is padding: its logit is left out of p.  A row without a kept logit (none left, or all of them -inf) and a row
// of weight 0 have loss 0 and gradient 0, whatever the student's logits are.
//
// Bound by HBM: one read and one write of the logits.  A row stays in the registers of its team (a wave, 256 or 1,024 threads, at most 64 elements each) from
// the load through maximum, exponential and sum to the store, so each exponential is taken once.  The few columns that the teacher names are corrected
// behind the store of the row by the threads that hold the teacher's entries, in the same block.  exp((z - m) / T) is 2^((z - m) c): the difference
// first, so that rows of the type's lowest value stay finite.
#include <tuple>

#include "rowops_dev.h"

namespace eg {

constexpr int kDistillTop = 1024;   // most teacher logits a row
constexpr int team_top(int nt) { return nt > 64 ? kDistillTop : 128; }   // ... that a team's LDS holds

struct Kept {   // a teacher's entry: its column (-1: padding), (u - max u) / T and then p; the student's logit and the old gradient of the column
  int idx;
  float p, z, old;
};

// A team's threads see each other's LDS and memory writes of before.
template <int NT>
__device__ __forceinline__ void team_sync() {
  if constexpr (NT > 64) __syncthreads();
  else {
    __threadfence_block();
    __builtin_amdgcn_wave_barrier();
  }
}

// The teacher's kept entries of row r; returns false if there is none.  log_norm: the log of their exponentials' sum.
template <int NT>
__device__ __forceinline__ bool load_teacher(const DistillArgs& a, long long r, int t, Kept* kept, float (&red)[2][NT > 64 ? NT / 64 : 1], float it, float& log_norm) {
  float m = -INFINITY;
  for (int k = t; k < a.top; k += NT) {
    const long long j = a.index64 ? ((const long long*)a.index)[r * a.ld_index + k] : (long long)((const int*)a.index)[r * a.ld_index + k];
    const bool in = j >= 0 && j < a.cols;
    const float u = in ? a.teacher[r * a.ld_teacher + k] : -INFINITY;
    kept[k].idx = in ? (int)j : -1;
    kept[k].p = u;
    m = max_nan(m, u);
  }
  m = team_max<NT>(m, red[0]);
  if (m == -INFINITY) return false;
  float s[1] = {0.f};
  for (int k = t; k < a.top; k += NT) {
    const float v = (kept[k].p - m) * it;
    kept[k].p = v;
    s[0] += expf(v);
  }
  team_sum<NT>(s, red[1]);
  log_norm = logf(s[0]);
  return true;
}
// What the row holds in the teacher's columns, before the row is stored (the gradient may lie in the logits' memory).
template <typename T, int NT>
__device__ __forceinline__ void read_named(const DistillArgs& a, const T* z, const T* g, int t, Kept* kept) {
  for (int k = t; k < a.top; k += NT) {
    const int j = kept[k].idx;
    kept[k].z = j >= 0 ? (float)z[j] : 0.f;
    kept[k].old = j >= 0 && a.acc && g ? (float)g[j] : 0.f;
  }
}
// sum_k p_k (log p_k - log q_k); the entries' p become probabilities.  m: the student's maximum, log_sum the log of its exponentials' sum.
template <int NT>
__device__ __forceinline__ float teacher_loss(const DistillArgs& a, int t, Kept* kept, float (&red)[NT > 64 ? NT / 64 : 1], float it, float log_norm, float m, float log_sum) {
  float l[1] = {0.f};
  for (int k = t; k < a.top; k += NT) {
    const float lp = kept[k].p - log_norm;
    const float p = kept[k].idx >= 0 ? expf(lp) : 0.f;
    if (p != 0.f) l[0] += p * (lp - ((kept[k].z - m) * it - log_sum));
    kept[k].p = p;
  }
  team_sum<NT>(l, red);
  return l[0];
}
// The gradient's columns lo .. hi - 1 that the teacher names; an index given several times is written several times, with the same value.
template <typename T, int NT>
__device__ __forceinline__ void write_named(const DistillArgs& a, T* g, int t, const Kept* kept, float c, float m, float inv, float f, int lo, int hi) {
  for (int k = t; k < a.top; k += NT) {
    const int j = kept[k].idx;
    if (j < lo || j >= hi) continue;
    float p = 0.f;
    for (int l = 0; l < a.top; ++l) p += kept[l].idx == j ? kept[l].p : 0.f;
    g[j] = (T)(kept[k].old + f * (__builtin_amdgcn_exp2f((kept[k].z - m) * c) * inv - p));
  }
}

constexpr float kLog2e = 1.44269504088896340736f;
// A row in a team's registers.
template <typename T, int NT, int NE, int V>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void distill_rows(DistillArgs a) {
  constexpr int NB = NT > 256 ? NT : 256, TEAMS = NB / NT, NV = NE / V;
  __shared__ Kept all_kept[TEAMS][team_top(NT)];
  __shared__ float red_t[2][NT > 64 ? NT / 64 : 1], red[3][NT > 64 ? NT / 64 : 1];   // (one wave needs none)
  const int t = threadIdx.x % NT, team = threadIdx.x / NT;
  Kept* kept = all_kept[team];
  const float it = 1.f / a.temperature, c = it * kLog2e;
  for (long long r = (long long)blockIdx.x * TEAMS + team; r < a.rows; r += (long long)gridDim.x * TEAMS) {
    const T* z = (const T*)a.logits + r * a.ld;
    T* g = a.grad ? (T*)a.grad + r * a.ldg : nullptr;
    const float w = (a.row_weight ? a.row_weight[r] : 1.f) * a.weight;
    float v[NV][V], log_norm = 0.f;
    bool alive = w != 0.f;
    if (alive) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = (i * NT + t) * V;
        load_pack<T, V>(z + (at < a.cols ? at : 0), v[i]);   // (columns past the last repeat the first ones; they are left out of the sum)
      }
      alive = load_teacher<NT>(a, r, t, kept, red_t, it, log_norm);
    }
    if (!alive) {
      if (g && !a.acc) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int at = (i * NT + t) * V;
          const float zero[V] = {};
          if (at < a.cols) store_pack<T, V>(g + at, zero);
        }
      }
      if (t == 0) a.loss[r] = 0.f;
      team_sync<NT>();
      continue;
    }
    read_named<T, NT>(a, z, g, t, kept);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) m = max_nan(m, v[i][j]);
    m = team_max<NT>(m, red[0]);
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = (i * NT + t) * V < a.cols ? __builtin_amdgcn_exp2f((v[i][j] - m) * c) : 0.f;
        s[0] += v[i][j];
      }
    team_sum<NT>(s, red[1]);
    const float loss = teacher_loss<NT>(a, t, kept, red[2], it, log_norm, m, logf(s[0]));
    if (t == 0) a.loss[r] = w * a.temperature * a.temperature * loss;
    if (g) {
      const float f = w * a.temperature, inv = 1.f / s[0], fi = f * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = (i * NT + t) * V;
        if (at >= a.cols) continue;
        float o[V] = {};
        if (a.acc) load_pack<T, V>(g + at, o);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] += v[i][j] * fi;
        store_pack<T, V>(g + at, o);
      }
      team_sync<NT>();
      write_named<T, NT>(a, g, t, kept, c, m, inv, f, 0, a.cols);
    }
    team_sync<NT>();
  }
}

// ---- a row over several blocks ----------------------------------------------------------------------------------------------------
// Rows too long for a team's registers, or long ones too few for the chip's 256 compute units: blocks of kChunk columns, first their maximum and sum of
// exponentials (and the student's logits in the teacher's columns) into the workspace [rows][2 chunks + top], then, in a second launch, the
// loss and the gradient.  The row is read twice.
constexpr int kChunkThreads = 256, kChunk = 8192;
static int chunks_of(int cols) { return (cols + kChunk - 1) / kChunk; }

template <int V, typename F>
__device__ __forceinline__ void walk(int lo, int hi, F f) {
#pragma unroll 4
  for (int c = lo + threadIdx.x * V; c < hi; c += kChunkThreads * V) f(c);
}
template <typename T, int V>
__global__ __launch_bounds__(kChunkThreads) void distill_chunk_sums(DistillArgs a, int chunks) {
  __shared__ float red[2][kChunkThreads / 64];
  const float c = 1.f / a.temperature * kLog2e;
  const long long tasks = a.rows * chunks;
  for (long long q = blockIdx.x; q < tasks; q += gridDim.x) {
    const long long r = q / chunks;
    const int chunk = (int)(q - r * chunks), lo = chunk * kChunk, hi = min(lo + kChunk, a.cols);
    const T* z = (const T*)a.logits + r * a.ld;
    float* out = a.partial + r * (2 * chunks + a.top);
    float m = -INFINITY;
    walk<V>(lo, hi, [&](int at) {
      float v[V];
      load_pack<T, V>(z + at, v);
#pragma unroll
      for (int j = 0; j < V; ++j) m = max_nan(m, v[j]);
    });
    m = team_max<kChunkThreads>(m, red[0]);
    float s[1] = {0.f};
    if (m != -INFINITY)
      walk<V>(lo, hi, [&](int at) {
        float v[V];
        load_pack<T, V>(z + at, v);
#pragma unroll
        for (int j = 0; j < V; ++j) s[0] += __builtin_amdgcn_exp2f((v[j] - m) * c);
      });
    team_sum<kChunkThreads>(s, red[1]);
    if (threadIdx.x == 0) {
      out[2 * chunk] = m;
      out[2 * chunk + 1] = s[0];
    }
    if (chunk == 0)
      for (int k = threadIdx.x; k < a.top; k += kChunkThreads) {
        const long long j = a.index64 ? ((const long long*)a.index)[r * a.ld_index + k] : (long long)((const int*)a.index)[r * a.ld_index + k];
        out[2 * chunks + k] = j >= 0 && j < a.cols ? (float)z[j] : 0.f;
      }
    __syncthreads();
  }
}
template <typename T, int V>
__global__ __launch_bounds__(kChunkThreads) void distill_chunk_grad(DistillArgs a, int chunks) {
  __shared__ Kept kept[kDistillTop];
  __shared__ float red_t[2][kChunkThreads / 64], red[3][kChunkThreads / 64];
  const int t = threadIdx.x;
  const float it = 1.f / a.temperature, c = it * kLog2e;
  const int per = a.grad ? chunks : 1;   // (without a gradient one block a row forms the loss)
  const long long tasks = a.rows * per;
  for (long long q = blockIdx.x; q < tasks; q += gridDim.x) {
    const long long r = q / per;
    const int chunk = (int)(q - r * per), lo = chunk * kChunk, hi = min(lo + kChunk, a.cols);
    const T* z = (const T*)a.logits + r * a.ld;
    T* g = a.grad ? (T*)a.grad + r * a.ldg : nullptr;
    const float* in = a.partial + r * (2 * chunks + a.top);
    const float w = (a.row_weight ? a.row_weight[r] : 1.f) * a.weight;
    float log_norm = 0.f;
    if (w == 0.f || !load_teacher<kChunkThreads>(a, r, t, kept, red_t, it, log_norm)) {
      if (g && !a.acc)
        for (int j = lo + t; j < hi; j += kChunkThreads) g[j] = (T)0.f;
      if (t == 0 && chunk == 0) a.loss[r] = 0.f;
      __syncthreads();
      continue;
    }
    for (int k = t; k < a.top; k += kChunkThreads) {
      const int j = kept[k].idx;
      kept[k].z = in[2 * chunks + k];
      kept[k].old = j >= lo && j < hi && a.acc && g ? (float)g[j] : 0.f;   // (read_named, of this block's columns)
    }
    float m = -INFINITY;
    for (int k = t; k < chunks; k += kChunkThreads) m = max_nan(m, in[2 * k]);
    m = team_max<kChunkThreads>(m, red[0]);
    float s[1] = {0.f};
    for (int k = t; k < chunks; k += kChunkThreads)
      if (in[2 * k] != -INFINITY) s[0] += in[2 * k + 1] * __builtin_amdgcn_exp2f((in[2 * k] - m) * c);
    team_sum<kChunkThreads>(s, red[1]);
    const float loss = teacher_loss<kChunkThreads>(a, t, kept, red[2], it, log_norm, m, logf(s[0]));
    if (t == 0 && chunk == 0) a.loss[r] = w * a.temperature * a.temperature * loss;
    if (g) {
      const float f = w * a.temperature, inv = 1.f / s[0], fi = f * inv;
      walk<V>(lo, hi, [&](int at) {
        float v[V], o[V] = {};
        load_pack<T, V>(z + at, v);
        if (a.acc) load_pack<T, V>(g + at, o);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] += __builtin_amdgcn_exp2f((v[j] - m) * c) * fi;
        store_pack<T, V>(g + at, o);
      });
      __syncthreads();
      write_named<T, kChunkThreads>(a, g, t, kept, c, m, inv, f, lo, hi);
    }
    __syncthreads();
  }
}

// One row a team where the registers hold it and the rows are enough for the chip, else chunks.
static bool distill_in_chunks(long long rows, int cols) { return cols > 65536 || (cols > 2 * kChunk && rows < 64); }

size_t distill_partial_floats(long long rows, int cols, int top) {
  return distill_in_chunks(rows, cols) ? (size_t)rows * (2 * chunks_of(cols) + top) : 0;
}

template <typename T, int V>
static void distill_team(const DistillArgs& a, hipStream_t s) {
  auto go = [&](auto nt, auto ne) {
    constexpr int NT = decltype(nt)::value, NE = decltype(ne)::value, TEAMS = NT > 256 ? 1 : 256 / NT;
    row_launch(distill_rows<T, NT, NE, V>, dim3((unsigned)std::min<long long>((a.rows + TEAMS - 1) / TEAMS, 1 << 16)), dim3(NT > 256 ? NT : 256), s, a);
  };
  using std::integral_constant;
#define EG_TEAM(NT, NE) if (a.cols <= (NT) * (NE) && a.top <= team_top(NT)) return go(integral_constant<int, NT>{}, integral_constant<int, NE>{})
  EG_TEAM(64, 8);
  EG_TEAM(64, 16);
  EG_TEAM(256, 16);
  EG_TEAM(256, 32);
  EG_TEAM(1024, 16);
  EG_TEAM(1024, 32);
  EG_TEAM(1024, 64);
#undef EG_TEAM
}

void launch_distill(const DistillArgs& a, int type, hipStream_t s) {
  if (!a.rows) return;
  EG_CHECK(a.top <= kDistillTop, "distillation: at most %d teacher logits a row", kDistillTop);
  by_type(type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto v) {
      constexpr int V = decltype(v)::value;
      if (!distill_in_chunks(a.rows, a.cols)) return distill_team<T, V>(a, s);
      const int chunks = chunks_of(a.cols);
      row_launch(distill_chunk_sums<T, V>, dim3((unsigned)std::min<long long>(a.rows * chunks, 1 << 16)), dim3(kChunkThreads), s, a, chunks);
      row_launch(distill_chunk_grad<T, V>, dim3((unsigned)std::min<long long>(a.rows * (a.grad ? chunks : 1), 1 << 16)), dim3(kChunkThreads), s, a, chunks);
    };
    constexpr int V = 16 / sizeof(T);
    const bool packs = a.cols % V == 0 && (uintptr_t)a.logits % 16 == 0 && a.ld * sizeof(T) % 16 == 0 && (!a.grad || ((uintptr_t)a.grad % 16 == 0 && a.ldg * sizeof(T) % 16 == 0));
    if (packs) go(std::integral_constant<int, V>{});
    else go(std::integral_constant<int, 1>{});
  });
}

}  // namespace eg
