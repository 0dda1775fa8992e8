// Distillation from a teacher's top logits, loss and gradient in one launch.  For each row, with T the temperature and w the row's weight:
//   p = softmax(u / T) over the teacher's kept logits u,  q = softmax(z / T) over all of the student's logits z
//   loss = w T^2 sum_k p_k (log p_k - log q_i(k)),   dz_j = w T (q_j - sum of the p_k whose index is j)
// An index outside [0, cols) is padding: its logit is left out of p.  A row without a kept logit (none left, or all of them -inf) and a row
// of weight 0 have loss 0 and gradient 0, whatever the student's logits are.
//
// Bound by HBM: one read and one write of the logits.  A row stays in the registers of its team (a wave, 256 or 1,024 threads, at most 64 elements each) from
// the load through maximum and sum to the store: in 16 bits as loaded (half the registers: two rows of
// 65,536 a compute unit; the exponentials are taken twice), in
// 32 bits as exponentials.  The few columns that the teacher names are corrected
// behind the store of the row by the threads that hold the teacher's entries, in the same block.  exp((z - m) / T) is 2^((z - m) c): the difference
// first, so that rows of the type's lowest value stay finite.
// Measured: 4,096 x 65,536 bf16 218 - 224 us (4.9 TB/s; a copy of 1 GB 4.8 - 5.3), 511 x 10,007 f16 12.5 us, 64 x 14 f32 4.7 us.
#include <cmath>
#include <tuple>

#include "rowops_dev.h"

namespace eg {

constexpr int kDistillTop = 1024;   // most teacher logits a row
constexpr int team_top(int nt) { return nt > 64 ? kDistillTop : 128; }   // ... that a team's LDS holds

struct Kept {   // a teacher's entry: its column (-1: padding), (u - max u) / T and then p; the student's logit in the column
  int idx;
  float p, z;
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
#pragma unroll 1
  for (int k = t; k < a.top; k += NT) {
    const long long j = a.index64 ? ((const long long*)a.index)[r * a.ld_index + k] : (long long)((const int*)a.index)[r * a.ld_index + k];
    const float given = a.teacher[r * a.ld_teacher + k];   // (beside the index, not behind it)
    const bool in = j >= 0 && j < a.cols;
    const float u = in ? given : -INFINITY;
    kept[k].idx = in ? (int)j : -1;
    kept[k].p = u;
    m = max_nan(m, u);
  }
  m = team_max<NT>(m, red[0]);
  if (m == -INFINITY) return false;
  float s[1] = {0.f};
#pragma unroll 1
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
__device__ __forceinline__ void read_named(const DistillArgs& a, const T* z, int t, Kept* kept) {
#pragma unroll 1
  for (int k = t; k < a.top; k += NT) kept[k].z = kept[k].idx >= 0 ? (float)z[kept[k].idx] : 0.f;
}
// sum_k p_k (log p_k - log q_k); the entries' p become probabilities.  m: the student's maximum, log_sum the log of its exponentials' sum.
template <int NT>
__device__ __forceinline__ float teacher_loss(const DistillArgs& a, int t, Kept* kept, float (&red)[NT > 64 ? NT / 64 : 1], float it, float log_norm, float m, float log_sum) {
  float l[1] = {0.f};
#pragma unroll 1
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
// log_q: of a logit.
template <typename T, int NT, typename L>
__device__ __forceinline__ void write_named(const DistillArgs& a, T* g, int t, const Kept* kept, float f, L log_q, int lo, int hi) {
#pragma unroll 1
  for (int k = t; k < a.top; k += NT) {
    const int j = kept[k].idx;
    if (j < lo || j >= hi) continue;
    float p = 0.f;
#pragma unroll 4
    for (int l = 0; l < a.top; ++l) p += kept[l].idx == j ? kept[l].p : 0.f;
    g[j] = (T)(f * (expf(log_q(kept[k].z)) - p));
  }
}

constexpr float kLog2e = 1.44269504088896340736f;
// Tells the compiler that a pack may have changed: it then forms what follows from the pack again instead of keeping its converted elements and their
// exponentials in registers from one pass over the row to the next.
template <typename T, int V>
__device__ __forceinline__ void opaque(LoosePack<T, V>& p) {
  if constexpr (sizeof(p) == 2) {
    unsigned u = __builtin_bit_cast(unsigned short, p);
    asm volatile("" : "+v"(u));
    p = __builtin_bit_cast(LoosePack<T, V>, (unsigned short)u);
  } else {
    struct Words {
      unsigned w[sizeof(p) / 4];
    } k = __builtin_bit_cast(Words, p);
#pragma unroll
    for (unsigned& w : k.w) asm volatile("" : "+v"(w));
    p = __builtin_bit_cast(LoosePack<T, V>, k);
  }
}

// The largest of packs.  In 16 bits two elements an instruction: as signed whole numbers non-negative floats keep their order and negative ones lie
// below them in reversed order, so the row's maximum is the largest whole number if that is a non-negative float, else the smallest.  (A NaN need not be kept: the sum is then NaN.)
template <typename T>
struct RowMax {
  using i16x2 = __attribute__((ext_vector_type(2))) short;
  float m = -INFINITY;
  i16x2 hi = {-32768, -32768}, lo = {32767, 32767};
  template <int V>
  __device__ __forceinline__ void take(const LoosePack<T, V>& p) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < V; ++j) m = fmaxf(m, p.e[j]);
    } else if constexpr (V == 1) {
      const short k = __builtin_bit_cast(short, p);
      hi.x = hi.x > k ? hi.x : k;
      lo.x = lo.x < k ? lo.x : k;
    } else {
      struct Words {
        i16x2 w[V / 2];
      } k = __builtin_bit_cast(Words, p);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        hi = __builtin_elementwise_max(hi, k.w[j]);
        lo = __builtin_elementwise_min(lo, k.w[j]);
      }
    }
  }
  __device__ __forceinline__ float value() const {
    if constexpr (sizeof(T) == 4) return m;
    else {
      const short h = hi.x > hi.y ? hi.x : hi.y, l = lo.x < lo.y ? lo.x : lo.y;
      return (float)__builtin_bit_cast(T, h >= 0 ? h : l);
    }
  }
};
// A row in a team's registers.  A long row is alone in its registers: the teacher's part lies before the load and behind the
// store (with it in between the compiler spilt the row).  The other block of a compute unit fills the waits.
template <typename T, int NT, int NE, int V>
__global__ __launch_bounds__(NT > 256 ? NT : 256) void distill_rows(DistillArgs a) {
  constexpr int NB = NT > 256 ? NT : 256, TEAMS = NB / NT, NV = NE / V;
  __shared__ Kept all_kept[TEAMS][team_top(NT)];
  __shared__ float red_t[2][NT > 64 ? NT / 64 : 1], red[3][NT > 64 ? NT / 64 : 1];   // (one wave needs none)
  const int t = TEAMS > 1 ? threadIdx.x % NT : threadIdx.x, team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
  const long long r = (long long)blockIdx.x * TEAMS + team;
  if (r >= a.rows) return;   // (a whole wave)
  Kept* kept = all_kept[team];
  const float it = 1.f / a.temperature, c = it * kLog2e;
  const T* z = (const T*)a.logits + r * a.ld;
  T* g = a.grad ? (T*)a.grad + r * a.ldg : nullptr;
  const float w = (a.row_weight ? a.row_weight[r] : 1.f) * a.weight;
  LoosePack<T, V> v[NV];
  auto load_row = [&] { request_row<T, NT, NV, V>(z, a.cols, t, v); };   // (packs past the end repeat the last ones: left out of the sum)
  auto store = [&](int i, int th, const float (&o)[V]) {
    const int at = (th + i * NT) * V;
    if (at < a.cols) store_row_pack<T, V, true>(g, at, a.cols, o);
  };
  constexpr bool EARLY = NE <= 16;   // few registers: the row is on its way while the teacher's part is worked on
  if constexpr (EARLY) load_row();
  float log_norm = 0.f;
  if (w == 0.f || !load_teacher<NT>(a, r, t, kept, red_t, it, log_norm)) {
    if (g)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float zero[V] = {};
        store(i, t, zero);
      }
    if (t == 0) a.loss[r] = 0.f;
    return;
  }
  read_named<T, NT>(a, z, t, kept);
  if constexpr (!EARLY) load_row();
  if (V > 1 && a.cols % V) settle_row<T, NT, NV, V, true>(a.cols, t, v, (T)-INFINITY);
  RowMax<T> most;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    most.take(v[i]);
    if constexpr (NE > 16) __builtin_amdgcn_sched_barrier(0);   // (pack by pack: the scheduler would convert the whole row at once)
  }
  const float m = team_max<NT>(most.value(), red[0]);
  float s[1] = {0.f};
  const int t1 = fresh(t);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    opaque(v[i]);
    float part = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float e = __builtin_amdgcn_exp2f(((float)v[i].e[j] - m) * c);
      if constexpr (sizeof(T) == 4) v[i].e[j] = e;
      part += e;
    }
    s[0] += (t1 + i * NT) * V < a.cols ? part : 0.f;
    opaque(v[i]);
    if constexpr (NE > 16) __builtin_amdgcn_sched_barrier(0);
  }
  team_sum<NT>(s, red[1]);
  const float f = w * a.temperature;
  if (g) {
    const float fi = f / s[0];
    const int t2 = fresh(t);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = (sizeof(T) == 4 ? (float)v[i].e[j] : __builtin_amdgcn_exp2f(((float)v[i].e[j] - m) * c)) * fi;
      store(i, t2, o);
      if constexpr (NE > 16) __builtin_amdgcn_sched_barrier(0);
    }
  }
  const float log_sum = logf(s[0]);
  const float loss = teacher_loss<NT>(a, t, kept, red[2], it, log_norm, m, log_sum);
  if (t == 0) a.loss[r] = f * (a.temperature * loss);   // (T^2 may leave f32's range where T^2 KL does not)
  team_sync<NT>();
  if (g) write_named<T, NT>(a, g, t, kept, f, [&](float x) { return it * (x - m) - log_sum; }, 0, a.cols);
}

// ---- a row over several blocks ----------------------------------------------------------------------------------------------------
// Rows too long for a team's registers, or a few that would fill them: blocks of kChunk columns, first their maximum and sum of
// exponentials (and the student's logits in the teacher's columns) into the workspace [rows][2 chunks + top], then, in a second launch, the
// loss and the gradient.  The row is read twice.
constexpr int kChunkThreads = 256, kChunk = 8192;
static int chunks_of(int cols) { return (cols + kChunk - 1) / kChunk; }

// f(column, elements as a type): packs of V at any address, then what is left one by one
template <int V, typename F>
__device__ __forceinline__ void walk(int lo, int hi, F f) {
#pragma unroll 4
  for (int c = lo + threadIdx.x * V; c + V <= hi; c += kChunkThreads * V) f(c, std::integral_constant<int, V>{});
  if ((int)threadIdx.x < (hi - lo) % V) f(hi - (hi - lo) % V + (int)threadIdx.x, std::integral_constant<int, 1>{});
}
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void distill_chunk_sums(DistillArgs a, int chunks) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float red[2][kChunkThreads / 64];
  const float c = 1.f / a.temperature * kLog2e;
  const long long tasks = a.rows * chunks;
  for (long long q = blockIdx.x; q < tasks; q += gridDim.x) {
    const long long r = q / chunks;
    const int chunk = (int)(q - r * chunks), lo = chunk * kChunk, hi = min(lo + kChunk, a.cols);
    const T* z = (const T*)a.logits + r * a.ld;
    float* out = a.partial + r * (2 * chunks + a.top);
    float m = -INFINITY;
    walk<V>(lo, hi, [&](int at, auto n) {
      const auto k = *reinterpret_cast<const LoosePack<T, decltype(n)::value>*>(z + at);
#pragma unroll
      for (int j = 0; j < decltype(n)::value; ++j) m = max_nan(m, (float)k.e[j]);
    });
    m = team_max<kChunkThreads>(m, red[0]);
    float s[1] = {0.f};
    if (m != -INFINITY)
      walk<V>(lo, hi, [&](int at, auto n) {
        const auto k = *reinterpret_cast<const LoosePack<T, decltype(n)::value>*>(z + at);
#pragma unroll
        for (int j = 0; j < decltype(n)::value; ++j) s[0] += __builtin_amdgcn_exp2f(((float)k.e[j] - m) * c);
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
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void distill_chunk_grad(DistillArgs a, int chunks) {
  constexpr int V = 16 / sizeof(T);
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
      if (g)
        for (int j = lo + t; j < hi; j += kChunkThreads) g[j] = (T)0.f;
      if (t == 0 && chunk == 0) a.loss[r] = 0.f;
      __syncthreads();
      continue;
    }
    for (int k = t; k < a.top; k += kChunkThreads) kept[k].z = in[2 * chunks + k];
    float m = -INFINITY;
    for (int k = t; k < chunks; k += kChunkThreads) m = max_nan(m, in[2 * k]);
    m = team_max<kChunkThreads>(m, red[0]);
    float s[1] = {0.f};
    for (int k = t; k < chunks; k += kChunkThreads)
      if (in[2 * k] != -INFINITY) s[0] += in[2 * k + 1] * __builtin_amdgcn_exp2f((in[2 * k] - m) * c);
    team_sum<kChunkThreads>(s, red[1]);
    const float log_sum = logf(s[0]);
    const float loss = teacher_loss<kChunkThreads>(a, t, kept, red[2], it, log_norm, m, log_sum);
    if (t == 0 && chunk == 0) a.loss[r] = w * a.temperature * (a.temperature * loss);
    if (g) {
      const float f = w * a.temperature, fi = f / s[0];
      walk<V>(lo, hi, [&](int at, auto n) {
        using P = LoosePack<T, decltype(n)::value>;
        P k = *reinterpret_cast<const P*>(z + at);
#pragma unroll
        for (int j = 0; j < decltype(n)::value; ++j) k.e[j] = (T)(__builtin_amdgcn_exp2f(((float)k.e[j] - m) * c) * fi);
        *reinterpret_cast<P*>(g + at) = k;
      });
      __syncthreads();
      write_named<T, kChunkThreads>(a, g, t, kept, f, [&](float z) { return it * (z - m) - log_sum; }, lo, hi);
    }
    __syncthreads();
  }
}

// A row a team while its registers hold the row, else chunks; chunks also for rows that fill those registers where they are few. us, team / chunks, bf16:
//   32,768 columns: 9.2 / 10.7 for one row, 10.1 / 11.8 for 64, 13.3 / 18.0 for 256;  65,536: 12.6 / 10.9, 14.0 / 13.3, 20.0 / 29.5 (128 rows: 16.3 / 17.4)
static bool distill_in_chunks(long long rows, int cols) { return cols > 65536 || (cols > 32768 && rows <= 64); }

// (the kernels scale by its reciprocal and by log2 e times that)
bool distill_temperature(float t) { return t > 0.f && std::isfinite(t) && std::isfinite(1.f / t * kLog2e); }

size_t distill_partial_floats(long long rows, int cols, int top) {
  return distill_in_chunks(rows, cols) ? (size_t)rows * (2 * chunks_of(cols) + top) : 0;
}

template <typename T, int NT, int NE, int V>
static void distill_launch(const DistillArgs& a, hipStream_t s) {
  constexpr int TEAMS = NT > 256 ? 1 : 256 / NT;
  constexpr long long slab = 1 << 20;   // rows of a launch (a grid has fewer than 2^32 threads)
  for (long long r = 0; r < a.rows; r += slab) {
    DistillArgs p = a;
    p.rows = std::min(slab, a.rows - r);
    p.logits = (const T*)a.logits + r * a.ld;
    p.index = (const char*)a.index + r * a.ld_index * (a.index64 ? 8 : 4);
    p.teacher = a.teacher + r * a.ld_teacher;
    if (a.row_weight) p.row_weight = a.row_weight + r;
    p.loss = a.loss + r;
    if (a.grad) p.grad = (T*)a.grad + r * a.ldg;
    row_launch(distill_rows<T, NT, NE, V>, dim3((unsigned)((p.rows + TEAMS - 1) / TEAMS)), dim3(NT > 256 ? NT : 256), s, p);
  }
}
// The smallest team that holds the row; us with it / with the next one, bf16: 16,384 x 1,000 20.5 (a wave of 16 elements a thread) / 43 (256 threads), 8,192 x 7,000 48 (256 of
// 32) / 104 (1,024 of 16), 2,048 x 30,000 55 (1,024 of 32) / 67 (1,024 of 64); 16,384 x 300 15.0 / 17.1, 4,096 x 14,000 61 / 77; 64 rows of 7,000 5.6 / 6.3.
template <typename T>
static void distill_team(const DistillArgs& a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
#define EG_TEAM(NT, NE) if (a.cols <= (NT) * (NE) && a.top <= team_top(NT)) return distill_launch<T, NT, NE, V>(a, s)
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
  by_type(type, [&](auto t) {
    using T = decltype(t);
    if (distill_in_chunks(a.rows, a.cols)) {
      const int chunks = chunks_of(a.cols);
      row_launch(distill_chunk_sums<T>, dim3((unsigned)std::min<long long>(a.rows * chunks, 1 << 16)), dim3(kChunkThreads), s, a, chunks);
      return row_launch(distill_chunk_grad<T>, dim3((unsigned)std::min<long long>(a.rows * (a.grad ? chunks : 1), 1 << 16)), dim3(kChunkThreads), s, a, chunks);
    }
    constexpr int V = 16 / sizeof(T);
    if (a.cols >= V) distill_team<T>(a, s);
    else if (a.top <= team_top(64)) distill_launch<T, 64, 8, 1>(a, s);   // (shorter than a pack)
    else distill_launch<T, 256, 16, 1>(a, s);
  });
}

__global__ __launch_bounds__(256) void distill_join(const float* more, float* grad, int n, const float* loss, int rows, float* total) {
  __shared__ float red[4];
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) grad[i] += more[i];
  if (blockIdx.x) return;
  float s[1] = {0.f};
  for (int r = threadIdx.x; r < rows; r += 256) s[0] += loss[r];
  team_sum<256>(s, red);
  if (threadIdx.x == 0) *total = s[0];
}
void launch_distill_join(const float* more, float* grad, int n, const float* loss, int rows, float* total, hipStream_t s) {
  row_launch(distill_join, dim3((unsigned)std::min((n + 255) / 256, 256)), dim3(256), s, more, grad, n, loss, rows, total);
}

}  // namespace eg
