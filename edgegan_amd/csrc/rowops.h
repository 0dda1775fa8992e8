// Operators over rows in device memory (C entries: rowops.cpp; kernels: k_layer_norm.hip, k_int8.hip, k_distill.hip).
// A row is `cols` consecutive elements; rows are `ld` elements apart (ld >= cols, any alignment).
#pragma once
#include <hip/hip_runtime.h>

namespace eg {

enum RowType { ROW_F32 = 0, ROW_BF16 = 1, ROW_F16 = 2 };

struct LayerNormArgs {
  const void* x;
  long long ldx;
  const void *gamma, *beta;   // [cols] or null
  long long rows;
  int cols;
  float eps;
  int act;                    // ACT_NONE / ACT_RELU / ACT_LRELU
  void* y;
  long long ldy;
  float *mean, *rstd;         // [rows]; null: not stored (forward), required (backward)
};
// LeakyReLU's derivative at a pre-activation of exactly 0, where a row of one value has all of its elements unless there is a shift: the operators of
// include/edgegan_hip.h take its slope, the engine 1, as its LeakyReLUs everywhere (max(z, 0.2 z), whose gradient goes to z where both are equal)
constexpr float kLreluAtZero = 0.2f, kEngineLreluAtZero = 1.f;
struct LayerNormGradArgs {
  const void *dy, *x;
  long long lddy, ldx;
  const float *mean, *rstd;
  const void *gamma, *beta;
  long long rows;
  int cols;
  int act;
  float at_zero;              // kLreluAtZero / kEngineLreluAtZero
  void* dx;                   // null: not wanted
  long long lddx;
  int acc_x;                  // dx += (f32 only)
  void *dgamma, *dbeta;       // null: not wanted
  int acc_w;                  // bit 0: dgamma +=, bit 1: dbeta +=
  float* partial;             // layer_norm_partial_floats()
};
// J_v of the layer norm at x and its reverse (f32; the gradient penalty of a critic; LeakyReLU's derivative at 0 is kEngineLreluAtZero)
struct LayerNormTangentArgs {
  const float *x, *mean, *rstd, *gamma, *beta, *tx;
  long long rows;
  int cols;
  int act;
  float* ty;                  // forward: act' gamma P tx
  const float* dty;           // reverse: the gradient of ty ...
  float* dtx;                 //   ... gives that of tx, x and gamma
  int acc_t;
  float* dx;
  int acc_x;
  float* dgamma;
  int acc_w;
  float* partial;
};
struct QuantizeArgs {
  const void* x;
  long long ldx;
  const float *gamma, *beta;  // the fused layer norm's (null: 1, 0)
  bool norm;
  float eps;
  long long rows;
  int cols;
  signed char* q;
  long long ldq;
  float* scale;
};
struct Int8Args {
  const signed char* a;
  long long lda;
  const float* a_scale;
  const signed char* b;
  long long ldb;
  const float* b_scale;
  const float* bias;          // [n] or null
  long long m;
  int n, k;
  void* out;
  long long ldo;
};
struct DistillArgs {
  const void* logits;
  long long ld;
  const void* index;          // int32 or int64
  long long ld_index;
  int index64;
  const float* teacher;
  long long ld_teacher;
  const float* row_weight;    // [rows] or null
  long long rows;
  int cols, top;
  float temperature;
  float weight;               // a factor of every row
  float* loss;                // [rows]
  void* grad;                 // null: not wanted
  long long ldg;
  float* partial;             // distill_partial_floats()
};

bool layer_norm_gradient_in_one(long long rows, int cols);   // one launch, which needs no partial sums
size_t layer_norm_partial_floats(long long rows, int cols);
void launch_layer_norm(const LayerNormArgs& a, int type, int wtype, hipStream_t s);
void launch_layer_norm_backward(const LayerNormGradArgs& a, int type, int wtype, hipStream_t s);
void launch_layer_norm_tangent(const LayerNormTangentArgs& a, hipStream_t s);
void launch_layer_norm_tangent_backward(const LayerNormTangentArgs& a, hipStream_t s);
void launch_quantize_rows(const QuantizeArgs& a, int type, hipStream_t s);
void launch_int8_matmul(const Int8Args& a, int out_type, hipStream_t s);
size_t int8_linear_bytes(long long m, int k);
bool int8_linear_in_one(const QuantizeArgs& q, const Int8Args& a, int type, int out_type);   // one launch, which needs no workspace
void launch_int8_linear(const QuantizeArgs& q, const Int8Args& a, int type, int out_type, void* workspace, hipStream_t s);
bool distill_temperature(float t);   // one that the kernels take
size_t distill_partial_floats(long long rows, int cols, int top);
void launch_distill(const DistillArgs& a, int type, hipStream_t s);
// grad[i] += more[i] (n values), *total = the sum of loss[0 .. rows)
void launch_distill_join(const float* more, float* grad, int n, const float* loss, int rows, float* total, hipStream_t s);

}  // namespace eg
