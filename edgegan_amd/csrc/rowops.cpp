// C entries of the row operators (include/edgegan_hip.h): argument checks, the device, error codes.
#include <cmath>
#include <initializer_list>

#include "../../include/edgegan_hip.h"
#include "common.h"
#include "kernels.h"
#include "rowops.h"

using namespace eg;

void eg_set_global_error(const char* what);   // capi.cpp: eg_last_error(NULL)

namespace {

// the operands' device, current for the length of a call
struct OnDevice {
  int before = -1;
  explicit OnDevice(int device) {
    int now = -1, count = 0;
    EG_HIP(hipGetDevice(&now));
    if (now == device) return;
    EG_HIP(hipGetDeviceCount(&count));
    EG_CHECK(device >= 0 && device < count, "device %d of %d", device, count);
    EG_HIP(hipSetDevice(device));
    before = now;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

int type_of(int t, const char* what) {
  EG_CHECK(t == EG_F32 || t == EG_BF16 || t == EG_F16, "%s: unknown element type %d", what, t);
  return t;
}
constexpr long long kMaxCols = 1 << 24;   // (32-bit sums of more elements than 2^24 stop to be sums)
void check_rows(const char* what, long long rows, long long cols) {
  EG_CHECK(rows >= 0 && cols >= 0 && cols <= kMaxCols, "%s: %lld rows of %lld columns (columns: 0 .. 2^24)", what, rows, cols);
}
void check_matrix(const char* what, const void* p, long long ld, long long rows, long long cols, int elem) {
  if (rows == 0 || cols == 0) return;
  EG_CHECK(p, "%s: null pointer", what);
  EG_CHECK(ld >= cols || rows == 1, "%s: rows %lld elements apart hold %lld columns", what, ld, cols);
  EG_CHECK(ld >= 0 && (rows == 1 || ld <= (1ll << 62) / rows / elem), "%s: too large", what);
  EG_CHECK((uintptr_t)p % elem == 0, "%s: misaligned for its type", what);
}
void check_parameters(const char* what, int dtype, int wtype, const void* gamma, const void* beta) {
  type_of(wtype, what);
  EG_CHECK(wtype == dtype || wtype == EG_F32, "%s: gamma and beta of the rows' type or f32, not %d beside %d", what, wtype, dtype);
  const uintptr_t e = wtype == EG_F32 ? 4 : 2;
  EG_CHECK((uintptr_t)gamma % e == 0 && (uintptr_t)beta % e == 0, "%s: gamma or beta misaligned for its type", what);
}
void check_floats(const char* what, std::initializer_list<const float*> v) {
  for (const float* p : v) EG_CHECK((uintptr_t)p % 4 == 0, "%s: a vector of f32 is misaligned", what);
}
void check_act(int act) { EG_CHECK(act == EG_ACT_NONE || act == EG_ACT_RELU || act == EG_ACT_LRELU, "unknown activation %d", act); }
void check_eps(float eps) { EG_CHECK(eps > 0.f && std::isfinite(eps), "eps must be positive and finite"); }
int bytes_of(int type) { return type == EG_F32 ? 4 : 2; }
void check_workspace(const char* what, const void* p, long long have, size_t floats) {
  EG_CHECK(floats == 0 || (p && have >= 0 && (size_t)have >= floats * 4 && (uintptr_t)p % 16 == 0),
           "%s: the workspace needs %zu bytes at a multiple of 16", what, floats * 4);
}

template <typename F>
int entry(F f) {
  try {
    f();
    return 0;
  } catch (const eg::Error& e) {
    if (e.code == 2) (void)hipGetLastError();   // (reported here: the caller's next check is not to find it again)
    eg_set_global_error(e.what());
    return e.code;
  } catch (const std::exception& e) {
    eg_set_global_error(e.what());
    return 99;
  }
}

}  // namespace

extern "C" {

int eg_layer_norm(int device, void* stream, int dtype, const void* x, long long ldx, int wtype, const void* gamma, const void* beta, long long rows,
                  long long cols, float eps, int act, void* y, long long ldy, float* mean, float* rstd) {
  return entry([&] {
    type_of(dtype, "eg_layer_norm");
    check_parameters("eg_layer_norm", dtype, wtype, gamma, beta);
    check_floats("eg_layer_norm", {mean, rstd});
    check_rows("eg_layer_norm", rows, cols);
    check_matrix("eg_layer_norm x", x, ldx, rows, cols, bytes_of(dtype));
    check_matrix("eg_layer_norm y", y, ldy, rows, cols, bytes_of(dtype));
    check_act(act);
    check_eps(eps);
    EG_CHECK(!mean == !rstd, "eg_layer_norm: mean and rstd go together");
    if (rows == 0) return;
    EG_CHECK(cols > 0, "eg_layer_norm: rows without columns have no mean");
    OnDevice on(device);
    launch_layer_norm({x, ldx, gamma, beta, rows, (int)cols, eps, act, y, ldy, mean, rstd}, dtype, wtype, (hipStream_t)stream);
  });
}

long long eg_layer_norm_workspace(long long rows, long long cols) {
  if (rows < 0 || cols < 0 || cols > kMaxCols) return -1;
  return layer_norm_gradient_in_one(rows, (int)cols) ? 0 : (long long)layer_norm_partial_floats(rows, (int)cols) * 4;
}

int eg_layer_norm_backward(int device, void* stream, int dtype, const void* dy, long long lddy, const void* x, long long ldx, const float* mean,
                           const float* rstd, int wtype, const void* gamma, const void* beta, long long rows, long long cols, int act, void* dx,
                           long long lddx, void* dgamma, void* dbeta, void* workspace, long long workspace_bytes) {
  return entry([&] {
    type_of(dtype, "eg_layer_norm_backward");
    check_parameters("eg_layer_norm_backward", dtype, wtype, gamma, beta);
    check_parameters("eg_layer_norm_backward gradients", dtype, wtype, dgamma, dbeta);
    check_floats("eg_layer_norm_backward", {mean, rstd});
    check_rows("eg_layer_norm_backward", rows, cols);
    const int e = bytes_of(dtype);
    check_matrix("eg_layer_norm_backward dy", dy, lddy, rows, cols, e);
    check_matrix("eg_layer_norm_backward x", x, ldx, rows, cols, e);
    if (dx) check_matrix("eg_layer_norm_backward dx", dx, lddx, rows, cols, e);
    check_act(act);
    EG_CHECK(rows == 0 || (mean && rstd), "eg_layer_norm_backward: null statistics");
    if ((dgamma || dbeta) && (workspace_bytes || !layer_norm_gradient_in_one(rows, (int)cols)))
      check_workspace("eg_layer_norm_backward", workspace, workspace_bytes, layer_norm_partial_floats(rows, (int)cols));
    if (cols == 0) {
      EG_CHECK(rows == 0, "eg_layer_norm_backward: rows without columns have no mean");
      return;
    }
    OnDevice on(device);
    launch_layer_norm_backward({dy, x, lddy, ldx, mean, rstd, gamma, beta, rows, (int)cols, act, kLreluAtZero, dx, lddx, 0, dgamma, dbeta, 0, (float*)workspace}, dtype,
                               wtype, (hipStream_t)stream);
  });
}

int eg_quantize_rows(int device, void* stream, int dtype, const void* x, long long ldx, int norm, const float* gamma, const float* beta, float eps,
                     long long rows, long long cols, signed char* q, long long ldq, float* scale) {
  return entry([&] {
    type_of(dtype, "eg_quantize_rows");
    check_rows("eg_quantize_rows", rows, cols);
    check_matrix("eg_quantize_rows x", x, ldx, rows, cols, bytes_of(dtype));
    check_matrix("eg_quantize_rows q", q, ldq, rows, cols, 1);
    check_floats("eg_quantize_rows", {gamma, beta, scale});
    EG_CHECK(norm || (!gamma && !beta), "eg_quantize_rows: gamma and beta belong to the norm");
    if (norm) check_eps(eps);
    if (rows == 0) return;
    EG_CHECK(scale, "eg_quantize_rows: null scale");
    EG_CHECK(cols > 0, "eg_quantize_rows: rows without columns");
    OnDevice on(device);
    launch_quantize_rows({x, ldx, gamma, beta, norm != 0, eps, rows, (int)cols, q, ldq, scale}, dtype, (hipStream_t)stream);
  });
}

static void check_product(long long m, long long n, long long k) {
  EG_CHECK(m >= 0 && n >= 0 && k >= 0 && n < (1ll << 30), "int8 product: bad sizes %lld x %lld x %lld", m, n, k);
  EG_CHECK(k <= 131071, "int8 product: %lld terms can overflow a 32-bit sum (at most 131071)", k);
}

int eg_int8_matmul(int device, void* stream, const signed char* a, long long lda, const float* a_scale, const signed char* b, long long ldb,
                   const float* b_scale, const float* bias, long long m, long long n, long long k, int out_type, void* out, long long ldo) {
  return entry([&] {
    type_of(out_type, "eg_int8_matmul");
    check_product(m, n, k);
    check_matrix("eg_int8_matmul a", a, lda, m, k, 1);
    check_matrix("eg_int8_matmul b", b, ldb, n, k, 1);
    check_matrix("eg_int8_matmul out", out, ldo, m, n, bytes_of(out_type));
    if (m == 0 || n == 0) return;
    EG_CHECK(a_scale && b_scale, "eg_int8_matmul: null scale");
    check_floats("eg_int8_matmul", {a_scale, b_scale, bias});
    OnDevice on(device);
    launch_int8_matmul({a, lda, a_scale, b, ldb, b_scale, bias, m, (int)n, (int)k, out, ldo}, out_type, (hipStream_t)stream);
  });
}

long long eg_int8_linear_workspace(long long rows, long long inner) {
  if (rows < 0 || inner < 0 || inner > 131071) return -1;
  return (long long)int8_linear_bytes(rows, (int)inner);
}

int eg_int8_linear(int device, void* stream, int dtype, const void* x, long long ldx, int norm, const float* gamma, const float* beta, float eps,
                   const signed char* weight, long long ldw, const float* weight_scale, const float* bias, long long rows, long long cols, long long inner,
                   int out_type, void* out, long long ldo, void* workspace, long long workspace_bytes) {
  return entry([&] {
    type_of(dtype, "eg_int8_linear");
    type_of(out_type, "eg_int8_linear");
    check_product(rows, cols, inner);
    check_matrix("eg_int8_linear x", x, ldx, rows, inner, bytes_of(dtype));
    check_matrix("eg_int8_linear weight", weight, ldw, cols, inner, 1);
    check_matrix("eg_int8_linear out", out, ldo, rows, cols, bytes_of(out_type));
    EG_CHECK(norm || (!gamma && !beta), "eg_int8_linear: gamma and beta belong to the norm");
    if (norm) check_eps(eps);
    if (rows == 0 || cols == 0) return;
    EG_CHECK(inner > 0, "eg_int8_linear: rows without columns");
    EG_CHECK(weight_scale, "eg_int8_linear: null scale");
    check_floats("eg_int8_linear", {gamma, beta, weight_scale, bias});
    const QuantizeArgs q{x, ldx, gamma, beta, norm != 0, eps, rows, (int)inner, nullptr, 0, nullptr};
    const Int8Args a{nullptr, 0, nullptr, weight, ldw, weight_scale, bias, rows, (int)cols, (int)inner, out, ldo};
    if (workspace_bytes || !int8_linear_in_one(q, a, dtype, out_type))
      check_workspace("eg_int8_linear", workspace, workspace_bytes, int8_linear_bytes(rows, (int)inner) / 4);
    OnDevice on(device);
    launch_int8_linear(q, a, dtype, out_type, workspace, (hipStream_t)stream);
  });
}

int eg_int8_linear_in_one(int dtype, const void* x, long long ldx, int norm, const float* gamma, const float* beta, const signed char* weight, long long ldw,
                          long long rows, long long cols, long long inner, int out_type, long long ldo) {
  if (dtype < 0 || dtype > ROW_F16 || rows < 0 || cols < 0 || cols > INT_MAX || inner < 1 || inner > 131071) return 0;
  return int8_linear_in_one({x, ldx, gamma, beta, norm != 0, 1.f, rows, (int)inner, nullptr, 0, nullptr},
                            {nullptr, 0, nullptr, weight, ldw, nullptr, nullptr, rows, (int)cols, (int)inner, nullptr, ldo}, dtype, out_type);
}

long long eg_distill_loss_workspace(long long rows, long long cols, long long top) {
  if (rows < 0 || cols < 0 || cols > kMaxCols || top < 0 || top > 1024) return -1;
  return (long long)distill_partial_floats(rows, (int)cols, (int)top) * 4;
}

int eg_distill_loss(int device, void* stream, int dtype, const void* logits, long long ld, int index_bytes, const void* index, long long ld_index,
                    const float* teacher, long long ld_teacher, const float* row_weight, long long rows, long long cols, long long top,
                    float temperature, float* loss, void* grad, long long ldg, void* workspace, long long workspace_bytes) {
  return entry([&] {
    type_of(dtype, "eg_distill_loss");
    check_rows("eg_distill_loss", rows, cols);
    check_matrix("eg_distill_loss logits", logits, ld, rows, cols, bytes_of(dtype));
    if (grad) check_matrix("eg_distill_loss grad", grad, ldg, rows, cols, bytes_of(dtype));
    EG_CHECK(index_bytes == 4 || index_bytes == 8, "eg_distill_loss: indexes of 4 or 8 bytes, not %d", index_bytes);
    EG_CHECK(top >= 0 && top <= 1024, "eg_distill_loss: %lld teacher logits a row (0 .. 1024)", top);
    check_matrix("eg_distill_loss index", index, ld_index, rows, top, index_bytes);
    check_matrix("eg_distill_loss teacher", teacher, ld_teacher, rows, top, 4);
    EG_CHECK(distill_temperature(temperature), "eg_distill_loss: the temperature must be positive and finite, and log2(e) / temperature finite");
    if (rows == 0) return;
    EG_CHECK(loss, "eg_distill_loss: null loss");
    check_floats("eg_distill_loss", {row_weight, loss});
    EG_CHECK(cols > 0, "eg_distill_loss: rows without columns");
    check_workspace("eg_distill_loss", workspace, workspace_bytes, distill_partial_floats(rows, (int)cols, (int)top));
    OnDevice on(device);
    launch_distill({logits, ld, index, ld_index, index_bytes == 8, teacher, ld_teacher, row_weight, rows, (int)cols, (int)top, temperature, 1.f, loss, grad, ldg,
                    (float*)workspace},
                   dtype, (hipStream_t)stream);
  });
}

}  // extern "C"
