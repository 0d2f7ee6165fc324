// extern "C" entry points of the row operators and products with 8-bit operands (declared in include/fvsr_lcsa.h,
// section f4): argument validation before any device work, then launches on the caller's stream. They allocate nothing
// and keep nothing: what they need beside their operands is the caller's `workspace`, so calls on one context may
// overlap, on any streams, and may be captured into graphs.
#include "api.hpp"
#include "blocks8.hpp"

namespace fvsr {

int max_norm_channels();
int launch_layer_norm(int dtype, int param_dtype, const void* x, int64_t rows, int C, float eps, const void* w,
                      const void* b, void* y, Out8 y8, Out8 x8, float* stats, hipStream_t stream);
int64_t norm_grad_blocks(int64_t rows, int C);
int launch_layer_norm_grad(int dtype, int param_dtype, const void* dy, const void* x, In8 x8, const float* stats,
                           int64_t rows, int C, const void* w, void* dx, float* dw, float* db, float* part,
                           hipStream_t stream);
int launch_quantize(int dtype, const void* x, int64_t rows, int C, Out8 o, hipStream_t stream);
int launch_dequantize(In8 q, int64_t rows, int C, int dtype, void* out, hipStream_t stream);
size_t linear8_workspace(int64_t rows, int K, int N);
int launch_linear8(In8 x, int64_t rows, int K, In8 w, int N, int bias_dtype, const void* bias, int gelu, int out_dtype,
                   void* y, void* ws, hipStream_t stream);
size_t weight_grad_workspace(int64_t rows, int N, int K);
int launch_weight_grad(const void* dy, int64_t rows, int N, In8 x, int K, int out_dtype, void* dw, float* db, void* ws,
                       hipStream_t stream);

}  // namespace fvsr

using namespace fvsr;

extern "C" {

size_t fvsr_blocks8_code_bytes(int64_t rows, int channels) {
  return rows <= 0 || channels <= 0 ? 0 : (size_t)rows * runs_of(channels) * kRun;
}

size_t fvsr_blocks8_scale_bytes(int64_t rows, int channels) {
  return rows <= 0 || channels <= 0 ? 0 : (size_t)rows * scale_stride(channels);
}

int fvsr_quantize8(fvsr_ctx* ctx, int dtype, const void* x, int64_t rows, int channels, void* codes, void* scales,
                   void* stream) {
  int rc = check_rows(ctx, rows, channels, kMaxFeatures);
  if (rc) return rc;
  FVSR_REQUIRE(dtype_ok(dtype), FVSR_ERR_INVALID_ARG, "dtype must be FVSR_DTYPE_F32 or FVSR_DTYPE_BF16");
  if (rows == 0) return FVSR_OK;
  FVSR_REQUIRE(x != nullptr, FVSR_ERR_INVALID_ARG, "x is NULL");
  if ((rc = check_8(codes, scales, "quantize8"))) return rc;
  FVSR_ON_DEVICE(ctx);
  return launch_quantize(dtype, x, rows, channels, Out8{(uint8_t*)codes, (uint8_t*)scales}, (hipStream_t)stream);
}

int fvsr_dequantize8(fvsr_ctx* ctx, const void* codes, const void* scales, int64_t rows, int channels, int dtype, void* out,
                     void* stream) {
  int rc = check_rows(ctx, rows, channels, kMaxFeatures);
  if (rc) return rc;
  FVSR_REQUIRE(dtype_ok(dtype), FVSR_ERR_INVALID_ARG, "dtype must be FVSR_DTYPE_F32 or FVSR_DTYPE_BF16");
  if (rows == 0) return FVSR_OK;
  FVSR_REQUIRE(out != nullptr, FVSR_ERR_INVALID_ARG, "out is NULL");
  if ((rc = check_8(codes, scales, "dequantize8"))) return rc;
  FVSR_ON_DEVICE(ctx);
  return launch_dequantize(In8{(const uint8_t*)codes, (const uint8_t*)scales}, rows, channels, dtype, out,
                           (hipStream_t)stream);
}

int fvsr_layer_norm(fvsr_ctx* ctx, int dtype, const void* x, int64_t rows, int channels, float eps, int param_dtype,
                    const void* weight, const void* bias, void* y, void* y_codes, void* y_scales, void* x_codes,
                    void* x_scales, float* stats, void* stream) {
  int rc = check_rows(ctx, rows, channels, max_norm_channels());
  if (rc) return rc;
  if ((rc = check_params(dtype, param_dtype, weight, bias))) return rc;
  FVSR_REQUIRE(eps >= 0.f, FVSR_ERR_INVALID_ARG, "eps must be >= 0");
  if (rows == 0) return FVSR_OK;
  FVSR_REQUIRE(x != nullptr, FVSR_ERR_INVALID_ARG, "x is NULL");
  FVSR_REQUIRE(y || y_codes, FVSR_ERR_INVALID_ARG, "y and y_codes are both NULL");
  if (y_codes && (rc = check_8(y_codes, y_scales, "y"))) return rc;
  if (x_codes && (rc = check_8(x_codes, x_scales, "x"))) return rc;
  FVSR_ON_DEVICE(ctx);
  return launch_layer_norm(dtype, param_dtype, x, rows, channels, eps, weight, bias, y,
                           Out8{(uint8_t*)y_codes, (uint8_t*)y_scales}, Out8{(uint8_t*)x_codes, (uint8_t*)x_scales}, stats,
                           (hipStream_t)stream);
}

size_t fvsr_layer_norm_backward_workspace(int64_t rows, int channels) {
  return rows <= 0 || channels <= 0 ? 0 : (size_t)norm_grad_blocks(rows, channels) * 2 * channels * sizeof(float);
}

int fvsr_layer_norm_backward(fvsr_ctx* ctx, int dtype, const void* dy, const void* x, const void* x_codes,
                             const void* x_scales, const float* stats, int64_t rows, int channels, int param_dtype,
                             const void* weight, void* dx, float* dweight, float* dbias, void* workspace,
                             size_t workspace_bytes, void* stream) {
  int rc = check_rows(ctx, rows, channels, max_norm_channels());
  if (rc) return rc;
  if ((rc = check_params(dtype, param_dtype, weight, nullptr))) return rc;
  if (rows > 0) {
    FVSR_REQUIRE(dy && stats && dx, FVSR_ERR_INVALID_ARG, "dy, stats and dx must be non-NULL");
    FVSR_REQUIRE((x != nullptr) != (x_codes != nullptr), FVSR_ERR_INVALID_ARG, "give either x or x_codes");
    if (x_codes && (rc = check_8(x_codes, x_scales, "x"))) return rc;
    FVSR_REQUIRE((!dweight && !dbias) ||
                     (workspace && aligned(workspace, 16) &&
                      workspace_bytes >= fvsr_layer_norm_backward_workspace(rows, channels)),
                 FVSR_ERR_INVALID_ARG,
                 "dweight and dbias need a 16-byte aligned workspace of fvsr_layer_norm_backward_workspace bytes");
  }
  FVSR_ON_DEVICE(ctx);
  return launch_layer_norm_grad(dtype, param_dtype, dy, x, In8{(const uint8_t*)x_codes, (const uint8_t*)x_scales}, stats,
                                rows, channels, weight, dx, dweight, dbias, (float*)workspace, (hipStream_t)stream);
}

size_t fvsr_linear8_workspace(int64_t rows, int in_features, int out_features) {
  return rows <= 0 || in_features <= 0 || out_features <= 0 ? 0 : linear8_workspace(rows, in_features, out_features);
}

int fvsr_linear8(fvsr_ctx* ctx, int x_dtype, const void* x, int64_t rows, int in_features, void* x_codes, void* x_scales,
                 const void* w_codes, const void* w_scales, int out_features, int bias_dtype, const void* bias, int gelu,
                 int y_dtype, void* y, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_rows(ctx, rows, in_features, kMaxFeatures);
  if (rc) return rc;
  FVSR_REQUIRE(out_features > 0, FVSR_ERR_INVALID_ARG, "out_features must be > 0");
  FVSR_REQUIRE(out_features <= kMaxFeatures, FVSR_ERR_UNSUPPORTED, "at most " + std::to_string(kMaxFeatures) + " out_features");
  FVSR_REQUIRE(!x || dtype_ok(x_dtype), FVSR_ERR_INVALID_ARG, "x_dtype must be FVSR_DTYPE_F32 or FVSR_DTYPE_BF16");
  FVSR_REQUIRE(!bias || dtype_ok(bias_dtype), FVSR_ERR_INVALID_ARG, "bias_dtype must be FVSR_DTYPE_F32 or FVSR_DTYPE_BF16");
  FVSR_REQUIRE(dtype_ok(y_dtype), FVSR_ERR_INVALID_ARG, "y_dtype must be FVSR_DTYPE_F32 or FVSR_DTYPE_BF16");
  if (rows == 0) return FVSR_OK;
  FVSR_REQUIRE(y != nullptr, FVSR_ERR_INVALID_ARG, "y is NULL");
  if ((rc = check_8(x_codes, x_scales, "x"))) return rc;
  if ((rc = check_8(w_codes, w_scales, "weight"))) return rc;
  const size_t need = fvsr_linear8_workspace(rows, in_features, out_features);
  FVSR_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), FVSR_ERR_INVALID_ARG,
               "a 16-byte aligned workspace of fvsr_linear8_workspace bytes is needed");
  FVSR_ON_DEVICE(ctx);
  const Out8 q{(uint8_t*)x_codes, (uint8_t*)x_scales};
  if (x && (rc = launch_quantize(x_dtype, x, rows, in_features, q, (hipStream_t)stream))) return rc;
  return launch_linear8(In8{q.codes, q.scales}, rows, in_features, In8{(const uint8_t*)w_codes, (const uint8_t*)w_scales},
                        out_features, bias_dtype, bias, gelu ? 1 : 0, y_dtype, y, workspace, (hipStream_t)stream);
}

size_t fvsr_linear8_weight_grad_workspace(int64_t rows, int in_features, int out_features) {
  return rows < 0 || in_features <= 0 || out_features <= 0 ? 0 : weight_grad_workspace(rows, out_features, in_features);
}

int fvsr_linear8_weight_grad(fvsr_ctx* ctx, const void* dy, int64_t rows, int out_features, const void* x_codes,
                             const void* x_scales, int in_features, int dw_dtype, void* dw, float* db, void* workspace,
                             size_t workspace_bytes, void* stream) {
  int rc = check_rows(ctx, rows, in_features, kMaxFeatures);
  if (rc) return rc;
  FVSR_REQUIRE(out_features > 0, FVSR_ERR_INVALID_ARG, "out_features must be > 0");
  FVSR_REQUIRE(out_features <= kMaxFeatures, FVSR_ERR_UNSUPPORTED, "at most " + std::to_string(kMaxFeatures) + " out_features");
  FVSR_REQUIRE(dtype_ok(dw_dtype), FVSR_ERR_INVALID_ARG, "dw_dtype must be FVSR_DTYPE_F32 or FVSR_DTYPE_BF16");
  FVSR_REQUIRE(dw != nullptr, FVSR_ERR_INVALID_ARG, "dw is NULL");
  if (rows > 0) {
    FVSR_REQUIRE(dy != nullptr, FVSR_ERR_INVALID_ARG, "dy is NULL");
    FVSR_REQUIRE(out_features % 8 != 0 || aligned(dy, 16), FVSR_ERR_INVALID_ARG,
                 "dy must be 16-byte aligned where out_features is a multiple of 8");
    if ((rc = check_8(x_codes, x_scales, "x"))) return rc;
  }
  const size_t need = fvsr_linear8_weight_grad_workspace(rows, in_features, out_features);
  FVSR_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), FVSR_ERR_INVALID_ARG,
               "a 16-byte aligned workspace of fvsr_linear8_weight_grad_workspace bytes is needed");
  FVSR_ON_DEVICE(ctx);
  return launch_weight_grad(dy, rows, out_features, In8{(const uint8_t*)x_codes, (const uint8_t*)x_scales}, in_features,
                            dw_dtype, dw, db, workspace, (hipStream_t)stream);
}

}  // extern "C"
