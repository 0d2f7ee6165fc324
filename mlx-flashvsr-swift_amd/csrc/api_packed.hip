// extern "C" entry points of the self-attention's training and serving path (declared in include/fvsr_lcsa.h, section f5):
// argument validation before any device work, then launches on the caller's stream. They allocate nothing and keep nothing.
#include <cmath>

#include "api.hpp"
#include "blocks8.hpp"
#include "packed_attn.hpp"

namespace fvsr {

int max_norm_channels();
int launch_rms_norm(int dtype, int param_dtype, const void* x, int64_t x_stride, const void* r, int64_t rows, int C, float eps,
                    const void* w, void* y, Out8 y8, void* s, float* rstd, hipStream_t stream);
int64_t rms_grad_blocks(int64_t rows, int C);
int launch_rms_norm_grad(int dtype, int param_dtype, const void* dy, const void* s, int64_t s_stride, const float* rstd,
                         const void* ds, int64_t rows, int C, const void* w, void* dx, float* dw, float* part,
                         hipStream_t stream);
int launch_rotary(int dtype, const fvsr_heads* q, const fvsr_heads* q_out, const fvsr_heads* k, const fvsr_heads* k_out,
                  int64_t tokens, int D, const void* pos, int pos64, const double* freq, int axes, const int32_t* axis_pairs,
                  int halves, int back, hipStream_t stream);

// a launch's workgroups times 1024 threads stay below 2^32
constexpr int64_t kMostRows = (int64_t)1 << 22;
constexpr int kMostHeads = 1 << 16;

static int check_row_count(int64_t rows, int channels) {
  const int64_t groups = channels <= 128 ? rows / 16 : channels <= 512 ? rows / 4 : rows;
  FVSR_REQUIRE(groups < kMostRows, FVSR_ERR_UNSUPPORTED, "too many rows for one launch");
  return FVSR_OK;
}

static int check_view(const fvsr_heads* x, const char* what) {
  FVSR_REQUIRE(x != nullptr, FVSR_ERR_INVALID_ARG, std::string(what) + " is NULL");
  FVSR_REQUIRE(x->heads > 0 && x->token_stride >= 0 && x->head_stride >= 0, FVSR_ERR_INVALID_ARG,
               std::string(what) + ": heads must be > 0 and strides >= 0");
  FVSR_REQUIRE(x->heads <= kMostHeads, FVSR_ERR_UNSUPPORTED, std::string(what) + ": at most 65536 heads");
  return FVSR_OK;
}

// an operand of the matrix cores' kernels
static int check_bf16_view(const fvsr_heads* x, const char* what, int heads, int64_t tokens) {
  if (const int rc = check_view(x, what)) return rc;
  FVSR_REQUIRE(x->heads == heads, FVSR_ERR_INVALID_ARG, std::string(what) + ": expected " + std::to_string(heads) + " heads");
  if (tokens == 0) return FVSR_OK;
  FVSR_REQUIRE(x->data && aligned(x->data, 16), FVSR_ERR_INVALID_ARG, std::string(what) + ": data must be non-NULL and 16-byte aligned");
  FVSR_REQUIRE(x->token_stride % 8 == 0 && x->head_stride % 8 == 0, FVSR_ERR_INVALID_ARG,
               std::string(what) + ": strides must be multiples of 8 elements");
  FVSR_REQUIRE(x->token_stride < (int64_t)1 << 23, FVSR_ERR_UNSUPPORTED, std::string(what) + ": token_stride must be below 2^23 elements");
  return FVSR_OK;
}

static int check_packed(const fvsr_ctx* ctx, const fvsr_packed* p) {
  FVSR_REQUIRE(ctx != nullptr, FVSR_ERR_INVALID_ARG, "ctx is NULL");
  FVSR_REQUIRE(p != nullptr, FVSR_ERR_INVALID_ARG, "the sequences are NULL");
  FVSR_REQUIRE(p->sequences > 0 && p->cu_q && p->cu_k, FVSR_ERR_INVALID_ARG,
               "at least one sequence, with offsets of queries and keys, is needed");
  FVSR_REQUIRE(p->tokens_q >= 0 && p->tokens_k >= 0, FVSR_ERR_INVALID_ARG, "tokens must be >= 0");
  FVSR_REQUIRE(p->tokens_q <= 0x7fffff00 && p->tokens_k <= 0x7fffff00, FVSR_ERR_UNSUPPORTED, "more tokens than 31-bit offsets hold");
  FVSR_REQUIRE(p->channels > 0 && p->channels % 8 == 0 && p->channels <= 128, FVSR_ERR_UNSUPPORTED,
               "channels of a head must be a multiple of 8, at most 128");
  FVSR_REQUIRE(std::isfinite(p->scale) && p->scale > 0.f, FVSR_ERR_INVALID_ARG, "scale must be positive and finite");
  FVSR_REQUIRE(p->scale >= 1e-30f && p->scale <= 1e30f, FVSR_ERR_UNSUPPORTED,
               "scale must be from 1e-30 to 1e30");   // lse / scale stays finite
  return FVSR_OK;
}

static int check_grid(const fvsr_packed* p, int64_t tokens, int heads) {
  FVSR_REQUIRE((tokens / 128 + p->sequences + 1) * heads < kMostRows, FVSR_ERR_UNSUPPORTED,
               "too many blocks of queries or keys for one launch");
  return FVSR_OK;
}

static PackedArgs args_of(const fvsr_packed* p, const fvsr_heads* q, const fvsr_heads* k, const fvsr_heads* v) {
  PackedArgs a{};
  auto in = [](const fvsr_heads* x) { return HeadView<const bf16>{(const bf16*)x->data, x->token_stride, x->head_stride}; };
  a.q = in(q);
  a.k = in(k);
  a.v = in(v);
  a.cu_q = p->cu_q;
  a.cu_k = p->cu_k;
  a.used_k = p->used_k;
  a.seqs = p->sequences;
  a.tq = (int)p->tokens_q;
  a.tk = (int)p->tokens_k;
  a.heads = q->heads;
  a.kv_heads = k->heads;
  a.group = q->heads / k->heads;
  a.D = p->channels;
  a.causal = p->causal ? 1 : 0;
  a.scale = p->scale;
  a.c = p->scale * 1.4426950408889634f;
  return a;
}
static HeadView<bf16> out_of(const fvsr_heads* x) { return HeadView<bf16>{(bf16*)x->data, x->token_stride, x->head_stride}; }

}  // namespace fvsr

using namespace fvsr;

extern "C" {

int fvsr_rms_norm(fvsr_ctx* ctx, int dtype, const void* x, int64_t x_stride, const void* residual, int64_t rows, int channels,
                  float eps, int param_dtype, const void* weight, void* y, void* y_codes, void* y_scales, void* sum, float* rstd,
                  void* stream) {
  int rc = check_rows(ctx, rows, channels, max_norm_channels());
  if (rc) return rc;
  if ((rc = check_params(dtype, param_dtype, weight, nullptr))) return rc;
  FVSR_REQUIRE(eps >= 0.f, FVSR_ERR_INVALID_ARG, "eps must be >= 0");
  FVSR_REQUIRE(x_stride >= channels, FVSR_ERR_INVALID_ARG, "x_stride must be at least the channels");
  if (rows == 0) return FVSR_OK;
  if ((rc = check_row_count(rows, channels))) return rc;
  FVSR_REQUIRE(x != nullptr, FVSR_ERR_INVALID_ARG, "x is NULL");
  FVSR_REQUIRE(y || y_codes, FVSR_ERR_INVALID_ARG, "y and y_codes are both NULL");
  if (y_codes && (rc = check_8(y_codes, y_scales, "y"))) return rc;
  FVSR_ON_DEVICE(ctx);
  return launch_rms_norm(dtype, param_dtype, x, x_stride, residual, rows, channels, eps, weight, y,
                         Out8{(uint8_t*)y_codes, (uint8_t*)y_scales}, sum, rstd, (hipStream_t)stream);
}

size_t fvsr_rms_norm_backward_workspace(int64_t rows, int channels) {
  const int64_t blocks = rows <= 0 || channels <= 0 ? 0 : rms_grad_blocks(rows, channels);
  return blocks > 1 ? (size_t)blocks * channels * sizeof(float) : 0;
}

int fvsr_rms_norm_backward(fvsr_ctx* ctx, int dtype, const void* dy, const void* s, int64_t s_stride, const float* rstd,
                           const void* dsum, int64_t rows, int channels, int param_dtype, const void* weight, void* dx,
                           float* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_rows(ctx, rows, channels, max_norm_channels());
  if (rc) return rc;
  if ((rc = check_params(dtype, param_dtype, weight, nullptr))) return rc;
  FVSR_REQUIRE(s_stride >= channels, FVSR_ERR_INVALID_ARG, "s_stride must be at least the channels");
  if (rows > 0) {
    FVSR_REQUIRE(dy && s && rstd && dx, FVSR_ERR_INVALID_ARG, "dy, s, rstd and dx must be non-NULL");
    const size_t need = dweight ? fvsr_rms_norm_backward_workspace(rows, channels) : 0;
    FVSR_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need),
                 FVSR_ERR_INVALID_ARG, "dweight needs a 16-byte aligned workspace of fvsr_rms_norm_backward_workspace bytes");
  }
  FVSR_ON_DEVICE(ctx);
  return launch_rms_norm_grad(dtype, param_dtype, dy, s, s_stride, rstd, dsum, rows, channels, weight, dx, dweight,
                              (float*)workspace, (hipStream_t)stream);
}

int fvsr_rotary(fvsr_ctx* ctx, int dtype, const fvsr_heads* q, const fvsr_heads* q_out, const fvsr_heads* k,
                const fvsr_heads* k_out, int64_t tokens, int channels, const void* positions, int positions64,
                const double* frequencies, int axes, const int32_t* axis_pairs, int halves, int back, void* stream) {
  FVSR_REQUIRE(ctx != nullptr, FVSR_ERR_INVALID_ARG, "ctx is NULL");
  FVSR_REQUIRE(dtype_ok(dtype), FVSR_ERR_INVALID_ARG, "dtype must be FVSR_DTYPE_F32 or FVSR_DTYPE_BF16");
  FVSR_REQUIRE(tokens >= 0 && channels > 0 && channels % 2 == 0, FVSR_ERR_INVALID_ARG, "tokens must be >= 0, channels even and > 0");
  FVSR_REQUIRE(tokens <= (int64_t)1 << 32 && channels <= 1024, FVSR_ERR_UNSUPPORTED, "at most 2^32 tokens of 1024 channels a head");
  FVSR_REQUIRE(axes >= 1 && axes <= 3 && axis_pairs, FVSR_ERR_INVALID_ARG, "1 to 3 axes, with the pairs of each, are needed");
  int64_t pairs = 0;
  for (int i = 0; i < axes; ++i) {
    FVSR_REQUIRE(axis_pairs[i] >= 0, FVSR_ERR_INVALID_ARG, "an axis' pairs must be >= 0");
    pairs += axis_pairs[i];
  }
  FVSR_REQUIRE(pairs >= 1 && 2 * pairs <= channels, FVSR_ERR_INVALID_ARG, "the axes' pairs must be 1 to channels / 2 together");
  int rc = check_view(q, "q");
  if (rc || (rc = check_view(q_out, "q_out"))) return rc;
  FVSR_REQUIRE((k == nullptr) == (k_out == nullptr), FVSR_ERR_INVALID_ARG, "k and k_out go together");
  if (k && ((rc = check_view(k, "k")) || (rc = check_view(k_out, "k_out")))) return rc;
  FVSR_REQUIRE(q->heads == q_out->heads && (!k || k->heads == k_out->heads), FVSR_ERR_INVALID_ARG, "an output has its input's heads");
  if (tokens == 0) return FVSR_OK;
  FVSR_REQUIRE(q->data && q_out->data && (!k || (k->data && k_out->data)), FVSR_ERR_INVALID_ARG, "data is NULL");
  FVSR_REQUIRE(positions && frequencies, FVSR_ERR_INVALID_ARG, "positions and frequencies must be non-NULL");
  FVSR_ON_DEVICE(ctx);
  return launch_rotary(dtype, q, q_out, k, k_out, tokens, channels, positions, positions64 ? 1 : 0, frequencies, axes, axis_pairs,
                       halves ? 1 : 0, back ? 1 : 0, (hipStream_t)stream);
}

size_t fvsr_packed_attention_workspace(const fvsr_packed* p, int heads, int kv_heads) {
  return !p || p->sequences <= 0 || p->tokens_q <= 0 || kv_heads <= 0 || heads < kv_heads
             ? 0
             : packed_forward_workspace(p->sequences, p->tokens_q, p->tokens_k, heads, kv_heads, p->channels);
}

int fvsr_packed_attention(fvsr_ctx* ctx, const fvsr_packed* p, const fvsr_heads* q, const fvsr_heads* k, const fvsr_heads* v,
                          const fvsr_heads* o, float* lse, int clear, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_packed(ctx, p);
  if (rc || (rc = check_view(q, "q")) || (rc = check_view(k, "k"))) return rc;
  FVSR_REQUIRE(q->heads % k->heads == 0, FVSR_ERR_INVALID_ARG, "q's heads must be a multiple of k's");
  if ((rc = check_bf16_view(q, "q", q->heads, p->tokens_q)) || (rc = check_bf16_view(k, "k", k->heads, p->tokens_k)) ||
      (rc = check_bf16_view(v, "v", k->heads, p->tokens_k)) || (rc = check_bf16_view(o, "o", q->heads, p->tokens_q)))
    return rc;
  if (p->tokens_q == 0) return FVSR_OK;
  if ((rc = check_grid(p, p->tokens_q, q->heads))) return rc;
  const size_t need = fvsr_packed_attention_workspace(p, q->heads, k->heads);
  FVSR_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), FVSR_ERR_INVALID_ARG,
               "a 16-byte aligned workspace of fvsr_packed_attention_workspace bytes is needed");
  FVSR_ON_DEVICE(ctx);
  PackedArgs a = args_of(p, q, k, v);
  a.o = out_of(o);
  a.lse = lse;
  a.clear = clear == FVSR_CLEAR_LSE ? 2 : clear ? 3 : 0;
  return launch_packed_forward(a, workspace, (hipStream_t)stream);
}

size_t fvsr_packed_attention_backward_workspace(const fvsr_packed* p, int heads, int kv_heads) {
  return !p || p->sequences <= 0 || p->tokens_q < 0 || p->tokens_k < 0 || kv_heads <= 0 || heads < kv_heads
             ? 0
             : packed_backward_workspace(p->sequences, p->tokens_q, p->tokens_k, heads, kv_heads, p->channels, p->causal != 0);
}

int fvsr_packed_attention_backward(fvsr_ctx* ctx, const fvsr_packed* p, const fvsr_heads* d_o, const fvsr_heads* q,
                                   const fvsr_heads* k, const fvsr_heads* v, const fvsr_heads* o, const float* lse,
                                   const fvsr_heads* dq, const fvsr_heads* dk, const fvsr_heads* dv, int clear, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  int rc = check_packed(ctx, p);
  if (rc || (rc = check_view(q, "q")) || (rc = check_view(k, "k"))) return rc;
  FVSR_REQUIRE(q->heads % k->heads == 0, FVSR_ERR_INVALID_ARG, "q's heads must be a multiple of k's");
  const int64_t tq = p->tokens_q, tk = p->tokens_k;
  if ((rc = check_bf16_view(d_o, "d_o", q->heads, tq)) || (rc = check_bf16_view(q, "q", q->heads, tq)) ||
      (rc = check_bf16_view(k, "k", k->heads, tk)) || (rc = check_bf16_view(v, "v", k->heads, tk)) ||
      (rc = check_bf16_view(o, "o", q->heads, tq)) || (rc = check_bf16_view(dq, "dq", q->heads, tq)) ||
      (rc = check_bf16_view(dk, "dk", k->heads, tk)) || (rc = check_bf16_view(dv, "dv", k->heads, tk)))
    return rc;
  if (tq == 0 && tk == 0) return FVSR_OK;
  if ((rc = check_grid(p, tq, q->heads)) || (rc = check_grid(p, tk, k->heads))) return rc;   // (parts only where blocks are few)
  FVSR_REQUIRE(lse || tq == 0, FVSR_ERR_INVALID_ARG, "lse is NULL");
  const size_t need = fvsr_packed_attention_backward_workspace(p, q->heads, k->heads);
  FVSR_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), FVSR_ERR_INVALID_ARG,
               "a 16-byte aligned workspace of fvsr_packed_attention_backward_workspace bytes is needed");
  FVSR_ON_DEVICE(ctx);
  PackedArgs a = args_of(p, q, k, v);
  a.d_o = HeadView<const bf16>{(const bf16*)d_o->data, d_o->token_stride, d_o->head_stride};
  a.o = out_of(o);
  a.dq = out_of(dq);
  a.dk = out_of(dk);
  a.dv = out_of(dv);
  a.lse = const_cast<float*>(lse);
  a.clear = clear ? 1 : 0;
  return launch_packed_backward(a, workspace, (hipStream_t)stream);
}

}  // extern "C"
