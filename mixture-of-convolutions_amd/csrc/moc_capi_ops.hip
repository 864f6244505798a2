// C ABI of the operators that stand next to the MoC layers: layer norm, causal
// convolution, selective scan (declared in include/moc_hip.h).  Argument checks and
// dispatch; no exception leaves an entry (nothing here allocates or throws).
#include <hip/hip_runtime.h>

#include "../../include/moc_hip.h"
#include "moc_kernels.h"

namespace {

using moc::clear_error;
using moc::fail;

bool any_dt(int dt) { return dt == MOC_DT_F32 || dt == MOC_DT_BF16 || dt == MOC_DT_F16; }
bool x_dt_ok(int dt) { return dt == MOC_DT_F32 || dt == MOC_DT_BF16; }

constexpr int64_t kMaxTokens = int64_t(1) << 31;
constexpr int64_t kMaxStride = int64_t(1) << 31;  // elements between tokens
// a grid counts threads in 32 bits: workgroups of 256 threads, and chunks of a scan that is
// differentiated, whose backward has workgroups of 512
constexpr int64_t kMaxWorkgroups = int64_t(1) << 24, kMaxSavedChunks = int64_t(1) << 23;

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MOC_OK : fail(MOC_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

int check_space(size_t need, const void* ws, size_t got) {
  if (got < need || (need > 0 && ws == nullptr))
    return fail(MOC_ERR_WORKSPACE, "workspace too small: need %zu bytes, got %zu", need, got);
  return MOC_OK;
}

// ---------------------------------------------------------------------------
int check_norm(int64_t rows, int64_t dim, int x_dt, int w_dt, int b_dt) {
  if (rows <= 0 || dim <= 0)
    return fail(MOC_ERR_ARG, "rows and dim must be positive (got %lld, %lld)", (long long)rows, (long long)dim);
  if (rows >= kMaxTokens || dim >= kMaxTokens)
    return fail(MOC_ERR_ARG, "rows or dim too large: %lld, %lld", (long long)rows, (long long)dim);
  if (!x_dt_ok(x_dt)) return fail(MOC_ERR_DTYPE, "unsupported x dtype code %d (bf16 or f32 only)", x_dt);
  if (!any_dt(w_dt) || !any_dt(b_dt)) return fail(MOC_ERR_DTYPE, "unsupported weight or bias dtype code");
  return MOC_OK;
}

// ---------------------------------------------------------------------------
int check_seq(const void* cu, int64_t n_seqs, int64_t n_tokens, int64_t seq_len) {
  if (n_tokens <= 0 || n_tokens >= kMaxTokens)
    return fail(MOC_ERR_ARG, "n_tokens must be in [1, 2^31), got %lld", (long long)n_tokens);
  if (cu == nullptr) {
    if (seq_len <= 0 || n_tokens % seq_len != 0)
      return fail(MOC_ERR_ARG, "seq_len must be positive and divide n_tokens for fixed-length inputs");
  } else if (n_seqs <= 0 || n_seqs >= kMaxTokens) {
    return fail(MOC_ERR_ARG, "n_seqs must be positive when cu_seqlens is given");
  }
  return MOC_OK;
}

moc::SeqLayout layout(const void* cu, int cu64, int64_t n_seqs, int64_t n_tokens, int64_t seq_len) {
  moc::SeqLayout s;
  s.cu = cu;
  s.cu64 = cu64 ? 1 : 0;
  s.n_seqs = n_seqs;
  s.seq_len = seq_len;
  s.n_tokens = n_tokens;
  return s;
}

int check_conv(int64_t dim, int64_t ks, int x_dt, int w_dt, int b_dt, int activation) {
  // (a lane has two channels at least, so that 2^31 of them would take a grid of 2^32 threads)
  if (dim <= 0 || dim >= kMaxTokens / 2)
    return fail(MOC_ERR_ARG, "dim must be in [1, 2^30), got %lld", (long long)dim);
  if (ks < 1 || ks > moc::kConvMaxS)
    return fail(MOC_ERR_ARG, "kernel_size must be in [1, %d], got %lld", moc::kConvMaxS, (long long)ks);
  if (!x_dt_ok(x_dt)) return fail(MOC_ERR_DTYPE, "unsupported x dtype code %d (bf16 or f32 only)", x_dt);
  if (!any_dt(w_dt) || !any_dt(b_dt)) return fail(MOC_ERR_DTYPE, "unsupported weight or bias dtype code");
  if (activation != 0 && activation != 1) return fail(MOC_ERR_ARG, "activation must be 0 or 1, got %d", activation);
  return MOC_OK;
}

// ---------------------------------------------------------------------------
enum class Use { kStep, kForward, kSaved };  // (kSaved: the forward for a backward, and that)
int check_scan(const MocScan* s, Use use) {
  if (s == nullptr) return fail(MOC_ERR_ARG, "null scan");
  if (!s->x || !s->dt || !s->a || !s->b || !s->c) return fail(MOC_ERR_ARG, "null tensor pointer");
  if (s->heads <= 0 || s->head_dim <= 0 || s->groups <= 0 || s->state_dim <= 0 || s->heads % s->groups != 0)
    return fail(MOC_ERR_ARG, "heads, head_dim, groups and state_dim must be positive, groups a divisor of heads "
                             "(got %lld, %lld, %lld, %lld)",
                (long long)s->heads, (long long)s->head_dim, (long long)s->groups, (long long)s->state_dim);
  if (s->head_dim > moc::kScanMaxP || s->state_dim > moc::kScanMaxN)
    return fail(MOC_ERR_ARG, "head_dim must be at most %d and state_dim at most %d, got %lld and %lld", moc::kScanMaxP,
                moc::kScanMaxN, (long long)s->head_dim, (long long)s->state_dim);
  if (s->heads > 32767) return fail(MOC_ERR_ARG, "too many heads: %lld", (long long)s->heads);
  if (!x_dt_ok(s->x_dtype)) return fail(MOC_ERR_DTYPE, "unsupported x dtype code %d (bf16 or f32 only)", s->x_dtype);
  if (!any_dt(s->a_dtype) || !any_dt(s->d_dtype) || !any_dt(s->bias_dtype))
    return fail(MOC_ERR_DTYPE, "unsupported A, D or dt_bias dtype code");
  if (s->dt_softplus != 0 && s->dt_softplus != 1)
    return fail(MOC_ERR_ARG, "dt_softplus must be 0 or 1, got %d", s->dt_softplus);
  const int64_t xs = s->heads * s->head_dim, bs = s->groups * s->state_dim;
  if (s->n_tokens > 1 && (s->x_stride < xs || s->dt_stride < s->heads || s->b_stride < bs || s->c_stride < bs))
    return fail(MOC_ERR_ARG, "token strides must hold a token's values");
  if (s->n_tokens > 1 && (s->x_stride >= kMaxStride || s->dt_stride >= kMaxStride || s->b_stride >= kMaxStride ||
                          s->c_stride >= kMaxStride))
    return fail(MOC_ERR_ARG, "token strides must be below 2^31 elements");
  if (int rc = check_seq(s->cu_seqlens, s->n_seqs, s->n_tokens, s->seq_len)) return rc;
  if (use == Use::kStep) {
    if (s->cu_seqlens != nullptr || s->seq_len != 1) return fail(MOC_ERR_ARG, "a step has one token per sequence");
    if (s->n_tokens * s->heads >= kMaxWorkgroups) return fail(MOC_ERR_ARG, "too many sequences and heads for a step");
  } else if (s->n_tokens / 64 + (s->cu_seqlens != nullptr ? s->n_seqs + 2 : s->n_tokens / s->seq_len) >=
             (use == Use::kSaved ? kMaxSavedChunks : kMaxWorkgroups)) {
    return fail(MOC_ERR_ARG, "too many chunks of 64 tokens");
  }
  return MOC_OK;
}

moc::Scan problem(const MocScan* s) {
  moc::Scan p;
  p.seq = layout(s->cu_seqlens, s->cu_seqlens_i64, s->n_seqs, s->n_tokens, s->seq_len);
  p.H = s->heads;
  p.P = s->head_dim;
  p.G = s->groups;
  p.N = s->state_dim;
  p.x = s->x;
  p.dt = s->dt;
  p.A = s->a;
  p.B = s->b;
  p.C = s->c;
  p.D = s->d;
  p.bias = s->dt_bias;
  // (a single token's strides say nothing)
  const bool one = s->n_tokens == 1;
  p.x_stride = one ? s->heads * s->head_dim : s->x_stride;
  p.dt_stride = one ? s->heads : s->dt_stride;
  p.b_stride = one ? s->groups * s->state_dim : s->b_stride;
  p.c_stride = one ? s->groups * s->state_dim : s->c_stride;
  p.x_dt = s->x_dtype;
  p.a_dt = s->a_dtype;
  p.d_dt = s->d_dtype;
  p.bias_dt = s->bias_dtype;
  p.softplus = s->dt_softplus;
  return p;
}

int check_states(const MocScan* s, const void* a, const void* b) {
  if ((a != nullptr || b != nullptr) && s->cu_seqlens != nullptr)
    return fail(MOC_ERR_ARG, "states are only supported for fixed-length inputs");
  // (one workgroup reads the first while another writes the last)
  if (a != nullptr && a == b) return fail(MOC_ERR_ARG, "the state read and the state written must not be the same tensor");
  return MOC_OK;
}

}  // namespace

extern "C" {

int moc_norm_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                     int64_t rows, int64_t dim, int x_dtype, int weight_dtype, int bias_dtype, float eps,
                     void* stream) {
  clear_error();
  if (int rc = check_norm(rows, dim, x_dtype, weight_dtype, bias_dtype)) return rc;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return fail(MOC_ERR_ARG, "null tensor pointer");
  moc::norm_forward(x, weight, bias, y, mean, rstd, rows, dim, x_dtype, weight_dtype, bias_dtype, eps,
                    static_cast<hipStream_t>(stream));
  return launched("moc_norm_forward launch");
}

size_t moc_norm_backward_workspace_bytes(int64_t rows, int64_t dim) {
  return rows <= 0 || dim <= 0 ? 0 : moc::norm_backward_workspace(rows, dim);
}

int moc_norm_backward(const void* x, const void* weight, const void* dy, const float* mean, const float* rstd,
                      void* dx, void* dweight, void* dbias, int64_t rows, int64_t dim, int x_dtype, int weight_dtype,
                      int bias_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_norm(rows, dim, x_dtype, weight_dtype, bias_dtype)) return rc;
  if (!x || !dy || !mean || !rstd) return fail(MOC_ERR_ARG, "null tensor pointer");
  if (dweight != nullptr || dbias != nullptr)
    if (int rc = check_space(moc::norm_backward_workspace(rows, dim), workspace, workspace_bytes)) return rc;
  moc::norm_backward(x, weight, dy, mean, rstd, dx, dweight, dbias, rows, dim, x_dtype, weight_dtype, bias_dtype,
                     workspace, static_cast<hipStream_t>(stream));
  return launched("moc_norm_backward launch");
}

int moc_conv_forward(const void* x, const void* weight, const void* bias, const void* cache, void* y,
                     void* final_state, const void* cu_seqlens, int cu_seqlens_i64, int64_t n_seqs, int64_t n_tokens,
                     int64_t seq_len, int64_t dim, int64_t kernel_size, int x_dtype, int weight_dtype, int bias_dtype,
                     int activation, void* stream) {
  clear_error();
  if (int rc = check_conv(dim, kernel_size, x_dtype, weight_dtype, bias_dtype, activation)) return rc;
  if (int rc = check_seq(cu_seqlens, n_seqs, n_tokens, seq_len)) return rc;
  if (!x || !weight || !y) return fail(MOC_ERR_ARG, "null tensor pointer");
  if ((cache != nullptr || final_state != nullptr) && cu_seqlens != nullptr)
    return fail(MOC_ERR_ARG, "states are only supported for fixed-length inputs");
  if (cache != nullptr && cache == final_state)
    return fail(MOC_ERR_ARG, "the cache read and the final state written must not be the same tensor");
  const moc::Conv p{layout(cu_seqlens, cu_seqlens_i64, n_seqs, n_tokens, seq_len), dim, kernel_size, x_dtype,
                    weight_dtype, bias_dtype, activation};
  moc::conv_forward(p, x, weight, bias, cache, y, final_state, static_cast<hipStream_t>(stream));
  return launched("moc_conv_forward launch");
}

size_t moc_conv_backward_workspace_bytes(int64_t n_tokens, int64_t dim, int64_t kernel_size, int x_dtype) {
  if (n_tokens <= 0 || dim <= 0 || kernel_size <= 0) return 0;
  return moc::conv_backward_workspace({layout(nullptr, 0, 0, n_tokens, n_tokens), dim, kernel_size, x_dtype, 0, 0, 0});
}

int moc_conv_backward(const void* x, const void* weight, const void* bias, const void* dy, void* dx, void* dweight,
                      void* dbias, const void* cu_seqlens, int cu_seqlens_i64, int64_t n_seqs, int64_t n_tokens,
                      int64_t seq_len, int64_t dim, int64_t kernel_size, int x_dtype, int weight_dtype,
                      int bias_dtype, int activation, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_conv(dim, kernel_size, x_dtype, weight_dtype, bias_dtype, activation)) return rc;
  if (int rc = check_seq(cu_seqlens, n_seqs, n_tokens, seq_len)) return rc;
  if (!x || !weight || !dy) return fail(MOC_ERR_ARG, "null tensor pointer");
  const moc::Conv p{layout(cu_seqlens, cu_seqlens_i64, n_seqs, n_tokens, seq_len), dim, kernel_size, x_dtype,
                    weight_dtype, bias_dtype, activation};
  if (dweight != nullptr || dbias != nullptr)
    if (int rc = check_space(moc::conv_backward_workspace(p), workspace, workspace_bytes)) return rc;
  moc::conv_backward(p, x, weight, bias, dy, dx, dweight, dbias, workspace, static_cast<hipStream_t>(stream));
  return launched("moc_conv_backward launch");
}

int moc_conv_update(const void* x, const void* weight, const void* bias, void* cache, int64_t cache_stride_b,
                    int64_t cache_stride_d, int64_t cache_stride_s, void* y, int64_t batch, int64_t dim,
                    int64_t kernel_size, int x_dtype, int weight_dtype, int bias_dtype, int activation, void* stream) {
  clear_error();
  if (int rc = check_conv(dim, kernel_size, x_dtype, weight_dtype, bias_dtype, activation)) return rc;
  if (batch <= 0 || batch >= kMaxTokens) return fail(MOC_ERR_ARG, "batch must be positive, got %lld", (long long)batch);
  if (!x || !weight || !cache || !y) return fail(MOC_ERR_ARG, "null tensor pointer");
  moc::conv_update(x, weight, bias, cache, cache_stride_b, cache_stride_d, cache_stride_s, y, batch, dim, kernel_size,
                   x_dtype, weight_dtype, bias_dtype, activation, static_cast<hipStream_t>(stream));
  return launched("moc_conv_update launch");
}

size_t moc_scan_saved_bytes(const MocScan* s) {
  clear_error();
  return check_scan(s, Use::kSaved) != MOC_OK ? 0 : moc::scan_saved_bytes(problem(s));
}

size_t moc_scan_forward_workspace_bytes(const MocScan* s, int with_saved) {
  clear_error();
  return check_scan(s, with_saved != 0 ? Use::kSaved : Use::kForward) != MOC_OK
             ? 0
             : moc::scan_forward_workspace(problem(s), with_saved != 0);
}

int moc_scan_forward(const MocScan* s, void* y, const float* initial_state, float* final_state, void* saved,
                     size_t saved_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_scan(s, saved != nullptr ? Use::kSaved : Use::kForward)) return rc;
  if (!y) return fail(MOC_ERR_ARG, "null tensor pointer");
  if (int rc = check_states(s, initial_state, final_state)) return rc;
  const moc::Scan p = problem(s);
  if (saved != nullptr)
    if (int rc = check_space(moc::scan_saved_bytes(p), saved, saved_bytes)) return rc;
  if (int rc = check_space(moc::scan_forward_workspace(p, saved != nullptr), workspace, workspace_bytes)) return rc;
  moc::scan_forward(p, y, initial_state, final_state, saved, workspace, static_cast<hipStream_t>(stream));
  return launched("moc_scan_forward launch");
}

size_t moc_scan_backward_workspace_bytes(const MocScan* s) {
  clear_error();
  return check_scan(s, Use::kSaved) != MOC_OK ? 0 : moc::scan_backward_workspace(problem(s));
}

int moc_scan_backward(const MocScan* s, const void* dy, int has_initial_state, const float* dfinal_state,
                      const void* saved, size_t saved_bytes, const MocScanGrads* grads, void* workspace,
                      size_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_scan(s, Use::kSaved)) return rc;
  if (!dy || !saved || !grads || !grads->dx || !grads->ddt || !grads->da || !grads->db || !grads->dc)
    return fail(MOC_ERR_ARG, "null tensor pointer");
  if (int rc = check_states(s, dfinal_state, grads->dinitial_state)) return rc;
  if (has_initial_state != 0 && s->cu_seqlens != nullptr)
    return fail(MOC_ERR_ARG, "states are only supported for fixed-length inputs");
  const moc::Scan p = problem(s);
  if (int rc = check_space(moc::scan_saved_bytes(p), saved, saved_bytes)) return rc;
  if (int rc = check_space(moc::scan_backward_workspace(p), workspace, workspace_bytes)) return rc;
  const moc::ScanGrads g{grads->dx, grads->ddt, grads->da, grads->db, grads->dc, grads->dd, grads->ddt_bias,
                         grads->dinitial_state};
  moc::scan_backward(p, dy, has_initial_state != 0, dfinal_state, saved, g, workspace,
                     static_cast<hipStream_t>(stream));
  return launched("moc_scan_backward launch");
}

int moc_scan_update(const MocScan* s, float* state, void* y, void* stream) {
  clear_error();
  if (int rc = check_scan(s, Use::kStep)) return rc;
  if (!state || !y) return fail(MOC_ERR_ARG, "null tensor pointer");
  moc::scan_update(problem(s), state, y, s->n_tokens, static_cast<hipStream_t>(stream));
  return launched("moc_scan_update launch");
}

}  // extern "C"
