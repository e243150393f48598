// C entry points of the token half (include/spx.h): argument checks, job and
// workspace layout, launches.  No exception leaves them: nothing here throws.
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "sm100.cuh"

using namespace spx;

namespace {

__device__ int g_token_status;  // of callers without a word of their own

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

size_t round16(size_t n) { return (n + 15) & ~size_t(15); }

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

// Elements of 16 bytes, FP32 or BF16: a row stride is a multiple of them.
int64_t row_unit(int32_t f32) { return f32 != 0 ? 4 : 8; }

// ---------------------------------------------------------------- linear attention
int check_dims(const spx_linattn_dims* d) {
  if (d == nullptr) return SPX_ERR_INVALID_ARG;
  if (d->batch < 0 || d->seq_len < 0 || d->heads <= 0 || d->kv_heads <= 0 || d->heads % d->kv_heads != 0)
    return SPX_ERR_INVALID_ARG;
  if (d->key_dim <= 0 || d->value_dim <= 0 || !(d->scale < 0.0f || d->scale > 0.0f)) return SPX_ERR_INVALID_ARG;
  if (d->key_dim % 8 != 0 || d->value_dim % 8 != 0 || d->key_dim > kLaMaxD || d->value_dim > kLaMaxD)
    return SPX_ERR_UNSUPPORTED;
  // tokens and (sequence, head) pairs are 32-bit coordinates
  const int64_t lim = (int64_t(1) << 31) - 256;
  if (d->seq_len > lim || d->batch > lim || d->heads > 65535 || d->batch * d->heads > lim) return SPX_ERR_UNSUPPORTED;
  if (d->packed == 0 && d->batch > 0 && d->seq_len > lim / d->batch) return SPX_ERR_UNSUPPORTED;
  return SPX_OK;
}

int64_t total_tokens(const spx_linattn_dims& d) { return d.packed != 0 ? d.seq_len : d.batch * d.seq_len; }

// An output of tokens that belong to no sequence.
int zero_rows(void* p, size_t bytes, cudaStream_t stream) {
  if (bytes == 0) return SPX_OK;
  if (p == nullptr) return SPX_ERR_INVALID_ARG;
  return cudaMemsetAsync(p, 0, bytes, stream) == cudaSuccess ? SPX_OK : SPX_ERR_CUDA;
}

// Pointer, alignment and strides; the stride of a dimension of one element is not used.
int check_heads(const spx_heads* t, int64_t batch, int64_t tokens, int64_t heads) {
  if (t == nullptr || t->ptr == nullptr) return SPX_ERR_INVALID_ARG;
  const int64_t extent[3] = {batch, tokens, heads}, stride[3] = {t->batch_stride, t->token_stride, t->head_stride};
  bool misaligned = !aligned(t->ptr);
  for (int i = 0; i < 3; ++i) {
    if (extent[i] <= 1) continue;
    if (stride[i] < 0) return SPX_ERR_INVALID_ARG;
    if (stride[i] % 8 != 0) misaligned = true;
  }
  return misaligned ? SPX_ERR_ALIGNMENT : SPX_OK;
}

// Of q, k, v (and the output's gradient) of a call over sequences.
int check_sequences(const spx_linattn_dims& d, const spx_heads* q, const spx_heads* k, const spx_heads* v,
                    const spx_heads* d_out) {
  const int64_t rows = d.packed != 0 ? 1 : d.batch;
  if (int rc = check_heads(q, rows, d.seq_len, d.heads); rc != SPX_OK) return rc;
  if (int rc = check_heads(k, rows, d.seq_len, d.kv_heads); rc != SPX_OK) return rc;
  if (int rc = check_heads(v, rows, d.seq_len, d.kv_heads); rc != SPX_OK) return rc;
  return d_out == nullptr ? SPX_OK : check_heads(d_out, rows, d.seq_len, d.heads);
}

LaOperand operand(const spx_heads* t, int group) {
  return LaOperand{t->ptr, t->batch_stride, t->token_stride, t->head_stride, group};
}

LaArgs base_args(const spx_linattn_dims& d, const spx_decays* g, const int32_t* cu, int* status) {
  LaArgs a{};
  a.g = g->ptr;
  a.g_sb = g->batch_stride;
  a.g_st = g->token_stride;
  a.g_sh = g->head_stride;
  a.cu = d.packed != 0 ? cu : nullptr;
  a.T = d.seq_len;
  a.total = total_tokens(d);
  a.nseq = static_cast<int>(d.batch);
  a.H = d.heads;
  a.g_f32 = d.decay_f32;
  a.scale = d.scale;
  a.status = status;
  return a;
}

// Planes of the chunked form's dots: two for each 64 columns of an output.
int planes_of(int width) { return 2 * ((width + 63) / 64); }

template <typename T>
T* at(void* base, size_t off) {
  return reinterpret_cast<T*>(static_cast<uint8_t*>(base) + off);
}

// A few tokens go one by one: the chunked form would pad them to 128.  Forward,
// 4 x 12 heads of 64: 6, 9.7 and 14.5 us for 1, 4 and 8 tokens, chunked 12.5; 64 x 16
// heads of 128: 27, 50, 78 and 110 us for 1, 4, 8 and 12 tokens, chunked 110.
constexpr int64_t kRecurrentMax = 8;
bool recurrent(const LaArgs& a) { return a.cu == nullptr && a.T <= kRecurrentMax; }

// The widths, counts and lengths alone, for workspace sizes.
LaArgs shape_args(const spx_linattn_dims& d, bool backward) {
  static const int32_t some = 0;
  const spx_decays none{};
  LaArgs a = base_args(d, &none, &some, nullptr);
  a.njobs = backward ? 3 : 1;
  a.job[0].dc = backward ? d.key_dim : d.value_dim;
  a.job[1].dc = d.key_dim;
  a.job[2].dc = d.value_dim;
  return a;
}

size_t jobs_workspace(const LaArgs& a) { return a.nseq == 0 || recurrent(a) ? 0 : la_chunk_workspace(a); }

int run_jobs(const LaArgs& a, bool precise, void* workspace, cudaStream_t stream) {
  return recurrent(a) ? launch_la_recurrent(a, stream) : launch_la_chunk(a, precise, workspace, stream);
}

struct BackwardLayout {
  size_t q_dots, k_dots, last, dk, dv, segments, total;
};

BackwardLayout backward_layout(const spx_linattn_dims& d) {
  BackwardLayout L{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = round16(off + bytes);
    return at;
  };
  const size_t n = static_cast<size_t>(total_tokens(d)), h = static_cast<size_t>(d.heads);
  const size_t state = static_cast<size_t>(d.batch) * h * d.key_dim * d.value_dim * 4;
  L.q_dots = take(n * h * 4 * planes_of(d.key_dim));
  L.k_dots = take(n * h * 4 * planes_of(d.key_dim));
  L.last = take(state);
  if (d.heads != d.kv_heads) {
    L.dk = take(n * h * d.key_dim * 4);
    L.dv = take(n * h * d.value_dim * 4);
  }
  L.segments = take(jobs_workspace(shape_args(d, true)));
  L.total = off;
  return L;
}

}  // namespace

extern "C" {

int spx_add_rmsnorm_rows(const uint16_t* hidden, int64_t ld_hidden, const void* residual, int64_t ld_residual,
                         int32_t residual_f32, const uint16_t* norm_weight, float eps, int64_t rows, int32_t d,
                         void* sum, uint16_t* normed, uint8_t* mx_values, uint8_t* mx_scales, void* stream) {
  if (rows < 0 || d <= 0 || !(eps > 0.0f)) return SPX_ERR_INVALID_ARG;
  if (d % 8 != 0 || d > kNormMaxD) return SPX_ERR_UNSUPPORTED;
  const bool mx = mx_values != nullptr || mx_scales != nullptr;
  if (mx && (mx_values == nullptr || mx_scales == nullptr)) return SPX_ERR_INVALID_ARG;
  if (mx && d % kMxBlock != 0) return SPX_ERR_UNSUPPORTED;
  if (rows == 0) return SPX_OK;
  if (hidden == nullptr || norm_weight == nullptr || (!mx && normed == nullptr)) return SPX_ERR_INVALID_ARG;
  if ((residual == nullptr) != (sum == nullptr)) return SPX_ERR_INVALID_ARG;
  if (ld_hidden < 0 || (residual != nullptr && ld_residual < 0)) return SPX_ERR_INVALID_ARG;
  if (!aligned(hidden) || !aligned(norm_weight) || !aligned(residual) || !aligned(sum) || !aligned(normed) ||
      !aligned(mx_values) || ld_hidden % 8 != 0 || (residual != nullptr && ld_residual % row_unit(residual_f32) != 0))
    return SPX_ERR_ALIGNMENT;
  AddNormArgs a{};
  a.x = hidden;
  a.res = residual;
  a.w = norm_weight;
  a.sum = sum;
  a.y = normed;
  a.mx_values = mx_values;
  a.mx_scales = mx_scales;
  a.rows = rows;
  a.ld_x = ld_hidden;
  a.ld_res = ld_residual;
  a.d = d;
  a.res_f32 = residual != nullptr && residual_f32 != 0 ? 1 : 0;
  a.eps = eps;
  return launch_add_norm(a, as_stream(stream));
}

size_t spx_add_rmsnorm_backward_workspace(int64_t rows, int32_t d) {
  if (rows <= 0 || d <= 0) return 0;
  return static_cast<size_t>(add_norm_backward_parts(rows, d)) * d * sizeof(float);
}

int spx_add_rmsnorm_backward(const void* sum, int64_t ld_sum, int32_t residual_f32, const uint16_t* norm_weight,
                             float eps, const uint16_t* d_normed, int64_t ld_d_normed, const void* d_sum,
                             int64_t ld_d_sum, int64_t rows, int32_t d, uint16_t* d_hidden, float* d_residual,
                             uint16_t* d_weight, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || d <= 0 || !(eps > 0.0f)) return SPX_ERR_INVALID_ARG;
  if (d % 8 != 0 || d > kNormMaxD) return SPX_ERR_UNSUPPORTED;
  if (rows > 0) {
    if (sum == nullptr || norm_weight == nullptr || d_normed == nullptr || d_hidden == nullptr)
      return SPX_ERR_INVALID_ARG;
    if (d_residual != nullptr && residual_f32 == 0) return SPX_ERR_INVALID_ARG;
    if (ld_sum < 0 || ld_d_normed < 0 || (d_sum != nullptr && ld_d_sum < 0)) return SPX_ERR_INVALID_ARG;
    if (!aligned(sum) || !aligned(norm_weight) || !aligned(d_normed) || !aligned(d_sum) || !aligned(d_hidden) ||
        !aligned(d_residual) || ld_sum % row_unit(residual_f32) != 0 || ld_d_normed % 8 != 0 ||
        (d_sum != nullptr && ld_d_sum % row_unit(residual_f32) != 0))
      return SPX_ERR_ALIGNMENT;
    if (d_weight != nullptr) {
      if (workspace == nullptr || workspace_bytes < spx_add_rmsnorm_backward_workspace(rows, d)) return SPX_ERR_WORKSPACE;
      if (!aligned(workspace)) return SPX_ERR_ALIGNMENT;
    }
  }
  AddNormBackwardArgs a{};
  a.h = sum;
  a.w = norm_weight;
  a.dy = d_normed;
  a.dsum = d_sum;
  a.dx = d_hidden;
  a.dres = d_residual;
  a.dw_part = d_weight != nullptr ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows;
  a.ld_h = ld_sum;
  a.ld_dy = ld_d_normed;
  a.ld_dsum = ld_d_sum;
  a.d = d;
  a.res_f32 = residual_f32 != 0 ? 1 : 0;
  a.eps = eps;
  return launch_add_norm_backward(a, d_weight, as_stream(stream));
}

int spx_rotary(const spx_heads* q, int32_t q_heads, const spx_heads* k, int32_t k_heads, int64_t tokens,
               int32_t head_dim, int32_t pairs, const void* positions, int32_t positions_64, int64_t position_period,
               const double* frequencies, float factor, int32_t interleaved, int32_t inverse, uint16_t* q_out,
               uint16_t* k_out, void* stream) {
  if (tokens < 0 || head_dim <= 0 || pairs < 0 || 2 * static_cast<int64_t>(pairs) > head_dim || q_heads < 0 || k_heads < 0)
    return SPX_ERR_INVALID_ARG;
  if (head_dim > kRotMaxD || q_heads > 65535 || k_heads > 65535) return SPX_ERR_UNSUPPORTED;
  if (tokens == 0 || q_heads + k_heads == 0) return SPX_OK;
  if ((q_heads > 0 && (q == nullptr || q->ptr == nullptr || q_out == nullptr)) ||
      (k_heads > 0 && (k == nullptr || k->ptr == nullptr || k_out == nullptr)))
    return SPX_ERR_INVALID_ARG;
  if (pairs > 0 && (positions == nullptr || frequencies == nullptr)) return SPX_ERR_INVALID_ARG;
  if (position_period <= 0) return SPX_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(frequencies) & 7u) != 0) return SPX_ERR_ALIGNMENT;
  RotaryArgs a{};
  if (q_heads > 0) a.q = q->ptr, a.q_st = q->token_stride, a.q_sh = q->head_stride;
  if (k_heads > 0) a.k = k->ptr, a.k_st = k->token_stride, a.k_sh = k->head_stride;
  a.q_out = q_out;
  a.k_out = k_out;
  a.pos = positions;
  a.freq = frequencies;
  a.tokens = tokens;
  a.pos_period = position_period;
  a.heads_q = q_heads;
  a.heads_k = k_heads;
  a.d = head_dim;
  a.pairs = pairs;
  a.pos64 = positions_64 != 0 ? 1 : 0;
  a.interleaved = interleaved != 0 ? 1 : 0;
  a.inverse = inverse != 0 ? 1 : 0;
  a.factor = factor;
  return launch_rotary(a, as_stream(stream));
}

int spx_token_status_word(int** word) {
  if (word == nullptr) return SPX_ERR_INVALID_ARG;
  // the first use on a device loads the variable, which a capture under way would not allow in its own mode
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return SPX_ERR_CUDA;
  void* p = nullptr;
  const cudaError_t got = cudaGetSymbolAddress(&p, g_token_status);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (got != cudaSuccess || p == nullptr) return SPX_ERR_CUDA;
  *word = static_cast<int*>(p);
  return SPX_OK;
}

size_t spx_linear_attention_workspace(const spx_linattn_dims* dims) {
  if (check_dims(dims) != SPX_OK) return 0;
  return jobs_workspace(shape_args(*dims, false));
}

int spx_linear_attention(const spx_linattn_dims* dims, const spx_heads* q, const spx_heads* k, const spx_heads* v,
                         const spx_decays* decays, const int32_t* cu_seqlens, const float* initial_state,
                         uint16_t* out, float* final_state, void* workspace, size_t workspace_bytes, int* status,
                         void* stream) {
  if (int rc = check_dims(dims); rc != SPX_OK) return rc;
  const spx_linattn_dims& d = *dims;
  if (d.batch == 0) {
    const size_t n = static_cast<size_t>(total_tokens(d)) * d.heads;
    return zero_rows(out, n * d.value_dim * 2, as_stream(stream));
  }
  if (d.packed != 0 && cu_seqlens == nullptr) return SPX_ERR_INVALID_ARG;
  if (total_tokens(d) > 0) {
    if (int rc = check_sequences(d, q, k, v, nullptr); rc != SPX_OK) return rc;
    if (decays == nullptr || decays->ptr == nullptr || out == nullptr) return SPX_ERR_INVALID_ARG;
  } else if (q == nullptr || k == nullptr || v == nullptr || decays == nullptr) {
    return SPX_ERR_INVALID_ARG;
  }
  if (!aligned(out) || !aligned(initial_state) || !aligned(final_state)) return SPX_ERR_ALIGNMENT;
  const size_t need = spx_linear_attention_workspace(dims);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return SPX_ERR_WORKSPACE;
  if (!aligned(workspace)) return SPX_ERR_ALIGNMENT;
  const int group = d.heads / d.kv_heads;
  LaArgs a = base_args(d, decays, cu_seqlens, status);
  LaJob& j = a.job[0];
  a.njobs = 1;
  j.a = operand(q, 1);
  j.b = operand(k, group);
  j.c = operand(v, group);
  j.da = d.key_dim;
  j.dc = d.value_dim;
  j.out = out;
  j.init = initial_state;
  j.fin = final_state;
  j.s_row = d.value_dim;
  j.s_col = 1;
  j.init_scale = j.fin_scale = 1.0f;
  return run_jobs(a, false, workspace, as_stream(stream));
}

size_t spx_linear_attention_backward_workspace(const spx_linattn_dims* dims) {
  if (check_dims(dims) != SPX_OK) return 0;
  return backward_layout(*dims).total;
}

int spx_linear_attention_backward(const spx_linattn_dims* dims, const spx_heads* q, const spx_heads* k,
                                  const spx_heads* v, const spx_decays* decays, const int32_t* cu_seqlens,
                                  const float* initial_state, const spx_heads* d_out, const float* d_final_state,
                                  uint16_t* d_q, uint16_t* d_k, uint16_t* d_v, void* d_decay, float* d_initial_state,
                                  void* workspace, size_t workspace_bytes, int* status, void* stream) {
  if (int rc = check_dims(dims); rc != SPX_OK) return rc;
  const spx_linattn_dims& d = *dims;
  const int64_t total = total_tokens(d);
  if (d.batch == 0) {
    const size_t n = static_cast<size_t>(total), h = d.heads, kv = d.kv_heads;
    const cudaStream_t st = as_stream(stream);
    if (int rc = zero_rows(d_q, n * h * d.key_dim * 2, st); rc != SPX_OK) return rc;
    if (int rc = zero_rows(d_k, n * kv * d.key_dim * 2, st); rc != SPX_OK) return rc;
    if (int rc = zero_rows(d_v, n * kv * d.value_dim * 2, st); rc != SPX_OK) return rc;
    return zero_rows(d_decay, n * h * (d.decay_f32 != 0 ? 4 : 2), st);
  }
  if (d.packed != 0 && cu_seqlens == nullptr) return SPX_ERR_INVALID_ARG;
  if (total > 0) {
    if (d_out == nullptr) return SPX_ERR_INVALID_ARG;
    if (int rc = check_sequences(d, q, k, v, d_out); rc != SPX_OK) return rc;
    if (decays == nullptr || decays->ptr == nullptr || d_q == nullptr || d_k == nullptr || d_v == nullptr ||
        d_decay == nullptr)
      return SPX_ERR_INVALID_ARG;
  } else if (q == nullptr || k == nullptr || v == nullptr || decays == nullptr || d_out == nullptr) {
    return SPX_ERR_INVALID_ARG;
  }
  if (!aligned(d_q) || !aligned(d_k) || !aligned(d_v) || !aligned(initial_state) || !aligned(d_final_state) ||
      !aligned(d_initial_state) || !aligned(workspace))
    return SPX_ERR_ALIGNMENT;
  const BackwardLayout L = backward_layout(d);
  if (L.total > 0 && (workspace == nullptr || workspace_bytes < L.total)) return SPX_ERR_WORKSPACE;
  const int group = d.heads / d.kv_heads;
  const int K = d.key_dim, V = d.value_dim;
  const cudaStream_t st = as_stream(stream);
  LaArgs a = base_args(d, decays, cu_seqlens, status);
  a.njobs = 3;
  a.dg = d_decay;
  // d q_i = scale sum_{j <= i} w_ij (d out_i . v_j) k_j: the forward's sum on (d out, v, k), state transposed
  LaJob& jq = a.job[0];
  jq.a = operand(d_out, 1);
  jq.b = operand(v, group);
  jq.c = operand(k, group);
  jq.da = V;
  jq.dc = K;
  jq.out = d_q;
  jq.init = initial_state;
  jq.fin = d_final_state != nullptr ? at<float>(workspace, L.last) : nullptr;
  jq.s_row = 1;
  jq.s_col = V;
  jq.init_scale = jq.fin_scale = 1.0f;
  jq.e = operand(q, 1);
  jq.dots = at<float>(workspace, L.q_dots);
  // d k_j = scale sum_{i >= j} w_ij (v_j . d out_i) q_i
  LaJob& jk = a.job[1];
  jk.a = operand(v, group);
  jk.b = operand(d_out, 1);
  jk.c = operand(q, 1);
  jk.da = V;
  jk.dc = K;
  jk.reverse = 1;
  jk.out = group > 1 ? at<void>(workspace, L.dk) : d_k;
  jk.out_f32 = group > 1 ? 1 : 0;
  jk.init = d_final_state;
  jk.s_row = 1;
  jk.s_col = V;
  jk.init_scale = 1.0f / d.scale;  // the last state's gradient enters without `scale`
  jk.fin_scale = d.scale;
  if (group == 1) {  // else the sum over the group takes k . dk per query head
    jk.e = operand(k, 1);
    jk.dots = at<float>(workspace, L.k_dots);
  }
  // d v_j = scale sum_{i >= j} w_ij (k_j . q_i) d out_i, and the first state's gradient
  LaJob& jv = a.job[2];
  jv.a = operand(k, group);
  jv.b = operand(q, 1);
  jv.c = operand(d_out, 1);
  jv.da = K;
  jv.dc = V;
  jv.reverse = 1;
  jv.out = group > 1 ? at<void>(workspace, L.dv) : d_v;
  jv.out_f32 = group > 1 ? 1 : 0;
  jv.init = d_final_state;
  jv.fin = d_initial_state;
  jv.s_row = V;
  jv.s_col = 1;
  jv.init_scale = 1.0f / d.scale;
  jv.fin_scale = d.scale;
  if (int rc = run_jobs(a, true, at<void>(workspace, L.segments), st); rc != SPX_OK) return rc;
  if (group > 1) {
    LaGroupSumArgs sum{};
    sum.total = total;
    sum.T = d.packed != 0 ? total : d.seq_len;
    sum.H = d.heads;
    sum.group = group;
    sum.in = at<float>(workspace, L.dk);
    sum.out = d_k;
    sum.d = K;
    sum.e = operand(k, group);
    sum.dots = at<float>(workspace, L.k_dots);
    if (int rc = launch_la_group_sum(sum, st); rc != SPX_OK) return rc;
    sum.in = at<float>(workspace, L.dv);
    sum.out = d_v;
    sum.d = V;
    sum.e = LaOperand{};
    if (int rc = launch_la_group_sum(sum, st); rc != SPX_OK) return rc;
  }
  LaDecayGradArgs g{};
  g.q_dots = jq.dots;
  g.k_dots = at<float>(workspace, L.k_dots);
  g.q_slices = recurrent(a) ? 1 : planes_of(K);
  g.k_slices = group > 1 ? 1 : g.q_slices;
  g.last = jq.fin;
  g.d_last = d_final_state;
  g.dg = d_decay;
  g.cu = a.cu;
  g.T = a.T;
  g.total = total;
  g.state_elems = static_cast<int64_t>(K) * V;
  g.nseq = a.nseq;
  g.H = a.H;
  g.g_f32 = a.g_f32;
  g.from_zero = initial_state == nullptr;
  if (int rc = launch_la_decay_grad(g, st); rc != SPX_OK) return rc;
  return SPX_OK;
}

int spx_linear_attention_step(const spx_heads* q, const spx_heads* k, const spx_heads* v, const spx_decays* decays,
                              int32_t decay_f32, int64_t batch, int32_t heads, int32_t kv_heads, int32_t key_dim,
                              int32_t value_dim, float scale, float* state, int64_t slots, const int64_t* slot_index,
                              uint16_t* out, void* stream) {
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || slots < 0 || key_dim <= 0 || value_dim <= 0)
    return SPX_ERR_INVALID_ARG;
  if (key_dim % 8 != 0 || value_dim % 8 != 0 || key_dim > kLaMaxD || value_dim > kLaMaxD) return SPX_ERR_UNSUPPORTED;
  if (batch == 0) return SPX_OK;
  if (slot_index == nullptr && batch > slots) return SPX_ERR_INVALID_ARG;
  if (int rc = check_heads(q, batch, 1, heads); rc != SPX_OK) return rc;
  if (int rc = check_heads(k, batch, 1, kv_heads); rc != SPX_OK) return rc;
  if (int rc = check_heads(v, batch, 1, kv_heads); rc != SPX_OK) return rc;
  if (decays == nullptr || decays->ptr == nullptr || (state == nullptr && slots > 0) || out == nullptr)
    return SPX_ERR_INVALID_ARG;
  if (!aligned(state) || !aligned(out)) return SPX_ERR_ALIGNMENT;
  const int group = heads / kv_heads;
  LaStepArgs a{};
  a.q = operand(q, 1);
  a.k = operand(k, group);
  a.v = operand(v, group);
  a.g = decays->ptr;
  a.g_sb = decays->batch_stride;
  a.g_sh = decays->head_stride;
  a.g_f32 = decay_f32;
  a.state = state;
  a.slot = slot_index;
  a.slots = slots;
  a.out = out;
  a.batch = batch;
  a.H = heads;
  a.dk = key_dim;
  a.dv = value_dim;
  a.scale = scale;
  return launch_la_step(a, as_stream(stream));
}

}  // extern "C"
