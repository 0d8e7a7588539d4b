// C entry points of the operators between a state space layer's projections (declared in include/dfssm.h): checks, then
// the launches.
#include <hip/hip_runtime.h>

#include <initializer_list>

#include "dfssm.h"
#include "layer.h"

using namespace dfssm;

namespace {

int hip_status(hipError_t e) { return e == hipSuccess ? DFSSM_OK : (int)e; }
bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

constexpr int64_t kMaxScanLd = 1 << 23;       // the chunked kernel addresses a chunk's rows by 32-bit offsets
constexpr int64_t kMaxLd = (int64_t)1 << 30;  // (rows times this, in bytes, stays in 64 bits)
constexpr int64_t kMaxRows = (int64_t)1 << 30;
constexpr float kMinEps = 0x1p-126f;

bool type16(int t) { return t == DFSSM_TYPE_F16 || t == DFSSM_TYPE_BF16; }

// What the operators over sequences have in common.
template <class D>
int check_sequences(const D* d, bool step) {
  if (d->n_seq < 0 || d->n_tokens < 0 || d->n_tokens > kMaxRows || d->n_slots < 0) return DFSSM_E_RANGE;
  if (step && (d->n_tokens != d->n_seq || d->cu_seqlens)) return DFSSM_E_RANGE;
  if (!step && !d->cu_seqlens && d->n_seq > 0 && d->n_tokens % d->n_seq) return DFSSM_E_RANGE;
  return DFSSM_OK;
}

int check_conv(const dfssm_conv* d, bool step) {
  if (!d) return DFSSM_E_NULL;
  if (d->channels < 1 || d->channels > 1 << 24 || d->width < 2 || d->width > 4 || !type16(d->type)) return DFSSM_E_DIMS;
  const int rc = check_sequences(d, step);
  if (rc || d->n_seq == 0) return rc;
  if (!d->weight || !d->state || !d->state_out || (d->n_tokens && (!d->x || !d->out))) return DFSSM_E_NULL;
  if (!aligned(d->x, 2) || !aligned(d->weight, 2) || !aligned(d->bias, 2) || !aligned(d->state, 2) ||
      !aligned(d->state_out, 2) || !aligned(d->out, 2))
    return DFSSM_E_ALIGN;
  for (const int64_t ld : {d->ld_x, d->ld_out})
    if (ld < 0 || ld > kMaxLd) return DFSSM_E_RANGE;
  if (d->n_tokens > 1 && d->ld_out < d->channels) return DFSSM_E_DIMS;
  if (!step && d->n_tokens && d->out == d->x) return DFSSM_E_RANGE;
  return DFSSM_OK;
}

PackedConvArgs conv_args(const dfssm_conv* d) {
  PackedConvArgs a{};
  a.x = (const uint16_t*)d->x; a.weight = (const uint16_t*)d->weight; a.bias = (const uint16_t*)d->bias;
  a.state = (const uint16_t*)d->state; a.state_out = (uint16_t*)d->state_out;
  a.slots = d->slots; a.cu = d->cu_seqlens; a.out = (uint16_t*)d->out;
  a.ld_x = d->ld_x; a.ld_out = d->ld_out; a.n_tokens = d->n_tokens; a.len = d->n_tokens / d->n_seq;
  a.n_seq = d->n_seq; a.n_slots = d->n_slots; a.C = d->channels; a.W = d->width;
  a.bf16 = d->type == DFSSM_TYPE_BF16; a.silu = d->silu;
  return a;
}

int check_scan_dims(const dfssm_scan* d) {
  if (d->groups < 1 || d->heads < 1 || d->heads % d->groups) return DFSSM_E_DIMS;
  if ((d->cols != 64 && d->cols != 128) || d->dim < 16 || d->dim > 256 || d->dim % 16) return DFSSM_E_DIMS;
  return type16(d->type) && (d->dt_type == d->type || d->dt_type == DFSSM_TYPE_F32) ? DFSSM_OK : DFSSM_E_DIMS;
}

int check_scan(const dfssm_scan* d, bool step) {
  if (!d) return DFSSM_E_NULL;
  int rc = check_scan_dims(d);
  if (!rc) rc = check_sequences(d, step);
  if (rc || d->n_seq == 0) return rc;
  if (!d->A_log || !d->state || !d->state_out || (d->n_tokens && (!d->x || !d->dt || !d->B || !d->C || !d->out)))
    return DFSSM_E_NULL;
  if (!aligned(d->x, 16) || !aligned(d->B, 16) || !aligned(d->C, 16) || !aligned(d->out, 16) || !aligned(d->state, 16) ||
      !aligned(d->state_out, 16) || !aligned(d->dt, d->dt_type == DFSSM_TYPE_F32 ? 4 : 2))
    return DFSSM_E_ALIGN;
  for (const int64_t ld : {d->ld_x, d->ld_dt, d->ld_B, d->ld_C, d->ld_out})
    if (ld < 0 || ld > kMaxScanLd) return DFSSM_E_RANGE;
  if (d->n_tokens > 1 && d->ld_out < (int64_t)d->heads * d->dim) return DFSSM_E_DIMS;
  if (d->ld_x % 8 || d->ld_B % 8 || d->ld_C % 8 || d->ld_out % 8) return DFSSM_E_ALIGN;
  return DFSSM_OK;
}

PackedScanArgs scan_args(const dfssm_scan* d) {
  PackedScanArgs a{};
  a.x = (const uint16_t*)d->x; a.B = (const uint16_t*)d->B; a.C = (const uint16_t*)d->C; a.dt = d->dt;
  a.A_log = d->A_log; a.D = d->D; a.dt_bias = d->dt_bias;
  a.state = d->state; a.state_out = d->state_out;
  a.slots = d->slots; a.cu = d->cu_seqlens; a.out = (uint16_t*)d->out;
  a.ld_x = d->ld_x; a.ld_dt = d->ld_dt; a.ld_B = d->ld_B; a.ld_C = d->ld_C; a.ld_out = d->ld_out;
  a.n_tokens = d->n_tokens; a.len = d->n_tokens / d->n_seq;
  a.n_seq = d->n_seq; a.n_slots = d->n_slots; a.H = d->heads; a.G = d->groups; a.P = d->dim; a.N = d->cols;
  a.bf16 = d->type == DFSSM_TYPE_BF16; a.dt32 = d->dt_type == DFSSM_TYPE_F32; a.softplus = d->softplus;
  return a;
}

// Prompts that run token by token: too few tokens for a chunk's fixed work. The lengths behind cu_seqlens are on the device,
// so the rule there goes by all tokens, which any one sequence may have; without offsets it goes by the length, whatever the number
// of sequences. That is right for few of them: 32 and 64 of 7 or 8 tokens would take up to 15% less in chunks. Sequences of
// 4 | 6 | 8 | 12 tokens, token by token and in chunks, kernels in a replayed graph, fp16:
//   64 heads of 64 x 128                one 6.3, 11.9 | 7.8, 11.8 | 9.3, 11.9 | 12.1, 11.8 us   32: 31, 39 | 39, 39 | 45, 39 | 58, 40
//                                      four 8.6, 13.5 | 10.5, 13.5 | 12.4, 13.3 | 16.2, 13.4    64: 59, 70 | 72, 71 | 83, 72 | 116, 72
//   40 heads of 128 x 128, 5 groups     one 6.5, 11.8 | 8.1, 11.9 | 9.6, 11.9 | 12.4, 11.9      32: 39, 49 | 47, 49 | 54, 48 | 71, 49
//                                      four 9.7, 13.5 | 11.9, 13.5 | 14.3, 13.6 | 18.4, 13.5    64: 72, 90 | 89, 92 | 107, 92 | 139, 95
//   6 heads of 256 x 64                 one 5.7, 8.8 | 6.9, 8.8 | 8.3, 8.8 | 10.8, 8.9          32: 11, 14 | 14, 14 | 17, 14 | 22, 14
constexpr int kTokenPath = 8;
bool by_tokens(const PackedScanArgs& a) { return (a.cu ? a.n_tokens : a.len) <= kTokenPath; }

// Rows of a norm.
int check_rows(int64_t rows, int cols, std::initializer_list<int64_t> in, std::initializer_list<int64_t> out, float eps) {
  if (rows < 0 || rows > kMaxRows) return DFSSM_E_RANGE;
  for (const int64_t ld : in)
    if (ld < 0 || ld > kMaxLd) return DFSSM_E_RANGE;
  for (const int64_t ld : out) {
    if (ld < 0 || ld > kMaxLd) return DFSSM_E_RANGE;
    if (rows > 1 && ld < cols) return DFSSM_E_DIMS;
  }
  return eps >= kMinEps ? DFSSM_OK : DFSSM_E_RANGE;  // (a NaN is refused)
}

}  // namespace

extern "C" {

int dfssm_causal_conv_step(const dfssm_conv* args, void* stream) {
  const int rc = check_conv(args, true);
  if (rc || args->n_seq == 0) return rc;
  return hip_status(launch_conv_step(conv_args(args), (hipStream_t)stream));
}

int dfssm_causal_conv_prefill(const dfssm_conv* args, void* stream) {
  const int rc = check_conv(args, false);
  if (rc || args->n_seq == 0) return rc;
  return hip_status(launch_conv_prefill(conv_args(args), (hipStream_t)stream));
}

int dfssm_selective_scan_step(const dfssm_scan* args, void* stream) {
  const int rc = check_scan(args, true);
  if (rc || args->n_seq == 0) return rc;
  return hip_status(launch_scan_token(scan_args(args), (hipStream_t)stream));
}

size_t dfssm_selective_scan_workspace_bytes(const dfssm_scan* args) {
  if (!args || check_scan_dims(args) != DFSSM_OK || check_sequences(args, false) != DFSSM_OK || args->n_seq == 0) return 0;
  const PackedScanArgs a = scan_args(args);
  return by_tokens(a) ? 0 : scan_chunk_workspace(a);
}

int dfssm_selective_scan_prefill(const dfssm_scan* args, void* workspace, void* stream) {
  const int rc = check_scan(args, false);
  if (rc || args->n_seq == 0) return rc;
  const PackedScanArgs a = scan_args(args);
  if (by_tokens(a)) return hip_status(launch_scan_token(a, (hipStream_t)stream));
  if (scan_chunk_workspace(a)) {
    if (!workspace) return DFSSM_E_NULL;
    if (!aligned(workspace, 16)) return DFSSM_E_ALIGN;
  }
  return hip_status(launch_scan_chunked(a, workspace, (hipStream_t)stream));
}

int dfssm_gated_norm(const dfssm_gated* d, void* stream) {
  if (!d) return DFSSM_E_NULL;
  if (d->cols < 1 || d->groups < 1 || d->cols % d->groups || d->cols / d->groups > DFSSM_NORM_MAX_COLS || !type16(d->type))
    return DFSSM_E_DIMS;
  const int rc = check_rows(d->rows, d->cols, {d->ld_x, d->ld_gate}, {d->ld_out}, d->eps);
  if (rc || d->rows == 0) return rc;
  if (!d->x || !d->weight || !d->out) return DFSSM_E_NULL;
  if (!aligned(d->x, 2) || !aligned(d->gate, 2) || !aligned(d->out, 2) || !aligned(d->weight, 4)) return DFSSM_E_ALIGN;
  GatedNormArgs a{};
  a.x = (const uint16_t*)d->x; a.gate = (const uint16_t*)d->gate; a.weight = d->weight; a.out = (uint16_t*)d->out;
  a.ld_x = d->ld_x; a.ld_gate = d->ld_gate; a.ld_out = d->ld_out; a.rows = d->rows;
  a.cols = d->cols; a.groups = d->groups; a.bf16 = d->type == DFSSM_TYPE_BF16; a.gate_first = d->gate_first; a.eps = d->eps;
  return hip_status(launch_gated_norm(a, (hipStream_t)stream));
}

int dfssm_residual_norm(const dfssm_residual* d, void* stream) {
  if (!d) return DFSSM_E_NULL;
  if (d->cols < 1 || d->cols > DFSSM_NORM_MAX_COLS || !type16(d->type) ||
      (d->residual_type != d->type && d->residual_type != DFSSM_TYPE_F32))
    return DFSSM_E_DIMS;
  const int rc = check_rows(d->rows, d->cols, {d->ld_x, d->ld_residual}, {d->ld_out, d->ld_residual_out}, d->eps);
  if (rc || d->rows == 0) return rc;
  if (!d->x || !d->residual || !d->weight || !d->out || !d->residual_out) return DFSSM_E_NULL;
  const uintptr_t r = d->residual_type == DFSSM_TYPE_F32 ? 4 : 2;
  if (!aligned(d->x, 2) || !aligned(d->out, 2) || !aligned(d->residual, r) || !aligned(d->residual_out, r) ||
      !aligned(d->weight, 4) || !aligned(d->post_weight, 4) || !aligned(d->scales, 4))
    return DFSSM_E_ALIGN;
  ResidualNormArgs a{};
  a.x = (const uint16_t*)d->x; a.residual = d->residual;
  a.post_weight = d->post_weight; a.scales = d->scales; a.weight = d->weight;
  a.out = (uint16_t*)d->out; a.residual_out = d->residual_out;
  a.ld_x = d->ld_x; a.ld_res = d->ld_residual; a.ld_out = d->ld_out; a.ld_res_out = d->ld_residual_out; a.rows = d->rows;
  a.cols = d->cols; a.bf16 = d->type == DFSSM_TYPE_BF16; a.res32 = d->residual_type == DFSSM_TYPE_F32;
  a.scale = d->scale; a.eps = d->eps;
  return hip_status(launch_residual_norm(a, (hipStream_t)stream));
}

}  // extern "C"
