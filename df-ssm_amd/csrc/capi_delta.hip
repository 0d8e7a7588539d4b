// C entry points of the gated delta rule (declared in include/dfssm.h): checks, then the launches.
#include <hip/hip_runtime.h>

#include "delta.h"
#include "dfssm.h"

using namespace dfssm;

namespace {

int hip_status(hipError_t e) { return e == hipSuccess ? DFSSM_OK : (int)e; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

constexpr int64_t kMaxLd = 1 << 23;

int check_dims(const dfssm_delta* d) {
  if (d->n_seq < 0 || d->n_tokens < 0 || d->n_slots < 0) return DFSSM_E_RANGE;
  if (d->k_heads < 1 || d->v_heads < 1 || d->v_heads % d->k_heads) return DFSSM_E_DIMS;
  if ((d->k_dim != 64 && d->k_dim != 128) || d->v_dim < 16 || d->v_dim > 256 || d->v_dim % 16) return DFSSM_E_DIMS;
  if (d->type != DFSSM_TYPE_F16 && d->type != DFSSM_TYPE_BF16) return DFSSM_E_DIMS;
  return DFSSM_OK;
}

int check_delta(const dfssm_delta* d, bool step) {
  if (!d) return DFSSM_E_NULL;
  const int rc = check_dims(d);
  if (rc) return rc;
  if (step && (d->n_tokens != d->n_seq || d->cu_seqlens)) return DFSSM_E_RANGE;
  if (!step && !d->cu_seqlens && d->n_seq > 0 && d->n_tokens % d->n_seq) return DFSSM_E_RANGE;
  if (d->n_seq == 0) return DFSSM_OK;
  if (!d->state || !d->state_out) return DFSSM_E_NULL;
  if (d->n_tokens && (!d->q || !d->k || !d->v || !d->g || !d->beta || !d->out)) return DFSSM_E_NULL;
  if (!aligned16(d->q) || !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->out) || !aligned16(d->state) ||
      !aligned16(d->state_out))
    return DFSSM_E_ALIGN;
  // (the kernels address a chunk's rows by 32-bit offsets)
  for (const int64_t ld : {d->ld_q, d->ld_k, d->ld_v, d->ld_g, d->ld_beta, d->ld_out})
    if (ld < 0 || ld > kMaxLd) return DFSSM_E_RANGE;
  if (d->n_tokens > 1 && d->ld_out < (int64_t)d->v_heads * d->v_dim) return DFSSM_E_DIMS;
  if (d->ld_q % 8 || d->ld_k % 8 || d->ld_v % 8 || d->ld_out % 8) return DFSSM_E_ALIGN;
  return DFSSM_OK;
}

DeltaArgs delta_args(const dfssm_delta* d) {
  DeltaArgs a{};
  a.q = (const uint16_t*)d->q; a.k = (const uint16_t*)d->k; a.v = (const uint16_t*)d->v;
  a.g = d->g; a.beta = d->beta;
  a.state = d->state; a.state_out = d->state_out;
  a.slots = d->slots; a.cu = d->cu_seqlens;
  a.out = (uint16_t*)d->out;
  a.ld_q = d->ld_q; a.ld_k = d->ld_k; a.ld_v = d->ld_v; a.ld_g = d->ld_g; a.ld_beta = d->ld_beta; a.ld_out = d->ld_out;
  a.n_tokens = d->n_tokens; a.len = d->n_seq ? d->n_tokens / d->n_seq : 0;
  a.n_seq = d->n_seq; a.n_slots = d->n_slots;
  a.Hk = d->k_heads; a.Hv = d->v_heads; a.Dk = d->k_dim; a.Dv = d->v_dim;
  a.bf16 = d->type == DFSSM_TYPE_BF16; a.l2norm = d->l2norm; a.scale = d->scale;
  return a;
}

// Prompts that run token by token: too few tokens for a chunk's fixed work. The lengths behind cu_seqlens are
// on the device, so the rule there goes by all tokens, which any one sequence may have (32 packed sequences of one token
// run 32 chunks). Kernels in a replayed graph, token by token and in chunks, for sequences of 12 | 16 | 24 tokens, fp16:
//   64 heads of 64 x 128   one sequence 9.9, 12.5 | 12.1, 12.6 | 17.2, 12.8 us   32: 68, 78 | 84, 79 | 117, 81
//   80 heads of 64 x 128                10.3, 16.8 | 12.8, 17.3 | 18.0, 17.0         83, 93 | 99, 97 | 142, 100
//   2 heads of 256 x 64                 7.9, 11.2 | 9.7, 11.3 | 13.4, 11.3           12.5, 17.5 | 15.4, 16.8 | 20.8, 17.3
//   12 heads of 128 x 64                8.4, 11.5 | 10.5, 11.9 | 14.7, 11.9          20.7, 27.2 | 25.6, 27.4 | 35, 27
//   40 heads of 128 x 128               10.1, 17.3 | 12.6, 17.2 | 17.3, 17.8         78, 89 | 98, 89 | 139, 90
constexpr int kTokenPath = 12;
bool by_tokens(const DeltaArgs& a) { return (a.cu ? a.n_tokens : a.len) <= kTokenPath; }

}  // namespace

extern "C" {

int dfssm_gated_delta_step(const dfssm_delta* args, void* stream) {
  const int rc = check_delta(args, true);
  if (rc || args->n_seq == 0) return rc;
  return hip_status(launch_delta_token(delta_args(args), (hipStream_t)stream));
}

size_t dfssm_gated_delta_workspace_bytes(const dfssm_delta* args) {
  if (!args || args->n_seq <= 0 || check_dims(args) != DFSSM_OK) return 0;
  const DeltaArgs a = delta_args(args);
  return by_tokens(a) ? 0 : delta_chunk_workspace(a);
}

int dfssm_gated_delta_prefill(const dfssm_delta* args, void* workspace, void* stream) {
  const int rc = check_delta(args, false);
  if (rc || args->n_seq == 0) return rc;
  const DeltaArgs a = delta_args(args);
  if (by_tokens(a)) return hip_status(launch_delta_token(a, (hipStream_t)stream));
  if (!workspace) return DFSSM_E_NULL;
  if (!aligned16(workspace)) return DFSSM_E_ALIGN;
  return hip_status(launch_delta_chunked(a, workspace, (hipStream_t)stream));
}

}  // extern "C"
