// C ABI of the rotary positions and of the verification of drafted tokens (declared in include/moba_b200.h): argument checks and launches.
#include "common.cuh"
#include "moba_b200.h"
#include "rotary.cuh"
#include "verify.cuh"

using namespace moba;

extern "C" {

int moba_rotary_check(const moba_rotary_t* p) {
  if (p == nullptr) return MOBA_E_NULL;
  if (p->total_tokens <= 0 || p->num_q_heads <= 0 || p->num_kv_heads < 0 || p->head_dim <= 0) return MOBA_E_SHAPE;
  if (p->rotary_dim <= 0 || p->rotary_dim > p->head_dim || p->rotary_dim % 2 != 0) return MOBA_E_SHAPE;
  if (!(p->magnitude > 0.f) || p->magnitude > 3.0e38f) return MOBA_E_SHAPE;
  if (p->head_dim != 64 && p->head_dim != 96 && p->head_dim != 128 && p->head_dim != 256) return MOBA_E_UNSUPPORTED;
  if (p->dtype != MOBA_DTYPE_BF16 && p->dtype != MOBA_DTYPE_FP16) return MOBA_E_UNSUPPORTED;
  if ((p->interleaved != 0 && p->interleaved != 1) || (p->inverse != 0 && p->inverse != 1) || p->reserved != 0 || p->reserved2 != 0)
    return MOBA_E_UNSUPPORTED;
  // rows and blocks are counted in 32 bits
  if (p->total_tokens >= ((int64_t)1 << 31) / ((int64_t)p->num_q_heads + p->num_kv_heads)) return MOBA_E_UNSUPPORTED;
  const int64_t strides[8] = {p->q_stride_token, p->q_stride_head, p->k_stride_token, p->k_stride_head,
                              p->qo_stride_token, p->qo_stride_head, p->ko_stride_token, p->ko_stride_head};
  for (int i = 0; i < 8; ++i) {
    if (strides[i] < 0) return MOBA_E_SHAPE;
    if (strides[i] % 8 != 0) return MOBA_E_ALIGN;
    const int heads = i % 4 < 2 ? p->num_q_heads : p->num_kv_heads;
    if (i >= 4 && strides[i] == 0 && (i % 2 == 0 ? p->total_tokens > 1 && heads > 0 : heads > 1)) return MOBA_E_SHAPE;   // rows on one another
  }
  return MOBA_OK;
}

int moba_rotary(const moba_rotary_t* p, const void* q, const void* k, const int32_t* positions, const int64_t* turns, void* q_out,
                void* k_out, void* stream) {
  const int rc = moba_rotary_check(p);
  if (rc != MOBA_OK) return rc;
  if (!q || !q_out || !positions || !turns || (p->num_kv_heads > 0 && (!k || !k_out))) return MOBA_E_NULL;
  if (((uintptr_t)q | (uintptr_t)q_out | (p->num_kv_heads > 0 ? (uintptr_t)k | (uintptr_t)k_out : 0)) & 15) return MOBA_E_ALIGN;
  if (((uintptr_t)positions & 3) || ((uintptr_t)turns & 7)) return MOBA_E_ALIGN;
  // rows that are turned where they are lie there the same way (a single token or head is never stepped over)
  auto apart = [&](int64_t t, int64_t h, int64_t to, int64_t ho, int heads) { return (p->total_tokens > 1 && t != to) || (heads > 1 && h != ho); };
  if (q == q_out && apart(p->q_stride_token, p->q_stride_head, p->qo_stride_token, p->qo_stride_head, p->num_q_heads)) return MOBA_E_SHAPE;
  if (p->num_kv_heads > 0 && k == k_out && apart(p->k_stride_token, p->k_stride_head, p->ko_stride_token, p->ko_stride_head, p->num_kv_heads))
    return MOBA_E_SHAPE;
  RotaryParams r{};
  r.rows = p->total_tokens;
  r.heads_q = p->num_q_heads;
  r.heads_k = p->num_kv_heads;
  r.dim = p->head_dim;
  r.turned = p->rotary_dim;
  r.interleaved = p->interleaved;
  r.inverse = p->inverse;
  r.fp16 = p->dtype == MOBA_DTYPE_FP16;
  r.magnitude = p->magnitude;
  r.q_t = p->q_stride_token; r.q_h = p->q_stride_head;
  r.k_t = p->k_stride_token; r.k_h = p->k_stride_head;
  r.qo_t = p->qo_stride_token; r.qo_h = p->qo_stride_head;
  r.ko_t = p->ko_stride_token; r.ko_h = p->ko_stride_head;
  r.q = q;
  r.k = k;
  r.q_out = q_out;
  r.k_out = k_out;
  r.positions = positions;
  r.turns = reinterpret_cast<const long long*>(turns);
  return (int)launch_rotary(r, (cudaStream_t)stream);
}

int moba_drafts_check(const moba_drafts_t* p) {
  if (p == nullptr) return MOBA_E_NULL;
  if (p->total_tokens <= 0 || p->batch <= 0 || p->vocabulary <= 0 || p->max_new <= 0) return MOBA_E_SHAPE;
  if (p->target_stride < 0 || p->draft_stride < 0) return MOBA_E_SHAPE;
  if (p->dtype != MOBA_DTYPE_BF16 && p->dtype != MOBA_DTYPE_FP16 && p->dtype != MOBA_DTYPE_FP32) return MOBA_E_UNSUPPORTED;
  if ((p->token_bits != 32 && p->token_bits != 64) || p->reserved != 0) return MOBA_E_UNSUPPORTED;
  if (p->max_new > kVerifyMostRows || p->vocabulary > kVerifyMostTokens || p->batch >= (1 << 27)) return MOBA_E_UNSUPPORTED;
  if (p->total_tokens >= ((int64_t)1 << 31)) return MOBA_E_UNSUPPORTED;
  return MOBA_OK;
}

int moba_verify_drafts(const moba_drafts_t* p, const void* target, const void* draft, const void* tokens, const int32_t* cu,
                       const int32_t* parents, const float* accept, const float* sample, int32_t* path, int32_t* count, void* next,
                       void* stream) {
  const int rc = moba_drafts_check(p);
  if (rc != MOBA_OK) return rc;
  if (!target || !tokens || !cu || !accept || !sample || !path || !count || !next) return MOBA_E_NULL;
  const uintptr_t element = p->dtype == MOBA_DTYPE_FP32 ? 3 : 1, token = p->token_bits / 8 - 1;
  if (((uintptr_t)target | (uintptr_t)draft) & element) return MOBA_E_ALIGN;
  if (((uintptr_t)tokens | (uintptr_t)next) & token) return MOBA_E_ALIGN;
  if (((uintptr_t)cu | (uintptr_t)parents | (uintptr_t)accept | (uintptr_t)sample | (uintptr_t)path | (uintptr_t)count) & 3) return MOBA_E_ALIGN;
  VerifyParams a{};
  a.target = target;
  a.draft = draft;
  a.tokens = tokens;
  a.target_stride = p->target_stride;
  a.draft_stride = p->draft_stride;
  a.rows = p->total_tokens;
  a.vocabulary = p->vocabulary;
  a.batch = p->batch;
  a.max_new = p->max_new;
  a.tokens64 = p->token_bits == 64;
  a.cu = cu;
  a.parents = parents;
  a.accept = accept;
  a.sample = sample;
  a.path = path;
  a.count = count;
  a.next = next;
  return (int)launch_verify(a, p->dtype, (cudaStream_t)stream);
}

}  // extern "C"
