// C ABI of the paged keys and values (declared in include/moba_b200.h): argument checks and launches.  Host-side only.
#include "paged.cuh"

using namespace moba;

namespace {

int check_paged(const moba_paged_t* p) {
  if (p == nullptr) return MOBA_E_NULL;
  if (p->total_tokens <= 0 || p->batch <= 0 || p->num_q_heads <= 0 || p->num_kv_heads <= 0 || p->head_dim <= 0) return MOBA_E_SHAPE;
  if (p->num_q_heads % p->num_kv_heads != 0) return MOBA_E_SHAPE;
  if (p->num_pages <= 0 || p->page_size <= 0 || p->pages_per_seq <= 0 || p->max_new <= 0) return MOBA_E_SHAPE;
  if (p->head_dim != 64 && p->head_dim != 96 && p->head_dim != 128 && p->head_dim != 256) return MOBA_E_UNSUPPORTED;
  if (p->num_q_heads / p->num_kv_heads > 128) return MOBA_E_UNSUPPORTED;
  if (p->page_size < 16 || (p->page_size & (p->page_size - 1)) != 0) return MOBA_E_UNSUPPORTED;
  if ((p->dtype != MOBA_DTYPE_BF16 && p->dtype != MOBA_DTYPE_FP16) || p->reserved != 0) return MOBA_E_UNSUPPORTED;
  if (p->store != MOBA_STORE_SAME && p->store != MOBA_STORE_E4M3 && p->store != MOBA_STORE_INT8) return MOBA_E_UNSUPPORTED;
  if (!(p->softmax_scale >= 0.f) || p->softmax_scale > 2.3e38f) return MOBA_E_SHAPE;   // (times log2 e it is still finite)
  // rows and grids are counted in 32 bits, positions too
  if (p->total_tokens >= ((int64_t)1 << 31) / p->num_q_heads) return MOBA_E_UNSUPPORTED;
  if ((int64_t)p->pages_per_seq * p->page_size >= ((int64_t)1 << 30)) return MOBA_E_UNSUPPORTED;
  if (p->table_stride < (p->batch > 1 ? p->pages_per_seq : 0)) return MOBA_E_SHAPE;
  const int64_t strides[8] = {p->q_stride_token, p->q_stride_head, p->o_stride_token, p->o_stride_head,
                              p->k_stride_token, p->k_stride_head, p->v_stride_token, p->v_stride_head};
  for (int i = 0; i < 8; ++i) {
    if (strides[i] < 0) return MOBA_E_SHAPE;
    if (strides[i] % 8 != 0) return MOBA_E_ALIGN;
  }
  const int64_t pool[6] = {p->k_page_stride, p->k_page_token, p->k_page_head, p->v_page_stride, p->v_page_token, p->v_page_head};
  for (int i = 0; i < 6; ++i) {
    if (pool[i] <= 0) return MOBA_E_SHAPE;
    if (pool[i] % (p->store == MOBA_STORE_SAME ? 8 : 16) != 0) return MOBA_E_ALIGN;
  }
  return MOBA_OK;
}

PagedParams paged_params(const moba_paged_t* p, const int32_t* cu, const int32_t* lens, const int32_t* table) {
  PagedParams r;
  r.T = p->total_tokens;
  r.B = p->batch;
  r.Hq = p->num_q_heads;
  r.Hkv = p->num_kv_heads;
  r.G = r.Hq / r.Hkv;
  r.D = p->head_dim;
  r.pages = p->num_pages;
  r.page_shift = 0;
  while ((1 << r.page_shift) < p->page_size) ++r.page_shift;
  r.per_seq = p->pages_per_seq;
  r.max_new = p->max_new;
  r.fp16 = p->dtype == MOBA_DTYPE_FP16;
  r.store = p->store;
  r.sl2 = (p->softmax_scale > 0.f ? p->softmax_scale : 1.f / sqrtf((float)r.D)) * 1.4426950408889634f;
  r.sq_t = p->q_stride_token; r.sq_h = p->q_stride_head;
  r.so_t = p->o_stride_token; r.so_h = p->o_stride_head;
  r.sk_t = p->k_stride_token; r.sk_h = p->k_stride_head;
  r.sv_t = p->v_stride_token; r.sv_h = p->v_stride_head;
  r.kp_p = p->k_page_stride; r.kp_t = p->k_page_token; r.kp_h = p->k_page_head;
  r.vp_p = p->v_page_stride; r.vp_t = p->v_page_token; r.vp_h = p->v_page_head;
  r.table_stride = p->table_stride;
  r.cu = cu;
  r.lens = lens;
  r.table = table;
  return r;
}

// Pointers of every call; `a` and `b`: its packed tensors.
int check_pointers(const moba_paged_t* p, const void* a, const void* b, const int32_t* cu, const int32_t* lens,
                   const int32_t* table, const void* kp, const void* vp, const void* ks, const void* vs) {
  if (!a || !b || !cu || !lens || !table || !kp || !vp) return MOBA_E_NULL;
  if (p->store != MOBA_STORE_SAME && (!ks || !vs)) return MOBA_E_NULL;
  if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)kp | (uintptr_t)vp) & 15) return MOBA_E_ALIGN;
  if (p->store != MOBA_STORE_SAME && (((uintptr_t)ks | (uintptr_t)vs) & 15)) return MOBA_E_ALIGN;
  if (((uintptr_t)cu | (uintptr_t)lens | (uintptr_t)table) & 3) return MOBA_E_ALIGN;
  return MOBA_OK;
}

size_t workspace_of(const PagedParams& p) { return paged_few_rows(p) ? paged_few_workspace(p) : paged_rows_workspace(p); }

// Rows that are written must not lie on one another (a single token or head is never stepped over).
bool apart(const moba_paged_t* p, int64_t token, int64_t head, int heads) {
  return (token > 0 || p->total_tokens == 1) && (head > 0 || heads == 1);
}

}  // namespace

extern "C" {

int moba_paged_check(const moba_paged_t* p) { return check_paged(p); }

int moba_paged_store(const moba_paged_t* p, const void* k, const void* v, const int32_t* cu, const int32_t* lens, const int32_t* table,
                     void* kp, void* vp, uint8_t* ks, uint8_t* vs, void* stream) {
  int rc = check_paged(p);
  if (rc == MOBA_OK) rc = check_pointers(p, k, v, cu, lens, table, kp, vp, ks, vs);
  if (rc != MOBA_OK) return rc;
  return (int)launch_paged_store(paged_params(p, cu, lens, table), k, v, kp, vp, ks, vs, (cudaStream_t)stream);
}

int moba_paged_load(const moba_paged_t* p, const int32_t* cu, const int32_t* lens, const int32_t* table, const void* kp, const void* vp,
                    const uint8_t* ks, const uint8_t* vs, void* k, void* v, void* stream) {
  int rc = check_paged(p);
  if (rc == MOBA_OK) rc = check_pointers(p, k, v, cu, lens, table, kp, vp, ks, vs);
  if (rc != MOBA_OK) return rc;
  if (!apart(p, p->k_stride_token, p->k_stride_head, p->num_kv_heads) || !apart(p, p->v_stride_token, p->v_stride_head, p->num_kv_heads))
    return MOBA_E_SHAPE;
  return (int)launch_paged_load(paged_params(p, cu, lens, table), kp, vp, ks, vs, k, v, (cudaStream_t)stream);
}

int moba_paged_workspace_size(const moba_paged_t* p, size_t* bytes) {
  const int rc = check_paged(p);
  if (rc != MOBA_OK) return rc;
  if (bytes == nullptr) return MOBA_E_NULL;
  *bytes = workspace_of(paged_params(p, nullptr, nullptr, nullptr));
  return MOBA_OK;
}

int moba_paged_attention(const moba_paged_t* p, const void* q, const int32_t* cu, const int32_t* lens, const int32_t* table,
                         const void* kp, const void* vp, const uint8_t* ks, const uint8_t* vs, void* out, float* lse_out,
                         void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_paged(p);
  if (rc == MOBA_OK) rc = check_pointers(p, q, out, cu, lens, table, kp, vp, ks, vs);
  if (rc != MOBA_OK) return rc;
  if (!apart(p, p->o_stride_token, p->o_stride_head, p->num_q_heads)) return MOBA_E_SHAPE;
  if ((uintptr_t)lse_out & 3) return MOBA_E_ALIGN;
  const PagedParams r = paged_params(p, cu, lens, table);
  if (workspace == nullptr || workspace_bytes < workspace_of(r)) return MOBA_E_WORKSPACE;
  if ((uintptr_t)workspace & 31) return MOBA_E_ALIGN;
  return (int)(paged_few_rows(r) ? launch_paged_few : launch_paged_rows)(r, q, kp, vp, ks, vs, out, lse_out, workspace, (cudaStream_t)stream);
}

}  // extern "C"
