// extern "C" entry points of the 8-bit key/value cache: host-side checks and dispatch.  No allocation, no host
// synchronisation, no global state.
#include "cbk_cache8.h"
#include "cbk_cache_attn.h"
#include "cbk_cache_check.h"

namespace cbk {

int launch_cache8_write(const DCache8&, const DRows&, const CacheIo&, int dt, hipStream_t);
int launch_cache8_read(const DCache8&, const DRows&, const CacheIo&, int dt, hipStream_t);
int launch_cache8_attn(const DCache8&, const DRows&, AttnArgs, size_t ws_bytes, hipStream_t);
size_t cache8_attn_workspace(const DCache8&, const DRows&, int ratio);

static int to_dcache8(const cbk_cache8* in, DCache8* c, bool need_device_ptrs) {
  if (!in) return CBK_ERR_NULL;
  if (in->head_dim != 64 && in->head_dim != 128 && in->head_dim != 256) return CBK_ERR_LAYOUT;
  if (in->page < 16 || in->page > 256 || (in->page & (in->page - 1))) return CBK_ERR_LAYOUT;
  if (in->block < 16 || in->block > in->page || (in->block & (in->block - 1))) return CBK_ERR_LAYOUT;
  if (in->pages < 1 || in->pages > INT32_MAX || in->heads < 1 || in->heads > 4096) return CBK_ERR_SHAPE;
  if (need_device_ptrs) {
    if (!in->k_codes || !in->v_codes || !in->scales) return CBK_ERR_NULL;
    if (((uintptr_t)in->k_codes | (uintptr_t)in->v_codes | (uintptr_t)in->scales) & 15) return CBK_ERR_ALIGN;
  }
  c->kc = (uint8_t*)in->k_codes; c->vc = (uint8_t*)in->v_codes;
  c->sc = (float2*)in->scales;
  c->pages = in->pages; c->page = in->page; c->shift = __builtin_ctz((unsigned)in->page);
  c->heads = in->heads; c->dim = in->head_dim;
  c->block_shift = __builtin_ctz((unsigned)in->block); c->blocks = in->page / in->block;
  return CBK_OK;
}

static int cache8_io(const cbk_cache8* cache, const cbk_rows* rows, const CacheIo& io, int dt, bool write, void* stream) {
  DCache8 c;
  DRows r;
  int rc = to_dcache8(cache, &c, true);
  if (!rc) rc = to_drows(rows, c.page, &r, true);
  if (rc) return rc;
  if (dt != CBK_F16 && dt != CBK_BF16T && (write || dt != CBK_F32)) return CBK_ERR_DTYPE;
  if (r.tokens == 0 || r.seqs == 0) return CBK_OK;
  const int size = dt == CBK_F32 ? 4 : 2;
  rc = check_dense(io.k, io.kt, io.kh, size);
  if (!rc) rc = check_dense(io.v, io.vt, io.vh, size);
  if (rc) return rc;
  if ((int64_t)r.tokens * c.heads >= (int64_t)1 << 29) return CBK_ERR_SHAPE;       // 2^32 threads of a launch: 4 a row and head at least
  return write ? launch_cache8_write(c, r, io, dt, (hipStream_t)stream) : launch_cache8_read(c, r, io, dt, (hipStream_t)stream);
}

}  // namespace cbk

using namespace cbk;

extern "C" {

size_t cbk_cache_eight_code_bytes(const cbk_cache8* cache) {
  DCache8 c;
  return to_dcache8(cache, &c, false) ? 0 : (size_t)c.pages * c.heads * c.page * c.dim;
}
size_t cbk_cache_eight_scale_bytes(const cbk_cache8* cache) {
  DCache8 c;
  return to_dcache8(cache, &c, false) ? 0 : (size_t)c.pages * c.heads * c.blocks * sizeof(float2);
}

int cbk_cache_eight_write(const cbk_cache8* cache, const cbk_rows* rows, const void* k, int64_t k_row, int64_t k_head,
                          const void* v, int64_t v_row, int64_t v_head, int dtype, void* stream) {
  return cache8_io(cache, rows, CacheIo{(void*)k, (void*)v, k_row, k_head, v_row, v_head}, dtype, true, stream);
}

int cbk_cache_eight_read(const cbk_cache8* cache, const cbk_rows* rows, void* k, int64_t k_row, int64_t k_head,
                         void* v, int64_t v_row, int64_t v_head, int dtype, void* stream) {
  return cache8_io(cache, rows, CacheIo{k, v, k_row, k_head, v_row, v_head}, dtype, false, stream);
}

size_t cbk_cache_eight_attention_workspace_bytes(const cbk_cache8* cache, const cbk_rows* rows, int q_heads) {
  DCache8 c;
  DRows r;
  int ratio;
  if (to_dcache8(cache, &c, false) || to_drows(rows, c.page, &r, false) || attn_ratio(c.heads, r, q_heads, &ratio)) return 0;
  return r.tokens && r.seqs ? cache8_attn_workspace(c, r, ratio) : 0;
}

int cbk_cache_eight_attention(const cbk_cache8* cache, const cbk_rows* rows, const void* q, int64_t q_row, int64_t q_head,
                              void* out, int64_t out_row, int64_t out_head, int dtype, int q_heads, float scale, int window,
                              int sinks, void* workspace, size_t workspace_bytes, void* stream) {
  DCache8 c;
  DRows r;
  AttnArgs a{};
  int rc = to_dcache8(cache, &c, true);
  if (!rc) rc = to_drows(rows, c.page, &r, true);
  if (!rc) rc = attn_ratio(c.heads, r, q_heads, &a.ratio);
  if (rc) return rc;
  if (dtype != CBK_F16 && dtype != CBK_BF16T) return CBK_ERR_DTYPE;
  if (!(scale >= 1e-30f) || scale > 1e30f || window < 0 || sinks < 0) return CBK_ERR_SHAPE;
  if (r.tokens == 0 || r.seqs == 0) return CBK_OK;
  rc = check_dense(q, q_row, q_head, 2);
  if (!rc) rc = check_dense(out, out_row, out_head, 2);
  if (rc) return rc;
  if (((uintptr_t)workspace & 255)) return CBK_ERR_ALIGN;
  set_attn(&a, q, q_row, q_head, out, out_row, out_head, dtype, scale, window, sinks, workspace);
  return launch_cache8_attn(c, r, a, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
