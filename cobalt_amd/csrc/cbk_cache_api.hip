// extern "C" entry points of the 4-bit key/value cache: host-side checks and dispatch.  No allocation, no host
// synchronisation, no global state.
#include "cbk_cache.h"
#include "cbk_cache_attn.h"

namespace cbk {

int launch_cache_write(const DCache&, const DRows&, const CacheIo&, int dt, hipStream_t);
int launch_cache_read(const DCache&, const DRows&, const CacheIo&, int dt, hipStream_t);
int launch_cache_attn(const DCache&, const DRows&, AttnArgs, size_t ws_bytes, hipStream_t);
size_t cache_attn_workspace(const DCache&, const DRows&, int ratio);

static int to_dcache(const cbk_cache* in, DCache* c, bool need_device_ptrs) {
  if (!in) return CBK_ERR_NULL;
  if (in->head_dim != 64 && in->head_dim != 128 && in->head_dim != 256) return CBK_ERR_LAYOUT;
  if ((in->group != 32 && in->group != 64 && in->group != 128) || in->group > in->head_dim) return CBK_ERR_LAYOUT;
  if (in->page < 16 || in->page > 256 || (in->page & (in->page - 1))) return CBK_ERR_LAYOUT;
  if (in->pages < 1 || in->pages > INT32_MAX || in->heads < 1 || in->heads > 4096) return CBK_ERR_SHAPE;
  if (need_device_ptrs) {
    if (!in->k_codes || !in->v_codes || !in->k_meta || !in->v_meta) return CBK_ERR_NULL;
    if (((uintptr_t)in->k_codes | (uintptr_t)in->v_codes | (uintptr_t)in->k_meta | (uintptr_t)in->v_meta) & 15) return CBK_ERR_ALIGN;
  }
  c->kc = (uint8_t*)in->k_codes; c->vc = (uint8_t*)in->v_codes;
  c->km = (uint32_t*)in->k_meta; c->vm = (uint32_t*)in->v_meta;
  c->pages = in->pages; c->page = in->page; c->shift = __builtin_ctz((unsigned)in->page);
  c->heads = in->heads; c->dim = in->head_dim; c->group = in->group; c->groups = in->head_dim / in->group;
  return CBK_OK;
}

static int to_drows(const cbk_rows* in, const DCache& c, DRows* r, bool need_device_ptrs) {
  if (!in) return CBK_ERR_NULL;
  if (in->seqs < 0 || in->table_cols < 0 || in->ld_table < in->table_cols || in->tokens < 0 || in->tokens >= 1 << 30) return CBK_ERR_SHAPE;
  if (in->table_cols > (1 << 30) / c.page) return CBK_ERR_SHAPE;    // token positions are ints, tiles round them up
  if (in->seqs == 0 && in->tokens > 0 && !in->starts) return CBK_ERR_SHAPE;
  if (!in->starts && in->seqs && in->tokens % in->seqs) return CBK_ERR_SHAPE;
  if (need_device_ptrs && in->seqs > 0 && in->tokens > 0) {
    if (!in->lens || (in->table_cols && !in->table)) return CBK_ERR_NULL;
    if (((uintptr_t)in->lens | (uintptr_t)in->table | (uintptr_t)in->starts) & 3) return CBK_ERR_ALIGN;
  }
  r->table = (const int32_t*)in->table; r->lens = (const int32_t*)in->lens; r->starts = (const int32_t*)in->starts;
  r->ld = in->ld_table; r->seqs = in->seqs; r->cols = in->table_cols; r->tokens = (int)in->tokens;
  r->per = in->starts || !in->seqs ? 0 : (int)(in->tokens / in->seqs);
  r->cap = in->table_cols * c.page;
  return CBK_OK;
}

// Rows of `heads` heads of D elements: unit stride along D, 16-byte pieces
static int check_dense(const void* p, int64_t rs, int64_t hs, int size) {
  if (!p) return CBK_ERR_NULL;
  if (rs < 0 || hs < 0) return CBK_ERR_SHAPE;
  if (((uintptr_t)p & 15) || (rs * size & 15) || (hs * size & 15)) return CBK_ERR_ALIGN;
  return CBK_OK;
}

static int cache_io(const cbk_cache* cache, const cbk_rows* rows, const CacheIo& io, int dt, bool write, void* stream) {
  DCache c;
  DRows r;
  int rc = to_dcache(cache, &c, true);
  if (!rc) rc = to_drows(rows, c, &r, true);
  if (rc) return rc;
  if (dt != CBK_F16 && dt != CBK_BF16T && (write || dt != CBK_F32)) return CBK_ERR_DTYPE;
  if (r.tokens == 0 || r.seqs == 0) return CBK_OK;
  const int size = dt == CBK_F32 ? 4 : 2;
  rc = check_dense(io.k, io.kt, io.kh, size);
  if (!rc) rc = check_dense(io.v, io.vt, io.vh, size);
  if (rc) return rc;
  if ((int64_t)r.tokens * c.heads * c.dim >= (int64_t)1 << 36) return CBK_ERR_SHAPE;   // 2^32 threads of a launch: 16 numbers each
  return write ? launch_cache_write(c, r, io, dt, (hipStream_t)stream) : launch_cache_read(c, r, io, dt, (hipStream_t)stream);
}

static int attn_ratio(const DCache& c, const DRows& r, int q_heads, int* ratio) {
  if (q_heads < 1 || q_heads % c.heads || (int64_t)r.tokens * q_heads >= (int64_t)1 << 30) return CBK_ERR_SHAPE;
  *ratio = q_heads / c.heads;
  if (*ratio > 256) return CBK_ERR_SHAPE;                           // (weights of tiles are rows times tokens in 64 bits)
  return CBK_OK;
}

}  // namespace cbk

using namespace cbk;

extern "C" {

size_t cbk_cache_code_bytes(const cbk_cache* cache) {
  DCache c;
  return to_dcache(cache, &c, false) ? 0 : (size_t)c.pages * c.heads * c.page * (c.dim / 2);
}
size_t cbk_cache_meta_bytes(const cbk_cache* cache) {
  DCache c;
  return to_dcache(cache, &c, false) ? 0 : (size_t)c.pages * c.heads * c.page * c.groups * 4;
}

int cbk_cache_write(const cbk_cache* cache, const cbk_rows* rows, const void* k, int64_t k_row, int64_t k_head,
                    const void* v, int64_t v_row, int64_t v_head, int dtype, void* stream) {
  return cache_io(cache, rows, CacheIo{(void*)k, (void*)v, k_row, k_head, v_row, v_head}, dtype, true, stream);
}

int cbk_cache_read(const cbk_cache* cache, const cbk_rows* rows, void* k, int64_t k_row, int64_t k_head,
                   void* v, int64_t v_row, int64_t v_head, int dtype, void* stream) {
  return cache_io(cache, rows, CacheIo{k, v, k_row, k_head, v_row, v_head}, dtype, false, stream);
}

size_t cbk_cache_attention_workspace_bytes(const cbk_cache* cache, const cbk_rows* rows, int q_heads) {
  DCache c;
  DRows r;
  int ratio;
  if (to_dcache(cache, &c, false) || to_drows(rows, c, &r, false) || attn_ratio(c, r, q_heads, &ratio)) return 0;
  return r.tokens && r.seqs ? cache_attn_workspace(c, r, ratio) : 0;
}

int cbk_cache_attention(const cbk_cache* cache, const cbk_rows* rows, const void* q, int64_t q_row, int64_t q_head,
                        void* out, int64_t out_row, int64_t out_head, int dtype, int q_heads, float scale, int window,
                        int sinks, void* workspace, size_t workspace_bytes, void* stream) {
  DCache c;
  DRows r;
  AttnArgs a{};
  int rc = to_dcache(cache, &c, true);
  if (!rc) rc = to_drows(rows, c, &r, true);
  if (!rc) rc = attn_ratio(c, r, q_heads, &a.ratio);
  if (rc) return rc;
  if (dtype != CBK_F16 && dtype != CBK_BF16T) return CBK_ERR_DTYPE;
  if (!(scale >= 1e-30f) || scale > 1e30f || window < 0 || sinks < 0) return CBK_ERR_SHAPE;
  if (r.tokens == 0 || r.seqs == 0) return CBK_OK;
  rc = check_dense(q, q_row, q_head, 2);
  if (!rc) rc = check_dense(out, out_row, out_head, 2);
  if (rc) return rc;
  if (((uintptr_t)workspace & 255)) return CBK_ERR_ALIGN;
  a.q = q; a.out = out;
  a.qt = q_row; a.qh = q_head; a.ot = out_row; a.oh = out_head;
  a.bf = dtype == CBK_BF16T;
  a.scale = scale * 1.44269504088896341f;
  a.window = window >= 1 << 30 ? 0 : window;                        // (positions end below 2^31: such a window hides nothing a table holds)
  a.sinks = sinks < 1 << 30 ? sinks : 1 << 30;
  a.ws = (uint8_t*)workspace;
  return launch_cache_attn(c, r, a, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
