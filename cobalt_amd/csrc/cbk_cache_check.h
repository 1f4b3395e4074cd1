// Host-side checks that the entry points of the caches share.
#pragma once
#include "cbk_cache_attn.h"

namespace cbk {

inline int to_drows(const cbk_rows* in, int page, DRows* r, bool need_device_ptrs) {
  if (!in) return CBK_ERR_NULL;
  if (in->seqs < 0 || in->table_cols < 0 || in->ld_table < in->table_cols || in->tokens < 0 || in->tokens >= 1 << 30) return CBK_ERR_SHAPE;
  if (in->table_cols > (1 << 30) / page) return CBK_ERR_SHAPE;    // token positions are ints, tiles round them up
  if (in->seqs == 0 && in->tokens > 0 && !in->starts) return CBK_ERR_SHAPE;
  if (!in->starts && in->seqs && in->tokens % in->seqs) return CBK_ERR_SHAPE;
  if (need_device_ptrs && in->seqs > 0 && in->tokens > 0) {
    if (!in->lens || (in->table_cols && !in->table)) return CBK_ERR_NULL;
    if (((uintptr_t)in->lens | (uintptr_t)in->table | (uintptr_t)in->starts) & 3) return CBK_ERR_ALIGN;
  }
  r->table = (const int32_t*)in->table; r->lens = (const int32_t*)in->lens; r->starts = (const int32_t*)in->starts;
  r->ld = in->ld_table; r->seqs = in->seqs; r->cols = in->table_cols; r->tokens = (int)in->tokens;
  r->per = in->starts || !in->seqs ? 0 : (int)(in->tokens / in->seqs);
  r->cap = in->table_cols * page;
  return CBK_OK;
}

// Rows of `heads` heads of D elements: unit stride along D, 16-byte pieces
inline int check_dense(const void* p, int64_t rs, int64_t hs, int size) {
  if (!p) return CBK_ERR_NULL;
  if (rs < 0 || hs < 0) return CBK_ERR_SHAPE;
  if (((uintptr_t)p & 15) || (rs * size & 15) || (hs * size & 15)) return CBK_ERR_ALIGN;
  return CBK_OK;
}

inline int attn_ratio(int heads, const DRows& r, int q_heads, int* ratio) {
  if (q_heads < 1 || q_heads % heads || (int64_t)r.tokens * q_heads >= (int64_t)1 << 30) return CBK_ERR_SHAPE;
  *ratio = q_heads / heads;
  if (*ratio > 256) return CBK_ERR_SHAPE;                           // (weights of tiles are rows times tokens in 64 bits)
  return CBK_OK;
}

inline void set_attn(AttnArgs* a, const void* q, int64_t q_row, int64_t q_head, void* out, int64_t out_row, int64_t out_head, int dtype, float scale,
                     int window, int sinks, void* workspace) {
  a->q = q; a->out = out;
  a->qt = q_row; a->qh = q_head; a->ot = out_row; a->oh = out_head;
  a->bf = dtype == CBK_BF16T;
  a->scale = scale * 1.44269504088896341f;
  a->window = window >= 1 << 30 ? 0 : window;                       // (positions end below 2^31: such a window hides nothing a table holds)
  a->sinks = sinks < 1 << 30 ? sinks : 1 << 30;
  a->ws = (uint8_t*)workspace;
}

}  // namespace cbk
