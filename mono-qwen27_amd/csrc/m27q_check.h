// m27q_check.h -- argument checks that the entry points of the token mixers and of a batch's steps share (host).
#pragma once

#include <cmath>
#include <cstdint>

#include "m27q_mix.h"

namespace m27q {

constexpr uint32_t kMaxTokens = 1u << 24;   // rows of a call
constexpr uint32_t kMaxSeqs = 65535;        // a grid's y
constexpr uint32_t kMaxKv = 1u << 30;
constexpr uint32_t kMaxHeads = 1024;
constexpr long long kMaxGroups = (1ll << 23) - 1;  // workgroups of up to 512 in a grid's x: below 2^32 work-items

inline bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }

inline bool value_type(uint32_t t) { return t == M27Q_TYPE_F32 || t == M27Q_TYPE_F16 || t == M27Q_TYPE_BF16; }

inline m27q_status check_rows(const m27q_rows &r, uint32_t max_dim) {
    if (!r.ptr) return M27Q_ERR_NULL;
    if (!value_type(r.type)) return M27Q_ERR_TYPE;
    if (r.heads < 1 || r.heads > kMaxHeads || r.dim < 1 || r.dim > max_dim) return M27Q_ERR_SHAPE;
    if (r.token_stride < 0 || r.head_stride < 0 || r.token_stride > INT32_MAX) return M27Q_ERR_SHAPE;
    if (!aligned(r.ptr, (size_t)type_bytes(r.type))) return M27Q_ERR_LAYOUT;
    return M27Q_OK;
}

// Output rows: no head or token on top of the next one.
inline m27q_status check_out(const m27q_rows &r, uint32_t max_dim) {
    const m27q_status st = check_rows(r, max_dim);
    if (st != M27Q_OK) return st;
    if ((r.heads > 1 && r.head_stride < (int64_t)r.dim) || r.token_stride < (int64_t)r.dim) return M27Q_ERR_SHAPE;
    return M27Q_OK;
}

inline bool rows_aligned(const m27q_rows &r, int bytes) {
    const int b = type_bytes(r.type);
    return aligned(r.ptr, (size_t)bytes) && r.token_stride * b % bytes == 0 && r.head_stride * b % bytes == 0;
}

inline bool same_shape(const m27q_rows &a, const m27q_rows &b) { return a.heads == b.heads && a.dim == b.dim; }

inline m27q_status hip_status(hipError_t e) { return e == hipSuccess ? M27Q_OK : M27Q_ERR_HIP; }

inline m27q_status check_cache(const m27q_cache *c) {
    if (!c || !c->k || !c->v) return M27Q_ERR_NULL;
    if (c->type != M27Q_TYPE_F16 && c->type != M27Q_TYPE_BF16) return M27Q_ERR_TYPE;
    if (c->pages < 1 || c->pages > (1u << 30) || c->heads < 1 || c->heads > kMaxHeads || c->dim < 1 || c->dim > 1024)
        return M27Q_ERR_SHAPE;
    if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1))) return M27Q_ERR_SHAPE;
    if (c->page_stride < (int64_t)c->heads * c->page_size * c->dim) return M27Q_ERR_SHAPE;
    if (!aligned(c->k, 2) || !aligned(c->v, 2)) return M27Q_ERR_LAYOUT;
    return M27Q_OK;
}

inline m27q_status check_seqs(const m27q_seqs *s) {
    if (!s || !s->start || !s->kv_len || !s->table) return M27Q_ERR_NULL;
    if (s->n < 1 || s->n > kMaxSeqs || s->table_stride < 1 || s->table_stride > (1u << 30)) return M27Q_ERR_SHAPE;
    if (s->tokens < 1 || s->tokens > kMaxTokens || s->max_q < 1 || s->max_q > s->tokens) return M27Q_ERR_SHAPE;
    if (s->max_kv < 1 || s->max_kv > kMaxKv) return M27Q_ERR_SHAPE;
    if (!aligned(s->start, 4) || !aligned(s->kv_len, 4) || !aligned(s->table, 4)) return M27Q_ERR_LAYOUT;
    return M27Q_OK;
}

// The launch bound on keys: no table reaches further.
inline m27q_seqs bounded(const m27q_seqs &s, const m27q_cache &c) {
    m27q_seqs r = s;
    const unsigned long long reach = (unsigned long long)s.table_stride * c.page_size;
    if (r.max_kv > reach) r.max_kv = (uint32_t)reach;
    return r;
}

inline bool attn_shape(const m27q_seqs *s, uint32_t q_heads, const m27q_cache *c) {
    if (check_seqs(s) != M27Q_OK || check_cache(c) != M27Q_OK) return false;
    if (c->dim != 64 && c->dim != 128 && c->dim != 256) return false;
    if (q_heads < 1 || q_heads > kMaxHeads || q_heads % c->heads || q_heads / c->heads > 64) return false;
    return attn_groups(*s, q_heads, *c) <= kMaxGroups;
}

// What every attention over pages asks of its arguments.
inline m27q_status check_attn(const m27q_seqs *seqs, const m27q_cache *cache, const m27q_rows &q, const m27q_rows &out,
                              float scale, const void *scratch) {
    m27q_status st = check_seqs(seqs);
    if (st == M27Q_OK) st = check_cache(cache);
    if (st == M27Q_OK) st = check_rows(q, 256);
    if (st == M27Q_OK) st = check_out(out, 256);
    if (st != M27Q_OK) return st;
    if (q.type != cache->type || (out.type != cache->type && out.type != M27Q_TYPE_F32)) return M27Q_ERR_TYPE;
    if (!same_shape(q, out) || q.dim != cache->dim || !attn_shape(seqs, q.heads, cache)) return M27Q_ERR_SHAPE;
    if (!std::isfinite(scale)) return M27Q_ERR_RANGE;
    if (!rows_aligned(q, 16) || !rows_aligned(out, out.type == M27Q_TYPE_F32 ? 16 : 8)) return M27Q_ERR_LAYOUT;
    if (!aligned(cache->k, 16) || !aligned(cache->v, 16) || cache->page_stride % 8 || !aligned(scratch, 16))
        return M27Q_ERR_LAYOUT;
    return M27Q_OK;
}

}  // namespace m27q
