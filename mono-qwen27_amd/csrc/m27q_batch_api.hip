// m27q_batch_api.hip -- entry points of the steps that a batch takes around its products and mixers (norms, attention
// behind shared prefixes, sampling): argument checks, then launches (as m27q_api.hip: every check runs on the host
// before the first HIP call).
#include <cmath>

#include "m27q_internal.h"
#include "m27q_check.h"
#include "m27q_mix.h"

using namespace m27q;

namespace {

constexpr uint32_t kMaxDim = 1u << 20;     // of a norm, as a product's K
constexpr uint32_t kMaxActRows = 1u << 16; // as m27q_quant_act
constexpr uint32_t kMaxVocab = 1u << 24;
constexpr uint32_t kMaxSampled = 65535;

// Written where x is read: a thread reads a value before it writes there, if both are at the same place.
bool in_place(const m27q_rows &a, const m27q_rows &b) {
    return a.ptr != b.ptr || (a.type == b.type && a.token_stride == b.token_stride && a.head_stride == b.head_stride);
}

m27q_status check_prefixes(const m27q_prefixes *x, const m27q_seqs *s) {
    if (!x || !x->first || !x->len) return M27Q_ERR_NULL;
    if (x->groups < 1 || x->groups > s->n || x->max_rows < 1 || x->max_rows > s->tokens) return M27Q_ERR_SHAPE;
    if (x->max_len < 1 || x->max_len > kMaxKv) return M27Q_ERR_SHAPE;
    if (!aligned(x->first, 4) || !aligned(x->len, 4)) return M27Q_ERR_LAYOUT;
    return M27Q_OK;
}

bool shared_shape(const m27q_seqs *s, const m27q_prefixes *x, uint32_t q_heads, const m27q_cache *c) {
    return attn_shape(s, q_heads, c) && check_prefixes(x, s) == M27Q_OK && shared_groups(*s, *x, q_heads, *c) <= kMaxGroups;
}

}  // namespace

extern "C" {

M27Q_API m27q_status m27q_rms_norm(const m27q_rows *x, const m27q_rows *add, int tokens, const float *weight, float eps,
                                   const m27q_rows *sum, const m27q_rows *out, void *xq, hipStream_t stream) {
    if (!x || (!sum && !out && !xq)) return M27Q_ERR_NULL;
    m27q_status st = check_rows(*x, kMaxDim);
    if (st == M27Q_OK && add) st = check_rows(*add, kMaxDim);
    if (st == M27Q_OK && sum) st = check_out(*sum, kMaxDim);
    if (st == M27Q_OK && out) st = check_out(*out, kMaxDim);
    if (st != M27Q_OK) return st;
    if ((add && !same_shape(*x, *add)) || (sum && !same_shape(*x, *sum)) || (out && !same_shape(*x, *out)))
        return M27Q_ERR_SHAPE;
    if (tokens < 1 || (uint32_t)tokens > kMaxTokens) return M27Q_ERR_SHAPE;
    const long long K = (long long)x->heads * x->dim;
    if (xq && ((uint32_t)tokens > kMaxActRows || x->dim % 32 || K > kMaxDim)) return M27Q_ERR_SHAPE;
    if (!std::isfinite(eps) || !(eps > 0.0f)) return M27Q_ERR_RANGE;
    if (!aligned(weight, 4) || !aligned(xq, 16)) return M27Q_ERR_LAYOUT;
    for (const m27q_rows *to : {sum, out})
        if (to && (!in_place(*x, *to) || (add && !in_place(*add, *to)))) return M27Q_ERR_LAYOUT;
    if (sum && out && sum->ptr == out->ptr) return M27Q_ERR_LAYOUT;
    NormParams p{};
    p.x = *x;
    if (add) p.add = *add;
    if (sum) p.sum = *sum;
    if (out) p.out = *out;
    p.tokens = tokens;
    p.weight = weight;
    p.eps = eps;
    if (xq) {
        p.q = (int8_t *)xq;
        p.d = (float *)((uint8_t *)xq + m27q_act_d_offset(tokens, (int)K));
        p.s = (uint32_t *)((uint8_t *)xq + m27q_act_s_offset(tokens, (int)K));
    }
    if (!norm_fits(p)) return M27Q_ERR_SHAPE;
    return hip_status(launch_norm(p, stream));
}

M27Q_API size_t m27q_attn_shared_scratch_bytes(const m27q_seqs *seqs, const m27q_prefixes *prefix, uint32_t q_heads,
                                               const m27q_cache *cache) {
    if (!shared_shape(seqs, prefix, q_heads, cache)) return 0;
    const m27q_seqs s = bounded(*seqs, *cache);
    const SharedPlan plan = shared_plan(s, *prefix, q_heads, *cache, cu_count());
    return attn_scratch(s, q_heads, cache->dim, plan.prefix.splits + plan.own);
}

M27Q_API m27q_status m27q_attn_shared(const m27q_seqs *seqs, const m27q_prefixes *prefix, const m27q_cache *cache,
                                      const m27q_rows *q, const m27q_rows *out, float scale, void *scratch,
                                      size_t scratch_bytes, hipStream_t stream) {
    if (!q || !out || !scratch) return M27Q_ERR_NULL;
    m27q_status st = check_attn(seqs, cache, *q, *out, scale, scratch);
    if (st != M27Q_OK) return st;
    st = check_prefixes(prefix, seqs);
    if (st != M27Q_OK) return st;
    if (!shared_shape(seqs, prefix, q->heads, cache)) return M27Q_ERR_SHAPE;
    AttnParams p{};
    p.seqs = bounded(*seqs, *cache);
    p.cache = *cache;
    p.q = *q;
    p.out = *out;
    p.scale = scale;
    p.prefix = *prefix;
    const SharedPlan plan = shared_plan(p.seqs, *prefix, q->heads, *cache, cu_count());
    p.prefix_parts = plan.prefix.splits;
    p.own_least = plan.own_least;
    p.splits = plan.prefix.splits + plan.own;
    if (scratch_bytes < attn_scratch(p.seqs, q->heads, cache->dim, p.splits)) return M27Q_ERR_SCRATCH;
    p.part = (float *)scratch;
    p.stat = (float2 *)(p.part + (size_t)p.seqs.tokens * q->heads * p.splits * cache->dim);
    return hip_status(launch_shared(p, plan, stream));
}

M27Q_API size_t m27q_sample_rows_scratch_bytes(uint32_t rows, uint32_t n) {
    if (rows < 1 || rows > kMaxSampled || n < 1 || n > kMaxVocab) return 0;
    return sample_scratch(rows, n);
}

M27Q_API m27q_status m27q_sample_rows(const m27q_sampling *s, void *scratch, size_t scratch_bytes, hipStream_t stream) {
    if (!s || !s->logits || !s->u || !s->token || !scratch) return M27Q_ERR_NULL;
    if (!value_type(s->type)) return M27Q_ERR_TYPE;
    const size_t need = m27q_sample_rows_scratch_bytes(s->rows, s->n);
    if (!need || s->stride < (int64_t)s->n) return M27Q_ERR_SHAPE;
    if (!aligned(s->logits, (size_t)type_bytes(s->type)) || !aligned(s->temperature, 4) || !aligned(s->top_k, 4) ||
        !aligned(s->top_p, 4) || !aligned(s->min_p, 4) || !aligned(s->u, 4) || !aligned(s->token, 4) ||
        !aligned(s->prob, 4) || !aligned(scratch, 16))
        return M27Q_ERR_LAYOUT;
    if (scratch_bytes < need) return M27Q_ERR_SCRATCH;
    return hip_status(launch_sample_rows(*s, scratch, stream));
}

}  // extern "C"
