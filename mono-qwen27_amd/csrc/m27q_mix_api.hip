// m27q_mix_api.hip -- entry points of the token mixers: argument checks, then
// launches (as m27q_api.hip: every check runs on the host before the first HIP
// call).
#include <cmath>

#include "m27q_internal.h"
#include "m27q_check.h"
#include "m27q_mix.h"

using namespace m27q;

namespace {

m27q_status check_rope(const m27q_rope_plan *r, const int32_t *pos, const m27q_rows &x, const m27q_rows &out) {
    if (!r || !r->turns || !pos) return M27Q_ERR_NULL;
    m27q_status st = check_rows(x, 1024);
    if (st == M27Q_OK) st = check_out(out, 1024);
    if (st != M27Q_OK) return st;
    if (!same_shape(x, out)) return M27Q_ERR_SHAPE;
    if (r->rot < 2 || r->rot % 2 || r->rot > x.dim) return M27Q_ERR_SHAPE;
    if (r->layout != M27Q_ROPE_HALF && r->layout != M27Q_ROPE_PAIRS) return M27Q_ERR_LAYOUT;
    if (!aligned(r->turns, 8) || !aligned(pos, 4)) return M27Q_ERR_LAYOUT;
    if (x.ptr == out.ptr &&
        (x.type != out.type || x.token_stride != out.token_stride || x.head_stride != out.head_stride))
        return M27Q_ERR_LAYOUT;
    return M27Q_OK;
}

}  // namespace

extern "C" {

M27Q_API m27q_status m27q_rope_turns(uint32_t rot, double base, int scaling, double factor, double trained,
                                     uint64_t *turns, float *mscale) {
    if (!turns || !mscale) return M27Q_ERR_NULL;
    if (rot < 2 || rot % 2 || rot > 1024) return M27Q_ERR_SHAPE;
    if (!(base >= 1.0) || std::isinf(base)) return M27Q_ERR_RANGE;
    if (scaling < M27Q_ROPE_PLAIN || scaling > M27Q_ROPE_YARN) return M27Q_ERR_RANGE;
    if (scaling != M27Q_ROPE_PLAIN && (!(factor >= 1.0) || std::isinf(factor))) return M27Q_ERR_RANGE;
    if (scaling == M27Q_ROPE_YARN && (!(trained >= 1.0) || std::isinf(trained) || !(base > 1.0))) return M27Q_ERR_RANGE;
    if (scaling == M27Q_ROPE_NTK && rot <= 2) return M27Q_ERR_SHAPE;
    const double pi = 3.14159265358979323846;
    double low = 0, high = 0;
    *mscale = 1.0f;
    if (scaling == M27Q_ROPE_NTK) base *= std::pow(factor, rot / (rot - 2.0));
    if (scaling == M27Q_ROPE_YARN) {
        // the pair index at which a pair turns that many times in the trained tokens
        auto at = [&](double n) { return rot * std::log(trained / (n * 2 * pi)) / (2 * std::log(base)); };
        low = std::fmax(0.0, std::floor(at(32)));
        high = std::fmin(rot - 1.0, std::ceil(at(1)));
        *mscale = (float)(0.1 * std::log(factor) + 1.0);
    }
    for (uint32_t j = 0; j < rot / 2; ++j) {
        double f = std::pow(base, -2.0 * j / rot);
        if (scaling == M27Q_ROPE_LINEAR) f /= factor;
        if (scaling == M27Q_ROPE_YARN) {
            const double ramp = std::fmin(1.0, std::fmax(0.0, (j - low) / std::fmax(high - low, 1e-3)));
            f = f / factor * ramp + f * (1 - ramp);
        }
        turns[j] = (uint64_t)(f / (2 * pi) * 18446744073709551616.0);  // f <= 1: below a sixth of a turn
    }
    return M27Q_OK;
}

M27Q_API m27q_status m27q_rope(const m27q_rope_plan *rope, const int32_t *pos, int tokens, const m27q_rows *x,
                               const m27q_rows *out, hipStream_t stream) {
    if (!x || !out) return M27Q_ERR_NULL;
    const m27q_status st = check_rope(rope, pos, *x, *out);
    if (st != M27Q_OK) return st;
    if (tokens < 1 || (uint32_t)tokens > kMaxTokens) return M27Q_ERR_SHAPE;
    RopeParams p{};
    p.rope = *rope;
    p.pos = pos;
    p.tokens = tokens;
    p.q = *x;
    p.q_out = *out;
    if (!rope_groups(p, rope_vectorizes(p))) return M27Q_ERR_SHAPE;
    return hip_status(launch_rope(p, stream));
}

M27Q_API m27q_status m27q_rope_append(const m27q_rope_plan *rope, const int32_t *pos, const m27q_seqs *seqs,
                                      const m27q_cache *cache, const m27q_rows *q, const m27q_rows *q_out,
                                      const m27q_rows *k, const m27q_rows *v, hipStream_t stream) {
    if (!q || !q_out || !k || !v) return M27Q_ERR_NULL;
    m27q_status st = check_seqs(seqs);
    if (st == M27Q_OK) st = check_cache(cache);
    if (st == M27Q_OK) st = check_rope(rope, pos, *q, *q_out);
    if (st == M27Q_OK) st = check_rows(*k, 1024);
    if (st == M27Q_OK) st = check_rows(*v, 1024);
    if (st != M27Q_OK) return st;
    if (!same_shape(*k, *v) || k->heads != cache->heads || k->dim != cache->dim || q->dim != cache->dim)
        return M27Q_ERR_SHAPE;
    RopeParams p{};
    p.rope = *rope;
    p.pos = pos;
    p.tokens = (int)seqs->tokens;
    p.q = *q;
    p.q_out = *q_out;
    p.has_cache = 1;
    p.k = *k;
    p.v = *v;
    p.seqs = *seqs;
    p.cache = *cache;
    if (!rope_groups(p, rope_vectorizes(p))) return M27Q_ERR_SHAPE;
    return hip_status(launch_rope(p, stream));
}

M27Q_API size_t m27q_attn_scratch_bytes(const m27q_seqs *seqs, uint32_t q_heads, const m27q_cache *cache) {
    if (!attn_shape(seqs, q_heads, cache)) return 0;
    const m27q_seqs s = bounded(*seqs, *cache);
    return attn_scratch(s, q_heads, cache->dim, attn_plan(s, q_heads, *cache, cu_count()).splits);
}

M27Q_API m27q_status m27q_attn_paged(const m27q_seqs *seqs, const m27q_cache *cache, const m27q_rows *q,
                                     const m27q_rows *out, float scale, int window, void *scratch,
                                     size_t scratch_bytes, hipStream_t stream) {
    if (!q || !out || !scratch) return M27Q_ERR_NULL;
    const m27q_status st = check_attn(seqs, cache, *q, *out, scale, scratch);
    if (st != M27Q_OK) return st;
    if (window < 0) return M27Q_ERR_RANGE;
    AttnParams p{};
    p.seqs = bounded(*seqs, *cache);
    p.cache = *cache;
    p.q = *q;
    p.out = *out;
    p.scale = scale;
    p.window = window;
    const AttnPlan plan = attn_plan(p.seqs, q->heads, *cache, cu_count());
    if (scratch_bytes < attn_scratch(p.seqs, q->heads, cache->dim, plan.splits)) return M27Q_ERR_SCRATCH;
    p.splits = plan.splits;
    p.part = (float *)scratch;
    p.stat = (float2 *)(p.part + (size_t)p.seqs.tokens * q->heads * plan.splits * cache->dim);
    return hip_status(launch_attn(p, plan, stream));
}

M27Q_API size_t m27q_delta_scratch_bytes(uint32_t n, uint32_t tokens, uint32_t max_len, uint32_t heads, uint32_t dk,
                                         uint32_t dv) {
    if (n < 1 || n > kMaxSeqs || tokens < 1 || tokens > kMaxTokens || max_len < 1 || max_len > tokens) return 0;
    if (heads < 1 || heads > kMaxHeads || (dk != 64 && dk != 128) || dv < 16 || dv > 256 || dv % 16) return 0;
    return delta_scratch(n, tokens, max_len, heads, dk, dv);
}

M27Q_API m27q_status m27q_delta_rule(const m27q_delta *d, void *scratch, size_t scratch_bytes, hipStream_t stream) {
    if (!d || !d->start || !d->g || !d->beta || !scratch) return M27Q_ERR_NULL;
    m27q_status st = check_rows(d->q, 128);
    if (st == M27Q_OK) st = check_rows(d->k, 128);
    if (st == M27Q_OK) st = check_rows(d->v, 256);
    if (st == M27Q_OK) st = check_out(d->out, 256);
    if (st != M27Q_OK) return st;
    if (d->q.type != d->v.type || d->k.type != d->v.type || d->out.type != d->v.type) return M27Q_ERR_TYPE;
    if (!same_shape(d->q, d->k) || !same_shape(d->v, d->out) || d->v.heads % d->k.heads) return M27Q_ERR_SHAPE;
    const size_t need = m27q_delta_scratch_bytes(d->n, d->tokens, d->max_len, d->v.heads, d->k.dim, d->v.dim);
    if (!need || d->n_slots > (1u << 24) || (long long)d->n * d->k.heads > kMaxGroups) return M27Q_ERR_SHAPE;
    if (!std::isfinite(d->scale) || d->head_map > M27Q_HEADS_CYCLED) return M27Q_ERR_RANGE;
    if (!rows_aligned(d->q, 16) || !rows_aligned(d->k, 16) || !rows_aligned(d->v, 16) || !rows_aligned(d->out, 16))
        return M27Q_ERR_LAYOUT;
    if (!aligned(d->start, 4) || !aligned(d->slots, 4) || !aligned(d->g, 4) || !aligned(d->beta, 4) ||
        !aligned(d->state_in, 16) || !aligned(d->state_out, 16) || !aligned(scratch, 16))
        return M27Q_ERR_LAYOUT;
    if (scratch_bytes < need) return M27Q_ERR_SCRATCH;
    return hip_status(launch_delta(*d, scratch, stream));
}

}  // extern "C"
