// m27q_attn_shared.hip -- attention of sequences that share prefixes.
#include <algorithm>

#include "m27q_attn.h"

namespace m27q {

namespace {

long long tiles_of(long long rows) { return (rows + kWaves * kRows - 1) / (kWaves * kRows); }

template <int D, bool BF, int NP, Kind KIND>
void launch_kind(const AttnParams &p, bool few, long long rows, unsigned units, int parts, hipStream_t s) {
    if (few) {
        const dim3 grid(units * p.cache.heads, parts);
        constexpr int NW = KIND == kOwn && D == 256 ? 2 : kWaves;
        if (rows <= 16) hipLaunchKernelGGL((k_attn_few<D, BF, NP, 16, KIND, NW>), grid, dim3(NW * 64), 0, s, p);
        else hipLaunchKernelGGL((k_attn_few<D, BF, NP, kRows, KIND, NW>), grid, dim3(NW * 64), 0, s, p);
    } else {
        const dim3 grid((unsigned)(tiles_of(rows) * units * p.cache.heads), parts);
        hipLaunchKernelGGL((k_attn<D, BF, NP, KIND>), grid, dim3(kWaves * 64), 0, s, p);
    }
}

template <int D, bool BF>
hipError_t launch_t(const AttnParams &p, const SharedPlan &plan, hipStream_t s) {
    constexpr int NP = BF ? 3 : 2;
    const int group = (int)(p.q.heads / p.cache.heads);
    const long long pr = (long long)p.prefix.max_rows * group, orows = (long long)p.seqs.max_q * group;
    if (p.out.type == M27Q_TYPE_F32) {
        launch_kind<D, BF, NP, kPrefix>(p, plan.prefix.few, pr, p.prefix.groups, plan.prefix.splits, s);
        launch_kind<D, BF, NP, kOwn>(p, plan.own.few, orows, p.seqs.n, plan.own.splits, s);
    } else {
        launch_kind<D, BF, 1, kPrefix>(p, plan.prefix.few, pr, p.prefix.groups, plan.prefix.splits, s);
        launch_kind<D, BF, 1, kOwn>(p, plan.own.few, orows, p.seqs.n, plan.own.splits, s);
    }
    constexpr int RPB = 4 * 64 / (D / 4);
    const dim3 g2((p.seqs.max_q * p.q.heads + RPB - 1) / RPB, p.seqs.n);
    hipLaunchKernelGGL((k_attn_join<D, BF, kOwn>), g2, dim3(256), 0, s, p);
    return hipGetLastError();
}

// Parts of `keys` keys, as many as run at once: two workgroups on each CU, or one of few rows of 256 (its tiles
// take the LDS).
int parts_of(long long wgs, long long slots, long long keys, long long least, long long limit) {
    return (int)std::max(1ll, std::min({slots / wgs, (keys + least - 1) / least, limit}));
}

}  // namespace

// Workgroups of a part of the keys, the larger of the prefixes' and the sequences'.
long long shared_groups(const m27q_seqs &seqs, const m27q_prefixes &prefix, uint32_t q_heads, const m27q_cache &cache) {
    const long long rows = (long long)prefix.max_rows * (q_heads / cache.heads);
    const long long a = tiles_of(rows) * prefix.groups * cache.heads, b = attn_groups(seqs, q_heads, cache);
    return a > b ? a : b;
}

// The prefix's parts, at most 48 of the join's 64, and those of a sequence's own keys, of which there are as
// many as the longest sequence has behind the longest prefix: parts of 64, a tile for each of two waves, at least.
// Measured, with other numbers of parts: 64 tokens behind 32768 places 150 us with 42 of the prefix, 151 with 21, 32
// and 40; 3 groups of 8 x 5 tokens behind 12000 places 80 with 21, 83 with 16, 98 with 10; 8 prompts of 301
// behind 8192 places 473 with 1, 507, 543 and 472 with 2, 3 and 4.  Own keys: 64 sequences 150 with 2, 156, 154 and 157
// with 1, 3 and 6; 4 sequences 23.1 with 5, 27.8, 25.5 and 24.0 with 1, 2 and 10.
SharedPlan shared_plan(const m27q_seqs &seqs, const m27q_prefixes &prefix, uint32_t q_heads, const m27q_cache &cache,
                       int cus) {
    const long long group = q_heads / cache.heads, slots = 2ll * cus;
    const long long rows = prefix.max_rows * group, wgs = tiles_of(rows) * prefix.groups * cache.heads;
    const long long shared = prefix.max_len < seqs.max_kv ? prefix.max_len : seqs.max_kv;
    SharedPlan r{};
    r.prefix.few = rows <= kRows;
    r.prefix.splits = parts_of(wgs, r.prefix.few && cache.dim == 256 ? cus : slots, shared, r.prefix.few ? 128 : 256, 48);
    r.own.few = (long long)seqs.max_q * group <= kRows;
    r.own.splits = parts_of(attn_groups(seqs, q_heads, cache), slots, (long long)seqs.max_kv - shared, r.own.few ? 64 : 256,
                            kMaxSplits - r.prefix.splits);
    return r;
}

hipError_t launch_shared(const AttnParams &p, const SharedPlan &plan, hipStream_t s) {
    const bool bf = p.cache.type == M27Q_TYPE_BF16;
    switch (p.cache.dim) {
        case 64: return bf ? launch_t<64, true>(p, plan, s) : launch_t<64, false>(p, plan, s);
        case 128: return bf ? launch_t<128, true>(p, plan, s) : launch_t<128, false>(p, plan, s);
        default: return bf ? launch_t<256, true>(p, plan, s) : launch_t<256, false>(p, plan, s);
    }
}

}  // namespace m27q
