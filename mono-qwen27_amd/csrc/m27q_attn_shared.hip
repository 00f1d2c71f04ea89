// m27q_attn_shared.hip -- attention of sequences that share prefixes.
#include <algorithm>

#include "m27q_attn.h"

namespace m27q {

namespace {

long long tiles_of(long long rows) { return (rows + kWaves * kRows - 1) / (kWaves * kRows); }

// A prefix of many rows and all sequences' own keys in one launch: the prefix's workgroups, bound by the matrix
// units, come first, one on each CU, and beside them those of the own keys, bound by memory.  64 tokens behind
// 32768 places and up to 1021 own ones, 24 heads of 256 on 4, F16 to F32: 117 to 126 us with 9 of joining, where
// 43 would do for the bytes (304 MB at a plain read's 7.15 TB/s) and 59 for the products (the second one in two pieces);
// BF16 to F32, in three pieces, 165 (the paged attention 465), BF16 103 (418); 8 prompts of up to 301 tokens behind
// 8192, BF16: 437 to 447 with 33 of joining, 0.85 PFLOP/s of the pairs that count.  Heads of 256 take all 256 registers:
// BF16 to F32 spills 19 (64 bytes a lane), the others one.
template <int D, bool BF, int NP>
__global__ __launch_bounds__(kWaves * 64, 2) void k_attn_both(const AttnParams p, unsigned px, unsigned prefix, unsigned ox) {
    if (blockIdx.x < prefix) {
        const unsigned by = blockIdx.x / px;
        attn_many<D, BF, NP, kPrefix>(p, blockIdx.x - by * px, by, px, (unsigned)p.prefix_parts);
    } else {
        const unsigned id = blockIdx.x - prefix, by = id / ox;
        attn_many<D, BF, NP, kOwn>(p, id - by * ox, by, ox, (unsigned)(p.splits - p.prefix_parts));
    }
}

// The same of few rows, bound by the latency of a part's steps: 4 tokens behind 32768 places and up to 300 own
// ones, 137 MB, 38.5 us with the join, 3.6 TB/s.
template <int D, bool BF, int NP, int PREFIX_ROWS, int OWN_ROWS>
__global__ __launch_bounds__(kWaves * 64, D == 256 ? 1 : 2) void k_attn_few_both(const AttnParams p, unsigned px, unsigned prefix,
                                                                                  unsigned ox) {
    if (blockIdx.x < prefix) {
        const unsigned by = blockIdx.x / px;
        attn_few<D, BF, NP, PREFIX_ROWS, kPrefix>(p, blockIdx.x - by * px, by);
    } else {
        const unsigned id = blockIdx.x - prefix, by = id / ox;
        attn_few<D, BF, NP, OWN_ROWS, kOwn>(p, id - by * ox, by);
    }
}

template <int D, bool BF, int NP>
void launch_parts(const AttnParams &p, const SharedPlan &plan, hipStream_t s) {
    const int group = (int)(p.q.heads / p.cache.heads);
    const long long pr = (long long)p.prefix.max_rows * group, orows = (long long)p.seqs.max_q * group;
    const unsigned tp = plan.prefix.few ? 1 : (unsigned)tiles_of(pr), to = plan.prefix.few ? 1 : (unsigned)tiles_of(orows);
    const unsigned px = tp * p.prefix.groups * p.cache.heads, ox = to * p.seqs.n * p.cache.heads;
    const unsigned prefix = px * plan.prefix.splits;
    const dim3 grid(prefix + ox * plan.own), block(kWaves * 64);
    auto k = k_attn_both<D, BF, NP>;
    if (plan.prefix.few)
        k = std::max(pr, orows) <= 16 ? k_attn_few_both<D, BF, NP, 16, 16>
            : orows <= 16             ? k_attn_few_both<D, BF, NP, kRows, 16>
                                      : k_attn_few_both<D, BF, NP, kRows, kRows>;
    hipLaunchKernelGGL(k, grid, block, 0, s, p, px, prefix, ox);
}

template <int D, bool BF>
hipError_t launch_t(const AttnParams &p, const SharedPlan &plan, hipStream_t s) {
    constexpr int NP = BF ? 3 : 2;
    if (p.out.type == M27Q_TYPE_F32) launch_parts<D, BF, NP>(p, plan, s);
    else launch_parts<D, BF, 1>(p, plan, s);
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

// Whether a prefix is read once for its group, or by each sequence as the rest of its keys (from the caches
// then, which hold it after the first): what is saved against what a pass of its own costs, from the bounds, as
// if all sequences shared.  In tiles of 32 places of 256 values, by times measured with 4 cache heads of 256
// (24 query heads, F16 to F32): 656 tiles a us of up to 16 rows and 496 of 32 by themselves, 160 of 128 rows of
// a group.  A few rows (of a group 32): what is saved has to be 1200 tiles, for lengths, groups and places are
// looked up one after another; 4 tokens behind 2048, 8192, 16384 and 32768 places 16.6, 24.3, 29.0 and 38.5 us,
// by themselves 13.0, 22.7, 31.1 and 48.3; 9 behind 1560 (8 heads) 15.0 and 19.9.  More: 6 us, and 1 for 400
// tiles of own keys, which have a wave of a workgroup here; 64 tokens and up to 600 own places behind 1024,
// 2048, 8192 and 32768 41.7, 44.1, 66 and 117 and 35.0, 46.4, 117 and 403; 8 x 5 tokens behind 8192, 16384 and
// 32768 37.9, 53.9 and 78.7 and 34.5, 50.5 and 83.4; 3 x 8 x 5 behind 12000 66 and 96.  Prompts save what is
// left over of tiles of 128 rows: 4 of 200 tokens behind 512, 1024 and 4096 49, 61 and 147 and 48, 74 and 165.
// Three numbers do not fit every shape.  Few rows: over 396 cases (2 to 32 sequences behind 1024 to 32768 places, 1 to
// 16 cache heads of 64 to 256) the way taken is 2.8% slower than the other one on average, by more than 10% in 37 of
// them, at most by 61% (5 tokens behind 1024 places, 8 heads of 256: by themselves 20.8 us, shared 12.9; 4 behind
// 8192, 4 heads: 22.5 and 24.3).  Prompts count as if all were as long as the longest: 301, 195, 206, 200, 183, 198, 266
// and 273 tokens behind 8192 places are shared for a saving of 34 of 120 tiles, of which they have 90, and take 445
// us, by themselves 455; one of 2000 and seven of 20 778 and 2640.
bool worth_sharing(const m27q_seqs &seqs, const m27q_prefixes &prefix, long long group, const m27q_cache &cache,
                   long long shared) {
    const double n = seqs.n, groups = prefix.groups;
    const double tile = (double)cache.heads * cache.dim / (256 * kKeys), tiles = shared * tile;
    const long long rows = seqs.max_q * group, together = prefix.max_rows * group;
    const double others = groups * tiles * tiles_of(together) / 160;
    if (rows > kRows) return n * tiles * tiles_of(rows) / 160 - others >= 1.5;
    if (together <= kRows) return (n - groups) * tiles >= 1200;
    return n * tiles / (rows <= 16 ? 656 : 496) - others >= 6 + n * (seqs.max_kv - shared) * tile / 400;
}

}  // namespace

// Workgroups of a part of the keys, the prefixes' and the sequences'.
long long shared_groups(const m27q_seqs &seqs, const m27q_prefixes &prefix, uint32_t q_heads, const m27q_cache &cache) {
    const long long rows = (long long)prefix.max_rows * (q_heads / cache.heads);
    const long long a = tiles_of(rows) * prefix.groups * cache.heads, b = attn_groups(seqs, q_heads, cache);
    return a + b;
}

// The prefix's parts, at most 48 of the join's 64, and those of a sequence's own keys: what runs at once, in one
// launch.  Many rows: a place on a CU for the own keys of each sequence and head, up to one of its two, and the
// others for the prefix.  Few: up to half of the places for the own keys, in parts of 128, a tile a wave, at
// least.  Measured, with other numbers of parts: 64 tokens behind 32768 places 130 us with 21 of the prefix, 161,
// 141, 138 and 150 with 14, 17, 32 and 42; 3 groups of 8 x 5 tokens behind 12000 places 66 with 17, 62, 64, 75
// and 72 with 16, 18, 10 and 21; 8 prompts of 301 behind 8192 places 438 with 1, 474, 500 and 433 with 2, 3 and 4.
// (Each kind in a launch of its own: 150, 80 and 473 us.)  Few rows: 4 tokens behind 2048 places 16.5 with 16,
// 17.2, 17.1 and 17.8 with 11, 22 and 32 (two launches: 23.1); behind 32768 places 38.9 with 48, 40.6, 37.7 and
// 38.4 with 24, 32 and 40; 8 tokens, 8 cache heads of 128, 4096 places and up to 1500 own ones 21.2, 18.5 with
// half as many parts of the own ones.
//
// A sequence usually has as many own keys as the longest has behind the longest prefix: `usual` parts.  But it may
// share less than the bounds say, or nothing: there are parts then as for all of its keys, filling half of the places
// (few rows) or all of them (many, whose tokens have a wave of four: two at least, for up to 32 rounds of workgroups).  A
// sequence that does not need them leaves them at once: 4 tokens behind 32768 places 38 us with and without them, 64
// behind 8192 63, the 3 x 8 x 5 71.2 and 69.9.  4 tokens of 32000 places that share 512 under bounds of 33000 take 113
// us so, with the usual parts 579 (the paged attention 97); 8 x 5 tokens behind 16384 places and 5 of a sequence of 17000
// by itself 112 and 313 (88); 64 tokens behind 32768 places and one of 33000 by itself 910 and 1715 (1110), as a group of
// one 200.
SharedPlan shared_plan(const m27q_seqs &seqs, const m27q_prefixes &prefix, uint32_t q_heads, const m27q_cache &cache,
                       int cus) {
    const long long group = q_heads / cache.heads, slots = 2ll * cus;
    const long long rows = prefix.max_rows * group, wgs = tiles_of(rows) * prefix.groups * cache.heads;
    const long long own = attn_groups(seqs, q_heads, cache);
    const long long shared = prefix.max_len < seqs.max_kv ? prefix.max_len : seqs.max_kv;
    SharedPlan r{};
    // (work-items of the join's grid, 256 for 1024 / dim rows, are less than 2^32)
    const bool joins = (long long)seqs.max_q * q_heads / (1024 / cache.dim) < (1ll << 24) - 1;
    if (!joins || !worth_sharing(seqs, prefix, group, cache, shared)) {
        const AttnPlan each = attn_plan(seqs, q_heads, cache, cus);
        return {{each.few, 0}, each.splits, 0};
    }
    r.prefix.few = rows <= kRows && seqs.max_q * group <= kRows;
    const int least = r.prefix.few ? 128 : 256;
    const long long places = r.prefix.few && cache.dim == 256 ? cus : slots;
    r.prefix.splits = parts_of(wgs, places - std::min(own, places / 2), shared, least, 48);
    const long long left = r.prefix.few ? places - wgs * r.prefix.splits : slots, behind = seqs.max_kv - shared;
    const long long limit = kMaxSplits - r.prefix.splits, usual = parts_of(own, left, behind, least, limit);
    const long long most = r.prefix.few ? places / 2
                           : tiles_of(seqs.max_q * group) > 1 ? places : std::max(places, std::min(2 * own, 64 * places));
    r.own = (int)std::max(usual, (long long)parts_of(own, most, seqs.max_kv, least, limit));
    r.own_least = (int)std::max((long long)least, ((behind + usual - 1) / usual + kKeys - 1) / kKeys * kKeys);
    return r;
}

hipError_t launch_shared(const AttnParams &p, const SharedPlan &plan, hipStream_t s) {
    if (plan.prefix.splits == 0) return launch_attn(p, {plan.prefix.few, plan.own}, s);
    const bool bf = p.cache.type == M27Q_TYPE_BF16;
    switch (p.cache.dim) {
        case 64: return bf ? launch_t<64, true>(p, plan, s) : launch_t<64, false>(p, plan, s);
        case 128: return bf ? launch_t<128, true>(p, plan, s) : launch_t<128, false>(p, plan, s);
        default: return bf ? launch_t<256, true>(p, plan, s) : launch_t<256, false>(p, plan, s);
    }
}

}  // namespace m27q
