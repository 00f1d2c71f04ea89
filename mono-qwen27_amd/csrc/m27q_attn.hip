#include "m27q_attn.h"

namespace m27q {

long long attn_groups(const m27q_seqs &seqs, uint32_t q_heads, const m27q_cache &cache) {
    const long long rows = (long long)seqs.max_q * (q_heads / cache.heads);
    return (rows + kWaves * kRows - 1) / (kWaves * kRows) * seqs.n * cache.heads;
}

namespace {

template <int D, bool BF>
hipError_t launch_t(const AttnParams &p, const AttnPlan &plan, hipStream_t s) {
    constexpr int NP = BF ? 3 : 2;
    const bool full = p.out.type == M27Q_TYPE_F32;
    if (plan.few) {
        const dim3 grid(p.seqs.n * p.cache.heads, p.splits);
        const bool half = p.seqs.max_q * (p.q.heads / p.cache.heads) <= 16;
        if (full && half) hipLaunchKernelGGL((k_attn_few<D, BF, NP, 16>), grid, dim3(kWaves * 64), 0, s, p);
        else if (full) hipLaunchKernelGGL((k_attn_few<D, BF, NP, kRows>), grid, dim3(kWaves * 64), 0, s, p);
        else if (half) hipLaunchKernelGGL((k_attn_few<D, BF, 1, 16>), grid, dim3(kWaves * 64), 0, s, p);
        else hipLaunchKernelGGL((k_attn_few<D, BF, 1, kRows>), grid, dim3(kWaves * 64), 0, s, p);
    } else {
        const dim3 grid((unsigned)attn_groups(p.seqs, p.q.heads, p.cache), p.splits);
        if (full) hipLaunchKernelGGL((k_attn<D, BF, NP>), grid, dim3(kWaves * 64), 0, s, p);
        else hipLaunchKernelGGL((k_attn<D, BF, 1>), grid, dim3(kWaves * 64), 0, s, p);
    }
    if (p.splits > 1) {
        constexpr int RPB = 4 * 64 / (D / 4);
        const dim3 g2((p.seqs.max_q * p.q.heads + RPB - 1) / RPB, p.seqs.n);
        hipLaunchKernelGGL((k_attn_join<D, BF>), g2, dim3(256), 0, s, p);
    }
    return hipGetLastError();
}

}  // namespace

// Parts of the keys.  Rows of several tiles: enough workgroups for two on each CU, parts of
// 256 keys at least.  Few rows: one workgroup on each CU (dim 256: its tiles take the LDS),
// or two, and twice that from 64 pairs of sequence and head on, for ragged ones to even out,
// unless the pairs fill the CUs; parts of 128 keys at least, a tile for each wave.  Measured
// at one, two and four times that: dim 256, 2 sequences of 32768 keys 60 / 71 / 70 us, 32 of
// 16381 293 / 289 / 291, 64 of 3000 112 / 118 / 123; dim 128, 2 of 16384 30 / 35 / 35, 16 of
// 8000 83 / 85 / 88; dim 64, 2 of 16384 20 / 23 / 23, 16 of 8000 49 / 48 / 49.
AttnPlan attn_plan(const m27q_seqs &seqs, uint32_t q_heads, const m27q_cache &cache, int cus) {
    const bool few = (long long)seqs.max_q * (q_heads / cache.heads) <= kRows;
    const long long wgs = attn_groups(seqs, q_heads, cache), least = few ? 128 : 256;
    const long long once = few ? (long long)cus * (cache.dim == 256 ? 1 : 2) * (wgs < 64 || wgs >= cus ? 1 : 2) : 2ll * cus;
    const long long want = (once + wgs - 1) / wgs, most = (seqs.max_kv + least - 1) / least;
    long long splits = want < most ? want : most;
    if (splits > kMaxSplits) splits = kMaxSplits;
    return {few, splits < 1 ? 1 : (int)splits};
}

size_t attn_scratch(const m27q_seqs &seqs, uint32_t q_heads, uint32_t dim, int splits) {
    if (splits <= 1) return 16;
    return (size_t)seqs.tokens * q_heads * splits * (dim * 4 + 8);
}

hipError_t launch_attn(const AttnParams &p, const AttnPlan &plan, hipStream_t s) {
    const bool bf = p.cache.type == M27Q_TYPE_BF16;
    switch (p.cache.dim) {
        case 64: return bf ? launch_t<64, true>(p, plan, s) : launch_t<64, false>(p, plan, s);
        case 128: return bf ? launch_t<128, true>(p, plan, s) : launch_t<128, false>(p, plan, s);
        default: return bf ? launch_t<256, true>(p, plan, s) : launch_t<256, false>(p, plan, s);
    }
}

}  // namespace m27q
