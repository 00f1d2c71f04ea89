// m27q_sample.hip -- a token for each row of logits.
//
// In order of value (equal ones in order of index) token i of a row has the weight
// w_i = e^((l_i - max) / T).  What is kept is a prefix of that order: the first
// top_k, of these the ones with w_i >= min_p, of these the shortest prefix whose
// sum reaches top_p times the sum of the first top_k.  The token is the first
// whose running sum reaches u times the sum of what is kept.
//
// Weights are summed as 64-bit integers, so that no order of adding changes a
// sum, each rounded by 2^-36 of its size at most.
//
// Nothing is sorted but the few hundred tokens among which the borders lie.  Four
// launches:
//   parts  the logits read once: a part's weights summed by bins of a sixteenth of an octave
//   plan   a row's bins from its parts', and those that can hold a border
//   list   the tokens of these bins, from a second reading (parts without any are passed over)
//   pick   a row's list in order, its running sums, the borders, the token
// Where the list would be too long (flat rows, thousands of equal logits at a border), pick reads the whole
// row once or twice more for each border, by pieces of its bin's keys.
//
// 200 rows of 248320 F32, top-p (199 MB): 92 to 103 us from card to card, of these 50 to 52 for parts, 8, 25 for
// list (7.8 TB/s: what parts read last still lies in the caches) and 10.  parts is bound by the vector units: some 30
// operations of a wave for each 64 tokens, half of them on 64 bits, and the LDS additions beside them (a
// plain read of the same bytes: 28).  64 rows of all rules 45 to 48 us (19, 8.5, 12, 8); one row
// 23 to 24: four launches of 5.3, 8, 5.3 and 6, each the latency of its steps (the 40 largest and the choice among them,
// m27q_topk and m27q_sample, take 14).  64 rows of normal logits
// (deviation 2.2) at temperature 2 or 5 with top-p, 10000 tokens a bin, 197 and 228 (342 and 402 where tokens near a border
// do not wait until they fill a wave, 850 and 890 by 11 bits of all keys at a time, 2100 and 2890 by 8); equal logits
// throughout 1070 without cuts, up to 3200 with all.
#include "m27q_device.h"
#include "m27q_mix.h"

namespace m27q {

namespace {

constexpr int kRowThreads = 1024;  // of a workgroup that works on one row

// Descending order of keys: value, then the lower index; -0 as +0; NaN behind every number.
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t b = __float_as_uint(v);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0;
    if ((b & 0x7fffffffu) == 0) return 0x80000000u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float v, int i) {
    return (uint64_t)order_bits(v) << 24 | (0xffffffu - (uint32_t)i);
}
constexpr uint64_t kLastKey = (uint64_t)0xff800000 << 24 | 0xffffff;  // of infinity
__device__ __forceinline__ int key_index(uint64_t key) { return (int)(0xffffffu - (uint32_t)(key & 0xffffffu)); }

__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 24);
    return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}

// What a row is sampled with.
struct Rule {
    double inv_t;   // 1 / T
    double top_p, min_p, u;
    int k;          // candidates
    bool greedy;
};
__device__ __forceinline__ Rule row_rule(const m27q_sampling &p, int row) {
    Rule r;
    const float t = p.temperature ? p.temperature[row] : 1.0f;
    r.greedy = !(t > 0.0f);
    r.inv_t = r.greedy ? 1.0 : 1.0 / (double)t;
    const int k = p.top_k ? p.top_k[row] : 0;
    r.k = k <= 0 || k > (int)p.n ? (int)p.n : k;
    const float tp = p.top_p ? p.top_p[row] : 1.0f, mp = p.min_p ? p.min_p[row] : 0.0f, u = p.u[row];
    r.top_p = tp < 1.0f ? fmax((double)tp, 0.0) : 1.0;  // (NaN cuts nothing)
    r.min_p = mp > 0.0f ? (double)mp : 0.0;
    r.u = u > 0.0f ? fmin((double)u, 1.0) : 0.0;
    return r;
}

// ------------------------------------------------------------------ bins --
//
// Weights are told apart by y = 16 log2(e) l / T, a sixteenth of an octave a unit.  The tokens of a
// row fall into bins by their distance from an anchor, the octave at or above the largest: 384
// bins of a unit, 127 of an octave, and what lies below those 151 octaves counts for nothing.
// Units are absolute (y rounded), anchors whole octaves: bins of parts of a row with anchors of
// their own add up.  A bin holds how many tokens and the sum of their weights, in 2^-36 of
// the weight at its octave's upper end.

constexpr int kUnit = 16;               // units of an octave
constexpr int kFine = 384, kCoarse = 127;
constexpr int kBins = kFine + kCoarse;  // bin kBins: nothing
constexpr int kOctaves = kFine / kUnit; // of the fine bins, whose sums a part has too
constexpr int kStored = kBins + 1 + kOctaves;
constexpr int kMassBits = 36, kSumBits = 50;
constexpr int kPart = 8192;             // tokens of a part: counts of 14 bits above sums of 50
constexpr double kUnitsPerNat = 16 * 1.4426950408889634074;

// Weights of places within an octave, k units and z down it: 2^(-(k + z) / 16), from a table for k and the
// Taylor polynomial for |z| <= 1 / 2 (degree 5: the next term is below 2^-42), in 2^-36.  The
// constants are kept in registers: scalar ones, but for what a product's or sum's second one has to be.
struct Weights {
    double c[6], add;
    const double *octave;  // 2^(36 - k / 16), in LDS
    __device__ __forceinline__ Weights(const double *octave) : octave(octave) {
        constexpr double a = -0.69314718055994530942 / kUnit;
        c[0] = 1.0;
        c[1] = a;
        c[2] = a * a / 2;
        c[3] = a * a * a / 6;
        c[4] = a * a * a * a / 24;
        c[5] = a * a * a * a * a / 120;
        add = 0x1p52;
        asm("" : "+s"(c[1]), "+s"(c[2]), "+s"(c[3]), "+v"(c[4]), "+s"(c[5]), "+v"(add));
    }
    // threads 0 .. 15
    static __device__ __forceinline__ double factor(int k) { return exp2(kMassBits - k * (1.0 / kUnit)); }
    // `count` above the bits of a sum.  Rounded by an addition that leaves the whole number in the low
    // bits; 2^52's exponent off and the count on in one subtraction.
    __device__ __forceinline__ unsigned long long mass(double z, int k, unsigned count) const {
        double p = c[5];
#pragma unroll
        for (int i = 4; i >= 0; --i) p = __builtin_fma(p, z, c[i]);
        const unsigned long long m = __builtin_bit_cast(unsigned long long, __builtin_fma(p, octave[k], add));
        return (unsigned long long)((uint32_t)(m >> 32) - (0x43300000u - (count << (kSumBits - 32)))) << 32 | (uint32_t)m;
    }
};

// What a row's logits are placed by.
constexpr int kReach = kFine + kUnit * kCoarse;  // units down to where weights end
struct Scale {
    double c;       // units of a logit
    double anchor;
    bool wide;      // distances from the anchor are not whole numbers of 2^26 at most, T is infinite, or a step of the
                    // smallest logits is no small part of a unit
};
__device__ __forceinline__ Scale row_scale(const Rule &r, double anchor) {
    const double far = fabs(anchor) + kReach;
    const double c = kUnitsPerNat * r.inv_t;
    return {c, anchor, __builtin_amdgcn_readfirstlane(!(far < 0x1p26) || !(c > 0.0) || c > 0x1p140) != 0};
}

// A logit in whole units, and what is left over: of the exact product, rounded once, whatever anchor it is
// measured from, so that parts of a row and the row count a token in the same bin.  From 2^50 units on a
// step of a logit is thousands of octaves and only equal ones have a weight: there the rounded product does.
__device__ __forceinline__ double units_of(double l, double c, double &z) {
    const double y = l * c;
    const bool near = fabs(y) < 0x1p50;
    const double b = near ? __builtin_fma(l, c, 0x1.8p52) - 0x1.8p52 : __builtin_rint(y);
    z = near ? __builtin_fma(l, -c, b) : 0.0;
    return b;
}

// The same for logits less than 2^26 units from the anchor: how far down from it, the whole number in the low bits of an
// addition.
__device__ __forceinline__ uint32_t units_down(double l, double c, double low, double &z) {
    const double t = __builtin_fma(l, -c, low);  // low = anchor + 1.5 2^52
    z = __builtin_fma(l, -c, low - t);           // (the difference is a whole number below 2^27)
    return (uint32_t)__builtin_bit_cast(unsigned long long, t);
}

// The bin of a logit, and its place in its octave.
struct Place {
    int bin, k;
    double z;
};
__device__ __forceinline__ int bin_of(uint32_t d) { return (int)min(d, (d >> 4) + (kFine - kFine / kUnit)); }
__device__ __forceinline__ Place place_of(float l, const Scale &s) {
    Place p{kBins, 0, 0};
    const double far = s.anchor - units_of((double)l, s.c, p.z);
    if (!(far < kReach)) return p;  // (-infinity and NaN too)
    const uint32_t d = (uint32_t)far;
    p.bin = bin_of(d);
    p.k = (int)(d & (kUnit - 1));
    return p;
}
// The weight at the upper end of a bin's octave, of that at the anchor.
__device__ __forceinline__ int bin_distance(int bin) { return bin < kFine ? bin : kFine + kUnit * (bin - kFine); }
__device__ __forceinline__ double bin_scale(int bin) { return __builtin_ldexp(1.0, -(bin_distance(bin) / kUnit)); }

// The logits of a range of bins, and a little more than those.
struct LogitRange {
    float lo, hi;
};
__device__ __forceinline__ LogitRange logits_of(const Scale &s, int first, int last) {
    if (!(s.c > 1e-30)) return {-__builtin_inff(), __builtin_inff()};
    const double up = (s.anchor - bin_distance(first) + 0.5) / s.c;
    const double down = (s.anchor - bin_distance(last) - (last < kFine ? 0.5 : kUnit - 0.5)) / s.c;
    return {(float)(down - fabs(down) * 0x1p-20), (float)(up + fabs(up) * 0x1p-20)};
}

// What is kept of a part of a row, and of a row.
struct Part {
    double anchor;        // -infinity: no token of any weight
    uint64_t best;        // the largest key
};
constexpr int kList = 8192;
constexpr int kRanges = 4;
constexpr int kMinBins = 3;  // at most, in which min_p's border lies
struct RowPlan {
    double anchor;
    uint64_t best;
    int state;            // 0: done; 1: the tokens of marked bins make a list; 2: the whole row is gone through
    uint32_t listed;      // tokens on the list
    unsigned long long min_p_sum;         // of the tokens that min_p leaves, where none of its border's bins cuts them
    int min_first, min_last;              // those bins
    int first[kRanges], last[kRanges];    // the marked bins
    float lo[kRanges], hi[kRanges];       // their logits lie within these
    float least;                          // and above this
    uint32_t before[kBins + 1];           // tokens of the bins above
    uint32_t at[kBins + 1];               // ... that are on the list
    unsigned long long sum[kBins + 1];    // their weights, in units of sum_unit
    double unit[kBins + 1];               // those units in 2^-36 of the weight at the bin's upper end
};
struct Scratch {
    Part *part;                 // [rows][parts]
    unsigned long long *bins;   // [rows][parts][kStored]
    RowPlan *plan;              // [rows]
    uint64_t *list;             // [rows][kList]
    int parts;                  // of a row
};

// 2^-36 of the anchor's weight, the unit of its octave's bins, in the units of a row's sums, which fit 62 bits.
__device__ __forceinline__ double sum_unit(uint32_t n) {
    return (double)(1ull << (62 - (32 - __builtin_clz(n)))) / (double)(1ull << kMassBits);
}
// A bin's weights in the units of a row's sums.
__device__ __forceinline__ unsigned long long row_mass(unsigned long long mass, double unit) {
    return (unsigned long long)__builtin_rint((double)mass * unit);
}

template <typename T>
__device__ __forceinline__ float logit(const void *p, long long at) { return (float)((const T *)p)[at]; }

constexpr int kPartThreads = 512;
constexpr int kEach = kPart / kPartThreads;
constexpr int kCopies = 4;  // of a part's bins: lanes that meet in a bin wait for each other

// The i-th of a thread's tokens in a part.
__device__ __forceinline__ int part_index(int i) { return i * kPartThreads + (int)threadIdx.x; }

// A part's logits, all on their way at once; NaN behind the end, which no comparison takes (a border's range may reach
// down to -infinity).
template <typename T>
__device__ __forceinline__ void load_part(const m27q_sampling &p, int row, int first, float (&v)[kEach]) {
    const int count = min(kPart, (int)p.n - first);
    const T *const from = (const T *)p.logits + ((long long)row * p.stride + first);
    if (count == kPart) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) v[i] = (float)(from + i * kPartThreads)[threadIdx.x];
        return;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] = (float)from[min(part_index(i), count - 1)];
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] = part_index(i) < count ? v[i] : __builtin_nanf("");
}

// A part's bins, and its largest token.
template <typename T>
__global__ __launch_bounds__(kPartThreads) void k_sample_parts(const m27q_sampling p, const Scratch sc) {
    static_assert(kPartThreads == kBins + 1, "a thread a bin");
    constexpr int W = kPartThreads / 64;
    __shared__ unsigned long long bins[(kBins + 1) * kCopies];
    __shared__ double octave[kUnit];
    __shared__ float top_s[W];
    __shared__ int at_s[W];
    const int row = blockIdx.y, first = (int)blockIdx.x * kPart;
    float v[kEach];
    load_part<T>(p, row, first, v);
    const Rule r = row_rule(p, row);
#pragma unroll
    for (int i = 0; i < kCopies; ++i) bins[i * (kBins + 1) + threadIdx.x] = 0;
    if (threadIdx.x < kUnit) octave[threadIdx.x] = Weights::factor(threadIdx.x);
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kEach; ++i) top = fmaxf(top, v[i]);
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float mine = top;
    if (lane == 0) top_s[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top = fmaxf(top, top_s[i]);
    int at = 0x7fffffff;
    if (__builtin_amdgcn_readfirstlane(mine == top)) {
#pragma unroll
        for (int i = kEach - 1; i >= 0; --i) at = v[i] == top ? part_index(i) : at;
#pragma unroll
        for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o));
    }
    if (lane == 0) at_s[wave] = at;

    const bool any = !r.greedy && __builtin_isfinite(top);
    double z;
    const double b = units_of((double)top, kUnitsPerNat * r.inv_t, z);
    const Scale s = row_scale(r, any ? ceil(b * (1.0 / kUnit)) * kUnit : -__builtin_inf());
    if (any) {
        const Weights w(octave);
        const int copy = lane & (kCopies - 1);
        if (s.wide) {
#pragma unroll 1
            for (int i = 0; i < kEach; ++i) {
                const Place a = place_of(v[i], s);
                if (a.bin < kBins) atomicAdd(&bins[a.bin * kCopies + copy], w.mass(a.z, a.k, 1));
            }
        } else {
            // the same without branches, several tokens' chains beside each other.  A logit above this one is
            // less than 16 units past the last bin (rounded to a float it is off by 4 units at most, 2^-24 of 2^26
            // or, among the smallest, c 2^-150): what is further down, -infinity and NaN are left out by it.
            const float least = fmaxf((float)((s.anchor - (kReach + kUnit / 2)) / s.c), -0x1.fffffep+127f);
            const double low = s.anchor + 0x1.8p52;
            constexpr int AT = 4;
#pragma unroll
            for (int i0 = 0; i0 < kEach; i0 += AT) {
                unsigned long long m[AT];
                int bin[AT];
#pragma unroll
                for (int j = 0; j < AT; ++j) {
                    double z;
                    const uint32_t d = units_down((double)v[i0 + j], s.c, low, z);
                    bin[j] = bin_of(d);
                    m[j] = w.mass(z, (int)(d & (kUnit - 1)), 1);
                }
#pragma unroll
                for (int j = 0; j < AT; ++j) asm volatile("" : "+v"(m[j]), "+v"(bin[j]));  // computed by now, for all lanes
#pragma unroll
                for (int j = 0; j < AT; ++j)
                    if (v[i0 + j] >= least) atomicAdd(&bins[bin[j] * kCopies + copy], m[j]);
            }
        }
    }
    __syncthreads();
    const long long me = (long long)row * sc.parts + blockIdx.x;
    if (threadIdx.x == 0) {
        for (int i = 0; i < W; ++i) at = min(at, at_s[i]);
        const bool none = at >= (int)p.n - first;  // NaN alone
        sc.part[me] = {s.anchor, order_key(none ? __builtin_nanf("") : top, first + (none ? 0 : at))};
    }
    if (!any) return;  // its anchor says so
    unsigned long long sum = 0;
#pragma unroll
    for (int j = 0; j < kCopies; ++j) sum += bins[threadIdx.x * kCopies + j];
    sc.bins[me * kStored + threadIdx.x] = sum;
    // the octaves of the fine bins, 16 lanes each, for a row whose anchor lies so far above that they are one bin there
    if (threadIdx.x < kFine) {
#pragma unroll
        for (int o = kUnit / 2; o; o >>= 1) sum += __shfl_xor(sum, o);
        if ((threadIdx.x & (kUnit - 1)) == 0) sc.bins[me * kStored + kBins + 1 + threadIdx.x / kUnit] = sum;
    }
}

// Lanes' values moved up by DPP within a wave, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long moved(unsigned long long v) {
    return (unsigned long long)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | moved<CTRL, ROWS>((uint32_t)v);
}
// The running sum over a wave's lanes, the lane's own included: 1, 2, 4, 8 lanes up within rows of 16,
// then a row's last to the next row, and the lower half's last to the upper half.
template <typename T>
__device__ __forceinline__ T scan_wave(T v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}

// The running sums of a workgroup's values, one a thread: before this thread's, and all of them.
// `lds` is used once between barriers of the caller's.
template <int THREADS, typename T>
__device__ __forceinline__ T scan_group(T v, T *lds, T &all) {
    constexpr int W = THREADS / 64;
    const int wave = threadIdx.x >> 6;
    const T run = scan_wave(v);
    if ((threadIdx.x & 63) == 63) lds[wave] = run;
    __syncthreads();
    T before = 0;
    all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const T x = lds[i];
        before += i < wave ? x : T(0);
        all += x;
    }
    return before + run - v;
}

// Where a part whose anchor lies `off` units (whole octaves) below the row's has the sum for the row's bin J: the same
// bin's, or, where an octave of the row lies among the part's fine bins, their octave's.  -1: it has none.
__device__ __forceinline__ int part_bin(int J, int off) {
    const int oct = kOctaves + J - kFine - off / kUnit;
    if (J < kFine) return max(J - off, -1);
    return J >= kBins ? -1 : oct >= kOctaves ? kFine + oct - kOctaves : oct >= 0 ? kBins + 1 + oct : -1;
}

constexpr int kPlanThreads = 512, kHalves = 2;
static_assert(kBins + 1 == kPlanThreads, "a thread a bin");

// The largest of a wave's values, all above 0, for every lane.
__device__ __forceinline__ unsigned long long max_wave(unsigned long long v) {
    v = max(v, moved<0x111, 0xf>(v));
    v = max(v, moved<0x112, 0xf>(v));
    v = max(v, moved<0x114, 0xf>(v));
    v = max(v, moved<0x118, 0xf>(v));
    v = max(v, moved<0x142, 0xa>(v));
    v = max(v, moved<0x143, 0xc>(v));
    const uint32_t high = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63);
    return (unsigned long long)high << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// Numbers in their order as bits, and back.
__device__ __forceinline__ unsigned long long ordered(double v) {
    const long long b = __builtin_bit_cast(long long, v);
    return (unsigned long long)(b ^ (b >> 63 | (long long)(1ull << 63)));
}
__device__ __forceinline__ double unordered(unsigned long long u) {
    return __builtin_bit_cast(double, u >> 63 ? u ^ 1ull << 63 : ~u);
}

// The first of `n` <= 512 values that do not descend which reaches a target (n: none does), by a wave: of every
// eighth, then of eight.
template <typename T, typename F>
__device__ __forceinline__ int first_of(const T *v, int n, F reaches) {
    const int lane = threadIdx.x & 63;
    const unsigned long long far = __ballot(8 * lane < n && reaches(v[min(8 * lane + 7, n - 1)]));
    if (!far) return n;
    const int i = 8 * __builtin_ctzll(far), j = min(i + (lane & 7), n - 1);
    return i + __builtin_ctzll(__ballot(reaches(v[j])));
}

// A row's bins from those of its parts, and the bins in which its borders can lie: of the top_k-th
// token, of top_p, of min_p and of the pick.  What is not known before another border is found
// leaves a range of bins.  A chain of steps that wait for each other bounds it: each wave does
// for itself what is not a bin's (it took 11.4 us with the workgroup's threads looking for each border, 8.9
// with all parts by the same threads; 8 now, of which loading and adding the parts' bins is a half).
__global__ __launch_bounds__(kHalves * kPlanThreads) void k_sample_plan(const m27q_sampling p, const Scratch sc) {
    constexpr int W = kPlanThreads / 64;
    __shared__ unsigned long long mass_s[W], sum[kBins + 2];
    __shared__ uint32_t count_s[W], tokens_s[kBins + 2];  // down to a bin, without it
    const int row = blockIdx.x, J = threadIdx.x & (kPlanThreads - 1), lane = J & 63, wave = J >> 6;
    const int half = __builtin_amdgcn_readfirstlane(threadIdx.x / kPlanThreads);
    const Part *part = sc.part + (long long)row * sc.parts;
    const Rule r = row_rule(p, row);
    RowPlan &out = sc.plan[row];
    unsigned long long best = 0, high = 0;
    double anchors = 0;  // of the first 64 parts, a lane each
    for (int i = lane; i < sc.parts; i += 64) {
        const Part x = part[i];
        if (i == lane) anchors = x.anchor;
        high = max(high, ordered(x.anchor));
        best = max(best, (unsigned long long)x.best);
    }
    best = max_wave(best);
    const double anchor = unordered(max_wave(high));
    const float top = key_value(best);
    if (r.greedy || !__builtin_isfinite(top)) {
        if (threadIdx.x == 0) {
            p.token[row] = key_index(best);
            if (p.prob) p.prob[row] = 1.0f;
            out.state = 0;
        }
        return;
    }

    // this thread's bin, from one stored sum of each part; half of the threads have the one half of the parts
    unsigned long long mass = 0;
    uint32_t count = 0;
    constexpr unsigned long long kMask = (1ull << kSumBits) - 1;
    constexpr int kSkip = 1 << 20, AT = 16;  // parts on their way at a time
    int offs = kSkip;
    for (int i0 = half * AT; i0 < sc.parts; i0 += kHalves * AT) {
        if (i0 % 64 < kHalves * AT) {
            const int i = i0 - i0 % 64 + lane;
            if (i0 >= 64) anchors = part[min(i, sc.parts - 1)].anchor;
            offs = i < sc.parts && anchor - anchors < kReach ? (int)(anchor - anchors) : kSkip;
        }
        const unsigned long long *bins = sc.bins + ((long long)row * sc.parts + i0) * kStored;
        unsigned long long x[AT];
        bool ok[AT];
#pragma unroll
        for (int k = 0; k < AT; ++k) {
            const int off = __builtin_amdgcn_readlane(offs, i0 % 64 + k), from = part_bin(J, off);
            ok[k] = off != kSkip && from >= 0;
            x[k] = bins[(off != kSkip ? k * kStored : 0) + (ok[k] ? from : 0)];
        }
#pragma unroll
        for (int k = 0; k < AT; ++k) {
            count += ok[k] ? (uint32_t)(x[k] >> kSumBits) : 0u;
            mass += ok[k] ? x[k] & kMask : 0ull;
        }
    }
    if (half) {
        sum[J] = mass;
        tokens_s[J] = count;
    }
    __syncthreads();
    if (half) return;
    mass += sum[J];
    count += tokens_s[J];
    const double unit = sum_unit(p.n) * bin_scale(J);
    mass = row_mass(mass, unit);
    unsigned long long above = scan_wave(mass);
    uint32_t before = scan_wave(count);
    if (lane == 63) {
        mass_s[wave] = above;
        count_s[wave] = before;
    }
    __syncthreads();
    above -= mass;
    before -= count;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        above += i < wave ? mass_s[i] : 0ull;
        before += i < wave ? count_s[i] : 0u;
    }
    sum[J] = above;
    tokens_s[J] = before;
    if (J == kBins) {
        sum[kBins + 1] = above + mass;
        tokens_s[kBins + 1] = before + count;
    }
    __syncthreads();

    const unsigned long long total = sum[kBins];
    const uint32_t tokens = tokens_s[kBins];
    // the bin in which the running sum reaches a target, the last one that holds a token if none does
    const auto bin_at = [&](double target) {
        const double t = fmax(target, 1.0);   // (the first token's own bin holds far more)
        return first_of(sum + 1, kBins, [&](unsigned long long v) { return (double)v >= t || v == total; });
    };
    const bool k_cuts = (uint32_t)r.k < tokens;
    const int kb = k_cuts ? first_of(tokens_s + 1, kBins, [&](uint32_t v) { return v >= (uint32_t)r.k; }) : kBins;
    // the sum of the first top_k
    const double s_lo = (double)(k_cuts ? sum[kb] : total), s_hi = (double)(k_cuts ? sum[kb + 1] : total);
    double t_lo = s_lo, t_hi = s_hi;  // the sum of what is kept
    int p0 = kBins, p1 = -1, m0 = kBins, m1 = -1;
    unsigned long long min_p_sum = total;
    if (r.top_p < 1.0) {
        p0 = bin_at(r.top_p * s_lo);
        p1 = bin_at(r.top_p * s_hi);
        t_lo = fmin(t_lo, (double)sum[p0]);
        t_hi = fmin(t_hi, (double)sum[p1 + 1]);
    }
    if (r.min_p > 0.0) {
        // the bin of the weight min_p, and its neighbours for what rounding does
        const double y = (double)top * (kUnitsPerNat * r.inv_t) + kUnit * log2(r.min_p), d = anchor - __builtin_rint(y);
        if (d < kReach) {
            const int m = d < 0 ? 0 : d < kFine ? (int)d : kFine + ((int)d - kFine) / kUnit;
            m0 = max(m - 1, 0);
            m1 = min(m + 1, kBins - 1);
            min_p_sum = sum[m1 + 1];
            t_lo = fmin(t_lo, (double)sum[m0]);
            t_hi = fmin(t_hi, (double)min_p_sum);
        }
    }
    const int q0 = bin_at(r.u * t_lo), q1 = bin_at(r.u * t_hi);
    // the marked ranges in order, without what an earlier one has
    int b0[kRanges] = {k_cuts ? kb : kBins, p0, m0, q0}, b1[kRanges] = {k_cuts ? kb : -1, p1, m1, q1};
#pragma unroll
    for (int i = 1; i < kRanges; ++i)
#pragma unroll
        for (int j = kRanges - 1; j >= i; --j)
            if (b0[j] < b0[j - 1]) {
                const int x = b0[j], y = b1[j];
                b0[j] = b0[j - 1];
                b1[j] = b1[j - 1];
                b0[j - 1] = x;
                b1[j - 1] = y;
            }
    uint32_t at = 0, listed = 0;
    int end = -1;
#pragma unroll
    for (int j = 0; j < kRanges; ++j) {
        b0[j] = max(b0[j], end + 1);
        end = max(end, b1[j]);
        if (b1[j] < b0[j]) continue;
        const uint32_t from = tokens_s[b0[j]];
        at += tokens_s[min(max(J, b0[j]), b1[j] + 1)] - from;
        listed += tokens_s[b1[j] + 1] - from;
    }
    out.sum[J] = above;
    out.unit[J] = unit;
    out.before[J] = before;
    out.at[J] = at;
    // a lane a range
    float lo = __builtin_inff();
    if (J < kRanges) {
        const double c = kUnitsPerNat * r.inv_t;
        int first = b0[0], last = b1[0];
#pragma unroll
        for (int j = 1; j < kRanges; ++j) {
            first = J == j ? b0[j] : first;
            last = J == j ? b1[j] : last;
        }
        const LogitRange near = logits_of({c, anchor, false}, first, last);
        const bool none = last < first;
        lo = none ? __builtin_inff() : near.lo;
        out.first[J] = first;
        out.last[J] = last;
        out.lo[J] = lo;
        out.hi[J] = none ? -__builtin_inff() : near.hi;
    }
    static_assert(kRanges == 4, "lanes that meet");
    lo = fminf(lo, __shfl_xor(lo, 1));
    lo = fminf(lo, __shfl_xor(lo, 2));
    if (J == 0) {
        out.least = lo;
        out.anchor = anchor;
        out.best = best;
        out.min_p_sum = min_p_sum;
        out.min_first = m0;
        out.min_last = m1;
        out.state = listed <= (uint32_t)kList ? 1 : 2;
        out.listed = 0;  // counted by the next launch
    }
}

// The tokens of marked bins, in no order.  Those within the bins' ranges of logits, hardly more, are
// gathered first and told apart side by side: in their places, a few lanes of most waves would work.  One
// atomic a workgroup: those of a row meet at one address, one after another.
template <typename T>
__global__ __launch_bounds__(kPartThreads) void k_sample_list(const m27q_sampling p, const Scratch sc) {
    __shared__ uint16_t near_at[kPart];
    __shared__ uint32_t near_s, count_s, to_s;
    const int row = blockIdx.y, first = (int)blockIdx.x * kPart, lane = threadIdx.x & 63;
    RowPlan &plan = sc.plan[row];
    // a part whose largest token lies below all of them has none
    if (plan.state != 1 || key_value(sc.part[(long long)row * sc.parts + blockIdx.x].best) < plan.least) return;
    float v[kEach];
    load_part<T>(p, row, first, v);
    if (threadIdx.x == 0) near_s = count_s = 0;
    unsigned long long near[kEach];  // a bit a lane
    int b0[kRanges], b1[kRanges], up = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) near[i] = 0;
#pragma unroll
    for (int j = 0; j < kRanges; ++j) {
        b0[j] = plan.first[j];
        b1[j] = plan.last[j];
        const float lo = plan.lo[j], hi = plan.hi[j];
        if (b1[j] < b0[j]) continue;
#pragma unroll
        for (int i = 0; i < kEach; ++i) near[i] |= __ballot(v[i] >= lo) & __ballot(v[i] <= hi);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) up += __popcll(near[i]);
    __syncthreads();
    if (up) {
        uint32_t to = 0;
        if (lane == 0) to = atomicAdd(&near_s, (uint32_t)up);
        to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (near[i] >> lane & 1) near_at[to + __popcll(near[i] & ((1ull << lane) - 1))] = (uint16_t)part_index(i);
            to += (uint32_t)__popcll(near[i]);
        }
    }
    __syncthreads();
    const int m = (int)near_s;
    if (m == 0) return;
    const Scale s = row_scale(row_rule(p, row), plan.anchor);
    const long long base = (long long)row * p.stride + first;
    uint64_t *const list = sc.list + (long long)row * kList;
    for (int i0 = 0; i0 < m; i0 += kPartThreads) {
        const int i = i0 + (int)threadIdx.x, at = near_at[min(i, m - 1)];
        const float l = logit<T>(p.logits, base + at);
        const int bin = place_of(l, s).bin;
        bool ok = false;
#pragma unroll
        for (int j = 0; j < kRanges; ++j) ok |= bin >= b0[j] && bin <= b1[j];
        ok &= i < m && bin < kBins;
        const unsigned long long mine = __ballot(ok);
        uint32_t to = 0;
        if (lane == 0 && mine) to = atomicAdd(&count_s, (uint32_t)__popcll(mine));
        __syncthreads();
        if (threadIdx.x == 0) {
            to_s = atomicAdd(&plan.listed, count_s);
            count_s = 0;
        }
        __syncthreads();
        to = __builtin_amdgcn_readfirstlane(to) + to_s + (uint32_t)__popcll(mine & ((1ull << lane) - 1));
        if (ok && to < (uint32_t)kList) list[to] = order_key(l, first + at);
    }
}

// The smallest of a workgroup's values that do not descend from thread to thread, but for the largest of
// their type, which stands for none: that of each wave's first.
template <typename T>
__device__ __forceinline__ void min_of_first(T v, T &to) {
    const T none = sizeof(T) == 8 ? (T)~0ull : (T)0x7fffffff;
    const unsigned long long m = __ballot(v != none);
    if (m && (int)(threadIdx.x & 63) == __builtin_ctzll(m)) atomicMin(&to, v);
}

// What a workgroup that goes through a whole row keeps in LDS.
constexpr int kDigitBits = 11, kDigits = 1 << kDigitBits;
struct WholeRow {
    unsigned long long mass[kDigits];
    uint64_t key[kDigits];               // of a piece's only token
    uint32_t count[kDigits];
    float2 wait[kRowThreads / 64][128];  // a wave's tokens near a border: logit, and index as bits
    uint64_t found_key;
    unsigned long long found_sum, found_own;
    uint32_t found_count, found_held;
    int found;
};
struct Border {
    uint64_t key;              // of the token at the border
    unsigned long long down;   // the running sum, itself included
    double own;                // its weight in that sum's units
};

constexpr int kCrowd = 1024;
struct PickShared {
    union {
        struct {
            uint64_t keys[kList];
            uint32_t count[kList];  // of the tokens in a bucket, then of those before it
        };
        WholeRow whole;
    };
    uint32_t scan32[kRowThreads / 64];
    unsigned long long scan[kRowThreads / 64];
    // the plan's
    uint32_t before[kBins + 1], at[kBins + 1];
    unsigned long long sum[kBins + 1];
    double unit[kBins + 1];
    unsigned long long start[kBins + 1];  // the list's running sum in front of a bin
    // sums down to the top_k-th token, the one that reaches top_p and the last one that min_p leaves
    unsigned long long among, top_p, min_p;
    int pick;
    uint32_t most;
    double octave[kUnit];
};

// How far down in its bin a logit lies, of 1: by what it is off a whole unit.
__device__ __forceinline__ float part_of(const Place &a) {
    return a.bin < kFine ? (float)a.z + 0.5f : ((float)a.k + (float)a.z + 0.5f) * (1.0f / kUnit);
}
// The same for logits of 16 bits (`low` bits of theirs as floats are 0), of which hundreds are equal: by how many
// 16-bit numbers lie between it and the bin's upper end, equal ones by index.  Whole numbers, so that what is
// before another in the row's order is never behind it here.  24 rows of 248320, BF16, top-p: 35 us, by z 64.
__device__ __forceinline__ float part_of(uint64_t key, int bin, const Scale &s, int low, uint32_t n) {
    const double d = s.anchor - bin_distance(bin);
    const int up = (int)(order_bits((float)((d + 0.5) / s.c)) >> low) + 1;  // (rounding, of less than one number)
    const int down = (int)(order_bits((float)((d - (bin < kFine ? 0.5 : kUnit - 0.5)) / s.c)) >> low);
    const int at = up - (int)((uint32_t)(key >> 24) >> low);
    return ((float)at + (float)key_index(key) / (float)n) / (float)(up - down + 1);
}

// A row's list in order, the running sums of its tokens, and the borders among them.  E tokens a thread.
// In order: a bin's tokens have as many buckets as they are, by their place in it, so that few share one; a
// token's place in its bucket is how many of it are larger.  False: some bucket holds so many
// (equal logits of 32 bits) that this would take long.
template <int E>
__device__ __forceinline__ bool pick_from_list(const m27q_sampling &p, const Scratch &sc, const RowPlan &plan, const Rule &r,
                                               int n, PickShared &s) {
    const int row = blockIdx.x, tid = threadIdx.x, i0 = tid * E;
    const Scale scale = row_scale(r, plan.anchor);
    const Weights x(s.octave);
    uint64_t key[E];
    uint32_t bucket[E], slot[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = e * kRowThreads + tid;
        key[e] = i < n ? sc.list[(long long)row * kList + i] : 0;
        if (e * kRowThreads < kList) s.count[i] = 0;
    }
    __syncthreads();  // the plan's arrays are there too
#pragma unroll
    for (int e = 0; e < E; ++e) {
        bucket[e] = slot[e] = 0;
        if (e * kRowThreads + tid >= n) continue;
        const Place a = place_of(key_value(key[e]), scale);
        const uint32_t at = s.at[a.bin], count = s.at[a.bin + 1] - at;
        const int low = p.type == M27Q_TYPE_BF16 ? 16 : 13;
        const float part = p.type == M27Q_TYPE_F32 ? part_of(a) : part_of(key[e], a.bin, scale, low, p.n);
        // (below n even if somebody writes to the logits meanwhile)
        bucket[e] = min(at + min((uint32_t)fmaxf(part * (float)count, 0.0f), count - 1), (uint32_t)n - 1);
        slot[e] = atomicAdd(&s.count[bucket[e]], 1u);
    }
    __syncthreads();
    uint32_t c[E], sum32 = 0, most = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        c[e] = s.count[i0 + e];
        sum32 += c[e];
        most = max(most, c[e]);
    }
    if (most > (uint32_t)kCrowd) s.most = most;
    uint32_t all32, run32 = scan_group<kRowThreads>(sum32, s.scan32, all32);
    if (s.most) return false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        s.count[i0 + e] = run32;
        run32 += c[e];
    }
    __syncthreads();
    uint32_t first[E], held[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        first[e] = held[e] = 0;
        if (e * kRowThreads + tid >= n) continue;
        first[e] = s.count[bucket[e]];
        held[e] = (bucket[e] + 1 < (uint32_t)(E * kRowThreads) ? s.count[bucket[e] + 1] : (uint32_t)n) - first[e];
        s.keys[first[e] + slot[e]] = key[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        uint32_t larger = 0;
        for (uint32_t j = 0; j < held[e]; ++j) larger += s.keys[first[e] + j] > key[e];
        slot[e] = first[e] + larger;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e * kRowThreads + tid < n) s.keys[slot[e]] = key[e];
    __syncthreads();

    // the sums of the row down to each token of the list.  In front of a bin, and at its end, they are the plan's.
    unsigned long long own[E], sum = 0;
    int bin[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        own[e] = 0;
        bin[e] = 0;
        if (i0 + e < n) {
            key[e] = s.keys[i0 + e];
            const Place a = place_of(key_value(key[e]), scale);
            bin[e] = a.bin;
            own[e] = x.mass(a.z, a.k, 0);
        }
        sum += own[e];
    }
    unsigned long long all, run = scan_group<kRowThreads>(sum, s.scan, all);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (i0 + e < n && (uint32_t)(i0 + e) == s.at[bin[e]]) s.start[bin[e]] = run;
        run += own[e];
    }
    run -= sum;
    __syncthreads();
    const float top = key_value(plan.best);
    unsigned long long down[E], dropped = ~0ull;
    int rank[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t i = (uint32_t)(i0 + e);
        const unsigned long long lo = s.sum[bin[e]], hi = s.sum[bin[e] + 1], in = run - s.start[bin[e]];
        const auto to = [&](unsigned long long x) { return min(lo + row_mass(x, s.unit[bin[e]]), hi); };
        down[e] = i + 1 == s.at[bin[e] + 1] ? hi : to(in + own[e]);
        rank[e] = i < (uint32_t)n ? (int)(s.before[bin[e]] + i - s.at[bin[e]]) : 0x7fffffff;
        run += own[e];
        if (rank[e] == r.k - 1) s.among = down[e];
        if (r.min_p > 0.0 && i < (uint32_t)n && dropped == ~0ull &&
            exp(((double)key_value(key[e]) - (double)top) * r.inv_t) < r.min_p)
            dropped = to(in);
    }
    if (r.min_p > 0.0) min_of_first(dropped, s.min_p);
    __syncthreads();
    if (r.top_p < 1.0) {
        const double reach = r.top_p * (double)s.among;
        unsigned long long at = ~0ull;
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
            if (i0 + e < n && (double)down[e] >= reach) at = down[e];
        min_of_first(at, s.top_p);
        __syncthreads();
    }
    // the first token is kept whatever the rest says
    const Place f = place_of(top, scale);
    const unsigned long long one = min(row_mass(x.mass(f.z, f.k, 0), s.unit[f.bin]), s.sum[f.bin + 1]);
    const unsigned long long total = max(one, min(s.among, min(s.top_p, s.min_p)));
    const double target = r.u * (double)total;
    int at = 0x7fffffff;
#pragma unroll
    for (int e = E - 1; e >= 0; --e)
        if (i0 + e < n && (double)down[e] >= target) at = rank[e];
    min_of_first(at, s.pick);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (i0 + e < n && rank[e] == s.pick) {
            p.token[row] = key_index(key[e]);
            if (p.prob) p.prob[row] = (float)((double)own[e] * s.unit[bin[e]] / (double)total);
        }
    return true;
}

// U logits of a row, all on their way at once.
template <int U>
__device__ __forceinline__ void load_some(const m27q_sampling &p, long long base, int i0, float (&v)[U]) {
    const int last = (int)p.n - 1;
    if (p.type == M27Q_TYPE_F32) {
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = logit<float>(p.logits, base + min(i0 + j * kRowThreads, last));
    } else if (p.type == M27Q_TYPE_F16) {
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = logit<_Float16>(p.logits, base + min(i0 + j * kRowThreads, last));
    } else {
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = logit<__bf16>(p.logits, base + min(i0 + j * kRowThreads, last));
    }
}

// A row whose borders lie among more tokens than a list holds (flat ones, thousands of equal logits): the
// token of a border's bin at which a count or a sum of weights in descending order reaches its target, by 2048 pieces
// of the keys that are left at a time, the row read once for each, until one token is left.
__device__ __forceinline__ void sample_whole_row(const m27q_sampling &p, int row, const Rule &r, const RowPlan &plan,
                                                 PickShared &s) {
    const int n = (int)p.n, tid = threadIdx.x, lane = tid & 63;
    const long long base_at = (long long)row * p.stride;
    const float top = key_value(plan.best);
    const Scale scale = row_scale(r, plan.anchor);
    const Weights x(s.octave);
    WholeRow &o = s.whole;
    constexpr int U = 4;

    // Among the tokens of a bin the first at which their count reaches `most` or the row's running sum `target`; the
    // last one if none does.
    const auto border = [&](int bin, uint32_t most, double target) -> Border {
        const unsigned long long lo = s.sum[bin], hi = s.sum[bin + 1];
        const uint32_t tokens = s.before[bin + 1] - s.before[bin];
        const double unit = s.unit[bin];
        const auto down = [&](uint32_t count, unsigned long long mass) {
            return count == tokens ? hi : min(lo + row_mass(mass, unit), hi);
        };
        const LogitRange near = logits_of(scale, bin, bin);
        uint64_t first = (uint64_t)order_bits(near.lo) << 24, span = ((uint64_t)order_bits(near.hi) << 24 | 0xffffff) - first + 1;
        unsigned long long sum = 0;
        uint32_t seen = 0;
        while (true) {
            const int shift = max(64 - __builtin_clzll((span - 1) | 1) - kDigitBits, 0);
            // (the piece of the largest numbers reaches past infinity, where keys stand for none)
            const uint64_t last = first + span - 1;
            const float least = key_value(first), most_l = key_value(last < kLastKey ? last : kLastKey);
            for (int i = tid; i < kDigits; i += kRowThreads) o.mass[i] = 0, o.count[i] = 0;
            if (tid == 0) o.found = 0x7fffffff;
            __syncthreads();
            // few tokens of most waves lie near: those wait until they fill one
            float2 *const wait = o.wait[tid >> 6];
            int waiting = 0;
            const auto add = [&](bool there) {
                const float2 e = wait[lane];
                const uint64_t key = order_key(e.x, __float_as_int(e.y)), at = key - first;
                const Place a = place_of(e.x, scale);
                const bool in = there && at < span && a.bin == bin;
                const unsigned long long some = __ballot(in);
                if (!some) return;
                const int digit = (int)(at >> shift) & (kDigits - 1), one = __builtin_ctzll(some);
                const int same = __builtin_amdgcn_readlane(digit, one);
                unsigned long long w = in ? x.mass(a.z, a.k, 0) : 0;
                if (__ballot(in && digit != same) == 0) {  // lanes that would meet in one place
                    w = scan_wave(w);
                    if (lane == 63) {
                        atomicAdd(&o.mass[same], w);
                        atomicAdd(&o.count[same], (uint32_t)__popcll(some));
                    }
                    if (lane == one) o.key[same] = key;
                } else if (in) {
                    atomicAdd(&o.mass[digit], w);
                    atomicAdd(&o.count[digit], 1u);
                    o.key[digit] = key;
                }
            };
            for (int i0 = tid; i0 - tid < n; i0 += U * kRowThreads) {
                float v[U];
                load_some(p, base_at, i0, v);
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    const int i = i0 + j * kRowThreads;
                    const bool close = i < n && v[j] >= least && v[j] <= most_l;
                    const unsigned long long some = __ballot(close);
                    if (!some) continue;
                    if (close) wait[waiting + __popcll(some & ((1ull << lane) - 1))] = make_float2(v[j], __int_as_float(i));
                    waiting += (int)__popcll(some);
                    wave_order();
                    if (waiting >= 64) {
                        add(true);
                        waiting -= 64;
                        const float2 rest = wait[64 + lane];
                        wave_order();
                        wait[lane] = rest;
                        wave_order();
                    }
                }
            }
            add(lane < waiting);
            __syncthreads();
            // the pieces in descending order, two a thread
            constexpr int E = kDigits / kRowThreads;
            static_assert(E == 2, "two pieces a thread");
            const int d0 = kDigits - 1 - E * tid, d1 = d0 - 1;
            const uint32_t c0 = o.count[d0], c1 = o.count[d1];
            const unsigned long long m0 = o.mass[d0], m1 = o.mass[d1];
            uint32_t left;
            unsigned long long all;
            const uint32_t c = scan_group<kRowThreads>(c0 + c1, s.scan32, left);
            const unsigned long long m = scan_group<kRowThreads>(m0 + m1, s.scan, all);
            const auto reaches = [&](uint32_t count, unsigned long long mass) {
                return seen + count >= most || (double)down(seen + count, sum + mass) >= target || count == left;
            };
            int hit = 0x7fffffff;
            if (c1 && reaches(c + c0 + c1, m + m0 + m1)) hit = E * tid + 1;
            if (c0 && reaches(c + c0, m + m0)) hit = E * tid;
            min_of_first(hit, o.found);
            __syncthreads();
            if (o.found / E == tid) {
                const bool second = o.found % E;
                o.found_key = second ? o.key[d1] : o.key[d0];
                o.found_count = seen + c + (second ? c0 : 0);
                o.found_held = second ? c1 : c0;
                o.found_sum = sum + m + (second ? m0 : 0);
                o.found_own = second ? m1 : m0;
            }
            __syncthreads();
            seen = o.found_count;
            sum = o.found_sum;
            first += (uint64_t)(kDigits - 1 - o.found) << shift;
            span = 1ull << shift;
            const Border found{o.found_key, down(seen + 1, sum + o.found_own), (double)o.found_own * unit};
            const bool done = o.found_held == 1 || shift == 0;
            __syncthreads();  // all have read it
            if (done) return found;
        }
    };
    const auto bin_at = [&](double target) {  // as the plan's
        const double t = fmax(target, 1.0);
        const unsigned long long all = s.sum[kBins];
        return min(first_of(s.sum + 1, kBins, [&](unsigned long long v) { return (double)v >= t || v == all; }), kBins - 1);
    };

    unsigned long long among = s.sum[kBins], total;
    if ((uint32_t)r.k < s.before[kBins]) {
        const int bin = min(first_of(s.before + 1, kBins, [&](uint32_t v) { return v >= (uint32_t)r.k; }), kBins - 1);
        among = border(bin, (uint32_t)r.k - s.before[bin], __builtin_inf()).down;
    }
    total = among;
    if (r.top_p < 1.0) {
        const double target = r.top_p * (double)among;
        total = min(total, border(bin_at(target), 0xffffffffu, target).down);
    }
    if (r.min_p > 0.0) {
        // in the bins where its border can lie
        if (tid < kMinBins) o.mass[tid] = 0, o.count[tid] = 0;
        __syncthreads();
        const LogitRange near = logits_of(scale, plan.min_first, plan.min_last);
        for (int i0 = tid; i0 - tid < n; i0 += U * kRowThreads) {
            float v[U];
            load_some(p, base_at, i0, v);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (!(i0 + j * kRowThreads < n && v[j] >= near.lo && v[j] <= near.hi)) continue;
                const Place a = place_of(v[j], scale);
                if (a.bin < plan.min_first || a.bin > plan.min_last) continue;
                const int at = a.bin - plan.min_first;
                if (exp(((double)v[j] - (double)top) * r.inv_t) >= r.min_p) atomicAdd(&o.mass[at], x.mass(a.z, a.k, 0));
                else o.count[at] = 1;
            }
        }
        __syncthreads();
        unsigned long long sum = plan.min_p_sum;
        for (int i = plan.min_last - plan.min_first; i >= 0; --i) {
            const int bin = plan.min_first + i;
            if (o.count[i]) sum = min(s.sum[bin] + row_mass(o.mass[i], s.unit[bin]), s.sum[bin + 1]);
        }
        total = min(total, sum);
        __syncthreads();
    }
    // the first token is kept whatever the rest says
    const Place f = place_of(top, scale);
    total = max(total, min(row_mass(x.mass(f.z, f.k, 0), s.unit[f.bin]), s.sum[f.bin + 1]));
    const double target = r.u * (double)total;
    const Border pick = border(bin_at(target), 0xffffffffu, target);
    if (tid == 0) {
        p.token[row] = key_index(pick.key);
        if (p.prob) p.prob[row] = (float)(pick.own / (double)total);
    }
}

__global__ __launch_bounds__(kRowThreads) void k_sample_pick(const m27q_sampling p, const Scratch sc) {
    __shared__ PickShared s;
    const int row = blockIdx.x;
    const RowPlan &plan = sc.plan[row];
    const int state = plan.state;
    if (state == 0) return;
    const Rule r = row_rule(p, row);
    bool done = false;
    if (threadIdx.x < kUnit) s.octave[threadIdx.x] = Weights::factor(threadIdx.x);
    if (threadIdx.x <= kBins) {
        s.before[threadIdx.x] = plan.before[threadIdx.x];
        s.at[threadIdx.x] = plan.at[threadIdx.x];
        s.sum[threadIdx.x] = plan.sum[threadIdx.x];
        s.unit[threadIdx.x] = plan.unit[threadIdx.x];
    }
    if (state == 1) {
        if (threadIdx.x == 0) {
            s.among = plan.sum[kBins];  // unless the top_k-th is on the list
            s.top_p = ~0ull;
            s.min_p = plan.min_p_sum;
            s.pick = 0x7fffffff;
            s.most = 0;
        }
        const int n = (int)min(plan.listed, (uint32_t)kList);
        if (n <= kRowThreads) done = pick_from_list<1>(p, sc, plan, r, n, s);
        else if (n <= 2 * kRowThreads) done = pick_from_list<2>(p, sc, plan, r, n, s);
        else if (n <= 4 * kRowThreads) done = pick_from_list<4>(p, sc, plan, r, n, s);
        else done = pick_from_list<8>(p, sc, plan, r, n, s);
    }
    __syncthreads();
    if (!done) sample_whole_row(p, row, r, plan, s);
}

struct Sizes {
    int parts;
    size_t part, bins, plan, list;
    Sizes(uint32_t rows, uint32_t n)
        : parts((int)((n + kPart - 1) / kPart)), part(align((size_t)rows * parts * sizeof(Part))),
          bins((size_t)rows * parts * kStored * 8), plan(align((size_t)rows * sizeof(RowPlan))), list((size_t)rows * kList * 8) {}
    static size_t align(size_t v) { return (v + 255) & ~(size_t)255; }
};

template <typename T>
hipError_t launch_t(const m27q_sampling &p, const Scratch &sc, hipStream_t s) {
    const dim3 parts(sc.parts, p.rows);
    hipLaunchKernelGGL((k_sample_parts<T>), parts, dim3(kPartThreads), 0, s, p, sc);
    hipLaunchKernelGGL(k_sample_plan, dim3(p.rows), dim3(kHalves * kPlanThreads), 0, s, p, sc);
    hipLaunchKernelGGL((k_sample_list<T>), parts, dim3(kPartThreads), 0, s, p, sc);
    hipLaunchKernelGGL(k_sample_pick, dim3(p.rows), dim3(kRowThreads), 0, s, p, sc);
    return hipGetLastError();
}

}  // namespace

size_t sample_scratch(uint32_t rows, uint32_t n) {
    const Sizes z(rows, n);
    return z.part + z.bins + z.plan + z.list;
}

hipError_t launch_sample_rows(const m27q_sampling &p, void *scratch, hipStream_t s) {
    const Sizes z(p.rows, p.n);
    Scratch sc;
    char *at = (char *)scratch;
    sc.part = (Part *)at;
    sc.bins = (unsigned long long *)(at += z.part);
    sc.plan = (RowPlan *)(at += z.bins);
    sc.list = (uint64_t *)(at + z.plan);
    sc.parts = z.parts;
    if (p.type == M27Q_TYPE_F32) return launch_t<float>(p, sc, s);
    return p.type == M27Q_TYPE_F16 ? launch_t<_Float16>(p, sc, s) : launch_t<__bf16>(p, sc, s);
}

}  // namespace m27q
