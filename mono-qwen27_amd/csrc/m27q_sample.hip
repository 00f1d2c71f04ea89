// m27q_sample.hip -- a token for each row of logits.
//
// In order of value (equal ones in order of index) token i of a row has the weight
// w_i = e^((l_i - max) / T).  What is kept is a prefix of that order: the first
// top_k, of these the ones with w_i >= min_p, of these the shortest prefix whose
// sum reaches top_p times the sum of the first top_k.  The token is the first
// whose running sum reaches u times the sum of what is kept.
//
// Weights are summed as 64-bit integers, so that no order of adding changes a
// sum, and a border is where the weights put it: 2^-44 of the largest weight for
// each token of a vocabulary of 250000.
#include "m27q_mix.h"

namespace m27q {

namespace {

constexpr int kThreads = 1024;

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
constexpr int kKeyBits = 56;
__device__ __forceinline__ int key_index(uint64_t key) { return (int)(0xffffffu - (uint32_t)(key & 0xffffffu)); }

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

struct Found {
    uint64_t key;    // of the token at the border
    uint64_t sum;    // of the weights down to it, itself included
};

// One workgroup a row: the token at which a count or a sum of weights in descending order
// reaches its target, by 8 bits of the keys at a time, the row read once for each.
__global__ __launch_bounds__(kThreads) void k_sample_row(const m27q_sampling p) {
    __shared__ unsigned long long mass[256];
    __shared__ uint32_t count[256];
    __shared__ unsigned long long best_s, total_s;
    __shared__ uint64_t found_key, found_sum;
    __shared__ uint32_t found_count;
    const int row = blockIdx.x, n = (int)p.n, tid = threadIdx.x;
    const long long base = (long long)row * p.stride;
    auto value = [&](int i) { return load1(p.logits, base + i, p.type); };
    const Rule r = row_rule(p, row);

    if (tid == 0) best_s = total_s = 0;
    __syncthreads();
    unsigned long long best = 0;
    for (int i = tid; i < n; i += kThreads) best = max(best, (unsigned long long)order_key(value(i), i));
    atomicMax(&best_s, best);
    __syncthreads();
    best = best_s;
    const float top = value(key_index(best));
    if (r.greedy || !__builtin_isfinite(top)) {
        if (tid == 0) {
            p.token[row] = key_index(best);
            if (p.prob) p.prob[row] = 1.0f;
        }
        return;
    }
    const double one = (double)(1ull << (62 - (64 - __builtin_clzll((unsigned long long)n))));
    auto weight = [&](float v) {
        const double w = exp(((double)v - (double)top) * r.inv_t);
        return w > 0.0 ? w : 0.0;  // (NaN: none)
    };
    auto fixed = [&](double w) { return (unsigned long long)__builtin_rint(w * one); };

    // The first token in order at which the running count reaches `most` or the running sum `target`.
    auto border = [&](uint32_t most, double target) {
        uint64_t prefix = 0, sum = 0;
        uint32_t seen = 0;
        for (int shift = kKeyBits - 8; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) mass[tid] = 0, count[tid] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const float v = value(i);
                const uint64_t key = order_key(v, i);
                if ((key >> (shift + 8)) != prefix) continue;
                const int digit = (int)(key >> shift) & 255;
                atomicAdd(&count[digit], 1u);
                atomicAdd(&mass[digit], fixed(weight(v)));
            }
            __syncthreads();
            if (tid == 0) {
                int digit = 255, last = -1;
                for (; digit >= 0; --digit) {
                    if (count[digit] == 0) continue;
                    last = digit;
                    if (seen + count[digit] >= most || (double)(sum + mass[digit]) >= target) break;
                    seen += count[digit];
                    sum += mass[digit];
                }
                if (digit < 0) {  // never reached: the last one
                    digit = last;
                    seen -= count[digit];
                    sum -= mass[digit];
                }
                found_key = prefix << 8 | (uint64_t)digit;
                found_sum = sum;
                found_count = seen;
            }
            __syncthreads();
            prefix = found_key;
            sum = found_sum;
            seen = found_count;
        }
        return Found{prefix, sum + fixed(weight(value(key_index(prefix))))};
    };

    const Found all = border((uint32_t)r.k, __builtin_inf());
    uint64_t cut = all.key;
    if (r.top_p < 1.0) cut = max(cut, border(0xffffffffu, r.top_p * (double)all.sum).key);
    unsigned long long part = 0;
    for (int i = tid; i < n; i += kThreads) {
        const float v = value(i);
        const uint64_t key = order_key(v, i);
        const double w = weight(v);
        if (key == best || (key >= cut && w >= r.min_p)) part += fixed(w);
    }
    atomicAdd(&total_s, part);
    __syncthreads();
    const Found pick = border(0xffffffffu, r.u * (double)total_s);
    if (tid == 0) {
        const int i = key_index(pick.key);
        p.token[row] = i;
        if (p.prob) p.prob[row] = (float)(weight(value(i)) * one / (double)total_s);
    }
}

}  // namespace

size_t sample_scratch(uint32_t, uint32_t) { return 16; }

hipError_t launch_sample_rows(const m27q_sampling &p, void *, hipStream_t s) {
    hipLaunchKernelGGL(k_sample_row, dim3(p.rows), dim3(kThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace m27q
