// m27q_rope.hip -- rotary positions, and k and v into the pages of a cache.
//
// Pair j of a head at position p becomes
//   (a, b) -> mscale (a cos t - b sin t, a sin t + b cos t),  t = 2 pi p turn_j,
// with p turn_j taken modulo one turn in 64-bit fixed point, which is exact:
// integer products wrap where turns do.  Memory bounds it: every value is read
// and written once.  A workgroup takes one token (a part of its heads where
// they are more than 256 units): the cosines and sines of the token's pairs
// are computed once into LDS (one per thread), then each thread turns one
// unit, 8 pairs or 8 values that stay.  The loads of a unit are issued before
// the barrier.  A unit is read and written by one thread, so out may be x.
//
// One token (24 query and 4 + 4 cache heads of 256) takes 3.6 us, 64 take 4.6: launch, one
// round trip for the table entry, one for the store.  2999 and 2903 of them from fp32 into a
// BF16 cache, 290 MB: 72 us, 4.0 TB/s (a plain conversion of as much takes 50, 5.8 TB/s).  Four
// units a thread (fewer, longer workgroups) took 110 us, loads past the caches 77, a workgroup
// of queries that leaves the table alone 71.
#include "m27q_mix.h"

namespace m27q {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 512;

// cos and sin of a phase in 2^-64 turns: the nearest quarter turn is taken
// off, the rest (|x| <= pi / 4, its upper 32 bits: 1.5e-9 rad) goes through
// the Taylor polynomials, cut where the next term is below 3e-9.
__device__ __forceinline__ float2 cos_sin(uint64_t phase) {
    const uint64_t quarter = (phase + (1ull << 61)) >> 62;
    const int32_t rest = (int32_t)((int64_t)(phase - (quarter << 62)) >> 32);
    const float x = (float)rest * 0x1.921fb6p-30f;  // 2 pi / 2^32
    const float y = x * x;
    float s = 0x1.71de3ap-19f;  // 1 / 9!
    s = __builtin_fmaf(s, y, -0x1.a01a02p-13f);
    s = __builtin_fmaf(s, y, 0x1.111112p-7f);
    s = __builtin_fmaf(s, y, -0x1.555556p-3f);
    s = __builtin_fmaf(s * y, x, x);
    float c = -0x1.27e4fcp-22f;  // 1 / 10!
    c = __builtin_fmaf(c, y, 0x1.a01a02p-16f);
    c = __builtin_fmaf(c, y, -0x1.6c16c2p-10f);
    c = __builtin_fmaf(c, y, 0x1.555556p-5f);
    c = __builtin_fmaf(c, y, -0.5f);
    c = __builtin_fmaf(c, y, 1.0f);
    const float a = (quarter & 1) ? s : c, b = (quarter & 1) ? c : s;
    return make_float2(((quarter + 1) & 2) ? -a : a, (quarter & 2) ? -b : b);
}

// The sequence of row t: the last one that starts at or before t, by a search
// of 64 starts at a time (lane l looks at l of 64 steps through the range).
__device__ __forceinline__ int seq_of(const int32_t *start, int n, int t) {
    int lo = 0, len = n;  // the answer is in [lo, lo + len), if any sequence starts that early
    while (len > 1) {
        const int step = (len + 63) / 64;
        const int at = lo + (int)(threadIdx.x & 63) * step;
        const bool early = at < lo + len && start[at] <= t;
        const int k = __popcll(__ballot(early));
        if (k == 0) return -1;
        const int next = lo + (k - 1) * step;
        len = min(step, lo + len - next);
        lo = next;
    }
    return start[lo] <= t && t < start[lo + 1] ? lo : -1;
}

// Units of a head that turns: pairs, then what stays (8 of each, or one where
// a launch is not vectorized).
template <bool VEC>
__host__ __device__ inline int pair_units(uint32_t rot, uint32_t layout) {
    return VEC ? (int)(layout == M27Q_ROPE_HALF ? rot / 16 : rot / 8) : (int)rot / 2;
}
template <bool VEC>
__host__ __device__ inline int head_units(uint32_t rot, uint32_t layout, uint32_t dim) {
    return pair_units<VEC>(rot, layout) + (int)(dim - rot) / (VEC ? 8 : 1);
}
template <bool VEC>
__host__ __device__ inline int token_units(const RopeParams &p) {
    const int u = head_units<VEC>(p.rope.rot, p.rope.layout, p.q.dim) * (int)p.q.heads;
    if (!p.has_cache) return u;
    return u + (head_units<VEC>(p.rope.rot, p.rope.layout, p.k.dim) + (int)p.v.dim / (VEC ? 8 : 1)) * (int)p.k.heads;
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void k_rope(const RopeParams p, int parts) {
    __shared__ float2 cs[kMaxPairs];
    const int t = blockIdx.x / parts;
    const int pairs = (int)p.rope.rot / 2;
    const bool half = p.rope.layout == M27Q_ROPE_HALF;

    // this thread's unit: which head of q, k or v, and which part of it
    int u = (int)(blockIdx.x - (unsigned)t * parts) * kThreads + (int)threadIdx.x;
    const bool live = u < token_units<VEC>(p);
    const int per = head_units<VEC>(p.rope.rot, p.rope.layout, p.q.dim);  // q and k alike
    const int pu = pair_units<VEC>(p.rope.rot, p.rope.layout);
    const int nq = (int)p.q.heads * per, nk = p.has_cache ? (int)p.k.heads * per : 0;
    int kind = 0, head = 0, unit = 0;  // kind 0: q, 1: k, 2: v
    if (live) {
        if (u < nq) {
            head = u / per;
            unit = u - head * per;
        } else if (u < nq + nk) {
            kind = 1;
            head = (u - nq) / per;
            unit = u - nq - head * per;
        } else {
            kind = 2;
            const int pv = (int)p.v.dim / (VEC ? 8 : 1);
            head = (u - nq - nk) / pv;
            unit = u - nq - nk - head * pv;
        }
    }
    const m27q_rows &x = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const long long from = (long long)t * x.token_stride + (long long)head * x.head_stride;
    const bool turns = kind != 2 && unit < pu;
    // values of the unit within its head: e0 .. and, for a turning one, e1 ..
    const int W = VEC ? 8 : 1;
    const int e0 = turns ? (half ? unit * W : unit * 2 * W / (VEC ? 2 : 1))
                         : (kind == 2 ? unit * W : (int)p.rope.rot + (unit - pu) * W);
    const int e1 = half ? e0 + pairs : e0 + 1;
    f32x8 a = {}, b = {};
    if (live) {
        if constexpr (VEC) {
            a = load8(x.ptr, from + e0, x.type);
            if (turns && half) b = load8(x.ptr, from + e1, x.type);
        } else {
            a[0] = load1(x.ptr, from + e0, x.type);
            if (turns) b[0] = load1(x.ptr, from + e1, x.type);
        }
    }

    const int64_t pos = p.pos[t];
    for (int j = threadIdx.x; j < pairs; j += kThreads) {
        const float2 v = cos_sin((uint64_t)pos * p.rope.turns[j]);
        cs[j] = make_float2(v.x * p.rope.mscale, v.y * p.rope.mscale);
    }
    // where the token's keys and values go
    long long place = -1;
    if (p.has_cache) {
        const int s = seq_of(p.seqs.start, (int)p.seqs.n, t);
        if (s >= 0) {
            const long long at = (long long)p.seqs.kv_len[s] - (min(p.seqs.start[s + 1], p.tokens) - t);
            const int shift = __builtin_ctz(p.cache.page_size), row = t - max(p.seqs.start[s], 0);
            const long long page = at >> shift;
            if (at >= 0 && at < (long long)p.seqs.max_kv && page < (long long)p.seqs.table_stride &&
                row < (int)p.seqs.max_q) {
                const int32_t id = p.seqs.table[(long long)s * p.seqs.table_stride + page];
                if (id >= 0 && (uint32_t)id < p.cache.pages)
                    place = (long long)id * p.cache.page_stride + (at & (p.cache.page_size - 1)) * p.cache.dim;
            }
        }
    }
    __syncthreads();
    if (!live) return;

    if (turns) {
        if constexpr (VEC) {
            if (half) {
                const f32x8 a0 = a, b0 = b;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 v = cs[e0 + i];
                    a[i] = a0[i] * v.x - b0[i] * v.y;
                    b[i] = a0[i] * v.y + b0[i] * v.x;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float2 v = cs[e0 / 2 + i / 2];
                    const float c = a[i], d = a[i + 1];
                    a[i] = c * v.x - d * v.y;
                    a[i + 1] = c * v.y + d * v.x;
                }
            }
        } else {
            const float2 v = cs[unit];
            const float c = a[0], d = b[0];
            a[0] = c * v.x - d * v.y;
            b[0] = c * v.y + d * v.x;
        }
    }
    void *out;
    long long to;
    uint32_t type;
    if (kind == 0) {
        out = p.q_out.ptr;
        type = p.q_out.type;
        to = (long long)t * p.q_out.token_stride + (long long)head * p.q_out.head_stride;
    } else {
        if (place < 0) return;
        out = kind == 1 ? p.cache.k : p.cache.v;
        type = p.cache.type;
        to = place + (long long)head * p.cache.page_size * p.cache.dim;
    }
    if constexpr (VEC) {
        store8(out, to + e0, type, a);
        if (turns && half) store8(out, to + e1, type, b);
    } else {
        store1(out, to + e0, type, a[0]);
        if (turns) store1(out, to + e1, type, b[0]);
    }
}

bool rows16(const m27q_rows &r) {
    const int b = type_bytes(r.type);
    return (uintptr_t)r.ptr % 16 == 0 && r.token_stride * b % 16 == 0 && r.head_stride * b % 16 == 0;
}

}  // namespace

// Units of 8 values need whole units in a head and 16-byte aligned rows.
bool rope_vectorizes(const RopeParams &p) {
    if (p.q.dim % 8 || p.rope.rot % (p.rope.layout == M27Q_ROPE_HALF ? 16 : 8)) return false;
    if (!rows16(p.q) || !rows16(p.q_out)) return false;
    if (!p.has_cache) return true;
    return rows16(p.k) && rows16(p.v) && (uintptr_t)p.cache.k % 16 == 0 && (uintptr_t)p.cache.v % 16 == 0 &&
           p.cache.page_stride % 8 == 0;
}

long long rope_groups(const RopeParams &p, bool vec) {
    const long long units = vec ? token_units<true>(p) : token_units<false>(p);
    const long long groups = p.tokens * ((units + kThreads - 1) / kThreads);
    return groups * kThreads < (1ll << 32) ? groups : 0;
}

hipError_t launch_rope(const RopeParams &p, hipStream_t s) {
    const bool vec = rope_vectorizes(p);
    const long long groups = rope_groups(p, vec);
    const int parts = (int)(groups / p.tokens);
    if (vec) hipLaunchKernelGGL((k_rope<true>), dim3((unsigned)groups), dim3(kThreads), 0, s, p, parts);
    else hipLaunchKernelGGL((k_rope<false>), dim3((unsigned)groups), dim3(kThreads), 0, s, p, parts);
    return hipGetLastError();
}

}  // namespace m27q
