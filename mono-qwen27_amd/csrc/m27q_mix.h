// m27q_mix.h -- launch interface and device helpers of the token mixers
// (rotary positions, attention over pages, the gated delta rule) and of a
// batch's steps beside them (norms, sampling).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/m27q.h"

namespace m27q {

struct RopeParams {
    m27q_rope_plan rope;
    const int32_t *pos;
    int tokens;
    m27q_rows q, q_out;
    // append only (has_cache): the rows of k and v, and where they go
    int has_cache;
    m27q_rows k, v;
    m27q_seqs seqs;
    m27q_cache cache;
};
// Workgroups of a rope launch, 0 if they would pass the dispatch's limit.
long long rope_groups(const RopeParams &p, bool vec);
bool rope_vectorizes(const RopeParams &p);
hipError_t launch_rope(const RopeParams &p, hipStream_t s);

struct AttnParams {
    m27q_seqs seqs;
    m27q_cache cache;
    m27q_rows q, out;
    float scale;
    int window;
    int splits;     // parts of each sequence's keys
    float *part;    // [tokens * heads][splits][dim] sums of the parts, where splits > 1
    float2 *stat;   // [tokens * heads][splits] their maximum (log2) and weight
    // behind shared prefixes: parts 0 .. prefix_parts - 1 are of the prefix, the others of a sequence's own keys
    m27q_prefixes prefix;
    int prefix_parts;
    int own_least;  // keys of a part of those at least
};
struct AttnPlan {
    int few;        // the kernel for few rows
    int splits;
};
// Workgroups of a part of the keys.
long long attn_groups(const m27q_seqs &seqs, uint32_t q_heads, const m27q_cache &cache);
AttnPlan attn_plan(const m27q_seqs &seqs, uint32_t q_heads, const m27q_cache &cache, int cus);
size_t attn_scratch(const m27q_seqs &seqs, uint32_t q_heads, uint32_t dim, int splits);
hipError_t launch_attn(const AttnParams &p, const AttnPlan &plan, hipStream_t s);

// Attention behind shared prefixes: the prefixes' keys for the rows of a group, then each
// sequence's own, as parts of one softmax.
struct SharedPlan {
    AttnPlan prefix;  // no parts: not worth a pass of its own, every sequence reads all of its keys
    int own;          // parts of a sequence's own keys
    int own_least;    // keys of one of them at least, whole tiles
};
long long shared_groups(const m27q_seqs &seqs, const m27q_prefixes &prefix, uint32_t q_heads, const m27q_cache &cache);
SharedPlan shared_plan(const m27q_seqs &seqs, const m27q_prefixes &prefix, uint32_t q_heads, const m27q_cache &cache,
                       int cus);
hipError_t launch_shared(const AttnParams &p, const SharedPlan &plan, hipStream_t s);

struct NormParams {
    m27q_rows x, add, sum, out;  // of add, sum and out any may have no ptr
    int tokens;
    const float *weight;         // or NULL
    float eps;
    int8_t *q;                   // codes, or NULL; their scales and sums
    float *d;
    uint32_t *s;
};
bool norm_fits(const NormParams &p);
hipError_t launch_norm(const NormParams &p, hipStream_t s);

size_t sample_scratch(uint32_t rows, uint32_t n);
hipError_t launch_sample_rows(const m27q_sampling &p, void *scratch, hipStream_t s);

hipError_t launch_delta(const m27q_delta &d, void *scratch, hipStream_t s);
size_t delta_scratch(uint32_t n, uint32_t tokens, uint32_t max_len, uint32_t heads, uint32_t dk, uint32_t dv);

// ------------------------------------------------------------------ device --

__host__ __device__ __forceinline__ int type_bytes(uint32_t t) { return t == M27Q_TYPE_F32 ? 4 : 2; }

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x8a __attribute__((ext_vector_type(8), aligned(16)));  // eight fp32 values in memory
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Eight values at a 16-byte aligned place, in fp32; the type is the same for
// the whole launch, so the branch is scalar.
__device__ __forceinline__ f32x8 load8(const void *p, long long at, uint32_t type) {
    if (type == M27Q_TYPE_F32) return *(const f32x8a *)((const float *)p + at);
    if (type == M27Q_TYPE_F16) return __builtin_convertvector(*(const f16x8 *)((const _Float16 *)p + at), f32x8);
    return __builtin_convertvector(*(const bf16x8 *)((const __bf16 *)p + at), f32x8);
}
__device__ __forceinline__ void store8(void *p, long long at, uint32_t type, f32x8 v) {
    if (type == M27Q_TYPE_F32) *(f32x8a *)((float *)p + at) = v;
    else if (type == M27Q_TYPE_F16) *(f16x8 *)((_Float16 *)p + at) = __builtin_convertvector(v, f16x8);
    else *(bf16x8 *)((__bf16 *)p + at) = __builtin_convertvector(v, bf16x8);
}
__device__ __forceinline__ float load1(const void *p, long long at, uint32_t type) {
    if (type == M27Q_TYPE_F32) return ((const float *)p)[at];
    if (type == M27Q_TYPE_F16) return (float)((const _Float16 *)p)[at];
    return (float)((const __bf16 *)p)[at];
}
__device__ __forceinline__ void store1(void *p, long long at, uint32_t type, float v) {
    if (type == M27Q_TYPE_F32) ((float *)p)[at] = v;
    else if (type == M27Q_TYPE_F16) ((_Float16 *)p)[at] = (_Float16)v;
    else ((__bf16 *)p)[at] = (__bf16)v;
}

// Rows of sequence s within the call's bounds: first row, the end of all its
// rows (places count back from there) and how many of them are worked on.
struct SeqRows {
    int first, end, count;
};
__device__ __forceinline__ SeqRows seq_rows(const int32_t *start, int s, int tokens, int most) {
    const int a = min(max(start[s], 0), tokens), b = min(max(start[s + 1], a), tokens);
    return {a, b, min(b - a, most)};
}

}  // namespace m27q
