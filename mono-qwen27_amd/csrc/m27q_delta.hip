// m27q_delta.hip -- the gated delta rule: for each head a state S[dv][dk] and
//   S <- e^g S;  u = beta (v - S k);  S <- S + u k^T;  out = scale S q.
#include "m27q_internal.h"
#include "m27q_mix.h"

namespace m27q {

namespace {

__device__ __forceinline__ float quad_sum(float x) {
    x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0xB1, 0xF, 0xF, true));
    x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x4E, 0xF, 0xF, true));
    return x;
}

template <typename T>
struct Vec4;
template <>
struct Vec4<float> {
    typedef f32x4 t;
};
template <>
struct Vec4<_Float16> {
    typedef f16x4 t;
};
template <>
struct Vec4<__bf16> {
    typedef bf16x4 t;
};

// Row by row: a wave holds 16 rows of a head's state in registers, four lanes a
// row (dk = 16 i + 4 (lane % 4) + 0 .. 3 in its i-th quadruple, so that a load
// covers 64 contiguous bytes of a row and a row's sum is two DPP steps).  For a
// single row the state's bytes bound it: it is read and written once.  The two
// products of a row (S k, S q) are taken from the old state, with
// S_new q = e^g S q + u (k.q): one pass, then the update.
template <int DK, typename T>
__global__ __launch_bounds__(64) void k_delta_rows(const m27q_delta d) {
    typedef typename Vec4<T>::t T4;
    constexpr int N = DK / 16;
    const int parts = d.v.dim / 16;
    const int head = blockIdx.x / parts, part = blockIdx.x - head * parts, s = blockIdx.y;
    const int kh = d.head_map == M27Q_HEADS_CYCLED ? head % (int)d.k.heads : head / (int)(d.v.heads / d.k.heads);
    const int lane = threadIdx.x, r = part * 16 + (lane >> 2), c = 4 * (lane & 3);
    const SeqRows sr = seq_rows(d.start, s, (int)d.tokens, (int)d.max_len);
    const int slot = d.slots ? d.slots[s] : s;
    const bool held = slot >= 0 && (uint32_t)slot < d.n_slots;
    const long long at = (((long long)slot * d.v.heads + head) * d.v.dim + r) * DK + c;

    f32x4 S[N];
#pragma unroll
    for (int i = 0; i < N; ++i) S[i] = f32x4{0, 0, 0, 0};
    if (held && d.state_in) {
#pragma unroll
        for (int i = 0; i < N; ++i) S[i] = *(const f32x4 *)(d.state_in + at + 16 * i);
    }
    const T *q = (const T *)d.q.ptr + (long long)sr.first * d.q.token_stride + (long long)kh * d.q.head_stride + c;
    const T *k = (const T *)d.k.ptr + (long long)sr.first * d.k.token_stride + (long long)kh * d.k.head_stride + c;
    const T *v = (const T *)d.v.ptr + (long long)sr.first * d.v.token_stride + (long long)head * d.v.head_stride + r;
    T *out = (T *)d.out.ptr + (long long)sr.first * d.out.token_stride + (long long)head * d.out.head_stride + r;
    const float *g = d.g + (long long)sr.first * d.v.heads + head, *beta = d.beta + (long long)sr.first * d.v.heads + head;
    for (int t = 0; t < sr.count; ++t) {
        f32x4 kk[N], qq[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            kk[i] = __builtin_convertvector(*(const T4 *)(k + 16 * i), f32x4);
            qq[i] = __builtin_convertvector(*(const T4 *)(q + 16 * i), f32x4);
        }
        const float e = expf(*g), b = *beta, vv = (float)*v;
        f32x4 sk = {}, sq = {}, kq = {};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sk += S[i] * kk[i];
            sq += S[i] * qq[i];
            kq += kk[i] * qq[i];
        }
        const float u = b * (vv - e * quad_sum(sk[0] + sk[1] + sk[2] + sk[3]));
        const float o = e * quad_sum(sq[0] + sq[1] + sq[2] + sq[3]) + u * quad_sum(kq[0] + kq[1] + kq[2] + kq[3]);
#pragma unroll
        for (int i = 0; i < N; ++i) S[i] = S[i] * e + kk[i] * u;
        if ((lane & 3) == 0) *out = (T)(d.scale * o);
        k += d.k.token_stride;
        q += d.q.token_stride;
        v += d.v.token_stride;
        out += d.out.token_stride;
        g += d.v.heads;
        beta += d.v.heads;
    }
    if (held && d.state_out) {
#pragma unroll
        for (int i = 0; i < N; ++i) *(f32x4 *)(d.state_out + at + 16 * i) = S[i];
    }
}

template <int DK, typename T>
hipError_t launch_t(const m27q_delta &d, void *scratch, hipStream_t s) {
    hipLaunchKernelGGL((k_delta_rows<DK, T>), dim3(d.v.heads * (d.v.dim / 16), d.n), dim3(64), 0, s, d);
    return hipGetLastError();
}

}  // namespace

size_t delta_scratch(uint32_t n, uint32_t tokens, uint32_t max_len, uint32_t heads, uint32_t dk, uint32_t dv) {
    return 16;
}

hipError_t launch_delta(const m27q_delta &d, void *scratch, hipStream_t s) {
    switch (d.v.type) {
        case M27Q_TYPE_F32:
            return d.k.dim == 64 ? launch_t<64, float>(d, scratch, s) : launch_t<128, float>(d, scratch, s);
        case M27Q_TYPE_F16:
            return d.k.dim == 64 ? launch_t<64, _Float16>(d, scratch, s) : launch_t<128, _Float16>(d, scratch, s);
        default:
            return d.k.dim == 64 ? launch_t<64, __bf16>(d, scratch, s) : launch_t<128, __bf16>(d, scratch, s);
    }
}

}  // namespace m27q
