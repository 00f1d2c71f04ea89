// m27q_norm.hip -- root-mean-square norm of rows with a residual's addition, and
// the normed rows as the quantized activation of the next product.
//
//   h = x + add;  y = w h / sqrt(mean(h^2) + eps)
//
// of each head's dim values; h and y as rows of any type, y's per-32 codes as
// m27q_quant_act makes them.  h is fp32 until the end: y is of h before the
// rounding to the sum's type.
#include "m27q_device.h"
#include "m27q_mix.h"

namespace m27q {

namespace {

constexpr int kThreads = 256;

// The sum over a workgroup's threads, in an order that does not vary.
__device__ __forceinline__ float sum_group(float v, float *lds, int waves) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = lds[0];
    for (int i = 1; i < waves; ++i) s += lds[i];
    return s;
}

// Any dim and alignment, a value a thread at a time: a workgroup a row, which it reads twice.
__global__ __launch_bounds__(kThreads) void k_norm_any(const NormParams p) {
    __shared__ float lds[kThreads / 64];
    const int t = blockIdx.x / p.x.heads, head = blockIdx.x - t * p.x.heads, dim = (int)p.x.dim;
    const long long xr = (long long)t * p.x.token_stride + (long long)head * p.x.head_stride;
    const long long ar = (long long)t * p.add.token_stride + (long long)head * p.add.head_stride;
    const long long sr = (long long)t * p.sum.token_stride + (long long)head * p.sum.head_stride;
    const long long yr = (long long)t * p.out.token_stride + (long long)head * p.out.head_stride;
    auto at = [&](int i) {
        const float x = load1(p.x.ptr, xr + i, p.x.type);
        return p.add.ptr ? x + load1(p.add.ptr, ar + i, p.add.type) : x;
    };
    float ss = 0;
    for (int i = threadIdx.x; i < dim; i += kThreads) {
        const float h = at(i);
        ss = __builtin_fmaf(h, h, ss);
    }
    const float r = 1.0f / __builtin_sqrtf(sum_group(ss, lds, kThreads / 64) / (float)dim + p.eps);
    const long long base = ((long long)t * p.x.heads + head) * dim;
    for (int i = threadIdx.x; i < dim; i += kThreads) {  // (codes: dim % 32 == 0, so half waves are whole or out)
        const float h = at(i);
        float y = h * r;
        if (p.weight) y *= p.weight[i];
        if (p.sum.ptr) store1(p.sum.ptr, sr + i, p.sum.type, h);
        if (p.out.ptr) store1(p.out.ptr, yr + i, p.out.type, y);
        if (p.q) {
            float d;
            uint32_t s;
            p.q[base + i] = (int8_t)quant32(y, &d, &s);
            if ((threadIdx.x & 31) == 0) {
                p.d[(base + i) / 32] = d;
                p.s[(base + i) / 32] = s;
            }
        }
    }
}

}  // namespace

bool norm_fits(const NormParams &p) { return (long long)p.tokens * p.x.heads * kThreads < (1ll << 32); }

hipError_t launch_norm(const NormParams &p, hipStream_t s) {
    hipLaunchKernelGGL(k_norm_any, dim3((unsigned)(p.tokens * p.x.heads)), dim3(kThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace m27q
