// m27q_norm.hip -- root-mean-square norm of rows with a residual's addition, and
// the normed rows as the quantized activation of the next product.
//
//   h = x + add;  y = w h / sqrt(mean(h^2) + eps)
//
// of each head's dim values; h and y as rows of any type, y's per-32 codes as
// m27q_quant_act makes them.  h is fp32 until the end: y is of h before the
// rounding to the sum's type.
//
// Memory bounds it: a row is read once, kept in registers between the sum of its squares and the
// outputs (k_norm_row, k_norm_heads), and the codes are made where y is, which saves the
// quantizer's launch and 8 bytes a value.  4096 rows of 5120, residual, sum and codes (278 MB): 49 us, 5.7 TB/s;
// 1531 x 24 heads of 256, BF16 (38 MB): 10; a row of 5120: 3.6, a launch.
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

// Any dim and alignment, a value a thread at a time: a workgroup a row, which it reads twice.  4096 rows of 5120,
// F32 with sum and y: 92 us, 63 by units of 8; BF16 92 and 31; 98304 heads of 256 168 and 33.
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

// Eight of a row's values: h, with the residual's loads beside x's.
struct Unit8 {
    f32x8 x, a;
};
__device__ __forceinline__ void load_unit(const NormParams &p, long long xr, long long ar, int i, Unit8 &u) {
    u.x = load8(p.x.ptr, xr + 8 * i, p.x.type);
    if (p.add.ptr) u.a = load8(p.add.ptr, ar + 8 * i, p.add.type);
}
__device__ __forceinline__ f32x8 unit_h(const NormParams &p, const Unit8 &u) { return p.add.ptr ? u.x + u.a : u.x; }
__device__ __forceinline__ float unit_squares(f32x8 h, float s) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_fmaf(h[j], h[j], s);
    return s;
}
__device__ __forceinline__ void store_unit(const NormParams &p, long long sr, long long yr, long long base, int i, f32x8 h, f32x8 w,
                                           float r) {
    f32x8 y = h * r;
    if (p.weight) y *= w;
    if (p.sum.ptr) store8(p.sum.ptr, sr + 8 * i, p.sum.type, h);
    if (p.out.ptr) store8(p.out.ptr, yr + 8 * i, p.out.type, y);
    if (p.q) {  // four lanes have a group of 32
        float d;
        uint32_t s;
        const uint2 q = quant32x8(make_float4(y[0], y[1], y[2], y[3]), make_float4(y[4], y[5], y[6], y[7]), &d, &s);
        const long long at = base + 8 * i;
        *(uint2 *)(p.q + at) = q;
        if ((i & 3) == 0) {
            p.d[at / 32] = d;
            p.s[at / 32] = s;
        }
    }
}

// Long rows: a workgroup a row, U units of 8 values a thread, in registers between the two passes.
template <int U, int THREADS>
__global__ __launch_bounds__(THREADS) void k_norm_row(const NormParams p, int threads) {
    __shared__ float lds[THREADS / 64];
    const int t = blockIdx.x / p.x.heads, head = blockIdx.x - t * p.x.heads, units = (int)p.x.dim / 8;
    const long long xr = (long long)t * p.x.token_stride + (long long)head * p.x.head_stride;
    const long long ar = (long long)t * p.add.token_stride + (long long)head * p.add.head_stride;
    Unit8 u[U];
    f32x8 w[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int i = (int)threadIdx.x + k * threads;
        if (i < units) load_unit(p, xr, ar, i, u[k]);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int i = (int)threadIdx.x + k * threads;
        if (i < units && p.weight) w[k] = *(const f32x8a *)(p.weight + 8 * i);
    }
    float ss = 0;
    f32x8 h[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
        if ((int)threadIdx.x + k * threads < units) {
            h[k] = unit_h(p, u[k]);
            ss = unit_squares(h[k], ss);
        }
    const float r = 1.0f / __builtin_sqrtf(sum_group(ss, lds, threads / 64) / (float)(int)p.x.dim + p.eps);
    const long long sr = (long long)t * p.sum.token_stride + (long long)head * p.sum.head_stride;
    const long long yr = (long long)t * p.out.token_stride + (long long)head * p.out.head_stride;
    const long long base = ((long long)t * p.x.heads + head) * p.x.dim;
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int i = (int)threadIdx.x + k * threads;
        if (i < units) store_unit(p, sr, yr, base, i, h[k], w[k], r);
    }
}

// Short rows (a head's): L lanes a row.
template <int L>
__global__ __launch_bounds__(kThreads) void k_norm_heads(const NormParams p, long long rows) {
    const long long row = (long long)blockIdx.x * (kThreads / L) + threadIdx.x / L;
    const int i = threadIdx.x & (L - 1), units = (int)p.x.dim / 8;
    if (row >= rows) return;
    const int t = (int)(row / p.x.heads), head = (int)(row - (long long)t * p.x.heads);
    const bool live = i < units;
    Unit8 u;
    f32x8 w, h = {};
    if (live) {
        load_unit(p, (long long)t * p.x.token_stride + (long long)head * p.x.head_stride,
                  (long long)t * p.add.token_stride + (long long)head * p.add.head_stride, i, u);
        if (p.weight) w = *(const f32x8a *)(p.weight + 8 * i);
        h = unit_h(p, u);
    }
    float ss = unit_squares(h, 0);
#pragma unroll
    for (int o = L / 2; o; o >>= 1) ss += __shfl_xor(ss, o);
    const float r = 1.0f / __builtin_sqrtf(ss / (float)(int)p.x.dim + p.eps);
    if (live)
        store_unit(p, (long long)t * p.sum.token_stride + (long long)head * p.sum.head_stride,
                   (long long)t * p.out.token_stride + (long long)head * p.out.head_stride, row * p.x.dim, i, h, w, r);
}

bool rows16(const m27q_rows &r) {
    const int b = type_bytes(r.type);
    return !r.ptr || ((uintptr_t)r.ptr % 16 == 0 && r.token_stride * b % 16 == 0 && r.head_stride * b % 16 == 0);
}

}  // namespace

// Units of 8 values need whole units in a head and 16-byte aligned rows.
static bool norm_vectorizes(const NormParams &p) {
    return p.x.dim % 8 == 0 && p.x.dim <= 4 * 8 * 1024 && rows16(p.x) && rows16(p.add) && rows16(p.sum) && rows16(p.out) &&
           (uintptr_t)p.weight % 16 == 0;
}

// The kernel for a call, and a row's threads.  A head's lanes for up to 512 values: 98304 heads of 96 15.8 us, a workgroup
// each 35.5; of 256 32.6 and 36.9 (65536 of 512: 43.1 and 41.4).  Longer rows: a unit a thread, two of 16 bits (BF16, 4096
// rows of 5120: two 30.5 us, one 32.9, four 34.3; of 2048 12.9, 14.5 and 13.1; of 8192 46.4, 49.5 and 49.7.  F32: 63.9, 62.6
// and 66.0, a single row 3.7, 3.4 and 4.2).  Not by the number of rows: the squares are summed in one order in any batch.
enum NormKind { kAny, kLanes, kUnits1, kUnits2, kUnits4 };
struct NormForm {
    NormKind kind;
    int threads;
};
static NormForm norm_form(const NormParams &p) {
    const int units = (int)p.x.dim / 8;
    if (!norm_vectorizes(p)) return {kAny, kThreads};
    if (units <= 64) {
        int L = 4;
        while (L < units) L *= 2;
        return {kLanes, L};
    }
    if (units > 128 && units <= 2048 && p.x.type != M27Q_TYPE_F32) return {kUnits2, (units + 127) / 128 * 64};
    if (units <= 1024) return {kUnits1, (units + 63) / 64 * 64};
    return {units <= 2048 ? kUnits2 : kUnits4, 1024};
}

// Work-items of a grid's x are less than 2^32.
bool norm_fits(const NormParams &p) {
    return (long long)p.tokens * p.x.heads * norm_form(p).threads <= (1ll << 32) - kThreads;
}

hipError_t launch_norm(const NormParams &p, hipStream_t s) {
    const long long rows = (long long)p.tokens * p.x.heads;
    const NormForm f = norm_form(p);
    const dim3 grid((unsigned)(f.kind == kLanes ? (rows * f.threads + kThreads - 1) / kThreads : rows)), block(f.threads);
    switch (f.kind) {
        case kAny: hipLaunchKernelGGL(k_norm_any, grid, block, 0, s, p); break;
        case kLanes: {
            auto k = f.threads == 4 ? k_norm_heads<4> : f.threads == 8 ? k_norm_heads<8> : f.threads == 16 ? k_norm_heads<16>
                     : f.threads == 32 ? k_norm_heads<32> : k_norm_heads<64>;
            hipLaunchKernelGGL(k, grid, dim3(kThreads), 0, s, p, rows);
            break;
        }
        case kUnits1: hipLaunchKernelGGL((k_norm_row<1, 1024>), grid, block, 0, s, p, f.threads); break;
        case kUnits2: hipLaunchKernelGGL((k_norm_row<2, 1024>), grid, block, 0, s, p, f.threads); break;
        default: hipLaunchKernelGGL((k_norm_row<4, 1024>), grid, block, 0, s, p, f.threads);
    }
    return hipGetLastError();
}

}  // namespace m27q
