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
// S_new q = e^g S q + u (k.q): one pass, then the update.  64 sequences of 48 heads of 128 x
// 128: 407 MB in 71 us, 5.7 TB/s (x / 2 from as many states into others runs at 6.1, in place at
// 5.9).  Of more rows the 160 fp32 operations a lane and row bound it, 0.5 us where a SIMD has one
// wave; the next row's loads ahead of them changed nothing (16 rows 12.3 and 12.1 us), and cost
// the single row registers.
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
        float e = expf(*g);
        const float b = *beta, vv = (float)*v;
        f32x4 sk = {}, sq = {}, kq = {};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sk += S[i] * kk[i];
            sq += S[i] * qq[i];
            kq += kk[i] * qq[i];
        }
        float u = b * (vv - e * quad_sum(sk[0] + sk[1] + sk[2] + sk[3]));
        float o = e * quad_sum(sq[0] + sq[1] + sq[2] + sq[3]) + u * quad_sum(kq[0] + kq[1] + kq[2] + kq[3]);
        if (__builtin_expect(__any(!__builtin_isfinite(u) || !__builtin_isfinite(o)), 0)) {
            // in the rule's order: these products may pass fp32 where its own do not
            sk = sq = f32x4{};
#pragma unroll
            for (int i = 0; i < N; ++i) {
                S[i] *= e;
                sk += S[i] * kk[i];
                __builtin_amdgcn_sched_barrier(0);  // few registers
            }
            u = b * (vv - quad_sum(sk[0] + sk[1] + sk[2] + sk[3]));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                S[i] += kk[i] * u;
                sq += S[i] * qq[i];
                __builtin_amdgcn_sched_barrier(0);
            }
            o = quad_sum(sq[0] + sq[1] + sq[2] + sq[3]);
            e = 1, u = 0;
        }
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

// ---------------------------------------------------------------- chunks --
//
// C = 64 rows at a time.  With G_i the sum of g over the chunk's rows up to i,
// the rule within a chunk that starts from S is
//   (I + A) U = diag(beta) (V - diag(e^G) K S^T),
//       A_ij = beta_i e^(G_i - G_j) k_i.k_j   for j < i,
//   out = scale diag(e^G) Q S^T + P U,  P_ij = scale e^(G_i - G_j) q_i.k_j  for j <= i,
//   S <- e^(G_C) S + (diag(e^(G_C - G)) U)^T K.
// A first launch, parallel over chunks, makes T = (I + A)^-1 diag(beta), P and the
// factors; a second one walks the chunks of a sequence with 32 rows of a head's
// state, three products that wait for each other a chunk.
//
// Products are fp32-accurate on the bf16 matrix units, 16 times the rate of the
// fp32 ones: a value is the sum of three bf16 values (8 + 8 + 8 bits; F16 takes
// two, BF16 one) and a product the six partial products above 2^-24 of it, which
// is 6 / 16 of the fp32 instructions' time.

constexpr int kC = 64;       // rows of a chunk
constexpr int kSlice = 32;   // state rows of a workgroup

template <typename T>
struct In;  // an input type's values as bf16 pieces
template <>
struct In<float> {
    static constexpr int N = 3;
    typedef f32x8a raw;
};
template <>
struct In<_Float16> {
    static constexpr int N = 2;
    typedef f16x8 raw;
};
template <>
struct In<__bf16> {
    static constexpr int N = 1;
    typedef bf16x8 raw;
};

// x as N bf16 values each, rounded to nearest: what the ones before leave over.  Two values
// at a time, their fp32 forms taken from the packed word (one conversion for both).
template <int N>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        p[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
        if (j + 1 < N) {
            asm("" : "+v"(p[j]));  // one conversion, not one more for each half
            x -= __builtin_bit_cast(float, p[j] << 16);
            y -= __builtin_bit_cast(float, p[j] & 0xffff0000u);
        }
    }
}
template <int N>
__device__ __forceinline__ void split(f32x8 x, bf16x8 (&p)[N]) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    u4 w[N];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t t[N];
        split2<N>(x[2 * i], x[2 * i + 1], t);
#pragma unroll
        for (int j = 0; j < N; ++j) w[j][i] = t[j];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) p[j] = __builtin_bit_cast(bf16x8, w[j]);
}
template <int N>
__device__ __forceinline__ void split(f32x4 x, bf16x4 (&p)[N]) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    uint32_t a[N], b[N];
    split2<N>(x[0], x[1], a);
    split2<N>(x[2], x[3], b);
#pragma unroll
    for (int j = 0; j < N; ++j) p[j] = __builtin_bit_cast(bf16x4, u2{a[j], b[j]});
}

// Whether the pieces of a value are finite: from the middle between the largest bf16 value and
// the next that there would be, the first one is not.
__device__ __forceinline__ bool fits(float x) { return fabsf(x) < 0x1.ffp127f; }

// c[j] += a[j] b over 16x16 tiles and 32 of the contraction, the smallest parts first; the
// tiles in turn, so that a product does not wait for the one before.
template <int NC, int NA, int NB>
__device__ __forceinline__ void mma(const bf16x8 (&a)[NC][NA], const bf16x8 (&b)[NB], f32x4 (&c)[NC]) {
#pragma unroll
    for (int o = 2; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (o - i >= 0 && o - i < NB)
#pragma unroll
                for (int j = 0; j < NC; ++j)
                    c[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j][i], b[o - i], c[j], 0, 0, 0);
}

#define LDS_AS __attribute__((address_space(3)))

// What the first launch leaves for a chunk and a head: the pieces of T and of P as operand
// rows, six blocks of 16 rows and 32 columns (row tile m's first, and its second where that
// is not above the diagonal) of [3][64 lanes][8]; then the factors.
constexpr int kBlocks = 6, kBlockHalves = 3 * 64 * 8;
constexpr int kT = 0, kP = kBlocks * kBlockHalves / 2, kEg = 2 * kP, kEc = kEg + kC, kLast = kEc + kC,
              kRecord = kLast + 64;  // in floats
__device__ __forceinline__ int block_of(int m, int i) { return m < 2 ? m : 2 * m - 2 + i; }

// The place of a sequence's first chunk among all: places do not meet, as a
// sequence has at most one chunk more than whole ones.
__device__ __forceinline__ long long chunk_place(int first, int s) { return first / kC + s; }

// NI steps of the sequence's 16 rows from t0 as operand rows: lane m = lane % 16, values
// 32 (i0 + i) + 8 (lane / 16) + 0 .. 7 of row t0 + m.  Past the end it is the last row again,
// without a branch (a load under one would keep later waits from telling it from others):
// beta is 0 there, which keeps such rows out of U and of the state.
template <int NI, typename T>
__device__ __forceinline__ void load_rows(const m27q_rows &r, long long first, int head, int t0, int count, int i0,
                                          typename In<T>::raw (&x)[NI]) {
    const int lane = threadIdx.x & 63, t = min(t0 + (lane & 15), count - 1);
    const T *p = (const T *)r.ptr + first * r.token_stride + (long long)head * r.head_stride + 32 * i0;
    const unsigned long long at = (unsigned long long)(uint32_t)t * (uint32_t)r.token_stride + 8 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < NI; ++i) x[i] = *(const typename In<T>::raw *)(p + at + 32 * i);
}
template <typename T>
__device__ __forceinline__ void pieces(typename In<T>::raw x, bf16x8 (&p)[In<T>::N]) {
    if constexpr (In<T>::N == 1) p[0] = x;
    else split<In<T>::N>(__builtin_convertvector(x, f32x8), p);
}

// Place of a value in LDS, rows of W values: the 16-byte chunks of a row are exchanged by the row,
// so that 16 rows' reads of a column of chunks, and two groups of a transposing read (32-byte
// units of rows r .. r + 3 and r + 8 .. r + 11), meet different ones of the 64 banks.
template <int W>
__device__ __forceinline__ int lds_at(int row, int col) {
    const int x = (W == 128 ? row : row >> 1) & (W == 128 ? 15 : 7), top = x >> (W == 128 ? 3 : 2);
    const int swap = W == 128 ? ((x & 7) << 1) ^ (top * 9) : ((x & 3) << 1) ^ (top * 5);
    return row * W + (((col >> 3) ^ swap) << 3) + (col & 7);
}

// A chunk of a key head: K K^T and Q K^T once, then for its value heads (every `parts`-th
// of them) the triangular inverse.  Chains of dependent steps bound it (vector and matrix
// instructions fill 27 of 63 us), so it is made small, for four workgroups a CU: K lies in LDS
// 64 columns at a time, P takes A's place there (4096 rows of 16 key heads of 3, fp32: 49 us;
// with two workgroups a CU 63).  It writes 36 KB a chunk and head.
template <int DK, typename T>
__global__ __launch_bounds__(256, 4) void k_delta_prepare(const m27q_delta d, float *scratch, int parts) {
    constexpr int N = In<T>::N, LM = kC + 4;
    constexpr size_t planes = sizeof(__bf16) * N * kC * 64, mats = sizeof(float) * 2 * kC * LM;
    __shared__ __attribute__((aligned(16))) char mem[planes > mats ? planes : mats];
    __shared__ double Gs[3][kC];
    __shared__ float Bs[3][kC];
    __bf16 *kp = (__bf16 *)mem;                                        // K's pieces, 64 columns at a time, [N][kC][64]
    float *Am = (float *)mem, *Xm = Am + kC * LM;  // then A, P after it, and the inverse of I + A
    const int s = blockIdx.z, kh = blockIdx.y / parts, part = blockIdx.y - kh * parts, t0 = blockIdx.x * kC;
    const SeqRows sr = seq_rows(d.start, s, (int)d.tokens, (int)d.max_len);
    if (t0 >= sr.count) return;
    const int kheads = (int)d.k.heads, per = (int)d.v.heads / kheads;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;

    const auto head_of = [&](int which) {
        return d.head_map == M27Q_HEADS_CYCLED ? which * kheads + kh : kh * per + which;
    };
    const auto record = [&](int which) {
        return scratch + ((chunk_place(sr.first, s) + blockIdx.x) * d.v.heads + head_of(which)) * (long long)kRecord;
    };
    // A head's factors, three heads at a time, a wave each.  The sums of g are in 64 bits, as
    // differences of them are taken.
    const auto factors = [&](int which) {
        if (wave == 3 || which >= per) return;
        float *rec = record(which);
        const bool in = t0 + lane < sr.count;
        const long long at = (long long)(sr.first + t0 + lane) * d.v.heads + head_of(which);
        const float gf = in ? d.g[at] : 0.0f, beta = in ? d.beta[at] : 0.0f;
        double x = gf < -1e4f ? -1e4 : (double)gf;  // e^-10000 is 0 as e^-inf is, and no inf - inf
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(x, o);
            x += lane >= o ? y : 0.0;
        }
        const double last = __shfl(x, 63);
        Gs[wave][lane] = x;
        Bs[wave][lane] = beta;
        rec[kEg + lane] = __builtin_isfinite(beta) ? expf((float)x) : __builtin_nanf("");  // to be seen by the walk
        rec[kEc + lane] = expf((float)(last - x));
        if (lane == 0) rec[kLast] = expf((float)last);
    };

    typename In<T>::raw x[2], y[2];
    load_rows<2, T>(d.k, sr.first, kh, t0 + 16 * wave, sr.count, 0, x);
    load_rows<2, T>(d.q, sr.first, kh, t0 + 16 * wave, sr.count, 0, y);
    factors(part + wave * parts);
    f32x4 prod[4][2] = {};  // tiles of K K^T and Q K^T at rows 16 wave, columns 16 j
#pragma unroll
    for (int h = 0; h < DK / 64; ++h) {
        bf16x8 a[2][2][N];  // K's and Q's
        if (h) __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            pieces<T>(x[i], a[i][0]);
            pieces<T>(y[i], a[i][1]);
#pragma unroll
            for (int j = 0; j < N; ++j)
                *(bf16x8 *)(kp + j * kC * 64 + lds_at<64>(16 * wave + n, 32 * i + 8 * g)) = a[i][0][j];
        }
        if (h + 1 < DK / 64) {
            load_rows<2, T>(d.k, sr.first, kh, t0 + 16 * wave, sr.count, 2, x);
            load_rows<2, T>(d.q, sr.first, kh, t0 + 16 * wave, sr.count, 2, y);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > wave) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                bf16x8 b[N];
#pragma unroll
                for (int u = 0; u < N; ++u)
                    b[u] = *(const bf16x8 *)(kp + u * kC * 64 + lds_at<64>(16 * j + n, 32 * i + 8 * g));
                mma<2, N, N>(a[i], b, prod[j]);
            }
        }
    }

    for (int which = part, slot = 0; which < per; which += parts, ++slot) {
        __syncthreads();  // K's pieces, or the last head's matrices, make room
        if (slot == 3) {
            slot = 0;
            factors(which + wave * parts);
            __syncthreads();
        }
        const double *G = Gs[slot];
        const float *B = Bs[slot];
        float *rec = record(which);
        f32x4 P[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > (wave | 1)) break;  // read by nothing
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 16 * wave + 4 * g + i, col = 16 * j + n;
                float x = 0;
                P[j][i] = 0;
                if (col <= row) {
                    const float e = expf((float)(G[row] - G[col]));
                    P[j][i] = d.scale * e * prod[j][1][i];
                    if (col < row) x = B[row] * e * prod[j][0][i];
                }
                Am[row * LM + col] = x;
                Xm[row * LM + col] = 0;
            }
        }
        __syncthreads();
        // the inverse's 16x16 blocks: on the diagonal by forward substitution, a column a lane
        const int r0 = 16 * wave;
        if (lane < 16) {
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float v = i == lane ? 1.0f : 0.0f;
#pragma unroll
                for (int k = 0; k < i; ++k) v = __builtin_fmaf(-Am[(r0 + i) * LM + r0 + k], x[k], v);
                x[i] = v;
                Xm[(r0 + i) * LM + r0 + lane] = v;
            }
        }
        // below it by diagonals: X_ij = -X_ii sum_(j <= k < i) A_ik X_kj.  The sum's rows lie
        // in the lanes as 4 g + t, so the second product takes X_ii's columns in that order.
#pragma unroll
        for (int o = 1; o < 4; ++o) {
            __syncthreads();
            if (wave < o) continue;
            const int c0 = 16 * (wave - o);
            f32x4 y[4] = {}, x = {};
#pragma unroll
            for (int k = 0; k < 4 * o; ++k)
                y[k & 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(Am[(r0 + n) * LM + c0 + 4 * k + g],
                                                                Xm[(c0 + 4 * k + g) * LM + c0 + n], y[k & 3], 0, 0, 0);
            y[0] = (y[0] + y[1]) + (y[2] + y[3]);
#pragma unroll
            for (int t = 0; t < 4; ++t)
                x = __builtin_amdgcn_mfma_f32_16x16x4f32(-Xm[(r0 + n) * LM + r0 + 4 * g + t], y[0][t], x, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) Xm[(r0 + 4 * g + i) * LM + c0 + n] = x[i];
        }
        __syncthreads();
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // a wave's own rows: written and read without a barrier
            if (j > (wave | 1)) break;
#pragma unroll
            for (int i = 0; i < 4; ++i) Am[(r0 + 4 * g + i) * LM + 16 * j + n] = P[j][i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i == 1 && wave < 2) break;
            const int at = (r0 + n) * LM + 32 * i + 8 * g;
            __bf16 *to = (__bf16 *)(rec + kT) + block_of(wave, i) * kBlockHalves + lane * 8;
            const f32x8 tt = *(const f32x8a *)(Xm + at) * *(const f32x8a *)(B + 32 * i + 8 * g);
            const f32x8 pp = *(const f32x8a *)(Am + at);
#pragma unroll
            for (int u = 0; u < 8; ++u) bad |= !fits(tt[u]) || !fits(pp[u]);
            bf16x8 x[3], y[3];
            split<3>(tt, x);
            split<3>(pp, y);
#pragma unroll
            for (int u = 0; u < 3; ++u) {
                *(bf16x8 *)(to + u * 512) = x[u];
                *(bf16x8 *)(to + 2 * (kP - kT) + u * 512) = y[u];
            }
        }
        // T or P of products or factors that pass fp32, or of values that are not finite: the walk sees this
        if (__builtin_expect(__any(bad), 0)) rec[kEg + lane] = __builtin_nanf("");
    }
}

// c[j] += a b[j], as above with one left operand.
template <int NC, int NA, int NB>
__device__ __forceinline__ void mma(const bf16x8 (&a)[NA], const bf16x8 (&b)[NC][NB], f32x4 (&c)[NC]) {
#pragma unroll
    for (int o = 2; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (o - i >= 0 && o - i < NB)
#pragma unroll
                for (int j = 0; j < NC; ++j)
                    c[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j][o - i], c[j], 0, 0, 0);
}

// A record's operand blocks of row tile m (see kT): its first, and its second or the first again.
__device__ __forceinline__ void load_blocks(const float *from, int m, bf16x8 (&x)[2][3]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __bf16 *b = (const __bf16 *)from + block_of(m, m < 2 ? 0 : i) * kBlockHalves + (threadIdx.x & 63) * 8;
#pragma unroll
        for (int u = 0; u < 3; ++u) x[i][u] = *(const bf16x8 *)(b + u * 512);
    }
}

// A chunk's rows one by one, for a chunk with a value that is not finite, or whose products come
// to one: they would carry it, times zeros, to the rows before it.  The four waves that hold the state (as in
// k_delta_chunks) sum over their columns and, through `sums`, over each other's; two barriers
// a row.
template <int DK, typename T>
__device__ __forceinline__ void row_by_row(const m27q_delta &d, const SeqRows &sr, int kh, int head, int t0, int v0,
                                                     int mt, f32x4 (&S)[DK / 64][2], float *sums, T *out) {
    constexpr int MT = DK / 64;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    auto total = [&](float x) {  // over the lanes of a state row
        x += __shfl_xor(x, 16);
        return x + __shfl_xor(x, 32);
    };
    for (int t = t0; t < min(t0 + kC, sr.count); ++t) {
        const long long row = sr.first + t;
        const T *k = (const T *)d.k.ptr + row * d.k.token_stride + (long long)kh * d.k.head_stride + 16 * MT * mt + 4 * g;
        const T *q = (const T *)d.q.ptr + row * d.q.token_stride + (long long)kh * d.q.head_stride + 16 * MT * mt + 4 * g;
        const T *v = (const T *)d.v.ptr + row * d.v.token_stride + (long long)head * d.v.head_stride;
        const float e = expf(d.g[row * d.v.heads + head]), beta = d.beta[row * d.v.heads + head];
        float kk[MT][4], part[2] = {};
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                kk[m][i] = (float)k[16 * m + i];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    S[m][j][i] *= e;
                    part[j] += S[m][j][i] * kk[m][i];
                }
            }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float x = total(part[j]);
            if (g == 0) sums[mt * kSlice + 16 * j + n] = x;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float x = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) x += sums[w * kSlice + 16 * j + n];
            const float u = beta * ((float)v[min(v0 + 16 * j, (int)d.v.dim - 16) + n] - x);
            part[j] = 0;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    S[m][j][i] += u * kk[m][i];
                    part[j] += S[m][j][i] * (float)q[16 * m + i];
                }
            const float y = total(part[j]);
            if (g == 0) sums[(4 + mt) * kSlice + 16 * j + n] = y;
        }
        __syncthreads();
        if (mt == 0 && lane < kSlice && v0 + lane < (int)d.v.dim) {
            float o = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) o += sums[(4 + w) * kSlice + lane];
            out[(long long)t * d.out.token_stride + lane] = (T)(d.scale * o);
        }
    }
}

// The walk over a sequence's chunks, 32 state rows of a head a workgroup.  Four waves carry
// the state (16 MT of its columns each, in accumulators) through the three products that wait
// for each other; four more, one on each SIMD beside them, do what nothing waits for: Q S^T
// and P U, the outputs, and the next chunk's K in pieces.  Wave m of either four has rows
// 16 m .. of the chunk.  Three barriers a chunk part
//   1  X = K S^T, R = V - diag(e^G) X        | K of the next chunk into pieces
//   2  U = T R                               | Q S^T
//   3  S <- e^(G_C) S + K^T diag(..) U       | K's pieces to LDS, out = .. Q S^T + P U
// What in R, U or diag(..) U does not fit its pieces (T and P: by a NaN in e^G) is seen before the
// third part, which then takes the chunk's rows one by one from the state that it started from.
// Operands that come from memory are asked for again, for the next chunk, as soon as they have
// been used, without branches (a load under one would keep later waits from telling it apart).
// The chain of the three products bounds it: 4096 rows of 48 heads of 128 (192 workgroups),
// fp32, 64 chunks of 3.7 us, 7000 to 8500 cycles of which the matrix units work 2900, LDS 3400;
// Q S^T in pieces is the longest of part 2.  237 us after 49 of preparation; four BF16 sequences
// of up to 1531 rows (768 workgroups, one a CU at a time) 193 after 59.  Measured before reads
// stood in front of the products: Q cut into pieces in part 1 instead 333 us against 304 in all,
// K's loads and pieces with the state's waves 337; BF16 in the 128 registers of two workgroups a
// CU, which spill, 296 against 258.
template <int DK, typename T>
__global__ __launch_bounds__(512) void k_delta_chunks(const m27q_delta d, const float *scratch) {
    constexpr int N = In<T>::N, KS = DK / 32, MT = DK / 64;
    __shared__ __attribute__((aligned(16))) __bf16 kp[N * kC * DK];         // K's pieces [N][row][dk]
    __shared__ __attribute__((aligned(16))) __bf16 sb[3 * kSlice * DK];     // the state's [3][dv][dk]
    __shared__ __attribute__((aligned(16))) __bf16 rb[3 * kSlice * kC];     // the right-hand sides' [3][dv][row]
    __shared__ __attribute__((aligned(16))) __bf16 ub[3 * kSlice * kC];     // U's
    __shared__ __attribute__((aligned(16))) __bf16 wb[3 * kSlice * kC];     // diag(e^(G_C - G)) U's
    __shared__ int odd[2];                                                  // this chunk's products hold: no, and the next one's
    // workgroups of one key head and sequence are gridDim.x apart, so that where that is a
    // multiple of the XCDs they share an L2
    const int kheads = (int)d.k.heads, per = (int)d.v.heads / kheads, slices = (int)(d.v.dim + kSlice - 1) / kSlice;
    const int s = blockIdx.x / kheads, kh = blockIdx.x - s * kheads;
    const int which = blockIdx.y / slices, v0 = (blockIdx.y - which * slices) * kSlice;
    const int head = d.head_map == M27Q_HEADS_CYCLED ? which * kheads + kh : kh * per + which;
    const SeqRows sr = seq_rows(d.start, s, (int)d.tokens, (int)d.max_len);
    const int slot = d.slots ? d.slots[s] : s;
    const bool held = slot >= 0 && (uint32_t)slot < d.n_slots;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mt = wave & 3;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, row = 16 * mt + 4 * g;
    const float *rec = scratch + (chunk_place(sr.first, s) * d.v.heads + head) * (long long)kRecord;
    const long long step = (long long)d.v.heads * kRecord;  // behind the last chunk's there is room for one more
    const bool in[2] = {v0 < (int)d.v.dim, v0 + 16 < (int)d.v.dim};
    const long long at = (((long long)slot * d.v.heads + head) * d.v.dim + v0 + n) * DK + 16 * MT * mt + 4 * g;
    T *const out = (T *)d.out.ptr + (long long)sr.first * d.out.token_stride + (long long)head * d.out.head_stride + v0;

    if (sr.count == 0) {  // its state stays
        if (wave < 4 && held && d.state_out)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    if (in[j])
                        *(f32x4 *)(d.state_out + at + 16 * j * DK + 16 * m) =
                            d.state_in ? *(const f32x4 *)(d.state_in + at + 16 * j * DK + 16 * m) : f32x4{};
        return;
    }
    if (threadIdx.x < 2) odd[threadIdx.x] = 0;

    auto get_rows = [&](const __bf16 *from, int j, int i, bf16x8(&b)[3]) {
#pragma unroll
        for (int u = 0; u < 3; ++u)
            b[u] = *(const bf16x8 *)(from + u * kSlice * kC + lds_at<kC>(16 * j + n, 32 * i + 8 * g));
    };
    // Reads stay in front of the matrix instructions: left alone, the compiler puts each before
    // its own, to wait for it.
    auto reads_first = [] { __builtin_amdgcn_sched_barrier(0x476); };  // vector, scalar and memory instructions may pass
    auto get_both = [&](const __bf16 *from, bf16x8(&b)[2][2][3]) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) get_rows(from, j, i, b[i][j]);
        reads_first();
    };
    auto get_state = [&](int i, bf16x8(&b)[2][3]) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int u = 0; u < 3; ++u)
                b[j][u] = *(const bf16x8 *)(sb + u * kSlice * DK + lds_at<DK>(16 * j + n, 32 * i + 8 * g));
    };

    if (wave < 4) {
        // dk = 16 (MT mt + m) + 4 g + i of row v0 + 16 j + n
        f32x4 S[MT][2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                S[m][j] = f32x4{};
                if (held && d.state_in && in[j]) S[m][j] = *(const f32x4 *)(d.state_in + at + 16 * j * DK + 16 * m);
            }
        auto put_state = [&]() {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    bf16x4 p[3];
                    split<3>(S[m][j], p);
#pragma unroll
                    for (int u = 0; u < 3; ++u)
                        *(bf16x4 *)(sb + u * kSlice * DK + lds_at<DK>(16 * j + n, 16 * (MT * mt + m) + 4 * g)) = p[u];
                }
        };
        // rows `row` .. of value 16 j + n of the slice
        auto put_rows = [&](__bf16 *to, int j, f32x4 x) {
            bf16x4 p[3];
            split<3>(x, p);
#pragma unroll
            for (int u = 0; u < 3; ++u) *(bf16x4 *)(to + u * kSlice * kC + lds_at<kC>(16 * j + n, row)) = p[u];
        };
        bf16x8 t[2][3];
        T v[2][4];
        f32x4 eg, ec;
        float last;
        auto load_v = [&](int t0) {
            const T *x = (const T *)d.v.ptr + (long long)sr.first * d.v.token_stride + (long long)head * d.v.head_stride;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned long long o =
                    (unsigned long long)(uint32_t)min(t0 + row + i, sr.count - 1) * (uint32_t)d.v.token_stride + n;
#pragma unroll
                for (int j = 0; j < 2; ++j) v[j][i] = x[min(v0 + 16 * j, (int)d.v.dim - 16) + o];
            }
        };
        load_v(0);
        eg = *(const f32x4 *)(rec + kEg + row);
        load_blocks(rec + kT, mt, t);
        ec = *(const f32x4 *)(rec + kEc + row);
        last = rec[kLast];
        put_state();
        __syncthreads();
        for (int t0 = 0; t0 < sr.count; t0 += kC) {
            rec += step;
            int *const mark = odd + (t0 / kC & 1);
            f32x4 x[2] = {};
            {
                bf16x8 a[2][N], b[2][2][3];
                auto get = [&](int i) {
#pragma unroll
                    for (int u = 0; u < N; ++u)
                        a[i & 1][u] = *(const bf16x8 *)(kp + u * kC * DK + lds_at<DK>(16 * mt + n, 32 * i + 8 * g));
                    get_state(i, b[i & 1]);
                };
                get(0);
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    if (i + 1 < KS) get(i + 1);
                    reads_first();
                    mma<2, N, 3>(a[i & 1], b[i & 1], x);
                }
            }
            bf16x8 kt[2][MT][N];  // K^T: dk = 16 (MT mt + m) + n, rows 32 i + 8 g + 0 .. 7
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int u = 0; u < N; ++u) {
                        typedef short s4 __attribute__((ext_vector_type(4)));
                        const int r = 32 * i + 8 * g + (n >> 2), c = 16 * (MT * mt + m) + 4 * (n & 3);
                        const s4 y0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (LDS_AS s4 *)(kp + u * kC * DK + lds_at<DK>(r, c)));
                        const s4 y1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (LDS_AS s4 *)(kp + u * kC * DK + lds_at<DK>(r + 4, c)));
                        kt[i][m][u] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(y0, y1, 0, 1, 2, 3, 4, 5, 6, 7));
                    }
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f32x4 r;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    r[i] = (float)v[j][i] - eg[i] * x[j][i];
                    bad |= !fits(r[i]);
                }
                put_rows(rb, j, r);
            }
            load_v(t0 + kC);
            eg = *(const f32x4 *)(rec + kEg + row);
            __syncthreads();
            {
                f32x4 u[2] = {};
                bf16x8 b[2][2][3];
                get_both(rb, b);
                mma<2, 3, 3>(t[0], b[0], u);
                if (mt >= 2) mma<2, 3, 3>(t[1], b[1], u);  // otherwise above the diagonal
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const f32x4 w = u[j] * ec;
                    put_rows(ub, j, u[j]);
                    put_rows(wb, j, w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) bad |= !fits(u[j][i]) || !fits(w[i]);
                }
            }
            if (bad) *mark = 1;
            if (threadIdx.x == 0) odd[(t0 / kC & 1) ^ 1] = 0;  // the last chunk's: read before the barrier above
            load_blocks(rec + kT, mt, t);
            const float decay = last;
            ec = *(const f32x4 *)(rec + kEc + row);
            last = rec[kLast];
            __syncthreads();
            if (__builtin_expect(*mark, 0)) {
                row_by_row<DK, T>(d, sr, kh, head, t0, v0, mt, S, (float *)ub, out);
            } else {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int j = 0; j < 2; ++j) S[m][j] *= decay;
                bf16x8 b[2][2][3];
                get_both(wb, b);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma<2, N, 3>(kt[i][m], b[i], S[m]);
            }
            put_state();
            __syncthreads();
        }
        if (held && d.state_out)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    if (in[j]) *(f32x4 *)(d.state_out + at + 16 * j * DK + 16 * m) = S[m][j];
        return;
    }

    typename In<T>::raw k[KS], q[KS];
    bf16x8 p[2][3], ka[KS][N];
    auto cut = [&]() {
#pragma unroll
        for (int i = 0; i < KS; ++i) pieces<T>(k[i], ka[i]);
    };
    auto put_k = [&]() {
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int u = 0; u < N; ++u)
                *(bf16x8 *)(kp + u * kC * DK + lds_at<DK>(16 * mt + n, 32 * i + 8 * g)) = ka[i][u];
    };
    load_rows<KS, T>(d.k, sr.first, kh, 16 * mt, sr.count, 0, k);
    load_rows<KS, T>(d.q, sr.first, kh, 16 * mt, sr.count, 0, q);
    load_blocks(rec + kP, mt, p);
    f32x4 eg = *(const f32x4 *)(rec + kEg + row);
    cut();
    load_rows<KS, T>(d.k, sr.first, kh, kC + 16 * mt, sr.count, 0, k);
    put_k();
    __syncthreads();
    for (int t0 = 0; t0 < sr.count; t0 += kC) {
        rec += step;
        cut();
        load_rows<KS, T>(d.k, sr.first, kh, t0 + 2 * kC + 16 * mt, sr.count, 0, k);
        __syncthreads();
        f32x4 x[2] = {};
        {
            bf16x8 b[2][2][3];
            get_state(0, b[0]);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                bf16x8 a[N];
                pieces<T>(q[i], a);
                if (i + 1 < KS) get_state(i + 1, b[(i + 1) & 1]);
                reads_first();
                mma<2, N, 3>(a, b[i & 1], x);
            }
        }
        load_rows<KS, T>(d.q, sr.first, kh, t0 + kC + 16 * mt, sr.count, 0, q);
#pragma unroll
        for (int j = 0; j < 2; ++j) x[j] *= eg * d.scale;
        eg = *(const f32x4 *)(rec + kEg + row);
        __syncthreads();
        const bool slow = odd[t0 / kC & 1];
        put_k();
        if (__builtin_expect(slow, 0)) {
            for (int i = 0; i < 2 * min(kC, sr.count - t0); ++i) __syncthreads();  // those of row_by_row
        } else {
            bf16x8 b[2][2][3];
            get_both(ub, b);
            mma<2, 3, 3>(p[0], b[0], x);
            if (mt >= 2) mma<2, 3, 3>(p[1], b[1], x);
        }
        load_blocks(rec + kP, mt, p);
        // last, behind all loads: a wait for one of those would be one for these too
        if (!slow) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + row + i;
                if (t >= sr.count) break;
                T *o = out + (unsigned long long)(uint32_t)t * (uint32_t)d.out.token_stride + n;
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (in[j]) o[16 * j] = (T)x[j][i];
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------- few --
//
// The same products for 16 rows at a time in one launch: a wave holds 16 rows of the state,
// lane n = lane % 16 the row n, g = lane / 16 its values 16 m + 4 g + 0 .. 3.  That is where
// a matrix instruction leaves a 16x16 result, and two such tiles side by side are its right
// operand over 32 of the contraction if the left one's columns are taken in the same order;
// a result's 4 g + 0 .. 3 are the operand of the instructions over 16.  So state, right-hand
// sides and U go from product to product in registers.  The four waves of a workgroup share
// K and Q in LDS, as operand blocks [step][piece][64 lanes][8], a step of 32 columns a wave.
// A wave's chain of products bounds it where a SIMD has one (16 more rows 4.2 us).  With several
// neither that nor the bytes do alone: 16 rows of 8 sequences, 48 heads of 128 x 128, take 17.1 us
// in fp32 and 15.1 in BF16 (row by row 35) for 50 MB of states, 3 TB/s.  All waves are there at
// once, so all load, then all compute, then all store; what needs no state (A and its inverse)
// stands behind the products that wait for it.

template <int NA, int NB>
__device__ __forceinline__ void mma16(const bf16x4 (&a)[NA], const bf16x4 (&b)[NB], f32x4 &c) {
    typedef short s4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int o = 2; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (o - i >= 0 && o - i < NB)
                c = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a[i]), __builtin_bit_cast(s4, b[o - i]),
                                                              c, 0, 0, 0);
}

// Lane (n, g)'s 16 bytes of an operand block: for a transposing read (rows 4 g + 0 .. 3, every
// g' of them) the rows of a g lie apart by banks.
__device__ __forceinline__ int few_at(int n, int g) { return (16 * g + (n ^ (4 * g))) * 8; }

constexpr int kFew = 16;

template <int DK, typename T>
__global__ __launch_bounds__(256, 3) void k_delta_few(const m27q_delta d) {
    typedef typename Vec4<T>::t T4;
    constexpr int N = In<T>::N, KS = DK / 32, M = DK / 16, LA = kFew + 4;
    __shared__ __attribute__((aligned(16))) __bf16 kb[KS * N * 512], qb[KS * N * 512];
    __shared__ f32x4 part[KS][2][64];
    __shared__ __attribute__((aligned(16))) float At[4][kFew * LA];
    __shared__ __attribute__((aligned(16))) double Gs[kFew];
    __shared__ __attribute__((aligned(16))) float egs[kFew], ecs[kFew], bs[kFew];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int groups = ((int)d.v.dim + 63) / 64;
    const int head = blockIdx.x / groups, v0 = 64 * (blockIdx.x - head * groups) + 16 * wave, s = blockIdx.y;
    const int kh = d.head_map == M27Q_HEADS_CYCLED ? head % (int)d.k.heads : head / (int)(d.v.heads / d.k.heads);
    const SeqRows sr = seq_rows(d.start, s, (int)d.tokens, (int)d.max_len);
    const int slot = d.slots ? d.slots[s] : s;
    const bool in = v0 < (int)d.v.dim, held = in && slot >= 0 && (uint32_t)slot < d.n_slots;
    const int vc = min(v0, (int)d.v.dim - 16) + n;
    const long long at = (((long long)slot * d.v.heads + head) * d.v.dim + vc) * DK + 4 * g;

    f32x4 S[M];
#pragma unroll
    for (int m = 0; m < M; ++m) S[m] = f32x4{};
    if (held && d.state_in) {
#pragma unroll
        for (int m = 0; m < M; ++m) S[m] = *(const f32x4 *)(d.state_in + at + 16 * m);
    }
    const T *kr = (const T *)d.k.ptr + (long long)sr.first * d.k.token_stride + (long long)kh * d.k.head_stride + 4 * g;
    const T *qr = (const T *)d.q.ptr + (long long)sr.first * d.q.token_stride + (long long)kh * d.q.head_stride + 4 * g;
    const T *vr = (const T *)d.v.ptr + (long long)sr.first * d.v.token_stride + (long long)head * d.v.head_stride + vc;
    T *out = (T *)d.out.ptr + (long long)sr.first * d.out.token_stride + (long long)head * d.out.head_stride + vc;
    const float *gs = d.g + (long long)sr.first * d.v.heads + head, *betas = d.beta + (long long)sr.first * d.v.heads + head;

    // Past the end the last row again, with beta = 0.
    T4 k[2], q[2];
    T v[4];
    float gf, beta;
    const auto load = [&](int t0) {
        const unsigned long long t = (uint32_t)min(t0 + n, sr.count - 1);
        if (wave < KS) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                k[h] = *(const T4 *)(kr + t * (uint32_t)d.k.token_stride + 32 * wave + 16 * h);
                q[h] = *(const T4 *)(qr + t * (uint32_t)d.q.token_stride + 32 * wave + 16 * h);
            }
        }
        gf = gs[t * d.v.heads], beta = betas[t * d.v.heads];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = vr[(unsigned long long)(uint32_t)min(t0 + 4 * g + i, sr.count - 1) * (uint32_t)d.v.token_stride];
    };
    if (sr.count > 0) load(0);
    for (int t0 = 0; t0 < sr.count; t0 += kFew) {
        if (wave < KS) {
            bf16x8 a[N], b[2][N];
            f32x4 kk[2] = {};  // of rows j = 4 g + 0 .. 3 and the row n: k_j.k_n and k_j.q_n
            const f32x4 k0 = __builtin_convertvector(k[0], f32x4), k1 = __builtin_convertvector(k[1], f32x4);
            const f32x4 q0 = __builtin_convertvector(q[0], f32x4), q1 = __builtin_convertvector(q[1], f32x4);
            split<N>(__builtin_shufflevector(k0, k1, 0, 1, 2, 3, 4, 5, 6, 7), a);
            split<N>(__builtin_shufflevector(q0, q1, 0, 1, 2, 3, 4, 5, 6, 7), b[1]);
#pragma unroll
            for (int u = 0; u < N; ++u) {
                b[0][u] = a[u];
                *(bf16x8 *)(kb + (wave * N + u) * 512 + few_at(n, g)) = a[u];
                *(bf16x8 *)(qb + (wave * N + u) * 512 + few_at(n, g)) = b[1][u];
            }
            mma<2, N, N>(a, b, kk);
            part[wave][0][lane] = kk[0];
            part[wave][1][lane] = kk[1];
        }
        float last;  // sums of g in 64 bits: differences of them are taken
        {
            const bool row = t0 + n < sr.count;
            const float gn = row ? gf : 0.0f, b = row ? beta : 0.0f;
            double x = gn < -1e4f ? -1e4 : (double)gn;  // e^-10000 is 0 as e^-inf is, and no inf - inf
#pragma unroll
            for (int o = 1; o < kFew; o <<= 1) {
                const double y = __shfl_up(x, o, kFew);
                x += n >= o ? y : 0.0;
            }
            const double end = __shfl(x, kFew - 1, kFew);
            last = expf((float)end);
            if (wave == 0 && g == 0) {
                Gs[n] = x;
                egs[n] = expf((float)x);
                ecs[n] = expf((float)(end - x));
                bs[n] = b;
            }
        }
        f32x4 vt;
#pragma unroll
        for (int i = 0; i < 4; ++i) vt[i] = (float)v[i];
        if (t0 + kFew < sr.count) load(t0 + kFew);
        __syncthreads();

        f32x4 xy[2] = {};  // K S^T and Q S^T
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            bf16x8 a[2][N], b[3];
            split<3>(__builtin_shufflevector(S[2 * i], S[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7), b);
#pragma unroll
            for (int u = 0; u < N; ++u) {
                a[0][u] = *(const bf16x8 *)(kb + (i * N + u) * 512 + few_at(n, g));
                a[1][u] = *(const bf16x8 *)(qb + (i * N + u) * 512 + few_at(n, g));
            }
            mma<2, N, 3>(a, b, xy);
        }
        // Row n of A (into LDS, by columns) and of P, at 4 g + 0 .. 3
        f32x4 kk = part[0][0][lane], P = part[0][1][lane];
#pragma unroll
        for (int i = 1; i < KS; ++i) kk += part[i][0][lane], P += part[i][1][lane];
        const f32x4 eg = *(const f32x4 *)(egs + 4 * g), ec = *(const f32x4 *)(ecs + 4 * g), bt = *(const f32x4 *)(bs + 4 * g);
        const double Gn = Gs[n];
        const float bn = bs[n];
        double Gj[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) Gj[i] = Gs[4 * g + i];
        float *A = At[wave];
        int row = n;
        asm("" : "+v"(row));  // what is compared with it is not kept in registers over the loop
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = 4 * g + i;
            const float e = expf((float)(Gn - Gj[i])), p = d.scale * e * P[i], a = bn * e * kk[i];
            P[i] = j <= row ? p : 0.0f;
            A[j * LA + n] = j < row ? a : 0.0f;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // Row n of (I + A)^-1 from its last value back: x_j = [j = n] - sum_(k > j) x_k A_kj
        float x[kFew];
#pragma unroll
        for (int j = kFew - 1; j >= 0; --j) {
            float y = j == row ? 1.0f : 0.0f;
#pragma unroll
            for (int o = (kFew - 1) / 4; o >= (j + 1) / 4; --o) {
                const f32x4 a = *(const f32x4 *)(A + j * LA + 4 * o);
#pragma unroll
                for (int i = 3; i >= 0; --i)
                    if (4 * o + i > j) y = __builtin_fmaf(-x[4 * o + i], a[i], y);
            }
            x[j] = y;
            if (j % 4 == 0) asm volatile("" : "+v"(x[j]) : : "memory");  // not all of A at once in registers
        }
        f32x4 t, r, u = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x0 = x[i], x1 = x[4 + i], x2 = x[8 + i], x3 = x[12 + i], lo = g & 1 ? x1 : x0, hi = g & 1 ? x3 : x2;
            t[i] = (g & 2 ? hi : lo) * bt[i];
            r[i] = vt[i] - eg[i] * xy[0][i];
        }
        bf16x4 tp[3], pp[3], rp[3], up[3], wp[3];
        split<3>(t, tp);
        split<3>(r, rp);
        split<3>(P, pp);
        mma16(tp, rp, u);
        const f32x4 w = u * ec;
        f32x4 y = xy[1] * (eg * d.scale);
        split<3>(u, up);
        split<3>(w, wp);
        mma16(pp, up, y);
        bool bad = !__builtin_isfinite(last);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            bad |= !(fits(r[i]) && fits(u[i]) && fits(w[i]) && __builtin_isfinite(y[i]));
        if (__builtin_expect(__any(bad), 0)) {
            // Row by row: products would carry a value that is not finite, times zeros, to the rows before it.
            for (int i = t0; i < min(t0 + kFew, sr.count); ++i) {
                const float e = expf(gs[(unsigned long long)i * d.v.heads]), b = betas[(unsigned long long)i * d.v.heads];
                const T *ki = kr + (unsigned long long)i * (uint32_t)d.k.token_stride;
                const T *qi = qr + (unsigned long long)i * (uint32_t)d.q.token_stride;
                const float vi = (float)vr[(unsigned long long)i * (uint32_t)d.v.token_stride];
                float sk = 0, sq = 0;
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    __builtin_amdgcn_sched_barrier(0);  // few registers
#pragma unroll
                    for (int o = 0; o < 4; ++o) {
                        S[m][o] *= e;
                        sk += S[m][o] * (float)ki[16 * m + o];
                    }
                }
                sk += __shfl_xor(sk, 16);
                sk += __shfl_xor(sk, 32);
                const float ui = b * (vi - sk);
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int o = 0; o < 4; ++o) {
                        S[m][o] += ui * (float)ki[16 * m + o];
                        sq += S[m][o] * (float)qi[16 * m + o];
                    }
                }
                sq += __shfl_xor(sq, 16);
                sq += __shfl_xor(sq, 32);
                if (in && g == 0) out[(unsigned long long)i * (uint32_t)d.out.token_stride] = (T)(d.scale * sq);
            }
        } else {
#pragma unroll
            for (int m = 0; m < M; ++m) {
                typedef short s4 __attribute__((ext_vector_type(4)));
                bf16x4 a[N];  // K^T: value 16 m + n of rows 4 g + 0 .. 3
#pragma unroll
                for (int j = 0; j < N; ++j)
                    a[j] = __builtin_bit_cast(
                        bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (LDS_AS s4 *)(kb + ((m >> 1) * N + j) * 512 + few_at(4 * g + (n >> 2), n & 3) + 4 * (m & 1))));
                S[m] *= last;
                mma16(a, wp, S[m]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (in && t0 + 4 * g + i < sr.count)
                    out[(unsigned long long)(uint32_t)(t0 + 4 * g + i) * (uint32_t)d.out.token_stride] = (T)y[i];
        }
        __syncthreads();
    }
    if (held && d.state_out) {
#pragma unroll
        for (int m = 0; m < M; ++m) *(f32x4 *)(d.state_out + at + 16 * m) = S[m];
    }
}

// Which of the three.  A wave of 16 state rows takes 0.3 to 0.6 us a row, or 3.5 us for 16 and
// at first 4 more; the chunks take 3.7 us for 64 with a quarter of the waves, after 15 us of
// two launches and the rows' preparation.  48 heads of 128, fp32, us by rows, 16 rows and chunks:
//   1 sequence   8 rows 7.6 and 8.5, 10 rows 9.0 and 8.7; 64 rows 22.8 and 23.3, 96 rows 31.7 and 26.7
//   4 sequences  6 rows 12.4 and 12.8, 8 rows 14.6 and 12.9; 128 rows 53 and 58, 256 rows 97 and 88
//   8 sequences  5 rows 17 and 17, 16 rows 35 and 18; 128 rows 72 and 107, 384 rows 194 and 211
// (bf16: 1 sequence 6 rows 7.2 and 7.8, 8 rows 8.8 and 8.0; 4 sequences 5 rows 11.9 and 11.2;
// 4 sequences of 128 rows 44 and 41.)  The longest sequence of a call chooses for all of them: 2048
// rows beside 63 single tokens take 1407 us by chunks, apart 151 and 70.
constexpr uint32_t kMostFew = 64;
// Waves of 16 state rows that have rows to the end, about: short sequences beside a long one do not keep the card busy.
unsigned long long waves(const m27q_delta &d) {
    return (unsigned long long)d.tokens * (d.v.heads * (d.v.dim / 16)) / (d.max_len ? d.max_len : 1);
}
bool by_chunks(uint32_t rows, unsigned long long waves) { return rows > kMostFew && rows > waves / 8; }
bool by_rows(uint32_t rows, unsigned long long waves, bool wide) {
    return rows < (waves <= 1024 ? 8u : wide ? 6u : 5u);
}

template <int DK, typename T>
hipError_t launch_t(const m27q_delta &d, void *scratch, hipStream_t s) {
    const unsigned long long w = waves(d);
    if (by_rows(d.max_len, w, sizeof(T) == 4)) {
        hipLaunchKernelGGL((k_delta_rows<DK, T>), dim3(d.v.heads * (d.v.dim / 16), d.n), dim3(64), 0, s, d);
        return hipGetLastError();
    }
    if (!by_chunks(d.max_len, w)) {
        hipLaunchKernelGGL((k_delta_few<DK, T>), dim3(d.v.heads * ((d.v.dim + 63) / 64), d.n), dim3(256), 0, s, d);
        return hipGetLastError();
    }
    const unsigned chunks = (d.max_len + kC - 1) / kC, per = d.v.heads / d.k.heads;
    // A workgroup makes all value heads of a key head where that leaves enough of them: at 16 key
    // heads of 3, fp32, 1024 rows 92 against 88 us (256 workgroups), 1500 rows 127 against 132.
    const unsigned parts = (unsigned long long)chunks * d.k.heads * d.n >= 384 ? 1 : per;
    hipLaunchKernelGGL((k_delta_prepare<DK, T>), dim3(chunks, d.k.heads * parts, d.n), dim3(256), 0, s, d,
                       (float *)scratch, (int)parts);
    const unsigned slices = (d.v.dim + kSlice - 1) / kSlice;
    hipLaunchKernelGGL((k_delta_chunks<DK, T>), dim3(d.n * d.k.heads, per * slices), dim3(512), 0, s, d,
                       (const float *)scratch);
    return hipGetLastError();
}

}  // namespace

size_t delta_scratch(uint32_t n, uint32_t tokens, uint32_t max_len, uint32_t heads, uint32_t dk, uint32_t dv) {
    if (max_len <= kMostFew) return 16;  // not by the number of sequences: what does for many does for fewer
    return ((size_t)tokens / kC + n + 1) * heads * kRecord * sizeof(float);
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
