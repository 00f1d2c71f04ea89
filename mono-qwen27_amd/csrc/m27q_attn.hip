// m27q_attn.hip -- attention of a chunk of new tokens over a paged cache.
//
// The rows of one sequence and one cache head (tokens x the query heads that
// share it, token by token) are taken 32 to a wave, so that a key is read once
// for all of its query heads.  Everything is computed transposed: S^T = K Q^T
// leaves a query per lane (a column of the 32x32 tile), so a row's maximum and
// sum are in-lane up to one exchange between the wave's halves, and the
// weights P^T are, as they lie in the registers, the right operand of
// O^T += V^T P^T (the keys of a 16-key step in the order that the first
// product leaves them, V read in the same order).
//
// Two kernels.  Many rows (k_attn) share tiles of keys that a workgroup brings into LDS once:
// the matrix units bound it.  Up to 32 rows of a sequence and cache head (k_attn_few) are one
// wave's, so its waves take keys apart from each other, and the cache's bytes bound it.
// Such rows through k_attn: one token over 1021 keys 22.6 us, by k_attn_few 11.2; 32 tokens over
// up to 16381 keys 312 and 287; 2 x 5 rows over 32768 keys 62.4 and 59.8; 64 tokens over 3000
// keys 125 and 112.  The longest sequence of a call chooses for all of them: 512 rows beside 31
// single tokens over 13400 to 16384 keys take 1411 us, apart 44 and 340.
#include "m27q_device.h"
#include "m27q_internal.h"
#include "m27q_mix.h"

namespace m27q {

namespace {

constexpr float kLog2e = 0x1.715476p+0f;
constexpr int kWaves = 4;        // of a workgroup
constexpr int kRows = 32;        // of a wave
constexpr int kKeys = 32;        // of a tile in LDS
constexpr int kMaxSplits = 64;

#define LDS_AS __attribute__((address_space(3)))

template <bool BF>
struct Num;
template <>
struct Num<false> {
    typedef _Float16 t;
    typedef f16x2 t2;
    typedef f16x4 t4;
    typedef f16x8 t8;
    static __device__ __forceinline__ f32x16 mma(t8 a, t8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mma(t8 a, t8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Num<true> {
    typedef __bf16 t;
    typedef bf16x2 t2;
    typedef bf16x4 t4;
    typedef bf16x8 t8;
    static __device__ __forceinline__ f32x16 mma(t8 a, t8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mma(t8 a, t8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// The maximum and the sum of a value over the lanes of a row: l and l ^ 32, for rows of a
// 16-row tile l ^ 16 and l ^ 48 as well.
template <int RW>
__device__ __forceinline__ float max_row(float x) {
    unsigned u = __builtin_bit_cast(unsigned, x);
    if constexpr (RW == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        u = __builtin_bit_cast(unsigned, fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1])));
    }
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
template <int RW>
__device__ __forceinline__ float sum_row(float x) {
    unsigned u = __builtin_bit_cast(unsigned, x);
    if constexpr (RW == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        u = __builtin_bit_cast(unsigned, __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]));
    }
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// What one workgroup works on.
struct Work {
    int s, head;        // sequence, cache head
    int row0, rows;     // its first row of the sequence's rows, and all of those
    int first, end;     // the sequence's rows among the call's
    int kv_end;         // place of row r's own key: kv_end - q_count + r / group
    int lo, hi;         // keys it looks at
    bool gaps;          // some page of them is not one
};

// Tiles of K and V in LDS: kKeys rows of D values, 16-byte chunks exchanged within a row so
// that no kind of read meets bank conflicts (64 banks, 16 lanes of 16 bytes or 32 of 8 at a
// time): K's chunk c of row r lies at c ^ (r & 15) (a read takes one chunk column of 16 rows;
// D = 64, two rows to the banks: c ^ (r / 2 & 7)), V's 32-byte unit u at u ^ v_swap(r) (a
// transposing read takes two units of 4 rows, or one of 8).  Exchanges of row bits add up.
template <int D>
__device__ __forceinline__ int k_chunk(int row, int c) {
    return c ^ (D >= 128 ? row & 15 : (row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_swap(int row) {
    return D >= 128 ? ((row & 3) << 1) ^ ((row >> 2) & 1) : (row & 2) ^ ((row >> 2) & 1);
}
template <int D>
__device__ __forceinline__ int v_chunk(int row, int c) {
    return c ^ (v_swap<D>(row) << 1);
}

// The page of the keys that this wave brings into the tile at k0 (a multiple
// of 32): kKeys / kWaves of them in a row, which no page boundary parts.  In a
// vector register, so that nothing waits for it before its use.
__device__ __forceinline__ int tile_page(const AttnParams &p, const Work &w, int k0) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int page = min(k0 + wave * (kKeys / kWaves), w.hi - 1) >> __builtin_ctz(p.cache.page_size);
    asm("" : "+v"(page));
    return (p.seqs.table + (long long)w.s * p.seqs.table_stride)[page];
}

// The tile of keys k0 .. k0 + 31 into LDS, straight from memory: a wave's load
// fills 1 KiB, 512 / D rows.  CHECKED: keys past `hi` or on a page that is not
// one are not read; their rows of V become zeros (their weights are 0, which a
// NaN left in LDS would turn into NaN), their scores are masked later.
template <int D, bool CHECKED>
__device__ __forceinline__ void load_tile(const AttnParams &p, const Work &w, int k0, int page, LDS_AS char *kt,
                                          LDS_AS char *vt) {
    constexpr int RPI = 512 / D, CPR = D / 8, RPW = kKeys / kWaves;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int key = k0 + wave * RPW, id = __builtin_amdgcn_readfirstlane(page);
    const int rows = CHECKED ? ((uint32_t)id < p.cache.pages ? w.hi - key : 0) : RPW;
    const long long at = ((long long)(CHECKED && rows <= 0 ? 0 : id) * p.cache.page_stride +
                          ((long long)w.head * p.cache.page_size + (key & (int)(p.cache.page_size - 1))) * D) * 2;
    const __amdgpu_buffer_rsrc_t kg = buf_rsrc((const char *)p.cache.k + at, RPW * D * 2);
    const __amdgpu_buffer_rsrc_t vg = buf_rsrc((const char *)p.cache.v + at, RPW * D * 2);
    const int r0 = lane / CPR, pc = lane % CPR, first = wave * RPW + r0;
    const uint32_t ko = r0 * D * 2 + k_chunk<D>(first, pc) * 16, vo = r0 * D * 2 + v_chunk<D>(first, pc) * 16;
#pragma unroll
    for (int i = 0; i < RPW / RPI; ++i) {  // row first + i RPI: its chunks are the first's with i RPI exchanged as well
        LDS_AS char *kd = kt + (wave * RPW + i * RPI) * D * 2, *vd = vt + (wave * RPW + i * RPI) * D * 2;
        if (!CHECKED || i * RPI + r0 < rows) {
            const uint32_t ka = ko ^ (k_chunk<D>(i * RPI, 0) * 16), va = vo ^ (v_chunk<D>(i * RPI, 0) * 16);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(kg, (LDS_AS void *)kd, 16, ka, i * 1024, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(vg, (LDS_AS void *)vd, 16, va, i * 1024, 0, 0);
        } else {
            *(LDS_AS f32x4 *)(vd + lane * 16) = f32x4{0, 0, 0, 0};
        }
    }
}

// A barrier behind which the tiles that the waves asked for are there: loads
// into LDS count as memory loads, which a plain barrier does not wait for.
__device__ __forceinline__ void tile_barrier() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Puts zeros for the values of V that are not finite, in ROWS rows that this
// wave brought into LDS: some row of queries may not see their key, and
// its weight of 0 would make NaN of them.  Returns whether there were any.
template <int D, bool BF, int ROWS>
__device__ __forceinline__ bool clear_odd(LDS_AS char *at) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
    constexpr int N = ROWS * D / 512;
    at += (threadIdx.x & 63) * 16;
    u4 v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = *(LDS_AS u4 *)(at + i * 1024);
    u16x2 top = {0, 0};  // the largest of the values without their signs
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[i][j] & 0x7fff7fffu));
    const bool odd = top[0] >= E || top[1] >= E;
    if (__builtin_expect(odd, 0)) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool a = (v[i][j] & E) == E, b = ((v[i][j] >> 16) & E) == E;
                v[i][j] &= (a ? 0xffff0000u : ~0u) & (b ? 0xffffu : ~0u);
            }
            *(LDS_AS u4 *)(at + i * 1024) = v[i];
        }
    }
    return odd;
}

// One wave's rows, RW of them (32, or 16 where there are no more): the statistics and sums
// of a softmax in one pass.  Lane l has row l % RW and, as part g = l / RW of 64 / RW, four
// consecutive keys of every 4 * 64 / RW, and likewise of the values of a sum.
template <int D, bool BF, int NP, int RW>
struct Rows {
    typedef Num<BF> N;
    typedef typename N::t T;
    typedef typename N::t4 T4;
    typedef typename N::t8 T8;
    static constexpr int G = 64 / RW, STEP = 4 * G;   // parts, and the keys that they share out
    static constexpr int NS = kKeys / G;              // scores of a tile in a lane
    static constexpr int KD = 8 * G;                  // values of a product's step
    static constexpr int NV = NS / 8;                 // steps of the keys in the second product
    template <int W, int X = 0>
    struct Acc {
        typedef f32x16 t;
    };
    template <int X>
    struct Acc<16, X> {
        typedef f32x4 t;
    };
    typedef typename Acc<RW>::t acc;
    static constexpr int NA = RW * RW / 64;           // values of an accumulator
    T8 q[D / KD];
    acc o[D / RW];
    float m, l;      // maximum of the scores (before scale) that weights are taken from; this part's sum of weights
    int place;       // of this lane's row (-1: none)

    static __device__ __forceinline__ int part() { return (threadIdx.x & 63) / RW; }
    // the i-th of this lane's keys in a tile; the j-th value of accumulator t
    static __device__ __forceinline__ int key_at(int i) { return STEP * (i / 4) + 4 * part() + i % 4; }
    static __device__ __forceinline__ int value_at(int t, int j) { return RW * t + STEP * (j / 4) + 4 * part() + j % 4; }

    __device__ __forceinline__ void clear() {
        m = -__builtin_inff();
        l = 0;
#pragma unroll
        for (int i = 0; i < D / RW; ++i) o[i] = acc{};
    }

    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    struct Raw {
        u4 v[D / KD];
    };
    // token and head: a row of the call's, also for a lane that has none (and takes zeros)
    static __device__ __forceinline__ void load_q(const AttnParams &p, int token, int head, Raw &r) {
        const T *from =
            (const T *)p.q.ptr + (long long)token * p.q.token_stride + (long long)head * p.q.head_stride + 8 * part();
#pragma unroll
        for (int i = 0; i < D / KD; ++i) r.v[i] = *(const u4 *)(from + KD * i);
    }
    __device__ __forceinline__ void set_q(const AttnParams &p, const Raw &r, bool live) {
        // a negative scale goes into q, exactly: scores are then compared before scaling
        const uint32_t flip = p.scale < 0 ? 0x80008000u : 0, keep = live ? ~0u : 0u;
#pragma unroll
        for (int i = 0; i < D / KD; ++i) q[i] = __builtin_bit_cast(T8, (r.v[i] ^ flip) & keep);
    }

    // The tile in LDS.  MASK: some of its keys may be hidden from some row, or missing.  AHEAD:
    // all of a product's reads before its first instruction, for a wave that has its SIMD (and
    // its registers) to itself; otherwise the compiler leaves each to wait for its own.
    template <bool MASK, bool AHEAD>
    __device__ __forceinline__ void tile(const AttnParams &p, const Work &w, float sc, int k0, const LDS_AS char *kt,
                                         const LDS_AS char *vt) {
        float s[NS];
        T8 pc[NV][NP];
        scores<AHEAD>(kt, s);
        weights<MASK>(p, w, sc, s, k0, pc);
        values<AHEAD>(vt, pc);
    }

    template <bool AHEAD>
    __device__ __forceinline__ void scores(const LDS_AS char *kt, float (&s)[NS]) const {
        const int r = threadIdx.x & (RW - 1);
        // chunk G i + part of key row r (and r + 16): k_chunk of it is (y ^ (G i & M)) + (G i & ~M),
        // a few addresses, the rest offsets
        constexpr int M = D >= 128 ? 15 : 7;
        const LDS_AS char *kr = kt + r * D * 2;
        int y = k_chunk<D>(r, part());
        asm("" : "+v"(y));  // addresses are made here, not kept
#pragma unroll
        for (int b = 0; b < kKeys / RW; ++b) {
            acc c = {};
            T8 a[D / KD];
#pragma unroll
            for (int i = 0; i < D / KD; ++i) {
                a[i] = *(const LDS_AS T8 *)(kr + b * RW * D * 2 + (y ^ (G * i & M)) * 16 + (G * i & ~M) * 16);
                if constexpr (!AHEAD) c = N::mma(a[i], q[i], c);
            }
            if constexpr (AHEAD) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < D / KD; ++i) c = N::mma(a[i], q[i], c);
            }
#pragma unroll
            for (int i = 0; i < NA; ++i) s[b * NA + i] = c[i];
        }
    }

    // Their weights, as NP pieces of the cache's type, each what the ones before left over.
    template <bool MASK>
    __device__ __forceinline__ void weights(const AttnParams &p, const Work &w, float sc, float (&s)[NS], int k0,
                                            T8 (&pc)[NV][NP]) {
        if constexpr (MASK) {
#pragma unroll
            for (int i = 0; i < NS; ++i) s[i] = sees(p, w, k0 + key_at(i)) ? s[i] : -__builtin_inff();
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < NS; ++i) top = fmaxf(top, s[i]);
        top = max_row<RW>(top);
        // The maximum that weights are taken from follows the rows' own only
        // when one has grown by 2^8: weights reach 2^(6 + 8) then, and lie 2^6
        // above the type's small values otherwise.  (m = -inf: no key yet.)
        if (__any(!((top - m) * sc <= 8.0f) && top != m)) {
            const float next = fmaxf(m, top);
            const bool none = m == -__builtin_inff();
            const float f = none ? 1.0f : __builtin_amdgcn_exp2f((m - next) * sc);
            m = next;
            if (__any(!none)) {
                l *= f;
#pragma unroll
                for (int i = 0; i < D / RW; ++i) o[i] *= f;
            }
        }
        const float off = 6.0f - (m == -__builtin_inff() ? 0.0f : m) * sc;
        float part = 0;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sc, off));
            part += s[i];
        }
        l += part;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            f32x8 x;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = s[8 * i + j];
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                pc[i][j] = __builtin_convertvector(x, T8);
                if (j + 1 < NP) x -= __builtin_convertvector(pc[i][j], f32x8);
            }
        }
    }

    // O += weights times values.  V^T: lane (value RW t + lane % RW, part g) takes the keys of its
    // weights, STEP (2 i + e) + 4 g + 0 .. 3.
    template <bool AHEAD>
    __device__ __forceinline__ void values(const LDS_AS char *vt, const T8 (&pc)[NV][NP]) {
        const int lane = threadIdx.x & 63, x = 4 * part() + ((lane & 15) >> 2);  // the key this lane's 16 lanes read for
        const LDS_AS char *vr = vt + x * D * 2 + (lane & 3) * 8;
        constexpr int M = D >= 128 ? 7 : 3, U = RW / 16;
        const int y = v_swap<D>(x) ^ ((lane >> 4) & (U - 1));  // 32-byte unit U t + .. of a row, exchanged
        T8 v[D / RW][NV];
#pragma unroll
        for (int t = 0; t < D / RW; ++t)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const LDS_AS char *at = vr + 2 * i * STEP * D * 2 + ((U * t & M) ^ y) * 32 + (U * t & ~M) * 32;
                v[t][i] = __builtin_shufflevector(tr4(at), tr4(at + STEP * D * 2), 0, 1, 2, 3, 4, 5, 6, 7);
                if constexpr (!AHEAD) {
#pragma unroll
                    for (int j = 0; j < NP; ++j) o[t] = N::mma(v[t][i], pc[i][j], o[t]);
                }
            }
        if constexpr (AHEAD) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < NP; ++j)
#pragma unroll
                    for (int t = 0; t < D / RW; ++t) o[t] = N::mma(v[t][i], pc[i][j], o[t]);
        }
    }

    // Whether this lane's row sees a key.
    __device__ __forceinline__ bool sees(const AttnParams &p, const Work &w, int key) const {
        bool ok = key <= place && key < w.hi && (p.window == 0 || key > place - p.window);
        if (w.gaps && ok) {
            const int32_t id =
                p.seqs.table[(long long)w.s * p.seqs.table_stride + (key >> __builtin_ctz(p.cache.page_size))];
            ok = (uint32_t)id < p.cache.pages;
        }
        return ok;
    }

    static __device__ __forceinline__ T4 tr4(const LDS_AS char *at) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(T4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s4 *)at));
    }

    // Whether some sum of this lane is not finite.
    __device__ __forceinline__ bool odd_sums() const {
        float top = 0;
#pragma unroll
        for (int t = 0; t < D / RW; ++t)
#pragma unroll
            for (int j = 0; j < NA; ++j) top = __builtin_elementwise_maximum(top, fabsf(o[t][j]));
        return !__builtin_isfinite(top);
    }

    // O += the values of V that are not finite, where they are seen: the whole of
    // their effect, as a weight is positive.
    __device__ __forceinline__ void add_odd(const AttnParams &p, const Work &w, int k0, const LDS_AS char *vt) {
        const int lane = threadIdx.x & 63;
        for (int key = 0; key < kKeys; ++key) {
            const LDS_AS char *vk = vt + key * D * 2;
            bool odd = false;
            for (int i = lane; i < D; i += 64) odd |= !__builtin_isfinite((float)*(const LDS_AS T *)(vk + i * 2));
            if (!__any(odd)) continue;
            const bool ok = sees(p, w, k0 + key);
#pragma unroll
            for (int t = 0; t < D / RW; ++t) {
#pragma unroll
                for (int j = 0; j < NA; ++j) {
                    const int d = value_at(t, j);
                    const float v = (float)*(const LDS_AS T *)(vk + (v_chunk<D>(key, d / 8) * 8 + d % 8) * 2);
                    o[t][j] += ok && !__builtin_isfinite(v) ? v : 0.0f;
                }
                __builtin_amdgcn_sched_barrier(0);  // one step's registers at a time
            }
        }
    }
};

// What a part's sums count beside the largest part's, never 0: an infinite sum stays what it is
// (and 2^-126 of a finite one is nothing beside the largest part's weight of 2^6 and more).
__device__ __forceinline__ float join_factor(float log2) { return fmaxf(__builtin_amdgcn_exp2f(log2), 0x1p-126f); }

// The first key that a row at a place sees.  Rows before place 0 see none; a window may be as
// long as its type holds, so nothing is taken off below 0.
__device__ __forceinline__ int first_key(const AttnParams &p, int place) {
    return p.window ? max(0, max(place, 0) - p.window + 1) : 0;
}

// The keys of a workgroup whose rows stand at first .. last (of len >= 0 cached tokens, so none
// of these sums passes 32 bits), and its part of them: lo a multiple of a tile, hi >= lo, and
// hi <= max_kv where there are any.
__device__ __forceinline__ void set_keys(const AttnParams &p, Work &w, int len, int first, int last) {
    w.lo = first_key(p, first) & ~(kKeys - 1);  // tiles lie whole within pages or the other way round
    w.hi = max(w.lo, min(min(len, (int)p.seqs.max_kv), last + 1));
    if (p.splits > 1) {
        const int tiles = (w.hi - w.lo + kKeys - 1) / kKeys, each = (tiles + p.splits - 1) / p.splits;
        const int end = w.hi;
        w.lo += (int)blockIdx.y * each * kKeys;
        w.hi = max(w.lo, min(end, w.lo + each * kKeys));
    }
}

// Looks at every page of the keys once, the threads of a workgroup in turn: tiles trust them then.
__device__ __forceinline__ bool has_gaps(const AttnParams &p, const Work &w) {
    const int shift = __builtin_ctz(p.cache.page_size);
    const int32_t *table = p.seqs.table + (long long)w.s * p.seqs.table_stride;
    bool bad = false;
    if (w.lo < w.hi)
        for (int i = (w.lo >> shift) + (int)threadIdx.x; i <= (w.hi - 1) >> shift; i += kWaves * 64)
            bad |= (uint32_t)table[i] >= p.cache.pages;
    return bad;
}

// Many rows: four waves of 32 rows a workgroup, K and V of a tile of 32 keys in LDS, the next
// tile on its way while this one is worked on (two workgroups a CU: what one waits for, the
// other works).  Tiles that every row sees whole are taken without masks, those at the ends of
// the causal or window mask apart.  4096 rows over 8192 keys, 24 heads of 256, BF16: 632 to 651
// us from card to card, 950 to 980 TFLOP/s of the pairs that the mask lets through (a product of
// 8192^3 runs at 1208), F16 676; to F32, with the second product once for each piece of a weight,
// 1170 and 937.  A window shorter than a workgroup's tokens leaves no tile whole, so that nothing
// is on its way while a tile is worked on: 2048 rows 114 us without a window, 73 with one of 128.
template <int D, bool BF, int NP>
__global__ __launch_bounds__(kWaves * 64, 2) void k_attn(const AttnParams p) {
    typedef Rows<D, BF, NP, kRows> R;
    typedef typename R::T T;
    __shared__ __attribute__((aligned(1024))) char kt0[kKeys * D * 2], vt0[kKeys * D * 2];
    __shared__ __attribute__((aligned(1024))) char kt1[kKeys * D * 2], vt1[kKeys * D * 2];
    const int group = (int)(p.q.heads / p.cache.heads);
    // workgroups of one (sequence, head) are seqs * heads apart in dispatch order, so that
    // where that is a multiple of the XCDs they share an L2; the last rows see the most keys
    // and go first
    const unsigned pairs = p.seqs.n * p.cache.heads, fromlast = blockIdx.x / pairs, pair = blockIdx.x - fromlast * pairs;
    const int s = pair / p.cache.heads;
    Work w;
    w.s = s;
    w.head = pair - s * p.cache.heads;
    const SeqRows sr = seq_rows(p.seqs.start, s, (int)p.seqs.tokens, (int)p.seqs.max_q);
    w.rows = sr.count * group;
    w.row0 = (int)(gridDim.x / pairs - 1 - fromlast) * kWaves * kRows;
    if (w.row0 >= w.rows) return;
    const int len = max(p.seqs.kv_len[s], 0), place0 = len - (sr.end - sr.first);  // of the sequence's first row
    const int first = place0 + w.row0 / group;
    const int last = place0 + (min(w.row0 + kWaves * kRows, w.rows) - 1) / group;
    set_keys(p, w, len, first, last);

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    const int wrow = w.row0 + wave * kRows;  // this wave's first row
    const bool live = wrow + (lane & 31) < w.rows;
    const int row = min(wrow + (lane & 31), w.rows - 1);
    const int token = sr.first + row / group, qh = w.head * group + row % group;
    R x;
    x.place = live ? place0 + row / group : -1;
    x.clear();
    typename R::Raw q;
    R::load_q(p, token, qh, q);
    x.set_q(p, q, live);
    // (a scale of 0 would make NaN of a masked score's -inf)
    const float sc = fmaxf(fabsf(p.scale) * kLog2e, 1e-37f);

    w.gaps = __syncthreads_or(has_gaps(p, w));
    // tiles [ta, tb) are seen whole by every row of the workgroup: the next one is
    // on its way while one is worked on; the others, at the ends, go one by one
    const int tiles = (w.hi - w.lo + kKeys - 1) / kKeys;
    int ta = 0, tb = 0;
    if (!w.gaps) {
        tb = max(0, min(first + 1, w.hi) - w.lo) / kKeys;
        ta = p.window ? min(tb, (max(0, first_key(p, last) - w.lo) + kKeys - 1) / kKeys) : 0;
    }
    const bool any = wrow < w.rows;
    LDS_AS char *const ka = (LDS_AS char *)kt0, *const va = (LDS_AS char *)vt0;
    LDS_AS char *const kb = (LDS_AS char *)kt1, *const vb = (LDS_AS char *)vt1;
    int id = ta < tb ? tile_page(p, w, w.lo + ta * kKeys) : 0;
    if (ta < tb) {
        load_tile<D, false>(p, w, w.lo + ta * kKeys, id, ka, va);
        id = tile_page(p, w, w.lo + (ta + 1) * kKeys);
    }
    for (int t = ta; t < tb; t += 2) {
        tile_barrier();  // tile t is there; nobody reads the other buffers any more
        if (t + 1 < tb) {
            load_tile<D, false>(p, w, w.lo + (t + 1) * kKeys, id, kb, vb);
            id = tile_page(p, w, w.lo + (t + 2) * kKeys);
        }
        if (any) x.template tile<false, false>(p, w, sc, w.lo + t * kKeys, ka, va);
        if (t + 1 >= tb) break;
        tile_barrier();
        if (t + 2 < tb) {
            load_tile<D, false>(p, w, w.lo + (t + 2) * kKeys, id, ka, va);
            id = tile_page(p, w, w.lo + (t + 3) * kKeys);
        }
        if (any) x.template tile<false, false>(p, w, sc, w.lo + (t + 1) * kKeys, kb, vb);
    }
    bool odd = false;
    for (int i = 0; i < tiles - (tb - ta); ++i) {
        const int k0 = w.lo + (i < ta ? i : i + tb - ta) * kKeys;
        __syncthreads();
        load_tile<D, true>(p, w, k0, tile_page(p, w, k0), ka, va);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        odd |= clear_odd<D, BF, kKeys / kWaves>(va + wave * (kKeys / kWaves) * D * 2);
        __syncthreads();
        if (any) x.template tile<true, false>(p, w, sc, k0, ka, va);
    }
    // sums that are not finite: of values in the tiles seen whole, whose weights' pieces may be
    // 0 or negative.  Once more then, all tiles as those at the ends.
    const bool again = ta < tb && x.odd_sums();
    if (__builtin_expect(__syncthreads_or(odd || again), 0)) {
        if (__syncthreads_or(again)) {
            x.clear();
            ta = tb = 0;
            for (int k0 = w.lo; k0 < w.hi; k0 += kKeys) {
                __syncthreads();
                load_tile<D, true>(p, w, k0, tile_page(p, w, k0), ka, va);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                clear_odd<D, BF, kKeys / kWaves>(va + wave * (kKeys / kWaves) * D * 2);
                __syncthreads();
                if (any) x.template tile<true, false>(p, w, sc, k0, ka, va);
            }
        }
        for (int i = 0; i < tiles - (tb - ta); ++i) {
            const int k0 = w.lo + (i < ta ? i : i + tb - ta) * kKeys;
            __syncthreads();
            load_tile<D, true>(p, w, k0, tile_page(p, w, k0), ka, va);
            tile_barrier();
            if (any) x.add_odd(p, w, k0, va);
        }
    }

    x.l = sum_row<kRows>(x.l);
    if (!live) return;
    if (p.splits > 1) {
        const long long at = ((long long)token * p.q.heads + qh) * p.splits + blockIdx.y;
        if (h == 0) p.stat[at] = make_float2(x.m * sc, x.l);
        if (x.l == 0) return;
        float *o = p.part + at * D;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *(f32x4 *)(o + 32 * t + 8 * j + 4 * h) =
                    f32x4{x.o[t][4 * j], x.o[t][4 * j + 1], x.o[t][4 * j + 2], x.o[t][4 * j + 3]};
        return;
    }
    const float inv = x.l == 0 ? 0.0f : 1.0f / x.l;
    const long long to = (long long)token * p.out.token_stride + (long long)qh * p.out.head_stride;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 v = {x.o[t][4 * j], x.o[t][4 * j + 1], x.o[t][4 * j + 2], x.o[t][4 * j + 3]};
            v = x.l == 0 ? f32x4{0, 0, 0, 0} : v * inv;
            const long long at = to + 32 * t + 8 * j + 4 * h;
            if (p.out.type == M27Q_TYPE_F32) *(f32x4 *)((float *)p.out.ptr + at) = v;
            else *(typename R::T4 *)((T *)p.out.ptr + at) = __builtin_convertvector(v, typename R::T4);
        }
}

// Few rows (up to 32 of a sequence and cache head): the cache's bytes bound it.  The waves
// of a workgroup take tiles in turn, each for itself with K and V tiles of its own: K of
// its next tile is on its way from the moment its scores are there, V from when its values
// are added, and nothing waits for another wave.  At the end the four sums are joined.
// 32 sequences of up to 16381 keys, 4 cache heads of 256, F16: 1.58 GB in 287 us, 5.5 TB/s (a
// plain read of as much runs at 7.1); 2 of up to 32768 keys and 5 rows each, 253 MB in 54 us and
// 6 of joining, 4.2 TB/s (a plain read: 6.8): a wave has some 9 tiles between its start and the
// join.  One token over 1021 keys: a tile a wave, and a chain of 16000 cycles (lengths 3500, page
// and loads 2700, their arrival 2500, products and weights 2800, the waves' join 4300), then 3 us
// of the parts' join.
template <int D, bool BF, int NP, int RW>
__global__ __launch_bounds__(kWaves * 64, D == 256 ? 1 : 2) void k_attn_few(const AttnParams p) {
    typedef Rows<D, BF, NP, RW> R;
    typedef typename R::T T;
    constexpr int TB = kKeys * D * 2;  // bytes of a tile
    __shared__ __attribute__((aligned(1024))) char kts[kWaves * TB], vts[kWaves * TB];
    __shared__ float ms[kWaves][RW], ls[kWaves][RW];
    const int group = (int)(p.q.heads / p.cache.heads);
    const int s = blockIdx.x / p.cache.heads;
    Work w;
    w.s = s;
    w.head = blockIdx.x - s * p.cache.heads;
    const SeqRows sr = seq_rows(p.seqs.start, s, (int)p.seqs.tokens, (int)p.seqs.max_q);
    int len = p.seqs.kv_len[s];
    asm("" : "+s"(len));  // asked for with the rows, not behind the branch
    w.rows = sr.count * group;
    if (w.rows == 0) return;
    len = max(len, 0);
    const int first = len - (sr.end - sr.first), last = first + sr.count - 1;
    set_keys(p, w, len, first, last);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const bool live = (lane & (RW - 1)) < w.rows;
    const int row = min(lane & (RW - 1), w.rows - 1), at = row / group;
    const int token = sr.first + at, qh = w.head * group + row - at * group;
    const unsigned long long part = (unsigned long long)((uint32_t)token * p.q.heads + qh) * (uint32_t)p.splits + blockIdx.y;
    // loads end in order: what is needed first is asked for first
    typename R::Raw q;
    R::load_q(p, token, qh, q);
    const bool gaps = has_gaps(p, w);
    LDS_AS char *const kt = (LDS_AS char *)kts + wave * TB, *const vt = (LDS_AS char *)vts + wave * TB;
    const int32_t *table = p.seqs.table + (long long)s * p.seqs.table_stride;
    const int shift = __builtin_ctz(p.cache.page_size);
    // the pages of a tile's two halves
    auto page = [&](int k0, int half) {
        int at = min(k0 + 16 * half, w.hi - 1) >> shift;
        asm("" : "+v"(at));
        return table[at];
    };
    constexpr int RPI = 512 / D, CPR = D / 8;
    const int r0 = lane / CPR, pc = lane % CPR;
    const uint32_t ko = r0 * D * 2 + k_chunk<D>(r0, pc) * 16, vo = r0 * D * 2 + v_chunk<D>(r0, pc) * 16;
    // K (or V) of the tile at k0.  `checked`: of keys past `hi` or on a page that is not one,
    // another row of the cache is read (their weights are 0); otherwise all 16 rows of each half
    // are there, a page that is none is read as the first, and what it gives is not used.
    auto load = [&](const void *from, LDS_AS char *to, bool keys, int k0, const int (&pages)[2], bool checked) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int id = __builtin_amdgcn_readfirstlane(pages[half]), key = k0 + 16 * half;
            const bool ok = (uint32_t)id < p.cache.pages && (!checked || key < w.hi);
            const int rows = checked ? (ok ? min(w.hi - key, 16) : 1) : 16;
            const long long at = ((long long)(ok ? id : 0) * p.cache.page_stride +
                                  ((long long)w.head * p.cache.page_size + (key & (int)(p.cache.page_size - 1))) * D) * 2;
            const __amdgpu_buffer_rsrc_t rs = buf_rsrc((const char *)from + at, rows * D * 2);
#pragma unroll
            for (int i = 0; i < 16 / RPI; ++i) {
                LDS_AS char *d = to + (16 * half + i * RPI) * D * 2;
                const uint32_t o = keys ? ko ^ (k_chunk<D>(i * RPI, 0) * 16) : vo ^ (v_chunk<D>(i * RPI, 0) * 16);
                const uint32_t back = checked ? max(i * RPI + r0 - (rows - 1), 0) * D * 2 : 0;
                const uint32_t oo = i * 1024 + o - back;
                if (checked) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LDS_AS void *)d, 16, oo, 0, 0, 0);
                else __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LDS_AS void *)d, 16, o, i * 1024, 0, 0);
            }
        }
    };

    // tiles [ta, tb): seen whole by every row (if no page is missing, which is found out
    // while the first of them is on its way)
    const int tiles = (w.hi - w.lo + kKeys - 1) / kKeys;
    int tb = max(0, min(first + 1, w.hi) - w.lo) / kKeys;
    int ta = p.window ? min(tb, (max(0, first_key(p, last) - w.lo) + kKeys - 1) / kKeys) : 0;
    int t = ta + ((wave - ta) & (kWaves - 1));  // this wave's first
    int ids[2];
    if (t < tb) {
        ids[0] = page(w.lo + t * kKeys, 0);
        ids[1] = page(w.lo + t * kKeys, 1);
        load(p.cache.k, kt, true, w.lo + t * kKeys, ids, false);
        load(p.cache.v, vt, false, w.lo + t * kKeys, ids, false);
    }
    // a wave that has none of them asks for its first one of the others
    int there = -1;
    if (t >= tb) {
        for (there = wave; there >= ta && there < tb;) there += kWaves;
        if (there < tiles) {
            ids[0] = page(w.lo + there * kKeys, 0);
            ids[1] = page(w.lo + there * kKeys, 1);
            load(p.cache.k, kt, true, w.lo + there * kKeys, ids, true);
            load(p.cache.v, vt, false, w.lo + there * kKeys, ids, true);
        }
    }
    R x;
    x.place = live ? first + at : -1;
    x.clear();
    x.set_q(p, q, live);
    const float sc = fmaxf(fabsf(p.scale) * kLog2e, 1e-37f);
    w.gaps = __syncthreads_or(gaps);
    if (w.gaps) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        ta = tb = 0;
    }
    typename R::T8 pcs[R::NV][NP];
    float sco[R::NS];
    for (; t < tb; t += kWaves) {
        const int k0 = w.lo + t * kKeys, k1 = k0 + kWaves * kKeys;
        ids[0] = page(k1, 0);
        ids[1] = page(k1, 1);
        // K is there when no more than V's loads are on their way
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(32 / RPI) : "memory");
        x.template scores<true>(kt, sco);
        x.template weights<false>(p, w, sc, sco, k0, pcs);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (t + kWaves < tb) load(p.cache.k, kt, true, k1, ids, false);
        x.template values<true>(vt, pcs);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V has been read
        if (t + kWaves < tb) load(p.cache.v, vt, false, k1, ids, false);
    }
    // the others, which begin where none of those is
    const auto other = [&](int t) { return t >= ta && t < tb ? t + ((tb - t + kWaves - 1) & ~(kWaves - 1)) : t; };
    bool odd = false;
    for (int t = other(wave); t < tiles; t = other(t + kWaves)) {
        const int k0 = w.lo + t * kKeys;
        if (t != there) {
            ids[0] = page(k0, 0);
            ids[1] = page(k0, 1);
            load(p.cache.k, kt, true, k0, ids, true);
            load(p.cache.v, vt, false, k0, ids, true);
        }
        there = -1;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        odd |= clear_odd<D, BF, kKeys>(vt);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        x.template tile<true, true>(p, w, sc, k0, kt, vt);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    // as in k_attn: a value that is not finite in a tile seen whole
    if (__builtin_expect(ta < tb && __any(x.odd_sums()), 0)) {
        x.clear();
        ta = tb = 0;
        for (int t = wave; t < tiles; t += kWaves) {
            const int k0 = w.lo + t * kKeys, ids[2] = {page(k0, 0), page(k0, 1)};
            load(p.cache.k, kt, true, k0, ids, true);
            load(p.cache.v, vt, false, k0, ids, true);
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            odd |= clear_odd<D, BF, kKeys>(vt);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            x.template tile<true, false>(p, w, sc, k0, kt, vt);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
    if (__builtin_expect(__any(odd), 0))
        for (int t = other(wave); t < tiles; t = other(t + kWaves)) {
            const int k0 = w.lo + t * kKeys, ids[2] = {page(k0, 0), page(k0, 1)};
            load(p.cache.v, vt, false, k0, ids, true);
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            x.add_odd(p, w, k0, vt);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }

    // the waves' sums: to a common maximum, into LDS (a quadruple of values of the rows side by
    // side; the first TB bytes in the wave's K tile, what is more in its V tile), then added in order
    const int col = lane & (RW - 1);
    x.l = sum_row<RW>(x.l);
    if (lane < RW) {
        ms[wave][col] = x.m;
        ls[wave][col] = x.l;
    }
    __syncthreads();
    float m = ms[0][col];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) m = fmaxf(m, ms[i][col]);
    constexpr int HALF = TB / (RW * 16);  // quadruples of a tile's room
    if (x.l != 0) {
        const float f = join_factor((x.m - m) * sc);
#pragma unroll
        for (int t = 0; t < D / RW; ++t)
#pragma unroll
            for (int j = 0; j < R::NA / 4; ++j) {
                const int quad = R::value_at(t, 4 * j) / 4;
                f32x4 v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = x.o[t][4 * j + i] * f;
                *(LDS_AS f32x4 *)((RW * t < 4 * HALF ? kt : vt - TB) + (quad * RW + col) * 16) = v;
            }
    }
    __syncthreads();
    float fs[kWaves], l = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        fs[i] = ls[i][col];
        const float e = ms[i][col] == -__builtin_inff() ? 0.0f : join_factor((ms[i][col] - m) * sc);
        l += ls[i][col] * e;
    }
    if (!live) return;
    constexpr int Q = D / 4 * RW / (kWaves * 64);  // quadruples of a thread
    f32x4 y[Q][kWaves], o[Q];
#pragma unroll
    for (int u = 0; u < Q; ++u)  // all reads at once: what a wave without keys left is read and dropped
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const int quad = threadIdx.x / RW + u * (kWaves * 64 / RW);
            y[u][i] = *(const LDS_AS f32x4 *)((LDS_AS char *)(quad < HALF ? kts : vts - TB) + i * TB + (quad * RW + col) * 16);
        }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < Q; ++u) {
        o[u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kWaves; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[u][j] += fs[i] != 0 ? y[u][i][j] : 0.0f;
    }
    if (p.splits > 1) {
        if (threadIdx.x < RW) p.stat[part] = make_float2(m * sc, l);
        if (l == 0) return;
#pragma unroll
        for (int u = 0; u < Q; ++u)
            *(f32x4 *)(p.part + part * D + 4 * (threadIdx.x / RW + u * (kWaves * 64 / RW))) = o[u];
        return;
    }
    const long long to = (long long)token * p.out.token_stride + (long long)qh * p.out.head_stride;
    const float inv = l == 0 ? 0.0f : 1.0f / l;
#pragma unroll
    for (int u = 0; u < Q; ++u) {
        const int quad = threadIdx.x / RW + u * (kWaves * 64 / RW);
        const f32x4 x = l == 0 ? f32x4{0, 0, 0, 0} : o[u] * inv;
        if (p.out.type == M27Q_TYPE_F32) *(f32x4 *)((float *)p.out.ptr + to + 4 * quad) = x;
        else *(typename R::T4 *)((T *)p.out.ptr + to + 4 * quad) = __builtin_convertvector(x, typename R::T4);
    }
}

// Joins the parts of each row, in order of the parts: a wave a row (two for D = 128, four
// for 64), each part's statistics in a lane (at most 64 parts), then the sums, several on
// their way at a time.
template <int D, bool BF>
__global__ __launch_bounds__(256) void k_attn_join(const AttnParams p) {
    constexpr int L = D / 4, RPW = 64 / L;
    const SeqRows sr = seq_rows(p.seqs.start, blockIdx.y, (int)p.seqs.tokens, (int)p.seqs.max_q);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first = (blockIdx.x * 4 + wave) * RPW, d = 4 * (lane % L), rows = sr.count * (int)p.q.heads;
    if (first >= rows) return;
    const long long base = (long long)sr.first * p.q.heads;
    const int mine = lane / L, row = first + mine;
    const bool live = row < rows;
    const float *from = p.part + (base + (live ? row : first)) * p.splits * D + d;
    constexpr int AT = 8;  // parts on their way at a time, the first before the statistics are there
    f32x4 v[AT];
#pragma unroll
    for (int i = 0; i < AT; ++i) v[i] = *(const f32x4 *)(from + (long long)min(i, p.splits - 1) * D);
    float f[RPW], inv[RPW];  // lane i: part i's factor of each of the wave's rows
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
        float2 st = p.stat[(base + min(first + r, rows - 1)) * p.splits + min(lane, p.splits - 1)];
        if (lane >= p.splits) st.y = 0;
        float m = st.y != 0 ? st.x : -__builtin_inff();
#pragma unroll
        for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        f[r] = st.y != 0 ? join_factor(st.x - m) : 0.0f;
        float l = st.y * f[r];
        f[r] = st.y != 0 ? f[r] : -1.0f;  // no key: its sums were not written
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
        inv[r] = l == 0 ? 0.0f : 1.0f / l;
    }
    f32x4 o = {};
    for (int i0 = 0; i0 < p.splits; i0 += AT) {
        f32x4 u[AT];
#pragma unroll
        for (int i = 0; i < AT; ++i) u[i] = v[i];
        if (i0 + AT < p.splits) {
#pragma unroll
            for (int i = 0; i < AT; ++i) v[i] = *(const f32x4 *)(from + (long long)min(i0 + AT + i, p.splits - 1) * D);
        }
#pragma unroll
        for (int i = 0; i < AT; ++i) {
            float w = __shfl(f[0], (i0 + i) & 63);
#pragma unroll
            for (int r = 1; r < RPW; ++r) {
                const float y = __shfl(f[r], (i0 + i) & 63);
                w = mine == r ? y : w;
            }
            o = i0 + i >= p.splits || w == -1.0f ? o : o + u[i] * w;
        }
    }
    if (!live) return;
    float scale = inv[0];
#pragma unroll
    for (int r = 1; r < RPW; ++r) scale = mine == r ? inv[r] : scale;
    o = scale == 0 ? f32x4{0, 0, 0, 0} : o * scale;
    const int token = sr.first + row / (int)p.q.heads, qh = row % (int)p.q.heads;
    const long long to = (long long)token * p.out.token_stride + (long long)qh * p.out.head_stride + d;
    if (p.out.type == M27Q_TYPE_F32) *(f32x4 *)((float *)p.out.ptr + to) = o;
    else if constexpr (BF) *(bf16x4 *)((__bf16 *)p.out.ptr + to) = __builtin_convertvector(o, bf16x4);
    else *(f16x4 *)((_Float16 *)p.out.ptr + to) = __builtin_convertvector(o, f16x4);
}

}  // namespace

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
