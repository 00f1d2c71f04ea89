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
};

// The maximum of a value over the wave's two halves (lane l and l ^ 32).
__device__ __forceinline__ float max_halves(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
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

// Tiles of K and V in LDS: kKeys rows of D values, 16-byte chunks exchanged
// within a row so that neither kind of read meets bank conflicts: K's chunk c
// of row r lies at c ^ (r & 7) (a read takes one chunk column of 32 rows), V's
// 32-byte unit u at u ^ (r & 7) (D = 64: r & 3; a transposing read takes one
// unit of 4 rows per 16 lanes).
template <int D>
__device__ __forceinline__ int k_chunk(int row, int c) {
    return c ^ (row & 7);
}
template <int D>
__device__ __forceinline__ int v_chunk(int row, int c) {
    return c ^ ((row & (D >= 128 ? 7 : 3)) << 1);
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
    const int r0 = lane / CPR, pc = lane % CPR;
    const uint32_t ko = r0 * D * 2 + k_chunk<D>(r0, pc) * 16, vo = r0 * D * 2 + v_chunk<D>(r0, pc) * 16;
#pragma unroll
    for (int i = 0; i < RPW / RPI; ++i) {  // row i RPI + r0: its chunks are r0's with i RPI exchanged as well
        LDS_AS char *kd = kt + (wave * RPW + i * RPI) * D * 2, *vd = vt + (wave * RPW + i * RPI) * D * 2;
        if (!CHECKED || i * RPI + r0 < rows) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(kg, (LDS_AS void *)kd, 16, ko ^ (i * RPI * 16), i * 1024, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(vg, (LDS_AS void *)vd, 16, vo ^ (i * RPI * 32), i * 1024, 0, 0);
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

// Puts zeros for the values of V that are not finite, in the rows that this
// wave brought into the tile: some row of queries may not see their key, and
// its weight of 0 would make NaN of them.  Returns whether there were any.
template <int D, bool BF>
__device__ __forceinline__ bool clear_odd(LDS_AS char *vt) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
    bool odd = false;
    LDS_AS char *at = vt + (threadIdx.x >> 6) * (kKeys / kWaves) * D * 2 + (threadIdx.x & 63) * 16;
#pragma unroll
    for (int i = 0; i < kKeys / kWaves * D / 512; ++i) {
        u4 v = *(LDS_AS u4 *)(at + i * 1024);
        bool here = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool a = (v[j] & E) == E, b = ((v[j] >> 16) & E) == E;
            v[j] &= (a ? 0xffff0000u : ~0u) & (b ? 0xffffu : ~0u);
            here |= a || b;
        }
        if (here) *(LDS_AS u4 *)(at + i * 1024) = v;
        odd |= here;
    }
    return odd;
}

// One wave's rows: the statistics and sums of a softmax in one pass.
template <int D, bool BF, int NP>
struct Rows {
    typedef Num<BF> N;
    typedef typename N::t T;
    typedef typename N::t4 T4;
    typedef typename N::t8 T8;
    T8 q[D / 16];
    f32x16 o[D / 32];
    float m, l;      // maximum of the scores (before scale) that weights are taken from; this half's sum of weights
    int place;       // of this lane's row (-1: none)

    // The tile in LDS.  MASK: some of its keys may be hidden from some row, or missing.
    template <bool MASK>
    __device__ __forceinline__ void tile(const AttnParams &p, const Work &w, float sc, int k0, const LDS_AS char *kt,
                                         const LDS_AS char *vt) {
        const int lane = threadIdx.x & 63, h = lane >> 5, r = lane & 31;
        f32x16 s = {};
        // K: row r, chunks 2 i + h
        const LDS_AS char *kr = kt + r * D * 2;
        const int y = (r & 7) ^ h;  // k_chunk(r, 2 i + h) = (y ^ (2 i & 6)) + (2 i & ~7): four addresses, the rest offsets
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const T8 a = *(const LDS_AS T8 *)(kr + (y ^ (2 * i & 6)) * 16 + (2 * i & ~7) * 16);
            s = N::mma(a, q[i], s);
        }
        if constexpr (MASK) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = sees(p, w, k0 + 8 * (i / 4) + 4 * h + i % 4) ? s[i] : -__builtin_inff();
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        top = max_halves(top);
        // The maximum that weights are taken from follows the rows' own only
        // when one has grown by 2^8: weights reach 2^(6 + 8) then, and lie 2^6
        // above the type's small values otherwise.  (m = -inf: no key yet.)
        if (__any(!((top - m) * sc <= 8.0f) && top != m)) {
            const float next = fmaxf(m, top);
            const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - next) * sc);
            m = next;
            l *= f;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] *= f;
        }
        const float off = 6.0f - (m == -__builtin_inff() ? 0.0f : m) * sc;
        float part = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sc, off));
            part += s[i];
        }
        l += part;
        // P as NP pieces of the cache's type, each what the ones before left over
        T8 pc[2][NP];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f32x8 x = i ? __builtin_shufflevector(s, s, 8, 9, 10, 11, 12, 13, 14, 15)
                        : __builtin_shufflevector(s, s, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                pc[i][j] = __builtin_convertvector(x, T8);
                if (j + 1 < NP) x -= __builtin_convertvector(pc[i][j], f32x8);
            }
        }
        // V^T: lane (d = 32 t + lane % 32, half h) takes keys 16 i + 8 e + 4 h + 0 .. 3
        const int x = 4 * h + ((lane & 15) >> 2);  // key mod 8 of the row this lane reads
        const LDS_AS char *vr = vt + x * D * 2 + (lane & 3) * 8;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const T8 v = values(vr + 16 * i * D * 2, x, t);
#pragma unroll
                for (int j = 0; j < NP; ++j) o[t] = N::mma(v, pc[i][j], o[t]);
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

    // This lane's eight values of V^T in the 16 keys at vr: d = 32 t + lane % 32.
    static __device__ __forceinline__ T8 values(const LDS_AS char *vr, int x, int t) {
        constexpr int M = D >= 128 ? 7 : 3;
        const int y = (x & M) ^ ((threadIdx.x >> 4) & 1);  // its 32-byte unit, exchanged as in v_chunk
        const int c = ((2 * t & (M - 1)) ^ y) * 32 + (2 * t & ~M) * 32;
        return __builtin_shufflevector(tr4(vr + c), tr4(vr + c + 8 * D * 2), 0, 1, 2, 3, 4, 5, 6, 7);
    }

    static __device__ __forceinline__ T4 tr4(const LDS_AS char *at) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(T4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s4 *)at));
    }

    // O += the values of V that are not finite, where they are seen: the whole of
    // their effect, as a weight is positive.
    __device__ __forceinline__ void add_odd(const AttnParams &p, const Work &w, int k0, const LDS_AS char *vt) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        for (int key = 0; key < kKeys; ++key) {
            const LDS_AS char *vk = vt + key * D * 2;
            bool odd = false;
            for (int i = lane; i < D; i += 64) odd |= !__builtin_isfinite((float)*(const LDS_AS T *)(vk + i * 2));
            if (!__any(odd)) continue;
            const bool ok = sees(p, w, k0 + key);
#pragma unroll
            for (int t = 0; t < D / 32; ++t) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int d = 32 * t + 8 * (j / 4) + 4 * h + j % 4;
                    const float v = (float)*(const LDS_AS T *)(vk + (v_chunk<D>(key, d / 8) * 8 + d % 8) * 2);
                    o[t][j] += ok && !__builtin_isfinite(v) ? v : 0.0f;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
};

template <int D, bool BF, int NP>
__global__ __launch_bounds__(kWaves * 64, 2) void k_attn(const AttnParams p) {
    typedef Rows<D, BF, NP> R;
    typedef typename R::T T;
    typedef typename R::T8 T8;
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
    const int kv = min(max(p.seqs.kv_len[s], 0), (int)p.seqs.max_kv);
    const int place0 = p.seqs.kv_len[s] - (sr.end - sr.first);  // of the sequence's first row
    const int first = place0 + w.row0 / group;
    const int last = place0 + (min(w.row0 + kWaves * kRows, w.rows) - 1) / group;
    int lo = p.window ? max(0, first - p.window + 1) & ~(kKeys - 1) : 0;  // tiles lie whole within pages or the other way round
    int hi = min(kv, last + 1);
    if (p.splits > 1) {
        const int tiles = max(0, hi - lo + kKeys - 1) / kKeys;
        const int each = (tiles + p.splits - 1) / p.splits;
        lo += (int)blockIdx.y * each * kKeys;
        hi = min(hi, lo + each * kKeys);
    }
    w.lo = lo;
    w.hi = hi;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    const int wrow = w.row0 + wave * kRows;  // this wave's first row
    const int row = wrow + (lane & 31);
    const bool live = row < w.rows;
    const int token = sr.first + row / group, qh = w.head * group + row % group;
    R x;
    x.place = live ? place0 + row / group : -1;
    x.m = -__builtin_inff();
    x.l = 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) x.o[i] = f32x16{};
    {
        const T *q = (const T *)p.q.ptr + (long long)token * p.q.token_stride + (long long)qh * p.q.head_stride;
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        // a negative scale goes into q, exactly: scores are then compared before scaling
        const uint32_t flip = p.scale < 0 ? 0x80008000u : 0;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            u4 v = {0, 0, 0, 0};
            if (live) v = *(const u4 *)(q + 16 * i + 8 * h);
            x.q[i] = __builtin_bit_cast(T8, v ^ flip);
        }
    }
    // (a scale of 0 would make NaN of a masked score's -inf)
    const float sc = fmaxf(fabsf(p.scale) * kLog2e, 1e-37f);

    // every page of the keys, looked at once: the tiles below trust them
    w.gaps = false;
    {
        const int shift = __builtin_ctz(p.cache.page_size);
        const int32_t *table = p.seqs.table + (long long)s * p.seqs.table_stride;
        bool bad = false;
        if (w.lo < w.hi)
            for (int i = (w.lo >> shift) + (int)threadIdx.x; i <= (w.hi - 1) >> shift; i += kWaves * 64)
                bad |= (uint32_t)table[i] >= p.cache.pages;
        w.gaps = __syncthreads_or(bad);
    }
    // tiles [ta, tb) are seen whole by every row of the workgroup: the next one is
    // on its way while one is worked on; the others, at the ends, go one by one
    const int tiles = max(0, w.hi - w.lo + kKeys - 1) / kKeys;
    int ta = 0, tb = 0;
    if (!w.gaps) {
        tb = max(0, min(first + 1, w.hi) - w.lo) / kKeys;
        ta = p.window ? min(tb, (max(0, last - p.window + 1 - w.lo) + kKeys - 1) / kKeys) : 0;
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
        if (any) x.template tile<false>(p, w, sc, w.lo + t * kKeys, ka, va);
        if (t + 1 >= tb) break;
        tile_barrier();
        if (t + 2 < tb) {
            load_tile<D, false>(p, w, w.lo + (t + 2) * kKeys, id, ka, va);
            id = tile_page(p, w, w.lo + (t + 3) * kKeys);
        }
        if (any) x.template tile<false>(p, w, sc, w.lo + (t + 1) * kKeys, kb, vb);
    }
    bool odd = false;
    for (int i = 0; i < tiles - (tb - ta); ++i) {
        const int k0 = w.lo + (i < ta ? i : i + tb - ta) * kKeys;
        __syncthreads();
        load_tile<D, true>(p, w, k0, tile_page(p, w, k0), ka, va);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        odd |= clear_odd<D, BF>(va);
        __syncthreads();
        if (any) x.template tile<true>(p, w, sc, k0, ka, va);
    }
    if (__builtin_expect(__syncthreads_or(odd), 0))
        for (int i = 0; i < tiles - (tb - ta); ++i) {
            const int k0 = w.lo + (i < ta ? i : i + tb - ta) * kKeys;
            __syncthreads();
            load_tile<D, true>(p, w, k0, tile_page(p, w, k0), ka, va);
            tile_barrier();
            if (any) x.add_odd(p, w, k0, va);
        }

    x.l = sum_halves(x.l);
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

// Joins the parts of each row, in order of the parts: D / 4 lanes a row.
template <int D, bool BF>
__global__ __launch_bounds__(256) void k_attn_join(const AttnParams p) {
    constexpr int L = D / 4, RPB = 256 / L;
    const SeqRows sr = seq_rows(p.seqs.start, blockIdx.y, (int)p.seqs.tokens, (int)p.seqs.max_q);
    const int row = blockIdx.x * RPB + threadIdx.x / L, d = 4 * (threadIdx.x % L);
    if (row >= sr.count * (int)p.q.heads) return;
    const int token = sr.first + row / (int)p.q.heads, qh = row % (int)p.q.heads;
    const long long at = ((long long)token * p.q.heads + qh) * p.splits;
    float m = -__builtin_inff();
    for (int i = 0; i < p.splits; ++i) {
        const float2 st = p.stat[at + i];
        if (st.y != 0) m = fmaxf(m, st.x);
    }
    float l = 0;
    f32x4 o = {};
    for (int i = 0; i < p.splits; ++i) {
        const float2 st = p.stat[at + i];
        if (st.y == 0) continue;  // no key: its sums were not written
        const float f = __builtin_amdgcn_exp2f(st.x - m);
        l += st.y * f;
        o += *(const f32x4 *)(p.part + (at + i) * D + d) * f;
    }
    o = l == 0 ? f32x4{0, 0, 0, 0} : o * (1.0f / l);
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
    const dim3 grid((unsigned)attn_groups(p.seqs, p.q.heads, p.cache), p.splits);
    constexpr int NP = BF ? 3 : 2;
    if (p.out.type == M27Q_TYPE_F32) hipLaunchKernelGGL((k_attn<D, BF, NP>), grid, dim3(kWaves * 64), 0, s, p);
    else hipLaunchKernelGGL((k_attn<D, BF, 1>), grid, dim3(kWaves * 64), 0, s, p);
    if (p.splits > 1) {
        constexpr int RPB = 256 / (D / 4);
        const dim3 g2((p.seqs.max_q * p.q.heads + RPB - 1) / RPB, p.seqs.n);
        hipLaunchKernelGGL((k_attn_join<D, BF>), g2, dim3(256), 0, s, p);
    }
    return hipGetLastError();
}

}  // namespace

// Parts of the keys: enough workgroups for two on each CU, parts of 256 keys at least.
AttnPlan attn_plan(const m27q_seqs &seqs, uint32_t q_heads, const m27q_cache &cache, int cus) {
    const long long wgs = attn_groups(seqs, q_heads, cache);
    const long long want = (2ll * cus + wgs - 1) / wgs, most = (seqs.max_kv + 255) / 256;
    long long splits = want < most ? want : most;
    if (splits > kMaxSplits) splits = kMaxSplits;
    return {0, splits < 1 ? 1 : (int)splits};
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
