// The tiles of matrix products C(m, n) = sum_k A(m, k) B(n, k): operands to
// LDS, the matrix instructions, and the fp32 sums that an epilogue takes.
#pragma once
#include "fl_abi.h"
#include "fl_common.h"
#include <type_traits>

namespace fl {
namespace {

constexpr int LN_NT = 256;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Planes {
    static constexpr int N = 1;
};
template <>
struct Planes<float> {
    static constexpr int N = 3;
};

template <typename T>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma<_Float16>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

// N consecutive values at an element-aligned address, as few wide loads.
template <typename T, int N>
struct Vec {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T *p) {
    Vec<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T *p, const Vec<T, N> &r) {
    __builtin_memcpy(p, &r, sizeof(r));
}

// The first m of them.
template <typename T, int N>
__device__ __forceinline__ void store_some(T *p, const Vec<T, N> &r, int m) {
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < m) p[e] = r.v[e];
}

// Up to four values as floats, the others 0.
template <typename T>
__device__ __forceinline__ void load_some(const T *p, int have, float (&out)[4]) {
    if (have == 4) {
        const Vec<T, 4> r = load_vec<T, 4>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = (float)r.v[e];
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = e < have ? (float)p[e] : 0.0f;
}

// The upper halves of two words, lo's first.
__device__ __forceinline__ uint32_t upper_halves(uint32_t lo, uint32_t hi) {
    return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}

// Eight consecutive k of one row as the chunk of every plane.
template <typename T>
__device__ __forceinline__ void chunk_planes(const T (&v)[8], u32x4 (&out)[Planes<T>::N]) {
    static_assert(sizeof(T) == 2, "16-bit operands");
    union {
        T t[8];
        u32x4 u;
    } c;
#pragma unroll
    for (int j = 0; j < 8; ++j) c.t[j] = v[j];
    out[0] = c.u;
}
template <>
__device__ __forceinline__ void chunk_planes<float>(const float (&v)[8], u32x4 (&out)[3]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t x0 = __float_as_uint(v[2 * j]), x1 = __float_as_uint(v[2 * j + 1]);
        const float r0 = v[2 * j] - __uint_as_float(x0 & 0xffff0000u);
        const float r1 = v[2 * j + 1] - __uint_as_float(x1 & 0xffff0000u);
        const uint32_t m = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{r0, r1}), bf16x2));
        out[0][j] = upper_halves(x0, x1);
        out[1][j] = m;
        out[2][j] = upper_halves(__float_as_uint(r0 - __uint_as_float(m << 16)),
                                 __float_as_uint(r1 - __uint_as_float(m & 0xffff0000u)));
    }
}

// LDS element offset of chunk c of row r in a tile of BK values a row.  A
// 128-bit LDS read takes 16 lanes a cycle, lanes 0-3, 12-15, 20-23, 24-27 of
// each half wave together and then the rest, so an MFMA operand read has 8
// rows at chunk c and 8 others at chunk c ^ 1 in one cycle; the permutation of
// a row's chunks keeps those 16 in different banks, and 16 consecutive rows at
// one chunk (the stores of k-strided operands) too.  (Permuted by r ^ (r >> 3)
// a third of the LDS cycles were conflicts.)
template <int BK>
__device__ __forceinline__ int lds_at(int r, int c) {
    const int f = BK == 32 ? (0x78 >> (2 * ((r >> 2) & 3))) & 3 : (r >> 1) & 7;
    return r * BK + ((c ^ f) << 3);
}

// Operand rows with k contiguous: a pointer a row, 8 k a load.  The part of K
// that is no whole tile is taken first (fetch_tail, guarded), the whole tiles
// without guards.
template <typename T, int BR, int BK>
struct ContigTile {
    static constexpr int CPR = BK / 8, RP = LN_NT / CPR, PASSES = BR / RP;
    static_assert(BR % RP == 0, "whole passes");
    const T *row[PASSES];
    Vec<T, 8> raw[PASSES];

    template <typename F>
    __device__ __forceinline__ void init(F &&row_ptr) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) row[i] = row_ptr(threadIdx.x / CPR + i * RP) + (threadIdx.x % CPR) * 8;
    }
    // The first `left` < BK values of every row.
    __device__ __forceinline__ void fetch_tail(int64_t left) {
        const int have = (int)left - (int)(threadIdx.x % CPR) * 8;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) raw[i].v[j] = j < have ? row[i][j] : (T)0.0f;
            row[i] += left;
        }
    }
    __device__ __forceinline__ void fetch() {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            raw[i] = load_vec<T, 8>(row[i]);
            row[i] += BK;
        }
    }
    __device__ __forceinline__ void stage(uint16_t *lds, int plane) const {
        const int c = threadIdx.x % CPR;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            u32x4 ch[Planes<T>::N];
            chunk_planes<T>(raw[i].v, ch);
#pragma unroll
            for (int p = 0; p < Planes<T>::N; ++p)
                *reinterpret_cast<u32x4 *>(lds + p * plane + lds_at<BK>(threadIdx.x / CPR + i * RP, c)) = ch[p];
        }
    }
};

// Operand rows with k strided: element (k, r) at base + row_of(k) * ld + r.
// Lanes take consecutive r, a word's worth of them each, a thread 8 k.  Lanes
// behind the last of the R columns read it again: their products are not
// stored.  (Two columns a word need R >= 2; at an odd end the pair before it
// is read and shifted.)
template <typename T, int BR, int BK>
struct StridedTile {
    static constexpr int V = BR >= 128 ? 4 / (int)sizeof(T) : 1;
    static constexpr int LR = BR / V < FL_WAVE ? BR / V : FL_WAVE;  // lanes along r
    static constexpr int RPASS = BR / (LR * V), SLOTS = LN_NT / LR, CPR = BK / 8, CP = CPR / SLOTS;
    static_assert(CP >= 1 && CPR % SLOTS == 0 && BR % (LR * V) == 0, "whole passes");
    const T *col[RPASS];
    const int32_t *order;
    int64_t ld, k;  // k: first place of the thread's slot
    uint32_t raw[CP][RPASS][8];
    int slot, shift[RPASS];

    __device__ __forceinline__ void init(const T *base, int64_t stride, int64_t R, const int32_t *ord) {
        ld = stride;
        order = ord;
        k = 0;
        slot = threadIdx.x / LR;
        if (LR == FL_WAVE) slot = __builtin_amdgcn_readfirstlane(slot);
#pragma unroll
        for (int i = 0; i < RPASS; ++i) {
            const int64_t r = (threadIdx.x % LR) * V + i * LR * V;
            col[i] = base + (r < R - V ? r : R - V);
            shift[i] = V == 2 && r == R - 1 ? 16 : 0;
        }
    }
    __device__ __forceinline__ uint32_t load(const T *p) const {
        if constexpr (sizeof(T) == 2 && V == 1) return __builtin_bit_cast(uint16_t, *p);
        uint32_t w;
        __builtin_memcpy(&w, p, 4);
        return w;
    }
    __device__ __forceinline__ int64_t at(int64_t place) const { return (order ? (int64_t)order[place] : place) * ld; }
    __device__ __forceinline__ void fetch_tail(int64_t left) {
#pragma unroll
        for (int cp = 0; cp < CP; ++cp)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t q = (slot + cp * SLOTS) * 8 + j;
                const int64_t o = at(q < left ? q : left - 1);
#pragma unroll
                for (int i = 0; i < RPASS; ++i) {
                    const uint32_t w = load(col[i] + o);
                    raw[cp][i][j] = q < left ? w : 0u;
                }
            }
        k = left;
    }
    __device__ __forceinline__ void fetch() {
#pragma unroll
        for (int cp = 0; cp < CP; ++cp)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t o = at(k + (slot + cp * SLOTS) * 8 + j);
#pragma unroll
                for (int i = 0; i < RPASS; ++i) raw[cp][i][j] = load(col[i] + o);
            }
        k += BK;
    }
    __device__ __forceinline__ void stage(uint16_t *lds, int plane) const {
#pragma unroll
        for (int cp = 0; cp < CP; ++cp)
#pragma unroll
            for (int i = 0; i < RPASS; ++i) {
                const uint32_t(&w)[8] = raw[cp][i];
                const int r = (threadIdx.x % LR) * V + i * LR * V, c = slot + cp * SLOTS;
                if constexpr (sizeof(T) == 4) {
                    float one[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) one[j] = __uint_as_float(w[j]);
                    u32x4 ch[3];
                    chunk_planes<float>(one, ch);
#pragma unroll
                    for (int p = 0; p < 3; ++p)
                        *reinterpret_cast<u32x4 *>(lds + p * plane + lds_at<BK>(r, c)) = ch[p];
                } else {
                    u32x4 lo, hi;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t w0 = w[2 * j] >> shift[i], w1 = w[2 * j + 1] >> shift[i];
                        lo[j] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
                        hi[j] = upper_halves(w0, w1);
                    }
                    *reinterpret_cast<u32x4 *>(lds + lds_at<BK>(r, c)) = lo;
                    if (V == 2) *reinterpret_cast<u32x4 *>(lds + lds_at<BK>(r + 1, c)) = hi;
                }
            }
    }
};

// A workgroup's product: waves WAVES_M x WAVES_N, each MT x NTL tiles of 16 x 16.
template <typename T, int BM, int BN, int BK>
struct Product {
    static constexpr int P = Planes<T>::N;
    static constexpr int WAVES_M = 2, WAVES_N = 2;
    static constexpr int MT = BM / WAVES_M / 16, NTL = BN / WAVES_N / 16;
    static constexpr int PLANE_A = BM * BK, PLANE_B = BN * BK;
    static constexpr int LDS_ELEMS = P * (PLANE_A + PLANE_B);
    f32x4 acc[MT][NTL];

    __device__ __forceinline__ int wave_m() const { return (fl_wave_id() / WAVES_N) * (BM / WAVES_M); }
    __device__ __forceinline__ int wave_n() const { return (fl_wave_id() % WAVES_N) * (BN / WAVES_N); }

    __device__ __forceinline__ void step(const uint16_t *la, const uint16_t *lb) {
        const int r = fl_lane() & 15, q = fl_lane() >> 4;
#pragma unroll
        for (int ks = 0; ks < BK / 32; ++ks) {
            u32x4 b[NTL][P];
#pragma unroll
            for (int j = 0; j < NTL; ++j)
#pragma unroll
                for (int p = 0; p < P; ++p)
                    b[j][p] = *reinterpret_cast<const u32x4 *>(
                        lb + p * PLANE_B + lds_at<BK>(wave_n() + j * 16 + r, ks * 4 + q));
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                u32x4 a[P];
#pragma unroll
                for (int p = 0; p < P; ++p)
                    a[p] = *reinterpret_cast<const u32x4 *>(
                        la + p * PLANE_A + lds_at<BK>(wave_m() + i * 16 + r, ks * 4 + q));
#pragma unroll
                for (int j = 0; j < NTL; ++j) {
                    if (P == 3) {  // smallest products first
                        acc[i][j] = mfma<T>(b[j][2], a[0], acc[i][j]);
                        acc[i][j] = mfma<T>(b[j][1], a[1], acc[i][j]);
                        acc[i][j] = mfma<T>(b[j][0], a[2], acc[i][j]);
                        acc[i][j] = mfma<T>(b[j][1], a[0], acc[i][j]);
                        acc[i][j] = mfma<T>(b[j][0], a[1], acc[i][j]);
                    }
                    acc[i][j] = mfma<T>(b[j][0], a[0], acc[i][j]);
                }
            }
        }
    }

    template <typename TA, typename TB>
    __device__ __forceinline__ void run(TA &ta, TB &tb, int64_t K, uint16_t *lds) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
        uint16_t *la = lds, *lb = lds + P * PLANE_A;
        if (K <= 0) return;
        const int64_t left = K % BK;
        if (left) {
            ta.fetch_tail(left);
            tb.fetch_tail(left);
        } else {
            ta.fetch();
            tb.fetch();
        }
        for (int64_t more = (K - 1) / BK;; --more) {
            ta.stage(la, PLANE_A);
            tb.stage(lb, PLANE_B);
            __syncthreads();
            if (more > 0) {
                ta.fetch();
                tb.fetch();
            }
            step(la, lb);
            if (more == 0) break;
            __syncthreads();
        }
    }
};

// The same products for large 16-bit operands at the matrix unit's pace.  512
// threads take BM x 256 outputs, 8 waves of BM/2 x 64; BK values of k a step.
// Operands go from memory to LDS without registers (global_load_lds, 16 bytes
// a lane), into one of STAGES buffers while others are multiplied, so that a
// load has STAGES - 1 steps to arrive.  The waves work in two halves, one wave
// of each on every SIMD, half a step apart: while one half reads its operands
// from LDS (and issues its share of the loads), the other multiplies; barriers
// keep them in turn.  (With all waves in step the matrix unit was busy 45% of
// the time.)  A wave's load fills 1 KB of LDS in lane order, so the permutation
// of the chunks that spreads the later reads over the banks is made on the
// memory side: a lane loads the chunk that belongs to its place.
// k-strided operands lie in LDS as they do in memory, rows of k, and are read
// transposed (ds_read_b64_tr_b16: of 16 lanes, lane s gives the address of
// row s/4, columns 4 (s%4)..+3, and lane i receives column i of the 4 rows).
// Needs 16-byte aligned rows of whole 8-value chunks.
constexpr int WD_NT = 512;
constexpr int WD_WAVES = WD_NT / FL_WAVE;
constexpr int WD_BN = 256;

// What lanes outside an operand load.
__device__ __align__(16) const uint32_t wd_zeros[4] = {0, 0, 0, 0};

typedef __attribute__((address_space(3))) void lds_ptr;
typedef __attribute__((address_space(1))) const void mem_ptr;

__device__ __forceinline__ void load_lds(const void *p, uint16_t *lds) {
    __builtin_amdgcn_global_load_lds((mem_ptr *)p, (lds_ptr *)lds, 16, 0, 0);
}

template <int BR, int BK>
struct WideContig {
    static constexpr int CPR = BK / 8, RPL = FL_WAVE / CPR;  // chunks of a row, rows of a load
    static constexpr int LOADS = BR / RPL / WD_WAVES;
    static constexpr int ELEMS = BR * BK;
    const uint16_t *p[LOADS];

    // The row and the chunk that this lane loads i-th.
    static __device__ __forceinline__ int row(int i) { return (fl_wave_id() * LOADS + i) * RPL + fl_lane() / CPR; }
    static __device__ __forceinline__ int chunk(int i) { return (lds_at<BK>(row(i), fl_lane() % CPR) % BK) / 8; }

    template <typename F>
    __device__ __forceinline__ void init(F &&row_ptr) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) p[i] = row_ptr(row(i)) + chunk(i) * 8;
    }
    // The next `count` values of k, BK if WHOLE.
    template <bool WHOLE>
    __device__ __forceinline__ void issue(uint16_t *lds, int count) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const void *q = WHOLE || chunk(i) * 8 < count ? (const void *)p[i] : (const void *)wd_zeros;
            load_lds(q, lds + (fl_wave_id() * LOADS + i) * 512);
            p[i] += count;
        }
    }
    // The operands of N 16-row tiles from row0 on.
    template <int N>
    __device__ __forceinline__ void read(const uint16_t *lds, int row0, u32x4 (&f)[BK / 32][N]) const {
#pragma unroll
        for (int ks = 0; ks < BK / 32; ++ks)
#pragma unroll
            for (int i = 0; i < N; ++i)
                f[ks][i] = *reinterpret_cast<const u32x4 *>(
                    lds + lds_at<BK>(row0 + i * 16 + (fl_lane() & 15), ks * 4 + (fl_lane() >> 4)));
    }
};

// A value that the compiler takes for new at this place, so that what is made of
// it is not kept in registers over a loop.
__device__ __forceinline__ int made_here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// fp32 values as three bfloat16 planes (chunk_planes): a row holds 32 values of the
// first, the same 32 of the second and of the third, and so on.
__device__ __forceinline__ int64_t plane_at(int64_t c) { return c / 32 * 96 + c % 32; }

// The same for rows of whole steps, from a base that all lanes have and with
// 32-bit offsets (half the registers): rows of less than 2^23 values.  P: planes of
// a value; a step is 64 k of one, 32 of three.  A plane's part of a step lies in LDS
// as a tile of its own.
template <int BR, int P>
struct StepsContig {
    static constexpr int BK = P == 1 ? 64 : 32;
    using At = WideContig<BR, BK>;
    static constexpr int LOADS = P * At::LOADS, ELEMS = P * At::ELEMS;
    static constexpr bool BLOCKING = false;
    const uint16_t *base;      // of the next step
    uint32_t at[At::LOADS];    // bytes

    // Row r of the tile is row row_at(r) from b on.
    template <typename F>
    __device__ __forceinline__ void init(const uint16_t *b, int64_t ld, F &&row_at) {
        const int lane = made_here(fl_lane());
        base = b;
#pragma unroll
        for (int i = 0; i < At::LOADS; ++i) {
            const int r = (fl_wave_id() * At::LOADS + i) * At::RPL + lane / At::CPR;
            at[i] = (uint32_t)row_at(r) * (uint32_t)(ld * 2) + lds_at<BK>(r, lane % At::CPR) % BK * 2;
        }
    }
    __device__ __forceinline__ void issue(uint16_t *lds, int i) {
        const int p = i / At::LOADS, j = i % At::LOADS;
        load_lds((const char *)base + p * (BK * 2) + at[j], lds + p * At::ELEMS + (fl_wave_id() * At::LOADS + j) * 512);
    }
    __device__ __forceinline__ void next() { base += P * BK; }
    // The operands of N 16-row tiles from row0 on: the step's first or second 32
    // values, or those of a plane.
    template <int KS, int N>
    __device__ __forceinline__ void read(const uint16_t *lds, int row0, u32x4 (&f)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row0 + i * 16 + (fl_lane() & 15), c = fl_lane() >> 4;
            f[i] = *reinterpret_cast<const u32x4 *>(
                lds + (P == 1 ? lds_at<BK>(r, KS * 4 + c) : KS * At::ELEMS + lds_at<BK>(r, c)));
        }
    }
};

// k-strided: the rows of k one after the other, or in an order if GATHER.
template <int BR, int BK, bool GATHER>
struct WideStrided {
    static constexpr int CH = BR / 8;                // chunks a row of k
    static constexpr int RPL = FL_WAVE / CH;         // rows of k a load
    static constexpr int LOADS = BK / RPL / WD_WAVES;
    static constexpr int ELEMS = BR * BK;
    const uint16_t *base;  // of the next step, if not GATHER
    int64_t ld;
    uint32_t at[LOADS];  // bytes from there, or from a row's first column

    // The permutation of a row's chunks, in steps of the two chunks that a
    // transposed read takes of each of 4 rows.
    static __device__ __forceinline__ int turn(int k) { return 2 * ((k & 3) | ((((k >> 3) ^ (k >> 4)) & 1) << 2)); }
    static __device__ __forceinline__ int row(int i) { return (fl_wave_id() * LOADS + i) * RPL + fl_lane() / CH; }

    __device__ __forceinline__ void init(const uint16_t *b, int64_t stride, int64_t R) {
        base = b;
        ld = stride;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int64_t c = ((fl_lane() % CH) ^ turn(row(i))) * 8;
            at[i] = (uint32_t)((c <= R - 8 ? c : R - 8) * 2);
            if constexpr (!GATHER) at[i] += (uint32_t)(row(i) * stride * 2);
        }
    }
    // The next `count` rows of k, BK if WHOLE; r: this lane's, if GATHER.
    template <bool WHOLE>
    __device__ __forceinline__ void issue(uint16_t *lds, int count, const int (&r)[LOADS]) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const char *q = (const char *)base + at[i];
            if constexpr (GATHER) q += (int64_t)r[i] * ld * 2;
            if (!WHOLE && row(i) >= count) q = (const char *)wd_zeros;
            load_lds(q, lds + (fl_wave_id() * LOADS + i) * 512);
        }
        if constexpr (!GATHER) base += count * ld;
    }
    // The operands of N 16-column tiles from col0 on.  In asm, with the wait:
    // the builtin's reads are made to wait for every load to LDS under way, so
    // the half of the waves that has just issued some began each step by
    // waiting for them.
    template <int N>
    __device__ __forceinline__ void read(const uint16_t *lds, int col0, u32x4 (&f)[BK / 32][N]) const {
        static_assert(BK == 64 && N % 4 == 0, "four tiles of two k steps a block");
        const int s = fl_lane() & 15, k = (fl_lane() >> 4) * 8 + (s >> 2);  // turn() is that of k's multiples of 4 and 32 on
        const uint32_t base =
            (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)lds + k * (BR * 2) + (s & 1) * 8;
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            uint32_t at[4];
#pragma unroll
            for (int t = 0; t < 4; ++t)
                at[t] = base + ((((col0 >> 3) + (i + t) * 2 + ((s & 3) >> 1)) ^ turn(k)) << 4);
            uint64_t v[4][4];  // [tile][4 rows, the next 4, those of k + 32]
            asm volatile(
                "ds_read_b64_tr_b16 %0, %16\n"
                "ds_read_b64_tr_b16 %1, %16 offset:%20\n"
                "ds_read_b64_tr_b16 %2, %16 offset:%21\n"
                "ds_read_b64_tr_b16 %3, %16 offset:%22\n"
                "ds_read_b64_tr_b16 %4, %17\n"
                "ds_read_b64_tr_b16 %5, %17 offset:%20\n"
                "ds_read_b64_tr_b16 %6, %17 offset:%21\n"
                "ds_read_b64_tr_b16 %7, %17 offset:%22\n"
                "ds_read_b64_tr_b16 %8, %18\n"
                "ds_read_b64_tr_b16 %9, %18 offset:%20\n"
                "ds_read_b64_tr_b16 %10, %18 offset:%21\n"
                "ds_read_b64_tr_b16 %11, %18 offset:%22\n"
                "ds_read_b64_tr_b16 %12, %19\n"
                "ds_read_b64_tr_b16 %13, %19 offset:%20\n"
                "ds_read_b64_tr_b16 %14, %19 offset:%21\n"
                "ds_read_b64_tr_b16 %15, %19 offset:%22\n"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[1][0]), "=&v"(v[1][1]),
                  "=&v"(v[1][2]), "=&v"(v[1][3]), "=&v"(v[2][0]), "=&v"(v[2][1]), "=&v"(v[2][2]), "=&v"(v[2][3]),
                  "=&v"(v[3][0]), "=&v"(v[3][1]), "=&v"(v[3][2]), "=&v"(v[3][3])
                : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(4 * BR * 2), "n"(32 * BR * 2), "n"(36 * BR * 2)
                : "memory");
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
                    f[ks][i + t] = u32x4{(uint32_t)v[t][2 * ks], (uint32_t)(v[t][2 * ks] >> 32),
                                         (uint32_t)v[t][2 * ks + 1], (uint32_t)(v[t][2 * ks + 1] >> 32)};
        }
    }
};

// The same, k rows one after the other, without guards: rows behind the last one
// read it again, so that the other operand has to be 0 there.  P: planes of a value,
// each of which lies in LDS as a tile of its own.
template <int BR, int P>
struct StepsStrided {
    static constexpr int STEP = P == 1 ? 64 : 32;
    using At = WideStrided<BR, STEP, false>;
    static constexpr int LOADS = P * At::LOADS, ELEMS = P * At::ELEMS;
    static constexpr bool BLOCKING = true;
    const uint16_t *base;  // of the next step
    int64_t ld;
    uint32_t at[At::LOADS];  // bytes

    // From column 0 of b on, R columns; `rows`: of k that there are, STEP at most.
    __device__ __forceinline__ void init(const uint16_t *b, int64_t stride, int64_t R, int rows) {
        const int lane = made_here(fl_lane());
        base = b;
        ld = stride;
        const int most = R - 8 < BR ? (int)R - 8 : BR;
#pragma unroll
        for (int i = 0; i < At::LOADS; ++i) {
            const int r = (fl_wave_id() * At::LOADS + i) * At::RPL + lane / At::CH;
            const int c0 = ((lane % At::CH) ^ At::turn(r)) * 8, c = c0 < most ? c0 : most;
            at[i] = (uint32_t)(P == 1 ? c : (int)plane_at(c)) * 2 +
                    (uint32_t)(r < rows ? r : rows - 1) * (uint32_t)(stride * 2);
        }
    }
    __device__ __forceinline__ void issue(uint16_t *lds, int i) {
        const int p = i / At::LOADS, j = i % At::LOADS;
        load_lds((const char *)base + p * 64 + at[j], lds + p * At::ELEMS + (fl_wave_id() * At::LOADS + j) * 512);
    }
    __device__ __forceinline__ void next() { base += STEP * ld; }
    // Of N 16-column tiles from col0 on: the step's first or second 32 rows, or those
    // of a plane.  In asm, with the wait, as WideStrided's.
    template <int KS, int N>
    __device__ __forceinline__ void read(const uint16_t *lds, int col0, u32x4 (&f)[N]) const {
        static_assert(N == 2 || N % 4 == 0, "two or four tiles a block");
        const int s = fl_lane() & 15, k = (fl_lane() >> 4) * 8 + (s >> 2);
        const uint32_t from =
            (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t *)lds + k * (BR * 2) + (s & 1) * 8;
        constexpr int LO = KS * 32 * BR * 2, HI = LO + 4 * BR * 2;
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            uint32_t a[4];
            uint64_t v[4][2];
#pragma unroll
            for (int t = 0; t < 4; ++t)
                a[t] = from + ((((col0 >> 3) + (i + t) * 2 + ((s & 3) >> 1)) ^ At::turn(k)) << 4);
            if constexpr (N == 2)
                asm volatile(
                    "ds_read_b64_tr_b16 %0, %4 offset:%6\n"
                    "ds_read_b64_tr_b16 %1, %4 offset:%7\n"
                    "ds_read_b64_tr_b16 %2, %5 offset:%6\n"
                    "ds_read_b64_tr_b16 %3, %5 offset:%7\n"
                    "s_waitcnt lgkmcnt(0)"
                    : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1])
                    : "v"(a[0]), "v"(a[1]), "n"(LO), "n"(HI)
                    : "memory");
            else
                asm volatile(
                    "ds_read_b64_tr_b16 %0, %8 offset:%12\n"
                    "ds_read_b64_tr_b16 %1, %8 offset:%13\n"
                    "ds_read_b64_tr_b16 %2, %9 offset:%12\n"
                    "ds_read_b64_tr_b16 %3, %9 offset:%13\n"
                    "ds_read_b64_tr_b16 %4, %10 offset:%12\n"
                    "ds_read_b64_tr_b16 %5, %10 offset:%13\n"
                    "ds_read_b64_tr_b16 %6, %11 offset:%12\n"
                    "ds_read_b64_tr_b16 %7, %11 offset:%13\n"
                    "s_waitcnt lgkmcnt(0)"
                    : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[2][0]), "=&v"(v[2][1]),
                      "=&v"(v[3][0]), "=&v"(v[3][1])
                    : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(LO), "n"(HI)
                    : "memory");
#pragma unroll
            for (int t = 0; t < (N < 4 ? N : 4); ++t)
                f[i + t] = u32x4{(uint32_t)v[t][0], (uint32_t)(v[t][0] >> 32), (uint32_t)v[t][1],
                                 (uint32_t)(v[t][1] >> 32)};
        }
    }
};

// The rows of k that a lane loads for strided operands, in the order `order`.
template <typename Tile>
struct WideRows {
    static constexpr int LOADS = Tile::LOADS, RPL = Tile::RPL, OWN = LOADS * RPL;
    const int32_t *order;  // of the next step
    int32_t next;          // lane j: the index of the wave's j-th row of that step

    __device__ __forceinline__ void init(const int32_t *ord, int first) {
        order = ord;
        look(first);
    }
    // One load of a wave, which arrives with the operands issued before it.
    // (Scalar loads of the eight rows were waited for with the LDS reads of
    // the same phase.)
    __device__ __forceinline__ void look(int count) {
        const int r = fl_wave_id() * OWN + fl_lane() % OWN;
        next = r < count ? order[r] : 0;
    }
    // The step of `count` rows, which `after` more follow.
    __device__ __forceinline__ void step(int count, int after, int (&r)[LOADS]) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) r[i] = __shfl(next, i * RPL + fl_lane() / Tile::CH);
        order += count;
        look(after);
    }
};

template <typename T, int BM, int BK, int STAGES, typename TA, typename TB>
struct WideProduct {
    static constexpr int MT = BM / 2 / 16, NTL = 4;
    static constexpr int ELEMS = TA::ELEMS + TB::ELEMS;
    static constexpr int LOADS = TA::LOADS + TB::LOADS;
    f32x4 acc[MT][NTL];

    static __device__ __forceinline__ int wave_m() { return (fl_wave_id() >> 2) * (BM / 2); }
    static __device__ __forceinline__ int wave_n() { return (fl_wave_id() & 3) * 64; }

    // feed(lds_a, lds_b, i, whole) issues the loads of step i, a whole one of
    // BK values or the first.
    template <typename F>
    __device__ __forceinline__ void run(const TA &ta, const TB &tb, int64_t steps, uint16_t *lds, F &&feed) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
        if (steps <= 0) return;
        const bool second = fl_wave_id() >= WD_WAVES / 2;
        const auto load = [&](int64_t step) {
            uint16_t *to = lds + (int)(step % STAGES) * ELEMS;
            feed(to, to + TA::ELEMS, step, std::true_type());
        };
        feed(lds, lds + TA::ELEMS, (int64_t)0, std::false_type());
#pragma unroll
        for (int s = 1; s < STAGES; ++s)
            if (s < steps) load(s);
        if (steps < STAGES) wait<0>();
        else wait<LOADS *(STAGES - 1)>();
        meet();
        if (second) meet();
        // Phase 2s: the first half reads step s, phase 2s + 1: it multiplies;
        // the second half one phase later.  In phase 2s + 2 both have read
        // step s and both load step s + STAGES over it; step s + 1 has to
        // have landed when phase 2s + 1 ends.
        for (int64_t s = 0; s < steps; ++s) {
            const uint16_t *la = lds + (int)(s % STAGES) * ELEMS, *lb = la + TA::ELEMS;
            const bool full = s + STAGES - 1 < steps;  // as many steps under way as there can be
            u32x4 fa[BK / 32][MT], fb[BK / 32][NTL];
            tb.read(lb, wave_n(), fb);
            ta.read(la, wave_m(), fa);
            if (!second && s > 0 && full) load(s + STAGES - 1);
            if (second) {
                if (full) wait<LOADS *(STAGES - 2)>();
                else wait<0>();
            } else wait_lds();
            meet();
            if (second && s + STAGES < steps) load(s + STAGES);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int ks = 0; ks < BK / 32; ++ks)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NTL; ++j) acc[i][j] = mfma<T>(fb[ks][j], fa[ks][i], acc[i][j]);
            __builtin_amdgcn_s_setprio(0);
            if (!second) {
                if (full) wait<LOADS *(STAGES - 2)>();
                else wait<0>();
            }
            meet();
        }
        if (!second) meet();
    }
    static __device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xc07f); }
    // Waits for this wave's LDS reads and for all but its last VM memory loads
    // (s_waitcnt: vmcnt in bits 0-3 and 14-15, expcnt 4-6, lgkmcnt 8-11).
    template <int VM>
    static __device__ __forceinline__ void wait() {
        __builtin_amdgcn_s_waitcnt((VM & 15) | ((VM >> 4) << 14) | 0x0070);
    }
    static __device__ __forceinline__ void meet() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
};

// Tiles one after the other as one sequence of steps, `steps` a tile: the loads
// run ahead over the tiles' ends.  Tiles of BM rows and WN x 64 columns, a step of
// 64 values (P = 3: 32 of three planes, six products).
//
// Operands are read from LDS beside the products of others: of small tiles those
// of the next step; of 256 x 256 tiles, whose sums leave fewer registers, a step's
// come in two halves, the first of the next step's beside the second's products.
// A barrier a step says that it is read by all and the next one there.  Loads of a
// later step are issued one at a time between the products.  (Read and multiplied
// in turns, by half the waves each or by all together, the matrix unit was busy 46%
// of the time, whatever the tile.)
//
// feed(i, lds_a, lds_b) issues load i of the next step, and after the last one
// goes on to the step behind it; behind the last step it may load anything that
// can be read.  out(tile) takes a tile's sums.
template <typename T, int P, int BM, int WN, int STAGES, typename TA, typename TB>
struct WideTiles {
    static constexpr int WM = WD_WAVES / WN, MT = BM / WM / 16, NTL = 4, BN = WN * 64;
    static constexpr int ELEMS = TA::ELEMS + TB::ELEMS, LOADS = TA::LOADS + TB::LOADS;
    using Waits = WideProduct<T, BM, 64, STAGES, TA, TB>;
    f32x4 acc[MT][NTL];

    static __device__ __forceinline__ int wave_m() { return (fl_wave_id() / WN) * (BM / WM); }
    static __device__ __forceinline__ int wave_n() { return (fl_wave_id() % WN) * 64; }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    }
    // between(i) comes behind the i-th of LOADS equal parts.
    template <typename F>
    __device__ __forceinline__ void multiply(const u32x4 (&fa)[MT], const u32x4 (&fb)[NTL], F &&between) {
        constexpr int ALL = MT * NTL, EACH = ALL / LOADS;
        static_assert(EACH >= 1, "a load between matrix instructions");
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) {
                acc[i][j] = mfma<T>(fb[j], fa[i], acc[i][j]);
                const int n = i * NTL + j + 1;
                if (n % EACH == 0 && n / EACH <= LOADS) between(n / EACH - 1);
            }
    }

    // ONE: a single tile.
    template <bool ONE, typename F, typename O>
    __device__ __forceinline__ void run(const TA &ta, const TB &tb, int tiles, int steps, uint16_t *lds, F &&feed,
                                        O &&out) {
        const int all = tiles * steps;
        clear();
        if (all <= 0) {
            for (int t = 0; t < tiles; ++t) out(t);
            return;
        }
        uint16_t *to = lds;
        const auto load = [&](int i) {
            feed(i, to, to + TA::ELEMS);
            if (i == LOADS - 1) to = to == lds + (STAGES - 1) * ELEMS ? lds : to + ELEMS;
        };
        const auto load_between = [&](int i) {
            __builtin_amdgcn_sched_barrier(0);
            load(i);
        };
        const auto none = [](int) {};
#pragma unroll
        for (int s = 0; s < STAGES; ++s)
#pragma unroll
            for (int i = 0; i < LOADS; ++i) load(i);
        Waits::template wait<LOADS *(STAGES - 1)>();
        Waits::meet();
        const uint16_t *la = lds;
        int at = 0, tile = 0;
        const auto go_on = [&]() { la = la == lds + (STAGES - 1) * ELEMS ? lds : la + ELEMS; };
        const auto finished = [&]() {
            if (ONE || ++at < steps) return;
            out(tile++);
            clear();
            at = 0;
        };
        if constexpr (MT * NTL <= 16) {
            // a whole step's operands beside those that are multiplied; half the waves read first, half multiply first
            struct Operands {
                u32x4 a[P == 1 ? 2 : 3][MT], b[P == 1 ? 2 : 3][NTL];
            };
            const bool second = fl_wave_id() >= WD_WAVES / 2;
            const auto read = [&](Operands &o) {
                tb.template read<0>(la + TA::ELEMS, wave_n(), o.b[0]);
                ta.template read<0>(la, wave_m(), o.a[0]);
                tb.template read<1>(la + TA::ELEMS, wave_n(), o.b[1]);
                ta.template read<1>(la, wave_m(), o.a[1]);
                if constexpr (P == 3) {
                    tb.template read<2>(la + TA::ELEMS, wave_n(), o.b[2]);
                    ta.template read<2>(la, wave_m(), o.a[2]);
                }
            };
            const auto step = [&](const Operands &now, Operands &next) {
                Waits::template wait<LOADS *(STAGES - 2)>();
                Waits::meet();
                go_on();
                if (!second) read(next);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (P == 3) {  // smallest products first
                    multiply(now.a[0], now.b[2], load_between);
                    multiply(now.a[1], now.b[1], none);
                    multiply(now.a[2], now.b[0], none);
                    multiply(now.a[0], now.b[1], none);
                    multiply(now.a[1], now.b[0], none);
                    multiply(now.a[0], now.b[0], none);
                } else {
                    multiply(now.a[0], now.b[0], load_between);
                    multiply(now.a[1], now.b[1], none);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (second) read(next);
                finished();
            };
            Operands even, odd;
            read(even);
            for (int s = 0;; s += 2) {
                step(even, odd);
                if (s + 1 >= all) break;
                step(odd, even);
                if (s + 2 >= all) break;
            }
        } else {
            static_assert(P == 1, "three planes of such tiles have no registers");
            // operands whose reads are waited for at once: half the waves read first, half multiply first
            const bool later = TA::BLOCKING && TB::BLOCKING && fl_wave_id() >= WD_WAVES / 2;
            u32x4 a0[MT], b0[NTL], a1[MT], b1[NTL];
            ta.template read<0>(la, wave_m(), a0);
            tb.template read<0>(la + TA::ELEMS, wave_n(), b0);
            const auto second_half = [&]() {
                tb.template read<1>(la + TA::ELEMS, wave_n(), b1);
                ta.template read<1>(la, wave_m(), a1);
            };
            const auto first_half = [&]() {
                tb.template read<0>(la + TA::ELEMS, wave_n(), b0);
                ta.template read<0>(la, wave_m(), a0);
            };
            for (int s = 0; s < all; ++s) {
                if (!later) second_half();
                __builtin_amdgcn_sched_barrier(0);
                multiply(a0, b0, none);
                __builtin_amdgcn_sched_barrier(0);
                if (later) second_half();
                Waits::template wait<LOADS *(STAGES - 2)>();
                Waits::meet();
                go_on();
                if (!later) first_half();
                __builtin_amdgcn_sched_barrier(0);
                multiply(a1, b1, load_between);
                __builtin_amdgcn_sched_barrier(0);
                if (later) first_half();
                finished();
            }
        }
        Waits::template wait<0>();  // loads behind the last step
        if (ONE) out(0);
    }
};

// A wave's tiles through its own slice of the LDS, 64 rows at a time, so that
// eight lanes store (and read the residual of) a whole 128-byte line of a row:
// straight from the accumulators a store has 32 bytes a row, and the epilogue
// took 15 us of a 256 x 256 tile.  f(row, col, v): eight columns of one row of
// the wave's tile.
constexpr int WD_SLICE = 64 * 64;  // floats; a row's 16-byte chunks turned by the row

__device__ __forceinline__ int slice_at(int row, int chunk) { return row * 64 + ((chunk ^ row) & 15) * 4; }

template <int MT, typename F>
__device__ __forceinline__ void wide_rows_out(const f32x4 (&acc)[MT][4], float *slice, F &&f) {
    const int lane = fl_lane();
#pragma unroll
    for (int h = 0; h < MT / 4; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f32x4 *>(slice + slice_at(i * 16 + (lane & 15), j * 4 + (lane >> 4))) =
                    acc[h * 4 + i][j];
        fl_wave_sync();
#pragma unroll 1
        for (int r = 0; r < 8; ++r) {
            const int row = r * 8 + (lane >> 3), col = (lane & 7) * 8;
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(slice + slice_at(row, col / 4));
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(slice + slice_at(row, col / 4 + 1));
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = lo[e];
                v[4 + e] = hi[e];
            }
            f(h * 64 + row, col, v);
        }
        fl_wave_sync();
    }
}

typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));

// The first `have` of eight values as floats, the others 0.  PAST: past the
// caches.
template <bool PAST = false, typename U>
__device__ __forceinline__ void load_eight(const U *p, int have, float (&out)[8]) {
    if (have >= 8) {
        Vec<U, 8> r;
        if constexpr (PAST) {
            Words q[sizeof(r) / 16];
#pragma unroll
            for (int i = 0; i < (int)sizeof(r) / 16; ++i)
                q[i] = __builtin_nontemporal_load(reinterpret_cast<const Words *>(p) + i);
            __builtin_memcpy(&r, q, sizeof(r));
        } else r = load_vec<U, 8>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = (float)r.v[e];
    } else
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = e < have ? (float)p[e] : 0.0f;
}
template <bool PAST, typename U>
__device__ __forceinline__ void store_eight(U *p, int have, const float (&v)[8]) {
    Vec<U, 8> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.v[e] = (U)v[e];
    if (have >= 8) {
        Words q[sizeof(o) / 16];
        __builtin_memcpy(q, &o, sizeof(o));
#pragma unroll
        for (int i = 0; i < (int)sizeof(o) / 16; ++i) {
            if constexpr (PAST) __builtin_nontemporal_store(q[i], reinterpret_cast<Words *>(p) + i);
            else reinterpret_cast<Words *>(p)[i] = q[i];
        }
    } else store_some<U, 8>(p, o, have);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a product is cut: tiles of `rows` rows (and 128 or 64 columns), and
// parts of its inner dimension whose sums a second launch joins.
struct Cut {
    int rows, parts;
};

// The fastest cut of an [M, N] product over K, by what the kernels measured.
// A 32-value step of a tile takes `alone` microseconds where CUs hold one
// workgroup, `shared` times the workgroups of a CU where they hold more (fp32:
// [1536 x 2048 -> 1645] takes 147 us in 156 tiles of 128, 101 us in 624 tiles
// of 64; [8192 x 2048 -> 2048] 383 us in tiles of 128); joining parts takes a
// launch and their traffic.
inline Cut best_cut(int64_t M, int64_t N, int64_t K, bool f32, bool small_tiles) {
    struct Tile {
        int rows, cols;
        double alone, shared;
    };
    static const Tile wide[3] = {{128, 128, 2.3, 1.45}, {64, 64, 1.2, 0.52}, {32, 64, 0.52, 0.3}};
    const double scale = f32 ? 1.0 : 0.35;
    const double steps = (double)ceil_div(K, 32);
    Cut best{64, 1};
    double least = 1e30;
    for (const Tile &t : wide) {
        if (t.rows == 32 && !small_tiles) continue;
        const int64_t tiles = ceil_div(M, t.rows) * ceil_div(N, t.rows == 128 && N <= 64 ? 64 : t.cols);
        for (int parts = 1; parts <= 16 && (parts == 1 || K / parts >= 128); ++parts) {
            const double shared = t.shared * (double)ceil_div(tiles * parts, 256);
            double us = steps / parts * scale * (shared > t.alone ? shared : t.alone);
            if (parts > 1) us += 4.0 + (double)parts * M * N * 8e-6 / 4.0;
            if (us < least) {
                least = us;
                best = Cut{t.rows, parts};
            }
        }
    }
    return best;
}

// LDS of a wide kernel: its operands' buffers, or the waves' slices behind them.
constexpr unsigned wide_bytes(int bm, int bk, int stages) {
    const int operands = stages * (bm + WD_BN) * bk * 2, slices = WD_WAVES * WD_SLICE * 4;
    return (unsigned)(operands > slices ? operands : slices);
}

// For the wide kernels: rows on 16 bytes, and offsets of a step's rows of k in 32 bits.
inline bool aligned(const void *p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && ld < (1 << 24); }

}  // namespace
}  // namespace fl
