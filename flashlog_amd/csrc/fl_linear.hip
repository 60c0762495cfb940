// Matrix products with bias, activation and residual in the epilogue, plain
// and grouped by relation, and their gradients:
//
//   y  = act(x W_g^T + b_g) + residual      rows of x in their groups g
//   d  = gy * act'(p)                       p = x W_g^T + b_g, kept by the forward
//   dx = d W_g      dW_g = sum over the group's rows of d^T x      db_g = sum of d
//
// One kernel body: C(m, n) = sum_k A(m, k) B(n, k), whose operands are read
// with k contiguous in memory (x, W in the forward; d in dx) or with k
// strided (W in dx; d and x in dW).  A workgroup stages BM + BN rows of BK
// values in LDS as 16-byte chunks of 8 consecutive k -- for k-strided
// operands a thread reads 8 k of its columns and transposes them in registers
// -- with the chunks of a row permuted so that the MFMA operand reads of 16
// rows touch all banks, and multiplies with v_mfma_f32_16x16x32.  The next
// tile's values are loaded to registers while the present one is multiplied.
// The operands are given to the instruction as (B, A), so that a lane holds
// four consecutive n of one row m: one 16-byte store, and the row's address
// once per 16 rows.
//
// bfloat16 and half operands feed the instruction as they are, sums are fp32.
// fp32 operands are cut into three bfloat16 planes, v = v0 + v1 + v2 exactly: v0
// truncated (no value overflows), v1 the rest rounded to the nearest, so that
// |v1| is below 2^-7 and |v2| at most 2^-16 of |v|, of either sign.  The six
// products whose weight is at least 2^-16 are added; what is dropped, mostly
// v1 w2 + v2 w1, is below 2^-22 of a product and as often above 0 as below
// (with both planes truncated it was up to 2^-21, always towards 0).  An fp32
// product is rounded by up to 2^-24 of itself.  The matrix unit
// takes bfloat16 16 times faster than fp32, so the six products run at 2.7 times the
// fp32 instruction's rate.  The planes of an infinity or NaN hold a NaN: sums
// that such a value enters are NaN.
#include "fl_abi.h"
#include "fl_common.h"
#include "fl_parts.h"
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

// exp by the hardware's 2^x: off by |x| 2^-24 of itself besides its own step.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// Phi(p) = erfc(-p / sqrt 2) / 2 by Abramowitz and Stegun 7.1.26 (off by at
// most 1.5e-7; the factor exp(-p^2/2) keeps the lower tail's own scale).
__device__ __forceinline__ float normal_cdf(float p) {
    const float x = fabsf(p) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.0f));
    float q = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
    q = __builtin_fmaf(t, q, 1.421413741f);
    q = __builtin_fmaf(t, q, -0.284496736f);
    q = __builtin_fmaf(t, q, 0.254829592f);
    const float tail = 0.5f * t * q * fast_exp(-x * x);
    return p < 0.0f ? tail : 1.0f - tail;
}

// The activations of the epilogue, in a few instructions each: with the
// library's erff the epilogue of a 128 x 128 tile took a third of a product
// over 2048 inputs (9000 vector instructions a wave).
__device__ __forceinline__ float act_value(float p, int act) {
    switch (act) {
        case FL_ACT_RELU: return p > 0.0f ? p : (p != p ? p : 0.0f);
        case FL_ACT_GELU: return p * normal_cdf(p);
        case FL_ACT_SILU: return p * __builtin_amdgcn_rcpf(1.0f + fast_exp(-p));
        case FL_ACT_TANH: {
            // near 0 the odd series, off by 4e-7 of itself at 1/4
            const float s = p * p;
            const float near = p + p * s * (-0.33333333f + s * (0.13333333f + s * -0.053968254f));
            const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + fast_exp(2.0f * p));
            return s < 0.0625f ? near : far;
        }
        case FL_ACT_SIGMOID: return __builtin_amdgcn_rcpf(1.0f + fast_exp(-p));
        default: return p;
    }
}

// f with the activation as a constant.
template <typename F>
__device__ __forceinline__ void by_act(int act, F &&f) {
    switch (act) {
        case FL_ACT_RELU: return f(std::integral_constant<int, FL_ACT_RELU>());
        case FL_ACT_GELU: return f(std::integral_constant<int, FL_ACT_GELU>());
        case FL_ACT_SILU: return f(std::integral_constant<int, FL_ACT_SILU>());
        case FL_ACT_TANH: return f(std::integral_constant<int, FL_ACT_TANH>());
        case FL_ACT_SIGMOID: return f(std::integral_constant<int, FL_ACT_SIGMOID>());
        default: return;
    }
}

template <int N>
__device__ __forceinline__ void act_values(float (&v)[N], int act) {
    by_act(act, [&](auto known) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = act_value(v[e], decltype(known)::value);
    });
}

// act'(p), from the same pieces (gelu's of [16384 x 2048] bf16 44 us, 48 with
// the library's erff and expf).
__device__ __forceinline__ float act_slope(float p, int act) {
    switch (act) {
        case FL_ACT_RELU: return p > 0.0f ? 1.0f : (p != p ? p : 0.0f);
        case FL_ACT_GELU: return normal_cdf(p) + p * (0.39894228040143268f * fast_exp(-0.5f * p * p));
        case FL_ACT_SILU: {
            const float q = __builtin_amdgcn_rcpf(1.0f + fast_exp(-p));
            return q * (1.0f + p * (1.0f - q));
        }
        case FL_ACT_TANH: {
            const float t = act_value(p, FL_ACT_TANH);
            return 1.0f - t * t;
        }
        case FL_ACT_SIGMOID: {
            const float q = act_value(p, FL_ACT_SIGMOID);
            return q * (1.0f - q);
        }
        default: return 1.0f;
    }
}

template <int N>
__device__ __forceinline__ void act_slopes(float (&v)[N], int act) {
    by_act(act, [&](auto known) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = act_slope(v[e], decltype(known)::value);
    });
}

struct RowsArgs {
    const void *a, *b;
    void *c;
    int64_t lda, ldb, b_group, ldc;  // elements
    int64_t M, N, K;                 // C is [M, N]
    int64_t groups;
    uint32_t n_tiles;
    const int32_t *order, *offsets, *tiles;
    const void *bias, *residual;
    int64_t bias_group, ldres;
    float *pre;
    int act, bias_f32, block;
    uint32_t parts;  // of K
    float *part;     // [parts][M][N] sums without the epilogue, when parts > 1
};

// A tile of a product: its group (`none`: the rows of no group) and the places
// pos0 .. end of its rows.
struct RowTile {
    int64_t g, pos0, end;
    bool none;
};

// The BM rows of tile mt; the plan's tiles are `block` rows.
template <int BM>
__device__ __forceinline__ bool row_tile(const RowsArgs &a, uint32_t mt, RowTile *t) {
    if (!a.tiles) {
        *t = RowTile{0, (int64_t)mt * BM, a.M, false};
        return true;
    }
    const uint32_t sub = a.block / BM;
    const int32_t *e = a.tiles + 2 * (int64_t)(mt / sub);
    const int64_t g = e[0];
    if (g < 0) return false;
    const int64_t end = g < a.groups ? (int64_t)a.offsets[g + 1] : a.M;
    *t = RowTile{g, e[1] + (int64_t)(mt % sub) * BM, end, g >= a.groups};
    return t->pos0 < end;
}

// Stores a wave's tiles, whose first row is at place `pos` and first column
// `col`: bias, activation, residual, one rounding.
template <typename T, int MT, int NTL>
__device__ __forceinline__ void store_rows(const RowsArgs &a, const f32x4 (&acc)[MT][NTL], const RowTile &t,
                                           int64_t pos, int64_t col) {
    const int lane = fl_lane();
    const int64_t n0 = col + (lane >> 4) * 4;
    int have[NTL];  // columns of the lane's j-th four
    float bias[NTL][4];
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
        const int64_t left = a.N - (n0 + j * 16);
        have[j] = left < 0 ? 0 : left < 4 ? (int)left : 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[j][e] = 0.0f;
        if (a.bias && !t.none) {
            const int64_t at = t.g * a.bias_group + n0 + j * 16;
            if (a.bias_f32) load_some<float>((const float *)a.bias + at, have[j], bias[j]);
            else load_some<T>((const T *)a.bias + at, have[j], bias[j]);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t p = pos + i * 16 + (lane & 15);
        if (p >= t.end) continue;
        const int64_t row = a.order ? (int64_t)a.order[p] : p;
        float res[NTL][4];
        if (a.residual)
#pragma unroll
            for (int j = 0; j < NTL; ++j)
                load_some<T>((const T *)a.residual + row * a.ldres + n0 + j * 16, have[j], res[j]);
#pragma unroll
        for (int j = 0; j < NTL; ++j) {
            if (!have[j]) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] + bias[j][e];
            if (a.pre) {
                // kept in 32 bits: rounded to the operands' type it would move the slopes by as much as the
                // gradients' own rounding does
                const Vec<float, 4> f{{v[0], v[1], v[2], v[3]}};
                float *q = a.pre + row * a.N + n0 + j * 16;
                if (have[j] == 4) store_vec<float, 4>(q, f);
                else store_some<float, 4>(q, f, have[j]);
            }
            if (!t.none)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = act_value(v[e], a.act);
            if (a.residual)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += res[j][e];
            Vec<T, 4> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[e] = (T)v[e];
            T *q = (T *)a.c + row * a.ldc + n0 + j * 16;
            if (have[j] == 4) store_vec<T, 4>(q, o);
            else store_some<T, 4>(q, o, have[j]);
        }
    }
}

// The sums of a part of K (one group of all rows).
template <int MT, int NTL>
__device__ __forceinline__ void store_part(const RowsArgs &a, const f32x4 (&acc)[MT][NTL], uint32_t part, int64_t pos,
                                           int64_t col) {
    const int lane = fl_lane();
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t row = pos + i * 16 + (lane & 15);
        if (row >= a.M) continue;
#pragma unroll
        for (int j = 0; j < NTL; ++j) {
            const int64_t n = col + j * 16 + (lane >> 4) * 4;
            if (n >= a.N) continue;
            float *q = a.part + ((int64_t)part * a.M + row) * a.N + n;
            const Vec<float, 4> f{{acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]}};
            if (a.N - n >= 4) store_vec<float, 4>(q, f);
            else store_some<float, 4>(q, f, (int)(a.N - n));
        }
    }
}

// Joins the parts of K in order and finishes as store_rows does, four columns
// a thread ([1536 x 1645] fp32 of two parts: 10 us).
template <typename T>
__global__ __launch_bounds__(LN_NT) void k_lin_finish(RowsArgs a) {
    const uint32_t quads = (uint32_t)((a.N + 3) / 4);
    const int64_t i = fl_block() * LN_NT + threadIdx.x;
    if (i >= a.M * quads) return;
    const int64_t row = i / quads, n = (i % quads) * 4;
    const int have = a.N - n < 4 ? (int)(a.N - n) : 4;
    float v[4] = {0, 0, 0, 0}, t[4];
    for (uint32_t p = 0; p < a.parts; ++p) {
        load_some<float>(a.part + ((int64_t)p * a.M + row) * a.N + n, have, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += t[e];
    }
    if (a.bias) {
        if (a.bias_f32) load_some<float>((const float *)a.bias + n, have, t);
        else load_some<T>((const T *)a.bias + n, have, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += t[e];
    }
    if (a.pre) store_some<float, 4>(a.pre + row * a.N + n, Vec<float, 4>{{v[0], v[1], v[2], v[3]}}, have);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = act_value(v[e], a.act);
    if (a.residual) {
        load_some<T>((const T *)a.residual + row * a.ldres + n, have, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += t[e];
    }
    Vec<T, 4> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.v[e] = (T)v[e];
    T *q = (T *)a.c + row * a.ldc + n;
    if (have == 4) store_vec<T, 4>(q, o);
    else store_some<T, 4>(q, o, have);
}

// Products whose C rows are the batch's rows (the forward, and dx): a tile is
// BM rows of one group.  fp32 [1536 x 2048 -> 1645]: 65 us = 159 TFLOP/s, dx 86,
// bound by the six products' matrix instructions and the LDS reads before them;
// [15000 x 128 -> 75] in 74 groups 17 us, four steps of latency.
template <typename T, bool B_CONTIG, int BM, int BN, int BK>
__global__ __launch_bounds__(LN_NT) void k_lin_rows(RowsArgs a) {
    using Prod = Product<T, BM, BN, BK>;
    __shared__ __align__(16) uint16_t lds[Prod::LDS_ELEMS];
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const uint32_t tile = w / a.parts, part = w % a.parts;
    RowTile t;
    if (!row_tile<BM>(a, tile / a.n_tiles, &t)) return;
    const int64_t n0 = (int64_t)(tile % a.n_tiles) * BN;
    // whole steps of K a part; the last has the end of K
    const int64_t steps = (a.K + BK - 1) / BK, k0 = steps * part / a.parts * BK;
    const int64_t k1 = part + 1 == a.parts ? a.K : steps * (part + 1) / a.parts * BK;
    const T *A = (const T *)a.a;
    const T *B = (const T *)a.b + (t.none ? 0 : t.g * a.b_group);
    ContigTile<T, BM, BK> ta;
    ta.init([&](int r) {
        const int64_t p = t.pos0 + r < t.end ? t.pos0 + r : t.end - 1;
        return A + (a.order ? (int64_t)a.order[p] : p) * a.lda + k0;
    });
    Prod prod;
    const int64_t K = t.none ? 0 : k1 - k0;
    if constexpr (B_CONTIG) {
        ContigTile<T, BN, BK> tb;
        tb.init([&](int r) { return B + (n0 + r < a.N ? n0 + r : a.N - 1) * a.ldb + k0; });
        prod.run(ta, tb, K, lds);
    } else {
        StridedTile<T, BN, BK> tb;
        tb.init(B + k0 * a.ldb + n0, a.ldb, a.N - n0, nullptr);
        prod.run(ta, tb, K, lds);
    }
    if (a.part) store_part(a, prod.acc, part, t.pos0 + prod.wave_m(), n0 + prod.wave_n());
    else store_rows<T>(a, prod.acc, t, t.pos0 + prod.wave_m(), n0 + prod.wave_n());
}

struct OuterArgs {
    const void *d, *x;
    int64_t ldd, ldx;
    int64_t M, N, K;  // rows; dW_g is [N, K]
    int64_t groups;
    uint32_t n_tiles, k_tiles, parts;
    const int32_t *order, *offsets;
    void *dw;
    float *part;  // [parts][groups][N][K] when parts > 1
};

// A group's positions, cut into equal parts.
__device__ __forceinline__ void part_range(const int32_t *offsets, int64_t M, int64_t g, int parts, int p,
                                           int64_t *begin, int64_t *end) {
    const int64_t b = offsets ? (int64_t)offsets[g] : 0;
    const int64_t n = (offsets ? (int64_t)offsets[g + 1] : M) - b;
    *begin = b + n * p / parts;
    *end = b + n * (p + 1) / parts;
}

// Stores a wave's tiles of dW_g, or of a part of its sum.
template <typename T, int MT, int NTL>
__device__ __forceinline__ void store_outer(const OuterArgs &a, const f32x4 (&acc)[MT][NTL], int64_t g, int part,
                                            int64_t row, int64_t col) {
    const int lane = fl_lane();
    const int64_t NK = a.N * a.K;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = row + i * 16 + (lane & 15);
        if (m >= a.N) continue;
#pragma unroll
        for (int j = 0; j < NTL; ++j) {
            const int64_t c = col + j * 16 + (lane >> 4) * 4;
            if (c >= a.K) continue;
            const int n = a.K - c < 4 ? (int)(a.K - c) : 4;
            if (a.part) {
                float *q = a.part + ((int64_t)part * a.groups + g) * NK + m * a.K + c;
                const Vec<float, 4> f{{acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]}};
                if (n == 4) store_vec<float, 4>(q, f);
                else store_some<float, 4>(q, f, n);
            } else {
                T *q = (T *)a.dw + g * NK + m * a.K + c;
                Vec<T, 4> o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o.v[e] = (T)acc[i][j][e];
                if (n == 4) store_vec<T, 4>(q, o);
                else store_some<T, 4>(q, o, n);
            }
        }
    }
}

// dW_g = sum over the group's rows (a part of them) of d^T x.  fp32 [1645 x
// 2048] over 1536 rows: 86 us; [75 x 128] over 15000 rows in 74 groups 21 us.
template <typename T, int BM, int BN, int BK>
__global__ __launch_bounds__(LN_NT) void k_lin_outer(OuterArgs a) {
    using Prod = Product<T, BM, BN, BK>;
    __shared__ __align__(16) uint16_t lds[Prod::LDS_ELEMS];
    uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const int64_t nt = w % a.n_tiles;
    w /= a.n_tiles;
    const int64_t kt = w % a.k_tiles;
    w /= a.k_tiles;
    const int part = (int)(w % a.parts);
    const int64_t g = w / a.parts;
    int64_t begin, end;
    part_range(a.offsets, a.M, g, (int)a.parts, part, &begin, &end);
    const int64_t m0 = nt * BM, c0 = kt * BN, len = end - begin;
    const T *D = (const T *)a.d + m0, *X = (const T *)a.x + c0;
    const int32_t *ord = a.order ? a.order + begin : nullptr;
    if (!ord) {
        D += begin * a.ldd;
        X += begin * a.ldx;
    }
    StridedTile<T, BM, BK> ta;
    StridedTile<T, BN, BK> tb;
    ta.init(D, a.ldd, a.N - m0, ord);
    tb.init(X, a.ldx, a.K - c0, ord);
    Prod prod;
    prod.run(ta, tb, len, lds);
    store_outer<T>(a, prod.acc, g, part, m0 + prod.wave_m(), c0 + prod.wave_n());
}

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

template <typename T, int MT>
__device__ __forceinline__ void wide_store_rows(const RowsArgs &a, const f32x4 (&acc)[MT][4], const RowTile &t,
                                                int64_t pos, int64_t col, float *slice) {
    const int64_t n = col + (fl_lane() & 7) * 8;
    const int have = a.N - n < 8 ? (int)(a.N - n) : 8;
    float bias[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (a.bias && !t.none && have > 0) {
        if (a.bias_f32) load_eight<false, float>((const float *)a.bias + t.g * a.bias_group + n, have, bias);
        else load_eight<false, T>((const T *)a.bias + t.g * a.bias_group + n, have, bias);
    }
    wide_rows_out<MT>(acc, slice, [&](int r, int, float (&v)[8]) {
        const int64_t p = pos + r;
        if (p >= t.end || have <= 0) return;
        const int64_t row = a.order ? (int64_t)a.order[p] : p;
        float res[8];
        if (a.residual) load_eight<false, T>((const T *)a.residual + row * a.ldres + n, have, res);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bias[e];
        if (a.pre) store_eight<true, float>(a.pre + row * a.N + n, have, v);
        if (!t.none) act_values(v, a.act);
        if (a.residual)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += res[e];
        store_eight<false, T>((T *)a.c + row * a.ldc + n, have, v);
    });
}

template <typename T, int MT>
__device__ __forceinline__ void wide_store_outer(const OuterArgs &a, const f32x4 (&acc)[MT][4], int64_t g, int part,
                                                 int64_t row, int64_t col, float *slice) {
    const int64_t NK = a.N * a.K, c = col + (fl_lane() & 7) * 8;
    const int have = a.K - c < 8 ? (int)(a.K - c) : 8;
    wide_rows_out<MT>(acc, slice, [&](int r, int, float (&v)[8]) {
        const int64_t m = row + r;
        if (m >= a.N || have <= 0) return;
        if (a.part) store_eight<false, float>(a.part + ((int64_t)part * a.groups + g) * NK + m * a.K + c, have, v);
        else store_eight<true, T>((T *)a.dw + g * NK + m * a.K + c, have, v);
    });
}

// The forward (B_CONTIG) and dx.  [8192 x 8192 -> 8192] bf16: 900 us = 1221
// TFLOP/s; [16384 x 2048 -> 2048] 121 us = 1136 TFLOP/s (two rounds of 256
// tiles, whose first loads and last stores nothing overlaps), 163 us in fp16 with
// silu, a residual and the argument kept: its fp32 values go past the caches
// (through them an eighth more).
template <typename T, bool B_CONTIG, int BM, int BK, int STAGES>
__global__ __launch_bounds__(WD_NT) void k_wide_rows(RowsArgs a) {
    using TA = WideContig<BM, BK>;
    using TB = std::conditional_t<B_CONTIG, WideContig<WD_BN, BK>, WideStrided<WD_BN, BK, false>>;
    using Prod = WideProduct<T, BM, BK, STAGES, TA, TB>;
    extern __shared__ __align__(16) uint16_t wide_lds[];
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    RowTile t;
    if (!row_tile<BM>(a, w / a.n_tiles, &t)) return;
    const int64_t n0 = (int64_t)(w % a.n_tiles) * WD_BN;
    const uint16_t *A = (const uint16_t *)a.a;
    const uint16_t *B = (const uint16_t *)a.b + (t.none ? 0 : t.g * a.b_group);
    const int64_t steps = t.none ? 0 : (a.K + BK - 1) / BK;
    const int first = (int)(a.K - (steps - 1) * BK);  // the step that is no whole one comes first
    TA ta;
    TB tb;
    ta.init([&](int r) {
        const int64_t p = t.pos0 + r < t.end ? t.pos0 + r : t.end - 1;
        return A + (a.order ? (int64_t)a.order[p] : p) * a.lda;
    });
    if constexpr (B_CONTIG) tb.init([&](int r) { return B + (n0 + r < a.N ? n0 + r : a.N - 1) * a.ldb; });
    else tb.init(B + n0, a.ldb, a.N - n0);
    Prod prod;
    prod.run(ta, tb, steps, wide_lds, [&](uint16_t *la, uint16_t *lb, int64_t, auto whole) {
        const int count = decltype(whole)::value ? BK : first;
        ta.template issue<decltype(whole)::value>(la, count);
        if constexpr (B_CONTIG) tb.template issue<decltype(whole)::value>(lb, count);
        else tb.template issue<decltype(whole)::value>(lb, count, {});
    });
    __syncthreads();  // the operands in the LDS are read
    wide_store_rows<T>(a, prod.acc, t, t.pos0 + prod.wave_m(), n0 + prod.wave_n(),
                       reinterpret_cast<float *>(wide_lds) + fl_wave_id() * WD_SLICE);
}

// The tile of a workgroup of dW of several groups: an XCD takes whole groups
// (or parts of them) in turn, there and back, so that the large ones spread
// over all.  (16384 rows in 24 groups, the size falling with the root of the
// group's number: 105 us, 144 where an XCD takes groups that lie together;
// sizes in no order: 119 and 115.)
__device__ __forceinline__ uint32_t outer_item(const OuterArgs &a) {
    const uint32_t unit = a.n_tiles * a.k_tiles, whole = gridDim.x / unit / FL_XCDS * FL_XCDS * unit;
    if (blockIdx.x >= whole) return blockIdx.x;
    const uint32_t x = blockIdx.x % FL_XCDS, p = blockIdx.x / FL_XCDS, j = p / unit;
    return (j * FL_XCDS + (j & 1 ? FL_XCDS - 1 - x : x)) * unit + p % unit;
}

// dW.  [2048 x 2048] over 16384 fp16 rows: 119 us = 1155 TFLOP/s in four parts
// of the rows, that fold_parts joins in 12 us.
template <typename T, bool GATHER, int BK, int STAGES>
__global__ __launch_bounds__(WD_NT) void k_wide_outer(OuterArgs a) {
    using Tile = WideStrided<WD_BN, BK, GATHER>;
    using Prod = WideProduct<T, WD_BN, BK, STAGES, Tile, Tile>;
    extern __shared__ __align__(16) uint16_t wide_lds[];
    uint32_t w = GATHER ? outer_item(a) : (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const int64_t nt = w % a.n_tiles;
    w /= a.n_tiles;
    const int64_t kt = w % a.k_tiles;
    w /= a.k_tiles;
    const int part = (int)(w % a.parts);
    const int64_t g = w / a.parts;
    int64_t begin, end;
    part_range(a.offsets, a.M, g, (int)a.parts, part, &begin, &end);
    const int64_t m0 = nt * WD_BN, c0 = kt * WD_BN, len = end - begin;
    const uint16_t *D = (const uint16_t *)a.d + m0, *X = (const uint16_t *)a.x + c0;
    if constexpr (!GATHER) {
        D += begin * a.ldd;
        X += begin * a.ldx;
    }
    const int64_t steps = (len + BK - 1) / BK;
    const int first = (int)(len - (steps - 1) * BK);
    Tile ta, tb;
    ta.init(D, a.ldd, a.N - m0);
    tb.init(X, a.ldx, a.K - c0);
    WideRows<Tile> rows;
    if constexpr (GATHER) rows.init(a.order + begin, len > 0 ? first : 0);
    Prod prod;
    prod.run(ta, tb, steps, wide_lds, [&](uint16_t *la, uint16_t *lb, int64_t s, auto whole) {
        const int count = decltype(whole)::value ? BK : first;
        int r[Tile::LOADS] = {};
        if constexpr (GATHER) rows.step(count, s + 1 < steps ? BK : 0, r);
        ta.template issue<decltype(whole)::value>(la, count, r);
        tb.template issue<decltype(whole)::value>(lb, count, r);
    });
    __syncthreads();  // the operands in the LDS are read
    wide_store_outer<T>(a, prod.acc, g, part, m0 + prod.wave_m(), c0 + prod.wave_n(),
                        reinterpret_cast<float *>(wide_lds) + fl_wave_id() * WD_SLICE);
}

// d = gy * act'(p), rounded to the operands' type: it is an operand of two
// products.  HBM-bound: [16384 x 2048] bf16 44 us = 6.1 TB/s.
template <typename T>
__global__ __launch_bounds__(LN_NT) void k_act_grad(const T *__restrict__ gy, const float *__restrict__ pre, int64_t n,
                                                    int act, T *__restrict__ d) {
    const int64_t i = ((int64_t)blockIdx.x * LN_NT + threadIdx.x) * 4;
    if (i >= n) return;
    if (i + 4 <= n) {
        const Vec<T, 4> g = load_vec<T, 4>(gy + i);
        const Vec<float, 4> p = load_vec<float, 4>(pre + i);
        Vec<T, 4> o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] = (T)((float)g.v[e] * act_slope(p.v[e], act));
        store_vec<T, 4>(d + i, o);
    } else
        for (int64_t e = i; e < n; ++e) d[e] = (T)((float)gy[e] * act_slope(pre[e], act));
}

// The same and the column sums of a part of a group's rows in one pass, added
// before d is rounded: a workgroup takes 512 columns, eight a lane, each wave a
// quarter of its rows, in the plan's order if GATHER (rows of no group have no
// d).  [16384 x 2048] fp16: 51 us = 5.3 TB/s, 63 in two passes; bf16 in 24
// groups 77 us (the workgroups of a row's columns on one XCD; 82 spread over
// all, 93 with half as many workgroups).  What it reads is not read again and
// goes past the caches, which keep d for dx (there 114 -> 104 us) and dW
// (113 -> 107).
constexpr int AS_COLS = 8 * FL_WAVE;
constexpr int AS_GROUPS = 2048;  // workgroups, where the rows give as many

template <typename T, bool GATHER>
__global__ __launch_bounds__(LN_NT) void k_act_sums(const T *__restrict__ gy, const float *__restrict__ pre, int64_t M,
                                                    int64_t N, int64_t groups, int parts, int act,
                                                    const int32_t *__restrict__ order,
                                                    const int32_t *__restrict__ offsets, T *__restrict__ d,
                                                    float *__restrict__ out) {
    constexpr int AHEAD = 4;
    constexpr int WAVES = LN_NT / FL_WAVE;
    __shared__ float sums[WAVES][AS_COLS];
    const uint32_t w = GATHER ? (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x) : blockIdx.x;
    const uint32_t blocks = (uint32_t)((N + AS_COLS - 1) / AS_COLS), item = w / blocks;
    const int64_t c0 = (int64_t)(w % blocks) * AS_COLS, c = c0 + fl_lane() * 8;
    const int64_t g = GATHER ? item / parts : 0, part = GATHER ? item % parts : item;
    const int have = N - c < 8 ? (int)(N - c) : 8;
    int64_t begin, end;
    part_range(GATHER ? offsets : nullptr, M, g, parts * WAVES, (int)part * WAVES + fl_wave_id(), &begin, &end);
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    int rows = 0;  // lane j: the j-th of 64 in the order
    for (int64_t p = begin; p < end; p += AHEAD) {
        float v[AHEAD][8], q[AHEAD][8];
        int64_t row[AHEAD];
        const int at = (int)(p - begin) % FL_WAVE;
        if (GATHER && at == 0) rows = order[p + fl_lane() < end ? p + fl_lane() : end - 1];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            row[j] = GATHER ? (int64_t)__builtin_amdgcn_readlane(rows, at + j) : p + j < end ? p + j : end - 1;
        if (have <= 0) continue;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            load_eight<true, T>(gy + row[j] * N + c, have, v[j]);
            load_eight<true, float>(pre + row[j] * N + c, have, q[j]);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (p + j >= end) break;
            act_slopes(q[j], act);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[j][e] *= q[j][e];
                s[e] += v[j][e];
            }
            store_eight<false, T>(d + row[j] * N + c, have, v[j]);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[fl_wave_id()][fl_lane() * 8 + e] = s[e];
    __syncthreads();
#pragma unroll
    for (int i = threadIdx.x; i < AS_COLS; i += LN_NT)
        if (c0 + i < N) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) t += sums[w][i];
            out[(part * groups + g) * N + c0 + i] = t;
        }
}

// Column sums of a group's rows (a part of them), one thread a column: [16384 x
// 2048] fp16 15 us = 4.5 TB/s.  With an activation (ACT) d's terms are made
// again from the gradient gy and the argument, unrounded.
template <typename T, bool ACT>
__global__ __launch_bounds__(LN_NT) void k_col_sums(const T *__restrict__ d, const float *__restrict__ pre, int act,
                                                    int64_t M, int64_t N, int64_t groups, int parts,
                                                    const int32_t *__restrict__ order,
                                                    const int32_t *__restrict__ offsets, float *__restrict__ out) {
    const int64_t blocks = (N + LN_NT - 1) / LN_NT, w = blockIdx.x / blocks;
    const int64_t c = (blockIdx.x % blocks) * LN_NT + threadIdx.x;
    const int64_t g = w / parts;
    const int part = (int)(w % parts);
    if (c >= N) return;
    int64_t begin, end;
    part_range(offsets, M, g, parts, part, &begin, &end);
    float s = 0.0f;
    int64_t p = begin;
    for (; p + 8 <= end; p += 8) {
        float v[8], q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t at = (order ? (int64_t)order[p + j] : p + j) * N + c;
            v[j] = (float)d[at];
            if (ACT) q[j] = pre[at];
        }
        if (ACT) act_slopes(q, act);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += ACT ? v[j] * q[j] : v[j];
    }
    for (; p < end; ++p) {
        const int64_t at = (order ? (int64_t)order[p] : p) * N + c;
        const float v = (float)d[at];
        s += ACT ? v * act_slope(pre[at], act) : v;
    }
    out[((int64_t)part * groups + g) * N + c] = s;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

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
Cut best_cut(int64_t M, int64_t N, int64_t K, bool f32, bool small_tiles) {
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
bool aligned(const void *p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && ld < (1 << 24); }

// Rows of the wide kernels' tiles, 0: the operands or the sizes are not for
// them.  bf16 [M x 2048 -> 2048], us with other tiles, 128 rows and 256 rows:
// M = 1024 24, 32, 47; 2048 43, 34, 49; 4096 65, 41, 51; 6144 96, 74, 55; 8192
// 115, 77, 62.  So 128 rows from half the CUs on, and 256 where the tiles of 128
// would be more than the CUs.  Groups: 256 rows (16384 rows in 24 groups, bf16
// [1024 -> 2048]: 137 us, 165 with 128 rows) from 64 tiles on (8192 rows in 4
// groups, [1024 -> 512], 64 tiles: 34 us, 38 with others; [1024 -> 256] 33, 30).
int wide_rows(const fl_linear *op, const RowsArgs &a, bool b_contig) {
    if (op->dtype == FL_F32 || !aligned(a.a, a.lda) || !aligned(a.b, a.ldb) || a.b_group % 8 || a.K % 8 || a.K < 64 ||
        (!b_contig && a.N % 8) || a.N < 192)
        return 0;
    const int64_t cols = ceil_div(a.N, WD_BN);
    if (op->offsets) return fl_group_block(op->M, op->groups) == 256 && ceil_div(op->M, 256) * cols >= 64 ? 256 : 0;
    const int64_t tiles = ceil_div(op->M, 128) * cols;
    return tiles < 128 ? 0 : tiles <= 256 ? 128 : 256;
}

// The cut of y's or dx's product that the wide kernels do not take.
Cut rows_cut(const fl_linear *op, int64_t N, int64_t K) {
    if (op->offsets) {
        const int block = (int)fl_group_block(op->M, op->groups);
        return Cut{block < 128 ? block : 128, 1};
    }
    return best_cut(op->M, N, K, op->dtype == FL_F32, true);
}

size_t rows_bytes(const fl_linear *op, int64_t N, int64_t K) {
    const Cut c = rows_cut(op, N, K);
    return c.parts > 1 ? (size_t)c.parts * op->M * N * 4 : 0;
}

template <typename T, bool B_CONTIG>
int launch_rows(hipStream_t st, const fl_linear *op, RowsArgs &a, float *ws, const char *what) {
    a.block = (int)fl_group_block(op->M, op->groups);
    const int wide = sizeof(T) == 2 ? wide_rows(op, a, B_CONTIG) : 0;
    const Cut cut = wide ? Cut{wide, 1} : rows_cut(op, a.N, a.K);
    const int bm = cut.rows;
    a.parts = (uint32_t)cut.parts;
    a.part = cut.parts > 1 ? ws : nullptr;
    constexpr int BIG_K = sizeof(T) == 4 ? 32 : 64;
    const int bn = wide ? WD_BN : bm == 128 && a.N > 64 ? 128 : 64;
    const int64_t m_tiles = op->offsets ? fl_group_tiles(op->M, op->groups) * (a.block / bm) : ceil_div(op->M, bm);
    a.n_tiles = (uint32_t)ceil_div(a.N, bn);
    const int64_t grid = m_tiles * a.n_tiles * a.parts;
    if (!launch_fits(grid, wide ? WD_NT : LN_NT))
        return fl_fail(FL_ERR_ARG, "%s: too many tiles for one launch (shape)", what);
    if (grid == 0) return FL_OK;
    const dim3 g((unsigned)grid), nt(LN_NT);
    if constexpr (sizeof(T) == 2) {
        if (wide == 256)
            FL_LAUNCH("k_wide_rows", (k_wide_rows<T, B_CONTIG, 256, 64, 2>), g, dim3(WD_NT), wide_bytes(256, 64, 2), st, a);
        else if (wide)
            FL_LAUNCH("k_wide_rows", (k_wide_rows<T, B_CONTIG, 128, 64, 3>), g, dim3(WD_NT), wide_bytes(128, 64, 3), st, a);
        if (wide) return fl_check_launch(what);
    }
    if (bn == 128) FL_LAUNCH("k_lin_rows", (k_lin_rows<T, B_CONTIG, 128, 128, BIG_K>), g, nt, 0, st, a);
    else if (bm == 128) FL_LAUNCH("k_lin_rows", (k_lin_rows<T, B_CONTIG, 128, 64, BIG_K>), g, nt, 0, st, a);
    else if (bm == 64) FL_LAUNCH("k_lin_rows", (k_lin_rows<T, B_CONTIG, 64, 64, BIG_K>), g, nt, 0, st, a);
    else FL_LAUNCH("k_lin_rows", (k_lin_rows<T, B_CONTIG, 32, 64, 64>), g, nt, 0, st, a);
    if (a.part)
        FL_LAUNCH("k_lin_finish", k_lin_finish<T>, grid_of(ceil_div(a.M * ceil_div(a.N, 4), LN_NT)), nt, 0, st, a);
    return fl_check_launch(what);
}

// Parts of a group's rows in dW and db: enough workgroups for the chip where
// the tiles alone are few, of at least 256 rows on average.
int outer_parts(int64_t M, int64_t groups, int64_t tiles, int64_t workgroups) {
    int64_t want = workgroups / (tiles * groups), most = M / (256 * groups);
    int64_t p = want < most ? want : most;
    return (int)(p < 1 ? 1 : p > 64 ? 64 : p);
}

// Whether d and db are made in one pass: with few columns most lanes of its
// waves would have none.  In several groups where d is rounded, so that db's
// terms would be made twice otherwise, from 32 rows a group on (bf16 gelu, us
// in one pass and in two, sizes falling with the group's number: 16384 rows of
// 475 in 100 groups 68, 101; 4000 rows in 100 groups 60, 104, in 300 groups 225,
// 92, where a part is a whole group and the largest one's rows are walked by
// one workgroup).
bool act_and_sums(const fl_linear *op) {
    if (op->act == FL_ACT_NONE || op->N < 256) return false;
    return !op->offsets || (op->dtype != FL_F32 && op->M >= 32 * op->groups);
}

// Parts of a group's rows in db's sums.
int sum_parts(const fl_linear *op) {
    const int64_t M = op->M, N = op->N, groups = op->groups;
    if (act_and_sums(op)) {
        const int64_t want = ceil_div(AS_GROUPS, ceil_div(N, AS_COLS) * groups), most = M / (8 * groups);
        const int64_t p = want < most ? want : most;
        return (int)(p < 1 ? 1 : p > 512 ? 512 : p);
    }
    int64_t want = ceil_div(4096, ceil_div(N, LN_NT) * groups), most = M / (32 * groups);
    int64_t p = want < most ? want : most;
    return (int)(p < 1 ? 1 : p > 256 ? 256 : p);
}

// Tiles of dW: N and K extents, and the parts of the rows.  Wide ones where
// the operands allow it, a part keeps 256 rows and they are 64 or more (bf16,
// us, other tiles and wide ones: 256 x 256 over 16384 rows 34, 30; 1024 x 1024
// over 1024 rows 33, 31, over 4096 68, 42); 64 x 64 where 128 x 128
// would leave CUs idle.
struct OuterPlan {
    int tn, tk, parts;
    bool wide;
    int64_t tiles;
};

OuterPlan outer_plan(const fl_linear *op) {
    OuterPlan p{};
    const auto fill = [&](int tn, int tk) {
        p.tn = tn;
        p.tk = tk;
        p.tiles = ceil_div(op->N, tn) * ceil_div(op->K, tk);
    };
    // d is contiguous [M, N], on a 256-byte boundary of the workspace or the caller's gradient
    if (op->dtype != FL_F32 && aligned(nullptr, op->N) && aligned(op->x, op->ldx) && op->K % 8 == 0 && op->N >= 192 &&
        op->K >= 192) {
        fill(256, 256);
        p.parts = outer_parts(op->M, op->groups, p.tiles, 256);
        p.wide = p.tiles * op->groups * p.parts >= 64;
        if (p.wide) return p;
    }
    if (op->groups == 1) {
        const Cut c = best_cut(op->N, op->K, op->M, op->dtype == FL_F32, false);
        const int t = c.rows == 128 && op->N >= 2 && op->K >= 2 ? 128 : 64;
        fill(t, t);
        p.parts = c.parts;
        return p;
    }
    fill(128, 128);
    if (op->N < 128 || op->K < 128 || p.tiles * op->groups < 384) fill(64, 64);
    p.parts = outer_parts(op->M, op->groups, p.tiles < 1 ? 1 : p.tiles, 1024);
    return p;
}

int check_op(const fl_linear *op, const char *what) {
    if (!op) return fl_fail(FL_ERR_ARG, "%s: null operator", what);
    if (op->dtype < FL_F32 || op->dtype > FL_F16) return fl_fail(FL_ERR_ARG, "%s: unknown type", what);
    if (op->act < FL_ACT_NONE || op->act > FL_ACT_SIGMOID)
        return fl_fail(FL_ERR_ARG, "%s: unknown activation", what);
    if (op->M < 0 || op->N < 0 || op->K < 0 || op->groups < 1 || op->M > 0x7fffffffll || op->N > 0x7fffffffll ||
        op->K > 0x7fffffffll)
        return fl_fail(FL_ERR_ARG, "%s: bad shape", what);
    if (op->offsets ? op->M > 0 && (!op->order || !op->tiles) : op->groups != 1)
        return fl_fail(FL_ERR_ARG, "%s: several groups need the plan of their rows", what);
    return FL_OK;
}

template <typename T>
int forward(hipStream_t st, const fl_linear *op, void *y, float *pre, float *ws) {
    RowsArgs a{};
    a.a = op->x;
    a.lda = op->ldx;
    a.b = op->weight;
    a.ldb = op->ldw;
    a.b_group = op->w_group;
    a.c = y;
    a.ldc = op->N;
    a.M = op->M;
    a.N = op->N;
    a.K = op->K;
    a.groups = op->groups;
    a.order = op->order;
    a.offsets = op->offsets;
    a.tiles = op->tiles;
    a.bias = op->bias;
    a.bias_group = op->N;
    a.bias_f32 = op->bias_f32;
    a.residual = op->residual;
    a.ldres = op->ldres;
    a.pre = pre;
    a.act = op->act;
    return launch_rows<T, true>(st, op, a, ws, "linear_forward");
}

template <typename T>
int input_grad(hipStream_t st, const fl_linear *op, const void *d, void *dx, float *ws) {
    RowsArgs a{};
    a.a = d;
    a.lda = op->N;
    a.b = op->weight;
    a.ldb = op->ldw;
    a.b_group = op->w_group;
    a.c = dx;
    a.ldc = op->K;
    a.M = op->M;
    a.N = op->K;
    a.K = op->N;
    a.groups = op->groups;
    a.order = op->order;
    a.offsets = op->offsets;
    a.tiles = op->tiles;
    return launch_rows<T, false>(st, op, a, ws, "linear_backward");
}

template <typename T>
int weight_grad(hipStream_t st, const fl_linear *op, const void *d, void *dw, float *ws) {
    OuterArgs a{};
    OuterPlan p = outer_plan(op);
    if (p.wide && (uintptr_t)d % 16) return fl_fail(FL_ERR_ARG, "linear_backward: gy must be 16-byte aligned");
    a.d = d;
    a.x = op->x;
    a.ldd = op->N;
    a.ldx = op->ldx;
    a.M = op->M;
    a.N = op->N;
    a.K = op->K;
    a.groups = op->groups;
    a.n_tiles = (uint32_t)ceil_div(op->N, p.tn);
    a.k_tiles = (uint32_t)ceil_div(op->K, p.tk);
    a.parts = (uint32_t)p.parts;
    a.order = op->order;
    a.offsets = op->offsets;
    a.dw = dw;
    a.part = a.parts > 1 ? ws : nullptr;
    const int64_t grid = p.tiles * a.parts * a.groups;
    if (!launch_fits(grid, p.wide ? WD_NT : LN_NT))
        return fl_fail(FL_ERR_ARG, "linear_backward: too many tiles for one launch (shape)");
    if (grid == 0) return FL_OK;
    constexpr int BIG_K = sizeof(T) == 4 ? 32 : 64;
    const dim3 g((unsigned)grid), nt(LN_NT);
    if constexpr (sizeof(T) == 2) {
        if (p.wide && a.order)
            FL_LAUNCH("k_wide_outer", (k_wide_outer<T, true, 64, 2>), g, dim3(WD_NT), wide_bytes(256, 64, 2), st, a);
        else if (p.wide)
            FL_LAUNCH("k_wide_outer", (k_wide_outer<T, false, 64, 2>), g, dim3(WD_NT), wide_bytes(256, 64, 2), st, a);
    }
    if (p.wide) {
    } else if (p.tn == 128) FL_LAUNCH("k_lin_outer", (k_lin_outer<T, 128, 128, BIG_K>), g, nt, 0, st, a);
    else FL_LAUNCH("k_lin_outer", (k_lin_outer<T, 64, 64, BIG_K>), g, nt, 0, st, a);
    if (a.part) fold_parts<T>(st, ws, (int)a.parts, a.groups * a.N * a.K, (T *)dw);
    return fl_check_launch("linear_backward");
}

template <typename T>
int bias_grad(hipStream_t st, const fl_linear *op, const void *gy, const float *pre, const void *d, void *db,
              int db_f32, float *ws) {
    const int parts = sum_parts(op);
    const int64_t grid = (int64_t)parts * op->groups * ceil_div(op->N, LN_NT);
    if (!launch_fits(grid, LN_NT))
        return fl_fail(FL_ERR_ARG, "linear_bias_grad: too many groups for one launch (shape)");
    const dim3 g((unsigned)grid), nt(LN_NT);
    if (sizeof(T) == 2 && op->act != FL_ACT_NONE)
        FL_LAUNCH("k_col_sums", (k_col_sums<T, true>), g, nt, 0, st, (const T *)gy, pre, op->act, op->M, op->N,
                  op->groups, parts, op->order, op->offsets, ws);
    else
        FL_LAUNCH("k_col_sums", (k_col_sums<T, false>), g, nt, 0, st, (const T *)d, pre, op->act, op->M, op->N,
                  op->groups, parts, op->order, op->offsets, ws);
    if (db_f32) fold_parts<float>(st, ws, parts, op->groups * op->N, (float *)db);
    else fold_parts<T>(st, ws, parts, op->groups * op->N, (T *)db);
    return fl_check_launch("linear_bias_grad");
}

template <typename T>
int act_and_bias_grad(hipStream_t st, const fl_linear *op, const void *gy, const float *pre, void *d, void *db,
                      int db_f32, float *ws) {
    const int parts = sum_parts(op);
    const int64_t grid = parts * op->groups * ceil_div(op->N, AS_COLS);
    if (!launch_fits(grid, LN_NT))
        return fl_fail(FL_ERR_ARG, "linear_backward: too many columns or groups for one launch (shape)");
    const dim3 g((unsigned)grid), nt(LN_NT);
    if (op->offsets)
        FL_LAUNCH("k_act_sums", (k_act_sums<T, true>), g, nt, 0, st, (const T *)gy, pre, op->M, op->N, op->groups,
                  parts, op->act, op->order, op->offsets, (T *)d, ws);
    else
        FL_LAUNCH("k_act_sums", (k_act_sums<T, false>), g, nt, 0, st, (const T *)gy, pre, op->M, op->N, op->groups,
                  parts, op->act, op->order, op->offsets, (T *)d, ws);
    if (db_f32) fold_parts<float>(st, ws, parts, op->groups * op->N, (float *)db);
    else fold_parts<T>(st, ws, parts, op->groups * op->N, (T *)db);
    return fl_check_launch("linear_backward");
}

template <typename T>
int act_grad(hipStream_t st, int act, const void *gy, const float *pre, int64_t n, void *d) {
    const int64_t grid = ceil_div(n, LN_NT * 4);
    if (!launch_fits(grid, LN_NT))
        return fl_fail(FL_ERR_ARG, "linear_backward: too many values for one launch (shape)");
    FL_LAUNCH("k_act_grad", k_act_grad<T>, dim3((unsigned)grid), dim3(LN_NT), 0, st, (const T *)gy, pre, n, act,
              (T *)d);
    return fl_check_launch("linear_backward");
}

// The backward's workspace: d (when there is an activation), and the parts of
// dx, dW and db, one after the other in the same place.
struct BackwardSpace {
    size_t d, parts, bytes;
};

BackwardSpace backward_space(const fl_linear *op, int with_dx, int with_dw, int with_db) {
    BackwardSpace s{0, 0, 0};
    const auto take = [&](size_t n) {
        const size_t at = s.bytes;
        s.bytes += (n + 255) / 256 * 256;
        return at;
    };
    if (op->act != FL_ACT_NONE) s.d = take((size_t)op->M * op->N * (op->dtype == FL_F32 ? 4 : 2));
    size_t most = 0;
    const auto need = [&](size_t n) { most = n > most ? n : most; };
    if (with_dx && op->M && op->K) need(rows_bytes(op, op->K, op->N));
    if (with_dw && op->N && op->K) {
        const int parts = outer_plan(op).parts;
        if (parts > 1) need((size_t)parts * op->groups * op->N * op->K * 4);
    }
    if (with_db && op->N) need((size_t)sum_parts(op) * op->groups * op->N * 4);
    s.parts = take(most);
    return s;
}

template <typename T>
int backward(hipStream_t st, const fl_linear *op, const void *gy, const float *pre, void *dx, void *dw, void *db,
             int db_f32, char *ws) {
    const BackwardSpace s = backward_space(op, dx != nullptr, dw != nullptr, db != nullptr);
    float *parts = (float *)(ws + s.parts);
    const void *d = gy;
    int rc = FL_OK;
    const bool both = db && act_and_sums(op) && op->M;
    if (op->act != FL_ACT_NONE && op->M && op->N) {
        d = ws + s.d;
        if (both) rc = act_and_bias_grad<T>(st, op, gy, pre, ws + s.d, db, db_f32, parts);
        else rc = act_grad<T>(st, op->act, gy, pre, op->M * op->N, ws + s.d);
    }
    if (!rc && dx && op->M && op->K) rc = input_grad<T>(st, op, d, dx, parts);
    if (!rc && dw && op->N && op->K) rc = weight_grad<T>(st, op, d, dw, parts);
    if (!rc && db && op->N && !both) rc = bias_grad<T>(st, op, gy, pre, d, db, db_f32, parts);
    return rc;
}

}  // namespace
}  // namespace fl

#define FL_BY_TYPE(dtype, call)                     \
    switch (dtype) {                                \
        case FL_F32: { using T = float; return call; }    \
        case FL_BF16: { using T = __bf16; return call; }  \
        default: { using T = _Float16; return call; }     \
    }

extern "C" {

size_t fl_linear_op_bytes(void) { return sizeof(fl_linear); }

size_t fl_linear_forward_bytes(const fl_linear *op) {
    if (!op || op->M < 1 || op->N < 1 || op->K < 0 || op->groups < 1) return 0;
    return fl::rows_bytes(op, op->N, op->K);
}

int fl_linear_forward(void *stream, const fl_linear *op, void *y, float *pre, void *ws, size_t ws_bytes) {
    const int rc = fl::check_op(op, "linear_forward");
    if (rc) return rc;
    if (op->M == 0 || op->N == 0) return FL_OK;
    if (!y || (op->K > 0 && (!op->x || !op->weight)))
        return fl::fl_fail(FL_ERR_ARG, "linear_forward: null pointer");
    const size_t need = fl_linear_forward_bytes(op);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "linear_forward: workspace too small");
    FL_BY_TYPE(op->dtype, fl::forward<T>((hipStream_t)stream, op, y, pre, (float *)ws))
}

size_t fl_linear_backward_bytes(const fl_linear *op, int with_dx, int with_dw, int with_db) {
    if (!op || op->M < 0 || op->N < 0 || op->K < 0 || op->groups < 1) return 0;
    return fl::backward_space(op, with_dx, with_dw, with_db).bytes;
}

int fl_linear_backward(void *stream, const fl_linear *op, const void *gy, const float *pre, void *dx, void *dw,
                       void *db, int db_f32, void *ws, size_t ws_bytes) {
    const int rc = fl::check_op(op, "linear_backward");
    if (rc) return rc;
    const bool any = op->M > 0 && op->N > 0;
    if ((any && (!gy || (op->act != FL_ACT_NONE && !pre))) || (any && dx && op->K > 0 && !op->weight) ||
        (any && dw && op->K > 0 && !op->x))
        return fl::fl_fail(FL_ERR_ARG, "linear_backward: null pointer");
    const size_t need = fl_linear_backward_bytes(op, dx != nullptr, dw != nullptr, db != nullptr);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "linear_backward: workspace too small");
    if ((uintptr_t)ws % 16) return fl::fl_fail(FL_ERR_ARG, "linear_backward: workspace must be 16-byte aligned");
    FL_BY_TYPE(op->dtype, fl::backward<T>((hipStream_t)stream, op, gy, pre, dx, dw, db, db_f32, (char *)ws))
}

}  // extern "C"
