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
#include "fl_product.h"

namespace fl {
namespace {

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
