// The losses of rows that are a product z = x W^T + b, which is not kept: the
// forward joins the tiles' maxima and sums of exponentials, and the backward
// makes the tiles again with dz in place of z, for a piece of the vocabulary at
// a time (fl_loss.hip has the formulas):
//
//   dx = dz W      dW = dz^T x      db = sum over the rows of dz
//
// The piece of dz is what a call holds of [rows x vocabulary], in 16 bits (an
// operand of two products; fp32: as it is or in three bfloat16 planes).  The
// listed columns' own u comes from a dot product each; their entries of dz are
// made apart, since p - q of values rounded before would keep few bits where p is
// near 1.
//
// Bound by the matrix instructions: four products where logits that are kept
// would need three, beside 2 or 4 bytes of dz a logit written once and read twice.
// Small products go by k_vocab_*, the others, and bfloat16 in training, by k_wide_*:
// tiles one after the other, so that the loads of a tile begin while the one
// before it is finished.  There fp32 operands are laid out as their three bfloat16
// planes, and 16-bit rows that do not lie on 16 bytes as copies that do.
#include "fl_abi.h"
#include "fl_common.h"
#include "fl_loss.h"
#include "fl_product.h"
#include <type_traits>

namespace fl {
namespace {

constexpr int LS_NT = 256;
constexpr int LS_WAVES = LS_NT / FL_WAVE;
// Bytes of dz: with 128 MB, which the last level cache holds, [8192 x 512 -> 41000]
// bf16 train takes 1850 us, with 512 MB and 1 GB 1640 ([512 x 128 -> 4.6M] 6480,
// 6460 and 6100): fewer beginnings and ends of kernels.
constexpr size_t LS_PIECE = 1u << 30;

// The wide kernels' dz lies in blocks of so many columns, each row of a block
// behind the one before it: a tile's rows are one piece of memory.
constexpr int D_BLOCK = 256;

struct VocabArgs {
    fl_vocab op;
    float scale;          // log2(e) / tau
    // the vocabulary's piece [v0, v0 + width)
    int64_t v0, width;
    uint32_t m_tiles, n_tiles, parts;
    Running *part;        // [M][parts]
    const float2 *rows;
    float2 *listed;
    const float *coef;    // tau g of every row, 0 where it has no gradient; over a power of two where dz is half:
    const float *factor;  // that power, or null
    void *d;              // dz of the piece: [M][ldd], wide: blocks of D_BLOCK columns, [d_rows][ldd] each
    int64_t ldd, d_block;  // d_block: from one to the next
    int64_t dz_rows;      // rows of dz: M, or 2 M where the second M are what rounding left of the first
    float *sums;          // dx: [parts][dz_rows][K]; dW: [parts][width][K]
    void *dw;
    void *dx;             // where one part and one piece are all of it
    // x as dW takes it, and the exponent of what undoes its power of two, or null
    const void *y;
    int64_t ldy;
    const int *y_exp;
    int add;
    // wide kernels: operands laid out (or as they are), their columns and dz's with those that pad them to whole steps
    // (dz: 0 there, and in the rows that pad it), and what undoes the powers of two of x's rows and of weight (or null)
    const uint16_t *x, *w;
    int64_t ldx, ldw, cols, d_cols, d_rows;
    const float *undo_x, *undo_w;
};

// u of four listed ids of a row (-1: none), by one wave; the same in all lanes.
// Four rows of the weight at once, since a wave's gathered rows are bound by the
// time of a load: 4096 x 64 ids of 1024 fp16 values in 74 us, 7.2 TB/s of the
// weight from the caches.
constexpr int DOT_IDS = 4;

template <typename T>
__device__ __forceinline__ void dots(const VocabArgs &a, int64_t row, const int64_t (&id)[DOT_IDS],
                                     float (&s)[DOT_IDS]) {
    const int64_t K = a.op.K;
    const T *x = (const T *)a.op.x + row * a.op.ldx;
    const T *w[DOT_IDS];
#pragma unroll
    for (int i = 0; i < DOT_IDS; ++i) {
        s[i] = 0.0f;
        w[i] = (const T *)a.op.weight + (id[i] < 0 ? 0 : id[i]) * a.op.ldw;
    }
    int64_t c = fl_lane() * 8;
    for (; c + 8 <= K; c += FL_WAVE * 8) {
        const Vec<T, 8> xv = load_vec<T, 8>(x + c);
        Vec<T, 8> wv[DOT_IDS];
#pragma unroll
        for (int i = 0; i < DOT_IDS; ++i) wv[i] = load_vec<T, 8>(w[i] + c);
#pragma unroll
        for (int i = 0; i < DOT_IDS; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[i] = __builtin_fmaf((float)xv.v[e], (float)wv[i].v[e], s[i]);
    }
    for (int64_t e = c; e < K && e < c + 8; ++e)
#pragma unroll
        for (int i = 0; i < DOT_IDS; ++i) s[i] = __builtin_fmaf((float)x[e], (float)w[i][e], s[i]);
#pragma unroll
    for (int i = 0; i < DOT_IDS; ++i) {
        float b = 0.0f;
        if (a.op.bias && id[i] >= 0)
            b = a.op.bias_f32 ? ((const float *)a.op.bias)[id[i]] : (float)((const T *)a.op.bias)[id[i]];
        s[i] = (fl_wave_sum_f32(s[i]) + b) * a.scale;
    }
}
__device__ __forceinline__ void ids_of(const VocabArgs &a, int64_t row, int64_t j0, int64_t (&id)[DOT_IDS]) {
#pragma unroll
    for (int i = 0; i < DOT_IDS; ++i) {
        id[i] = j0 + i < a.op.lists.k ? a.op.lists.ids[row * a.op.lists.k + j0 + i] : -1;
        if (id[i] >= a.op.V) id[i] = -1;
    }
}

// A wave a row and four of its ids.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_vocab_dots(VocabArgs a) {
    const int64_t k = a.op.lists.k, quads = (k + DOT_IDS - 1) / DOT_IDS;
    const int64_t item = fl_block() * LS_WAVES + fl_wave_id();
    if (item >= a.op.M * quads) return;
    const int64_t row = item / quads, j0 = item % quads * DOT_IDS;
    int64_t id[DOT_IDS];
    float s[DOT_IDS];
    ids_of(a, row, j0, id);
    dots<T>(a, row, id, s);
#pragma unroll
    for (int i = 0; i < DOT_IDS; ++i)
        if (fl_lane() == i && j0 + i < k) a.listed[row * k + j0 + i] = float2{s[i], 0.0f};
}

// The rows' sums, dots and losses in one, for lists of up to four ids (a launch
// less): a wave a row.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_vocab_rows(VocabArgs a, ListArgs l) {
    __shared__ float2 lists[LS_WAVES][DOT_IDS];
    const int64_t row = fl_block() * LS_WAVES + fl_wave_id();
    if (row >= a.op.M) return;
    const Running r = joined_parts(a.part + row * a.parts, a.parts, 0, 1, 1.0f);
    int64_t id[DOT_IDS];
    float s[DOT_IDS];
    ids_of(a, row, 0, id);
    dots<T>(a, row, id, s);
    list_row(l, row, r, lists[fl_wave_id()], [&](int64_t j, int64_t) {
        return j == 0 ? s[0] : j == 1 ? s[1] : j == 2 ? s[2] : s[3];
    });
}

// Planes of a value in the wide kernels' operands, and what they and dz are; dz in
// the others.
template <typename T>
constexpr int planes_of() {
    return sizeof(T) == 4 ? 3 : 1;
}
template <typename T>
using WideDz = typename std::conditional<sizeof(T) == 4, __bf16, _Float16>::type;
template <typename T>
using PlainDz = typename std::conditional<sizeof(T) == 4, float, _Float16>::type;

// Where the wide kernels' dz of row m and column c (of the piece) is; of three
// planes the first one's, the others are each 32 values behind the one before.
template <int P>
__device__ __forceinline__ int64_t dz_at(const VocabArgs &a, int64_t m, int64_t c) {
    const int in = (int)(c % D_BLOCK);
    return c / D_BLOCK * a.d_block + m * a.ldd + (P == 1 ? in : plane_at(in));
}

// The logits of a lane's tiles in units of log 2, -inf behind the vocabulary:
// f(i, j, u[4]) of the row i * 16 + (lane & 15) and four columns from
// col + j * 16 + (lane >> 4) * 4 on, both within the wave's part of the tile.
template <typename T, int MT, int NTL, typename F>
__device__ __forceinline__ void each_u(const VocabArgs &a, const f32x4 (&acc)[MT][NTL], int64_t col, int64_t end,
                                       F &&f) {
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
        const int64_t n = col + j * 16 + (fl_lane() >> 4) * 4;
        const int have = end - n < 0 ? 0 : end - n < 4 ? (int)(end - n) : 4;
        float b[4] = {0, 0, 0, 0};
        if (a.op.bias) {
            if (a.op.bias_f32) load_some<float>((const float *)a.op.bias + n, have, b);
            else load_some<T>((const T *)a.op.bias + n, have, b);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            float u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = e < have ? (acc[i][j][e] + b[e]) * a.scale : -INFINITY;
            f(i, j, u);
        }
    }
}

// Joins the lanes' sums of a wave's rows and the waves' of a tile's columns,
// and stores them as one part of the rows.
template <int BM, int WAVES_N, int MT>
__device__ __forceinline__ void store_running(const VocabArgs &a, Running (&r)[MT], Running *lds, int wave_row,
                                              int wave_col, int64_t row0, uint32_t part) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        r[i] = joined(r[i], Running{__shfl_xor(r[i].m, 16), __shfl_xor(r[i].s, 16)});
        r[i] = joined(r[i], Running{__shfl_xor(r[i].m, 32), __shfl_xor(r[i].s, 32)});
        if (fl_lane() < 16) lds[wave_col * BM + wave_row + i * 16 + fl_lane()] = r[i];
    }
    __syncthreads();
    for (int t = threadIdx.x; t < BM; t += blockDim.x) {
        Running s = lds[t];
#pragma unroll
        for (int w = 1; w < WAVES_N; ++w) s = joined(s, lds[w * BM + t]);
        if (row0 + t < a.op.M) a.part[(row0 + t) * a.parts + part] = s;
    }
}

// The rows' running maxima and sums over a part of the vocabulary's tiles, a pair a
// row and part.  Bound by a step's load time where there are few tiles: fp32
// [96 x 256 -> 475] 7.7 us; by the fp32 planes' six products and LDS reads where
// there are many: [128 x 256 -> 41000] 28 us = 96 TFLOP/s.
template <typename T, int BM, int BN, int BK>
__global__ __launch_bounds__(LN_NT) void k_vocab_stats(VocabArgs a) {
    using Prod = Product<T, BM, BN, BK>;
    __shared__ __align__(16) uint16_t lds[Prod::LDS_ELEMS];
    __shared__ Running join[Prod::WAVES_N * BM];
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const uint32_t mt = w % a.m_tiles, part = w / a.m_tiles;
    const int64_t row0 = (int64_t)mt * BM, V = a.op.V;
    const int64_t t0 = (int64_t)a.n_tiles * part / a.parts, t1 = (int64_t)a.n_tiles * (part + 1) / a.parts;
    Running r[Prod::MT];
#pragma unroll
    for (int i = 0; i < Prod::MT; ++i) r[i] = Running{-INFINITY, 0.0f};
    Prod prod;
    for (int64_t t = t0; t < t1; ++t) {
        const int64_t n0 = t * BN;
        ContigTile<T, BM, BK> ta;
        ContigTile<T, BN, BK> tb;
        ta.init([&](int i) { return (const T *)a.op.x + (row0 + i < a.op.M ? row0 + i : a.op.M - 1) * a.op.ldx; });
        tb.init([&](int i) { return (const T *)a.op.weight + (n0 + i < V ? n0 + i : V - 1) * a.op.ldw; });
        prod.run(ta, tb, a.op.K, lds);
        __syncthreads();
        float u[Prod::MT][Prod::NTL * 4];
        each_u<T>(a, prod.acc, n0 + prod.wave_n(), V, [&](int i, int j, const float (&v)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) u[i][j * 4 + e] = v[e];
        });
#pragma unroll
        for (int i = 0; i < Prod::MT; ++i) {
            float m = r[i].m, s = 0.0f;
#pragma unroll
            for (int e = 0; e < Prod::NTL * 4; ++e) m = fmaxf(m, u[i][e]);
            const float at = base_of(m);
#pragma unroll
            for (int e = 0; e < Prod::NTL * 4; ++e) s += exp2_of(u[i][e] - at);
            r[i] = Running{m, r[i].s * exp2_of(r[i].m - at) + s};
        }
    }
    store_running<BM, Prod::WAVES_N>(a, r, join, prod.wave_m(), prod.wave_n() / (BN / Prod::WAVES_N), row0, part);
}

// What a row's dz is multiplied by.
__global__ __launch_bounds__(1024) void k_vocab_coef(const float2 *__restrict__ rows, const float *__restrict__ g,
                                                     float tau, int64_t M, float *__restrict__ coef) {
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < M; i += (int64_t)gridDim.x * 1024)
        coef[i] = rows[i].y != 0.0f ? tau * g[i] : 0.0f;
}

// Where dz is half: a row's tau g as a number of 2^14..2^15, which its dz is multiplied
// by, and a power of two, which its row of dx, its terms of db and its row of dW's
// other operand are multiplied by.  So what half can hold is that of p - q, 2^-39
// absolute, in every row, whatever the rows' gradients are to each other.  A wave a
// row, [8192 x 512] bf16 5.7 us; most: the largest exponent of a workgroup's rows of x
// times that power.
constexpr int LAY_PARTS = 1024;
constexpr int NO_EXP = -(1 << 20);

template <typename T>
__global__ __launch_bounds__(LS_NT) void k_row_scale(VocabArgs a, const float *__restrict__ g, float tau, int with_y,
                                                     float *__restrict__ coef, float *__restrict__ factor,
                                                     int *__restrict__ most) {
    __shared__ int waves[LS_WAVES];
    int top = NO_EXP;
    for (int64_t r = (int64_t)blockIdx.x * LS_WAVES + fl_wave_id(); r < a.op.M; r += (int64_t)gridDim.x * LS_WAVES) {
        float c = a.rows[r].y != 0.0f ? tau * g[r] : 0.0f;
        int e = 15;
        const bool some = c != 0.0f && fabsf(c) < INFINITY;
        if (some) {
            frexpf(c, &e);  // |c| < 2^e
            e = e < -110 ? -110 : e;
            c = ldexpf(c, 15 - e);
        }
        if (fl_lane() == 0) {
            coef[r] = c;
            factor[r] = ldexpf(1.0f, e - 15);
        }
        if (!with_y || !some) continue;
        const T *x = (const T *)a.op.x + r * a.op.ldx;
        float m = 0.0f;
        const auto see = [&](T v) {
            const float t = fabsf((float)v);
            m = fmaxf(m, t < INFINITY ? t : 0.0f);
        };
        for (int64_t k = fl_lane() * 8; k < a.op.K; k += FL_WAVE * 8) {
            if (k + 8 <= a.op.K) {
                const Vec<T, 8> v = load_vec<T, 8>(x + k);
#pragma unroll
                for (int i = 0; i < 8; ++i) see(v.v[i]);
            } else
                for (int64_t i = k; i < a.op.K; ++i) see(x[i]);
        }
#pragma unroll
        for (int o = FL_WAVE / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        int xe;
        frexpf(m, &xe);
        if (m > 0.0f && xe + e - 15 > top) top = xe + e - 15;
    }
    if (fl_lane() == 0) waves[fl_wave_id()] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < LS_WAVES; ++w) top = waves[w] > top ? waves[w] : top;
        most[blockIdx.x] = top;
    }
}

// dW's other operand in half: rows of x times their power of two and one of all rows,
// which brings the largest value to 2^13..2^14; 0 in rows without a gradient.
// HBM-bound: [8192 x 512] bf16 6.6 us.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_lay_y(VocabArgs a, const int *__restrict__ most, int parts,
                                                 _Float16 *__restrict__ y, int *__restrict__ y_exp) {
    __shared__ int waves[LS_WAVES];
    int top = NO_EXP;
    for (int i = threadIdx.x; i < parts; i += LS_NT) top = most[i] > top ? most[i] : top;
#pragma unroll
    for (int o = FL_WAVE / 2; o > 0; o >>= 1) {
        const int t = __shfl_xor(top, o);
        top = t > top ? t : top;
    }
    if (fl_lane() == 0) waves[fl_wave_id()] = top;
    __syncthreads();
    for (int w = 0; w < LS_WAVES; ++w) top = waves[w] > top ? waves[w] : top;
    if (top == NO_EXP) top = 14;
    if (blockIdx.x == 0 && threadIdx.x == 0) *y_exp = top - 14;
    const int64_t chunks = a.ldy / 8;
    for (int64_t i = (int64_t)blockIdx.x * LS_NT + threadIdx.x; i < a.op.M * chunks; i += (int64_t)gridDim.x * LS_NT) {
        const int64_t r = i / chunks, c = i % chunks * 8, have = a.coef[r] != 0.0f ? a.op.K : 0;
        const T *x = (const T *)a.op.x + r * a.op.ldx;
        Vec<T, 8> v;
        if (c + 8 <= have) v = load_vec<T, 8>(x + c);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = c + e < have ? x[c + e] : (T)0.0f;
        int e;
        frexpf(a.factor[r], &e);  // its power plus 1
        Vec<_Float16, 8> o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o.v[k] = (_Float16)ldexpf((float)v.v[k], e - 1 + 14 - top);
        store_vec<_Float16, 8>(y + r * a.ldy + c, o);
    }
}

// A value of dW from its sum.
template <typename T>
__device__ __forceinline__ T dw_of(float sum, int y_exp) {
    return (T)(sizeof(T) == 2 ? ldexpf(sum, y_exp) : sum);
}

// dz of a piece but for the listed columns: the product again, an exponential in
// place of the sums.  fp32 [128 x 256 -> 41000] 32 us, bound as k_vocab_stats.
template <typename T, int BM, int BN, int BK>
__global__ __launch_bounds__(LN_NT) void k_vocab_grad(VocabArgs a) {
    using Prod = Product<T, BM, BN, BK>;
    __shared__ __align__(16) uint16_t lds[Prod::LDS_ELEMS];
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const int64_t row0 = (int64_t)(w % a.m_tiles) * BM, n0 = a.v0 + (int64_t)(w / a.m_tiles) * BN, V = a.op.V;
    ContigTile<T, BM, BK> ta;
    ContigTile<T, BN, BK> tb;
    ta.init([&](int i) { return (const T *)a.op.x + (row0 + i < a.op.M ? row0 + i : a.op.M - 1) * a.op.ldx; });
    tb.init([&](int i) { return (const T *)a.op.weight + (n0 + i < V ? n0 + i : V - 1) * a.op.ldw; });
    Prod prod;
    prod.run(ta, tb, a.op.K, lds);
    const int64_t row = row0 + prod.wave_m() + (fl_lane() & 15), col = n0 + prod.wave_n();
    float top[Prod::MT], c[Prod::MT];  // c: times the sum's reciprocal
#pragma unroll
    for (int i = 0; i < Prod::MT; ++i) {
        const int64_t m = row + i * 16 < a.op.M ? row + i * 16 : a.op.M - 1;
        const float2 sum = a.rows[m];
        top[i] = sum.x;
        c[i] = a.coef[m] * sum.y;
    }
    each_u<T>(a, prod.acc, col, a.v0 + a.width, [&](int i, int j, const float (&u)[4]) {
        const int64_t n = col + j * 16 + (fl_lane() >> 4) * 4 - a.v0;
        if (row + i * 16 >= a.op.M || n >= a.ldd) return;
        using D = PlainDz<T>;
        Vec<D, 4> o, rest;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float d = c[i] == 0.0f ? 0.0f : c[i] * exp2_of(u[e] - top[i]);
            o.v[e] = (D)d;
            rest.v[e] = (D)(d - (float)o.v[e]);
        }
        store_vec<D, 4>((D *)a.d + (row + i * 16) * a.ldd + n, o);
        if (a.dz_rows > a.op.M) store_vec<D, 4>((D *)a.d + (a.op.M + row + i * 16) * a.ldd + n, rest);
    });
}

// A listed column's p from its u and the row's sums, 1 at most (its product is not the
// one in the sums: where logits are so large that their rounding passes 1, it could be
// anything above, and nothing that half holds).
__device__ __forceinline__ float listed_share(float u, float2 sum) {
    const float p = exp2_of(u - sum.x) * sum.y;
    return p > 1.0f ? 1.0f : p;
}

// dz of the listed columns in the piece: scattered stores of 2 or 4 bytes, 4096 x 64
// of them 12.5 us.
template <typename T, bool WIDE>
__global__ __launch_bounds__(LS_NT) void k_vocab_listed(VocabArgs a) {
    const int64_t i = fl_block() * LS_NT + threadIdx.x, k = a.op.lists.k;
    if (i >= a.op.M * k) return;
    const int64_t row = i / k, v = a.op.lists.ids[i] - a.v0;
    const float c = a.coef[row];
    if (v < 0 || v >= a.width || c == 0.0f) return;
    const float2 l = a.listed[i];
    const float d = c * (listed_share(l.x, a.rows[row]) - l.y);
    if constexpr (WIDE && sizeof(T) == 4) {
        const float chunk[8] = {d, 0, 0, 0, 0, 0, 0, 0};
        u32x4 plane[3];
        chunk_planes<float>(chunk, plane);
        uint16_t *to = (uint16_t *)a.d + dz_at<3>(a, row, v);
#pragma unroll
        for (int p = 0; p < 3; ++p) to[p * 32] = (uint16_t)plane[p][0];
    } else if constexpr (WIDE) ((_Float16 *)a.d)[dz_at<1>(a, row, v)] = (_Float16)d;
    else {
        using D = PlainDz<T>;
        const D o = (D)d;
        ((D *)a.d)[row * a.ldd + v] = o;
        if (a.dz_rows > a.op.M) ((D *)a.d)[(a.op.M + row) * a.ldd + v] = (D)(d - (float)o);
    }
}

// A piece's part of dx, added to what is there if `add`: the vocabulary is the long
// axis and is cut into parts.  fp32 [128 x 256 -> 41000] 35 us in 256 workgroups (46
// in 160, of at least 512 columns each).
template <typename T, int BM, int BN, int BK>
__global__ __launch_bounds__(LN_NT) void k_vocab_dx(VocabArgs a) {
    using Prod = Product<T, BM, BN, BK>;
    __shared__ __align__(16) uint16_t lds[Prod::LDS_ELEMS];
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const uint32_t tile = w / a.parts, part = w % a.parts;
    const int64_t row0 = (int64_t)(tile / a.n_tiles) * BM, n0 = (int64_t)(tile % a.n_tiles) * BN, M = a.dz_rows;
    const int64_t steps = (a.width + BK - 1) / BK, k0 = steps * part / a.parts * BK;
    const int64_t k1 = part + 1 == a.parts ? a.width : steps * (part + 1) / a.parts * BK;
    ContigTile<T, BM, BK> ta;
    StridedTile<T, BN, BK> tb;
    ta.init([&](int r) { return (const T *)a.d + (row0 + r < M ? row0 + r : M - 1) * a.ldd + k0; });
    tb.init((const T *)a.op.weight + (a.v0 + k0) * a.op.ldw + n0, a.op.ldw, a.op.K - n0, nullptr);
    Prod prod;
    prod.run(ta, tb, k1 - k0, lds);
#pragma unroll
    for (int i = 0; i < Prod::MT; ++i) {
        const int64_t row = row0 + prod.wave_m() + i * 16 + (fl_lane() & 15);
        if (row >= M) continue;
#pragma unroll
        for (int j = 0; j < Prod::NTL; ++j) {
            const int64_t n = n0 + prod.wave_n() + j * 16 + (fl_lane() >> 4) * 4;
            if (n >= a.op.K) continue;
            const int have = a.op.K - n < 4 ? (int)(a.op.K - n) : 4;
            float *q = a.sums + ((int64_t)part * M + row) * a.op.K + n;
            Vec<float, 4> f{{prod.acc[i][j][0], prod.acc[i][j][1], prod.acc[i][j][2], prod.acc[i][j][3]}};
            if (a.add) {
                float old[4];
                load_some<float>(q, have, old);
#pragma unroll
                for (int e = 0; e < 4; ++e) f.v[e] += old[e];
            }
            if (have == 4) store_vec<float, 4>(q, f);
            else store_some<float, 4>(q, f, have);
        }
    }
}

// The parts of a sum added and rounded: four values a lane, a quarter of the
// parts a wave, each in order and then the quarters.  HBM-bound: 67 MB of
// parts in 17 us.
// undo, factor (of rows of K values), exponent: what the sum is multiplied by, or null.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_vocab_fold(const float *__restrict__ part, uint32_t parts, int64_t n,
                                                      const float *__restrict__ undo,
                                                      const float *__restrict__ factor, int64_t K,
                                                      const int *__restrict__ exponent, T *__restrict__ out) {
    __shared__ float runs[LS_WAVES][4 * FL_WAVE];
    const int64_t i = (fl_block() * FL_WAVE + fl_lane()) * 4;
    const int have = n - i < 0 ? 0 : n - i < 4 ? (int)(n - i) : 4;
    float s[4] = {0, 0, 0, 0};
    uint32_t p = parts * fl_wave_id() / LS_WAVES;
    const uint32_t p1 = parts * (fl_wave_id() + 1) / LS_WAVES;
    const auto add = [&](auto many) {
        constexpr int N = decltype(many)::value;
        float v[N][4];
#pragma unroll
        for (int j = 0; j < N; ++j) load_some<float>(part + (p + j) * n + i, have, v[j]);
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += v[j][e];
        p += N;
    };
    while (p + 8 <= p1) add(std::integral_constant<int, 8>());
    while (p < p1) add(std::integral_constant<int, 1>());
#pragma unroll
    for (int e = 0; e < 4; ++e) runs[fl_wave_id()][fl_lane() * 4 + e] = s[e];
    __syncthreads();
    if (fl_wave_id() || !have) return;
    const float f = undo ? *undo : 1.0f;
    const int e2 = exponent ? *exponent : 0;
    Vec<T, 4> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int at = fl_lane() * 4 + e;
        float v = ((runs[0][at] + runs[1][at]) + (runs[2][at] + runs[3][at])) * f;
        if (factor) v *= factor[(i + (e < have ? e : 0)) / K];
        o.v[e] = (T)(exponent ? ldexpf(v, e2) : v);
    }
    if (have == 4) store_vec<T, 4>(out + i, o);
    else store_some<T, 4>(out + i, o, have);
}

// A piece's rows of dW, or of a part of the rows' sum.  fp32 [128 x 256 -> 41000]
// 40 us: four steps a tile, so that much of it is beginnings and stores.
template <typename T, int BM, int BN, int BK>
__global__ __launch_bounds__(LN_NT) void k_vocab_dw(VocabArgs a) {
    using Prod = Product<T, BM, BN, BK>;
    __shared__ __align__(16) uint16_t lds[Prod::LDS_ELEMS];
    uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const int64_t m0 = (int64_t)(w % a.m_tiles) * BM;
    w /= a.m_tiles;
    const int64_t c0 = (int64_t)(w % a.n_tiles) * BN;
    const uint32_t part = w / a.n_tiles;
    const int64_t begin = a.op.M * part / a.parts, end = a.op.M * (part + 1) / a.parts;
    StridedTile<T, BM, BK> ta;
    StridedTile<T, BN, BK> tb;
    ta.init((const T *)a.d + begin * a.ldd + m0, a.ldd, a.ldd - m0, nullptr);
    tb.init((const T *)a.y + begin * a.ldy + c0, a.ldy, a.op.K - c0, nullptr);
    Prod prod;
    prod.run(ta, tb, end - begin, lds);
    const int y_exp = a.y_exp ? *a.y_exp : 0;
#pragma unroll
    for (int i = 0; i < Prod::MT; ++i) {
        const int64_t m = m0 + prod.wave_m() + i * 16 + (fl_lane() & 15);
        if (m >= a.width) continue;
#pragma unroll
        for (int j = 0; j < Prod::NTL; ++j) {
            const int64_t c = c0 + prod.wave_n() + j * 16 + (fl_lane() >> 4) * 4;
            if (c >= a.op.K) continue;
            const int n = a.op.K - c < 4 ? (int)(a.op.K - c) : 4;
            if (a.sums) {
                float *q = a.sums + ((int64_t)part * a.width + m) * a.op.K + c;
                const Vec<float, 4> o{{prod.acc[i][j][0], prod.acc[i][j][1], prod.acc[i][j][2], prod.acc[i][j][3]}};
                if (n == 4) store_vec<float, 4>(q, o);
                else store_some<float, 4>(q, o, n);
            } else {
                T *q = (T *)a.dw + (a.v0 + m) * a.op.K + c;
                Vec<T, 4> o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o.v[e] = dw_of<T>(prod.acc[i][j][e], y_exp);
                if (n == 4) store_vec<T, 4>(q, o);
                else store_some<T, 4>(q, o, n);
            }
        }
    }
}

// dW of up to 32 KS rows, which is as good as a copy of W: HBM-bound by its stores.  A
// wave keeps x's columns of its band in registers and walks the vocabulary, 16
// columns of dz a tile, whose loads are a tile ahead.  The tile's values go through
// the wave's own LDS, so that a store takes whole rows of the band; of rows of whole
// 16 bytes nothing is masked, and lanes behind the end store what others do.  fp32 [23
// x 1152 -> 431394] 420 us = 4.7 TB/s (stores of 64 bytes of 16 rows, masked, 686;
// tiles of 128 x 128 1011), fp16 [4 x 1024 -> 400000] 167 (363; 610), bf16 [16 x 512 ->
// 200000] 46 (101; 160).  The stores of a tile are waited for with the next one's loads:
// left in flight 474 for 420, [17 x 544 -> 1001465] 583 for 510 and bf16 [60 x 512 ->
// 200000] 72 for 64, against 162 for 167, 42 for 46 and [120 x 512 -> 200000] 119 for 127.
// Up to 128 rows of 16-bit values and 64 of fp32 ([120 x 512 -> 200000] bf16 127 us,
// 189 by k_wide_dw's tiles, fp32 319 and 303).
inline int64_t few_rows(int dtype) { return dtype == FL_F32 ? 64 : 128; }
constexpr int64_t FEW_WALKS = 512;  // workgroups

template <typename T, int KS>
constexpr int few_cols() {
    return 512 / (int)sizeof(T) / KS;  // of x in registers: three planes of fp32
}

template <typename T, bool WIDE, int KS>
__global__ __launch_bounds__(LS_NT) void k_few_dw(VocabArgs a) {
    using H = typename std::conditional<WIDE, _Float16, T>::type;
    constexpr int P = Planes<H>::N, PAIR = sizeof(T) == 2 ? 2 : 1, COLS = few_cols<T, KS>(), NT = COLS / 16;
    using Out = Vec<T, 4 * PAIR>;
    constexpr int G = 4 * PAIR, PITCH = COLS + G, STORES = 16 * COLS / G / FL_WAVE;
    __shared__ __align__(16) T rows[LS_WAVES][16 * PITCH];
    T *mine = rows[fl_wave_id()];
    const int64_t M = a.dz_rows, K = a.op.K, bands = (K + COLS - 1) / COLS, tiles = (a.width + 15) / 16;
    const int64_t item = (int64_t)blockIdx.x * LS_WAVES + fl_wave_id(), runs = (int64_t)gridDim.x * LS_WAVES / bands;
    const int64_t run = item / bands, c0 = item % bands * COLS;
    if (run >= runs || run >= tiles) return;
    const int r = fl_lane() & 15, q = fl_lane() >> 4;
    const H *xs = (const H *)a.y;
    u32x4 x[KS][NT][P];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            // 16-bit tiles come in pairs whose columns alternate by fours: eight in a row a lane
            const int64_t c = c0 + (PAIR == 1 ? j * 16 + r : j / 2 * 32 + (r >> 2) * 8 + (j & 1) * 4 + (r & 3));
            // loads without branches around them, from places that there are: the compiler moved values of earlier rows to
            // other registers within the last branch, for the lanes that took it alone
            H v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t m = s * 32 + q * 8 + i, row = m < M ? m : M - 1;
                v[i] = xs[(row < a.op.M ? row : row - a.op.M) * a.ldy + (c < K ? c : K - 1)];
                if (m >= M || c >= K) v[i] = (H)0.0f;
            }
            chunk_planes<H>(v, x[s][j]);
        }
    H next[KS][8];
    const auto load = [&](int64_t t) {
        const int64_t v = t * 16 + r < a.width ? t * 16 + r : a.width - 1;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t m = s * 32 + q * 8 + i < M ? s * 32 + q * 8 + i : M - 1;
                next[s][i] = ((const H *)a.d)[WIDE ? dz_at<1>(a, m, v) : m * a.ldd + v];
            }
    };
    const int y_exp = a.y_exp ? *a.y_exp : 0;
    // the chunks of G columns that a lane stores
    const int band = (int)(K - c0 < COLS ? K - c0 : COLS), chunks = (band + G - 1) / G;
    const auto walk = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        load(run);
        for (int64_t t = run; t < tiles; t += runs) {
            if constexpr (WHOLE) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
            u32x4 d[KS][P];
#pragma unroll
            for (int s = 0; s < KS; ++s) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (s * 32 + q * 8 + i >= M) next[s][i] = (H)0.0f;
                chunk_planes<H>(next[s], d[s]);
            }
            load(t + runs < tiles ? t + runs : t);
            fl_wave_sync();
#pragma unroll
            for (int p = 0; p < NT / PAIR; ++p) {
                Vec<T, G> o;
#pragma unroll
                for (int h = 0; h < PAIR; ++h) {
                    f32x4 acc{0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        const u32x4(&b)[P] = x[s][p * PAIR + h];
                        if constexpr (P == 3) {  // smallest products first
                            acc = mfma<H>(b[2], d[s][0], acc);
                            acc = mfma<H>(b[1], d[s][1], acc);
                            acc = mfma<H>(b[0], d[s][2], acc);
                            acc = mfma<H>(b[1], d[s][0], acc);
                            acc = mfma<H>(b[0], d[s][1], acc);
                        }
                        acc = mfma<H>(b[0], d[s][0], acc);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) o.v[h * 4 + e] = dw_of<T>(acc[e], y_exp);
                }
                *reinterpret_cast<u32x4 *>(mine + r * PITCH + (p * 4 + q) * G) = __builtin_bit_cast(u32x4, o);
            }
            fl_wave_sync();
            const int have = (int)(a.width - t * 16 < 16 ? a.width - t * 16 : 16) * chunks;
            T *out = (T *)a.dw + (a.v0 + t * 16) * K + c0;
#pragma unroll
            for (int i = 0; i < STORES; ++i) {
                int at = i * FL_WAVE + fl_lane();
                if (!WHOLE && at >= have) continue;
                at = at < have ? at : have - 1;
                const int row = at / chunks, c = (at - row * chunks) * G;
                const Vec<T, G> o = __builtin_bit_cast(
                    Out, *reinterpret_cast<const u32x4 *>(mine + row * PITCH + c));
                if (WHOLE || c + G <= band) store_vec<T, G>(out + row * K + c, o);
                else store_some<T, G>(out + row * K + c, o, band - c);
            }
        }
    };
    if (K % G == 0) walk(std::true_type());
    else walk(std::false_type());
}

// Column sums of a part of the rows of dz, a thread a column: 21 MB in 7.7 us, from
// the last level cache.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_vocab_cols(VocabArgs a) {
    const int64_t blocks = (a.width + LS_NT - 1) / LS_NT, item = fl_block(), part = item / blocks;
    const int64_t c = item % blocks * LS_NT + threadIdx.x;
    if (part >= a.parts || c >= a.width) return;
    float s = 0.0f;
    for (int64_t m = a.dz_rows * part / a.parts; m < a.dz_rows * (part + 1) / a.parts; ++m) {
        const float d = (float)((const PlainDz<T> *)a.d)[m * a.ldd + c];
        s += a.factor ? d * a.factor[m < a.op.M ? m : m - a.op.M] : d;
    }
    a.sums[part * a.width + c] = s;
}

// ---------------------------------------------------------------------------
// The same for large products

// The power of two that brings m to 2^13..2^14 is 2^(14 - e).
__device__ __forceinline__ int exponent_of(float m) {
    int e;
    frexpf(m, &e);  // m < 2^e
    return e < -100 ? -100 : e;
}

// bfloat16 in training: rows of x laid out, a wave each (blockIdx.y 0), and the largest
// finite magnitude of weight, a part of it a workgroup.  HBM-bound: 1.18 GB of weight in
// 263 us = 4.5 TB/s.  A row of x is multiplied by a power of two of its own, so that rows
// of any sizes keep their bits beside each other (as operands of the logits: dW takes
// them from k_lay_y); one in which nothing is listed is zeros (padded rows may hold
// anything).
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_lay_max(VocabArgs a, float *__restrict__ most, _Float16 *__restrict__ out,
                                                   float *__restrict__ undo_x) {
    constexpr int G = 16 / (int)sizeof(T);
    __shared__ float waves[LS_WAVES];
    float m = 0.0f;
    const auto see = [&](const Vec<T, G> &v) {
#pragma unroll
        for (int e = 0; e < G; ++e) {
            const float t = fabsf((float)v.v[e]);
            m = fmaxf(m, t < INFINITY ? t : 0.0f);
        }
    };
    const auto see_row = [&](const T *row, int64_t c, int64_t step, int64_t K) {
        for (; c + 7 * step + G <= K; c += 8 * step) {
            Vec<T, G> v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = load_vec<T, G>(row + c + j * step);
#pragma unroll
            for (int j = 0; j < 8; ++j) see(v[j]);
        }
        for (; c < K; c += step) {
            Vec<T, G> v;
            if (c + G <= K) v = load_vec<T, G>(row + c);
            else
#pragma unroll
                for (int e = 0; e < G; ++e) v.v[e] = c + e < K ? row[c + e] : (T)0.0f;
            see(v);
        }
    };
    if (blockIdx.y == 0) {
        const int64_t k = a.op.lists.k;
        for (int64_t r = (int64_t)blockIdx.x * LS_WAVES + fl_wave_id(); r < a.op.M; r += LAY_PARTS * LS_WAVES) {
            bool any = false;
            for (int64_t j = fl_lane(); j < k; j += FL_WAVE) {
                const int64_t id = a.op.lists.ids[r * k + j];
                any = any || (id >= 0 && id < a.op.V);
            }
            any = __any(any);
            const T *row = (const T *)a.op.x + r * a.op.ldx;
            m = 0.0f;
            if (any) see_row(row, fl_lane() * G, FL_WAVE * G, a.op.K);
#pragma unroll
            for (int o = FL_WAVE / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
            const int e = exponent_of(m);
            const float scale = ldexpf(1.0f, 14 - e);
            if (fl_lane() == 0) undo_x[r] = ldexpf(1.0f, e - 14);
            const int64_t have = any ? a.op.K : 0;
            for (int64_t c = fl_lane() * 8; c < a.cols; c += FL_WAVE * 8) {
                Vec<T, 8> v;
                if (c + 8 <= have) v = load_vec<T, 8>(row + c);
                else
#pragma unroll
                    for (int i = 0; i < 8; ++i) v.v[i] = c + i < have ? row[c + i] : (T)0.0f;
                Vec<_Float16, 8> o;
#pragma unroll
                for (int i = 0; i < 8; ++i) o.v[i] = (_Float16)((float)v.v[i] * scale);
                store_vec<_Float16, 8>(out + r * a.cols + c, o);
            }
        }
        return;
    } else {
        // rows without gaps are one, of all workgroups
        const bool one = a.op.ldw == a.op.K;
        const int64_t R = one ? 1 : a.op.V, K = one ? a.op.V * a.op.K : a.op.K;
        const int64_t c0 = ((one ? (int64_t)blockIdx.x : 0) * LS_NT + threadIdx.x) * G;
        for (int64_t r = one ? 0 : blockIdx.x; r < R; r += LAY_PARTS)
            see_row((const T *)a.op.weight + r * a.op.ldw, c0, (one ? LAY_PARTS : 1) * (int64_t)LS_NT * G, K);
    }
#pragma unroll
    for (int o = FL_WAVE / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (fl_lane() == 0) waves[fl_wave_id()] = m;
    __syncthreads();
    if (threadIdx.x == 0)
        most[blockIdx.x] = fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3]));
}

// x and weight as rows on 16 bytes: fp32 as its planes (plane_at), half, and bfloat16
// that no backward follows, as they are; SCALED, bfloat16 in training: weight as half
// times a power of two that brings the largest to 2^13..2^14 (what is above 2^-31 of
// it is held exactly, and what is lost below 2^-38).  Zeros behind a row.  (dz, in
// half, is then rounded by 2^-11 of itself; by 2^-8 in bfloat16 it made the
// gradients' error 1.4 to 1.5 times that of their own rounding.)  HBM-bound: 1.18
// GB of bfloat16 read and written in 443 us = 5.3 TB/s.
template <typename T, bool SCALED>
__global__ __launch_bounds__(LS_NT) void k_lay(VocabArgs a, const float *__restrict__ most, uint16_t *__restrict__ x,
                                               uint16_t *__restrict__ w, float *__restrict__ undo) {
    const bool second = SCALED || blockIdx.y;
    const int64_t R = second ? a.op.V : a.op.M, ld = second ? a.op.ldw : a.op.ldx, chunks = a.cols / 8, K = a.op.K;
    const T *p = (const T *)(second ? a.op.weight : a.op.x);
    uint16_t *out = second ? w : x;
    float scale = 1.0f;
    if constexpr (SCALED) {
        __shared__ float waves[LS_WAVES];
        float m = 0.0f;
        for (int i = threadIdx.x; i < LAY_PARTS; i += LS_NT) m = fmaxf(m, most[i]);
#pragma unroll
        for (int o = FL_WAVE / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        if (fl_lane() == 0) waves[fl_wave_id()] = m;
        __syncthreads();
        const int e = exponent_of(fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3])));
        scale = ldexpf(1.0f, 14 - e);
        if (blockIdx.x == 0 && threadIdx.x == 0) *undo = ldexpf(1.0f, e - 14);
    }
    for (int64_t i = (int64_t)blockIdx.x * LS_NT + threadIdx.x; i < R * chunks; i += (int64_t)gridDim.x * LS_NT) {
        const int64_t r = i / chunks, c = i % chunks * 8;
        Vec<T, 8> v;
        if (c + 8 <= K) v = load_vec<T, 8>(p + r * ld + c);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = c + e < K ? p[r * ld + c + e] : (T)0.0f;
        if constexpr (sizeof(T) == 4) {
            u32x4 plane[3];
            chunk_planes<float>(v.v, plane);
            uint16_t *q = out + r * 3 * a.cols + plane_at(c);
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4 *>(q + p * 32) = plane[p];
        } else if constexpr (SCALED) {
            Vec<_Float16, 8> o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o.v[e] = (_Float16)((float)v.v[e] * scale);
            store_vec<_Float16, 8>((_Float16 *)out + r * a.cols + c, o);
        } else store_vec<T, 8>((T *)out + r * a.cols + c, v);
    }
}

// Logit tiles: row tiles of x against row tiles of weight from n0 on, whose
// order in LDS gives a lane 16 columns in a row (16 (lane / 16) .. of the
// wave's 64).
template <typename T, typename H, int BM, int WN, int STAGES>
struct LogitTiles {
    static constexpr int P = planes_of<T>();
    using TA = StepsContig<BM, P>;
    using TB = StepsContig<WN * 64, P>;
    using Run = WideTiles<H, P, BM, WN, STAGES, TA, TB>;
    TA ta;
    TB tb;
    int steps, at;  // of a tile's row; of the next load
    int64_t n_next;

    static __device__ __forceinline__ int column(int r) {
        return (r & ~63) + ((r >> 2) & 3) * 16 + ((r >> 4) & 3) * 4 + (r & 3);
    }
    __device__ __forceinline__ void aim(const VocabArgs &a) {
        const int64_t n0 = n_next < a.op.V ? n_next : a.op.V - 1;
        const int most = (int)(a.op.V - 1 - n0 < WN * 64 ? a.op.V - 1 - n0 : WN * 64);
        tb.init(a.w + n0 * a.ldw, a.ldw, [&](int r) { return column(r) < most ? column(r) : most; });
    }
    __device__ __forceinline__ void init(const VocabArgs &a, int64_t row0, int64_t n0) {
        steps = (int)(a.cols / TA::BK);
        at = 0;
        n_next = n0;
        const int most = (int)(a.op.M - 1 - row0 < BM ? a.op.M - 1 - row0 : BM);
        ta.init(a.x + row0 * a.ldx, a.ldx, [&](int r) { return r < most ? r : most; });
        aim(a);
    }
    __device__ __forceinline__ void feed(const VocabArgs &a, int i, uint16_t *la, uint16_t *lb) {
        if (i < TA::LOADS) ta.issue(la, i);
        else tb.issue(lb, i - TA::LOADS);
        if (i < TA::LOADS + TB::LOADS - 1) return;
        ta.next();
        tb.next();
        if (++at < steps) return;
        at = 0;
        ta.base -= steps * (P * TA::BK);
        n_next += WN * 64;
        aim(a);
    }
};

// A workgroup's row tile and part: eight row tiles and four parts are near each
// other, so that an XCD's workgroups share both operands.
__device__ __forceinline__ void row_and_part(const VocabArgs &a, uint32_t *mt, uint32_t *part) {
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const uint32_t g = w / (8 * a.parts), n = a.m_tiles - 8 * g < 8 ? a.m_tiles - 8 * g : 8, l = w - g * 8 * a.parts;
    // quotients come in vector registers
    *mt = (uint32_t)__builtin_amdgcn_readfirstlane((int)(8 * g + l % n));
    *part = (uint32_t)__builtin_amdgcn_readfirstlane((int)(l / n));
}

// Where the part of `all` things begins.
__device__ __forceinline__ int64_t part_begin(int64_t all, uint32_t part, uint32_t parts) {
    return fl_uniform_i64(all * part / parts);
}

// What a row's products are multiplied by, in units of log 2 (finite: a product of 0 stays 0).
__device__ __forceinline__ float product_scale(const VocabArgs &a, int64_t row) {
    if (!a.undo_x) return a.scale;
    return fminf(a.undo_x[row < a.op.M ? row : a.op.M - 1] * *a.undo_w * a.scale, 0x1.fffffep127f);
}
// Whether the operands' rows have powers of two.
template <typename T, typename H>
constexpr bool is_scaled() {
    return std::is_same<T, __bf16>::value && std::is_same<H, _Float16>::value;
}

// A lane's bias for its 16 columns from n on, in units of log 2.
template <typename T>
__device__ __forceinline__ void lane_bias(const VocabArgs &a, int64_t n, float (&b)[16]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const int64_t left = a.op.V - n - h * 4;
        const int have = left < 0 ? 0 : left < 4 ? (int)left : 4;
        float v[4];
        if (a.op.bias_f32) load_some<float>((const float *)a.op.bias + n + h * 4, have, v);
        else load_some<T>((const T *)a.op.bias + n + h * 4, have, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) b[h * 4 + e] = v[e] * a.scale;
    }
}

// The rows' running maxima and sums over a part of the vocabulary's tiles: a lane
// keeps those of its own columns in LDS over all tiles, and they are joined at the
// end.  An exponent is one multiply-add from the product; the maximum is the
// lane's first until a sum passes 2^20, so that it is not looked for in every tile
// (and an exponent that counts is rounded by no more than 2^-20).
// bf16 [8192 x 512 -> 41000] 339 to 348 us = 988 to 1014 TFLOP/s, fp16 [4096 x 1024
// -> 123000] 945 to 994 us = 1038 to 1092 (a large library product 1313 and 1451 on the same card), fp32
// [1536 x 2048 -> 1645] 78 us = 132 (153), six products each in 156 tiles on 256
// CUs; [512 x 128 -> 4.6M] bf16 954 us = 632: of two steps a tile, the exponentials
// are half.
template <typename T, typename H, int BM, int WN, int STAGES>
__global__ __launch_bounds__(WD_NT) void k_wide_stats(VocabArgs a) {
    using Tiles = LogitTiles<T, H, BM, WN, STAGES>;
    using Run = typename Tiles::Run;
    constexpr int MT = Run::MT;
    extern __shared__ __align__(16) uint16_t wide_lds[];
    uint32_t mt, part;
    row_and_part(a, &mt, &part);
    const int64_t row0 = (int64_t)mt * BM, V = a.op.V;
    const int64_t t0 = part_begin(a.n_tiles, part, a.parts), t1 = part_begin(a.n_tiles, part + 1, a.parts);
    // a lane's sums over its own columns, a pair a row
    Running *sums = reinterpret_cast<Running *>(wide_lds + STAGES * Run::ELEMS) + fl_wave_id() * MT * FL_WAVE;
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[i * FL_WAVE + fl_lane()] = Running{-INFINITY, 0.0f};
    Tiles tiles;
    tiles.init(a, row0, t0 * WN * 64);
    constexpr bool SCALED = is_scaled<T, H>();
    float scales[(MT + 3) / 4];  // of the wave's rows, one a lane
    Run run;
    if constexpr (SCALED)
#pragma unroll
        for (int h = 0; h < (MT + 3) / 4; ++h) scales[h] = product_scale(a, row0 + run.wave_m() + h * FL_WAVE + fl_lane());
    run.template run<false>(
        tiles.ta, tiles.tb, (int)(t1 - t0), tiles.steps, wide_lds,
        [&](int i, uint16_t *la, uint16_t *lb) { tiles.feed(a, i, la, lb); },
        [&](int64_t t) {
            const int lane = made_here(fl_lane());
            Running *state = sums + lane;
            const int64_t n = (t0 + t) * WN * 64 + run.wave_n() + (lane >> 4) * 16;
            const int have = V - n < 16 ? (int)(V - n) : 16;
            float b[16];
            if (a.op.bias) lane_bias<T>(a, n, b);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                __builtin_amdgcn_sched_barrier(0);  // a row's values at a time: few registers
                Running r = state[i * FL_WAVE];
                float s = 0.0f, scale = a.scale;
                if constexpr (SCALED) scale = __shfl(scales[i / 4], i % 4 * 16 + (lane & 15));
                const auto u = [&](int e, float less) {
                    const float v = run.acc[i][e / 4][e % 4];
                    const float t = a.op.bias ? b[e] - less : -less;
                    return e < have ? __builtin_fmaf(v, scale, t) : -INFINITY;
                };
                // what the lane had first serves as the maximum, until a sum passes 2^20 or is not a number
                if (__any(have < 16)) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s += exp2_of(u(e, r.m));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float v = run.acc[i][e / 4][e % 4];
                        s += exp2_of(__builtin_fmaf(v, scale, a.op.bias ? b[e] - r.m : -r.m));
                    }
                }
                s += r.s;
                if (r.m == -INFINITY || !(s < 0x1p20f)) {  // a lane's own: rows do not touch each other's bits
                    float m = r.m;
                    s = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; ++e) m = fmaxf(m, u(e, 0.0f));
                    const float at = base_of(m);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s += exp2_of(u(e, at));
                    s += r.s * exp2_of(r.m - at);
                    r.m = m;
                }
                r.s = s;
                state[i * FL_WAVE] = r;
            }
        });
    Running r[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) r[i] = sums[i * FL_WAVE + fl_lane()];
    __syncthreads();  // the operands in the LDS are read
    store_running<BM, WN>(a, r, reinterpret_cast<Running *>(wide_lds), run.wave_m(), run.wave_n() / 64, row0, part);
}

// dz of a piece but for the listed columns (a row's only one is made in its tile).
// 443, 1085 and 80 us where k_wide_stats takes 348, 994 and 78: what dz's stores
// add, 672 MB of them in the first.
template <typename T, int BM, int WN, int STAGES>
__global__ __launch_bounds__(WD_NT) void k_wide_grad(VocabArgs a) {
    using Tiles = LogitTiles<T, WideDz<T>, BM, WN, STAGES>;
    using Run = typename Tiles::Run;
    constexpr int MT = Run::MT;
    extern __shared__ __align__(16) uint16_t wide_lds[];
    uint32_t mt, part;
    row_and_part(a, &mt, &part);
    const int64_t row0 = (int64_t)mt * BM, end = a.v0 + a.width;
    const int64_t t0 = part_begin(a.n_tiles, part, a.parts), t1 = part_begin(a.n_tiles, part + 1, a.parts);
    // (maximum, coefficient over the sum, the row's only id or -1, its dz) of the tile's rows
    float4 *of = reinterpret_cast<float4 *>(wide_lds + STAGES * Run::ELEMS);
    for (int t = threadIdx.x; t < BM; t += WD_NT) {
        const int64_t m = row0 + t < a.op.M ? row0 + t : a.op.M - 1;
        const float2 sum = a.rows[m];
        const float c = row0 + t < a.op.M ? a.coef[m] : 0.0f;
        float id = __int_as_float(-1), d = 0.0f;
        if (a.op.lists.k == 1 && c != 0.0f) {
            const int64_t v = a.op.lists.ids[m];
            const float2 l = a.listed[m];
            if (v >= a.v0 && v < end) id = __int_as_float((int)(v - a.v0));
            d = c * (listed_share(l.x, sum) - l.y);
        }
        of[t] = float4{sum.x, c * sum.y, id, d};
    }
    constexpr bool SCALED = is_scaled<T, WideDz<T>>();
    float *scales = reinterpret_cast<float *>(of + BM);
    if constexpr (SCALED)
        for (int t = threadIdx.x; t < BM; t += WD_NT) scales[t] = product_scale(a, row0 + t);
    __syncthreads();
    Tiles tiles;
    tiles.init(a, row0, a.v0 + t0 * WN * 64);
    Run run;
    run.template run<false>(
        tiles.ta, tiles.tb, (int)(t1 - t0), tiles.steps, wide_lds,
        [&](int i, uint16_t *la, uint16_t *lb) { tiles.feed(a, i, la, lb); },
        [&](int64_t t) {
            const int lane = made_here(fl_lane());
            const int64_t c = (t0 + t) * WN * 64 + run.wave_n() + (lane >> 4) * 16, n = a.v0 + c;  // c: in the piece
            const int have = end - n < 16 ? (int)(end - n) : 16;
            float b[16];
            if (a.op.bias) lane_bias<T>(a, n, b);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                const int r = run.wave_m() + i * 16 + (lane & 15);
                const float4 q = of[r];
                const float scale = SCALED ? scales[r] : a.scale;
                const int64_t at = __float_as_int(q.z) - c;  // of the row's only id
                float u[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float v = run.acc[i][e / 4][e % 4];
                    u[e] = q.y * exp2_of(__builtin_fmaf(v, scale, a.op.bias ? b[e] - q.x : -q.x));
                }
                if (__any(q.y == 0.0f || have < 16))
#pragma unroll
                    for (int e = 0; e < 16; ++e) u[e] = q.y != 0.0f && e < have ? u[e] : 0.0f;
                if (__any(at >= 0 && at < 16))
#pragma unroll
                    for (int e = 0; e < 16; ++e) u[e] = at == e ? q.w : u[e];
                if (row0 + r >= a.d_rows) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (c + h * 8 >= a.d_cols) continue;
                    uint16_t *to = (uint16_t *)a.d + dz_at<planes_of<T>()>(a, row0 + r, c + h * 8);
                    if constexpr (sizeof(T) == 4) {
                        float one[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) one[e] = u[h * 8 + e];
                        u32x4 plane[3];
                        chunk_planes<float>(one, plane);
#pragma unroll
                        for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4 *>(to + p * 32) = plane[p];
                    } else {
                        Vec<_Float16, 8> o;
#pragma unroll
                        for (int e = 0; e < 8; ++e) o.v[e] = (_Float16)u[h * 8 + e];
                        store_vec<_Float16, 8>((_Float16 *)to, o);
                    }
                }
            }
        });
}

// Column sums of a part of the rows of dz: 512 columns a workgroup, eight a lane,
// a quarter of the rows a wave.  HBM-bound: 15 MB in 5.8 us, from the caches.
constexpr int COLS_WIDE = 8 * FL_WAVE;

template <typename T>
__global__ __launch_bounds__(LS_NT) void k_wide_cols(VocabArgs a) {
    constexpr int P = planes_of<T>(), AHEAD = P == 1 ? 4 : 2;
    using D = WideDz<T>;
    __shared__ float sums[LS_WAVES][COLS_WIDE];
    const int64_t blocks = (a.width + COLS_WIDE - 1) / COLS_WIDE, item = fl_block(), part = item / blocks;
    if (part >= a.parts) return;
    const int64_t c0 = item % blocks * COLS_WIDE, c = c0 + fl_lane() * 8;
    const int64_t runs = (int64_t)a.parts * LS_WAVES, run = part * LS_WAVES + fl_wave_id();
    const int64_t begin = a.op.M * run / runs, end = a.op.M * (run + 1) / runs;
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (c < a.d_cols)
        for (int64_t m = begin; m < end; m += AHEAD) {
            Vec<D, 8> v[AHEAD][P];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int64_t r = m + j < end ? m + j : end - 1;
                const D *d = (const D *)a.d + dz_at<P>(a, r, c);
#pragma unroll
                for (int p = 0; p < P; ++p) v[j][p] = load_vec<D, 8>(d + p * 32);
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (m + j >= end) break;
                const float f = P == 1 ? a.factor[m + j] : 1.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float t = (float)v[j][P - 1].v[e];
#pragma unroll
                    for (int p = P - 2; p >= 0; --p) t += (float)v[j][p].v[e];
                    s[e] += t * f;
                }
            }
        }
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[fl_wave_id()][fl_lane() * 8 + e] = s[e];
    __syncthreads();
    for (int i = threadIdx.x; i < COLS_WIDE && c0 + i < a.width; i += LS_NT)
        a.sums[part * a.width + c0 + i] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
}

// A piece's part of dx, added to what is there if `add`; with one part and one piece
// the result itself.  bf16 [8192 x 512 -> 41000] 333 us = 1033 TFLOP/s, fp16
// [4096 x 1024 -> 123000] 860 us = 1200, fp32 [1536 x 2048 -> 1645] 75 us = 138; the
// weight's steps are read transposed
// from LDS.
template <typename T, int BM, int WN, int STAGES>
__global__ __launch_bounds__(WD_NT) void k_wide_dx(VocabArgs a) {
    constexpr int P = planes_of<T>();
    using TA = StepsContig<BM, P>;
    using TB = StepsStrided<WN * 64, P>;
    using Run = WideTiles<WideDz<T>, P, BM, WN, STAGES, TA, TB>;
    constexpr int STEP = TB::STEP;
    extern __shared__ __align__(16) uint16_t wide_lds[];
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x), tiles = a.m_tiles * a.n_tiles;
    const uint32_t part = (uint32_t)__builtin_amdgcn_readfirstlane((int)(w / tiles)), tile = w - part * tiles;
    const uint32_t nt = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tile / a.m_tiles));
    const int64_t row0 = (int64_t)(tile - nt * a.m_tiles) * BM, n0 = (int64_t)nt * WN * 64, M = a.op.M;
    const int64_t all = (a.width + STEP - 1) / STEP;
    const int64_t s0 = part_begin(all, part, a.parts), s1 = part_begin(all, part + 1, a.parts);
    TA ta;
    TB tb;
    const int most = (int)(M - 1 - row0 < BM ? M - 1 - row0 : BM);
    constexpr int IN_BLOCK = D_BLOCK / STEP;  // steps
    ta.init((const uint16_t *)a.d + s0 / IN_BLOCK * a.d_block + row0 * a.ldd + s0 % IN_BLOCK * (P * STEP), a.ldd,
            [&](int r) { return r < most ? r : most; });
    const auto aim = [&](int64_t step) {  // dz is 0 behind the piece
        const int64_t v = step * STEP, left = a.width - v;
        tb.init(a.w + (a.v0 + v) * a.ldw + P * n0, a.ldw, a.cols - n0, left < STEP ? (int)left : STEP);
    };
    int64_t next = s0;
    aim(next);
    const float f = a.dx && a.undo_w ? *a.undo_w : 1.0f;
    Run run;
    run.template run<true>(
        ta, tb, 1, (int)(s1 - s0), wide_lds,
        [&](int i, uint16_t *la, uint16_t *lb) {
            if (i < TA::LOADS) ta.issue(la, i);
            else tb.issue(lb, i - TA::LOADS);
            if (i < Run::LOADS - 1 || ++next >= s1) return;
            ta.next();
            tb.next();
            if (next % IN_BLOCK == 0) ta.base += a.d_block - a.ldd;
            if (next == all - 1) aim(next);
        },
        [&](int64_t) {
            const int lane = made_here(fl_lane());
#pragma unroll
            for (int i = 0; i < Run::MT; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                const int64_t row = row0 + run.wave_m() + i * 16 + (lane & 15);
                if (row >= M) continue;
                const float f2 = a.dx && P == 1 ? a.factor[row] : 1.0f;
#pragma unroll
                for (int j = 0; j < Run::NTL; ++j) {
                    const int64_t n = n0 + run.wave_n() + j * 16 + (lane >> 4) * 4;
                    if (n >= a.op.K) continue;
                    const int have = a.op.K - n < 4 ? (int)(a.op.K - n) : 4;
                    if (a.dx) {
                        Vec<T, 4> o;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o.v[e] = (T)(run.acc[i][j][e] * f * f2);
                        T *q = (T *)a.dx + row * a.op.K + n;
                        if (have == 4) store_vec<T, 4>(q, o);
                        else store_some<T, 4>(q, o, have);
                        continue;
                    }
                    float *q = a.sums + ((int64_t)part * M + row) * a.op.K + n;
                    Vec<float, 4> f{{run.acc[i][j][0], run.acc[i][j][1], run.acc[i][j][2], run.acc[i][j][3]}};
                    if (a.add) {
                        float old[4];
                        load_some<float>(q, have, old);
#pragma unroll
                        for (int e = 0; e < 4; ++e) f.v[e] += old[e];
                    }
                    if (have == 4) store_vec<float, 4>(q, f);
                    else store_some<float, 4>(q, f, have);
                }
            }
        });
}

// A piece's rows of dW, or of a part of the rows' sum: tiles in a row.  Both
// operands lie with the rows of x one after the other and are read transposed, with
// twice the LDS instructions of k_wide_dx: 463 us = 743 TFLOP/s and 1172 us = 880 in
// its cases, fp32 [1536 x 2048 -> 1645] 76 us = 137.  (x could be laid out the other
// way round; it is not.)
template <typename T, int BM, int WN, int STAGES>
__global__ __launch_bounds__(WD_NT) void k_wide_dw(VocabArgs a) {
    constexpr int P = planes_of<T>();
    using TA = StepsStrided<BM, P>;
    using TB = StepsStrided<WN * 64, P>;
    using Run = WideTiles<WideDz<T>, P, BM, WN, STAGES, TA, TB>;
    constexpr int STEP = TB::STEP;
    extern __shared__ __align__(16) uint16_t wide_lds[];
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const uint32_t walks = (uint32_t)__builtin_amdgcn_readfirstlane((int)(gridDim.x / a.parts));
    const uint32_t part = (uint32_t)__builtin_amdgcn_readfirstlane((int)(w / walks)), walk = w - part * walks;
    const int64_t all = (int64_t)a.m_tiles * a.n_tiles;
    const int64_t t0 = part_begin(all, walk, walks), t1 = part_begin(all, walk + 1, walks);
    const int64_t rows = (a.op.M + STEP - 1) / STEP;
    const int64_t s0 = part_begin(rows, part, a.parts);
    const int steps = (int)(part_begin(rows, part + 1, a.parts) - s0);
    TA ta;
    TB tb;
    int64_t next = t0, m0, c0;
    int at = 0;
    const auto aim = [&](int64_t step) {  // dz is 0 in the rows behind the last
        const int64_t k = step * STEP, left = a.op.M - k;
        const int in = (int)(m0 % D_BLOCK);
        ta.init((const uint16_t *)a.d + m0 / D_BLOCK * a.d_block + k * a.ldd + P * in, a.ldd, D_BLOCK - in,
                STEP);
        tb.init((const uint16_t *)a.y + k * a.ldy + P * c0, a.ldy, a.cols - c0, left < STEP ? (int)left : STEP);
    };
    const auto aim_tile = [&]() {
        const int64_t mt = fl_uniform_i64(next / a.n_tiles);
        m0 = mt * BM;
        c0 = (next - mt * a.n_tiles) * (WN * 64);
        aim(s0);
    };
    aim_tile();
    const int y_exp = a.y_exp ? *a.y_exp : 0;
    Run run;
    run.template run<false>(
        ta, tb, (int)(t1 - t0), steps, wide_lds,
        [&](int i, uint16_t *la, uint16_t *lb) {
            if (i < TA::LOADS) ta.issue(la, i);
            else tb.issue(lb, i - TA::LOADS);
            if (i < Run::LOADS - 1 || next >= t1) return;
            if (++at == steps) {
                at = 0;
                if (++next < t1) aim_tile();
                return;
            }
            ta.next();
            tb.next();
            if (s0 + at == rows - 1 && a.op.M % STEP) aim(s0 + at);
        },
        [&](int64_t t) {
            const int lane = made_here(fl_lane());
            const int64_t mt = fl_uniform_i64((t0 + t) / a.n_tiles), m0 = mt * BM;
            const int64_t c0 = (t0 + t - mt * a.n_tiles) * (WN * 64);
#pragma unroll
            for (int i = 0; i < Run::MT; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                const int64_t m = m0 + run.wave_m() + i * 16 + (lane & 15);
                if (m >= a.width) continue;
#pragma unroll
                for (int j = 0; j < Run::NTL; ++j) {
                    const int64_t c = c0 + run.wave_n() + j * 16 + (lane >> 4) * 4;
                    if (c >= a.op.K) continue;
                    const int n = a.op.K - c < 4 ? (int)(a.op.K - c) : 4;
                    if (a.sums) {
                        float *q = a.sums + ((int64_t)part * a.width + m) * a.op.K + c;
                        const Vec<float, 4> o{{run.acc[i][j][0], run.acc[i][j][1], run.acc[i][j][2], run.acc[i][j][3]}};
                        if (n == 4) store_vec<float, 4>(q, o);
                        else store_some<float, 4>(q, o, n);
                    } else {
                        T *q = (T *)a.dw + (a.v0 + m) * a.op.K + c;
                        Vec<T, 4> o;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o.v[e] = dw_of<T>(run.acc[i][j][e], y_exp);
                        if (n == 4) store_vec<T, 4>(q, o);
                        else store_some<T, 4>(q, o, n);
                    }
                }
            }
        });
}

// ---------------------------------------------------------------------------
// Host side

// How the products of a vocabulary are cut.
struct VocabPlan {
    bool wide, lay, scaled;            // wide kernels; operands laid out, times powers of two
    bool small;                        // tiles of 128
    int bm, bn;                        // tiles of the logits
    uint32_t m_tiles, n_tiles, parts;  // parts: of the vocabulary, in the forward
    int64_t piece, d_cols, ldd;        // columns of dz in the backward, with those that pad them, and its row stride
    int64_t d_block;                   // wide: from one block of its columns to the next
    int64_t dz_rows, d_rows, cols;     // rows of dz; they and the inputs with those that pad them
    int64_t size;                      // bytes of a value of dz
};

// Inputs whose laid out rows have 32-bit offsets over a tile (255 and 127 of them, 2 and 6 bytes a value).
constexpr int64_t most_inputs(bool f32) { return f32 ? 1 << 22 : 1 << 23; }

VocabPlan vocab_plan(const fl_vocab *op) {
    VocabPlan p{};
    const bool f32 = op->dtype == FL_F32;
    const int64_t step = f32 ? 32 : 64, planes = f32 ? 3 : 1;  // inputs of a step of the wide kernels
    p.scaled = op->dtype == FL_BF16 && op->train;
    p.lay = f32 || p.scaled || !aligned(op->x, op->ldx) || !aligned(op->weight, op->ldw) || op->K % step ||
            op->ldx >= 1 << 23 || op->ldw >= 1 << 23;  // 32-bit offsets of 256 rows
    // Laying the weight out takes a pass over it or two, which few rows do not pay for.  fp32 (us laid out and as it is):
    // in training [1536 x 2048 -> 1645] 317 and 450, [4096 x 512 -> 4000] 414 and 463, [600 x 256 -> 41000] 414 and 468, but
    // [200 x 256 -> 41000] 214 and 216, [300 x 64 -> 41000] 161 and 133, [143 x 512 -> 200000] 1411 and 1304; in evaluation
    // 91 and 148, 99 and 102, 100 and 101, but [200 x 512 -> 8000] 45 and 26.  16-bit values, in units of 1e-12 s a value of
    // the weight: 0.9 to 1.3 and 2 rows / 1000 a product, against 2 rows / 430 (0.45 at least) from where it lies.  bfloat16
    // in training is laid out whatever it costs and at every size, so that dz is half.
    int64_t least = 65;
    double work = 1 << 27;
    if (f32) {
        least = op->train ? 256 : 512;
        work = op->train ? 1 << 30 : 1ll << 31;
    } else if (op->dtype == FL_BF16 && op->train) {
        least = 1;
        work = 0;
    } else if (p.lay) least = op->train ? 128 : 384;
    p.wide = op->K >= 1 && op->K <= most_inputs(f32) && op->M >= least && (double)op->M * op->V * op->K >= work;
    p.lay = p.lay && p.wide;
    p.scaled = p.scaled && p.wide;
    p.size = !f32 ? 2 : p.wide ? 6 : 4;
    if (p.wide) {
        p.cols = ceil_div(op->K, step) * step;
        p.small = f32 || op->M <= 128 || ceil_div(op->M, 256) * ceil_div(op->V, 256) < 192;
        p.bm = p.small ? 128 : 256;
        p.bn = p.bm;  // three planes of 256 x 256 have no registers
    } else {
        // tiles by the steps that the fullest CU takes: a step of 128 x 128 takes 2.3 us alone and 1.45 more a tile beside
        // others, of 64 x 64 1.2 and 0.52, of 32 x 64 0.52 and 0.3 (fp32)
        double least = 1e30;
        const int rows[3] = {128, 64, 32}, cols[3] = {128, 64, 64};
        const double alone[3] = {2.3, 1.2, 0.52}, beside[3] = {1.45, 0.52, 0.3};
        for (int i = 0; i < 3; ++i) {
            const double n = (double)ceil_div(ceil_div(op->M, rows[i]) * ceil_div(op->V, cols[i]), 256) * beside[i];
            const double us = n > alone[i] ? n : alone[i];
            if (us >= least) continue;
            least = us;
            p.bm = rows[i];
            p.bn = cols[i];
        }
    }
    p.m_tiles = (uint32_t)ceil_div(op->M, p.bm);
    p.n_tiles = (uint32_t)ceil_div(op->V, p.bn);
    const int64_t want = p.wide ? (p.m_tiles < 256 ? 256 / p.m_tiles : 1) : ceil_div(1024, p.m_tiles);
    p.parts = (uint32_t)(want < p.n_tiles ? want : p.n_tiles);
    // half: of few rows a gradient can be one term of dz, whose rounding would be as large as the gradient's own
    p.dz_rows = op->dtype == FL_F16 && !p.wide && op->M <= 64 ? 2 * op->M : op->M;
    int64_t piece = (int64_t)(LS_PIECE / p.size) / (p.dz_rows > 0 ? p.dz_rows : 1) / 256 * 256;
    if (piece < 256) piece = 256;
    p.piece = piece < op->V ? piece : op->V;
    p.d_cols = p.wide ? ceil_div(p.piece, D_BLOCK) * D_BLOCK : ceil_div(p.piece, 8) * 8;
    p.d_rows = p.wide ? ceil_div(op->M, step) * step : p.dz_rows;
    p.ldd = !p.wide ? p.d_cols : planes * D_BLOCK;
    p.d_block = p.d_rows * p.ldd;
    return p;
}

// The laid out operands: x, weight, what undoes the powers of two of x's rows and of weight, parts of weight's maximum.
struct VocabLayout {
    size_t x, w, undo_x, undo_w, most, bytes;
};

VocabLayout vocab_layout(const fl_vocab *op, const VocabPlan &p) {
    VocabLayout l{};
    if (!p.lay) return l;
    l.w = rounded((size_t)op->M * p.cols * p.size);
    l.bytes = l.w + rounded((size_t)op->V * p.cols * p.size);
    if (p.scaled) {
        l.undo_x = l.bytes;
        l.undo_w = l.undo_x + rounded((size_t)op->M * 4);
        l.most = l.undo_w + 256;
        l.bytes = l.most + LAY_PARTS * 4;
    }
    return l;
}

struct VocabSpace {
    size_t coef, factor, most, y_exp, y, d, dx, dw, db, bytes;
    bool half;  // dz: its rows' gradients as a number and a power of two
    int64_t ldy;
    int dx_parts, dw_parts, db_parts;
    int dx_tile, dx_cols, dw_cols, dw_tile;
    bool dx_direct, few_dw;
    uint32_t dw_walks;
};

VocabSpace vocab_space(const fl_vocab *op, const VocabPlan &p, bool with_dx, bool with_dw, bool with_db) {
    VocabSpace s{};
    const auto take = [&](size_t n) {
        const size_t at = s.bytes;
        s.bytes += rounded(n);
        return at;
    };
    const bool f32 = op->dtype == FL_F32;
    s.coef = take((size_t)op->M * 4);
    s.half = !f32;
    if (s.half) {
        s.factor = take((size_t)op->M * 4);
        s.most = take(LAY_PARTS * 4);
        s.y_exp = take(4);
        s.ldy = ceil_div(op->K, 64) * 64;
        if (with_dw) s.y = take((size_t)op->M * s.ldy * 2);
    }
    s.d = take((size_t)p.d_rows * p.d_cols * p.size);
    const int narrow = op->K <= 128 ? 128 : 256;
    if (with_dx) {
        if (p.wide) {
            s.dx_tile = p.small || ceil_div(op->M, 256) * ceil_div(op->K, narrow) < 16 ? 128 : 256;
            s.dx_cols = s.dx_tile == 128 ? 128 : narrow;
            const int64_t tiles = ceil_div(op->M, s.dx_tile) * ceil_div(op->K, s.dx_cols);
            const int64_t want = 256 / tiles, most = p.piece / 256;
            const int64_t n = want < most ? want : most;
            s.dx_parts = (int)(n < 1 ? 1 : n > 128 ? 128 : n);
        } else {
            // enough workgroups for the chip, of at least 256 columns
            s.dx_tile = p.dz_rows > 64 && op->K > 64 ? 128 : 64;
            const int64_t tiles = ceil_div(p.dz_rows, s.dx_tile) * ceil_div(op->K, s.dx_tile);
            const int64_t want = ceil_div(1024, tiles > 0 ? tiles : 1), most = p.piece / 256, n = want < most ? want : most;
            s.dx_parts = (int)(n < 1 ? 1 : n > 128 ? 128 : n);
        }
        s.dx_direct = p.wide && s.dx_parts == 1 && p.piece == op->V;
        if (!s.dx_direct) s.dx = take((size_t)s.dx_parts * p.dz_rows * op->K * 4);
    }
    s.few_dw = p.dz_rows <= few_rows(op->dtype);
    if (with_dw && s.few_dw) s.dw_parts = 1;
    else if (with_dw) {
        if (p.wide) {
            s.dw_tile = p.small ? 128 : 256;
            s.dw_cols = p.small ? 128 : narrow;
            const int64_t tiles = ceil_div(p.piece, s.dw_tile) * ceil_div(op->K, s.dw_cols), want = 256 / tiles, most = op->M / 256;
            const int64_t n = want < most ? want : most;
            s.dw_parts = (int)(n < 1 ? 1 : n > 16 ? 16 : n);
            s.dw_walks = (uint32_t)(tiles < 256 ? tiles : 256);
        } else {
            const Cut c = best_cut(p.piece, op->K, op->M, f32, false);
            s.dw_parts = c.parts;
            s.dw_tile = c.rows == 128 && op->K >= 2 && p.piece >= 2 ? 128 : 64;
        }
        if (s.dw_parts > 1) s.dw = take((size_t)s.dw_parts * p.piece * op->K * 4);
    }
    if (with_db) {
        const int64_t want = p.wide ? ceil_div(1024, ceil_div(p.piece, COLS_WIDE)) : ceil_div(2048, ceil_div(p.piece, LS_NT));
        const int64_t most = op->M / 16;
        const int64_t n = want < most ? want : most;
        s.db_parts = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
        s.db = take((size_t)s.db_parts * p.piece * 4);
    }
    return s;
}

VocabArgs vocab_args(const fl_vocab *op, const VocabPlan &p, void *state, void *layout) {
    VocabArgs a{};
    a.op = *op;
    a.scale = LOG2E / op->lists.temperature;
    a.rows = state_rows(state);
    a.listed = state_listed(&op->lists, state);
    a.width = op->V;
    a.cols = p.cols;
    if (p.lay) {
        const VocabLayout l = vocab_layout(op, p);
        a.x = (const uint16_t *)((char *)layout + l.x);
        a.w = (const uint16_t *)((char *)layout + l.w);
        a.ldx = a.ldw = op->dtype == FL_F32 ? 3 * p.cols : p.cols;
        if (p.scaled) {
            a.undo_x = (const float *)((char *)layout + l.undo_x);
            a.undo_w = (const float *)((char *)layout + l.undo_w);
        }
    } else {
        a.x = (const uint16_t *)op->x;
        a.w = (const uint16_t *)op->weight;
        a.ldx = op->ldx;
        a.ldw = op->ldw;
    }
    return a;
}

// Of tiles of 128 x 128, 256 x 128 and 256 x 256: stages, and bytes of LDS.
template <typename T>
constexpr int small_stages() {
    return planes_of<T>() == 1 ? 4 : 3;
}
template <typename T>
constexpr unsigned tiles_bytes(int bm, int bn, int stages) {
    return (unsigned)(stages * (bm + bn) * (planes_of<T>() == 1 ? 64 : 96) * 2);
}

template <typename T>
int vocab_forward(hipStream_t st, const fl_vocab *op, float *loss, void *state, void *layout, void *ws) {
    constexpr int BK = sizeof(T) == 4 ? 32 : 64, S = small_stages<T>();
    const VocabPlan p = vocab_plan(op);
    VocabArgs a = vocab_args(op, p, state, layout);
    a.m_tiles = p.m_tiles;
    a.n_tiles = p.n_tiles;
    a.parts = p.parts;
    a.part = (Running *)ws;
    const int64_t grid = (int64_t)p.m_tiles * p.parts;
    if (!launch_fits(grid, WD_NT)) return fl_fail(FL_ERR_ARG, "linear_loss: too many tiles for one launch (shape)");
    const dim3 g((unsigned)grid);
    if (p.lay) {
        const VocabLayout l = vocab_layout(op, p);
        const int64_t chunks = (op->M > op->V && !p.scaled ? op->M : op->V) * (p.cols / 8), want = ceil_div(chunks, LS_NT);
        const unsigned lg = (unsigned)(want < 4096 ? want : 4096);
        if constexpr (std::is_same<T, __bf16>::value)
            if (p.scaled) {
                float *most = (float *)((char *)layout + l.most);
                FL_LAUNCH("k_lay_max", k_lay_max<T>, dim3(LAY_PARTS, 2), dim3(LS_NT), 0, st, a, most, (_Float16 *)a.x,
                          (float *)a.undo_x);
                FL_LAUNCH("k_lay", (k_lay<T, true>), dim3(lg), dim3(LS_NT), 0, st, a, most, (uint16_t *)a.x,
                          (uint16_t *)a.w, (float *)a.undo_w);
            }
        if (!p.scaled)
            FL_LAUNCH("k_lay", (k_lay<T, false>), dim3(lg, 2), dim3(LS_NT), 0, st, a, (const float *)nullptr,
                      (uint16_t *)a.x, (uint16_t *)a.w, (float *)nullptr);
    }
    const bool few = op->lists.k <= DOT_IDS && p.parts <= 4 * FL_WAVE;
    if (!few && op->lists.k)
        FL_LAUNCH("k_vocab_dots", k_vocab_dots<T>,
                  grid_of(ceil_div(op->M * ceil_div(op->lists.k, DOT_IDS), LS_WAVES)), dim3(LS_NT), 0, st, a);
    if (p.wide) {
        const auto extra = [](int mt) { return (unsigned)(WD_WAVES * mt * FL_WAVE * sizeof(Running)); };
        const auto launch = [&](auto half) {
            using H = decltype(half);
            if (p.bm == 128)
                FL_LAUNCH("k_wide_stats", (k_wide_stats<T, H, 128, 2, S>), g, dim3(WD_NT), tiles_bytes<T>(128, 128, S) + extra(2), st, a);
            else if constexpr (planes_of<T>() == 1)
                FL_LAUNCH("k_wide_stats", (k_wide_stats<T, H, 256, 4, 2>), g, dim3(WD_NT), tiles_bytes<T>(256, 256, 2) + extra(8), st, a);
        };
        if constexpr (std::is_same<T, __bf16>::value) {
            if (p.scaled) launch(_Float16());
            else launch(T());
        } else launch(WideDz<T>());
    } else if (p.bm == 128)
        FL_LAUNCH("k_vocab_stats", (k_vocab_stats<T, 128, 128, BK>), g, dim3(LN_NT), 0, st, a);
    else if (p.bm == 64) FL_LAUNCH("k_vocab_stats", (k_vocab_stats<T, 64, 64, BK>), g, dim3(LN_NT), 0, st, a);
    else FL_LAUNCH("k_vocab_stats", (k_vocab_stats<T, 32, 64, 64>), g, dim3(LN_NT), 0, st, a);
    if (!few) return join_listed(st, &op->lists, op->V, a.part, p.parts, state, loss, "linear_loss");
    FL_LAUNCH("k_vocab_rows", k_vocab_rows<T>, grid_of(ceil_div(op->M, LS_WAVES)), dim3(LS_NT), 0, st, a,
              list_args(&op->lists, op->V, state, loss));
    return fl_check_launch("linear_loss");
}

template <typename T>
int vocab_backward(hipStream_t st, const fl_vocab *op, const float *grad, void *state, void *layout, void *dx, void *dw,
                   void *db, char *ws) {
    constexpr int BK = sizeof(T) == 4 ? 32 : 64, S = small_stages<T>();
    // dx and dW by the plain tiles: bfloat16 in training has them only where there are no inputs, and so neither
    constexpr bool PLAIN = !std::is_same<T, __bf16>::value;
    const VocabPlan p = vocab_plan(op);
    const VocabSpace s = vocab_space(op, p, dx, dw, db);
    VocabArgs a = vocab_args(op, p, state, layout);
    float *coef = (float *)(ws + s.coef);
    a.coef = coef;
    a.d = ws + s.d;
    a.ldd = p.ldd;
    a.d_block = p.d_block;
    a.d_cols = p.d_cols;
    a.d_rows = p.d_rows;
    a.dz_rows = p.dz_rows;
    const dim3 nt(LN_NT), wt(WD_NT);
    const float *none = nullptr;
    const auto fits = [&](int64_t grid) { return launch_fits(grid, WD_NT); };
    const auto fail = [&]() { return fl_fail(FL_ERR_ARG, "linear_loss: too many tiles for one launch (shape)"); };
    a.y = p.wide ? (const void *)a.x : op->x;
    a.ldy = p.wide ? a.ldx : op->ldx;
    if (!s.half)
        FL_LAUNCH("k_vocab_coef", k_vocab_coef, dim3((unsigned)(op->M > 65536 ? 64 : ceil_div(op->M, 1024))), dim3(1024),
                  0, st, a.rows, grad, op->lists.temperature, op->M, coef);
    if constexpr (sizeof(T) == 2)
        {
            float *factor = (float *)(ws + s.factor);
            int *most = (int *)(ws + s.most), *y_exp = (int *)(ws + s.y_exp);
            const int64_t all = ceil_div(op->M, LS_WAVES);
            const int parts = (int)(all < LAY_PARTS ? all : LAY_PARTS);
            a.factor = factor;
            FL_LAUNCH("k_row_scale", k_row_scale<T>, dim3(parts), dim3(LS_NT), 0, st, a, grad, op->lists.temperature,
                      dw && op->K, coef, factor, most);
            a.y = ws + s.y;
            a.ldy = s.ldy;
            a.y_exp = y_exp;
            if (dw && op->K) {
                const int64_t want = ceil_div(op->M * (s.ldy / 8), LS_NT);
                FL_LAUNCH("k_lay_y", k_lay_y<T>, dim3((unsigned)(want < 2048 ? want : 2048)), dim3(LS_NT), 0, st, a, most,
                          parts, (_Float16 *)(ws + s.y), y_exp);
            }
        }
    for (a.v0 = 0; a.v0 < op->V; a.v0 += p.piece) {
        a.width = op->V - a.v0 < p.piece ? op->V - a.v0 : p.piece;
        a.m_tiles = p.m_tiles;
        a.n_tiles = (uint32_t)ceil_div(a.width, p.bn);
        if (p.wide) {
            const int64_t want = p.m_tiles < 256 ? 256 / p.m_tiles : 1;
            a.parts = (uint32_t)(want < a.n_tiles ? want : a.n_tiles);
        } else a.parts = a.n_tiles;
        int64_t grid = (int64_t)a.m_tiles * a.parts;
        if (!fits(grid)) return fail();
        if (p.wide) {
            const auto extra = [](int bm) { return (unsigned)(bm * (sizeof(float4) + sizeof(float))); };
            const dim3 g((unsigned)grid);
            if (p.bm == 128)
                FL_LAUNCH("k_wide_grad", (k_wide_grad<T, 128, 2, S>), g, wt, tiles_bytes<T>(128, 128, S) + extra(128), st, a);
            else if constexpr (planes_of<T>() == 1)
                FL_LAUNCH("k_wide_grad", (k_wide_grad<T, 256, 4, 2>), g, wt, tiles_bytes<T>(256, 256, 2) + extra(256), st, a);
        } else if (p.bm == 128)
            FL_LAUNCH("k_vocab_grad", (k_vocab_grad<T, 128, 128, BK>), dim3((unsigned)grid), nt, 0, st, a);
        else if (p.bm == 64) FL_LAUNCH("k_vocab_grad", (k_vocab_grad<T, 64, 64, BK>), dim3((unsigned)grid), nt, 0, st, a);
        else FL_LAUNCH("k_vocab_grad", (k_vocab_grad<T, 32, 64, 64>), dim3((unsigned)grid), nt, 0, st, a);
        if (op->lists.k > 1 || (op->lists.k && !p.wide)) {
            const dim3 g = grid_of(ceil_div(op->M * op->lists.k, LS_NT));
            if (p.wide) FL_LAUNCH("k_vocab_listed", (k_vocab_listed<T, true>), g, dim3(LS_NT), 0, st, a);
            else FL_LAUNCH("k_vocab_listed", (k_vocab_listed<T, false>), g, dim3(LS_NT), 0, st, a);
        }
        if (dx && op->K) {
            a.m_tiles = (uint32_t)ceil_div(p.dz_rows, s.dx_tile);
            a.n_tiles = (uint32_t)ceil_div(op->K, p.wide ? s.dx_cols : s.dx_tile);
            a.parts = (uint32_t)s.dx_parts;
            a.sums = (float *)(ws + s.dx);
            a.dx = s.dx_direct ? dx : nullptr;
            a.add = a.v0 > 0;
            grid = (int64_t)a.m_tiles * a.n_tiles * a.parts;
            if (!fits(grid)) return fail();
            const dim3 g((unsigned)grid);
            if (p.wide) {
                if (s.dx_tile == 128)
                    FL_LAUNCH("k_wide_dx", (k_wide_dx<T, 128, 2, S>), g, wt, tiles_bytes<T>(128, 128, S), st, a);
                else if constexpr (planes_of<T>() == 1) {
                    if (s.dx_cols == 128)
                        FL_LAUNCH("k_wide_dx", (k_wide_dx<T, 256, 2, 3>), g, wt, tiles_bytes<T>(256, 128, 3), st, a);
                    else
                        FL_LAUNCH("k_wide_dx", (k_wide_dx<T, 256, 4, 2>), g, wt, tiles_bytes<T>(256, 256, 2), st, a);
                }
            } else if constexpr (PLAIN) {
                if (s.dx_tile == 128) FL_LAUNCH("k_vocab_dx", (k_vocab_dx<T, 128, 128, BK>), g, nt, 0, st, a);
                else FL_LAUNCH("k_vocab_dx", (k_vocab_dx<T, 64, 64, BK>), g, nt, 0, st, a);
            }
        }
        if (dw && op->K && s.few_dw) {
            const int cols = p.dz_rows <= 32 ? few_cols<T, 1>() : p.dz_rows <= 64 ? few_cols<T, 2>() : few_cols<T, 4>();
            const int64_t bands = ceil_div(op->K, cols), all = ceil_div(bands * ceil_div(a.width, 16), LS_WAVES);
            grid = ceil_div(bands, LS_WAVES);
            if (grid < FEW_WALKS) grid = all < FEW_WALKS ? all : FEW_WALKS;
            if (!fits(grid)) return fail();
            a.dw = dw;
            const dim3 g((unsigned)grid), t(LS_NT);
            const auto launch = [&](auto wide) {
                constexpr bool WIDE = decltype(wide)::value;
                if (p.dz_rows <= 32) FL_LAUNCH("k_few_dw", (k_few_dw<T, WIDE, 1>), g, t, 0, st, a);
                else if (p.dz_rows <= 64) FL_LAUNCH("k_few_dw", (k_few_dw<T, WIDE, 2>), g, t, 0, st, a);
                else if constexpr (sizeof(T) == 2) FL_LAUNCH("k_few_dw", (k_few_dw<T, WIDE, 4>), g, t, 0, st, a);
            };
            if constexpr (sizeof(T) == 2)
                if (p.wide) launch(std::true_type());
            if constexpr (PLAIN)
                if (!p.wide) launch(std::false_type());
        } else if (dw && op->K) {
            const int rows = s.dw_tile, cols = p.wide ? s.dw_cols : s.dw_tile;
            a.m_tiles = (uint32_t)ceil_div(a.width, rows);
            a.n_tiles = (uint32_t)ceil_div(op->K, cols);
            a.parts = (uint32_t)s.dw_parts;
            a.sums = s.dw_parts > 1 ? (float *)(ws + s.dw) : nullptr;
            a.dw = dw;
            grid = (int64_t)a.m_tiles * a.n_tiles;
            if (p.wide && grid > s.dw_walks) grid = s.dw_walks;
            grid *= a.parts;
            if (!fits(grid)) return fail();
            const dim3 g((unsigned)grid);
            if (p.wide) {
                if (rows == 128)
                    FL_LAUNCH("k_wide_dw", (k_wide_dw<T, 128, 2, S>), g, wt, tiles_bytes<T>(128, 128, S), st, a);
                else if constexpr (planes_of<T>() == 1) {
                    if (cols == 128)
                        FL_LAUNCH("k_wide_dw", (k_wide_dw<T, 256, 2, 3>), g, wt, tiles_bytes<T>(256, 128, 3), st, a);
                    else
                        FL_LAUNCH("k_wide_dw", (k_wide_dw<T, 256, 4, 2>), g, wt, tiles_bytes<T>(256, 256, 2), st, a);
                }
            } else if constexpr (PLAIN) {
                if (rows == 128) FL_LAUNCH("k_vocab_dw", (k_vocab_dw<T, 128, 128, BK>), g, nt, 0, st, a);
                else FL_LAUNCH("k_vocab_dw", (k_vocab_dw<T, 64, 64, BK>), g, nt, 0, st, a);
            }
            if (a.sums)
                FL_LAUNCH("k_vocab_fold", k_vocab_fold<T>, grid_of(ceil_div(a.width * op->K, FL_WAVE * 4)), dim3(LS_NT),
                          0, st, a.sums, a.parts, a.width * op->K, none, none, (int64_t)1, a.y_exp, (T *)dw + a.v0 * op->K);
        }
        if (db) {
            a.parts = (uint32_t)s.db_parts;
            a.sums = (float *)(ws + s.db);
            const dim3 g = grid_of(ceil_div(a.width, FL_WAVE * 4));
            if (p.wide)
                FL_LAUNCH("k_wide_cols", k_wide_cols<T>, grid_of(a.parts * ceil_div(a.width, COLS_WIDE)),
                          dim3(LS_NT), 0, st, a);
            else
                FL_LAUNCH("k_vocab_cols", k_vocab_cols<T>, grid_of(a.parts * ceil_div(a.width, LS_NT)), dim3(LS_NT), 0,
                          st, a);
            if (op->bias_f32)
                FL_LAUNCH("k_vocab_fold", k_vocab_fold<float>, g, dim3(LS_NT), 0, st, a.sums, a.parts, a.width,
                          none, none, (int64_t)1, (const int *)nullptr, (float *)db + a.v0);
            else
                FL_LAUNCH("k_vocab_fold", k_vocab_fold<T>, g, dim3(LS_NT), 0, st, a.sums, a.parts, a.width, none,
                          none, (int64_t)1, (const int *)nullptr, (T *)db + a.v0);
        }
    }
    if (dx && op->K && !s.dx_direct)
        FL_LAUNCH("k_vocab_fold", k_vocab_fold<T>, grid_of(ceil_div(op->M * op->K, FL_WAVE * 4)), dim3(LS_NT), 0, st,
                  (const float *)(ws + s.dx), (uint32_t)(s.dx_parts * (p.dz_rows / op->M)), op->M * op->K,
                  a.undo_w, a.factor, op->K, (const int *)nullptr, (T *)dx);
    return fl_check_launch("linear_loss");
}

int check_vocab(const fl_vocab *op, const char *what) {
    if (!op) return fl_fail(FL_ERR_ARG, "%s: null operator", what);
    if (op->dtype < FL_F32 || op->dtype > FL_F16) return fl_fail(FL_ERR_ARG, "%s: unknown type", what);
    if (op->M < 0 || op->V < 1 || op->K < 0 || op->V > 0x7fffffffll || op->K > 0x7fffffffll || op->M != op->lists.rows)
        return fl_fail(FL_ERR_ARG, "%s: bad shape", what);
    if (op->M && op->K && (!op->x || !op->weight)) return fl_fail(FL_ERR_ARG, "%s: null pointer", what);
    if (op->dtype == FL_BF16 && op->train && op->K > most_inputs(false))
        return fl_fail(FL_ERR_ARG, "%s: bfloat16 in training has up to %d inputs (shape)", what, (int)most_inputs(false));
    return check_lists(&op->lists, what);
}

}  // namespace
}  // namespace fl

#define FL_BY_TYPE(dtype, call)                           \
    switch (dtype) {                                      \
        case FL_F32: { using T = float; return call; }    \
        case FL_BF16: { using T = __bf16; return call; }  \
        default: { using T = _Float16; return call; }     \
    }

extern "C" {

size_t fl_vocab_op_bytes(void) { return sizeof(fl_vocab); }

size_t fl_vocab_layout_bytes(const fl_vocab *op) {
    if (!op || op->M < 1 || op->V < 1 || op->K < 0) return 0;
    return fl::vocab_layout(op, fl::vocab_plan(op)).bytes;
}

size_t fl_vocab_forward_bytes(const fl_vocab *op) {
    if (!op || op->M < 1 || op->V < 1 || op->K < 0) return 0;
    return (size_t)op->M * fl::vocab_plan(op).parts * 8;
}

int fl_vocab_forward(void *stream, const fl_vocab *op, float *loss, void *state, void *layout, void *ws,
                     size_t ws_bytes) {
    const int rc = fl::check_vocab(op, "linear_loss");
    if (rc) return rc;
    if (op->M == 0) return FL_OK;
    const size_t need = fl_vocab_forward_bytes(op);
    if (!loss || !state || (!layout && fl_vocab_layout_bytes(op))) return fl::fl_fail(FL_ERR_ARG, "linear_loss: null pointer");
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "linear_loss: workspace too small");
    if ((uintptr_t)layout % 16) return fl::fl_fail(FL_ERR_ARG, "linear_loss: layout must be 16-byte aligned");
    FL_BY_TYPE(op->dtype, fl::vocab_forward<T>((hipStream_t)stream, op, loss, state, layout, ws))
}

size_t fl_vocab_backward_bytes(const fl_vocab *op, int with_dx, int with_dw, int with_db) {
    if (!op || op->M < 1 || op->V < 1 || op->K < 0) return 0;
    return fl::vocab_space(op, fl::vocab_plan(op), with_dx, with_dw, with_db).bytes;
}

int fl_vocab_backward(void *stream, const fl_vocab *op, const float *grad, void *state, void *layout, void *dx,
                      void *dw, void *db, void *ws, size_t ws_bytes) {
    const int rc = fl::check_vocab(op, "linear_loss");
    if (rc) return rc;
    if (op->M == 0) return FL_OK;
    if (!op->train) return fl::fl_fail(FL_ERR_ARG, "linear_loss: a forward without `train` has no backward");
    if (!grad || !state || (!layout && fl_vocab_layout_bytes(op))) return fl::fl_fail(FL_ERR_ARG, "linear_loss: null pointer");
    const size_t need = fl_vocab_backward_bytes(op, dx != nullptr, dw != nullptr, db != nullptr);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "linear_loss: workspace too small");
    if ((uintptr_t)ws % 16) return fl::fl_fail(FL_ERR_ARG, "linear_loss: workspace must be 16-byte aligned");
    if ((uintptr_t)layout % 16) return fl::fl_fail(FL_ERR_ARG, "linear_loss: layout must be 16-byte aligned");
    FL_BY_TYPE(op->dtype, fl::vocab_backward<T>((hipStream_t)stream, op, grad, state, layout, dx, dw, db, (char *)ws))
}

}  // extern "C"
