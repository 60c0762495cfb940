// Losses of rows of logits over a vocabulary (relations, entities), and their
// gradients.  With u = z / tau over the columns of a row, lse = log sum exp u:
//
//   distillation   L = tau^2 sum_j q_j (log q_j - u[id_j] + lse)
//                  q = softmax of teacher / tau over the listed ids that count
//                  (inside the vocabulary, u[id] not -inf, teacher not -inf)
//                  dz_v = tau g (p_v - sum of the q_j with id_j = v),  p = exp(u - lse)
//   cross entropy  one id a row, q = 1, tau = 1: L = lse - z[id],  dz = g (p - 1 at id)
//
// A row in which nothing is listed, or nothing is left (every u -inf), has
// loss 0 and no gradient.
//
// The rows are either given (scores; a wave a segment of a row, HBM-bound), or
// the product z = x W^T + b, which is not kept: the forward joins every tile's
// maxima and sums of exponentials, and the backward makes the tiles again with
// dz in place of z, for a piece of the vocabulary at a time:
//
//   dx = dz W      dW = dz^T x      db = sum over the rows of dz
//
// The piece of dz is what a call holds of [rows x vocabulary], in the
// operands' type (an operand of two products), small enough for the last level
// cache.  The listed columns' own u comes from a dot product each; their
// entries of dz are made apart, since p - q of values rounded before would
// keep few bits where p is near 1.
//
// u is held in units of log 2: exponentials are the hardware's 2^x, off by
// 2^-24 |u| of themselves besides its own step.
#include "fl_abi.h"
#include "fl_common.h"
#include "fl_parts.h"
#include "fl_product.h"
#include <math.h>

namespace fl {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr int LS_SEG = 2048;  // columns of a wave
constexpr int LS_NT = 256;
constexpr int LS_WAVES = LS_NT / FL_WAVE;
constexpr size_t LS_PIECE = 128u << 20;  // bytes of dz

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// A running maximum and the sum of 2^(u - maximum).
struct Running {
    float m, s;
};
// What exponents are taken from: the maximum, 0 where nothing is above -inf.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ Running joined(Running a, Running b) {
    const float m = fmaxf(a.m, b.m), at = base_of(m);
    return Running{m, a.s * exp2_of(a.m - at) + b.s * exp2_of(b.m - at)};
}
__device__ __forceinline__ Running joined_over(Running r, int lanes) {
#pragma unroll
    for (int o = FL_WAVE / 2; o > 0; o >>= 1) {
        if (o >= lanes) continue;
        r = joined(r, Running{__shfl_xor(r.m, o), __shfl_xor(r.s, o)});
    }
    return r;
}

struct ListArgs {
    fl_lists op;
    float scale, tau2;  // log2(e) / tau, tau^2
    int64_t cols;
    const Running *part;  // [rows][parts]
    int64_t parts;
    const void *logits;   // scores; null: `listed` holds u
    int64_t ld;
    float *loss;
    float2 *rows, *listed;  // (lse, whether the row counts), (u, sum of q at the id)
};

// ---------------------------------------------------------------------------
// Rows that are given

struct ScoreArgs {
    fl_lists op;
    const void *logits;
    int64_t ld, cols;
    uint32_t segments;
    float scale;
    Running *part;
    const float2 *rows, *listed;
    const float *grad;
    void *dx;
};

template <typename T>
constexpr int cols_of() {
    return 16 / (int)sizeof(T);
}

// A wave's segment of a row in registers, behind its end `fill`.
template <typename T>
struct Segment {
    static constexpr int G = cols_of<T>(), N = LS_SEG / FL_WAVE / G;
    Vec<T, G> v[N];

    __device__ __forceinline__ void load(const T *row, int64_t c0, int64_t cols) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t c = c0 + (i * FL_WAVE + fl_lane()) * G;
            if (c + G <= cols) v[i] = load_vec<T, G>(row + c);
            else
#pragma unroll
                for (int e = 0; e < G; ++e) v[i].v[e] = c + e < cols ? row[c + e] : (T)-INFINITY;
        }
    }
};

template <typename T>
__global__ __launch_bounds__(LS_NT) void k_score_stats(ScoreArgs a) {
    constexpr int G = Segment<T>::G, N = Segment<T>::N;
    const int64_t item = fl_block() * LS_WAVES + fl_wave_id();
    if (item >= a.op.rows * a.segments) return;
    const int64_t row = item / a.segments, seg = item % a.segments;
    Segment<T> s;
    s.load((const T *)a.logits + row * a.ld, seg * LS_SEG, a.cols);
    Running r{-INFINITY, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < G; ++e) r.m = fmaxf(r.m, (float)s.v[i].v[e]);
#pragma unroll
    for (int o = FL_WAVE / 2; o > 0; o >>= 1) r.m = fmaxf(r.m, __shfl_xor(r.m, o));
    r.m *= a.scale;
    const float at = base_of(r.m);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < G; ++e) r.s += exp2_of((float)s.v[i].v[e] * a.scale - at);
    r.s = fl_wave_sum_f32(r.s);
    if (fl_lane() == 0) a.part[row * a.segments + seg] = r;
}

template <typename T>
__global__ __launch_bounds__(LS_NT) void k_score_grad(ScoreArgs a) {
    constexpr int G = Segment<T>::G, N = Segment<T>::N;
    const int64_t item = fl_block() * LS_WAVES + fl_wave_id();
    if (item >= a.op.rows * a.segments) return;
    const int64_t row = item / a.segments, c0 = (item % a.segments) * LS_SEG;
    const float2 of = a.rows[row];
    const float c = of.y != 0.0f ? a.op.temperature * a.grad[row] : 0.0f;
    T *out = (T *)a.dx + row * a.cols;
    Segment<T> s;
    s.load((const T *)a.logits + row * a.ld, c0, a.cols);
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int e = 0; e < G; ++e)
            s.v[i].v[e] = (T)(c == 0.0f ? 0.0f : c * exp2_of((float)s.v[i].v[e] * a.scale - of.x));
        const int64_t at = c0 + (i * FL_WAVE + fl_lane()) * G;
        if (at + G <= a.cols) store_vec<T, G>(out + at, s.v[i]);
        else store_some<T, G>(out + at, s.v[i], (int)(a.cols - at));
    }
    if (c == 0.0f) return;
    // the listed columns of this segment, behind the stores above
    const int64_t *ids = a.op.ids + row * a.op.k;
    bool waited = false;
    for (int64_t j0 = 0; j0 < a.op.k; j0 += FL_WAVE) {
        const int64_t j = j0 + fl_lane(), id = j < a.op.k ? ids[j] : -1;
        const bool here = id >= c0 && id < c0 + LS_SEG && id < a.cols;
        if (!__any(here)) continue;
        if (!waited) {
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
            __builtin_amdgcn_s_waitcnt(0);
        }
        waited = true;
        if (here) {
            const float2 l = a.listed[row * a.op.k + j];
            out[id] = (T)(c * (exp2_of(l.x - of.x) - l.y));
        }
    }
}

// ---------------------------------------------------------------------------
// Rows' sums joined, their lists, their losses: a wave a row.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_list_rows(ListArgs a) {
    extern __shared__ __align__(16) float2 list_lds[];
    const int waves = blockDim.x / FL_WAVE;
    const int64_t row = fl_block() * waves + fl_wave_id(), k = a.op.k;
    if (row >= a.op.rows) return;
    Running r{-INFINITY, 0.0f};
    for (int64_t p = fl_lane(); p < a.parts; p += FL_WAVE) r = joined(r, a.part[row * a.parts + p]);
    r = joined_over(r, FL_WAVE);
    const float lse = r.m + log2f(r.s);
    const int64_t *ids = a.op.ids + row * k;
    float2 *mine = list_lds + fl_wave_id() * k, *listed = a.listed + row * k;
    // (id, teacher in units of log 2), -inf where it does not count
    float top = -INFINITY;
    bool any = false;
    for (int64_t j = fl_lane(); j < k; j += FL_WAVE) {
        const int64_t id = ids[j];
        const bool in = id >= 0 && id < a.cols;
        float u = 0.0f;
        if (a.logits) u = in ? (float)((const T *)a.logits)[row * a.ld + id] * a.scale : 0.0f;
        else if (in) u = listed[j].x;
        float v = -INFINITY;
        if (in && a.op.teacher && u != -INFINITY) v = a.op.teacher[row * k + j] * a.scale;
        if (in && !a.op.teacher) v = 0.0f;
        mine[j] = float2{__int_as_float(in ? (int)id : -1), v};
        listed[j] = float2{u, 0.0f};
        top = fmaxf(top, v);
        any = any || v != -INFINITY;
    }
#pragma unroll
    for (int o = FL_WAVE / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const bool live = __any(any) && r.s != 0.0f;  // no sum: every u is -inf
    float total = 0.0f;
    for (int64_t j = fl_lane(); j < k; j += FL_WAVE) total += exp2_of(mine[j].y - top);
    total = fl_wave_sum_f32(total);
    const float of_total = 1.0f / total, log_total = log2f(total);
    float loss = 0.0f;
    for (int64_t j = fl_lane(); j < k; j += FL_WAVE) {
        const float v = mine[j].y, q = live ? exp2_of(v - top) * of_total : 0.0f;
        if (q != 0.0f) loss += q * ((v - top - log_total) - (listed[j].x - lse));
        mine[j].y = q;
    }
    loss = fl_wave_sum_f32(loss) * (a.tau2 * LN2);
    if (fl_lane() == 0) {
        a.loss[row] = live ? loss : 0.0f;
        a.rows[row] = float2{lse, live ? 1.0f : 0.0f};
    }
    fl_wave_sync();
    for (int64_t j = fl_lane(); j < k; j += FL_WAVE) {
        const int id = __float_as_int(mine[j].x);
        float q = 0.0f;
        if (id >= 0)
            for (int64_t i = 0; i < k; ++i) q += __float_as_int(mine[i].x) == id ? mine[i].y : 0.0f;
        listed[j].y = q;
    }
}

// ---------------------------------------------------------------------------
// Rows that are a product

struct VocabArgs {
    fl_vocab op;
    float scale;          // log2(e) / tau
    // the vocabulary's piece [v0, v0 + width)
    int64_t v0, width;
    uint32_t m_tiles, n_tiles, parts;
    Running *part;        // [M][parts]
    const float2 *rows;
    float2 *listed;
    const float *coef;    // tau g of every row (times a power of two), 0 where it has no gradient
    void *d;              // [M][ldd]
    int64_t ldd;
    float *sums;          // dx: [parts][M][K]; dW: [parts][width][K]
    void *dw;
    const float *unscale;  // what undoes the power of two
    int add;
};

// u of the listed columns: a wave a row and four of them.
constexpr int DOT_IDS = 4;

template <typename T>
__global__ __launch_bounds__(LS_NT) void k_vocab_dots(VocabArgs a) {
    const int64_t k = a.op.lists.k, quads = (k + DOT_IDS - 1) / DOT_IDS;
    const int64_t item = fl_block() * LS_WAVES + fl_wave_id();
    if (item >= a.op.M * quads) return;
    const int64_t row = item / quads, j0 = item % quads * DOT_IDS, K = a.op.K;
    const T *x = (const T *)a.op.x + row * a.op.ldx;
    const T *w[DOT_IDS];
    int64_t id[DOT_IDS];
    float s[DOT_IDS] = {};
#pragma unroll
    for (int i = 0; i < DOT_IDS; ++i) {
        id[i] = j0 + i < k ? a.op.lists.ids[row * k + j0 + i] : -1;
        if (id[i] >= a.op.V) id[i] = -1;
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
        s[i] = fl_wave_sum_f32(s[i]);
        if (fl_lane() == 0 && j0 + i < k) {
            float b = 0.0f;
            if (a.op.bias && id[i] >= 0)
                b = a.op.bias_f32 ? ((const float *)a.op.bias)[id[i]] : (float)((const T *)a.op.bias)[id[i]];
            a.listed[row * k + j0 + i] = float2{(s[i] + b) * a.scale, 0.0f};
        }
    }
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

// What a row's gradients are multiplied by.  SCALED (half): times the power of
// two that brings the largest to 2^14, so that small ones stay normal numbers.
template <bool SCALED>
__global__ __launch_bounds__(1024) void k_vocab_coef(const float2 *__restrict__ rows, const float *__restrict__ g,
                                                     float tau, int64_t M, float *__restrict__ coef,
                                                     float *__restrict__ unscale) {
    __shared__ float most[16];
    float scale = 1.0f;
    if constexpr (SCALED) {
        float m = 0.0f;
        for (int64_t i = threadIdx.x; i < M; i += 1024) {
            const float c = rows[i].y != 0.0f ? fabsf(tau * g[i]) : 0.0f;
            m = fmaxf(m, c < INFINITY ? c : 0.0f);
        }
#pragma unroll
        for (int o = FL_WAVE / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        if (fl_lane() == 0) most[threadIdx.x / FL_WAVE] = m;
        __syncthreads();
        for (int i = 0; i < 16; ++i) m = fmaxf(m, most[i]);
        int e;
        frexpf(m, &e);  // m < 2^e
        e = e < -100 ? -100 : e;
        scale = m > 0.0f ? ldexpf(1.0f, 14 - e) : 1.0f;
        if (threadIdx.x == 0) *unscale = m > 0.0f ? ldexpf(1.0f, e - 14) : 1.0f;
    } else if (fl_block() == 0 && threadIdx.x == 0) *unscale = 1.0f;
    const int64_t step = SCALED ? 1024 : (int64_t)gridDim.x * 1024;
    for (int64_t i = (SCALED ? 0 : (int64_t)blockIdx.x * 1024) + threadIdx.x; i < M; i += step)
        coef[i] = rows[i].y != 0.0f ? tau * g[i] * scale : 0.0f;
}

// dz of a piece but for the listed columns.
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
    float lse[Prod::MT], c[Prod::MT];
#pragma unroll
    for (int i = 0; i < Prod::MT; ++i) {
        const int64_t m = row + i * 16 < a.op.M ? row + i * 16 : a.op.M - 1;
        lse[i] = a.rows[m].x;
        c[i] = a.coef[m];
    }
    each_u<T>(a, prod.acc, col, a.v0 + a.width, [&](int i, int j, const float (&u)[4]) {
        const int64_t n = col + j * 16 + (fl_lane() >> 4) * 4 - a.v0;
        if (row + i * 16 >= a.op.M || n >= a.ldd) return;
        Vec<T, 4> o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] = (T)(c[i] == 0.0f ? 0.0f : c[i] * exp2_of(u[e] - lse[i]));
        store_vec<T, 4>((T *)a.d + (row + i * 16) * a.ldd + n, o);
    });
}

// dz of the listed columns in the piece.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_vocab_listed(VocabArgs a) {
    const int64_t i = fl_block() * LS_NT + threadIdx.x, k = a.op.lists.k;
    if (i >= a.op.M * k) return;
    const int64_t row = i / k, v = a.op.lists.ids[i] - a.v0;
    const float c = a.coef[row];
    if (v < 0 || v >= a.width || c == 0.0f) return;
    const float2 l = a.listed[i];
    ((T *)a.d)[row * a.ldd + v] = (T)(c * (exp2_of(l.x - a.rows[row].x) - l.y));
}

// A piece's part of dx, added to what is there if `add`.
template <typename T, int BM, int BN, int BK>
__global__ __launch_bounds__(LN_NT) void k_vocab_dx(VocabArgs a) {
    using Prod = Product<T, BM, BN, BK>;
    __shared__ __align__(16) uint16_t lds[Prod::LDS_ELEMS];
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const uint32_t tile = w / a.parts, part = w % a.parts;
    const int64_t row0 = (int64_t)(tile / a.n_tiles) * BM, n0 = (int64_t)(tile % a.n_tiles) * BN, M = a.op.M;
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

// The parts of a sum added in order and rounded: four values a thread.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_vocab_fold(const float *__restrict__ part, uint32_t parts, int64_t n,
                                                      const float *__restrict__ unscale, T *__restrict__ out) {
    const int64_t i = (fl_block() * LS_NT + threadIdx.x) * 4;
    if (i >= n) return;
    const int have = n - i < 4 ? (int)(n - i) : 4;
    const float f = *unscale;
    float s[4] = {0, 0, 0, 0}, v[4];
    for (uint32_t p = 0; p < parts; ++p) {
        load_some<float>(part + p * n + i, have, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
    Vec<T, 4> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.v[e] = (T)(s[e] * f);
    if (have == 4) store_vec<T, 4>(out + i, o);
    else store_some<T, 4>(out + i, o, have);
}

// A piece's rows of dW, or of a part of the rows' sum.
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
    tb.init((const T *)a.op.x + begin * a.op.ldx + c0, a.op.ldx, a.op.K - c0, nullptr);
    Prod prod;
    prod.run(ta, tb, end - begin, lds);
    const float f = a.sums ? 1.0f : *a.unscale;
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
                for (int e = 0; e < 4; ++e) o.v[e] = (T)(prod.acc[i][j][e] * f);
                if (n == 4) store_vec<T, 4>(q, o);
                else store_some<T, 4>(q, o, n);
            }
        }
    }
}

// Column sums of a part of the rows of dz, a thread a column.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_vocab_cols(VocabArgs a) {
    const int64_t blocks = (a.width + LS_NT - 1) / LS_NT, item = fl_block(), part = item / blocks;
    const int64_t c = item % blocks * LS_NT + threadIdx.x;
    if (part >= a.parts || c >= a.width) return;
    float s = 0.0f;
    for (int64_t m = a.op.M * part / a.parts; m < a.op.M * (part + 1) / a.parts; ++m)
        s += (float)((const T *)a.d)[m * a.ldd + c];
    a.sums[part * a.width + c] = s;
}

// ---------------------------------------------------------------------------
// Host side

constexpr int64_t LS_MOST_LISTED = 4096;

int check_lists(const fl_lists *l, const char *what) {
    if (l->rows < 0 || l->k < 0 || l->rows > 0x7fffffffll) return fl_fail(FL_ERR_ARG, "%s: bad shape", what);
    if (l->k > LS_MOST_LISTED)
        return fl_fail(FL_ERR_ARG, "%s: lists of more than %d ids (shape)", what, (int)LS_MOST_LISTED);
    if (l->rows && !l->teacher && l->k > 1) return fl_fail(FL_ERR_ARG, "%s: targets without a teacher are one a row (shape)", what);
    if (l->rows && l->k && !l->ids) return fl_fail(FL_ERR_ARG, "%s: null pointer", what);
    if (!(l->temperature >= 0x1p-100f && l->temperature <= 0x1p100f))
        return fl_fail(FL_ERR_ARG, "%s: temperature must be positive and finite", what);
    return FL_OK;
}

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }

// Bytes of the state that a forward leaves for the backward: rows, listed.
size_t state_bytes(const fl_lists *l) { return rounded((size_t)l->rows * 8) + (size_t)l->rows * l->k * 8; }
float2 *state_rows(void *state) { return (float2 *)state; }
float2 *state_listed(const fl_lists *l, void *state) { return (float2 *)((char *)state + rounded((size_t)l->rows * 8)); }

template <typename T>
int join_rows(hipStream_t st, ListArgs &a, const char *what) {
    const int64_t waves = a.op.k <= 512 ? LS_WAVES : 1;
    const size_t lds = (size_t)waves * a.op.k * 8;
    FL_LAUNCH("k_list_rows", k_list_rows<T>, grid_of(ceil_div(a.op.rows, waves)), dim3((unsigned)waves * FL_WAVE), lds,
              st, a);
    return fl_check_launch(what);
}

ListArgs list_args(const fl_lists *l, int64_t cols, void *state, float *loss) {
    ListArgs a{};
    a.op = *l;
    a.scale = LOG2E / l->temperature;
    a.tau2 = l->temperature * l->temperature;
    a.cols = cols;
    a.loss = loss;
    a.rows = state_rows(state);
    a.listed = state_listed(l, state);
    return a;
}

int64_t segments_of(int64_t cols) { return ceil_div(cols, LS_SEG); }

template <typename T>
int score_forward(hipStream_t st, const fl_scores *op, float *loss, void *state, void *ws) {
    ScoreArgs s{};
    s.op = op->lists;
    s.logits = op->logits;
    s.ld = op->ld;
    s.cols = op->cols;
    s.segments = (uint32_t)segments_of(op->cols);
    s.scale = LOG2E / op->lists.temperature;
    s.part = (Running *)ws;
    if (s.segments)
        FL_LAUNCH("k_score_stats", k_score_stats<T>, grid_of(ceil_div(op->lists.rows * s.segments, LS_WAVES)),
                  dim3(LS_NT), 0, st, s);
    ListArgs a = list_args(&op->lists, op->cols, state, loss);
    a.part = s.part;
    a.parts = s.segments;
    a.logits = op->logits;
    a.ld = op->ld;
    return join_rows<T>(st, a, "distillation");
}

template <typename T>
int score_backward(hipStream_t st, const fl_scores *op, const float *grad, void *state, void *dx) {
    ScoreArgs s{};
    s.op = op->lists;
    s.logits = op->logits;
    s.ld = op->ld;
    s.cols = op->cols;
    s.segments = (uint32_t)segments_of(op->cols);
    s.scale = LOG2E / op->lists.temperature;
    s.rows = state_rows(state);
    s.listed = state_listed(&op->lists, state);
    s.grad = grad;
    s.dx = dx;
    FL_LAUNCH("k_score_grad", k_score_grad<T>, grid_of(ceil_div(op->lists.rows * s.segments, LS_WAVES)), dim3(LS_NT),
              0, st, s);
    return fl_check_launch("distillation");
}

int check_scores(const fl_scores *op, const char *what) {
    if (!op) return fl_fail(FL_ERR_ARG, "%s: null operator", what);
    if (op->dtype < FL_F32 || op->dtype > FL_F16) return fl_fail(FL_ERR_ARG, "%s: unknown type", what);
    if (op->cols < 0 || op->cols > 0x7fffffffll) return fl_fail(FL_ERR_ARG, "%s: bad shape", what);
    if (op->lists.rows > 0 && op->cols > 0 && !op->logits) return fl_fail(FL_ERR_ARG, "%s: null pointer", what);
    return check_lists(&op->lists, what);
}

// How the products of a vocabulary are cut.
struct VocabPlan {
    int bm, bn;            // tiles of the logits
    uint32_t m_tiles, n_tiles, parts;  // parts: of the vocabulary, in the forward
    int64_t piece, ldd;    // columns of dz in the backward
};

VocabPlan vocab_plan(const fl_vocab *op) {
    VocabPlan p{};
    p.bm = op->M > 64 ? 128 : 64;
    p.bn = p.bm;
    p.m_tiles = (uint32_t)ceil_div(op->M, p.bm);
    p.n_tiles = (uint32_t)ceil_div(op->V, p.bn);
    const int64_t want = ceil_div(1024, p.m_tiles);
    p.parts = (uint32_t)(want < p.n_tiles ? want : p.n_tiles);
    const int64_t size = op->dtype == FL_F32 ? 4 : 2;
    int64_t piece = (int64_t)(LS_PIECE / size) / (op->M > 0 ? op->M : 1) / 256 * 256;
    if (piece < 256) piece = 256;
    p.piece = piece < op->V ? piece : op->V;
    p.ldd = ceil_div(p.piece, 8) * 8;
    return p;
}

struct VocabSpace {
    size_t coef, d, dx, dw, db, bytes;
    int dx_parts, dw_parts, db_parts;
    int dx_tile, dw_tile;
};

VocabSpace vocab_space(const fl_vocab *op, bool with_dx, bool with_dw, bool with_db) {
    const VocabPlan p = vocab_plan(op);
    VocabSpace s{};
    const auto take = [&](size_t n) {
        const size_t at = s.bytes;
        s.bytes += rounded(n);
        return at;
    };
    const bool f32 = op->dtype == FL_F32;
    s.coef = take((size_t)(op->M + 1) * 4);
    s.d = take((size_t)op->M * p.ldd * (f32 ? 4 : 2));
    if (with_dx) {
        const Cut c = best_cut(op->M, op->K, p.piece, f32, false);
        s.dx_parts = c.parts;
        s.dx_tile = c.rows == 128 && op->K >= 2 ? 128 : 64;
        s.dx = take((size_t)c.parts * op->M * op->K * 4);
    }
    if (with_dw) {
        const Cut c = best_cut(p.piece, op->K, op->M, f32, false);
        s.dw_parts = c.parts;
        s.dw_tile = c.rows == 128 && op->K >= 2 && p.piece >= 2 ? 128 : 64;
        if (c.parts > 1) s.dw = take((size_t)c.parts * p.piece * op->K * 4);
    }
    if (with_db) {
        const int64_t want = ceil_div(2048, ceil_div(p.piece, LS_NT)), most = op->M / 16;
        const int64_t n = want < most ? want : most;
        s.db_parts = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
        s.db = take((size_t)s.db_parts * p.piece * 4);
    }
    return s;
}

VocabArgs vocab_args(const fl_vocab *op, void *state) {
    VocabArgs a{};
    a.op = *op;
    a.scale = LOG2E / op->lists.temperature;
    a.rows = state_rows(state);
    a.listed = state_listed(&op->lists, state);
    a.width = op->V;
    return a;
}

template <typename T>
int vocab_forward(hipStream_t st, const fl_vocab *op, float *loss, void *state, void *ws) {
    constexpr int BK = sizeof(T) == 4 ? 32 : 64;
    const VocabPlan p = vocab_plan(op);
    VocabArgs a = vocab_args(op, state);
    a.m_tiles = p.m_tiles;
    a.n_tiles = p.n_tiles;
    a.parts = p.parts;
    a.part = (Running *)ws;
    const int64_t grid = (int64_t)p.m_tiles * p.parts;
    if (!launch_fits(grid, LN_NT)) return fl_fail(FL_ERR_ARG, "linear_loss: too many tiles for one launch (shape)");
    if (op->lists.k)
        FL_LAUNCH("k_vocab_dots", k_vocab_dots<T>,
                  grid_of(ceil_div(op->M * ceil_div(op->lists.k, DOT_IDS), LS_WAVES)), dim3(LS_NT), 0, st, a);
    if (p.bm == 128)
        FL_LAUNCH("k_vocab_stats", (k_vocab_stats<T, 128, 128, BK>), dim3((unsigned)grid), dim3(LN_NT), 0, st, a);
    else FL_LAUNCH("k_vocab_stats", (k_vocab_stats<T, 64, 64, BK>), dim3((unsigned)grid), dim3(LN_NT), 0, st, a);
    ListArgs l = list_args(&op->lists, op->V, state, loss);
    l.part = a.part;
    l.parts = p.parts;
    return join_rows<T>(st, l, "linear_loss");
}

template <typename T>
int vocab_backward(hipStream_t st, const fl_vocab *op, const float *grad, void *state, void *dx, void *dw, void *db,
                   char *ws) {
    constexpr int BK = sizeof(T) == 4 ? 32 : 64;
    const VocabPlan p = vocab_plan(op);
    const VocabSpace s = vocab_space(op, dx, dw, db);
    VocabArgs a = vocab_args(op, state);
    float *coef = (float *)(ws + s.coef);
    a.coef = coef;
    a.unscale = coef + op->M;
    a.d = ws + s.d;
    a.ldd = p.ldd;
    const dim3 nt(LN_NT);
    if (std::is_same<T, _Float16>::value)
        FL_LAUNCH("k_vocab_coef", k_vocab_coef<true>, dim3(1), dim3(1024), 0, st, a.rows, grad, op->lists.temperature,
                  op->M, coef, coef + op->M);
    else
        FL_LAUNCH("k_vocab_coef", k_vocab_coef<false>, dim3((unsigned)(op->M > 65536 ? 64 : ceil_div(op->M, 1024))),
                  dim3(1024), 0, st, a.rows, grad, op->lists.temperature, op->M, coef, coef + op->M);
    for (a.v0 = 0; a.v0 < op->V; a.v0 += p.piece) {
        a.width = op->V - a.v0 < p.piece ? op->V - a.v0 : p.piece;
        a.m_tiles = p.m_tiles;
        a.n_tiles = (uint32_t)ceil_div(a.width, p.bn);
        int64_t grid = (int64_t)a.m_tiles * a.n_tiles;
        if (!launch_fits(grid, LN_NT)) return fl_fail(FL_ERR_ARG, "linear_loss: too many tiles for one launch (shape)");
        if (p.bm == 128) FL_LAUNCH("k_vocab_grad", (k_vocab_grad<T, 128, 128, BK>), dim3((unsigned)grid), nt, 0, st, a);
        else FL_LAUNCH("k_vocab_grad", (k_vocab_grad<T, 64, 64, BK>), dim3((unsigned)grid), nt, 0, st, a);
        if (op->lists.k)
            FL_LAUNCH("k_vocab_listed", k_vocab_listed<T>, grid_of(ceil_div(op->M * op->lists.k, LS_NT)), dim3(LS_NT),
                      0, st, a);
        if (dx && op->K) {
            const int t = s.dx_tile;
            a.n_tiles = (uint32_t)ceil_div(op->K, t);
            a.parts = (uint32_t)s.dx_parts;
            a.sums = (float *)(ws + s.dx);
            a.add = a.v0 > 0;
            grid = ceil_div(op->M, t) * a.n_tiles * a.parts;
            if (!launch_fits(grid, LN_NT)) return fl_fail(FL_ERR_ARG, "linear_loss: too many tiles for one launch (shape)");
            if (t == 128) FL_LAUNCH("k_vocab_dx", (k_vocab_dx<T, 128, 128, BK>), dim3((unsigned)grid), nt, 0, st, a);
            else FL_LAUNCH("k_vocab_dx", (k_vocab_dx<T, 64, 64, BK>), dim3((unsigned)grid), nt, 0, st, a);
        }
        if (dw && op->K) {
            const int t = s.dw_tile;
            a.m_tiles = (uint32_t)ceil_div(a.width, t);
            a.n_tiles = (uint32_t)ceil_div(op->K, t);
            a.parts = (uint32_t)s.dw_parts;
            a.sums = s.dw_parts > 1 ? (float *)(ws + s.dw) : nullptr;
            a.dw = dw;
            grid = (int64_t)a.m_tiles * a.n_tiles * a.parts;
            if (!launch_fits(grid, LN_NT)) return fl_fail(FL_ERR_ARG, "linear_loss: too many tiles for one launch (shape)");
            if (t == 128) FL_LAUNCH("k_vocab_dw", (k_vocab_dw<T, 128, 128, BK>), dim3((unsigned)grid), nt, 0, st, a);
            else FL_LAUNCH("k_vocab_dw", (k_vocab_dw<T, 64, 64, BK>), dim3((unsigned)grid), nt, 0, st, a);
            if (a.sums)
                FL_LAUNCH("k_vocab_fold", k_vocab_fold<T>, grid_of(ceil_div(a.width * op->K, LS_NT * 4)), dim3(LS_NT),
                          0, st, a.sums, a.parts, a.width * op->K, a.unscale, (T *)dw + a.v0 * op->K);
        }
        if (db) {
            a.parts = (uint32_t)s.db_parts;
            a.sums = (float *)(ws + s.db);
            FL_LAUNCH("k_vocab_cols", k_vocab_cols<T>, grid_of(a.parts * ceil_div(a.width, LS_NT)), dim3(LS_NT), 0, st,
                      a);
            const dim3 g = grid_of(ceil_div(a.width, LS_NT * 4));
            if (op->bias_f32)
                FL_LAUNCH("k_vocab_fold", k_vocab_fold<float>, g, dim3(LS_NT), 0, st, a.sums, a.parts, a.width,
                          a.unscale, (float *)db + a.v0);
            else
                FL_LAUNCH("k_vocab_fold", k_vocab_fold<T>, g, dim3(LS_NT), 0, st, a.sums, a.parts, a.width, a.unscale,
                          (T *)db + a.v0);
        }
    }
    if (dx && op->K)
        FL_LAUNCH("k_vocab_fold", k_vocab_fold<T>, grid_of(ceil_div(op->M * op->K, LS_NT * 4)), dim3(LS_NT), 0, st,
                  (const float *)(ws + s.dx), (uint32_t)s.dx_parts, op->M * op->K, a.unscale, (T *)dx);
    return fl_check_launch("linear_loss");
}

int check_vocab(const fl_vocab *op, const char *what) {
    if (!op) return fl_fail(FL_ERR_ARG, "%s: null operator", what);
    if (op->dtype < FL_F32 || op->dtype > FL_F16) return fl_fail(FL_ERR_ARG, "%s: unknown type", what);
    if (op->M < 0 || op->V < 1 || op->K < 0 || op->V > 0x7fffffffll || op->K > 0x7fffffffll || op->M != op->lists.rows)
        return fl_fail(FL_ERR_ARG, "%s: bad shape", what);
    if (op->M && op->K && (!op->x || !op->weight)) return fl_fail(FL_ERR_ARG, "%s: null pointer", what);
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

size_t fl_scores_op_bytes(void) { return sizeof(fl_scores); }
size_t fl_vocab_op_bytes(void) { return sizeof(fl_vocab); }

size_t fl_lists_state_bytes(const fl_lists *lists) {
    if (!lists || lists->rows < 0 || lists->k < 0) return 0;
    return fl::state_bytes(lists);
}

size_t fl_scores_forward_bytes(const fl_scores *op) {
    if (!op || op->cols < 0 || op->lists.rows < 0) return 0;
    return (size_t)op->lists.rows * fl::segments_of(op->cols) * 8;
}

int fl_scores_forward(void *stream, const fl_scores *op, float *loss, void *state, void *ws, size_t ws_bytes) {
    const int rc = fl::check_scores(op, "distillation");
    if (rc) return rc;
    if (op->lists.rows == 0) return FL_OK;
    const size_t need = fl_scores_forward_bytes(op);
    if (!loss || !state) return fl::fl_fail(FL_ERR_ARG, "distillation: null pointer");
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "distillation: workspace too small");
    FL_BY_TYPE(op->dtype, fl::score_forward<T>((hipStream_t)stream, op, loss, state, ws))
}

int fl_scores_backward(void *stream, const fl_scores *op, const float *grad, void *state, void *dx) {
    const int rc = fl::check_scores(op, "distillation");
    if (rc) return rc;
    if (op->lists.rows == 0 || op->cols == 0) return FL_OK;
    if (!grad || !state || !dx) return fl::fl_fail(FL_ERR_ARG, "distillation: null pointer");
    FL_BY_TYPE(op->dtype, fl::score_backward<T>((hipStream_t)stream, op, grad, state, dx))
}

size_t fl_vocab_forward_bytes(const fl_vocab *op) {
    if (!op || op->M < 1 || op->V < 1 || op->K < 0) return 0;
    return (size_t)op->M * fl::vocab_plan(op).parts * 8;
}

int fl_vocab_forward(void *stream, const fl_vocab *op, float *loss, void *state, void *ws, size_t ws_bytes) {
    const int rc = fl::check_vocab(op, "linear_loss");
    if (rc) return rc;
    if (op->M == 0) return FL_OK;
    const size_t need = fl_vocab_forward_bytes(op);
    if (!loss || !state) return fl::fl_fail(FL_ERR_ARG, "linear_loss: null pointer");
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "linear_loss: workspace too small");
    FL_BY_TYPE(op->dtype, fl::vocab_forward<T>((hipStream_t)stream, op, loss, state, ws))
}

size_t fl_vocab_backward_bytes(const fl_vocab *op, int with_dx, int with_dw, int with_db) {
    if (!op || op->M < 1 || op->V < 1 || op->K < 0) return 0;
    return fl::vocab_space(op, with_dx, with_dw, with_db).bytes;
}

int fl_vocab_backward(void *stream, const fl_vocab *op, const float *grad, void *state, void *dx, void *dw, void *db,
                      void *ws, size_t ws_bytes) {
    const int rc = fl::check_vocab(op, "linear_loss");
    if (rc) return rc;
    if (op->M == 0) return FL_OK;
    if (!grad || !state) return fl::fl_fail(FL_ERR_ARG, "linear_loss: null pointer");
    const size_t need = fl_vocab_backward_bytes(op, dx != nullptr, dw != nullptr, db != nullptr);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "linear_loss: workspace too small");
    if ((uintptr_t)ws % 16) return fl::fl_fail(FL_ERR_ARG, "linear_loss: workspace must be 16-byte aligned");
    FL_BY_TYPE(op->dtype, fl::vocab_backward<T>((hipStream_t)stream, op, grad, state, dx, dw, db, (char *)ws))
}

}  // extern "C"
