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
// fp32 operands are cut into three bfloat16 planes by truncation, v = v0 + v1
// + v2 exactly (24 significant bits in 8 + 8 + 8), and the six products whose
// weight is at least 2^-16 are added: what is dropped is below 2^-22 of a
// product (2^-24 on average), as near as fp32 products are.  The matrix unit
// takes bfloat16 16 times faster than fp32, so the six products run at 2.7 times the
// fp32 instruction's rate.  The planes of an infinity or NaN hold a NaN: sums
// that such a value enters are NaN.
#include "fl_abi.h"
#include "fl_common.h"

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
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t w[2][3];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float x = v[2 * j + i];
            w[i][0] = __float_as_uint(x);
            const float r1 = x - __uint_as_float(w[i][0] & 0xffff0000u);
            w[i][1] = __float_as_uint(r1);
            w[i][2] = __float_as_uint(r1 - __uint_as_float(w[i][1] & 0xffff0000u));
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) out[p][j] = upper_halves(w[0][p], w[1][p]);
    }
}

// LDS element offset of chunk c of row r in a tile of BK values a row: the
// permutation spreads both 8 and 16 consecutive rows' chunks over the banks.
template <int BK>
__device__ __forceinline__ int lds_at(int r, int c) {
    const int f = BK == 32 ? ((r >> 1) ^ (r >> 3)) & 3 : (r ^ (r >> 3)) & 7;
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

__device__ __forceinline__ float act_value(float p, int act) {
    switch (act) {
        case FL_ACT_RELU: return p > 0.0f ? p : (p != p ? p : 0.0f);
        case FL_ACT_GELU: return 0.5f * p * (1.0f + erff(p * 0.70710678118654752f));
        case FL_ACT_SILU: return p / (1.0f + expf(-p));
        case FL_ACT_TANH: return tanhf(p);
        case FL_ACT_SIGMOID: return 1.0f / (1.0f + expf(-p));
        default: return p;
    }
}

__device__ __forceinline__ float act_slope(float p, int act) {
    switch (act) {
        case FL_ACT_RELU: return p > 0.0f ? 1.0f : (p != p ? p : 0.0f);
        case FL_ACT_GELU:
            return 0.5f * (1.0f + erff(p * 0.70710678118654752f)) + p * (0.39894228040143268f * expf(-0.5f * p * p));
        case FL_ACT_SILU: {
            const float q = 1.0f / (1.0f + expf(-p));
            return q * (1.0f + p * (1.0f - q));
        }
        case FL_ACT_TANH: {
            const float t = tanhf(p);
            return 1.0f - t * t;
        }
        case FL_ACT_SIGMOID: {
            const float q = 1.0f / (1.0f + expf(-p));
            return q * (1.0f - q);
        }
        default: return 1.0f;
    }
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
    int act, bias_f32;
};

// Products whose C rows are the batch's rows (the forward, and dx): a tile is
// BM rows of one group.
template <typename T, bool B_CONTIG, int BM, int BN, int BK>
__global__ __launch_bounds__(LN_NT) void k_lin_rows(RowsArgs a) {
    using Prod = Product<T, BM, BN, BK>;
    __shared__ __align__(16) uint16_t lds[Prod::LDS_ELEMS];
    const uint32_t w = (uint32_t)fl_xcd_contig(blockIdx.x, gridDim.x);
    const int64_t mt = w / a.n_tiles, nt = w % a.n_tiles;
    int64_t g = 0, pos0 = mt * BM, end = a.M;
    if (a.tiles) {
        g = a.tiles[2 * mt];
        if (g < 0) return;
        pos0 = a.tiles[2 * mt + 1];
        end = g < a.groups ? (int64_t)a.offsets[g + 1] : a.M;
    }
    const bool none = g >= a.groups;  // rows of no group
    const int64_t n0 = nt * BN;
    const T *A = (const T *)a.a;
    const T *B = (const T *)a.b + (none ? 0 : g * a.b_group);
    ContigTile<T, BM, BK> ta;
    ta.init(
        [&](int r) {
            int64_t p = pos0 + r < end ? pos0 + r : end - 1;
            return A + (a.order ? (int64_t)a.order[p] : p) * a.lda;
        });
    Prod prod;
    const int64_t K = none ? 0 : a.K;
    if constexpr (B_CONTIG) {
        ContigTile<T, BN, BK> tb;
        tb.init([&](int r) { return B + (n0 + r < a.N ? n0 + r : a.N - 1) * a.ldb; });
        prod.run(ta, tb, K, lds);
    } else {
        StridedTile<T, BN, BK> tb;
        tb.init(B + n0, a.ldb, a.N - n0, nullptr);
        prod.run(ta, tb, K, lds);
    }
    const int lane = fl_lane();
#pragma unroll
    for (int i = 0; i < Prod::MT; ++i) {
        const int64_t p = pos0 + prod.wave_m() + i * 16 + (lane & 15);
        if (p >= end) continue;
        const int64_t row = a.order ? (int64_t)a.order[p] : p;
#pragma unroll
        for (int j = 0; j < Prod::NTL; ++j) {
            const int64_t n = n0 + prod.wave_n() + j * 16 + (lane >> 4) * 4;
            if (n >= a.N) continue;
            const int m = a.N - n < 4 ? (int)(a.N - n) : 4;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = prod.acc[i][j][e];
            if (a.bias && !none) {
                const int64_t at = g * a.bias_group + n;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < m) v[e] += a.bias_f32 ? ((const float *)a.bias)[at + e] : (float)((const T *)a.bias)[at + e];
            }
            if (a.pre) {
                // kept in 32 bits: rounded to the operands' type it would move the slopes by as much as the
                // gradients' own rounding does
                const Vec<float, 4> f{{v[0], v[1], v[2], v[3]}};
                float *q = a.pre + row * a.N + n;
                if (m == 4) store_vec<float, 4>(q, f);
                else store_some<float, 4>(q, f, m);
            }
            Vec<T, 4> o;
            if (!none)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = act_value(v[e], a.act);
            if (a.residual) {
                const T *q = (const T *)a.residual + row * a.ldres + n;
                if (m == 4) {
                    const Vec<T, 4> r = load_vec<T, 4>(q);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += (float)r.v[e];
                } else
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < m) v[e] += (float)q[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[e] = (T)v[e];
            T *q = (T *)a.c + row * a.ldc + n;
            if (m == 4) store_vec<T, 4>(q, o);
            else store_some<T, 4>(q, o, m);
        }
    }
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

// dW_g = sum over the group's rows (a part of them) of d^T x.
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
    const int lane = fl_lane();
    const int64_t NK = a.N * a.K;
#pragma unroll
    for (int i = 0; i < Prod::MT; ++i) {
        const int64_t m = m0 + prod.wave_m() + i * 16 + (lane & 15);
        if (m >= a.N) continue;
#pragma unroll
        for (int j = 0; j < Prod::NTL; ++j) {
            const int64_t c = c0 + prod.wave_n() + j * 16 + (lane >> 4) * 4;
            if (c >= a.K) continue;
            const int n = a.K - c < 4 ? (int)(a.K - c) : 4;
            if (a.part) {
                float *q = a.part + ((int64_t)part * a.groups + g) * NK + m * a.K + c;
                #pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < n) q[e] = prod.acc[i][j][e];
            } else {
                T *q = (T *)a.dw + g * NK + m * a.K + c;
                Vec<T, 4> o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o.v[e] = (T)prod.acc[i][j][e];
                if (n == 4) store_vec<T, 4>(q, o);
                else store_some<T, 4>(q, o, n);
            }
        }
    }
}

// d = gy * act'(p), rounded to the operands' type: it is an operand of two products.
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

// Column sums of a group's rows (a part of them), one thread a column.
template <typename T>
__global__ __launch_bounds__(LN_NT) void k_col_sums(const T *__restrict__ d, int64_t ldd, int64_t M, int64_t N,
                                                    int64_t groups, int parts, const int32_t *__restrict__ order,
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
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)d[(order ? (int64_t)order[p + j] : p + j) * ldd + c];
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; p < end; ++p) s += (float)d[(order ? (int64_t)order[p] : p) * ldd + c];
    out[((int64_t)part * groups + g) * N + c] = s;
}

// out[i] = sum over the parts, in order.
template <typename TO>
__global__ __launch_bounds__(LN_NT) void k_part_sums(const float *__restrict__ part, int parts, int64_t n,
                                                     TO *__restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * LN_NT + threadIdx.x; i < n; i += (int64_t)gridDim.x * LN_NT) {
        float s = 0.0f;
        for (int p = 0; p < parts; ++p) s += part[(int64_t)p * n + i];
        out[i] = (TO)s;
    }
}

template <typename TO>
void part_sums(hipStream_t st, const float *part, int parts, int64_t n, void *out) {
    int64_t grid = (n + LN_NT - 1) / LN_NT;
    if (grid > 65536) grid = 65536;
    FL_LAUNCH("k_part_sums", k_part_sums<TO>, dim3((unsigned)grid), dim3(LN_NT), 0, st, part, parts, n, (TO *)out);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of a tile: the plan's, or for one group 128 where that gives the chip
// enough workgroups.
int tile_rows(const fl_linear *op, int64_t cols) {
    if (op->offsets) return (int)fl_group_block(op->M, op->groups);
    return ceil_div(op->M, 128) * ceil_div(cols, 128) >= 128 ? 128 : 32;
}

template <typename T, bool B_CONTIG>
int launch_rows(hipStream_t st, const fl_linear *op, RowsArgs &a, const char *what) {
    const int bm = tile_rows(op, a.N);
    constexpr int BIG_K = sizeof(T) == 4 ? 32 : 64;
    const int bn = bm == 128 && a.N > 64 ? 128 : 64;
    const int64_t m_tiles = op->offsets ? fl_group_tiles(op->M, op->groups) : ceil_div(op->M, bm);
    a.n_tiles = (uint32_t)ceil_div(a.N, bn);
    const int64_t grid = m_tiles * a.n_tiles;
    if (grid > 0x7fffffffll) return fl_fail(FL_ERR_ARG, "%s: too many tiles for one launch (shape)", what);
    if (grid == 0) return FL_OK;
    if (bn == 128)
        FL_LAUNCH("k_lin_rows", (k_lin_rows<T, B_CONTIG, 128, 128, BIG_K>), dim3((unsigned)grid), dim3(LN_NT), 0, st,
                  a);
    else if (bm == 128)
        FL_LAUNCH("k_lin_rows", (k_lin_rows<T, B_CONTIG, 128, 64, BIG_K>), dim3((unsigned)grid), dim3(LN_NT), 0, st,
                  a);
    else
        FL_LAUNCH("k_lin_rows", (k_lin_rows<T, B_CONTIG, 32, 64, 64>), dim3((unsigned)grid), dim3(LN_NT), 0, st, a);
    return fl_check_launch(what);
}

// Parts of a group's rows in dW and db: enough workgroups for the chip where
// the tiles alone are few, of at least 256 rows on average.
int outer_parts(int64_t M, int64_t groups, int64_t tiles) {
    int64_t want = ceil_div(512, tiles * groups), most = M / (256 * groups);
    int64_t p = want < most ? want : most;
    return (int)(p < 1 ? 1 : p > 64 ? 64 : p);
}

int sum_parts(int64_t M, int64_t N, int64_t groups) {
    int64_t want = ceil_div(1024, ceil_div(N, LN_NT) * groups), most = M / (32 * groups);
    int64_t p = want < most ? want : most;
    return (int)(p < 1 ? 1 : p > 256 ? 256 : p);
}

int outer_tile(const fl_linear *op) { return op->N >= 128 && op->K >= 128 ? 128 : 64; }

int64_t outer_tiles(const fl_linear *op) {
    const int t = outer_tile(op);
    return ceil_div(op->N, t) * ceil_div(op->K, t);
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
int forward(hipStream_t st, const fl_linear *op, void *y, float *pre) {
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
    return launch_rows<T, true>(st, op, a, "linear_forward");
}

template <typename T>
int input_grad(hipStream_t st, const fl_linear *op, const void *d, void *dx) {
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
    return launch_rows<T, false>(st, op, a, "linear_input_grad");
}

template <typename T>
int weight_grad(hipStream_t st, const fl_linear *op, const void *d, void *dw, float *ws) {
    OuterArgs a{};
    const int t = outer_tile(op);
    a.d = d;
    a.x = op->x;
    a.ldd = op->N;
    a.ldx = op->ldx;
    a.M = op->M;
    a.N = op->N;
    a.K = op->K;
    a.groups = op->groups;
    a.n_tiles = (uint32_t)ceil_div(op->N, t);
    a.k_tiles = (uint32_t)ceil_div(op->K, t);
    a.parts = (uint32_t)outer_parts(op->M, op->groups, outer_tiles(op));
    a.order = op->order;
    a.offsets = op->offsets;
    a.dw = dw;
    a.part = a.parts > 1 ? ws : nullptr;
    const int64_t grid = outer_tiles(op) * a.parts * a.groups;
    if (grid > 0x7fffffffll) return fl_fail(FL_ERR_ARG, "linear_weight_grad: too many tiles for one launch (shape)");
    if (grid == 0) return FL_OK;
    constexpr int BIG_K = sizeof(T) == 4 ? 32 : 64;
    if (t == 128)
        FL_LAUNCH("k_lin_outer", (k_lin_outer<T, 128, 128, BIG_K>), dim3((unsigned)grid), dim3(LN_NT), 0, st, a);
    else
        FL_LAUNCH("k_lin_outer", (k_lin_outer<T, 64, 64, 64>), dim3((unsigned)grid), dim3(LN_NT), 0, st, a);
    if (a.part) part_sums<T>(st, ws, (int)a.parts, a.groups * a.N * a.K, dw);
    return fl_check_launch("linear_weight_grad");
}

template <typename T>
int bias_grad(hipStream_t st, const fl_linear *op, const void *d, void *db, int db_f32, float *ws) {
    const int parts = sum_parts(op->M, op->N, op->groups);
    const int64_t grid = (int64_t)parts * op->groups * ceil_div(op->N, LN_NT);
    if (grid > 0x7fffffffll) return fl_fail(FL_ERR_ARG, "linear_bias_grad: too many groups for one launch (shape)");
    FL_LAUNCH("k_col_sums", k_col_sums<T>, dim3((unsigned)grid), dim3(LN_NT), 0, st,
              (const T *)d, op->N, op->M, op->N, op->groups, parts, op->order, op->offsets, ws);
    if (db_f32) part_sums<float>(st, ws, parts, op->groups * op->N, db);
    else part_sums<T>(st, ws, parts, op->groups * op->N, db);
    return fl_check_launch("linear_bias_grad");
}

template <typename T>
int act_grad(hipStream_t st, int act, const void *gy, const float *pre, int64_t n, void *d) {
    const int64_t grid = ceil_div(n, LN_NT * 4);
    if (grid > 0x7fffffffll) return fl_fail(FL_ERR_ARG, "linear_backward: too many values for one launch (shape)");
    FL_LAUNCH("k_act_grad", k_act_grad<T>, dim3((unsigned)grid), dim3(LN_NT), 0, st, (const T *)gy, pre, n, act,
              (T *)d);
    return fl_check_launch("linear_backward");
}

// The backward's workspace: d (when there is an activation), the parts of dW
// and those of db.
struct BackwardSpace {
    size_t d, dw, db, bytes;
};

BackwardSpace backward_space(const fl_linear *op, int with_dw, int with_db) {
    BackwardSpace s{0, 0, 0, 0};
    const auto take = [&](size_t n) {
        const size_t at = s.bytes;
        s.bytes += (n + 255) / 256 * 256;
        return at;
    };
    if (op->act != FL_ACT_NONE) s.d = take((size_t)op->M * op->N * (op->dtype == FL_F32 ? 4 : 2));
    const int64_t tiles = outer_tiles(op);
    if (with_dw && tiles) {
        const int parts = outer_parts(op->M, op->groups, tiles);
        s.dw = take(parts > 1 ? (size_t)parts * op->groups * op->N * op->K * 4 : 0);
    }
    if (with_db && op->N) s.db = take((size_t)sum_parts(op->M, op->N, op->groups) * op->groups * op->N * 4);
    return s;
}

template <typename T>
int backward(hipStream_t st, const fl_linear *op, const void *gy, const float *pre, void *dx, void *dw, void *db,
             int db_f32, char *ws) {
    const BackwardSpace s = backward_space(op, dw != nullptr, db != nullptr);
    const void *d = gy;
    int rc = FL_OK;
    if (op->act != FL_ACT_NONE && op->M && op->N) {
        rc = act_grad<T>(st, op->act, gy, pre, op->M * op->N, ws + s.d);
        d = ws + s.d;
    }
    if (!rc && dx && op->M && op->K) rc = input_grad<T>(st, op, d, dx);
    if (!rc && dw && op->N && op->K) rc = weight_grad<T>(st, op, d, dw, (float *)(ws + s.dw));
    if (!rc && db && op->N) rc = bias_grad<T>(st, op, d, db, db_f32, (float *)(ws + s.db));
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

int fl_linear_forward(void *stream, const fl_linear *op, void *y, float *pre) {
    const int rc = fl::check_op(op, "linear_forward");
    if (rc) return rc;
    if (op->M == 0 || op->N == 0) return FL_OK;
    if (!y || (op->K > 0 && (!op->x || !op->weight)))
        return fl::fl_fail(FL_ERR_ARG, "linear_forward: null pointer");
    FL_BY_TYPE(op->dtype, fl::forward<T>((hipStream_t)stream, op, y, pre))
}

size_t fl_linear_backward_bytes(const fl_linear *op, int with_dw, int with_db) {
    if (!op || op->M < 0 || op->N < 0 || op->K < 0 || op->groups < 1) return 0;
    return fl::backward_space(op, with_dw, with_db).bytes;
}

int fl_linear_backward(void *stream, const fl_linear *op, const void *gy, const float *pre, void *dx, void *dw,
                       void *db, int db_f32, void *ws, size_t ws_bytes) {
    const int rc = fl::check_op(op, "linear_backward");
    if (rc) return rc;
    const bool any = op->M > 0 && op->N > 0;
    if ((any && (!gy || (op->act != FL_ACT_NONE && !pre))) || (any && dx && op->K > 0 && !op->weight) ||
        (any && dw && op->K > 0 && !op->x))
        return fl::fl_fail(FL_ERR_ARG, "linear_backward: null pointer");
    const size_t need = fl_linear_backward_bytes(op, dw != nullptr, db != nullptr);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "linear_backward: workspace too small");
    FL_BY_TYPE(op->dtype, fl::backward<T>((hipStream_t)stream, op, gy, pre, dx, dw, db, db_f32, (char *)ws))
}

}  // extern "C"
