// Layer normalisation of rows and its gradients:
//
//   mean = sum x / N,  r = 1 / sqrt(sum (x - mean)^2 / N + eps),  h = (x - mean) r
//   y  = h w + b
//   dx = r (v - mean(v) - h mean(v h)),  v = gy w
//   dw = sum over the rows of gy h,      db = sum over the rows of gy
//
// HBM-bound: one read and one write of the rows forward, two reads and one
// write backward.  A row is in the registers of one wave (up to 512 columns) or
// of a workgroup's four (up to 8192), 16 bytes a lane and load, so that the mean
// is known before the deviations are squared (no cancellation, whatever the
// mean); longer rows are read again for each sum.  mean and r are kept in fp32
// for the backward, 8 bytes a row.  Waves walk the rows with the weight in
// registers and the next row's loads under way.
//
// dw and db: the sums of a lane's columns stay in registers over the walk, waves
// with rows of their own are added through LDS, and a second launch adds the
// workgroups in a fixed order.
//
// [16384 x 2048] bf16: 33 us forward, 46 + 5 backward = 4.1 and 4.4 TB/s (a copy
// 4.7 on the same card); with a wave a row of 2048 columns 35 and 60 + 4, without
// the next row's loads 49 and 56 + 7.
#include "fl_abi.h"
#include "fl_common.h"

namespace fl {
namespace {

constexpr int NM_WAVES = 4;
constexpr int NM_NT = NM_WAVES * FL_WAVE;
constexpr int NM_LANE = 32;                     // most values of a row that a lane holds
constexpr int NM_WAVE_COLS = 512;
constexpr int NM_ROW_COLS = NM_LANE * FL_WAVE * NM_WAVES;
// Most workgroups that walk the rows: forward ([16384 x 2048] bf16, us with 512, 1024,
// 1536, 4096 of them 53, 37, 31, 33) and backward, each of which leaves a row of sums
// (with 512, 1024, 1536, 2048 of them 68 + 4, 46 + 5, 56 + 6, 51 + 8).  Of fewer rows
// not chosen apart: 1536 are one or two a workgroup, 12 + 5 us of 2048 fp32 columns for 8.
constexpr int64_t NM_WALKS = 4096;
constexpr int64_t NM_GRAD_WALKS = 1024;

struct NormArgs {
    const void *x, *gy, *weight, *bias;
    void *y, *dx;
    const float *stats_in;  // [M][2]: mean, r
    float *stats, *part;    // part [workgroups][2][N]
    int64_t M, N, ldx;
    float eps;
    int with_dw;
};

// Four values at a time: columns c .. c + 3 of N, 0 behind the last.
template <typename U>
__device__ __forceinline__ void load_four(const U *row, int64_t c, int64_t N, float (&v)[4]) {
    if (c + 4 <= N) {
        U r[4];
        __builtin_memcpy(r, row + c, sizeof(r));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)r[e];
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < N ? (float)row[c + e] : 0.0f;
}
template <typename U>
__device__ __forceinline__ void store_four(U *row, int64_t c, int64_t N, const float (&v)[4]) {
    if (c + 4 <= N) {
        U r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (U)v[e];
        __builtin_memcpy(row + c, r, sizeof(r));
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < N) row[c + e] = (U)v[e];
}

// G columns of a lane, 16 bytes of the rows' type a load.
template <typename T, typename U>
__device__ __forceinline__ void load_cols(const U *row, int64_t c, int64_t N, float (&v)[16 / sizeof(T)]) {
    constexpr int G = 16 / (int)sizeof(T);
    if (c + G <= N) {
        U r[G];
        __builtin_memcpy(r, row + c, sizeof(r));
#pragma unroll
        for (int e = 0; e < G; ++e) v[e] = (float)r[e];
    } else
#pragma unroll
        for (int e = 0; e < G; ++e) v[e] = c + e < N ? (float)row[c + e] : 0.0f;
}
template <typename T, typename U>
__device__ __forceinline__ void store_cols(U *row, int64_t c, int64_t N, const float (&v)[16 / sizeof(T)]) {
    constexpr int G = 16 / (int)sizeof(T);
    if (c + G <= N) {
        U r[G];
#pragma unroll
        for (int e = 0; e < G; ++e) r[e] = (U)v[e];
        __builtin_memcpy(row + c, r, sizeof(r));
    } else
#pragma unroll
        for (int e = 0; e < G; ++e)
            if (c + e < N) row[c + e] = (U)v[e];
}

// A wave's sum, the same in all lanes: moves within the vector unit (through LDS,
// as shuffles go, a row's two sums took longer than its loads).
__device__ __forceinline__ float wave_sum(float v) {
    const auto add = [&](int moved) { v += __int_as_float(moved); };
    add(fl_dpp<0x111>(__float_as_int(v)));
    add(fl_dpp<0x112>(__float_as_int(v)));
    add(fl_dpp<0x114>(__float_as_int(v)));
    add(fl_dpp<0x118>(__float_as_int(v)));
    add(fl_dpp<0x142, 0xa>(__float_as_int(v)));
    add(fl_dpp<0x143, 0xc>(__float_as_int(v)));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), FL_WAVE - 1));
}

// Sums of S values a thread over the WPR waves of a row.  `lds`: [2][NM_WAVES][S],
// `turn` alternates, so that one barrier a sum is enough.
template <int WPR, int S>
__device__ __forceinline__ void row_sums(float (&v)[S], float *lds, int &turn) {
#pragma unroll
    for (int s = 0; s < S; ++s) v[s] = wave_sum(v[s]);
    if constexpr (WPR > 1) {
        float *at = lds + (turn & 1) * NM_WAVES * 2;
        ++turn;
        if (fl_lane() == 0)
#pragma unroll
            for (int s = 0; s < S; ++s) at[fl_wave_id() * 2 + s] = v[s];
        __syncthreads();
#pragma unroll
        for (int s = 0; s < S; ++s) v[s] = (at[s] + at[2 + s]) + (at[4 + s] + at[6 + s]);
    }
}

// A lane's part of a row as it lies in memory, so that the next row's can be under
// way while this one's is worked on.
template <typename T, int PER>
struct RowPart {
    static constexpr int G = 16 / (int)sizeof(T);
    T v[PER][G];

    // The columns c0 + p step .., 0 behind the last: loads without branches around
    // them (each would be waited for by itself).  The group that a row ends in is
    // read from its last G columns and moved.
    __device__ __forceinline__ void load(const T *row, int c0, int step, int N) {
        if (N < G) {
#pragma unroll
            for (int p = 0; p < PER; ++p)
#pragma unroll
                for (int e = 0; e < G; ++e) v[p][e] = c0 + p * step + e < N ? row[c0 + p * step + e] : (T)0.0f;
            return;
        }
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int c = c0 + p * step;
            __builtin_memcpy(v[p], row + (c < N - G ? c : N - G), sizeof(v[p]));
        }
        if (N % G == 0 && N == PER * step) return;
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int over = c0 + p * step - (N - G);
            if (over <= 0) continue;
#pragma unroll
            for (int d = 1; d < G; d *= 2)
                if (over & d)
#pragma unroll
                    for (int e = 0; e < G; ++e) v[p][e] = e + d < G ? v[p][e + d] : (T)0.0f;
            if (over >= G)
#pragma unroll
                for (int e = 0; e < G; ++e) v[p][e] = (T)0.0f;
        }
    }
};

// PER loads of a lane; WPR waves a row (1 or all), which walk the rows with the
// weight and bias in registers.
template <typename T, typename W, int PER, int WPR>
__global__ __launch_bounds__(NM_NT) void k_norm_rows(NormArgs a) {
    constexpr int G = 16 / (int)sizeof(T);
    __shared__ float lds[2 * NM_WAVES * 2];
    int turn = 0;
    const int64_t first = WPR == 1 ? (int64_t)blockIdx.x * NM_WAVES + fl_wave_id() : blockIdx.x;
    const int64_t stride = (int64_t)gridDim.x * (WPR == 1 ? NM_WAVES : 1);
    if (first >= a.M) return;
    const int64_t N = a.N, c0 = (int64_t)(WPR == 1 ? fl_lane() : threadIdx.x) * G, step = (int64_t)WPR * FL_WAVE * G;
    const T *x = (const T *)a.x;
    const float inv = 1.0f / (float)N;
    RowPart<T, PER> next;
    next.load(x + first * a.ldx, (int)c0, (int)step, (int)N);
    float w[PER][G], b[PER][G];
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        if (a.weight) load_cols<T, W>((const W *)a.weight, c0 + p * step, N, w[p]);
        if (a.bias) load_cols<T, W>((const W *)a.bias, c0 + p * step, N, b[p]);
    }
    for (int64_t row = first; row < a.M; row += stride) {
        float v[PER][G], s[1] = {0.0f};
#pragma unroll
        for (int p = 0; p < PER; ++p)
#pragma unroll
            for (int e = 0; e < G; ++e) {
                v[p][e] = (float)next.v[p][e];
                s[0] += v[p][e];
            }
        if (row + stride < a.M) next.load(x + (row + stride) * a.ldx, (int)c0, (int)step, (int)N);
        row_sums<WPR, 1>(s, lds, turn);
        const float mean = s[0] * inv;
        s[0] = 0.0f;
#pragma unroll
        for (int p = 0; p < PER; ++p)
#pragma unroll
            for (int e = 0; e < G; ++e) {
                v[p][e] = c0 + p * step + e < N ? v[p][e] - mean : 0.0f;
                s[0] = __builtin_fmaf(v[p][e], v[p][e], s[0]);
            }
        row_sums<WPR, 1>(s, lds, turn);
        const float r = 1.0f / sqrtf(s[0] * inv + a.eps);
        if (a.stats && (WPR == 1 ? fl_lane() : (int)threadIdx.x) == 0) {
            a.stats[row * 2] = mean;
            a.stats[row * 2 + 1] = r;
        }
        T *y = (T *)a.y + row * N;
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int64_t c = c0 + p * step;
            if (c >= N) continue;
#pragma unroll
            for (int e = 0; e < G; ++e) {
                float h = v[p][e] * r;
                if (a.weight) h *= w[p][e];
                if (a.bias) h += b[p][e];
                v[p][e] = h;
            }
            store_cols<T, T>(y, c, N, v[p]);
        }
    }
}

// Rows of any length: a workgroup a row, read once for each sum and once more, from the
// caches but for the first: [1024 x 20000] fp32 60 us = 2.7 TB/s of one read and one
// write, bf16 42.
template <typename T, typename W>
__global__ __launch_bounds__(NM_NT) void k_norm_long(NormArgs a) {
    __shared__ float lds[2 * NM_WAVES * 2];
    int turn = 0;
    const int64_t row = fl_block();
    if (row >= a.M) return;
    const int64_t N = a.N;
    const T *x = (const T *)a.x + row * a.ldx;
    float v[4], s[1] = {0.0f};
    for (int64_t c = threadIdx.x * 4; c < N; c += NM_NT * 4) {
        load_four<T>(x, c, N, v);
        s[0] += (v[0] + v[1]) + (v[2] + v[3]);
    }
    row_sums<NM_WAVES, 1>(s, lds, turn);
    const float inv = 1.0f / (float)N, mean = s[0] * inv;
    s[0] = 0.0f;
    for (int64_t c = threadIdx.x * 4; c < N; c += NM_NT * 4) {
        load_four<T>(x, c, N, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float d = c + e < N ? v[e] - mean : 0.0f;
            s[0] = __builtin_fmaf(d, d, s[0]);
        }
    }
    row_sums<NM_WAVES, 1>(s, lds, turn);
    const float r = 1.0f / sqrtf(s[0] * inv + a.eps);
    if (a.stats && threadIdx.x == 0) {
        a.stats[row * 2] = mean;
        a.stats[row * 2 + 1] = r;
    }
    T *y = (T *)a.y + row * N;
    for (int64_t c = threadIdx.x * 4; c < N; c += NM_NT * 4) {
        float w[4], b[4];
        load_four<T>(x, c, N, v);
        if (a.weight) load_four<W>((const W *)a.weight, c, N, w);
        if (a.bias) load_four<W>((const W *)a.bias, c, N, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float h = (v[e] - mean) * r;
            if (a.weight) h *= w[e];
            if (a.bias) h += b[e];
            v[e] = h;
        }
        store_four<T>(y, c, N, v);
    }
}

// dx, and the sums of gy h and gy over the rows that a workgroup walks.
template <typename T, typename W, int PER, int WPR>
__global__ __launch_bounds__(NM_NT) void k_norm_grad(NormArgs a) {
    constexpr int G = 16 / (int)sizeof(T);
    constexpr int OWN = WPR == 1 ? FL_WAVE : NM_NT;  // threads of a row
    __shared__ float lds[2 * NM_WAVES * 2];
    __shared__ float join[WPR == 1 ? NM_WAVES * OWN * G : 1];
    int turn = 0;
    const int64_t N = a.N, first = WPR == 1 ? (int64_t)blockIdx.x * NM_WAVES + fl_wave_id() : blockIdx.x;
    const int64_t stride = (int64_t)gridDim.x * (WPR == 1 ? NM_WAVES : 1);
    const int at = WPR == 1 ? fl_lane() : (int)threadIdx.x;
    const int64_t c0 = (int64_t)at * G, step = (int64_t)OWN * G;
    const float inv = 1.0f / (float)N;
    float w[PER][G], dw[PER][G], db[PER][G];
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        if (a.weight) load_cols<T, W>((const W *)a.weight, c0 + p * step, N, w[p]);
#pragma unroll
        for (int e = 0; e < G; ++e) {
            if (!a.weight) w[p][e] = 1.0f;
            dw[p][e] = db[p][e] = 0.0f;
        }
    }
    RowPart<T, PER> next_x, next_g;
    float2 next_of = {0.0f, 0.0f};
    const auto load = [&](int64_t row) {
        next_x.load((const T *)a.x + row * a.ldx, (int)c0, (int)step, (int)N);
        next_g.load((const T *)a.gy + row * N, (int)c0, (int)step, (int)N);
        next_of = *reinterpret_cast<const float2 *>(a.stats_in + row * 2);
    };
    if (first < a.M) load(first);
    for (int64_t row = first; row < a.M; row += stride) {
        const float mean = next_of.x, r = next_of.y;
        float h[PER][G], g[PER][G], s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < PER; ++p)
#pragma unroll
            for (int e = 0; e < G; ++e) {
                h[p][e] = (float)next_x.v[p][e];
                g[p][e] = (float)next_g.v[p][e];
            }
        if (row + stride < a.M) load(row + stride);
#pragma unroll
        for (int p = 0; p < PER; ++p)
#pragma unroll
            for (int e = 0; e < G; ++e) {
                h[p][e] = (h[p][e] - mean) * r;  // behind the row gy is 0, and nothing is stored
                dw[p][e] = __builtin_fmaf(g[p][e], h[p][e], dw[p][e]);
                db[p][e] += g[p][e];
                g[p][e] *= w[p][e];
                s[0] += g[p][e];
                s[1] = __builtin_fmaf(g[p][e], h[p][e], s[1]);
            }
        if (!a.dx) continue;
        row_sums<WPR, 2>(s, lds, turn);
        const float m1 = s[0] * inv, m2 = s[1] * inv;
        T *dx = (T *)a.dx + row * N;
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int64_t c = c0 + p * step;
            if (c >= N) continue;
#pragma unroll
            for (int e = 0; e < G; ++e) g[p][e] = r * (g[p][e] - m1 - h[p][e] * m2);
            store_cols<T, T>(dx, c, N, g[p]);
        }
    }
    if (!a.with_dw) return;
    float *out = a.part + (int64_t)blockIdx.x * 2 * N;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const int64_t c = c0 + p * step;
        if constexpr (WPR > 1) {
            if (c < N) {
                store_cols<T, float>(out, c, N, dw[p]);
                store_cols<T, float>(out + N, c, N, db[p]);
            }
        } else
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < G; ++e)
                    join[(fl_wave_id() * G + e) * FL_WAVE + fl_lane()] = which ? db[p][e] : dw[p][e];
                __syncthreads();
                // wave w adds columns e = w, w + 4, .. of every lane
                for (int e = fl_wave_id(); e < G; e += NM_WAVES) {
                    float t = 0.0f;
#pragma unroll
                    for (int k = 0; k < NM_WAVES; ++k) t += join[(k * G + e) * FL_WAVE + fl_lane()];
                    if (c + e < N) out[which * N + c + e] = t;
                }
            }
    }
}

// dx of rows of any length: [1024 x 20000] fp32 64 us = 3.8 TB/s of two reads and one
// write, bf16 49.
template <typename T, typename W>
__global__ __launch_bounds__(NM_NT) void k_norm_long_grad(NormArgs a) {
    __shared__ float lds[2 * NM_WAVES * 2];
    int turn = 0;
    const int64_t row = fl_block();
    if (row >= a.M) return;
    const int64_t N = a.N;
    const T *x = (const T *)a.x + row * a.ldx, *gy = (const T *)a.gy + row * N;
    const float mean = a.stats_in[row * 2], r = a.stats_in[row * 2 + 1], inv = 1.0f / (float)N;
    float s[2] = {0.0f, 0.0f};
    const auto pieces = [&](int64_t c, float (&h)[4], float (&g)[4]) {
        load_four<T>(x, c, N, h);
        load_four<T>(gy, c, N, g);
        float w[4];
        if (a.weight) load_four<W>((const W *)a.weight, c, N, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            h[e] = (h[e] - mean) * r;
            if (a.weight) g[e] *= w[e];
        }
    };
    float h[4], g[4];
    for (int64_t c = threadIdx.x * 4; c < N; c += NM_NT * 4) {
        pieces(c, h, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[0] += g[e];
            s[1] = __builtin_fmaf(g[e], h[e], s[1]);
        }
    }
    row_sums<NM_WAVES, 2>(s, lds, turn);
    const float m1 = s[0] * inv, m2 = s[1] * inv;
    T *dx = (T *)a.dx + row * N;
    for (int64_t c = threadIdx.x * 4; c < N; c += NM_NT * 4) {
        pieces(c, h, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = r * (g[e] - m1 - h[e] * m2);
        store_four<T>(dx, c, N, g);
    }
}

// The sums over a part of the rows, a column a thread: [1024 x 20000] fp32 29 us = 5.6
// TB/s, bf16 24.
template <typename T>
__global__ __launch_bounds__(NM_NT) void k_norm_cols(NormArgs a, int parts) {
    const int64_t blocks = (a.N + NM_NT - 1) / NM_NT, item = fl_block();
    const int64_t part = item / blocks, c = (item % blocks) * NM_NT + threadIdx.x;
    if (part >= parts || c >= a.N) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = a.M * part / parts; row < a.M * (part + 1) / parts; ++row) {
        const float g = (float)((const T *)a.gy)[row * a.N + c], x = (float)((const T *)a.x)[row * a.ldx + c];
        dw = __builtin_fmaf(g, (x - a.stats_in[row * 2]) * a.stats_in[row * 2 + 1], dw);
        db += g;
    }
    a.part[part * 2 * a.N + c] = dw;
    a.part[(part * 2 + 1) * a.N + c] = db;
}

// dw and db from the parts: 64 columns and sixteen runs of the parts a workgroup,
// each in order, then the runs.
constexpr int NM_FOLD = 16;

template <typename W>
__global__ __launch_bounds__(NM_FOLD *FL_WAVE) void k_norm_fold(const float *__restrict__ part, int parts, int64_t N,
                                                                 W *__restrict__ dw, W *__restrict__ db) {
    __shared__ float runs[NM_FOLD][FL_WAVE];
    const int64_t i = fl_block() * FL_WAVE + fl_lane();
    float s = 0.0f;
    if (i < 2 * N) {
        int p = parts * fl_wave_id() / NM_FOLD;
        const int p1 = parts * (fl_wave_id() + 1) / NM_FOLD;
        for (; p + 8 <= p1; p += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = part[(int64_t)(p + j) * 2 * N + i];
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
        }
        for (; p < p1; ++p) s += part[(int64_t)p * 2 * N + i];
    }
    runs[fl_wave_id()][fl_lane()] = s;
    __syncthreads();
    if (fl_wave_id() || i >= 2 * N) return;
    W *to = i < N ? dw : db;
    if (!to) return;
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < NM_FOLD; ++w) s += runs[w][fl_lane()];
    to[i < N ? i : i - N] = (W)s;
}

// Workgroups that walk the rows for dw and db.
int grad_groups(const fl_norm *op, bool with_dw) {
    const int64_t rows = op->N <= NM_WAVE_COLS ? NM_WAVES : 1;
    const int64_t all = (op->M + rows - 1) / rows;
    if (op->N > NM_ROW_COLS) {
        const int64_t p = op->M / 32;
        return (int)(p < 1 ? 1 : p > 64 ? 64 : p);
    }
    const int64_t most = with_dw ? NM_GRAD_WALKS : 1 << 22;
    return (int)(all < most ? all : most);
}

int check_op(const fl_norm *op, const char *what) {
    if (!op) return fl_fail(FL_ERR_ARG, "%s: null operator", what);
    if (op->dtype < FL_F32 || op->dtype > FL_F16) return fl_fail(FL_ERR_ARG, "%s: unknown type", what);
    if (op->M < 0 || op->N < 0 || op->M > 0x7fffffffll || op->N > 0x7fffffffll)
        return fl_fail(FL_ERR_ARG, "%s: bad shape", what);
    if (op->M && op->N && !op->x) return fl_fail(FL_ERR_ARG, "%s: null pointer", what);
    return FL_OK;
}

NormArgs args_of(const fl_norm *op) {
    NormArgs a{};
    a.x = op->x;
    a.ldx = op->ldx;
    a.weight = op->weight;
    a.bias = op->bias;
    a.M = op->M;
    a.N = op->N;
    a.eps = op->eps;
    return a;
}

// f(PER, WPR) for rows of N columns, PER a power of two.
template <typename T, typename F>
void by_cols(int64_t N, F &&f) {
    constexpr int G = 16 / (int)sizeof(T);
    const int wide = N > NM_WAVE_COLS;
    const int64_t per = (N + (int64_t)FL_WAVE * (wide ? NM_WAVES : 1) * G - 1) / ((int64_t)FL_WAVE * (wide ? NM_WAVES : 1) * G);
    const auto by_per = [&](auto wpr) {
        if (per <= 1) return f(std::integral_constant<int, 1>(), wpr);
        if (per <= 2) return f(std::integral_constant<int, 2>(), wpr);
        if (per <= 4 || G == 8) return f(std::integral_constant<int, 4>(), wpr);
        return f(std::integral_constant<int, NM_LANE / G>(), wpr);
    };
    if (wide) by_per(std::integral_constant<int, NM_WAVES>());
    else by_per(std::integral_constant<int, 1>());
}

template <typename T, typename W>
int forward(hipStream_t st, const fl_norm *op, void *y, float *stats) {
    NormArgs a = args_of(op);
    a.y = y;
    a.stats = stats;
    if (op->N > NM_ROW_COLS) {
        FL_LAUNCH("k_norm_long", (k_norm_long<T, W>), grid_of(op->M), dim3(NM_NT), 0, st, a);
        return fl_check_launch("layer_norm");
    }
    by_cols<T>(op->N, [&](auto per, auto wpr) {
        constexpr int PER = decltype(per)::value, WPR = decltype(wpr)::value;
        const int64_t rows = WPR == 1 ? NM_WAVES : 1, all = (op->M + rows - 1) / rows;
        FL_LAUNCH("k_norm_rows", (k_norm_rows<T, W, PER, WPR>), dim3((unsigned)(all < NM_WALKS ? all : NM_WALKS)),
                  dim3(NM_NT), 0, st, a);
    });
    return fl_check_launch("layer_norm");
}

template <typename T, typename W>
int backward(hipStream_t st, const fl_norm *op, const void *gy, const float *stats, void *dx, void *dw, void *db,
             float *ws) {
    NormArgs a = args_of(op);
    a.gy = gy;
    a.dx = dx;
    a.stats_in = stats;
    a.part = ws;
    a.with_dw = dw || db;
    const int groups = grad_groups(op, a.with_dw);
    if (op->N > NM_ROW_COLS) {
        if (dx) FL_LAUNCH("k_norm_long_grad", (k_norm_long_grad<T, W>), grid_of(op->M), dim3(NM_NT), 0, st, a);
        if (a.with_dw)
            FL_LAUNCH("k_norm_cols", k_norm_cols<T>, grid_of((int64_t)groups * ((op->N + NM_NT - 1) / NM_NT)),
                      dim3(NM_NT), 0, st, a, groups);
    } else
        by_cols<T>(op->N, [&](auto per, auto wpr) {
            constexpr int PER = decltype(per)::value, WPR = decltype(wpr)::value;
            FL_LAUNCH("k_norm_grad", (k_norm_grad<T, W, PER, WPR>), dim3(groups), dim3(NM_NT), 0, st, a);
        });
    if (a.with_dw)
        FL_LAUNCH("k_norm_fold", k_norm_fold<W>, grid_of((2 * op->N + FL_WAVE - 1) / FL_WAVE),
                  dim3(NM_FOLD * FL_WAVE), 0, st, ws,
                  groups, op->N, (W *)dw, (W *)db);
    return fl_check_launch("layer_norm");
}

}  // namespace
}  // namespace fl

// T: the rows' type, W: the weight's and bias's.
#define FL_BY_TYPES(op, call)                                                                 \
    switch ((op)->dtype) {                                                                    \
        case FL_F32: { using T = float; using W = float; return call; }                       \
        case FL_BF16: {                                                                       \
            using T = __bf16;                                                                 \
            if ((op)->wide) { using W = float; return call; }                                 \
            using W = __bf16;                                                                 \
            return call;                                                                      \
        }                                                                                     \
        default: {                                                                            \
            using T = _Float16;                                                               \
            if ((op)->wide) { using W = float; return call; }                                 \
            using W = _Float16;                                                               \
            return call;                                                                      \
        }                                                                                     \
    }

extern "C" {

size_t fl_norm_op_bytes(void) { return sizeof(fl_norm); }

int fl_norm_forward(void *stream, const fl_norm *op, void *y, float *stats) {
    const int rc = fl::check_op(op, "layer_norm");
    if (rc) return rc;
    if (op->M == 0 || op->N == 0) return FL_OK;
    if (!y) return fl::fl_fail(FL_ERR_ARG, "layer_norm: null pointer");
    FL_BY_TYPES(op, (fl::forward<T, W>((hipStream_t)stream, op, y, stats)))
}

size_t fl_norm_backward_bytes(const fl_norm *op, int with_dw) {
    if (!op || op->M < 1 || op->N < 1 || !with_dw) return 0;
    return (size_t)fl::grad_groups(op, true) * 2 * op->N * 4;
}

int fl_norm_backward(void *stream, const fl_norm *op, const void *gy, const float *stats, void *dx, void *dw, void *db,
                     void *ws, size_t ws_bytes) {
    const int rc = fl::check_op(op, "layer_norm");
    if (rc) return rc;
    if (op->N == 0 || (op->M == 0 && !dw && !db)) return FL_OK;
    if (op->M == 0) return fl::fl_fail(FL_ERR_ARG, "layer_norm: no rows (shape)");
    if (!gy || !stats) return fl::fl_fail(FL_ERR_ARG, "layer_norm: null pointer");
    const size_t need = fl_norm_backward_bytes(op, dw || db);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "layer_norm: workspace too small");
    FL_BY_TYPES(op, (fl::backward<T, W>((hipStream_t)stream, op, gy, stats, dx, dw, db, (float *)ws)))
}

}  // extern "C"
