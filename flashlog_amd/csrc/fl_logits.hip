// Constraints on logits and scores, the row softmax over what they leave, and
// the gradients of both.  For column j of row i, whose owner (the query of
// row i) has group g and a history of ids, with c = how often j is in it:
//
//   u = x + bias[g][j]
//   if c > 0: u = u > 0 ? u / repetition : u * repetition,
//             u -= presence + frequency c
//   v = u / temperature;   not allowed[g][j] -> `fill` (the softmax: 0)
//
//   softmax: w = exp(v - max) / sum over the allowed columns; a row with
//   nothing left (no column allowed, or all of them -inf) is all zeros
//   gradients: dv = g (softmax: w (g - sum w g)), dx = dv allowed slope with
//   slope = 1/temperature, for c > 0 times 1/repetition or repetition by the
//   sign of x + bias; dbias[g] = the sum of the dx of the group's rows
//
// All of it is one pass over the rows: HBM-bound, bytes = one read and one
// write of the rows (the gradients: what the slopes need besides).  A
// workgroup takes one row's segment of NT * 4 * VPT columns in registers
// (rows of up to 8192 columns whole; the softmax of longer rows joins the
// segments' maxima and sums in a second launch), a thread groups of 4 columns
// (16 or 8 bytes a load).  Masks are one bit a column; the repeats of the
// segment's columns are counted with LDS atomics (integers, so the order does
// not matter), once per segment.
//
// dbias adds fp32 terms in a fixed order: a workgroup keeps one table row's
// segment in registers and walks the group's rows, writing their dx on the
// way; groups of many rows are cut into parts whose sums are joined in order.
// The terms are the unrounded ones, so half-precision logits give the same
// dbias as fp32 ones.
#include "fl_abi.h"
#include "fl_common.h"

namespace fl {
namespace {

constexpr int LG_LONG = 8192;      // longest row held by one workgroup
constexpr int LG_SEG_VPT = 4;      // columns of a segment of longer rows: 256 * 4 * 4

enum { LG_CONSTRAIN = 0, LG_SOFTMAX = 1, LG_STATS = 2, LG_JOINED = 3 };

template <typename T>
struct Quad {
    T v[4];
};
template <typename T>
__device__ __forceinline__ Quad<T> load_quad(const T *p, int64_t left) {
    Quad<T> r;
    if (left >= 4) __builtin_memcpy(&r, p, sizeof(r));
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[e] = e < left ? p[e] : (T)0.0f;
    return r;
}
template <typename T>
__device__ __forceinline__ void store_quad(T *p, const Quad<T> &r, int64_t left) {
    if (left >= 4) __builtin_memcpy(p, &r, sizeof(r));
    else
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) p[e] = r.v[e];
}

struct LogitArgs {
    fl_logits op;
    float inv_temperature, inv_repetition;
    uint32_t segments;
};

// What a row's owner constrains it by.
struct RowView {
    const uint32_t *allowed;  // null: every column
    const float *bias;        // null: none
    const int64_t *ids;
    int64_t nids;
    bool none;                // nothing is allowed: the group is outside the tables
};

__device__ __forceinline__ RowView row_view(const fl_logits &op, int64_t row) {
    RowView r{nullptr, nullptr, nullptr, 0, false};
    const int64_t owner = (uint32_t)row / (uint32_t)op.inner;  // rows < 2^31
    int64_t g = 0;
    if (op.allowed_rows > 1 || op.bias_rows > 1) {
        g = op.group[owner];
        r.none = g < 0 || (op.allowed_rows > 1 && g >= op.allowed_rows) || (op.bias_rows > 1 && g >= op.bias_rows);
    }
    if (r.none) g = 0;
    if (op.allowed) r.allowed = (const uint32_t *)op.allowed + (op.allowed_rows > 1 ? g : 0) * op.allowed_ld;
    if (op.bias) r.bias = op.bias + (op.bias_rows > 1 ? g : 0) * op.cols;
    if (op.history) {
        if (op.history_ptr) {
            int64_t b = op.history_ptr[owner], e = op.history_ptr[owner + 1];
            b = b < 0 ? 0 : b > op.history_len ? op.history_len : b;
            e = e < b ? b : e > op.history_len ? op.history_len : e;
            r.ids = op.history + b;
            r.nids = e - b;
        } else {
            r.ids = op.history + owner * op.history_len;
            r.nids = op.history_len;
        }
    }
    return r;
}

template <int NT>
__device__ __forceinline__ float block_max(float v, float *red) {
#pragma unroll
    for (int o = FL_WAVE / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, FL_WAVE));
    if (NT == FL_WAVE) return v;
    if (fl_lane() == 0) red[fl_wave_id()] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NT / FL_WAVE; ++w) v = fmaxf(v, red[w]);
    __syncthreads();
    return v;
}

template <int NT>
__device__ __forceinline__ float block_sum(float v, float *red) {
    v = fl_wave_sum_f32(v);
    if (NT == FL_WAVE) return v;
    if (fl_lane() == 0) red[fl_wave_id()] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NT / FL_WAVE; ++w) v += red[w];
    __syncthreads();
    return v;
}

// Counts the ids of the row's history that fall into [base, base + SEG).
template <int NT, int SEG>
__device__ __forceinline__ void count_repeats(const RowView &r, int64_t base, int64_t cols, int *cnt) {
    __syncthreads();  // the last row's counts are read
    for (int i = threadIdx.x; i < SEG; i += NT) cnt[i] = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < r.nids; i += NT) {
        const int64_t id = r.ids[i];
        if (id >= base && id < base + SEG && id < cols) atomicAdd(&cnt[id - base], 1);
    }
    __syncthreads();
}

// The allowed bits of columns c .. c + 3 (those below cols).
__device__ __forceinline__ unsigned quad_bits(const RowView &r, int64_t c, int64_t cols) {
    if (c >= cols || r.none) return 0;
    unsigned b = r.allowed ? (r.allowed[c >> 5] >> (c & 31)) & 15u : 15u;
    return cols - c < 4 ? b & ((1u << (cols - c)) - 1) : b;
}

__device__ __forceinline__ float constrained(const LogitArgs &a, float x, float b, int c) {
    float u = x + b;
    if (c > 0) {
        u = u > 0.0f ? u * a.inv_repetition : u * a.op.repetition;
        u -= a.op.presence + a.op.frequency * (float)c;
    }
    return u * a.inv_temperature;
}

// Forward of one row's segment.  LG_STATS: the segment's maximum and sum to
// stats; LG_JOINED: the softmax with the row's joined statistics.
template <typename T, int NT, int VPT, int MODE, bool HIST>
__global__ __launch_bounds__(NT) void k_logits(LogitArgs a, void *out, float2 *stats) {
    constexpr int SEG = NT * 4 * VPT;
    __shared__ float red[NT / FL_WAVE];
    __shared__ int cnt[HIST ? SEG : 1];
    const int64_t cols = a.op.cols;
    const int64_t row = blockIdx.x / a.segments;
    const int64_t base = (int64_t)(blockIdx.x % a.segments) * SEG;
    const RowView r = row_view(a.op, row);
    const T *x = (const T *)a.op.x + row * a.op.ldx;
    float v[VPT][4];
    unsigned ok = 0;
    if (HIST) count_repeats<NT, SEG>(r, base, cols, cnt);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int local = (i * NT + threadIdx.x) * 4;
        const int64_t c = base + local;
        const unsigned bits = quad_bits(r, c, cols);
        ok |= bits << (4 * i);
        if (c >= cols) continue;
        const Quad<T> q = load_quad(x + c, cols - c);
        Quad<float> b{{0, 0, 0, 0}};
        if (r.bias) b = load_quad(r.bias + c, cols - c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[i][e] = constrained(a, (float)q.v[e], b.v[e], HIST ? cnt[local + e] : 0);
    }
    if constexpr (MODE == LG_CONSTRAIN) {
        T *y = (T *)out + row * cols;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + (i * NT + threadIdx.x) * 4;
            if (c >= cols) continue;
            Quad<T> q;
#pragma unroll
            for (int e = 0; e < 4; ++e) q.v[e] = (T)((ok >> (4 * i + e)) & 1 ? v[i][e] : a.op.fill);
            store_quad(y + c, q, cols - c);
        }
        return;
    }
    float m = -__builtin_inff(), s = 0.0f;
    if constexpr (MODE == LG_JOINED) {
        const float2 *st = stats + row * a.segments;
        for (int64_t i = threadIdx.x; i < a.segments; i += NT) m = fmaxf(m, st[i].x);
        m = block_max<NT>(m, red);
        if (m == -__builtin_inff()) m = 0.0f;
        for (int64_t i = threadIdx.x; i < a.segments; i += NT) s += st[i].y * expf(st[i].x - m);
        s = block_sum<NT>(s, red);
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((ok >> (4 * i + e)) & 1) m = fmaxf(m, v[i][e]);
        m = block_max<NT>(m, red);
        if (m == -__builtin_inff()) m = MODE == LG_STATS ? m : 0.0f;
    }
    const float shift = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[i][e] = (ok >> (4 * i + e)) & 1 ? expf(v[i][e] - shift) : 0.0f;
            if (MODE != LG_JOINED) s += v[i][e];
        }
    if (MODE != LG_JOINED) s = block_sum<NT>(s, red);
    if constexpr (MODE == LG_STATS) {
        // a segment of nothing but NaN keeps its sum: a maximum of 0 lets it through
        if (threadIdx.x == 0) stats[blockIdx.x] = make_float2(m == -__builtin_inff() && s != s ? 0.0f : m, s);
        return;
    }
    const float inv = 1.0f / (s == 0.0f ? 1.0f : s);
    float *y = (float *)out + row * cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int64_t c = base + (i * NT + threadIdx.x) * 4;
        if (c >= cols) continue;
        Quad<float> q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q.v[e] = v[i][e] * inv;
        store_quad(y + c, q, cols - c);
    }
}

struct GradArgs {
    LogitArgs l;
    const void *g;        // gradient of the output (T; the softmax: float)
    const float *w;       // the softmax's output
    const float *dots;    // [rows] sum w g, of rows longer than a segment
    void *dx;
    float *dbias;         // [parts][bias_rows][cols], or null
    const int32_t *order, *offsets;  // owners by group (null: every row its own list, or one list of all)
    int64_t lists;        // row lists (groups and one of no group; without dbias the rows)
    uint32_t parts;
};

// sum w g of one segment of a row.
template <int NT, int VPT>
__global__ __launch_bounds__(NT) void k_logits_dot(LogitArgs a, const float *__restrict__ g,
                                                   const float *__restrict__ w, float *__restrict__ dots) {
    constexpr int SEG = NT * 4 * VPT;
    __shared__ float red[NT / FL_WAVE];
    const int64_t cols = a.op.cols, row = blockIdx.x / a.segments;
    const int64_t base = (int64_t)(blockIdx.x % a.segments) * SEG;
    const RowView r = row_view(a.op, row);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int64_t c = base + (i * NT + threadIdx.x) * 4;
        const unsigned bits = quad_bits(r, c, cols);
        if (!bits) continue;
        const Quad<float> p = load_quad(w + row * cols + c, cols - c), q = load_quad(g + row * cols + c, cols - c);
#pragma unroll
        for (int e = 0; e < 4; ++e) s += (bits >> e) & 1 ? p.v[e] * q.v[e] : 0.0f;
    }
    s = block_sum<NT>(s, red);
    if (threadIdx.x == 0) dots[blockIdx.x] = s;
}

__global__ __launch_bounds__(FL_WAVE) void k_logits_join(const float *__restrict__ part, int64_t segments,
                                                         float *__restrict__ dots) {
    const int64_t row = blockIdx.x;
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < segments; i += FL_WAVE) s += part[row * segments + i];
    s = fl_wave_sum_f32(s);
    if (threadIdx.x == 0) dots[row] = s;
}

// Gradients of the rows of a list (a part of them), one segment of columns.
template <typename T, int NT, int VPT, bool SOFTMAX, bool HIST, bool WHOLE>
__global__ __launch_bounds__(NT) void k_logits_grad(GradArgs a) {
    constexpr int SEG = NT * 4 * VPT;
    __shared__ float red[NT / FL_WAVE];
    __shared__ int cnt[HIST ? SEG : 1];
    const fl_logits &op = a.l.op;
    const int64_t cols = op.cols;
    const uint32_t item = blockIdx.x / a.l.segments;
    const int64_t base = (int64_t)(blockIdx.x % a.l.segments) * SEG;
    const uint32_t part = item % a.parts;
    const int64_t list = item / a.parts;
    int64_t first = list, count = 1;  // rows (without a plan) or places of owners
    if (a.dbias) {
        const int64_t owners = op.rows / op.inner;
        first = a.order ? (int64_t)a.offsets[list] : 0;
        count = ((a.order && list + 1 < a.lists ? (int64_t)a.offsets[list + 1] : owners) - first) * op.inner;
    }
    const int64_t q0 = count * part / a.parts, q1 = count * (part + 1) / a.parts;
    float acc[VPT][4];
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
    for (int64_t q = q0; q < q1; ++q) {
        int64_t row = first;
        if (a.dbias) {
            const uint32_t inner = (uint32_t)op.inner, at = (uint32_t)q / inner;
            const int64_t place = first + at;
            row = (a.order ? (int64_t)a.order[place] : place) * inner + ((uint32_t)q - at * inner);
        }
        const RowView r = row_view(op, row);
        if (HIST) count_repeats<NT, SEG>(r, base, cols, cnt);
        float d[VPT][4];
        Quad<float> w[VPT];
        unsigned ok = 0;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + (i * NT + threadIdx.x) * 4;
            const unsigned bits = quad_bits(r, c, cols);
            ok |= bits << (4 * i);
            if (c >= cols) continue;
            if (SOFTMAX) {
                const Quad<float> g = load_quad((const float *)a.g + row * cols + c, cols - c);
                w[i] = load_quad(a.w + row * cols + c, cols - c);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    d[i][e] = g.v[e];
                    if (WHOLE) s += (bits >> e) & 1 ? w[i].v[e] * g.v[e] : 0.0f;
                }
            } else {
                const Quad<T> g = load_quad((const T *)a.g + row * cols + c, cols - c);
#pragma unroll
                for (int e = 0; e < 4; ++e) d[i][e] = (float)g.v[e];
            }
        }
        if (SOFTMAX) s = WHOLE ? block_sum<NT>(s, red) : a.dots[row];
        const T *x = (const T *)op.x + row * op.ldx;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int local = (i * NT + threadIdx.x) * 4;
            const int64_t c = base + local;
            if (c >= cols) continue;
            float slope[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) slope[e] = a.l.inv_temperature;
            if (HIST) {
                const Quad<T> xq = load_quad(x + c, cols - c);
                Quad<float> b{{0, 0, 0, 0}};
                if (r.bias) b = load_quad(r.bias + c, cols - c);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (cnt[local + e] > 0)
                        slope[e] *= (float)xq.v[e] + b.v[e] > 0.0f ? a.l.inv_repetition : op.repetition;
            }
            Quad<T> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float t = SOFTMAX ? w[i].v[e] * (d[i][e] - s) : d[i][e];
                const float u = (ok >> (4 * i + e)) & 1 ? t * slope[e] : 0.0f;
                acc[i][e] += u;
                o.v[e] = (T)u;
            }
            if (a.dx) store_quad((T *)a.dx + row * cols + c, o, cols - c);
        }
    }
    if (a.dbias && list < op.bias_rows) {
        float *b = a.dbias + ((int64_t)part * op.bias_rows + list) * cols;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + (i * NT + threadIdx.x) * 4;
            if (c >= cols) continue;
            store_quad(b + c, Quad<float>{{acc[i][0], acc[i][1], acc[i][2], acc[i][3]}}, cols - c);
        }
    }
}

__global__ __launch_bounds__(256) void k_logits_parts(const float *__restrict__ part, int parts, int64_t n,
                                                      float *__restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int p = 0; p < parts; ++p) s += part[(int64_t)p * n + i];
        out[i] = s;
    }
}

// One bit a column of a byte mask, 32 columns a word.
__global__ __launch_bounds__(256) void k_pack_bits(const uint8_t *__restrict__ mask, int64_t rows, int64_t cols,
                                                   int64_t words, uint32_t *__restrict__ out) {
    const int64_t per = (cols + FL_WAVE - 1) / FL_WAVE;  // ballots a row
    const int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) / FL_WAVE;
    if (t >= rows * per) return;
    const int64_t row = t / per, c = (t % per) * FL_WAVE + fl_lane();
    const unsigned long long b = __ballot(c < cols && mask[row * cols + c] != 0);
    const int64_t w = (t % per) * 2;
    if (fl_lane() < 2 && w + fl_lane() < words) out[row * words + w + fl_lane()] = (uint32_t)(b >> (32 * fl_lane()));
}

int64_t lg_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t seg_cols(int64_t cols, bool softmax) {
    if (cols <= 256) return 256;
    if (cols <= 1024) return 1024;
    if (cols <= 2048) return 2048;
    if (softmax && cols <= LG_LONG) return LG_LONG;
    return 256 * 4 * LG_SEG_VPT;
}

bool lg_long(int64_t cols) { return cols > LG_LONG; }

int lg_check(const fl_logits *op, const char *what) {
    if (!op) return fl_fail(FL_ERR_ARG, "%s: null operator", what);
    if (op->dtype < FL_F32 || op->dtype > FL_F16) return fl_fail(FL_ERR_ARG, "%s: unknown type", what);
    if (op->rows < 0 || op->cols < 0 || op->inner < 1 || op->rows % op->inner)
        return fl_fail(FL_ERR_ARG, "%s: bad shape", what);
    if (!(op->temperature > 0.0f) || !(op->repetition > 0.0f))
        return fl_fail(FL_ERR_ARG, "%s: temperature and repetition must lie in the range (0, inf)", what);
    if (op->allowed && (op->allowed_rows < 1 || op->allowed_ld < lg_ceil(op->cols, 32) ||
                        (op->allowed_rows > 1 && !op->group)))
        return fl_fail(FL_ERR_ARG, "%s: bad shape of the allowed table", what);
    if (op->bias && (op->bias_rows < 1 || (op->bias_rows > 1 && !op->group)))
        return fl_fail(FL_ERR_ARG, "%s: bad shape of the bias table", what);
    if (op->history && op->history_len < 0) return fl_fail(FL_ERR_ARG, "%s: bad shape of the history", what);
    if (op->rows > 0 && op->cols > 0 && !op->x) return fl_fail(FL_ERR_ARG, "%s: null pointer", what);
    const int64_t seg = seg_cols(op->cols, false);
    if (op->cols && op->rows > 0x7fffffffll / lg_ceil(op->cols, seg))
        return fl_fail(FL_ERR_ARG, "%s: too many rows for one launch (shape)", what);
    return FL_OK;
}

LogitArgs lg_args(const fl_logits *op, int64_t seg) {
    LogitArgs a;
    a.op = *op;
    if (!op->allowed) a.op.allowed_rows = 0;
    if (!op->bias) a.op.bias_rows = 0;
    a.inv_temperature = 1.0f / op->temperature;
    a.inv_repetition = 1.0f / op->repetition;
    a.segments = (uint32_t)lg_ceil(op->cols, seg);
    return a;
}

template <typename T, int NT, int VPT, int MODE>
void launch_fwd(hipStream_t st, const fl_logits *op, void *out, float2 *stats) {
    const LogitArgs a = lg_args(op, NT * 4 * VPT);
    const dim3 grid((unsigned)(op->rows * a.segments));
    if (op->history)
        FL_LAUNCH("k_logits", (k_logits<T, NT, VPT, MODE, true>), grid, dim3(NT), 0, st, a, out, stats);
    else
        FL_LAUNCH("k_logits", (k_logits<T, NT, VPT, MODE, false>), grid, dim3(NT), 0, st, a, out, stats);
}

template <typename T, int MODE>
int forward(hipStream_t st, const fl_logits *op, void *out, float2 *stats, const char *what) {
    const int64_t seg = seg_cols(op->cols, MODE == LG_SOFTMAX);
    if (seg == 256) launch_fwd<T, 64, 1, MODE>(st, op, out, stats);
    else if (seg == 1024) launch_fwd<T, 256, 1, MODE>(st, op, out, stats);
    else if (seg == 2048) launch_fwd<T, 256, 2, MODE>(st, op, out, stats);
    else if constexpr (MODE == LG_CONSTRAIN) launch_fwd<T, 256, LG_SEG_VPT, MODE>(st, op, out, stats);
    else if (seg == LG_LONG) launch_fwd<T, 256, LG_LONG / 1024, MODE>(st, op, out, stats);
    else {
        launch_fwd<T, 256, LG_SEG_VPT, LG_STATS>(st, op, out, stats);
        launch_fwd<T, 256, LG_SEG_VPT, LG_JOINED>(st, op, out, stats);
    }
    return fl_check_launch(what);
}

// Row lists of the gradient with a bias table: its groups and, with a plan,
// the owners of no group.
int64_t grad_lists(const fl_logits *op) { return op->bias_rows > 1 ? op->bias_rows + 1 : 1; }

int grad_parts(const fl_logits *op, int64_t lists, int64_t segments) {
    const int64_t want = lg_ceil(2048, lists * segments), most = op->rows / (8 * lists);
    const int64_t p = want < most ? want : most;
    return (int)(p < 1 ? 1 : p > 256 ? 256 : p);
}

template <typename T, int NT, int VPT, bool SOFTMAX, bool WHOLE>
void launch_grad(hipStream_t st, GradArgs &a, const fl_logits *op, float *dbias, float *ws) {
    a.l = lg_args(op, NT * 4 * VPT);
    const bool table = dbias != nullptr;
    a.lists = table ? grad_lists(op) : op->rows;
    a.parts = table ? (uint32_t)grad_parts(op, a.lists, a.l.segments) : 1;
    a.dbias = a.parts > 1 ? ws : dbias;
    const dim3 grid((unsigned)(a.lists * a.parts * a.l.segments));
    if (op->history && op->repetition != 1.0f)  // the slopes need the repeats
        FL_LAUNCH("k_logits_grad", (k_logits_grad<T, NT, VPT, SOFTMAX, true, WHOLE>), grid, dim3(NT), 0, st, a);
    else
        FL_LAUNCH("k_logits_grad", (k_logits_grad<T, NT, VPT, SOFTMAX, false, WHOLE>), grid, dim3(NT), 0, st, a);
    if (a.parts > 1) {
        const int64_t n = op->bias_rows * op->cols;
        FL_LAUNCH("k_logits_parts", k_logits_parts, dim3((unsigned)(lg_ceil(n, 256) < 8192 ? lg_ceil(n, 256) : 8192)),
                  dim3(256), 0, st, ws, (int)a.parts, n, dbias);
    }
}

template <typename T, bool SOFTMAX>
int gradient(hipStream_t st, GradArgs &a, const fl_logits *op, float *dbias, float *ws, const char *what) {
    const int64_t seg = seg_cols(op->cols, SOFTMAX);
    if (seg == 256) launch_grad<T, 64, 1, SOFTMAX, true>(st, a, op, dbias, ws);
    else if (seg == 1024) launch_grad<T, 256, 1, SOFTMAX, true>(st, a, op, dbias, ws);
    else if (seg == 2048) launch_grad<T, 256, 2, SOFTMAX, true>(st, a, op, dbias, ws);
    else if constexpr (!SOFTMAX) launch_grad<T, 256, LG_SEG_VPT, false, true>(st, a, op, dbias, ws);
    else if (seg == LG_LONG) launch_grad<T, 256, LG_LONG / 1024, true, true>(st, a, op, dbias, ws);
    else launch_grad<T, 256, LG_SEG_VPT, true, false>(st, a, op, dbias, ws);
    return fl_check_launch(what);
}

// Floats of workspace: the parts of dbias, then (long softmax) the segments'
// dots and the rows'.
size_t grad_floats(const fl_logits *op, int softmax, int with_dbias, int64_t *dots_at) {
    const int64_t segments = lg_ceil(op->cols, seg_cols(op->cols, softmax != 0));
    size_t n = 0;
    if (with_dbias) {
        const int parts = grad_parts(op, grad_lists(op), segments);
        if (parts > 1) n += (size_t)parts * op->bias_rows * op->cols;
    }
    *dots_at = (int64_t)n;
    if (softmax && lg_long(op->cols)) n += (size_t)op->rows * (segments + 1);
    return n;
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

size_t fl_logits_op_bytes(void) { return sizeof(fl_logits); }

int fl_pack_bits(void *stream, const uint8_t *mask, int64_t rows, int64_t cols, int32_t *words) {
    if (rows < 0 || cols < 0) return fl::fl_fail(FL_ERR_ARG, "pack_bits: bad shape");
    const int64_t waves = rows * fl::lg_ceil(cols, FL_WAVE);
    if (waves == 0) return FL_OK;
    if (!mask || !words) return fl::fl_fail(FL_ERR_ARG, "pack_bits: null pointer");
    if (fl::lg_ceil(waves, 4) > 0x7fffffffll) return fl::fl_fail(FL_ERR_ARG, "pack_bits: too many bits (shape)");
    FL_LAUNCH("k_pack_bits", fl::k_pack_bits, dim3((unsigned)fl::lg_ceil(waves, 4)), dim3(256), 0,
              (hipStream_t)stream, mask, rows, cols, fl::lg_ceil(cols, 32), (uint32_t *)words);
    return fl::fl_check_launch("pack_bits");
}

int fl_logits_constrain(void *stream, const fl_logits *op, void *out) {
    const int rc = fl::lg_check(op, "logits_constrain");
    if (rc) return rc;
    if (op->rows == 0 || op->cols == 0) return FL_OK;
    if (!out) return fl::fl_fail(FL_ERR_ARG, "logits_constrain: null pointer");
    FL_BY_TYPE(op->dtype, (fl::forward<T, fl::LG_CONSTRAIN>((hipStream_t)stream, op, out, nullptr,
                                                            "logits_constrain")))
}

size_t fl_logits_softmax_bytes(const fl_logits *op) {
    if (!op || !fl::lg_long(op->cols)) return 0;
    return (size_t)op->rows * fl::lg_ceil(op->cols, 256 * 4 * fl::LG_SEG_VPT) * sizeof(float2);
}

int fl_logits_softmax(void *stream, const fl_logits *op, float *w, void *ws, size_t ws_bytes) {
    const int rc = fl::lg_check(op, "logits_softmax");
    if (rc) return rc;
    if (op->rows == 0 || op->cols == 0) return FL_OK;
    if (!w) return fl::fl_fail(FL_ERR_ARG, "logits_softmax: null pointer");
    const size_t need = fl_logits_softmax_bytes(op);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "logits_softmax: workspace too small");
    FL_BY_TYPE(op->dtype, (fl::forward<T, fl::LG_SOFTMAX>((hipStream_t)stream, op, w, (float2 *)ws,
                                                          "logits_softmax")))
}

size_t fl_logits_grad_bytes(const fl_logits *op, int softmax, int with_dbias) {
    if (!op || op->rows < 1 || op->cols < 1) return 0;
    int64_t at;
    return fl::grad_floats(op, softmax, with_dbias, &at) * 4;
}

int fl_logits_grad(void *stream, const fl_logits *op, const float *w, const void *grad, const int32_t *order,
                   const int32_t *offsets, void *dx, float *dbias, void *ws, size_t ws_bytes) {
    const int rc = fl::lg_check(op, "logits_grad");
    if (rc) return rc;
    if (op->cols == 0) return FL_OK;
    if (dbias && (!op->bias || (op->bias_rows > 1 && (!order || !offsets))))
        return fl::fl_fail(FL_ERR_ARG, "logits_grad: the gradient of a bias table needs the owners by group");
    if (op->rows > 0 && !grad) return fl::fl_fail(FL_ERR_ARG, "logits_grad: null pointer");
    const size_t need = fl_logits_grad_bytes(op, w != nullptr, dbias != nullptr);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "logits_grad: workspace too small");
    if (op->rows == 0 && !dbias) return FL_OK;
    hipStream_t st = (hipStream_t)stream;
    fl::GradArgs a{};
    a.g = grad;
    a.w = w;
    a.dx = dx;
    if (dbias && op->bias_rows > 1) {
        a.order = order;
        a.offsets = offsets;
    }
    if (w && fl::lg_long(op->cols) && op->rows > 0) {
        int64_t at;
        fl::grad_floats(op, 1, dbias != nullptr, &at);
        const fl::LogitArgs l = fl::lg_args(op, 256 * 4 * fl::LG_SEG_VPT);
        float *part = (float *)ws + at, *dots = part + op->rows * l.segments;
        FL_LAUNCH("k_logits_dot", (fl::k_logits_dot<256, fl::LG_SEG_VPT>), dim3((unsigned)(op->rows * l.segments)),
                  dim3(256), 0, st, l, (const float *)grad, w, part);
        FL_LAUNCH("k_logits_join", fl::k_logits_join, dim3((unsigned)op->rows), dim3(FL_WAVE), 0, st, part,
                  (int64_t)l.segments, dots);
        a.dots = dots;
    }
    if (w) {
        FL_BY_TYPE(op->dtype, (fl::gradient<T, true>(st, a, op, dbias, (float *)ws, "logits_grad")))
    }
    FL_BY_TYPE(op->dtype, (fl::gradient<T, false>(st, a, op, dbias, (float *)ws, "logits_grad")))
}

}  // extern "C"
