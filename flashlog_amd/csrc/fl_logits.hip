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
// write of the rows.  Rows of up to 2048 columns are a wave's each, held in
// registers (up to 8 groups of 4 columns a lane), so that nothing waits for
// other waves; longer ones are cut into segments of 4096 columns, a workgroup
// each (the softmax: up to 8192 whole, beyond that the segments' maxima and
// sums are joined by a second launch).
//
// Masks are one bit a column.  Histories are short next to the rows: up to 8
// ids are compared with the columns in registers, more are looked at first and
// only a segment that holds some of them counts them in LDS (integers, so the
// order does not matter); the slopes read the logits of repeated columns only.
//
// dbias adds fp32 terms in a fixed order.  A workgroup keeps one table row's
// columns in registers and walks the group's rows, writing their dx on the
// way (rows of up to 2048 columns: four waves, a row each, joined in LDS);
// groups of many rows are cut into parts.  The terms are the unrounded ones,
// so half-precision logits give the same dbias as fp32 ones.
#include "fl_abi.h"
#include "fl_common.h"
#include "fl_parts.h"
#include <type_traits>

namespace fl {
namespace {

constexpr int LG_WAVE_COLS = 2048;  // longest row held by a wave
constexpr int LG_LONG = 8192;       // longest row held by a workgroup
constexpr int LG_NT = 256;
constexpr int LG_WAVES = LG_NT / FL_WAVE;
constexpr int LG_VPT = 4;           // groups of 4 columns a thread of a segment
constexpr int LG_SEG = LG_NT * 4 * LG_VPT;
constexpr int LG_FEW = 8;           // ids compared in registers

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

// Threads that share a row: a wave (nothing to wait for) or a workgroup.
template <int NT>
__device__ __forceinline__ void team_sync() {
    if (NT == FL_WAVE) fl_wave_sync();
    else __syncthreads();
}
template <int NT>
__device__ __forceinline__ bool team_any(bool v) {
    if (NT == FL_WAVE) return __any(v);
    return __syncthreads_or(v);
}
template <int NT>
__device__ __forceinline__ int team_thread() {
    return NT == FL_WAVE ? fl_lane() : (int)threadIdx.x;
}

template <int NT>
__device__ __forceinline__ float team_max(float v, float *red) {
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
__device__ __forceinline__ float team_sum(float v, float *red) {
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

// How often the row's history holds the columns [base, base + SEG).
template <int NT, int SEG>
struct Repeats {
    enum { NONE, FEW, BYTES, WORDS };
    int mode;
    int rel[LG_FEW];  // FEW: the ids' places in the segment, far below it for those outside
    const int *cnt;   // BYTES: a byte a column; WORDS: a word

    // lds: SEG words of the team.
    __device__ __forceinline__ void begin(const RowView &r, int64_t base, int64_t cols, int *lds) {
        const int64_t end = base + SEG < cols ? base + SEG : cols;
        const int t = team_thread<NT>();
        cnt = lds;
        mode = NONE;
        if (r.nids <= LG_FEW) {
            if (r.nids == 0) return;
            mode = FEW;
#pragma unroll
            for (int k = 0; k < LG_FEW; ++k) {
                const int64_t id = k < r.nids ? r.ids[k] : -1;
                rel[k] = id >= base && id < end ? (int)(id - base) : -8;
            }
            return;
        }
        bool hit = false;
        for (int64_t i = t; i < r.nids; i += NT) {
            const int64_t id = r.ids[i];
            hit |= id >= base && id < end;
        }
        if (!team_any<NT>(hit)) return;  // (behind it the last row's counts are read)
        const bool bytes = r.nids <= 255;
        mode = bytes ? BYTES : WORDS;
        const int words = bytes ? SEG / 4 : SEG;
        for (int i = t; i < words; i += NT) lds[i] = 0;
        team_sync<NT>();
        for (int64_t i = t; i < r.nids; i += NT) {
            const int64_t id = r.ids[i];
            if (id >= base && id < end) {
                const int c = (int)(id - base);
                if (bytes) atomicAdd(&lds[c >> 2], 1 << (8 * (c & 3)));
                else atomicAdd(&lds[c], 1);
            }
        }
        team_sync<NT>();
    }
    // The counts of the columns local .. local + 3; whether any is not 0.
    __device__ __forceinline__ bool quad(int local, int (&c)[4]) const {
        if (mode == NONE) return false;
        if (mode == WORDS) {
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = cnt[local + e];
            return (c[0] | c[1] | c[2] | c[3]) != 0;
        }
        unsigned w = 0;
        if (mode == BYTES) w = (unsigned)cnt[local >> 2];
        else
#pragma unroll
            for (int k = 0; k < LG_FEW; ++k) {
                const unsigned d = (unsigned)(rel[k] - local);
                w += d < 4 ? 1u << (8 * d) : 0u;
            }
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = (int)((w >> (8 * e)) & 255u);
        return w != 0;
    }
};

// The allowed bits of columns c .. c + 3 (those below cols).
__device__ __forceinline__ unsigned quad_bits(const RowView &r, int64_t c, int64_t cols) {
    if (c >= cols || r.none) return 0;
    unsigned b = r.allowed ? (r.allowed[c >> 5] >> (c & 31)) & 15u : 15u;
    return cols - c < 4 ? b & ((1u << (cols - c)) - 1) : b;
}

// A row's segment in a team's registers: the constrained values v and the
// allowed bits.
template <typename T, int NT, int VPT, bool HIST>
struct Segment {
    static constexpr int SEG = NT * 4 * VPT;
    float v[VPT][4];
    unsigned ok;

    static __device__ __forceinline__ int local(int i) { return (i * NT + team_thread<NT>()) * 4; }

    __device__ __forceinline__ void load(const LogitArgs &a, int64_t row, int64_t base, int *cnt) {
        const int64_t cols = a.op.cols;
        const RowView r = row_view(a.op, row);
        const T *x = (const T *)a.op.x + row * a.op.ldx;
        Quad<T> q[VPT];
        ok = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + local(i);
            if (c < cols) q[i] = load_quad(x + c, cols - c);
            ok |= quad_bits(r, c, cols) << (4 * i);
        }
        Repeats<NT, SEG> rep;
        if (HIST) rep.begin(r, base, cols, cnt);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + local(i);
            if (c >= cols) continue;
            Quad<float> b{{0, 0, 0, 0}};
            if (r.bias) b = load_quad(r.bias + c, cols - c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = (float)q[i].v[e] + b.v[e];
            int n[4];
            if (HIST && rep.quad(local(i), n)) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n[e] > 0) {
                        v[i][e] *= v[i][e] > 0.0f ? a.inv_repetition : a.op.repetition;
                        v[i][e] -= a.op.presence + a.op.frequency * (float)n[e];
                    }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] *= a.inv_temperature;
        }
    }
    __device__ __forceinline__ bool allowed(int i, int e) const { return (ok >> (4 * i + e)) & 1; }
    __device__ __forceinline__ float largest(float *red) const {
        float m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (allowed(i, e)) m = fmaxf(m, v[i][e]);
        return team_max<NT>(m, red);
    }
    // v = exp(v - shift) where allowed, 0 elsewhere; this thread's sum.
    __device__ __forceinline__ float exponentials(float shift) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[i][e] = allowed(i, e) ? expf(v[i][e] - shift) : 0.0f;
                s += v[i][e];
            }
        return s;
    }
    __device__ __forceinline__ void store_weights(float *y, int64_t base, int64_t cols, float inv) const {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + local(i);
            if (c < cols)
                store_quad(y + c, Quad<float>{{v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv}}, cols - c);
        }
    }
    __device__ __forceinline__ void store_values(T *y, int64_t base, int64_t cols, float fill) const {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + local(i);
            if (c >= cols) continue;
            Quad<T> q;
#pragma unroll
            for (int e = 0; e < 4; ++e) q.v[e] = (T)(allowed(i, e) ? v[i][e] : fill);
            store_quad(y + c, q, cols - c);
        }
    }
};

// Forward of rows held whole by a wave (NT = 64: a wave each) or a workgroup.
template <typename T, int NT, int VPT, bool SOFTMAX, bool HIST>
__global__ __launch_bounds__(LG_NT) void k_logits_rows(LogitArgs a, void *out) {
    using Seg = Segment<T, NT, VPT, HIST>;
    __shared__ float red[LG_WAVES];
    __shared__ int cnt[HIST ? LG_NT / NT : 1][HIST ? Seg::SEG : 1];
    const int team = NT == FL_WAVE ? fl_wave_id() : 0;
    const int64_t row = NT == FL_WAVE ? (int64_t)blockIdx.x * (blockDim.x / FL_WAVE) + team : (int64_t)blockIdx.x;
    if (row >= a.op.rows) return;  // NT = 64: no workgroup barriers
    const int64_t cols = a.op.cols;
    Seg s;
    s.load(a, row, 0, cnt[HIST ? team : 0]);
    if constexpr (!SOFTMAX) {
        s.store_values((T *)out + row * cols, 0, cols, a.op.fill);
    } else {
        const float m = s.largest(red);
        const float sum = team_sum<NT>(s.exponentials(m == -__builtin_inff() ? 0.0f : m), red);
        s.store_weights((float *)out + row * cols, 0, cols, 1.0f / (sum == 0.0f ? 1.0f : sum));
    }
}

// Forward of one segment of a longer row.  LG_STATS: its maximum and sum;
// LG_JOINED: the softmax with the row's joined ones.
template <typename T, int MODE, bool HIST>
__global__ __launch_bounds__(LG_NT) void k_logits_seg(LogitArgs a, void *out, float2 *stats) {
    using Seg = Segment<T, LG_NT, LG_VPT, HIST>;
    __shared__ float red[LG_WAVES];
    __shared__ int cnt[HIST ? LG_SEG : 1];
    const int64_t cols = a.op.cols, row = blockIdx.x / a.segments;
    const int64_t base = (int64_t)(blockIdx.x % a.segments) * LG_SEG;
    Seg s;
    s.load(a, row, base, cnt);
    if constexpr (MODE == LG_CONSTRAIN) {
        s.store_values((T *)out + row * cols, base, cols, a.op.fill);
    } else if constexpr (MODE == LG_STATS) {
        const float m = s.largest(red);
        const float sum = team_sum<LG_NT>(s.exponentials(m == -__builtin_inff() ? 0.0f : m), red);
        // a segment of nothing but NaN keeps its sum: a maximum of 0 lets it through
        if (threadIdx.x == 0) stats[blockIdx.x] = make_float2(m == -__builtin_inff() && sum != sum ? 0.0f : m, sum);
    } else {
        const float2 *st = stats + row * a.segments;
        float m = -__builtin_inff(), sum = 0.0f;
        for (uint32_t i = threadIdx.x; i < a.segments; i += LG_NT) m = fmaxf(m, st[i].x);
        m = team_max<LG_NT>(m, red);
        if (m == -__builtin_inff()) m = 0.0f;
        for (uint32_t i = threadIdx.x; i < a.segments; i += LG_NT) sum += st[i].y * expf(st[i].x - m);
        sum = team_sum<LG_NT>(sum, red);
        s.exponentials(m);
        s.store_weights((float *)out + row * cols, base, cols, 1.0f / (sum == 0.0f ? 1.0f : sum));
    }
}

struct GradArgs {
    LogitArgs l;
    const void *g;        // gradient of the output (T; the softmax: float)
    const float *w;       // the softmax's output
    const float *dots;    // [rows] sum w g, of rows longer than a workgroup holds
    void *dx;
    float *dbias;         // [parts][bias_rows][cols], or null: every row is a list of its own
    const int32_t *order, *offsets;  // owners by group (null: one list of all)
    int64_t lists;        // row lists: groups and one of no group
    uint32_t parts;
};

// The rows of a list, cut into parts.
struct RowList {
    int64_t first, q0, q1;
    __device__ __forceinline__ RowList(const GradArgs &a, int64_t list, uint32_t part) {
        const fl_logits &op = a.l.op;
        first = a.order ? (int64_t)a.offsets[list] : 0;
        const int64_t end = a.order && list + 1 < a.lists ? (int64_t)a.offsets[list + 1] : op.rows / op.inner;
        const int64_t n = (end - first) * op.inner;
        q0 = n * part / a.parts;
        q1 = n * (part + 1) / a.parts;
    }
    __device__ __forceinline__ int64_t row(const GradArgs &a, int64_t q) const {
        const uint32_t inner = (uint32_t)a.l.op.inner, at = (uint32_t)q / inner;
        const int64_t place = first + at;
        return (a.order ? (int64_t)a.order[place] : place) * inner + ((uint32_t)q - at * inner);
    }
};

// The gradient of a row's segment: what it reads, and its terms.
template <typename T, int NT, int VPT, bool SOFTMAX, bool HIST>
struct GradSegment {
    using TG = std::conditional_t<SOFTMAX, float, T>;
    static constexpr int SEG = NT * 4 * VPT;
    Quad<TG> g[VPT];
    Quad<float> w[SOFTMAX ? VPT : 1];
    int64_t row;

    static __device__ __forceinline__ int local(int i) { return (i * NT + team_thread<NT>()) * 4; }

    __device__ __forceinline__ void load(const GradArgs &a, int64_t at, int64_t base) {
        row = at;
        const int64_t cols = a.l.op.cols;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + local(i);
            if (c >= cols) continue;
            g[i] = load_quad((const TG *)a.g + row * cols + c, cols - c);
            if (SOFTMAX) w[i] = load_quad(a.w + row * cols + c, cols - c);
        }
    }
    // Writes the row's dx and adds its terms to acc.
    template <bool WHOLE>
    __device__ __forceinline__ void apply(const GradArgs &a, int64_t base, int *cnt, float *red, float (&acc)[VPT][4]) {
        const fl_logits &op = a.l.op;
        const int64_t cols = op.cols;
        const RowView r = row_view(op, row);
        unsigned ok = 0;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + local(i);
            const unsigned bits = quad_bits(r, c, cols);
            ok |= bits << (4 * i);
            if (SOFTMAX && WHOLE && c < cols)
#pragma unroll
                for (int e = 0; e < 4; ++e) s += (bits >> e) & 1 ? w[i].v[e] * (float)g[i].v[e] : 0.0f;
        }
        Repeats<NT, SEG> rep;
        if (HIST) rep.begin(r, base, cols, cnt);
        if (SOFTMAX) s = WHOLE ? team_sum<NT>(s, red) : a.dots[row];
        const T *x = (const T *)op.x + row * op.ldx;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = base + local(i);
            if (c >= cols) continue;
            float u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                u[e] = SOFTMAX ? w[i].v[e] * ((float)g[i].v[e] - s) : (float)g[i].v[e];
                u[e] *= a.l.inv_temperature;
            }
            int n[4];
            if (HIST && rep.quad(local(i), n)) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n[e] > 0) {
                        const float z = (float)x[c + e] + (r.bias ? r.bias[c + e] : 0.0f);
                        u[e] *= z > 0.0f ? a.l.inv_repetition : op.repetition;
                    }
            }
            Quad<T> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                u[e] = (ok >> (4 * i + e)) & 1 ? u[e] : 0.0f;
                acc[i][e] += u[e];
                o.v[e] = (T)u[e];
            }
            if (a.dx) store_quad((T *)a.dx + row * cols + c, o, cols - c);
        }
    }
};

// Rows held whole by a wave.  Without dbias a wave takes one row; with it a
// workgroup's waves take the rows of a list in turn, each loading its next
// row while it works on one, and join their sums.
template <typename T, int VPT, bool SOFTMAX, bool HIST>
__global__ __launch_bounds__(LG_NT) void k_logits_rows_grad(GradArgs a) {
    using Grad = GradSegment<T, FL_WAVE, VPT, SOFTMAX, HIST>;
    constexpr int SEG = Grad::SEG;
    __shared__ int cnt[HIST ? LG_WAVES : 1][HIST ? SEG : 1];
    __shared__ float sums[SEG];
    const int64_t cols = a.l.op.cols;
    const int wave = fl_wave_id(), waves = blockDim.x / FL_WAVE;
    int *mine = cnt[HIST ? wave : 0];
    float acc[VPT][4];
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
    if (!a.dbias) {
        const int64_t row = (int64_t)blockIdx.x * waves + wave;
        if (row >= a.l.op.rows) return;
        Grad g;
        g.load(a, row, 0);
        g.template apply<true>(a, 0, mine, nullptr, acc);
        return;
    }
    const int64_t list = blockIdx.x / a.parts;
    const uint32_t part = blockIdx.x % a.parts;
    const RowList rows(a, list, part);
    Grad g;
    if (rows.q0 + wave < rows.q1) g.load(a, rows.row(a, rows.q0 + wave), 0);
    for (int64_t q = rows.q0 + wave; q < rows.q1; q += LG_WAVES) {
        Grad next = g;
        if (q + LG_WAVES < rows.q1) next.load(a, rows.row(a, q + LG_WAVES), 0);
        g.template apply<true>(a, 0, mine, nullptr, acc);
        g = next;
    }
    if (list >= a.l.op.bias_rows) return;
    // in wave order
    for (int w = 0; w < LG_WAVES; ++w) {
        if (wave == w)
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float *at = sums + Grad::local(i) + e;
                    *at = w == 0 ? acc[i][e] : *at + acc[i][e];
                }
        __syncthreads();
    }
    float *b = a.dbias + ((int64_t)part * a.l.op.bias_rows + list) * cols;
    for (int64_t c = threadIdx.x; c < cols; c += LG_NT) b[c] = sums[c];
}

// One segment of the rows of a list (or of one row).  WHOLE: it is the row.
template <typename T, int VPT, bool SOFTMAX, bool HIST, bool WHOLE>
__global__ __launch_bounds__(LG_NT) void k_logits_seg_grad(GradArgs a) {
    using Grad = GradSegment<T, LG_NT, VPT, SOFTMAX, HIST>;
    __shared__ float red[LG_WAVES];
    __shared__ int cnt[HIST ? Grad::SEG : 1];
    const int64_t cols = a.l.op.cols;
    const uint32_t item = blockIdx.x / a.l.segments;
    const int64_t base = (int64_t)(blockIdx.x % a.l.segments) * Grad::SEG;
    float acc[VPT][4];
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
    Grad g;
    if (!a.dbias) {
        g.load(a, item, base);
        g.template apply<WHOLE>(a, base, cnt, red, acc);
        return;
    }
    const uint32_t part = item % a.parts;
    const int64_t list = item / a.parts;
    const RowList rows(a, list, part);
    if (rows.q0 < rows.q1) g.load(a, rows.row(a, rows.q0), base);
    for (int64_t q = rows.q0; q < rows.q1; ++q) {
        Grad next = g;
        if (q + 1 < rows.q1) next.load(a, rows.row(a, q + 1), base);
        g.template apply<WHOLE>(a, base, cnt, red, acc);
        g = next;
    }
    if (list >= a.l.op.bias_rows) return;
    float *b = a.dbias + ((int64_t)part * a.l.op.bias_rows + list) * cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int64_t c = base + Grad::local(i);
        if (c < cols) store_quad(b + c, Quad<float>{{acc[i][0], acc[i][1], acc[i][2], acc[i][3]}}, cols - c);
    }
}

// sum w g of one segment of a row.
__global__ __launch_bounds__(LG_NT) void k_logits_dot(LogitArgs a, const float *__restrict__ g,
                                                      const float *__restrict__ w, float *__restrict__ dots) {
    __shared__ float red[LG_WAVES];
    const int64_t cols = a.op.cols, row = blockIdx.x / a.segments;
    const int64_t base = (int64_t)(blockIdx.x % a.segments) * LG_SEG;
    const RowView r = row_view(a.op, row);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < LG_VPT; ++i) {
        const int64_t c = base + (i * LG_NT + threadIdx.x) * 4;
        const unsigned bits = quad_bits(r, c, cols);
        if (!bits) continue;
        const Quad<float> p = load_quad(w + row * cols + c, cols - c), q = load_quad(g + row * cols + c, cols - c);
#pragma unroll
        for (int e = 0; e < 4; ++e) s += (bits >> e) & 1 ? p.v[e] * q.v[e] : 0.0f;
    }
    s = team_sum<LG_NT>(s, red);
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
    if (op->cols && op->rows > 0x7fffffffll / lg_ceil(op->cols, LG_SEG))
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

// Waves of a workgroup whose waves take a row each: one where there are too
// few rows to give every CU a workgroup of four.
int row_waves(int64_t rows) { return rows < 1024 ? 1 : LG_WAVES; }

template <typename T, int NT, int VPT, bool SOFTMAX>
void launch_rows(hipStream_t st, const fl_logits *op, void *out) {
    const LogitArgs a = lg_args(op, NT * 4 * VPT);
    const int waves = NT == FL_WAVE ? row_waves(op->rows) : LG_WAVES;
    const dim3 grid((unsigned)(NT == FL_WAVE ? lg_ceil(op->rows, waves) : op->rows)), nt(waves * FL_WAVE);
    if (op->history) FL_LAUNCH("k_logits_rows", (k_logits_rows<T, NT, VPT, SOFTMAX, true>), grid, nt, 0, st, a, out);
    else FL_LAUNCH("k_logits_rows", (k_logits_rows<T, NT, VPT, SOFTMAX, false>), grid, nt, 0, st, a, out);
}

template <typename T, int MODE>
void launch_seg(hipStream_t st, const fl_logits *op, void *out, float2 *stats) {
    const LogitArgs a = lg_args(op, LG_SEG);
    const dim3 grid((unsigned)(op->rows * a.segments)), nt(LG_NT);
    if (op->history) FL_LAUNCH("k_logits_seg", (k_logits_seg<T, MODE, true>), grid, nt, 0, st, a, out, stats);
    else FL_LAUNCH("k_logits_seg", (k_logits_seg<T, MODE, false>), grid, nt, 0, st, a, out, stats);
}

template <typename T, bool SOFTMAX>
int forward(hipStream_t st, const fl_logits *op, void *out, float2 *stats, const char *what) {
    if (op->cols <= 256) launch_rows<T, FL_WAVE, 1, SOFTMAX>(st, op, out);
    else if (op->cols <= 512) launch_rows<T, FL_WAVE, 2, SOFTMAX>(st, op, out);
    else if (op->cols <= 1024) launch_rows<T, FL_WAVE, 4, SOFTMAX>(st, op, out);
    else if (op->cols <= LG_WAVE_COLS) launch_rows<T, FL_WAVE, 8, SOFTMAX>(st, op, out);
    else if constexpr (!SOFTMAX) launch_seg<T, LG_CONSTRAIN>(st, op, out, stats);
    else if (op->cols <= LG_LONG) launch_rows<T, LG_NT, LG_LONG / LG_NT / 4, true>(st, op, out);
    else {
        launch_seg<T, LG_STATS>(st, op, out, stats);
        launch_seg<T, LG_JOINED>(st, op, out, stats);
    }
    return fl_check_launch(what);
}

// Row lists of a bias table's gradient: its groups and, when there are
// several, the owners of none.
int64_t grad_lists(const fl_logits *op) { return op->bias_rows > 1 ? op->bias_rows + 1 : 1; }

int64_t grad_segments(const fl_logits *op, bool softmax) {
    return op->cols <= LG_WAVE_COLS || (softmax && op->cols <= LG_LONG) ? 1 : lg_ceil(op->cols, LG_SEG);
}

// Parts of a list: some 2048 workgroups in all, of at least 8 rows on average.
int grad_parts(const fl_logits *op, int64_t lists, int64_t segments) {
    const int64_t want = lg_ceil(2048, lists * segments), most = op->rows / (8 * lists);
    const int64_t p = want < most ? want : most;
    return (int)(p < 1 ? 1 : p > 256 ? 256 : p);
}

template <typename T, int VPT, bool SOFTMAX>
void launch_rows_grad(hipStream_t st, const GradArgs &a) {
    const fl_logits &op = a.l.op;
    const int waves = a.dbias ? LG_WAVES : row_waves(op.rows);
    const dim3 grid((unsigned)(a.dbias ? a.lists * a.parts : lg_ceil(op.rows, waves))), nt(waves * FL_WAVE);
    if (op.history && op.repetition != 1.0f)  // the slopes need the repeats
        FL_LAUNCH("k_logits_rows_grad", (k_logits_rows_grad<T, VPT, SOFTMAX, true>), grid, nt, 0, st, a);
    else FL_LAUNCH("k_logits_rows_grad", (k_logits_rows_grad<T, VPT, SOFTMAX, false>), grid, nt, 0, st, a);
}

template <typename T, int VPT, bool SOFTMAX, bool WHOLE>
void launch_seg_grad(hipStream_t st, const GradArgs &a) {
    const fl_logits &op = a.l.op;
    const dim3 grid((unsigned)((a.dbias ? a.lists * a.parts : op.rows) * a.l.segments)), nt(LG_NT);
    if (op.history && op.repetition != 1.0f)
        FL_LAUNCH("k_logits_seg_grad", (k_logits_seg_grad<T, VPT, SOFTMAX, true, WHOLE>), grid, nt, 0, st, a);
    else FL_LAUNCH("k_logits_seg_grad", (k_logits_seg_grad<T, VPT, SOFTMAX, false, WHOLE>), grid, nt, 0, st, a);
}

// The gradient's workspace: the parts of dbias, the segments' dots and the
// rows' (long softmax), and the owners by group.
struct GradSpace {
    size_t parts, dots, order, offsets, group, group_bytes, bytes;
};

GradSpace grad_space(const fl_logits *op, bool softmax, bool with_dbias) {
    GradSpace s{};
    const auto take = [&](size_t n) {
        const size_t at = s.bytes;
        s.bytes += (n + 255) / 256 * 256;
        return at;
    };
    const int64_t segments = grad_segments(op, softmax);
    if (with_dbias) {
        const int parts = grad_parts(op, grad_lists(op), segments);
        if (parts > 1) s.parts = take((size_t)parts * op->bias_rows * op->cols * 4);
        if (op->bias_rows > 1) {
            const int64_t owners = op->rows / op->inner;
            s.order = take((size_t)owners * 4 + 4);
            s.offsets = take((size_t)(op->bias_rows + 1) * 4);
            s.group_bytes = fl_group_rows_bytes(owners, op->bias_rows);
            s.group = take(s.group_bytes);
        }
    }
    if (softmax && op->cols > LG_LONG) s.dots = take((size_t)op->rows * (segments + 1) * 4);
    return s;
}

template <typename T, bool SOFTMAX>
int gradient(hipStream_t st, const fl_logits *op, const float *w, const void *grad, void *dx, float *dbias, char *ws) {
    const GradSpace sp = grad_space(op, SOFTMAX, dbias != nullptr);
    GradArgs a{};
    a.l = lg_args(op, LG_SEG);
    a.l.segments = (uint32_t)grad_segments(op, SOFTMAX);
    a.g = grad;
    a.w = w;
    a.dx = dx;
    a.parts = 1;
    if (dbias) {
        a.lists = grad_lists(op);
        a.parts = (uint32_t)grad_parts(op, a.lists, a.l.segments);
        a.dbias = a.parts > 1 ? (float *)(ws + sp.parts) : dbias;
        if (op->bias_rows > 1) {
            int32_t *order = (int32_t *)(ws + sp.order), *offsets = (int32_t *)(ws + sp.offsets);
            const int rc = fl_group_rows(st, op->group, op->rows / op->inner, op->bias_rows, order, offsets, nullptr,
                                         ws + sp.group, sp.group_bytes);
            if (rc) return rc;
            a.order = order;
            a.offsets = offsets;
        }
    } else if (op->rows == 0) return FL_OK;
    if (SOFTMAX && op->cols > LG_LONG && op->rows > 0) {
        float *part = (float *)(ws + sp.dots), *dots = part + op->rows * a.l.segments;
        FL_LAUNCH("k_logits_dot", k_logits_dot, dim3((unsigned)(op->rows * a.l.segments)), dim3(LG_NT), 0, st, a.l,
                  (const float *)grad, w, part);
        FL_LAUNCH("k_logits_join", k_logits_join, dim3((unsigned)op->rows), dim3(FL_WAVE), 0, st, part,
                  (int64_t)a.l.segments, dots);
        a.dots = dots;
    }
    if (op->cols <= 256) launch_rows_grad<T, 1, SOFTMAX>(st, a);
    else if (op->cols <= 512) launch_rows_grad<T, 2, SOFTMAX>(st, a);
    else if (op->cols <= 1024) launch_rows_grad<T, 4, SOFTMAX>(st, a);
    else if (op->cols <= LG_WAVE_COLS) launch_rows_grad<T, 8, SOFTMAX>(st, a);
    else if constexpr (!SOFTMAX) launch_seg_grad<T, LG_VPT, false, true>(st, a);
    else if (op->cols <= LG_LONG) launch_seg_grad<T, LG_LONG / LG_NT / 4, true, true>(st, a);
    else launch_seg_grad<T, LG_VPT, true, false>(st, a);
    if (a.parts > 1) fold_parts<float>(st, a.dbias, (int)a.parts, op->bias_rows * op->cols, dbias);
    return fl_check_launch("logits_grad");
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
    FL_BY_TYPE(op->dtype, (fl::forward<T, false>((hipStream_t)stream, op, out, nullptr,
                                                            "logits_constrain")))
}

size_t fl_logits_softmax_bytes(const fl_logits *op) {
    if (!op || op->cols <= fl::LG_LONG || op->rows < 1) return 0;
    return (size_t)op->rows * fl::lg_ceil(op->cols, fl::LG_SEG) * sizeof(float2);
}

int fl_logits_softmax(void *stream, const fl_logits *op, float *w, void *ws, size_t ws_bytes) {
    const int rc = fl::lg_check(op, "logits_softmax");
    if (rc) return rc;
    if (op->rows == 0 || op->cols == 0) return FL_OK;
    if (!w) return fl::fl_fail(FL_ERR_ARG, "logits_softmax: null pointer");
    const size_t need = fl_logits_softmax_bytes(op);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "logits_softmax: workspace too small");
    FL_BY_TYPE(op->dtype, (fl::forward<T, true>((hipStream_t)stream, op, w, (float2 *)ws,
                                                          "logits_softmax")))
}

size_t fl_logits_grad_bytes(const fl_logits *op, int softmax, int with_dbias) {
    if (!op || op->rows < 0 || op->cols < 1 || op->inner < 1) return 0;
    return fl::grad_space(op, softmax != 0, with_dbias != 0 && op->bias && op->bias_rows > 0).bytes;
}

int fl_logits_grad(void *stream, const fl_logits *op, const float *w, const void *grad, void *dx, float *dbias,
                   void *ws, size_t ws_bytes) {
    const int rc = fl::lg_check(op, "logits_grad");
    if (rc) return rc;
    if (op->cols == 0) return FL_OK;
    if (dbias && !op->bias) return fl::fl_fail(FL_ERR_ARG, "logits_grad: the gradient of no bias table");
    if (op->rows > 0 && !grad) return fl::fl_fail(FL_ERR_ARG, "logits_grad: null pointer");
    const size_t need = fl_logits_grad_bytes(op, w != nullptr, dbias != nullptr);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "logits_grad: workspace too small");
    if ((uintptr_t)ws % 16) return fl::fl_fail(FL_ERR_ARG, "logits_grad: workspace must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    if (w) {
        FL_BY_TYPE(op->dtype, (fl::gradient<T, true>(st, op, w, grad, dx, dbias, (char *)ws)))
    }
    FL_BY_TYPE(op->dtype, (fl::gradient<T, false>(st, op, w, grad, dx, dbias, (char *)ws)))
}

}  // extern "C"
