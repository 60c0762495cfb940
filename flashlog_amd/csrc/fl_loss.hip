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
// loss 0 and no gradient.  Here the rows that are given; fl_vocab.hip has those
// that are a product.
//
// HBM-bound: one read forward, one read and one write backward.  A wave takes a
// segment of a row in registers, a second launch joins the segments' maxima and
// sums and looks at the lists.  Exponentials are the hardware's 2^x of distances
// from the row's maximum, off by 2^-23 of their exponent besides its own step.
#include "fl_abi.h"
#include "fl_common.h"
#include "fl_loss.h"

namespace fl {
namespace {

constexpr int LS_SEG = 2048;  // columns of a wave
constexpr int LS_NT = 256;
constexpr int LS_WAVES = LS_NT / FL_WAVE;

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

template <typename T, int G>
struct Cols {
    T v[G];
};
template <typename T, int G>
__device__ __forceinline__ Cols<T, G> load_cols(const T *p) {
    Cols<T, G> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T, int G>
__device__ __forceinline__ void store_cols(T *p, const Cols<T, G> &r) {
    __builtin_memcpy(p, &r, sizeof(r));
}
// The first m of them.
template <typename T, int G>
__device__ __forceinline__ void store_first(T *p, const Cols<T, G> &r, int m) {
#pragma unroll
    for (int e = 0; e < G; ++e)
        if (e < m) p[e] = r.v[e];
}

// A wave's segment of a row in registers, behind its end `fill`.
template <typename T>
struct Segment {
    static constexpr int G = cols_of<T>(), N = LS_SEG / FL_WAVE / G;
    Cols<T, G> v[N];

    __device__ __forceinline__ void load(const T *row, int64_t c0, int64_t cols) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t c = c0 + (i * FL_WAVE + fl_lane()) * G;
            if (c + G <= cols) v[i] = load_cols<T, G>(row + c);
            else
#pragma unroll
                for (int e = 0; e < G; ++e) v[i].v[e] = c + e < cols ? row[c + e] : (T)-INFINITY;
        }
    }
};

// A segment's maximum and sum.  HBM-bound: fp32 [32 x 4.6M] 126 us = 4.7 TB/s, bf16
// [509 x 123000] 36 us = 3.5 (a large sum reads 4.0 on the same card).
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
    const float at = base_of(r.m);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < G; ++e) r.s += exp2_of(((float)s.v[i].v[e] - at) * a.scale);
    r.s = fl_wave_sum_f32(r.s);
    if (fl_lane() == 0) a.part[row * a.segments + seg] = r;
}

// A segment of the gradient, the listed columns behind it.  HBM-bound: fp32 [32 x
// 4.6M] 197 us = 6.0 TB/s, bf16 [509 x 123000] 47 us = 5.4.
template <typename T>
__global__ __launch_bounds__(LS_NT) void k_score_grad(ScoreArgs a) {
    constexpr int G = Segment<T>::G, N = Segment<T>::N;
    const int64_t item = fl_block() * LS_WAVES + fl_wave_id();
    if (item >= a.op.rows * a.segments) return;
    const int64_t row = item / a.segments, c0 = (item % a.segments) * LS_SEG;
    const float2 of = a.rows[row];
    const float c = of.y != 0.0f ? a.op.temperature * a.grad[row] : 0.0f, f = c * of.y;
    T *out = (T *)a.dx + row * a.cols;
    Segment<T> s;
    s.load((const T *)a.logits + row * a.ld, c0, a.cols);
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int e = 0; e < G; ++e)
            s.v[i].v[e] =
                (T)(c == 0.0f || (float)s.v[i].v[e] == -INFINITY
                        ? 0.0f  // masked, whatever its row holds
                        : f * exp2_of(((float)s.v[i].v[e] - of.x) * a.scale));
        const int64_t at = c0 + (i * FL_WAVE + fl_lane()) * G;
        if (at + G <= a.cols) store_cols<T, G>(out + at, s.v[i]);
        else store_first<T, G>(out + at, s.v[i], (int)(a.cols - at));
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
            if (l.x != -INFINITY) out[id] = (T)(c * (exp2_of((l.x - of.x) * a.scale) * of.y - l.y));
        }
    }
}

// ---------------------------------------------------------------------------
// Rows' sums joined, their lists, their losses: a wave a row, or the four of a
// workgroup where there are many parts (2247 of 32 rows: 25 us with one, 9 with
// four; 61 of 509 rows 8).  Bound by the time of its few loads.  An id's share adds
// the list's entries of that id, k^2 of them a row.
template <typename T, int WPR>
__global__ __launch_bounds__(LS_NT) void k_list_rows(ListArgs a) {
    extern __shared__ __align__(16) float2 list_lds[];
    __shared__ Running quarters[LS_WAVES];
    const int64_t waves = blockDim.x / FL_WAVE, row = WPR == 1 ? fl_block() * waves + fl_wave_id() : fl_block();
    if (row >= a.op.rows) return;
    Running r = joined_parts(a.part + row * a.parts, a.parts, WPR == 1 ? 0 : fl_wave_id(), WPR, a.unit);
    if constexpr (WPR > 1) {
        if (fl_lane() == 0) quarters[fl_wave_id()] = r;
        __syncthreads();
        if (fl_wave_id()) return;
        r = joined(joined(quarters[0], quarters[1], a.unit), joined(quarters[2], quarters[3], a.unit), a.unit);
    }
    list_row(a, row, r, list_lds + (WPR == 1 ? fl_wave_id() * a.op.k : 0), [&](int64_t j, int64_t id) {
        return a.logits ? (float)((const T *)a.logits)[row * a.ld + id] : a.listed[row * a.op.k + j].x;
    });
}

// ---------------------------------------------------------------------------
// Host side

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename T>
int join_rows(hipStream_t st, ListArgs &a, const char *what) {
    if (a.parts > 4 * FL_WAVE) {
        FL_LAUNCH("k_list_rows", (k_list_rows<T, LS_WAVES>), grid_of(a.op.rows), dim3(LS_NT), (size_t)a.op.k * 8, st, a);
        return fl_check_launch(what);
    }
    const int64_t waves = a.op.k <= 512 ? LS_WAVES : 1;
    FL_LAUNCH("k_list_rows", (k_list_rows<T, 1>), grid_of(ceil_div(a.op.rows, waves)), dim3((unsigned)waves * FL_WAVE),
              (size_t)waves * a.op.k * 8, st, a);
    return fl_check_launch(what);
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
    a.unit = a.scale;
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

}  // namespace

constexpr int64_t LS_MOST_LISTED = 4096;

int check_lists(const fl_lists *l, const char *what) {
    if (l->rows < 0 || l->k < 0 || l->rows > 0x7fffffffll) return fl_fail(FL_ERR_ARG, "%s: bad shape", what);
    if (l->k > LS_MOST_LISTED)
        return fl_fail(FL_ERR_ARG, "%s: lists of more than %d ids (shape)", what, (int)LS_MOST_LISTED);
    if (l->rows && !l->teacher && l->k > 1) return fl_fail(FL_ERR_ARG, "%s: targets without a teacher are one a row (shape)", what);
    if (l->rows && l->k && !l->ids) return fl_fail(FL_ERR_ARG, "%s: null pointer", what);
    if (!(l->temperature >= 0x1p-60f && l->temperature <= 0x1p60f))
        return fl_fail(FL_ERR_ARG, "%s: temperature must be within 2^-60 and 2^60", what);
    return FL_OK;
}

int join_listed(hipStream_t st, const fl_lists *l, int64_t cols, const Running *part, int64_t parts, void *state,
                float *loss, const char *what) {
    ListArgs a = list_args(l, cols, state, loss);
    a.part = part;
    a.parts = parts;
    return join_rows<float>(st, a, what);  // no logits: of no type
}

}  // namespace fl

#define FL_BY_TYPE(dtype, call)                           \
    switch (dtype) {                                      \
        case FL_F32: { using T = float; return call; }    \
        case FL_BF16: { using T = __bf16; return call; }  \
        default: { using T = _Float16; return call; }     \
    }

extern "C" {

size_t fl_scores_op_bytes(void) { return sizeof(fl_scores); }

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

}  // extern "C"
