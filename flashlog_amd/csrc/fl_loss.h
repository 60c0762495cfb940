// What the losses of given rows and of products share.
#pragma once
#include "fl_abi.h"
#include "fl_common.h"
#include <math.h>

namespace fl {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.69314718055994531f;

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// A running maximum m of a row's u and the sum of 2^((u - m) unit): what unit is
// depends on where u comes from.  Scores are held as they are given: their
// distance from m is exact at any size (a mask of the type's lowest value in
// every column leaves a uniform row).
struct Running {
    float m, s;
};
// What exponents are taken from: the maximum, 0 where nothing is above -inf.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ Running joined(Running a, Running b, float unit = 1.0f) {
    const float m = fmaxf(a.m, b.m), at = base_of(m);
    return Running{m, a.s * exp2_of((a.m - at) * unit) + b.s * exp2_of((b.m - at) * unit)};
}

// The state that a forward leaves for the backward: rows [rows] (the maximum, the
// sum's reciprocal; 0 where the row does not count), listed [rows][k] (u of the
// id, the sum of q at it).  A term's share is 2^((u - m) unit) times the reciprocal:
// the two as one number, log sum exp u, would be rounded by 2^-24 of its size, an
// error that all shares of the row have (sum(p) - 1 = 6e-4 at logits of 4000).
inline size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
inline size_t state_bytes(const fl_lists *l) { return rounded((size_t)l->rows * 8) + (size_t)l->rows * l->k * 8; }
inline float2 *state_rows(void *state) { return (float2 *)state; }
inline float2 *state_listed(const fl_lists *l, void *state) {
    return (float2 *)((char *)state + rounded((size_t)l->rows * 8));
}

__device__ __forceinline__ Running joined_over_lanes(Running r, float unit) {
#pragma unroll
    for (int o = FL_WAVE / 2; o > 0; o >>= 1) r = joined(r, Running{__shfl_xor(r.m, o), __shfl_xor(r.s, o)}, unit);
    return r;
}
// Of the parts [count], a wave's share (every `waves`-th 64 of them): the same in all lanes.
__device__ __forceinline__ Running joined_parts(const Running *part, int64_t count, int wave, int waves,
                                                float unit) {
    Running r{-INFINITY, 0.0f};
    const int64_t step = (int64_t)waves * FL_WAVE;
    int64_t p = (int64_t)wave * FL_WAVE + fl_lane();
    for (; p + 7 * step < count; p += 8 * step) {
        Running v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = part[p + j * step];
#pragma unroll
        for (int j = 0; j < 8; ++j) r = joined(r, v[j], unit);
    }
    for (; p < count; p += step) r = joined(r, part[p], unit);
    return joined_over_lanes(r, unit);
}

struct ListArgs {
    fl_lists op;
    float scale, tau2;  // log2(e) / tau, tau^2
    float unit;         // of u: scale where logits are given, 1 where u is in units of log 2
    int64_t cols;
    const Running *part;  // [rows][parts]
    int64_t parts;
    const void *logits;   // scores; null: `listed` holds u
    int64_t ld;
    float *loss;
    float2 *rows, *listed;  // the state
};

inline ListArgs list_args(const fl_lists *l, int64_t cols, void *state, float *loss) {
    ListArgs a{};
    a.op = *l;
    a.scale = LOG2E / l->temperature;
    a.tau2 = l->temperature * l->temperature;
    a.unit = 1.0f;
    a.cols = cols;
    a.loss = loss;
    a.rows = state_rows(state);
    a.listed = state_listed(l, state);
    return a;
}

// A row's list and loss, by one wave: r, the row's sums; mine [k], the wave's own
// LDS; u_of(j, id), u of the j-th id (inside the vocabulary).
template <typename U>
__device__ __forceinline__ void list_row(const ListArgs &a, int64_t row, Running r, float2 *mine, U &&u_of) {
    const int64_t k = a.op.k;
    const float log_sum = log2f(r.s);
    const int64_t *ids = a.op.ids + row * k;
    float2 *listed = a.listed + row * k;
    // (id, teacher), -inf where it does not count
    float top = -INFINITY;
    bool any = false;
    for (int64_t j = fl_lane(); j < k; j += FL_WAVE) {
        const int64_t id = ids[j];
        const bool in = id >= 0 && id < a.cols;
        const float u = in ? u_of(j, id) : 0.0f;
        float v = -INFINITY;
        if (in && a.op.teacher && u != -INFINITY) v = a.op.teacher[row * k + j];
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
    for (int64_t j = fl_lane(); j < k; j += FL_WAVE) total += exp2_of((mine[j].y - top) * a.scale);
    total = fl_wave_sum_f32(total);
    const float of_total = 1.0f / total, log_total = log2f(total);
    float loss = 0.0f;
    for (int64_t j = fl_lane(); j < k; j += FL_WAVE) {
        const float v = (mine[j].y - top) * a.scale, q = live ? exp2_of(v) * of_total : 0.0f;
        if (q != 0.0f) loss += q * ((v - log_total) - ((listed[j].x - r.m) * a.unit - log_sum));
        mine[j].y = q;
    }
    loss = fl_wave_sum_f32(loss) * (a.tau2 * LN2);
    if (fl_lane() == 0) {
        a.loss[row] = live ? loss : 0.0f;
        a.rows[row] = float2{r.m, live ? 1.0f / r.s : 0.0f};
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

int check_lists(const fl_lists *l, const char *what);

// Joins the parts of the rows' sums ([rows][parts]), and makes the losses and
// the state from the listed u that are there.
int join_listed(hipStream_t st, const fl_lists *l, int64_t cols, const Running *part, int64_t parts, void *state,
                float *loss, const char *what);

}  // namespace fl
