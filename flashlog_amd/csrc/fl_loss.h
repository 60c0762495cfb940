// What the losses of given rows and of products share.
#pragma once
#include "fl_abi.h"
#include "fl_common.h"
#include <math.h>

namespace fl {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.69314718055994531f;

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

// The state that a forward leaves for the backward: rows [rows] (lse, whether
// the row counts), listed [rows][k] (u of the id, the sum of q at it).
inline size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
inline size_t state_bytes(const fl_lists *l) { return rounded((size_t)l->rows * 8) + (size_t)l->rows * l->k * 8; }
inline float2 *state_rows(void *state) { return (float2 *)state; }
inline float2 *state_listed(const fl_lists *l, void *state) {
    return (float2 *)((char *)state + rounded((size_t)l->rows * 8));
}

int check_lists(const fl_lists *l, const char *what);

// Joins the parts of the rows' sums ([rows][parts]), and makes the losses and
// the state from the listed u that are there.
int join_listed(hipStream_t st, const fl_lists *l, int64_t cols, const Running *part, int64_t parts, void *state,
                float *loss, const char *what);

}  // namespace fl
