// Sums of partial results in a fixed order.
#pragma once
#include "fl_abi.h"
#include "fl_common.h"

namespace fl {

// out[i] = sum of part[p][i] over p: 64 outputs and 4 runs of parts a
// workgroup, each run added in order, then the runs.  (One thread an output
// has one chain of dependent loads: 13 us for 48 parts of 1645 columns.)
template <typename TO>
__global__ __launch_bounds__(256) void k_fold_parts(const float *__restrict__ part, int parts, int64_t n,
                                                    TO *__restrict__ out) {
    __shared__ float runs[4][64];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
    const int64_t i = fl_block() * 64 + lane;
    const int p1 = parts * (run + 1) / 4;
    float s = 0.0f;
    if (i < n) {
        int p = parts * run / 4;
        for (; p + 8 <= p1; p += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = part[(int64_t)(p + j) * n + i];
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
        }
        for (; p < p1; ++p) s += part[(int64_t)p * n + i];
    }
    runs[run][lane] = s;
    __syncthreads();
    if (run == 0 && i < n) out[i] = (TO)(((runs[0][lane] + runs[1][lane]) + runs[2][lane]) + runs[3][lane]);
}

// The same for many outputs of few parts: four outputs a thread.
template <typename TO>
__global__ __launch_bounds__(256) void k_fold_few(const float *__restrict__ part, int parts, int64_t n,
                                                  TO *__restrict__ out) {
    const int64_t i = (fl_block() * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    if (i + 4 <= n) {
        float s[4] = {0, 0, 0, 0};
        for (int p = 0; p < parts; ++p) {
            float v[4];
            __builtin_memcpy(v, part + (int64_t)p * n + i, 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += v[e];
        }
        TO o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (TO)s[e];
        __builtin_memcpy(out + i, o, sizeof(o));
    } else
        for (int64_t j = i; j < n; ++j) {
            float s = 0.0f;
            for (int p = 0; p < parts; ++p) s += part[(int64_t)p * n + j];
            out[j] = (TO)s;
        }
}

// By the number of parts.
template <typename TO>
inline void fold_parts(hipStream_t st, const float *part, int parts, int64_t n, TO *out) {
    if (parts > 8)
        FL_LAUNCH("k_fold_parts", k_fold_parts<TO>, grid_of((n + 63) / 64), dim3(256), 0, st, part, parts, n, out);
    else
        FL_LAUNCH("k_fold_few", k_fold_few<TO>, grid_of((n + 1023) / 1024), dim3(256), 0, st, part, parts, n, out);
}

}  // namespace fl
