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
//   gradients: dv = g (softmax: w (g - sum w g), 0 and no part of the sum where
//   w is 0, whatever g is), dx = dv allowed slope with
//   slope = 1/temperature, for c > 0 times 1/repetition or repetition by the
//   sign of x + bias; dbias[g] = the sum of the dx of the group's rows
//
// All of it is one pass over the rows: HBM-bound, bytes = one read and one
// write of the rows.  A wave takes a row's segment of up to 2048 columns in
// registers, 16 bytes a lane and load, so that nothing waits for other waves;
// rows of up to 2048 columns are one segment, the softmax of longer ones
// joins the segments' maxima and sums in a second launch.
//
// Masks are one bit a column.  Histories are short next to the rows: a wave
// looks at the ids 64 at a time, and every one that falls into its segment is
// counted by the lane that holds the column (a byte each; rows with more than
// 255 ids are counted in LDS, 16 bits each -- integers, so the order does not
// matter).  The
// slopes read the logits of repeated columns only.
//
// dbias adds fp32 terms in a fixed order: of longer rows a wave keeps one
// table row's segment in registers and walks the group's rows, writing their
// dx on the way; of rows of one segment, where that leaves too few waves, the
// terms are read back (fp32 dx as they are, of 16-bit logits a copy).  Groups
// of many rows are cut into parts.  The terms are the unrounded ones, so
// half-precision logits give the same dbias as fp32 ones.
#include "fl_abi.h"
#include "fl_common.h"
#include "fl_parts.h"
#include <math.h>
#include <type_traits>

namespace fl {
namespace {

constexpr int LG_SEG = 2048;  // columns of a wave
constexpr int LG_WAVES = 4;   // of a workgroup
constexpr int LG_NT = LG_WAVES * FL_WAVE;

// Columns of a lane's load.
template <typename T>
constexpr int group_cols() {
    return 16 / (int)sizeof(T);
}

template <typename U, int G>
struct Group {
    U v[G];
};

// Columns c .. c + G - 1 of a row of `cols`.  A group that the row ends in is
// read from its last G columns and shifted; lanes behind the row read those
// too and use nothing of it.
template <typename U, int G>
__device__ __forceinline__ Group<U, G> load_group(const U *row, int c, int cols) {
    Group<U, G> r;
    if (cols < G) {
#pragma unroll
        for (int e = 0; e < G; ++e) r.v[e] = c + e < cols ? row[c + e] : (U)0.0f;
        return r;
    }
    const int at = c + G <= cols ? c : cols - G;
    __builtin_memcpy(&r, reinterpret_cast<const char *>(row) + (uint32_t)at * (uint32_t)sizeof(U), sizeof(r));
    const int shift = c - at < G ? c - at : 0;
    if (__any(shift)) {
#pragma unroll
        for (int s = 1; s < G; s *= 2)
            if (shift & s)
#pragma unroll
                for (int e = 0; e + s < G; ++e) r.v[e] = r.v[e + s];
    }
    return r;
}
// PAST: past the caches.
template <bool PAST = false, typename U, int G>
__device__ __forceinline__ void store_group(U *row, int c, int cols, const Group<U, G> &r) {
    typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
    constexpr int N = (int)sizeof(r) / 16;
    static_assert(sizeof(r) == 16 * N, "whole 16-byte words");
    if (c + G <= cols) {
        Words *to = reinterpret_cast<Words *>(reinterpret_cast<char *>(row) + (uint32_t)c * (uint32_t)sizeof(U)), q[N];
        __builtin_memcpy(q, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < N; ++i)
            if constexpr (PAST) __builtin_nontemporal_store(q[i], to + i);
            else to[i] = q[i];
    } else
#pragma unroll
        for (int e = 0; e < G; ++e)
            if (c + e < cols) row[c + e] = r.v[e];
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

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = FL_WAVE / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, FL_WAVE));
    return v;
}

// A wave's columns of a row: VPT groups of G a lane from column `base` on.
template <int G, int VPT>
struct Columns {
    static constexpr int SEG = FL_WAVE * G * VPT;
    static __device__ __forceinline__ int local(int i) { return (i * FL_WAVE + fl_lane()) * G; }

    // The allowed bits of the lane's i-th group (those of columns below cols).
    static __device__ __forceinline__ unsigned bits(const RowView &r, int c, int cols) {
        if (c >= cols || r.none) return 0;
        const unsigned all = (1u << G) - 1;
        const unsigned b = r.allowed ? (r.allowed[c >> 5] >> (c & 31)) & all : all;
        return cols - c < G ? b & ((1u << (cols - c)) - 1) : b;
    }
};

// How often the row's history holds the wave's columns.
template <int G, int VPT>
struct Repeats {
    using C = Columns<G, VPT>;
    using Pack = std::conditional_t<G == 4, uint32_t, uint64_t>;
    Pack pack[VPT];         // a byte a column
    const uint32_t *halves;  // rows with more ids than a byte counts: LDS, 16 bits a column of the wave

    // head: this lane's id of the first 64.
    __device__ __forceinline__ void count(const RowView &r, int64_t head, int base, int cols, uint32_t *lds) {
        const int end = cols - base < C::SEG ? cols : base + C::SEG;
        halves = nullptr;
#pragma unroll
        for (int i = 0; i < VPT; ++i) pack[i] = 0;
        if (r.nids > 255) {
            halves = lds;
            fl_wave_sync();  // the last row's counts are read
            for (int i = fl_lane(); i < C::SEG / 2; i += FL_WAVE) lds[i] = 0;
            fl_wave_sync();
            for (int64_t j = fl_lane(); j < r.nids; j += FL_WAVE) {
                const int64_t id = r.ids[j];
                if (id >= base && id < end) {
                    const int c = (int)(id - base), up = 16 * (c & 1);
                    // at most 64 more a turn: a column that has come up 65000 times is counted no further
                    if (((volatile uint32_t *)lds)[c >> 1] >> up << 16 < 65000u << 16) atomicAdd(&lds[c >> 1], 1u << up);
                }
            }
            fl_wave_sync();
            return;
        }
        for (int j = 0; j < (int)r.nids; j += FL_WAVE) {
            const int64_t id = j == 0 ? head : j + fl_lane() < (int)r.nids ? r.ids[j + fl_lane()] : -1;
            const int o = (int)(id - base);
            unsigned long long m = __ballot(id >= base && id < end);
            while (m) {
                const int at = __builtin_amdgcn_readlane(o, __builtin_ctzll(m));
                m &= m - 1;
                const Pack one = fl_lane() == (at / G) % FL_WAVE ? (Pack)1 << (8 * (at % G)) : (Pack)0;
#pragma unroll
                for (int i = 0; i < VPT; ++i)
                    if (at / (G * FL_WAVE) == i) pack[i] += one;
            }
        }
    }
    __device__ __forceinline__ bool any(int i) const {
        if (halves) {
            uint32_t n = 0;
#pragma unroll
            for (int e = 0; e < G; e += 2) n |= halves[(C::local(i) + e) / 2];
            return n != 0;
        }
        return pack[i] != 0;
    }
    __device__ __forceinline__ int at(int i, int e) const {
        if (halves) return (int)(halves[(C::local(i) + e) / 2] >> (16 * (e & 1))) & 0xffff;
        return (int)((pack[i] >> (8 * e)) & 255);
    }
};

// This lane's id of the first 64 of the row's history.
__device__ __forceinline__ int64_t head_id(const RowView &r) {
    return fl_lane() < r.nids && r.nids <= 255 ? r.ids[fl_lane()] : -1;
}

// The constrained values v of a wave's segment and their allowed bits.
template <typename T, int VPT, bool HIST>
struct Segment : Columns<group_cols<T>(), VPT> {
    static constexpr int G = group_cols<T>();
    using C = Columns<G, VPT>;
    float v[VPT][G];
    unsigned ok[VPT];

    using Bias = Group<float, G>[VPT];

    static __device__ __forceinline__ void load_bias(const float *bias, int base, int cols, Bias &b) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) b[i] = load_group<float, G>(bias, base + C::local(i), cols);
    }
    // kept: the bias, if KEPT.
    template <bool KEPT>
    __device__ __forceinline__ void load(const LogitArgs &a, int64_t row, int base, uint32_t *lds, const Bias &kept) {
        const int cols = (int)a.op.cols;
        const RowView r = row_view(a.op, row);
        const T *x = (const T *)a.op.x + row * a.op.ldx;
        Group<T, G> q[VPT];
#pragma unroll
        for (int i = 0; i < VPT; ++i) q[i] = load_group<T, G>(x, base + C::local(i), cols);
        Repeats<G, VPT> rep;
        if (HIST) rep.count(r, head_id(r), base, cols, lds);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = base + C::local(i);
            ok[i] = C::bits(r, c, cols);
#pragma unroll
            for (int e = 0; e < G; ++e) v[i][e] = (float)q[i].v[e];
            if (KEPT || r.bias) {
                const Group<float, G> b = KEPT ? kept[i] : load_group<float, G>(r.bias, c, cols);
#pragma unroll
                for (int e = 0; e < G; ++e) v[i][e] += b.v[e];
            }
            if (HIST && rep.any(i)) {
#pragma unroll
                for (int e = 0; e < G; ++e) {
                    const int n = rep.at(i, e);
                    if (n > 0) {
                        v[i][e] *= v[i][e] > 0.0f ? a.inv_repetition : a.op.repetition;
                        v[i][e] -= a.op.presence + a.op.frequency * (float)n;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < G; ++e) v[i][e] *= a.inv_temperature;
        }
    }
    __device__ __forceinline__ bool allowed(int i, int e) const { return (ok[i] >> e) & 1; }
    __device__ __forceinline__ float largest() const {
        float m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < G; ++e)
                if (allowed(i, e)) m = fmaxf(m, v[i][e]);
        return wave_max(m);
    }
    // v = exp(v - shift) where allowed, 0 elsewhere; their sum.
    __device__ __forceinline__ float exponentials(float shift) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < G; ++e) {
                v[i][e] = allowed(i, e) ? expf(v[i][e] - shift) : 0.0f;
                s += v[i][e];
            }
        return fl_wave_sum_f32(s);
    }
    __device__ __forceinline__ void store_weights(float *y, int base, int cols, float inv) const {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            Group<float, G> q;
#pragma unroll
            for (int e = 0; e < G; ++e) q.v[e] = allowed(i, e) ? v[i][e] * inv : 0.0f;  // inv may be NaN
            store_group(y, base + C::local(i), cols, q);
        }
    }
    template <bool PAST>
    __device__ __forceinline__ void store_values(T *y, int base, int cols, float fill) const {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            Group<T, G> q;
#pragma unroll
            for (int e = 0; e < G; ++e) q.v[e] = (T)(allowed(i, e) ? v[i][e] : fill);
            store_group<PAST>(y, base + C::local(i), cols, q);
        }
    }
};

enum { LG_CONSTRAIN, LG_PAST, LG_SHARED, LG_SOFTMAX, LG_STATS, LG_JOINED };
constexpr int LG_SHARE = 4;  // rows of a wave, LG_SHARED

// Forward of a wave's segment.  LG_PAST: stores past the caches; LG_SHARED: so,
// of LG_SHARE rows with one bias, which is loaded once.  LG_SOFTMAX: it is the
// row.  LG_STATS: its maximum and sum; LG_JOINED: the softmax with the row's
// joined ones.  [32 x 4600000] fp32 with 60 ids a row 224 us = 5.3 TB/s,
// [509 x 123000] bf16 72 us = 3.5 TB/s of the rows (and as many bytes of the bias
// rows from the caches), the softmax of [4608 x 1645] 21 us = 2.9 TB/s: with 7
// or 8 waves a SIMD bound by how many loads are under way (bias loads ahead of
// the repeats took registers: 4 waves, 103 us for 79).
template <typename T, int VPT, int MODE, bool HIST>
__global__ __launch_bounds__(LG_NT) void k_logits(LogitArgs a, void *out, float2 *stats) {
    using Seg = Segment<T, VPT, HIST>;
    __shared__ uint32_t words[HIST ? LG_WAVES : 1][HIST ? Seg::SEG / 2 : 1];
    const uint32_t item = (uint32_t)fl_block() * (blockDim.x / FL_WAVE) + fl_wave_id();
    const int64_t row = item / a.segments * (MODE == LG_SHARED ? LG_SHARE : 1), cols = a.op.cols;
    const int base = (int)(item % a.segments) * Seg::SEG;
    if (row >= a.op.rows) return;
    Seg s;
    typename Seg::Bias bias;
    uint32_t *lds = words[HIST ? fl_wave_id() : 0];
    if constexpr (MODE == LG_SHARED) {
        Seg::load_bias(a.op.bias, base, (int)cols, bias);
        const int64_t end = row + LG_SHARE < a.op.rows ? row + LG_SHARE : a.op.rows;
        for (int64_t r = row; r < end; ++r) {
            s.template load<true>(a, r, base, lds, bias);
            s.template store_values<true>((T *)out + r * cols, base, (int)cols, a.op.fill);
        }
        return;
    }
    s.template load<false>(a, row, base, lds, bias);
    if constexpr (MODE == LG_CONSTRAIN || MODE == LG_PAST) {
        s.template store_values<MODE == LG_PAST>((T *)out + row * cols, base, (int)cols, a.op.fill);
    } else if constexpr (MODE == LG_JOINED) {
        const float2 *st = stats + row * a.segments;
        float m = -__builtin_inff(), sum = 0.0f;
        for (uint32_t i = fl_lane(); i < a.segments; i += FL_WAVE) m = fmaxf(m, st[i].x);
        m = wave_max(m);
        if (m == -__builtin_inff()) m = 0.0f;
        for (uint32_t i = fl_lane(); i < a.segments; i += FL_WAVE) sum += st[i].y * expf(st[i].x - m);
        sum = fl_wave_sum_f32(sum);
        s.exponentials(m);
        s.store_weights((float *)out + row * cols, base, (int)cols, 1.0f / (sum == 0.0f ? 1.0f : sum));
    } else {
        const float m = s.largest();
        const float sum = s.exponentials(m == -__builtin_inff() ? 0.0f : m);
        if constexpr (MODE == LG_STATS) {
            // a segment of nothing but NaN keeps its sum: a maximum of 0 lets it through
            if (fl_lane() == 0) stats[item] = make_float2(m == -__builtin_inff() && sum != sum ? 0.0f : m, sum);
        } else {
            s.store_weights((float *)out + row * cols, base, (int)cols, 1.0f / (sum == 0.0f ? 1.0f : sum));
        }
    }
}

struct GradArgs {
    LogitArgs l;
    const void *g;        // gradient of the output (T; the softmax: float)
    const float *w;       // the softmax's output
    const float *dots;    // [rows] sum w g, of rows of several segments
    void *dx;
    float *terms;         // [rows, cols] fp32 terms of dbias (rows of one segment), or null
    float *dbias;         // [parts][bias_rows][cols]
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

// What the gradient of a row's segment reads, and its terms.
template <typename T, int VPT, bool SOFTMAX, bool HIST>
struct GradSegment {
    static constexpr int G = group_cols<T>();
    using C = Columns<G, VPT>;
    using TG = std::conditional_t<SOFTMAX, float, T>;
    Group<TG, G> g[VPT];
    Group<float, G> w[SOFTMAX ? VPT : 1];
    int64_t row, head;
    RowView r;

    __device__ __forceinline__ void load(const GradArgs &a, int64_t at, int base) {
        row = at;
        r = row_view(a.l.op, row);
        const int64_t cols = a.l.op.cols;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            g[i] = load_group<TG, G>((const TG *)a.g + row * cols, base + C::local(i), (int)cols);
            if (SOFTMAX) w[i] = load_group<float, G>(a.w + row * cols, base + C::local(i), (int)cols);
        }
        if (HIST) head = head_id(r);
    }
    // Writes the row's dx and adds its terms to acc.
    template <bool WHOLE, bool PAST>
    __device__ __forceinline__ void apply(const GradArgs &a, int base, uint32_t *lds, float (&acc)[VPT][G]) {
        const fl_logits &op = a.l.op;
        const int cols = (int)op.cols;
        unsigned ok[VPT];
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            ok[i] = C::bits(r, base + C::local(i), cols);
            if (SOFTMAX && WHOLE)
#pragma unroll
                for (int e = 0; e < G; ++e)
                    s += ((ok[i] >> e) & 1) && w[i].v[e] != 0.0f ? w[i].v[e] * (float)g[i].v[e] : 0.0f;
        }
        if (SOFTMAX) s = WHOLE ? fl_wave_sum_f32(s) : a.dots[row];
        Repeats<G, VPT> rep;
        if (HIST) rep.count(r, head, base, cols, lds);
        const T *x = (const T *)op.x + row * op.ldx;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = base + C::local(i);
            float u[G];
#pragma unroll
            for (int e = 0; e < G; ++e) {
                u[e] = SOFTMAX ? w[i].v[e] * ((float)g[i].v[e] - s) : (float)g[i].v[e];
                if (SOFTMAX && w[i].v[e] == 0.0f) u[e] = 0.0f;
                u[e] *= a.l.inv_temperature;
            }
            if (HIST && rep.any(i)) {
#pragma unroll
                for (int e = 0; e < G; ++e)
                    if (rep.at(i, e) > 0 && c + e < cols) {
                        const float z = (float)x[c + e] + (r.bias ? r.bias[c + e] : 0.0f);
                        u[e] *= z > 0.0f ? a.l.inv_repetition : op.repetition;
                    }
            }
            Group<T, G> o;
#pragma unroll
            for (int e = 0; e < G; ++e) {
                u[e] = (ok[i] >> e) & 1 ? u[e] : 0.0f;
                acc[i][e] += u[e];
                o.v[e] = (T)u[e];
            }
            if (a.dx) store_group<PAST>((T *)a.dx + row * op.cols, c, cols, o);
            if (a.terms) {
                Group<float, G> f;
#pragma unroll
                for (int e = 0; e < G; ++e) f.v[e] = u[e];
                store_group(a.terms + row * op.cols, c, cols, f);
            }
        }
    }
};

// Gradients of the rows: a wave a segment.  WHOLE: it is the row.  (The softmax
// of [4608 x 1645]: 25 us = 3.6 TB/s.)
template <typename T, int VPT, bool SOFTMAX, bool HIST, bool WHOLE>
__global__ __launch_bounds__(LG_NT) void k_logits_grad(GradArgs a) {
    using Grad = GradSegment<T, VPT, SOFTMAX, HIST>;
    __shared__ uint32_t words[HIST ? LG_WAVES : 1][HIST ? Grad::C::SEG / 2 : 1];
    const uint32_t item = (uint32_t)fl_block() * (blockDim.x / FL_WAVE) + fl_wave_id();
    const int64_t row = item / a.l.segments;
    const int base = (int)(item % a.l.segments) * Grad::C::SEG;
    if (row >= a.l.op.rows) return;
    float acc[VPT][Grad::G] = {};
    Grad g;
    g.load(a, row, base);
    g.template apply<WHOLE, false>(a, base, words[HIST ? fl_wave_id() : 0], acc);
}

// Gradients of rows of several segments with dbias: a wave takes one segment
// of all the rows of a list.  (Loading the next row's values ahead took 256
// registers and was slower than the twice as many waves without.)  Its
// outputs go past the caches ([509 x 123000] bf16 with 74 table rows 122 -> 107 us).
template <typename T, int VPT, bool SOFTMAX, bool HIST>
__global__ __launch_bounds__(LG_NT) void k_logits_table_grad(GradArgs a) {
    using Grad = GradSegment<T, VPT, SOFTMAX, HIST>;
    constexpr int G = Grad::G, SEG = Grad::C::SEG;
    __shared__ uint32_t words[HIST ? LG_WAVES : 1][HIST ? SEG / 2 : 1];
    const int64_t cols = a.l.op.cols;
    const uint32_t segments = (uint32_t)((cols + SEG - 1) / SEG);
    uint32_t item = (uint32_t)fl_block() * LG_WAVES + fl_wave_id();
    const int base = (int)(item % segments) * SEG;
    item /= segments;
    const uint32_t part = item % a.parts;
    const int64_t list = item / a.parts;
    if (list >= a.lists) return;
    float acc[VPT][G] = {};
    const RowList rows(a, list, part);
    for (int64_t q = rows.q0; q < rows.q1; ++q) {
        Grad g;
        g.load(a, rows.row(a, q), base);
        g.template apply<false, true>(a, base, words[HIST ? fl_wave_id() : 0], acc);
    }
    if (list >= a.l.op.bias_rows) return;  // the rows of no group
    float *b = a.dbias + ((int64_t)part * a.l.op.bias_rows + list) * cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        Group<float, G> o;
#pragma unroll
        for (int e = 0; e < G; ++e) o.v[e] = acc[i][e];
        store_group<true>(b, base + Grad::C::local(i), (int)cols, o);
    }
}

// dbias of rows of one segment, from their fp32 terms: four columns a thread,
// the rows of a list (a part of them) in order ([4608 x 1645] into 1644 rows:
// 20 us = 2.0 TB/s).
__global__ __launch_bounds__(LG_NT) void k_logits_sums(GradArgs a) {
    const int64_t cols = a.l.op.cols;
    const uint32_t blocks = (uint32_t)((cols + 4 * LG_NT - 1) / (4 * LG_NT)), block = (uint32_t)fl_block(),
                   item = block / blocks;
    const int c = (int)((block % blocks) * LG_NT + threadIdx.x) * 4;
    const uint32_t part = item % a.parts;
    const int64_t list = item / a.parts;
    if (c >= cols || list >= a.l.op.bias_rows) return;
    const RowList rows(a, list, part);
    const float *terms = a.terms ? a.terms : (const float *)a.dx;  // fp32 dx are the terms themselves
    float s[4] = {0, 0, 0, 0};
    int64_t q = rows.q0;
    for (; q + 4 <= rows.q1; q += 4) {
        Group<float, 4> t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float *row = terms + rows.row(a, q + j) * cols;
            if (c + 4 <= cols) __builtin_memcpy(&t[j], row + c, 16);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) t[j].v[e] = c + e < cols ? row[c + e] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += t[j].v[e];
    }
    for (; q < rows.q1; ++q) {
        const float *row = terms + rows.row(a, q) * cols;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += c + e < cols ? row[c + e] : 0.0f;
    }
    float *b = a.dbias + ((int64_t)part * a.l.op.bias_rows + list) * cols;
    store_group(b, c, (int)cols, Group<float, 4>{{s[0], s[1], s[2], s[3]}});
}

// sum w g of one segment of a row.
__global__ __launch_bounds__(LG_NT) void k_logits_dot(LogitArgs a, const float *__restrict__ g,
                                                      const float *__restrict__ w, float *__restrict__ dots) {
    using C = Columns<4, LG_SEG / FL_WAVE / 4>;
    const uint32_t item = (uint32_t)fl_block() * LG_WAVES + fl_wave_id();
    const int64_t row = item / a.segments;
    const int cols = (int)a.op.cols, base = (int)(item % a.segments) * LG_SEG;
    if (row >= a.op.rows) return;
    const RowView r = row_view(a.op, row);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < C::SEG / FL_WAVE / 4; ++i) {
        const int c = base + C::local(i);
        const unsigned bits = C::bits(r, c, cols);
        const Group<float, 4> p = load_group<float, 4>(w + row * a.op.cols, c, cols);
        const Group<float, 4> q = load_group<float, 4>(g + row * a.op.cols, c, cols);
#pragma unroll
        for (int e = 0; e < 4; ++e) s += ((bits >> e) & 1) && p.v[e] != 0.0f ? p.v[e] * q.v[e] : 0.0f;
    }
    s = fl_wave_sum_f32(s);
    if (fl_lane() == 0) dots[item] = s;
}

__global__ __launch_bounds__(FL_WAVE) void k_logits_join(const float *__restrict__ part, int64_t rows,
                                                         int64_t segments, float *__restrict__ dots) {
    const int64_t row = fl_block();
    if (row >= rows) return;
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < segments; i += FL_WAVE) s += part[row * segments + i];
    s = fl_wave_sum_f32(s);
    if (threadIdx.x == 0) dots[row] = s;
}

// One bit a column of a byte mask, 32 columns a word.
__global__ __launch_bounds__(256) void k_pack_bits(const uint8_t *__restrict__ mask, int64_t rows, int64_t cols,
                                                   int64_t words, uint32_t *__restrict__ out) {
    const int64_t per = (cols + FL_WAVE - 1) / FL_WAVE;  // ballots a row
    const int64_t t = (fl_block() * 256 + threadIdx.x) / FL_WAVE;
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
    // the kernels multiply by their reciprocals, which have to be normal numbers as well
    const auto divides = [](float v) { return v >= 0x1p-126f && v <= 0x1p126f; };
    if (!divides(op->temperature) || !divides(op->repetition))
        return fl_fail(FL_ERR_ARG, "%s: temperature and repetition must lie in the range [2^-126, 2^126]", what);
    if (!(fabsf(op->presence) < INFINITY) || !(fabsf(op->frequency) < INFINITY))
        return fl_fail(FL_ERR_ARG, "%s: presence and frequency must lie in float32's range", what);
    if (op->allowed && (op->allowed_rows < 1 || op->allowed_ld < lg_ceil(op->cols, 32) ||
                        (op->allowed_rows > 1 && op->rows > 0 && !op->group)))
        return fl_fail(FL_ERR_ARG, "%s: bad shape of the allowed table", what);
    if (op->bias && (op->bias_rows < 1 || (op->bias_rows > 1 && op->rows > 0 && !op->group)))
        return fl_fail(FL_ERR_ARG, "%s: bad shape of the bias table", what);
    if (op->history && op->history_len < 0) return fl_fail(FL_ERR_ARG, "%s: bad shape of the history", what);
    if (op->rows > 0 && op->cols > 0 && !op->x) return fl_fail(FL_ERR_ARG, "%s: null pointer", what);
    if (op->cols >= 1ll << 29) return fl_fail(FL_ERR_ARG, "%s: rows of fewer than 2^29 columns (shape)", what);
    if (op->cols && op->rows > 0x7fffffffll / lg_ceil(op->cols, LG_SEG))
        return fl_fail(FL_ERR_ARG, "%s: too many rows for one launch (shape)", what);
    return FL_OK;
}

int64_t segments_of(const fl_logits *op) { return lg_ceil(op->cols, LG_SEG); }

LogitArgs lg_args(const fl_logits *op) {
    LogitArgs a;
    a.op = *op;
    if (!op->allowed) a.op.allowed_rows = 0;
    if (!op->bias) a.op.bias_rows = 0;
    a.inv_temperature = 1.0f / op->temperature;
    a.inv_repetition = 1.0f / op->repetition;
    a.segments = (uint32_t)segments_of(op);
    return a;
}

// Waves of a workgroup whose waves work alone: one where there are too few to
// give every CU a workgroup of four.
int lone_waves(int64_t items) { return items < 1024 ? 1 : LG_WAVES; }

template <typename T, int VPT, int MODE>
void launch(hipStream_t st, const fl_logits *op, void *out, float2 *stats) {
    LogitArgs a = lg_args(op);
    // without a softmax a row is cut anywhere: segments of half the columns take
    // fewer registers ([509 x 123000] bf16 79 -> 73 us)
    if (MODE <= LG_SHARED) a.segments = (uint32_t)lg_ceil(op->cols, FL_WAVE * group_cols<T>() * VPT);
    const int64_t items = (MODE == LG_SHARED ? lg_ceil(op->rows, LG_SHARE) : op->rows) * a.segments;
    const int waves = lone_waves(items);
    const dim3 grid = grid_of(lg_ceil(items, waves)), nt(waves * FL_WAVE);
    if (op->history) FL_LAUNCH("k_logits", (k_logits<T, VPT, MODE, true>), grid, nt, 0, st, a, out, stats);
    else FL_LAUNCH("k_logits", (k_logits<T, VPT, MODE, false>), grid, nt, 0, st, a, out, stats);
}

// The instance whose wave takes the columns: f(VPT), VPT in 1, 2, 4 (and 8).
template <typename T, typename F>
void by_columns(int64_t cols, F &&f) {
    constexpr int lane = FL_WAVE * group_cols<T>();
    if (cols <= lane) f(std::integral_constant<int, 1>{});
    else if (cols <= 2 * lane) f(std::integral_constant<int, 2>{});
    else if (LG_SEG == 4 * lane || cols <= 4 * lane) f(std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, LG_SEG / lane>{});
}

template <typename T, bool SOFTMAX>
int forward(hipStream_t st, const fl_logits *op, void *out, float2 *stats, const char *what) {
    if (SOFTMAX && op->cols > LG_SEG) {
        constexpr int V = LG_SEG / FL_WAVE / group_cols<T>();
        launch<T, V, LG_STATS>(st, op, out, stats);
        launch<T, V, LG_JOINED>(st, op, out, stats);
    } else {
        by_columns<T>(op->cols, [&](auto v) {
            constexpr int V = decltype(v)::value, HALF = LG_SEG / 2 / FL_WAVE / group_cols<T>();
            if constexpr (SOFTMAX) launch<T, V, LG_SOFTMAX>(st, op, out, stats);
            // an output that the L2s (32 MB) do not keep for its reader goes past
            // them ([32 x 4600000] fp32 254 -> 246 us); one bias for all rows is
            // loaded once for four (246 -> 224; two or eight: 228; rows taken in
            // the order of a table's groups left the rows' streams: 71 -> 92 us
            // for [509 x 123000] bf16)
            else if (op->cols > LG_SEG && op->rows * op->cols * (int64_t)sizeof(T) > (32 << 20)) {
                if (op->bias && op->bias_rows == 1) launch<T, HALF, LG_SHARED>(st, op, out, stats);
                else launch<T, HALF, LG_PAST>(st, op, out, stats);
            }
            else launch<T, V < HALF ? V : HALF, LG_CONSTRAIN>(st, op, out, stats);
        });
    }
    return fl_check_launch(what);
}

// Row lists of a bias table's gradient: its groups and, when there are
// several, the owners of none.
int64_t grad_lists(const fl_logits *op) { return op->bias_rows > 1 ? op->bias_rows + 1 : 1; }

// Parts of a list: some 8192 waves in all, of at least 8 rows on average.
int grad_parts(const fl_logits *op, int64_t lists) {
    const int64_t waves = op->cols <= LG_SEG ? lg_ceil(op->cols, 256) : lg_ceil(op->cols, LG_SEG / 2);
    const int64_t want = lg_ceil(8192, lists * waves), most = op->rows / (8 * lists);
    const int64_t p = want < most ? want : most;
    return (int)(p < 1 ? 1 : p > 256 ? 256 : p);
}

template <typename T, int VPT, bool SOFTMAX, bool HIST>
void launch_grad(hipStream_t st, const GradArgs &a) {
    const fl_logits &op = a.l.op;
    constexpr bool LONG = VPT == LG_SEG / FL_WAVE / group_cols<T>();
    const bool whole = op.cols <= LG_SEG;
    if constexpr (LONG) {
        if (!whole && a.dbias) {  // half as many columns a wave: more waves, fewer registers
            const int64_t waves = a.lists * a.parts * lg_ceil(op.cols, LG_SEG / 2);
            FL_LAUNCH("k_logits_table_grad", (k_logits_table_grad<T, VPT / 2, SOFTMAX, HIST>),
                      grid_of(lg_ceil(waves, LG_WAVES)), dim3(LG_NT), 0, st, a);
            return;
        }
    }
    const int64_t items = op.rows * a.l.segments;
    if (items > 0) {
        const int waves = lone_waves(items);
        const dim3 grid = grid_of(lg_ceil(items, waves)), nt(waves * FL_WAVE);
        if constexpr (SOFTMAX && LONG) {
            if (!whole) FL_LAUNCH("k_logits_grad", (k_logits_grad<T, VPT, true, HIST, false>), grid, nt, 0, st, a);
        }
        if (!SOFTMAX || whole)
            FL_LAUNCH("k_logits_grad", (k_logits_grad<T, VPT, SOFTMAX, HIST, true>), grid, nt, 0, st, a);
    }
    if (a.dbias) {
        const int64_t sums = op.bias_rows * a.parts * lg_ceil(op.cols, 4 * LG_NT);
        FL_LAUNCH("k_logits_sums", k_logits_sums, grid_of(sums), dim3(LG_NT), 0, st, a);
    }
}

// The gradient's workspace: the parts of dbias, its terms (rows of one segment
// whose dx does not hold them), the segments' dots and the rows' (softmax of
// several segments), and the owners by group.
struct GradSpace {
    size_t parts, terms, dots, order, offsets, group, group_bytes, bytes;
};

GradSpace grad_space(const fl_logits *op, bool softmax, bool with_dx, bool with_dbias) {
    GradSpace s{};
    const auto take = [&](size_t n) {
        const size_t at = s.bytes;
        s.bytes += (n + 255) / 256 * 256;
        return at;
    };
    if (with_dbias) {
        const int parts = grad_parts(op, grad_lists(op));
        if (parts > 1) s.parts = take((size_t)parts * op->bias_rows * op->cols * 4);
        if (op->cols <= LG_SEG && !(with_dx && op->dtype == FL_F32)) s.terms = take((size_t)op->rows * op->cols * 4);
        if (op->bias_rows > 1) {
            const int64_t owners = op->rows / op->inner;
            s.order = take((size_t)owners * 4 + 4);
            s.offsets = take((size_t)(op->bias_rows + 1) * 4);
            s.group_bytes = fl_group_rows_bytes(owners, op->bias_rows);
            s.group = take(s.group_bytes);
        }
    }
    if (softmax && op->cols > LG_SEG) s.dots = take((size_t)op->rows * (segments_of(op) + 1) * 4);
    return s;
}

template <typename T, bool SOFTMAX>
int gradient(hipStream_t st, const fl_logits *op, const float *w, const void *grad, void *dx, float *dbias, char *ws) {
    const GradSpace sp = grad_space(op, SOFTMAX, dx != nullptr, dbias != nullptr);
    GradArgs a{};
    a.l = lg_args(op);
    a.g = grad;
    a.w = w;
    a.dx = dx;
    a.parts = 1;
    if (dbias) {
        a.lists = grad_lists(op);
        a.parts = (uint32_t)grad_parts(op, a.lists);
        a.dbias = a.parts > 1 ? (float *)(ws + sp.parts) : dbias;
        if (op->cols <= LG_SEG && !(std::is_same_v<T, float> && dx)) a.terms = (float *)(ws + sp.terms);
        if (op->bias_rows > 1) {
            int32_t *order = (int32_t *)(ws + sp.order), *offsets = (int32_t *)(ws + sp.offsets);
            const int rc = fl_group_rows(st, op->group, op->rows / op->inner, op->bias_rows, order, offsets, nullptr,
                                         ws + sp.group, sp.group_bytes);
            if (rc) return rc;
            a.order = order;
            a.offsets = offsets;
        }
    } else if (op->rows == 0) return FL_OK;
    if (SOFTMAX && op->cols > LG_SEG && op->rows > 0) {
        float *part = (float *)(ws + sp.dots), *dots = part + op->rows * a.l.segments;
        FL_LAUNCH("k_logits_dot", k_logits_dot, grid_of(lg_ceil(op->rows * a.l.segments, LG_WAVES)), dim3(LG_NT),
                  0, st, a.l, (const float *)grad, w, part);
        FL_LAUNCH("k_logits_join", k_logits_join, grid_of(op->rows), dim3(FL_WAVE), 0, st, part, op->rows,
                  (int64_t)a.l.segments, dots);
        a.dots = dots;
    }
    const bool signs = op->history && op->repetition != 1.0f;  // the slopes need the repeats
    by_columns<T>(op->cols, [&](auto v) {
        if (signs) launch_grad<T, decltype(v)::value, SOFTMAX, true>(st, a);
        else launch_grad<T, decltype(v)::value, SOFTMAX, false>(st, a);
    });
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
    FL_LAUNCH("k_pack_bits", fl::k_pack_bits, fl::grid_of(fl::lg_ceil(waves, 4)), dim3(256), 0,
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
    if (!op || op->cols <= fl::LG_SEG || op->rows < 1) return 0;
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

size_t fl_logits_grad_bytes(const fl_logits *op, int softmax, int with_dx, int with_dbias) {
    if (!op || op->rows < 0 || op->cols < 1 || op->inner < 1) return 0;
    return fl::grad_space(op, softmax != 0, with_dx != 0, with_dbias != 0 && op->bias && op->bias_rows > 0).bytes;
}

int fl_logits_grad(void *stream, const fl_logits *op, const float *w, const void *grad, void *dx, float *dbias,
                   void *ws, size_t ws_bytes) {
    const int rc = fl::lg_check(op, "logits_grad");
    if (rc) return rc;
    if (op->cols == 0) return FL_OK;
    if (dbias && !op->bias) return fl::fl_fail(FL_ERR_ARG, "logits_grad: the gradient of no bias table");
    if (op->rows > 0 && !grad) return fl::fl_fail(FL_ERR_ARG, "logits_grad: null pointer");
    const size_t need = fl_logits_grad_bytes(op, w != nullptr, dx != nullptr, dbias != nullptr);
    if (ws_bytes < need || (need && !ws)) return fl::fl_fail(FL_ERR_ARG, "logits_grad: workspace too small");
    if ((uintptr_t)ws % 16) return fl::fl_fail(FL_ERR_ARG, "logits_grad: workspace must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    if (w) {
        FL_BY_TYPE(op->dtype, (fl::gradient<T, true>(st, op, w, grad, dx, dbias, (char *)ws)))
    }
    FL_BY_TYPE(op->dtype, (fl::gradient<T, false>(st, op, w, grad, dx, dbias, (char *)ws)))
}

}  // extern "C"
