// Rows grouped by an index (a query's head relation, the query of a known
// answer): the stable permutation that puts equal ids next to each other, the
// groups' offsets, and the list of row tiles that the grouped products take.
//
// A stable counting sort by digits of GR_BITS bits, so one pass for up to
// 4095 groups.  A wave takes a contiguous run of rows, 64 at a time: the lanes
// with an equal digit are found with one ballot a bit, a lane's rank among
// them is a popcount, and the wave's running count of every digit is in LDS
// (16 bits each: a wave takes at most GR_WAVE_ROWS rows).  The counts are then
// scanned over the waves of a workgroup and over the workgroups, so that a
// row's place is the same on every run.  Up to GR_BLOCK_ROWS rows and 4095
// groups are one launch, whose workgroups count all rows each (latency-bound:
// 15000 rows in 74 groups are 120 KB); more rows take three launches a digit.
//
// Ids outside [0, groups) come last, behind offsets[groups]: rows of no group.
#include "fl_abi.h"
#include "fl_common.h"

namespace fl {
namespace {

constexpr int GR_NT = 1024;
constexpr int GR_WAVES = GR_NT / FL_WAVE;
constexpr int GR_BITS = 12;
constexpr int GR_DIGITS = 1 << GR_BITS;
constexpr int64_t GR_WAVE_ROWS = 1024;
constexpr int64_t GR_BLOCK_ROWS = GR_WAVE_ROWS * GR_WAVES;

struct GroupArgs {
    const int64_t *index;
    int64_t rows, groups;
    const int32_t *in_order;  // null: the identity
    int32_t *out_order;
    int32_t *hist;            // [blocks][digits]: counts, then first places
    int32_t *offsets;         // [groups + 1]
    int32_t *tiles;           // [ntiles][2] (group, first position)
    int64_t ntiles, nblocks;
    int digits, shift, bits, block;
};

__device__ __forceinline__ int64_t group_key(const GroupArgs &a, int64_t row) {
    const int64_t k = a.index[row];
    return k >= 0 && k < a.groups ? k : a.groups;
}

// Lanes whose digit equals this one's (among the active rows).
__device__ __forceinline__ unsigned long long equal_lanes(int d, bool active, int bits) {
    const unsigned long long m = __ballot(active);
    unsigned lo = (unsigned)m, hi = (unsigned)(m >> 32);
    for (int b = 0; b < bits; ++b) {
        const int mine = (d << (31 - b)) >> 31;  // the bit, in every place
        const unsigned long long s = __ballot(mine != 0);
        lo &= ~((unsigned)s ^ (unsigned)mine);
        hi &= ~((unsigned)(s >> 32) ^ (unsigned)mine);
    }
    return ((unsigned long long)hi << 32) | lo;
}

// The rows of a wave's run, a strip of 64 at a time: all loaded before the
// first is worked on (one strip's loads after another's took 25 us for 15000
// rows, nothing but their latency).
struct WaveRows {
    static constexpr int STRIPS = (int)(GR_WAVE_ROWS / FL_WAVE);
    int32_t row[STRIPS];
    int digit[STRIPS], rank[STRIPS];
    int strips;
    int64_t begin, end;

    __device__ __forceinline__ void load(const GroupArgs &a) {
        // the workgroup's rows in equal contiguous runs of whole strips
        const int64_t b0 = (int64_t)blockIdx.x * GR_BLOCK_ROWS;
        const int64_t n = a.rows - b0 < GR_BLOCK_ROWS ? a.rows - b0 : GR_BLOCK_ROWS;
        const int64_t per = ((n + GR_WAVES - 1) / GR_WAVES + FL_WAVE - 1) / FL_WAVE * FL_WAVE;
        const int64_t s = fl_wave_id() * per;
        begin = b0 + (s < n ? s : n);
        end = b0 + (s + per < n ? s + per : n);
        strips = (int)((end - begin + FL_WAVE - 1) / FL_WAVE);
#pragma unroll
        for (int i = 0; i < STRIPS; ++i) {
            const int64_t p = begin + i * FL_WAVE + fl_lane();
            row[i] = p < end ? (a.in_order ? a.in_order[p] : (int32_t)p) : 0;
        }
#pragma unroll
        for (int i = 0; i < STRIPS; ++i)
            digit[i] = i < strips ? (int)((group_key(a, row[i]) >> a.shift) & (a.digits - 1)) : 0;
    }
    // Counts the digits in cnt (0 before); every row's rank among the wave's
    // rows of its digit.
    __device__ __forceinline__ void count(const GroupArgs &a, uint16_t *cnt) {
#pragma unroll
        for (int i = 0; i < STRIPS; ++i) {
            rank[i] = 0;
            if (i < strips) {
                const bool active = begin + i * FL_WAVE + fl_lane() < end;
                const unsigned long long eq = equal_lanes(digit[i], active, a.bits);
                if (active) {
                    const int before = __popcll(eq & ((1ull << fl_lane()) - 1));
                    const int old = cnt[digit[i]];
                    rank[i] = old + before;
                    if (before == 0) cnt[digit[i]] = (uint16_t)(old + __popcll(eq));
                }
                fl_wave_sync();
            }
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F &&f) const {
#pragma unroll
        for (int i = 0; i < STRIPS; ++i)
            if (begin + i * FL_WAVE + fl_lane() < end) f(row[i], digit[i], rank[i]);
    }
};

__device__ __forceinline__ void clear_counts(uint16_t *cnt, int digits) {
    uint32_t *c = reinterpret_cast<uint32_t *>(cnt);
    for (int i = threadIdx.x; i < GR_WAVES * digits / 2; i += GR_NT) c[i] = 0;
}

// Exclusive scan, by one workgroup, of f(i) for i < n; g(i, prefix) takes it.
template <typename F, typename G>
__device__ __forceinline__ void block_scan(int64_t n, int *lds, F &&f, G &&g) {
    int carry = 0;
    for (int64_t i0 = 0; i0 < n; i0 += GR_NT) {
        const int64_t i = i0 + threadIdx.x;
        const int v = i < n ? f(i) : 0;
        int total;
        const int pre = fl_block_excl_scan<GR_NT>(v, lds, &total);
        if (i < n) g(i, carry + pre);
        carry += total;
    }
}

// The tiles of every group (group `groups`: the rows of none), the rest of
// the list marked unused.
__device__ __forceinline__ void write_tiles(const GroupArgs &a, int *lds) {
    int used = 0;
    const int64_t ng = a.groups + 1;
    for (int64_t i0 = 0; i0 < ng; i0 += GR_NT) {
        const int64_t i = i0 + threadIdx.x;
        int b = 0, n = 0;
        if (i < ng) {
            b = a.offsets[i];
            const uint32_t rows = (uint32_t)((i < a.groups ? a.offsets[i + 1] : (int)a.rows) - b);
            n = (int)((rows + a.block - 1) / a.block);  // rows + block may pass 2^31
        }
        int total;
        const int pre = fl_block_excl_scan<GR_NT>(n, lds, &total);
        for (int t = 0; t < n; ++t) {
            a.tiles[2 * (int64_t)(used + pre + t)] = (int)i;
            a.tiles[2 * (int64_t)(used + pre + t) + 1] = b + t * a.block;
        }
        used += total;
    }
    for (int64_t t = used + threadIdx.x; t < a.ntiles; t += GR_NT) a.tiles[2 * t] = -1;
}

// One launch: every workgroup takes GR_NT rows, and counts the groups of all
// rows itself, those before its own apart, so that none waits for another
// (16384 rows in 24 groups 13 us; in one workgroup 20 to 25).
__global__ __launch_bounds__(GR_NT) void k_group_one(GroupArgs a) {
    extern __shared__ uint8_t mine[];  // [waves][digits] of the workgroup's own rows
    __shared__ int lds[GR_WAVES + 1];
    __shared__ int first[GR_DIGITS], rest[GR_DIGITS];
    const int64_t b0 = (int64_t)blockIdx.x * GR_NT, own = b0 + threadIdx.x;
    for (int i = threadIdx.x; i < a.digits; i += GR_NT) first[i] = rest[i] = 0;
    uint32_t *m32 = reinterpret_cast<uint32_t *>(mine);
    for (int i = threadIdx.x; i < GR_WAVES * a.digits / 4; i += GR_NT) m32[i] = 0;
    int key[GR_BLOCK_ROWS / GR_NT], digit = 0;
#pragma unroll
    for (int j = 0; j < (int)(GR_BLOCK_ROWS / GR_NT); ++j) {
        const int64_t p = (int64_t)j * GR_NT + threadIdx.x;
        key[j] = p < a.rows ? (int)group_key(a, p) : -1;
        if (p == own) digit = key[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < (int)(GR_BLOCK_ROWS / GR_NT); ++j)
        if (key[j] >= 0) atomicAdd(j < (int)blockIdx.x ? &first[key[j]] : &rest[key[j]], 1);
    const bool active = own < a.rows;
    const int wave = fl_wave_id();
    const unsigned long long eq = equal_lanes(digit, active, a.bits);
    int rank = 0;
    if (active) {
        rank = __popcll(eq & ((1ull << fl_lane()) - 1));
        if (rank == 0) mine[wave * a.digits + digit] = (uint8_t)__popcll(eq);
    }
    __syncthreads();
    block_scan(
        a.digits, lds, [&](int64_t d) { return first[d] + rest[d]; },
        [&](int64_t d, int pre) {
            first[d] += pre;
            if (blockIdx.x == 0 && d <= a.groups) a.offsets[d] = pre;
        });
    __syncthreads();
    if (active) {
        int at = first[digit] + rank;
        for (int w = 0; w < wave; ++w) at += mine[w * a.digits + digit];
        a.out_order[at] = (int32_t)own;
    }
    if (blockIdx.x == 0 && a.tiles) {
        __threadfence_block();
        __syncthreads();
        write_tiles(a, lds);
    }
}

__global__ __launch_bounds__(GR_NT) void k_group_count(GroupArgs a) {
    extern __shared__ uint16_t cnt[];
    WaveRows rows;
    rows.load(a);
    clear_counts(cnt, a.digits);
    __syncthreads();
    rows.count(a, cnt + fl_wave_id() * a.digits);
    __syncthreads();
    for (int d = threadIdx.x; d < a.digits; d += GR_NT) {
        int run = 0;
        for (int w = 0; w < GR_WAVES; ++w) run += cnt[w * a.digits + d];
        a.hist[(int64_t)blockIdx.x * a.digits + d] = run;
    }
}

__global__ __launch_bounds__(GR_NT) void k_group_scan(GroupArgs a) {
    __shared__ int lds[GR_WAVES + 1];
    block_scan(
        a.digits, lds,
        [&](int64_t d) {
            int run = 0;
            for (int64_t b = 0; b < a.nblocks; ++b) {
                const int c = a.hist[b * a.digits + d];
                a.hist[b * a.digits + d] = run;
                run += c;
            }
            return run;
        },
        [&](int64_t d, int pre) {
            for (int64_t b = 0; b < a.nblocks; ++b) a.hist[b * a.digits + d] += pre;
        });
}

__global__ __launch_bounds__(GR_NT) void k_group_place(GroupArgs a) {
    extern __shared__ uint16_t cnt[];
    WaveRows rows;
    rows.load(a);
    clear_counts(cnt, a.digits);
    __syncthreads();
    uint16_t *mine = cnt + fl_wave_id() * a.digits;
    rows.count(a, mine);
    __syncthreads();
    for (int d = threadIdx.x; d < a.digits; d += GR_NT) {
        int run = 0;
        for (int w = 0; w < GR_WAVES; ++w) {
            const int c = cnt[w * a.digits + d];
            cnt[w * a.digits + d] = (uint16_t)run;
            run += c;
        }
    }
    __syncthreads();
    const int32_t *first = a.hist + (int64_t)blockIdx.x * a.digits;
    rows.each([&](int32_t row, int d, int rank) { a.out_order[first[d] + mine[d] + rank] = row; });
}

// Offsets by binary search in the sorted rows (the multi-launch forms).
__global__ __launch_bounds__(GR_NT) void k_group_offsets(GroupArgs a) {
    const int64_t g = (int64_t)blockIdx.x * GR_NT + threadIdx.x;
    if (g > a.groups) return;
    int64_t lo = 0, hi = a.rows;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (group_key(a, a.out_order[mid]) < g) lo = mid + 1;
        else hi = mid;
    }
    a.offsets[g] = (int32_t)lo;
}

__global__ __launch_bounds__(GR_NT) void k_group_tiles(GroupArgs a) {
    __shared__ int lds[GR_WAVES + 1];
    write_tiles(a, lds);
}

int bits_for(int64_t n) {
    int b = 0;
    while ((1ll << b) < n) ++b;
    return b < 1 ? 1 : b;
}

bool one_launch(int64_t rows, int64_t groups) { return rows <= GR_BLOCK_ROWS && groups < GR_DIGITS; }

}  // namespace
}  // namespace fl

extern "C" {

int64_t fl_group_block(int64_t rows, int64_t groups) { return rows >= 512 * groups ? 256 : rows >= 32 * groups ? 64 : 32; }

int64_t fl_group_tiles(int64_t rows, int64_t groups) {
    if (rows <= 0) return 0;
    const int64_t block = fl_group_block(rows, groups);
    return (rows + block - 1) / block + (rows < groups + 1 ? rows : groups + 1);
}

size_t fl_group_rows_bytes(int64_t rows, int64_t groups) {
    if (rows <= 0 || groups < 0 || fl::one_launch(rows, groups)) return 0;
    const int64_t nb = (rows + fl::GR_BLOCK_ROWS - 1) / fl::GR_BLOCK_ROWS;
    // the workgroups' counts and one spare order
    return (size_t)nb * fl::GR_DIGITS * 4 + (size_t)rows * 4;
}

int fl_group_rows(void *stream, const int64_t *index, int64_t rows, int64_t groups, int32_t *order, int32_t *offsets,
                  int32_t *tiles, void *ws, size_t ws_bytes) {
    if (rows < 0 || rows > 0x7fffffffll || groups < 1 || groups >= (1ll << 24))
        return fl::fl_fail(FL_ERR_ARG, "group_rows: rows must lie in the range [0, 2^31), groups in [1, 2^24)");
    if (!offsets || (rows > 0 && (!index || !order)))
        return fl::fl_fail(FL_ERR_ARG, "group_rows: null pointer");
    if (ws_bytes < fl_group_rows_bytes(rows, groups) || (!ws && fl_group_rows_bytes(rows, groups)))
        return fl::fl_fail(FL_ERR_ARG, "group_rows: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    fl::GroupArgs a{};
    a.index = index;
    a.rows = rows;
    a.groups = groups;
    a.out_order = order;
    a.offsets = offsets;
    a.tiles = tiles;
    a.ntiles = fl_group_tiles(rows, groups);
    a.block = (int)fl_group_block(rows, groups);
    const int bits = fl::bits_for(groups + 1);
    if (rows == 0) {  // every group begins at 0, and there are no tiles
        FL_LAUNCH("k_group_offsets", fl::k_group_offsets, dim3((unsigned)((groups + fl::GR_NT) / fl::GR_NT)),
                  dim3(fl::GR_NT), 0, st, a);
        return fl::fl_check_launch("group_rows");
    }
    if (fl::one_launch(rows, groups)) {
        a.bits = bits;
        a.digits = 1 << bits;
        const int64_t nb = (rows + fl::GR_NT - 1) / fl::GR_NT;
        const size_t lds = (size_t)fl::GR_WAVES * (a.digits < 4 ? 4 : a.digits);
        FL_LAUNCH("k_group_one", fl::k_group_one, dim3((unsigned)nb), dim3(fl::GR_NT), lds, st, a);
        return fl::fl_check_launch("group_rows");
    }
    a.nblocks = (rows + fl::GR_BLOCK_ROWS - 1) / fl::GR_BLOCK_ROWS;
    a.hist = (int32_t *)ws;
    int32_t *spare = a.hist + a.nblocks * fl::GR_DIGITS;
    const int passes = (bits + fl::GR_BITS - 1) / fl::GR_BITS;  // 1 or 2
    for (int p = 0; p < passes; ++p) {
        a.shift = p * fl::GR_BITS;
        a.bits = bits - a.shift < fl::GR_BITS ? bits - a.shift : fl::GR_BITS;
        a.digits = 1 << a.bits;
        a.in_order = p ? spare : nullptr;
        a.out_order = p + 1 < passes ? spare : order;
        const size_t lds = (size_t)fl::GR_WAVES * a.digits * sizeof(uint16_t);
        const dim3 grid((unsigned)a.nblocks);
        FL_LAUNCH("k_group_count", fl::k_group_count, grid, dim3(fl::GR_NT), lds, st, a);
        FL_LAUNCH("k_group_scan", fl::k_group_scan, dim3(1), dim3(fl::GR_NT), 0, st, a);
        FL_LAUNCH("k_group_place", fl::k_group_place, grid, dim3(fl::GR_NT), lds, st, a);
    }
    FL_LAUNCH("k_group_offsets", fl::k_group_offsets, dim3((unsigned)((groups + fl::GR_NT) / fl::GR_NT)),
              dim3(fl::GR_NT), 0, st, a);
    if (tiles) FL_LAUNCH("k_group_tiles", fl::k_group_tiles, dim3(1), dim3(fl::GR_NT), 0, st, a);
    return fl::fl_check_launch("group_rows");
}

}  // extern "C"
