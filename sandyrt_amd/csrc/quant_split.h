// quant_split.h -- one column tile's keys over several workgroups: which keys each
// takes, and how their parts are joined, for column tiles of COLS (query, head) rows.
// The last workgroup to arrive joins them in the same launch (in a graph: 32 sequences
// of 512 to 4096 keys 15.9 us, 18.4 with the merge kernel; 64 with a window of 1024 20.0
// and 22.1; three short f32 ones 7.1 and 8.6; one of 32749 keys 14.3 and 14.8).  The
// merge kernel is for calls without counters and gives the same bits.
#pragma once
#include <algorithm>

#include "quant_mfma.h"

namespace sandy_hip {

constexpr int kMinPairs = 4;  // pairs of 16-key tiles a split has at least: one a wave

struct SplitArgs {
    QuantAttnArgs a;
    int32_t col_tiles;  // tiles of COLS columns of the (query, head) rows of a kv head
    int32_t splits;     // workgroups a column tile's keys may be split over
    int32_t few;        // and are, up to long_pairs each
    int32_t long_pairs;
    float* part_o;      // [unit, split][COLS][D] sums relative to the maximum
    float* part_ml;     // [unit, split][COLS][2] maximum and sum of weights
    uint32_t* arrived;  // [unit][counters_of(splits)][kCounterWords] zero between calls, or null: the merge kernel joins the splits
};

// Splits are joined by the last workgroup to arrive, in groups of 16 and then
// the groups: a unit's counters are one for the groups (or the only group) and,
// where there are several, one for each.  Each has 32 bytes of its own: next to each
// other, one sequence of 32749 keys takes 14.7 us instead of 13.4, 8 of 4000 keys of 16
// / 2 heads of 128 14.0 instead of 12.1 (64 bytes and more: no further gain).
constexpr int kCounterWords = 8;
__host__ __device__ constexpr int counters_of(int splits) { return splits <= 16 ? 1 : 1 + (splits + 15) / 16; }

// The keys of one column tile: pairs of 16-key tiles from `begin`, `per` of them a split.
struct TileKeys {
    int begin, last, pairs, per, active;
};

__device__ __forceinline__ TileKeys tile_keys(const SplitArgs& d, const SeqKeys& seq, int count, int t_lo, int t_hi) {
    TileKeys k{0, -1, 0, kMinPairs, 1};
    t_hi = min(t_hi, count - 1);
    if (t_lo <= t_hi) {
        k.begin = seq.of(t_lo).first & ~15;
        k.last = seq.of(t_hi).last;
        if (k.last >= k.begin) k.pairs = (k.last - k.begin + 32) >> 5;
        k.per = max((k.pairs + d.splits - 1) / d.splits, kMinPairs);
        if (d.few < d.splits) k.per = max(k.per, min((k.pairs + d.few - 1) / d.few, d.long_pairs));
        k.active = max((k.pairs + k.per - 1) / k.per, 1);
    }
    return k;
}

// Stores and loads that go through to memory (sc1): other XCDs' L2s see them once
// the storing thread has waited for them.  Whole 16-byte pieces: as 8-byte atomics
// the parts of 2 splits of a 2048-row prompt cost 33 us, so 26.
constexpr int kThrough = 16;

struct Through {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ explicit Through(float* base) : r(__builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7fffffff, kRsrcWord3)) {}
    // `at` in floats
    __device__ __forceinline__ void put(int at, f32x4_t v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), r, 4 * at, 0, kThrough);
    }
    __device__ __forceinline__ void put(int at, float x, float y) const {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(x), __float_as_uint(y)}, r, 4 * at, 0, kThrough);
    }
    __device__ __forceinline__ f32x4_t get4(int at) const {
        return __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, 4 * at, 0, kThrough));
    }
    __device__ __forceinline__ float2 get2(int at) const {
        const u32x2_t v = __builtin_amdgcn_raw_buffer_load_b64(r, 4 * at, 0, kThrough);
        return make_float2(__uint_as_float(v[0]), __uint_as_float(v[1]));
    }
};

// Counts this workgroup in once its stores are there; true for the last of n,
// which leaves the counter zero.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, int n) {
    __shared__ bool last;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<uint32_t>(n - 1);
        if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return last;
}

// Parts 0 .. n - 1 (n <= 16) of one row and 4 dims joined, in order: `ml` gives a part's
// maximum and sum of weights, `part` its sums.
struct Joined {
    float m, total;
    bool loud;
    f32x4_t o;
};

template <typename ML, typename PART>
__device__ __forceinline__ Joined join_parts(int n, ML ml, PART part) {
    Joined j{-INFINITY, 0.0f, false, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}};
    for (int s0 = 0; s0 < n; s0 += 8) {
        float2 w[8];
        f32x4_t x[8];
#pragma unroll
        for (int s = 0; s < 8; s++) {  // past the last: the last again, unused
            w[s] = ml(min(s0 + s, n - 1));
            x[s] = part(min(s0 + s, n - 1));
        }
        float top = j.m;
        bool any = false;
#pragma unroll
        for (int s = 0; s < 8; s++) {
            top = fmaxf(top, w[s].x);
            any |= is_loud(w[s].y);
        }
        const float shift = top == -INFINITY ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f(j.m - shift);
        j.total *= f;
        j.o *= f;
        j.m = top;
        if (any && !j.loud) j.o *= kLoudDown;
        j.loud |= any;
#pragma unroll
        for (int s = 0; s < 8; s++) {
            if (s0 + s >= n) continue;
            const float e = __builtin_amdgcn_exp2f(w[s].x - shift);
            j.total += fabsf(w[s].y) * e;
            j.o += x[s] * (j.loud && !is_loud(w[s].y) ? kLoudDown : 1.0f) * e;
        }
    }
    return j;
}

// Into row `row` of a kv head's rows, dims d .. d + 3.
template <typename T>
__device__ __forceinline__ void store_joined(const QuantAttnArgs& a, const Joined& j, int row, int d, int kh, int b) {
    const int qt = divide(row, a.group, a.group_magic), qg = row - qt * a.group;
    const float inv = j.total == 0.0f ? 0.0f : 1.0f / j.total;
    store4<T>(a.out, b * a.os[0] + (kh * a.group + qg) * a.os[1] + qt * a.os[2] + d, j.o * inv * (j.loud ? kLoudUp : 1.0f));
}

// Slots first, first + stride, .. (n <= 16) of a column tile joined: into the output,
// or into slot `first`.  A thread per column and 4 dims.
template <typename T, int COLS>
__device__ __forceinline__ void join_splits(const SplitArgs& da, int64_t first, int stride, int n, int ct, int kh, int b, bool final_out) {
    __shared__ float2 joined[COLS];
    const QuantAttnArgs& a = da.a;
    const int D = a.p.dim, rows = a.group * a.p.tokens;
    const int per_col = D / 4;
    const int cols = min(COLS, rows - COLS * ct);
    const Through po(da.part_o + first * COLS * D), pm(da.part_ml + first * COLS * 2);
    for (int i = threadIdx.x; i < cols * per_col; i += 256) {
        const int c = i / per_col, d = 4 * (i - c * per_col);
        const Joined j = join_parts(n, [&](int s) { return pm.get2(2 * (s * stride * COLS + c)); },
                                    [&](int s) { return po.get4((s * stride * COLS + c) * D + d); });
        if (final_out) {
            store_joined<T>(a, j, COLS * ct + c, d, kh, b);
        } else {
            po.put(c * D + d, j.o);
            if (d == 0) joined[c] = make_float2(j.m, mark_loud(j.total, j.loud));
        }
    }
    if (final_out) return;
    __syncthreads();  // every thread has read the slot's own maximum and sum
    if (threadIdx.x < cols) pm.put(2 * threadIdx.x, joined[threadIdx.x].x, joined[threadIdx.x].y);
}

// A workgroup's own part of a column tile, joined with the other splits' by the
// last to arrive (with the merge kernel's help where there are no counters).
template <typename T, int COLS>
__device__ __forceinline__ void finish_split(const SplitArgs& da, int64_t unit, int split, int active, int ct, int kh, int b) {
    if (!da.arrived) return;
    uint32_t* arrived = da.arrived + unit * counters_of(da.splits) * kCounterWords;
    const int groups = (active + 15) / 16, grp = split / 16;
    const int in_group = min(16, active - 16 * grp);
    if (!last_to_arrive(arrived + (groups > 1 ? 1 + grp : 0) * kCounterWords, in_group)) return;
    join_splits<T, COLS>(da, unit * da.splits + 16 * grp, 1, in_group, ct, kh, b, groups == 1);
    if (groups == 1 || !last_to_arrive(arrived, groups)) return;
    join_splits<T, COLS>(da, unit * da.splits, 16, groups, ct, kh, b, true);
}

// Joins the splits of one output row, in the order of the last workgroup's join and so
// to the same bits: a workgroup per row, a thread per 4 dims of a group of 16 splits.
template <typename T, int COLS>
__global__ __launch_bounds__(256) void quant_merge_kernel(SplitArgs da) {
    __shared__ f32x4_t group_o[16][64];
    __shared__ float2 group_ml[16];
    const QuantAttnArgs& a = da.a;
    const QuantPages& p = a.p;
    const int tid = threadIdx.x, D = p.dim;
    uint32_t at = blockIdx.x;
    const int rows = a.group * p.tokens;
    const int row = at % rows;
    at /= rows;
    const int kh = at % p.heads;
    const int b = at / p.heads;
    const int ct = row / COLS, col = row % COLS;
    const int t_lo = divide(COLS * ct, a.group, a.group_magic), t_hi = divide(min(rows - 1, COLS * ct + COLS - 1), a.group, a.group_magic);
    const int64_t pos = load_index(p.pos, p.pos_dt, b);
    const TileKeys tk = tile_keys(da, quant_keys(a, pos), pos < 0 ? 0 : quant_count(p, b), t_lo, t_hi);
    if (tk.active == 1) return;
    const int64_t unit = (static_cast<int64_t>(ct) * p.batch + b) * p.heads + kh;
    const float* ml = da.part_ml + (unit * da.splits * COLS + col) * 2;
    const float* po = da.part_o + (unit * da.splits * COLS + col) * D;
    const int pieces = D / 4, at_once = 256 / pieces, groups = (tk.active + 15) / 16;
    const int piece = tid % pieces, grp = tid / pieces;
    for (int g = grp; g < groups && grp < at_once; g += at_once) {
        const Joined j = join_parts(min(16, tk.active - 16 * g),
                                    [&](int s) { return *reinterpret_cast<const float2*>(ml + (16 * g + s) * 2 * COLS); },
                                    [&](int s) { return *reinterpret_cast<const f32x4_t*>(po + (16 * g + s) * COLS * D + 4 * piece); });
        if (groups == 1) {
            store_joined<T>(a, j, row, 4 * piece, kh, b);
            return;
        }
        group_o[g][piece] = j.o;
        if (piece == 0) group_ml[g] = make_float2(j.m, mark_loud(j.total, j.loud));
    }
    if (groups == 1) return;
    __syncthreads();
    if (tid < pieces)
        store_joined<T>(a, join_parts(groups, [&](int s) { return group_ml[s]; }, [&](int s) { return group_o[s][piece]; }), row,
                        4 * piece, kh, b);
}

// Splits of a column tile's keys: a workgroup a CU, rounded down -- one more to a CU
// halves nothing and is joined as well (D 128, 188 column tiles of 2000 keys 24.0 us in
// one piece, 26.2 in two, 29.1 in three; D 256, 80 of them 20.9 in 3, 24.6 in 4).  Where
// that leaves a tile more than long_pairs pairs, up to four a CU, so that the longest
// sequences end with the others: 300 tiles of 500 to 6000 keys, D 64 43.5 -> 39.0 us,
// D 128 75 -> 67, D 256 130 -> 115; of 8000 keys each 72 -> 67, 143 -> 125, 270 -> 228.
// long_pairs 64 (2048 keys), at D 64, whose tiles need least of a CU, 32: 32 sequences
// of 512 to 4096 keys 16.3 -> 14.9 (D 128 at 32: 150 tiles of 2000 keys 19.4 -> 24.2).
// None has less than kMinPairs pairs at the longest context the call can have.
inline void set_splits(SplitArgs* d, int64_t units, int64_t dim, int64_t cap, int64_t window, int64_t tokens) {
    const int64_t keys = window > 0 && window < cap ? std::min(cap, window + tokens + 16) : cap;
    // (and the threads of a launch stay below 2^32, however many are asked for)
    const int64_t most = std::clamp<int64_t>((keys + 31) / 32 / kMinPairs, 1, std::clamp<int64_t>((UINT32_MAX / 256) / units, 1, 256));
    const int forced = env_int("SANDY_QUANT_SPLITS", 0);
    auto of = [&](int64_t workgroups) {
        return static_cast<int>(std::clamp<int64_t>(forced > 0 ? forced : workgroups / units, 1, most));
    };
    d->long_pairs = dim > 64 ? 64 : 32;
    d->few = of(256);
    d->splits = keys > 32 * d->long_pairs * d->few ? of(1024) : d->few;
}

// Where the parts and counters of a split call are; the splits' launch.
template <int COLS>
int split_memory(SplitArgs* d, void* workspace, hipStream_t stream, Err e) {
    const QuantPages& p = d->a.p;
    const int64_t units = static_cast<int64_t>(p.batch) * p.heads * d->col_tiles;
    d->part_o = static_cast<float*>(workspace);
    d->part_ml = d->part_o + units * d->splits * COLS * p.dim;
    if (d->splits == 1 || env_int("SANDY_QUANT_MERGE_KERNEL", 0) != 0) return SANDY_OK;
    int status = 0;
    d->arrived = arrival_counters(static_cast<size_t>(units) * counters_of(d->splits) * kCounterWords, stream, e, &status);
    return status;
}

template <typename T, int COLS>
int launch_split(const void* kernel, SplitArgs d, size_t lds, hipStream_t stream, Err e) {
    const QuantPages& p = d.a.p;
    const int64_t wgs = static_cast<int64_t>(p.batch) * p.heads * d.col_tiles * d.splits;
    void* params[] = {&d};
    SANDY_HIP_TRY(hipLaunchKernel(kernel, dim3(static_cast<unsigned>(wgs)), dim3(256), params, lds, stream), e,
                  "quant_paged attention launch");
    if (d.splits > 1 && !d.arrived) {
        const int64_t rows = static_cast<int64_t>(p.batch) * d.a.hq * p.tokens;
        hipLaunchKernelGGL((quant_merge_kernel<T, COLS>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream, d);
        SANDY_HIP_TRY(hipGetLastError(), e, "quant_paged attention launch");
    }
    return ok(e);
}

} // namespace sandy_hip
