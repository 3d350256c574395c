// sample.hip -- one token a row drawn from its logits, on the device.  The reference samples on the host from logits it
// copies back (src/server/Sampler.cpp:69-79, 212).
//
//   w_i = exp((l_i - max) / T);  tokens ranked by logit, lowest id first among equals
//   K: the first top_k;  P: those of K before which less than top_p of K's weight lies;  M: those with w >= min_p
//   t = u * sum of the weights of P and M's common tokens;  the token where their running sum, in order of ids, passes t
//
// Weights are whole numbers: w_i rounded to 2^-s with s = 62 - log2(vocab) (44 bits of a 262144-token vocabulary).
// Sums of them are exact in any order, so that atomics, parts and workgroups leave no trace in the result, and so are
// comparisons of them (top_p's and the draw's, whose factors have 24 bits), in 128 bits.  min_p looks at w_i itself, in f64.
//
// Ranks are never formed.  Logits fall into 1023 bins of equal width from the maximum down to where weights
// vanish; counts and weights of the bins say in which the cuts of top_k, top_p and min_p lie, and only the tokens there
// (a list, or where it is too long all of them again) are narrowed down, 1024 steps of (logit, id) at a time, the
// last 64 by comparing each with each.  A small top_k needs counts alone: all it may keep is listed, and top_p looks at
// the list.
//
// Up to 8192 tokens a workgroup does a row in one launch, reading it up to four times, mostly from L2.  Longer rows are
// cut into parts, so that few rows fill the chip, and take five launches: peak, bins, cut, gather, draw.
#include "common.h"
#include "sample_parts.h"

#include <algorithm>
#include <type_traits>

namespace sandy_hip {
namespace {

constexpr int kChunk = 2048;      // a part is a whole number of these
constexpr int kParts = 64;        // at most, a row
constexpr int kBins = 1024;       // the last for tokens without weight
constexpr int kList = 8192;       // listed tokens of a row in parts
constexpr int kRowList = 2048;    // and of a row that one workgroup does
constexpr int kPartList = 1024;   // and of a part's
constexpr int kRowVocab = 8192;   // the longest such row
constexpr int kSmall = 1024;      // a top_k whose tokens are all listed
constexpr int kMaxVocab = 1 << 24;
// The cut, draw and whole-row kernels: 256 registers a thread, which 1024 threads would not have.  A thread has two bins.
constexpr int kThreads = 512, kWaves = kThreads / 64, kPer = kBins / kThreads;

struct Peak {
    float max, min;  // of the logits above -inf
    int32_t arg;     // lowest id of max; INT32_MAX: no token
    int32_t pad;
};

// A row's parameters and settings.
struct Row {
    double rate;        // log2(e) / temperature
    float max, half, scale;  // a logit's bin: (max / 2 - logit / 2) * scale, since max - logit may be beyond f32
    float top_p, least; // least: min_p
    float uniform;
    int32_t arg, bits;
    uint32_t top_k;     // 0: off
    bool greedy, bad;

    __device__ bool by_p() const { return top_p < 1.0f; }
    __device__ bool cuts() const { return top_k || by_p(); }
    __device__ bool small() const { return top_k > 0 && top_k <= kSmall; }  // top_k's tokens are all listed
};

// Where a row's cuts lie.  Bins below `sure` are kept; tokens of bins first .. last, m_first .. m_last and k_bin,
// as far as `limit`, are listed and kept up to the place that narrowing finds, if they are likely enough.
struct Cut {
    int32_t sure, first, last, m_first, m_last, k_bin, limit;
    uint32_t rank;      // how many of k_bin's tokens (a small top_k: of the listed ones) are in top_k; 0: all
    uint64_t weight;    // of top_k's tokens in bins below k_bin (k_bin < 0: of all of them)

    __device__ bool in_question(int bin) const {
        return (bin <= limit) & ((bin == k_bin) | ((bin >= first) & (bin <= last)) | ((bin >= m_first) & (bin <= m_last)));
    }
    __device__ bool listed_in(int bin, int b0, int b1) const { return (bin >= b0) & (bin <= b1) & in_question(bin); }
    // the logits between which all listed ones lie
    __device__ void logits(const Row& r, float* low, float* high) const;
    // whether a token of this bin and place stays, as far as top_k and top_p go
    __device__ bool keeps(int bin, uint64_t place, uint64_t last_place) const { return (bin < sure) | (in_question(bin) & (place <= last_place)); }
};

__device__ __forceinline__ Cut no_cut() {
    Cut cut{};
    cut.sure = cut.limit = cut.first = cut.m_first = kBins;
    cut.last = cut.m_last = cut.k_bin = -1;
    return cut;
}

struct SampleArgs {
    const void* logits;
    const float *temperature, *top_p, *min_p, *uniforms;
    const void* top_k;
    void* ids;
    float* probs;
    uint32_t* errw;
    int64_t stride;
    int32_t top_k_dt, ids_dt;
    int32_t rows, vocab;
    int32_t bits;         // s
    int32_t parts, per;   // a part is `per` chunks, one workgroup of the peak, bins and gather kernels
    // workspace of rows in parts
    Peak* peaks;          // [rows, parts]
    uint64_t* weights;    // [rows, parts, kBins]
    uint32_t* counts;     // [rows, parts, kBins]
    uint64_t* upto;       // [rows, kBins]: the row's weight up to and with each bin
    Row* settings;        // [rows]
    Cut* cuts;            // [rows]
    uint32_t* listed;     // [rows]
    uint64_t* list;       // [rows, kList]
    uint64_t* kept;       // [rows, parts]: kept weight of bins below the cuts
};

__device__ __forceinline__ bool token(float l) { return l > -__builtin_inff(); }  // not masked, not NaN

// logits as whole numbers whose order is the ranks': higher logits first
__device__ __forceinline__ uint32_t rank_key(float l) {
    const uint32_t u = __float_as_uint(l == 0.0f ? 0.0f : l);
    return u & 0x80000000u ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k : ~k & 0x7fffffffu); }
// (logit, id) in rank order
__device__ __forceinline__ uint64_t place_of(float l, uint32_t id) { return static_cast<uint64_t>(rank_key(l)) << 24 | id; }

// ------------------------------------------------------------------ sums over waves and workgroups
// The value `CTRL` names of another lane of the wave, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_move(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t lane_move(uint64_t v) {
    return static_cast<uint64_t>(lane_move<CTRL, ROWS>(static_cast<uint32_t>(v >> 32))) << 32 | lane_move<CTRL, ROWS>(static_cast<uint32_t>(v));
}
// Inclusive sums over a wave by DPP moves: within rows of 16 lanes, then each row's last lane to the next rows.
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
    v += lane_move<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v += lane_move<0x112, 0xf>(v);
    v += lane_move<0x114, 0xf>(v);
    v += lane_move<0x118, 0xf>(v);
    v += lane_move<0x142, 0xa>(v);  // row_bcast 15 to rows 1 and 3
    v += lane_move<0x143, 0xc>(v);  // row_bcast 31 to rows 2 and 3
    return v;
}
// Inclusive sums over a workgroup of WAVES waves; `waves` holds WAVES values, *total all of them.
template <int WAVES, typename V>
__device__ __forceinline__ V block_scan(V v, V* waves, V* total) {
    const int wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();  // the last use of `waves` is over
    if ((threadIdx.x & 63) == 63) waves[wave] = v;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (w < wave) before += waves[w];
        all += waves[w];
    }
    *total = all;
    return before + v;
}

// Two at once.
template <int WAVES>
__device__ __forceinline__ void block_scan(uint64_t& a, uint32_t& b, uint64_t* waves_a, uint32_t* waves_b, uint64_t* total_a) {
    const int wave = threadIdx.x >> 6;
    a = wave_scan(a);
    b = wave_scan(b);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) waves_a[wave] = a, waves_b[wave] = b;
    __syncthreads();
    uint64_t before_a = 0, all = 0;
    uint32_t before_b = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (w < wave) before_a += waves_a[w], before_b += waves_b[w];
        all += waves_a[w];
    }
    a += before_a;
    b += before_b;
    *total_a = all;
}

// ------------------------------------------------------------------ a row's settings
__device__ __forceinline__ void better_peak(float& mx, int& arg, float& mn, float ox, int oa, float on) {
    if (ox > mx || (ox == mx && oa < arg)) mx = ox, arg = oa;
    mn = fminf(mn, on);
}
__device__ __forceinline__ void wave_peak(float& mx, int& arg, float& mn) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) better_peak(mx, arg, mn, __shfl_xor(mx, m, 64), __shfl_xor(arg, m, 64), __shfl_xor(mn, m, 64));
}

__device__ __forceinline__ Row make_row(const SampleArgs& a, int row, float mx, int arg, float mn) {
    Row r;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const int64_t k = a.top_k ? load_index(a.top_k, a.top_k_dt, row) : 0;
    r.top_p = a.top_p ? a.top_p[row] : 1.0f;
    r.least = a.min_p ? a.min_p[row] : 0.0f;
    r.uniform = a.uniforms[row];
    r.max = mx;
    r.half = 0.5f * mx;
    r.arg = arg;
    r.bits = a.bits;
    r.top_k = k > 0 && k < a.vocab ? static_cast<uint32_t>(k) : 0;
    r.greedy = t == 0.0f;
    r.bad = !(t >= 0.0f) || r.top_p != r.top_p || !(r.least <= 1.0f) || !(r.uniform >= 0.0f && r.uniform < 1.0f);
    r.rate = 1.4426950408889634074 / static_cast<double>(t);
    // bins reach to where weights vanish (2^-bits-1, and a little on), or to the lowest logit where that is nearer
    const double width = fmin(static_cast<double>(mx) - static_cast<double>(mn), (a.bits + 1.5) / r.rate);
    r.scale = width > 0.0 ? static_cast<float>(fmin(2 * (kBins - 2) / width, 3.0e38)) : 0.0f;
    return r;
}

// (ln 2)^n / n!, n = kTerms .. 0
constexpr int kTerms = 12;
__device__ constexpr double kSeries[kTerms + 1] = {
    2.56784359934882055e-11,
    4.44553827187081162e-10, 7.05491162080112336e-09, 1.01780860092396999e-07,
    1.32154867901443095e-06, 1.52527338040598411e-05, 1.54035303933816088e-04,
    1.33335581464284433e-03, 9.61812910762847688e-03, 5.55041086648215831e-02,
    2.40226506959100722e-01, 6.93147180559945286e-01, 1.0};
// Weights of N logits at once, so that their series interleave: exp((l - max) / T) = 2^f 2^k, 1 at the maximum, f in
// -1/2 .. 1/2 by the Taylor series of e^(f ln 2) to the 12th power (the next term is below 2.4e-16 of the sum; an 11th power
// left 8.9e-15, 7 multiples of 2^-50), rounded to a multiple of 2^-bits, 52 bits of which lie behind 2^52: the nearest, or
// with roundings of the sum and its exponent (0.7 multiples of 2^-50 at most) one next to it.  Below 2^-200 it stays there,
// which weighs nothing.
// `all` false: 0 for those that min_p leaves out.  Masked logits weigh 0.
template <int N>
__device__ __forceinline__ void weigh(const Row& r, const float (&l)[N], bool all, uint64_t (&w)[N]) {
    double f[N], p[N];
    int k[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        const double d = l[j] == r.max ? 0.0 : static_cast<double>(l[j]) - static_cast<double>(r.max);
        const double x = fmax(d * r.rate, -200.0), whole = __builtin_rint(x);  // (inf less inf: -200 too)
        f[j] = x - whole;
        k[j] = static_cast<int>(whole);
        p[j] = kSeries[0];
    }
#pragma unroll
    for (int n = 1; n <= kTerms; n++)
#pragma unroll
        for (int j = 0; j < N; j++) p[j] = fma(p[j], f[j], kSeries[n]);
    auto two_to = [](int e) { return __longlong_as_double(static_cast<long long>(1023 + e) << 52); };
#pragma unroll
    for (int j = 0; j < N; j++) {
        w[j] = static_cast<uint64_t>(__double_as_longlong(fma(p[j], two_to(r.bits + k[j]), 4503599627370496.0))) - 0x4330000000000000ull;
        w[j] = token(l[j]) ? w[j] : 0;
    }
    if (__builtin_amdgcn_readfirstlane(!all & (r.least > 0.0f)))  // a row's own, the same for all
#pragma unroll
        for (int j = 0; j < N; j++) w[j] = p[j] * two_to(k[j]) >= static_cast<double>(r.least) ? w[j] : 0;
}
__device__ __forceinline__ uint64_t weight_of(const Row& r, float l, bool all = true) {
    const float v[1] = {l};
    uint64_t w[1];
    weigh(r, v, all, w);
    return w[0];
}
// Non-decreasing as logits fall; the last bin holds no token that weighs anything (those end a ninetieth before it, or
// the lowest logit ends at kBins - 2).
__device__ __forceinline__ int bin_of(const Row& r, float l) {
    const float at = l == r.max ? 0.0f : fmaf(l, -0.5f, r.half) * r.scale;
    const int bin = static_cast<int>(fminf(at, static_cast<float>(kBins - 2)));
    return at >= static_cast<float>(kBins - 1) ? kBins - 1 : bin;
}

// The logits between which all tokens of bins b0 .. b1 lie, a little widened: bins are rounded.
__device__ __forceinline__ void logits_of_bins(const Row& r, int b0, int b1, float* low, float* high) {
    const double most = r.max, wide = 2.0 / r.scale, edge = 1e-6 * fabs(most);
    const bool all = !(fabs(most) < 3.0e38) || r.scale == 0.0f;
    *high = b0 <= 0 || all ? r.max : static_cast<float>(most - b0 * wide * (1 - 1e-6) + edge);
    *low = b1 >= kBins - 2 || all ? -__builtin_inff() : static_cast<float>(most - (b1 + 1) * wide * (1 + 1e-6) - edge);
}

__device__ __forceinline__ void Cut::logits(const Row& r, float* low, float* high) const {
    int b0 = kBins, b1 = -1;
    if (k_bin >= 0) b0 = b1 = k_bin;
    if (first <= last) b0 = min(b0, first), b1 = max(b1, last);
    if (m_first <= m_last) b0 = min(b0, m_first), b1 = max(b1, m_last);
    logits_of_bins(r, b0, min(b1, limit), low, high);
}

// top_p's part of a weight, at least; 0 where it is that of the first token alone
__device__ __forceinline__ uint64_t nucleus(const Row& r, uint64_t weight) { return r.top_p > 0.0f ? part_of(r.top_p, weight, true) : 0; }

// Eight tokens from id `first` on of a row, what lies past the vocabulary as masked.
template <typename T>
__device__ __forceinline__ void load_tokens(const SampleArgs& a, int64_t at, int first, float (&v)[8]) {
    if (first + 8 <= a.vocab) {
        load8_unaligned<T>(a.logits, at + first, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = first + j < a.vocab ? Vec8<T>::load1(a.logits, at + first + j) : -__builtin_inff();
}

// f(logits, first id) for a thread's eights of a part's chunks, N loads at a time without a guard where they are whole, the
// next requested meanwhile.
template <typename T, int N, typename F>
__device__ __forceinline__ void part_tokens(const SampleArgs& a, int64_t at, int begin, int end, F f) {
    const int mine = static_cast<int>(threadIdx.x) * 8;
    float next[N][8];
    auto request = [&](int first) {
#pragma unroll
        for (int n = 0; n < N; n++) load8_unaligned<T>(a.logits, at + first + n * kChunk + mine, next[n]);
    };
    if (begin + N * kChunk <= end) request(begin);
    for (; begin + N * kChunk <= end; begin += N * kChunk) {
        float v[N][8];
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int j = 0; j < 8; j++) v[n][j] = next[n][j];
        request(min(begin + N * kChunk, end - N * kChunk));  // (past the last whole ones: tokens of before, not used)
#pragma unroll
        for (int n = 0; n < N; n++) f(v[n], begin + n * kChunk + mine);
    }
#pragma unroll 1
    for (; begin < end; begin += kChunk) {
        float v[8];
        load_tokens<T>(a, at, begin + mine, v);
        f(v, begin + mine);
    }
}

__device__ __forceinline__ void store_token(const SampleArgs& a, int row, int64_t id, float prob) {
    store_index(a.ids, a.ids_dt, row, id);
    if (a.probs) a.probs[row] = prob;
}
// Rows that need no draw: bad settings (recorded), no token, or greedy.
__device__ __forceinline__ bool drawn(const SampleArgs& a, const Row& r, int row) {
    const bool none = r.bad || r.arg == INT32_MAX;
    if (!none && !r.greedy) return false;
    if (threadIdx.x == 0) {
        if (r.bad) atomicOr(a.errw, static_cast<uint32_t>(SANDY_DEVERR_SAMPLE));
        store_token(a, row, none ? -1 : r.arg, none ? 0.0f : 1.0f);
    }
    return true;
}

// ------------------------------------------------------------------ where the cuts lie
struct CutShared {
    uint64_t waves64[kWaves], low, high;
    uint32_t waves32[kWaves], rank;
    int k_bin, k_last, p_first, p_last;
};

// Cuts of a row from its bins' counts and weights, bins kPer threadIdx .. of a thread; up_to: the weight up to and with each.
__device__ __forceinline__ Cut find_cuts(const Row& r, const uint32_t (&c)[kPer], const uint64_t (&w)[kPer], CutShared& sh, uint64_t (&up_to)[kPer]) {
    uint64_t all = 0, mine = 0;
    uint32_t tokens = 0, c_to[kPer], mine_c = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) up_to[i] = mine += w[i], c_to[i] = mine_c += c[i];
    if (!r.small()) {
        const uint64_t before = block_scan<kWaves>(mine, sh.waves64, &all) - mine;
#pragma unroll
        for (int i = 0; i < kPer; i++) up_to[i] += before;
    }
    if (r.top_k) {
        const uint32_t before = block_scan<kWaves>(mine_c, sh.waves32, &tokens) - mine_c;
#pragma unroll
        for (int i = 0; i < kPer; i++) c_to[i] += before;
    }
    if (threadIdx.x == 0) sh.k_bin = -1, sh.k_last = sh.p_first = sh.p_last = kBins, sh.low = sh.high = all, sh.rank = 0;
    __syncthreads();
    const uint32_t k = r.top_k;
    // the bin where top_k ends, if it ends inside one whose tokens weigh anything
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const int bin = kPer * threadIdx.x + i;
        if (!(k && k < tokens && c_to[i] >= k && c_to[i] - c[i] < k)) continue;
        sh.k_last = bin;
        if (c_to[i] == k || bin == kBins - 1) {
            sh.low = sh.high = up_to[i];
        } else {
            sh.k_bin = bin;
            sh.low = up_to[i] - w[i];
            sh.high = up_to[i];
            sh.rank = k - (c_to[i] - c[i]);
        }
    }
    __syncthreads();
    Cut cut = no_cut();
    cut.sure = 0;
    cut.limit = sh.k_last;
    if (r.small()) {
        // all that top_k may keep: to its last bin, or every token that weighs anything
        cut.first = 0;
        cut.last = min(sh.k_last, kBins - 2);
        cut.rank = k < tokens && sh.k_last < kBins - 1 ? k : 0;
        return cut;
    }
    cut.weight = sh.low;
    if (r.by_p()) {
        // top_p's cut lies where the sums reach its part of top_k's weight, which is between low and high
        const uint64_t from = nucleus(r, sh.low), to = nucleus(r, sh.high);
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int bin = kPer * threadIdx.x + i;
            const uint64_t before = up_to[i] - w[i];
            if (up_to[i] >= from && (bin == 0 || before < from)) sh.p_first = bin;
            if (up_to[i] >= to && (bin == 0 || before < to)) sh.p_last = bin;
        }
    }
    __syncthreads();
    const int k_bin = sh.k_bin;
    cut.sure = k_bin >= 0 ? k_bin : sh.k_last < kBins ? sh.k_last + 1 : kBins;
    int p_first = kBins;
    if (r.by_p()) cut.sure = min(cut.sure, p_first = sh.p_first);
    if (r.least > 0.0f) {
        // min_p's cut is at a logit: within a bin of where that falls
        const double at = -log2(static_cast<double>(r.least)) / r.rate * (0.5 * static_cast<double>(r.scale));
        if (at < kBins) {
            cut.m_first = max(static_cast<int>(at) - 1, 0);
            cut.m_last = static_cast<int>(at) + 1;
            cut.sure = min(cut.sure, cut.m_first);
            if (cut.m_last < p_first && cut.m_last < (k_bin >= 0 ? k_bin : kBins)) return cut;  // nothing else cuts
        }
    }
    if (r.by_p()) {
        cut.first = p_first;
        cut.last = sh.p_last;
    }
    if (k_bin >= 0) {
        cut.k_bin = k_bin;
        cut.rank = sh.rank;
    }
    return cut;
}

// ------------------------------------------------------------------ narrowing down
struct NarrowShared {
    uint64_t bin_weights[kBins], waves64[kWaves], places[64], weights[64];
    uint64_t lo, hi, weight_before;
    uint32_t bin_counts[kBins], waves32[kWaves], count_before, n;
};

// Of the tokens that each(f) names as f(place, weight), at most `most` and from `low` to `high`, in rank order: the place of
// the one with which they become `rank`, or (rank 0) with which their weights reach `weight`, the first token reaching 0;
// no less than the last of all if they never do.  sh.weight_before is then the sum up to and with it.
template <typename Each>
__device__ __forceinline__ uint64_t narrow(NarrowShared& sh, uint32_t rank, uint64_t weight, uint32_t most, uint64_t low, uint64_t high, Each each) {
    const int tid = threadIdx.x;
    if (tid == 0) sh.lo = low, sh.hi = high, sh.weight_before = 0, sh.count_before = 0, sh.n = most;
    __syncthreads();
    while (sh.n > 64) {  // a step of 1024 of the last one
        const uint64_t from = sh.lo, to = sh.hi;
        const int shift = max(0, 54 - __builtin_clzll((to - from) | 1));
#pragma unroll
        for (int i = 0; i < kPer; i++) sh.bin_weights[kPer * tid + i] = 0, sh.bin_counts[kPer * tid + i] = 0;
        __syncthreads();
        each([&](uint64_t place, uint64_t w) {
            if (place < from || place > to) return;
            const int q = static_cast<int>((place - from) >> shift);
            atomicAdd(&sh.bin_counts[q], 1u);
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bin_weights[q]), static_cast<unsigned long long>(w));
        });
        __syncthreads();
        uint64_t w[kPer], w_to[kPer], mine = 0, all;
        uint32_t c[kPer], c_to[kPer], mine_c = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            w_to[i] = mine += w[i] = sh.bin_weights[kPer * tid + i];
            c_to[i] = mine_c += c[i] = sh.bin_counts[kPer * tid + i];
        }
        uint64_t w_before = mine;
        uint32_t c_before = mine_c;
        block_scan<kWaves>(w_before, c_before, sh.waves64, sh.waves32, &all);
        w_before += sh.weight_before - mine;
        c_before += sh.count_before - mine_c;
        int here = -1;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            w_to[i] += w_before;
            c_to[i] += c_before;
            if (c[i] != 0 && (rank ? c_to[i] >= rank && c_to[i] - c[i] < rank : w_to[i] >= weight && (w_to[i] - w[i] < weight || c_to[i] == c[i]))) here = i;
        }
        if (!__syncthreads_or(here >= 0)) {
            if (tid == 0) sh.weight_before += all;
            __syncthreads();
            return to;
        }
#pragma unroll
        for (int i = 0; i < kPer; i++)
            if (here == i) {
                const uint64_t step = kPer * tid + i;
                sh.lo = from + (step << shift);
                sh.hi = min(to, from + ((step + 1) << shift) - 1);
                sh.weight_before = w_to[i] - w[i];
                sh.count_before = c_to[i] - c[i];
                sh.n = c[i];
            }
        __syncthreads();
    }
    // the last few: each with each
    const uint64_t from = sh.lo, to = sh.hi;
    __syncthreads();
    if (tid == 0) sh.n = 0;
    __syncthreads();
    each([&](uint64_t place, uint64_t w) {
        if (place < from || place > to) return;
        const uint32_t i = atomicAdd(&sh.n, 1u);
        sh.places[i] = place;
        sh.weights[i] = w;
    });
    __syncthreads();
    const uint32_t few = sh.n;
    if (tid < 64) {
        const bool in = tid < few;
        if (!in) sh.places[tid] = ~uint64_t{0}, sh.weights[tid] = 0;
        const uint64_t place = sh.places[tid], w = sh.weights[tid];
        uint64_t w_to = sh.weight_before + w, all = sh.weight_before;
        uint32_t c_to = sh.count_before + 1;
        __builtin_amdgcn_wave_barrier();
#pragma unroll 8
        for (uint32_t i = 0; i < (few + 7 & ~7u); i++) {
            const uint64_t other = sh.weights[i];
            const bool before = sh.places[i] < place;
            w_to += before ? other : 0;
            c_to += before ? 1 : 0;
            all += other;
        }
        const bool here = in && (rank ? c_to == rank : w_to >= weight && (w_to - w < weight || c_to == 1));
        const uint64_t found = __ballot(here);
        if (here) sh.lo = place, sh.weight_before = w_to;
        if (!found && tid == 0) sh.lo = to, sh.weight_before = all;
    }
    __syncthreads();
    return sh.lo;
}

// The last place that top_k and top_p keep: ~0 where no listed token is cut by them.  each(b0, b1, f) names the listed
// tokens of bins b0 .. b1, `most` of all; up_to(bin): the row's weight up to and with a bin.
template <typename Each, typename UpTo>
__device__ __forceinline__ uint64_t last_place(const Row& r, const Cut& cut, NarrowShared& sh, uint32_t most, Each each, UpTo up_to) {
    uint64_t last = ~uint64_t{0}, kept = cut.weight;  // top_k's
    const bool small = r.small();
#pragma unroll 1
    for (int step = 0; step < 2; step++) {
        // first where top_k ends (a small one with room for all: their weight), then where top_p does
        int b0 = 0, b1 = kBins;
        uint32_t rank = 0;
        uint64_t weight = 0;
        if (step == 0) {
            if (small ? !cut.rank && !r.by_p() : cut.k_bin < 0) continue;
            rank = cut.rank ? cut.rank : UINT32_MAX;
            if (!small) b0 = b1 = cut.k_bin;
        } else {
            if (small ? !r.by_p() : cut.last < 0) continue;
            weight = nucleus(r, kept);
            if (!small) {
                int bin = cut.first;
                while (bin < cut.last && up_to(bin) < weight) bin++;
                const uint64_t before = bin > 0 ? up_to(bin - 1) : 0;
                weight = weight > before ? weight - before : 0;
                b0 = b1 = bin;
            }
        }
        float low, high;
        logits_of_bins(r, b0, min(b1, cut.limit), &low, &high);
        const uint64_t place = narrow(sh, rank, weight, most, place_of(high, 0), place_of(low, 0xffffff), [&](auto f) { each(b0, b1, f); });
        last = min(last, place);
        if (step == 0) kept += sh.weight_before;
        __syncthreads();
    }
    return last;
}

// The tokens in question of bins b0 .. b1, from the row itself: for lists that are too long.
template <typename T, typename F>
__device__ __forceinline__ void each_of_row(const SampleArgs& a, int64_t at, const Row& r, const Cut& cut, int b0, int b1, F f) {
#pragma unroll 1
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
        const float l = Vec8<T>::load1(a.logits, at + i);
        if (token(l) && cut.listed_in(bin_of(r, l), b0, b1)) f(place_of(l, i), weight_of(r, l));
    }
}

// ------------------------------------------------------------------ a row a workgroup
constexpr int kBlock = 8 * kThreads;  // tokens a workgroup takes at a time

struct RowShared {
    uint64_t weights[kBins], up_to[kBins];
    uint32_t counts[kBins];
    uint64_t places[kRowList], held[kRowList];
    NarrowShared narrow;
    uint64_t sums[kRowVocab / kBlock * kWaves];  // of each wave's tokens of each block
    Peak peaks[kWaves];
    CutShared cuts;
    Row row;
    Cut cut;
    uint32_t listed;
};

// f(logits, first id) for this thread's eight tokens of each block of a row, the next eight requested meanwhile.
template <typename T, typename F>
__device__ __forceinline__ void row_tokens(const SampleArgs& a, int64_t at, F f) {
    float next[8];
    load_tokens<T>(a, at, static_cast<int>(threadIdx.x) * 8, next);
#pragma unroll 1
    for (int first = threadIdx.x * 8; first - static_cast<int>(threadIdx.x) * 8 < a.vocab; first += kBlock) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = next[j];
        load_tokens<T>(a, at, first + kBlock, next);
        f(v, first);
    }
}

// Bound by one CU's vector instructions (40 a token to weigh it, half of them in 64 bits) and the meetings of its waves: 512
// rows of 8000 bf16 tokens in two rounds 24 us by temperature alone, 41 with top-k 50, 43 with top-p 0.9.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ RowShared sh;
    const int tid = threadIdx.x, row = blockIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t at = row * a.stride;
    float mx = -__builtin_inff(), mn = __builtin_inff();
    int arg = INT32_MAX;
#pragma unroll
    for (int i = 0; i < kPer; i++) sh.weights[kPer * tid + i] = 0, sh.counts[kPer * tid + i] = 0;
    if (tid == 0) sh.listed = 0;
    row_tokens<T>(a, at, [&](const float (&v)[8], int first) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (token(v[j])) better_peak(mx, arg, mn, v[j], first + j, v[j]);
    });
    wave_peak(mx, arg, mn);
    if (lane == 0) sh.peaks[wave] = Peak{mx, mn, arg, 0};
    __syncthreads();
    if (wave == 0) {
        const Peak p = sh.peaks[lane & (kWaves - 1)];
        mx = p.max, arg = p.arg, mn = p.min;
        wave_peak(mx, arg, mn);
        if (lane == 0) sh.row = make_row(a, row, mx, arg, mn);
    }
    __syncthreads();
    const Row& r = sh.row;
    if (drawn(a, r, row)) return;
    const Cut& cut = sh.cut;
    if (tid == 0) sh.cut = no_cut();
    __syncthreads();
    uint64_t last = ~uint64_t{0};
    if (r.cuts()) {
        const bool count = r.top_k != 0, weighed = !r.small();
        row_tokens<T>(a, at, [&](const float (&v)[8], int) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (count && token(v[j])) atomicAdd(&sh.counts[bin_of(r, v[j])], 1u);
            if (!weighed) return;
            uint64_t w[8];
            weigh(r, v, true, w);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (w[j]) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.weights[bin_of(r, v[j])]), static_cast<unsigned long long>(w[j]));
        });
        __syncthreads();
        uint64_t w[kPer], up_to[kPer];
        uint32_t c[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) w[i] = sh.weights[kPer * tid + i], c[i] = sh.counts[kPer * tid + i];
        const Cut found = find_cuts(r, c, w, sh.cuts, up_to);
        if (tid == 0) sh.cut = found;
#pragma unroll
        for (int i = 0; i < kPer; i++) sh.up_to[kPer * tid + i] = up_to[i];
        __syncthreads();
        row_tokens<T>(a, at, [&](const float (&v)[8], int first) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (!token(v[j]) || !cut.in_question(bin_of(r, v[j]))) continue;
                const uint32_t i = atomicAdd(&sh.listed, 1u);
                if (i < kRowList) sh.places[i] = place_of(v[j], first + j);
            }
        });
        __syncthreads();
        const uint32_t listed = sh.listed;
        if (listed <= kRowList)
            for (uint32_t i = tid; i < listed; i += kThreads) sh.held[i] = weight_of(r, key_logit(static_cast<uint32_t>(sh.places[i] >> 24)));
        __syncthreads();
        auto each = [&](int b0, int b1, auto f) {
            if (listed <= kRowList) {
                for (uint32_t i = tid; i < listed; i += kThreads) {
                    const int b = bin_of(r, key_logit(static_cast<uint32_t>(sh.places[i] >> 24)));
                    if (b >= b0 && b <= b1) f(sh.places[i], sh.held[i]);
                }
                return;
            }
            each_of_row<T>(a, at, r, cut, b0, b1, f);
        };
        last = last_place(r, cut, sh.narrow, listed, each, [&](int bin) { return sh.up_to[bin]; });
    }
    // kept weights of eight tokens, and their sums over each wave's part of a block
    auto kept = [&](const float (&v)[8], int first, uint64_t (&w)[8]) {
        bool keep[8], any = false;
#pragma unroll
        for (int j = 0; j < 8; j++) any |= keep[j] = cut.keeps(bin_of(r, v[j]), place_of(v[j], first + j), last);  // (masked ones weigh 0)
        if (__any(any)) {
            weigh(r, v, false, w);
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = keep[j] ? w[j] : 0;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = 0;
        }
        return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    };
    row_tokens<T>(a, at, [&](const float (&v)[8], int first) {
        uint64_t w[8];
        const uint64_t sum = wave_scan(kept(v, first, w));
        if (lane == 63) sh.sums[first / kBlock * kWaves + wave] = sum;
    });
    __syncthreads();
    // the block and wave in which the sum of all passes the target: each wave looks, that one goes on
    constexpr int kSums = kRowVocab / kBlock * kWaves;
    static_assert(kSums <= 64);
    const uint64_t part_w = lane < (a.vocab + kBlock - 1) / kBlock * kWaves ? sh.sums[lane & (kSums - 1)] : 0, to = wave_scan(part_w);
    const uint64_t total = __shfl(to, 63, 64), target = part_of(r.uniform, total, false);
    const uint64_t past = __ballot(to > target);
    if (past == 0) {  // the total is above the target, unless logits change meanwhile: no place to go on from
        if (tid == 0) store_token(a, row, -1, 0.0f);
        return;
    }
    const int part = __builtin_ctzll(past);
    if (part % kWaves != wave) return;
    const uint64_t before = __shfl(to - part_w, part, 64);
    float v[8];
    uint64_t w[8];
    const int first = part / kWaves * kBlock + tid * 8;
    load_tokens<T>(a, at, first, v);
    const uint64_t mine = kept(v, first, w);
    uint64_t upto = before + wave_scan(mine) - mine;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (upto <= target && upto + w[j] > target)
            store_token(a, row, first + j, static_cast<float>(static_cast<double>(w[j]) / static_cast<double>(total)));
        upto += w[j];
    }
}

// ------------------------------------------------------------------ rows in parts
// Times of each: 64 rows of 262144 bf16 logits, 33.5 MB, with top-p 0.9.

// A stream from HBM: 9 to 14 us, 11 on average, 3.1 TB/s.  A thread keeps the eight with its maximum and looks them up again for the id.
template <typename T>
__global__ __launch_bounds__(256) void sample_peak_kernel(SampleArgs a) {
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const int64_t at = row * a.stride;
    const int begin = part * a.per * kChunk, end = min(begin + a.per * kChunk, a.vocab);
    float mx = -__builtin_inff(), mn = __builtin_inff();
    int eight = -1, arg = INT32_MAX;  // the first eight that hold the maximum, looked at again for its id
    part_tokens<T, 4>(a, at, begin, end, [&](const float (&v)[8], int i) {
        float top = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const bool in = token(v[j]);  // (a signalling NaN may win fmaxf, and with it hide what came before)
            top = fmaxf(top, in ? v[j] : -__builtin_inff());
            mn = fminf(mn, in ? v[j] : __builtin_inff());
        }
        eight = top > mx ? i : eight;
        mx = fmaxf(mx, top);
    });
    if (eight >= 0) {
        float v[8];
        load_tokens<T>(a, at, eight, v);
#pragma unroll
        for (int j = 7; j >= 0; j--) arg = v[j] == mx ? eight + j : arg;
    }
    wave_peak(mx, arg, mn);
    __shared__ Peak waves[4];
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = Peak{mx, mn, arg, 0};
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < 4; w++) better_peak(mx, arg, mn, waves[w].max, waves[w].arg, waves[w].min);
        a.peaks[blockIdx.x] = Peak{mx, mn, arg, 0};
    }
}

// Settings from the parts' peaks; every thread of the workgroup gets them.
__device__ __forceinline__ Row row_of(const SampleArgs& a, int row, Row* shared) {
    if (threadIdx.x < 64) {
        float mx = -__builtin_inff(), mn = __builtin_inff();
        int arg = INT32_MAX;
        if (static_cast<int>(threadIdx.x) < a.parts) {
            const Peak p = a.peaks[static_cast<int64_t>(row) * a.parts + threadIdx.x];
            mx = p.max, arg = p.arg, mn = p.min;
        }
        wave_peak(mx, arg, mn);
        if (threadIdx.x == 0) *shared = make_row(a, row, mx, arg, mn);
    }
    __syncthreads();
    return *shared;
}

// Counts where top_k asks for them, weights unless all of top_k's tokens are listed; the part's weight of rows that
// nothing cuts but min_p.  26 us, 17 of them issuing the 40 instructions a token of its weight and bin.
template <typename T>
__global__ __launch_bounds__(256) void sample_bins_kernel(SampleArgs a) {
    __shared__ uint64_t weights[kBins], waves[4];
    __shared__ uint32_t counts[kBins];
    __shared__ Row shared;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    for (int i = threadIdx.x; i < kBins; i += 256) weights[i] = 0, counts[i] = 0;
    const Row r = row_of(a, row, &shared);
    if (part == 0 && threadIdx.x == 0) a.settings[row] = r;
    if (r.greedy || r.bad) return;
    const int64_t at = row * a.stride;
    const int begin = part * a.per * kChunk, end = min(begin + a.per * kChunk, a.vocab);
    const bool cuts = r.cuts(), count = r.top_k != 0, weighed = !r.small();
    uint64_t sum = 0;
    part_tokens<T, 1>(a, at, begin, end, [&](const float (&v)[8], int) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (count && token(v[j])) atomicAdd(&counts[bin_of(r, v[j])], 1u);
        if (!weighed) return;
        uint64_t w[8];
        weigh(r, v, cuts, w);
        if (!cuts) {
            sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (w[j]) atomicAdd(reinterpret_cast<unsigned long long*>(&weights[bin_of(r, v[j])]), static_cast<unsigned long long>(w[j]));
    });
    if (!cuts) {
        uint64_t total;
        block_scan<4>(sum, waves, &total);
        if (threadIdx.x == 0) a.kept[blockIdx.x] = total;
        return;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += 256) {
        if (!r.small()) a.weights[static_cast<int64_t>(blockIdx.x) * kBins + i] = weights[i];
        if (r.top_k) a.counts[static_cast<int64_t>(blockIdx.x) * kBins + i] = counts[i];
    }
}

// Sums of the parts' bins, and the cuts: 5 us, a chain of dependent loads, scans and meetings.
__global__ __launch_bounds__(kThreads) void sample_cut_kernel(SampleArgs a) {
    __shared__ CutShared sh;
    const int row = blockIdx.x, bin = kPer * threadIdx.x;
    const Row r = a.settings[row];
    Cut cut = no_cut();
    if (!drawn(a, r, row) && r.cuts()) {
        uint64_t w[kPer] = {}, up_to[kPer];
        uint32_t c[kPer] = {};
        const int64_t first = static_cast<int64_t>(row) * a.parts * kBins + bin;
        if (!r.small())
#pragma unroll 8
            for (int p = 0; p < a.parts; p++)
#pragma unroll
                for (int i = 0; i < kPer; i++) w[i] += a.weights[first + p * kBins + i];
        if (r.top_k)
#pragma unroll 8
            for (int p = 0; p < a.parts; p++)
#pragma unroll
                for (int i = 0; i < kPer; i++) c[i] += a.counts[first + p * kBins + i];
        cut = find_cuts(r, c, w, sh, up_to);
#pragma unroll
        for (int i = 0; i < kPer; i++) a.upto[static_cast<int64_t>(row) * kBins + bin + i] = up_to[i];
    }
    if (bin == 0) {
        a.cuts[row] = cut;
        a.listed[row] = 0;
    }
}

// Lists the tokens in question, and sums up what a part keeps for sure from its bins.  A part lists its tokens in LDS,
// takes as many places of the row's list at once and copies them there; what LDS has no room for goes there by itself.
// 15 us, 2.3 TB/s: settings, bins and tokens one after the other, then a place of the list.
template <typename T>
__global__ __launch_bounds__(256) void sample_gather_kernel(SampleArgs a) {
    __shared__ uint64_t waves[4], places[kPartList];
    __shared__ uint32_t found, to;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const Row r = a.settings[row];
    if (r.greedy || r.bad || !r.cuts()) return;
    const Cut cut = a.cuts[row];
    const int64_t at = row * a.stride;
    uint64_t* const list = a.list + static_cast<int64_t>(row) * kList;
    uint64_t sum = 0, total;
    for (int i = threadIdx.x; i < min(cut.sure, kBins); i += 256) sum += a.weights[static_cast<int64_t>(blockIdx.x) * kBins + i];
    if (threadIdx.x == 0) found = 0;
    float low, high;
    cut.logits(r, &low, &high);
    block_scan<4>(sum, waves, &total);
    part_tokens<T, 4>(a, at, part * a.per * kChunk, min((part + 1) * a.per * kChunk, a.vocab), [&](const float (&v)[8], int first) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (v[j] >= low && v[j] <= high && token(v[j]) && cut.in_question(bin_of(r, v[j]))) {
                const uint64_t place = place_of(v[j], first + j);
                const uint32_t i = atomicAdd(&found, 1u);
                if (i < kPartList) {
                    places[i] = place;
                } else {
                    const uint32_t next = atomicAdd(&a.listed[row], 1u);
                    if (next < kList) list[next] = place;
                }
            }
    });
    __syncthreads();
    const uint32_t held = min(found, static_cast<uint32_t>(kPartList));
    if (threadIdx.x == 0) {
        a.kept[blockIdx.x] = total;
        to = held ? atomicAdd(&a.listed[row], held) : 0;
    }
    __syncthreads();
    const uint32_t next = to;
    for (uint32_t i = threadIdx.x; i < held; i += 256)
        if (next + i < kList) list[next + i] = places[i];
}

struct DrawShared {
    uint64_t places[kList], weights[kList];
    NarrowShared narrow;
    Row row;
    Cut cut;
    uint64_t waves64[kWaves], sums[kParts], before;
    int chosen;
};

// The listed tokens narrowed down, and the draw: the part, then the token.  A workgroup a row, 64 CUs of 256: 24 us, of which
// settings and list 2, narrowing 3 (50 listed tokens) to 9 (650), the part 1, a block of its tokens 3 each.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs a) {
    __shared__ DrawShared sh;
    const int tid = threadIdx.x, row = blockIdx.x;
    if (tid == 0) sh.row = a.settings[row], sh.cut = a.cuts[row], sh.chosen = -1;
    __syncthreads();
    const Row& r = sh.row;
    const Cut& cut = sh.cut;
    if (r.bad || r.greedy || r.arg == INT32_MAX) return;  // the cut kernel has stored those
    const int64_t at = row * a.stride;
    if (tid < a.parts) sh.sums[tid] = a.kept[static_cast<int64_t>(row) * a.parts + tid];
    uint64_t last = ~uint64_t{0};
    if (r.cuts()) {
        const uint32_t listed = a.listed[row];  // above kList: the list does not hold them, the row again
        if (listed <= kList)
            for (uint32_t i = tid; i < listed; i += kThreads) {
                const uint64_t place = a.list[static_cast<int64_t>(row) * kList + i];
                sh.places[i] = place;
                sh.weights[i] = weight_of(r, key_logit(static_cast<uint32_t>(place >> 24)));
            }
        __syncthreads();
        auto each = [&](int b0, int b1, auto f) {
            if (listed <= kList) {
                for (uint32_t i = tid; i < listed; i += kThreads) {
                    const int b = bin_of(r, key_logit(static_cast<uint32_t>(sh.places[i] >> 24)));
                    if (b >= b0 && b <= b1) f(sh.places[i], sh.weights[i]);
                }
                return;
            }
            each_of_row<T>(a, at, r, cut, b0, b1, f);
        };
        last = last_place(r, cut, sh.narrow, listed, each, [&](int bin) { return a.upto[static_cast<int64_t>(row) * kBins + bin]; });
        // the listed tokens that are kept join their parts' weights
        each(cut.sure, kBins, [&](uint64_t place, uint64_t w) {
            if (place > last) return;
            if (r.least > 0.0f) w = weight_of(r, key_logit(static_cast<uint32_t>(place >> 24)), false);
            if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.sums[(place & 0xffffff) / (a.per * kChunk)]), static_cast<unsigned long long>(w));
        });
    }
    __syncthreads();
    if (tid < 64) {
        const uint64_t w = tid < a.parts ? sh.sums[tid] : 0;
        const uint64_t to = wave_scan(w), total = __shfl(to, 63, 64);
        const uint64_t target = part_of(r.uniform, total, false);
        if (to > target && to - w <= target) sh.chosen = tid, sh.before = to - w;
        if (tid == 0) sh.waves64[0] = total;
    }
    __syncthreads();
    const uint64_t total = sh.waves64[0], target = part_of(r.uniform, total, false);
    const int part = sh.chosen;
    if (part < 0) {  // as above
        if (tid == 0) store_token(a, row, -1, 0.0f);
        return;
    }
    uint64_t run = sh.before;
    __syncthreads();
    // the tokens of the part in which the sum passes the target, eight a thread at a time, the next eight requested meanwhile
    const int end = min((part + 1) * a.per * kChunk, a.vocab);
    float next[8];
    load_tokens<T>(a, at, part * a.per * kChunk + tid * 8, next);
    for (int begin = part * a.per * kChunk; begin < end; begin += kBlock) {
        const int first = begin + tid * 8;
        float v[8];
        uint64_t w[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = next[j];
        load_tokens<T>(a, at, first + kBlock, next);
        bool in[8], any = false;
#pragma unroll
        for (int j = 0; j < 8; j++) any |= in[j] = (first + j < end) & cut.keeps(bin_of(r, v[j]), place_of(v[j], first + j), last);
        if (__any(any)) {
            weigh(r, v, false, w);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                // (a select of values: zeroed in branches, elements of this array kept their old values with hipcc 7.2)
                w[j] = in[j] ? w[j] : 0;
                sum += w[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = 0;
        }
        uint64_t all;
        uint64_t to = run + block_scan<kWaves>(sum, sh.waves64, &all) - sum;
        run += all;
        if (run <= target) continue;  // the same for all
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (to + w[j] > target && to <= target) store_token(a, row, first + j, static_cast<float>(static_cast<double>(w[j]) / static_cast<double>(total)));
            to += w[j];
        }
        return;
    }
}

// How a call's rows are cut, and its workspace; rows that a workgroup does need none.
struct Plan {
    int32_t parts, per;
    int64_t peaks, weights, counts, upto, settings, cuts, listed, list, kept, bytes;
};

// A workgroup a row where a row is two blocks at most: 512 rows of 8000 bf16 tokens 24 to 46 us, in parts 30 to 48; 16 rows
// 14 to 25, 18 to 27.  Longer ones are better in parts, also where workgroups of whole rows would fill the chip: 512 rows of
// 32000 61 to 121 us, in parts 63 to 91; 16 rows 31 to 62, 18 to 31 (weights alone, and top-p).
bool by_rows(int64_t vocab) { return vocab <= kRowVocab; }

// Rows in parts are done so many at a time, which fill the chip, and the workspace is that of no more.
constexpr int64_t kSlab = 1024;

Plan plan_of(int64_t rows, int64_t vocab) {
    Plan p{};
    if (by_rows(vocab)) return p;
    rows = std::min(rows, kSlab);
    const int64_t chunks = (vocab + kChunk - 1) / kChunk;
    // about four workgroups a CU, since each leaves 12 KB of bins behind (64 rows of 262144, top-p 0.9: 76 us; with eight 82,
    // with two 90; the peaks alone in as many parts as there may be: 78)
    const int64_t want = std::max<int64_t>(std::min<int64_t>({(1024 + rows - 1) / rows, chunks, kParts}), 1);
    p.per = static_cast<int32_t>((chunks + want - 1) / want);
    p.parts = static_cast<int32_t>((chunks + p.per - 1) / p.per);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.peaks = take(rows * p.parts * static_cast<int64_t>(sizeof(Peak)));
    p.weights = take(rows * p.parts * kBins * 8);
    p.counts = take(rows * p.parts * kBins * 4);
    p.upto = take(rows * kBins * 8);
    p.settings = take(rows * static_cast<int64_t>(sizeof(Row)));
    p.cuts = take(rows * static_cast<int64_t>(sizeof(Cut)));
    p.listed = take(rows * 4);
    p.list = take(rows * kList * 8);
    p.kept = take(rows * p.parts * 8);
    p.bytes = at;
    return p;
}

int check_logits(const SandyTensor* logits, Err e) {
    if (!valid_rank(logits) || logits->rank != 2 || !is_float(logits->dtype) || logits->dims[0] < 0 || logits->dims[1] < 0)
        return fail(e, SANDY_ERR_INVALID, "sample logits must be [rows, vocab] f32 or bf16");
    if (logits->dims[0] > 0 && logits->dims[1] < 1) return fail(e, SANDY_ERR_INVALID, "sample logits must have a vocabulary");
    if (logits->dims[1] > kMaxVocab) return fail(e, SANDY_ERR_UNSUPPORTED, "sample vocabulary above 2^24 tokens");
    if (logits->dims[0] > (1 << 17)) return fail(e, SANDY_ERR_UNSUPPORTED, "sample of more than 2^17 rows");
    return SANDY_OK;
}

template <typename T>
int launch_sample(SampleArgs a, Err e, hipStream_t s) {
    const int64_t all = a.rows, slab = by_rows(a.vocab) ? all : kSlab;
    for (int64_t first = 0; first < all; first += slab) {
        a.rows = static_cast<int32_t>(std::min(slab, all - first));
        const dim3 rows(static_cast<unsigned>(a.rows));
        if (by_rows(a.vocab)) {
            hipLaunchKernelGGL(sample_row_kernel<T>, rows, dim3(kThreads), 0, s, a);
            continue;
        }
        const dim3 parts(static_cast<unsigned>(a.rows) * a.parts);
        hipLaunchKernelGGL(sample_peak_kernel<T>, parts, dim3(256), 0, s, a);
        hipLaunchKernelGGL(sample_bins_kernel<T>, parts, dim3(256), 0, s, a);
        hipLaunchKernelGGL(sample_cut_kernel, rows, dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL(sample_gather_kernel<T>, parts, dim3(256), 0, s, a);
        hipLaunchKernelGGL(sample_draw_kernel<T>, rows, dim3(kThreads), 0, s, a);
        auto next = [](auto*& p, int64_t bytes) {
            if (p) p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(reinterpret_cast<uintptr_t>(p) + bytes);
        };
        auto index = [](int32_t dt) { return dt == SANDY_I32 ? 4 : 8; };
        next(a.logits, slab * a.stride * static_cast<int64_t>(sizeof(typename Vec8<T>::elem)));
        for (const float** p : {&a.temperature, &a.top_p, &a.min_p, &a.uniforms}) next(*p, slab * 4);
        next(a.top_k, slab * index(a.top_k_dt));
        next(a.ids, slab * index(a.ids_dt));
        next(a.probs, slab * 4);
    }
    SANDY_HIP_TRY(hipGetLastError(), e, "sample launch");
    return ok(e);
}

} // namespace
} // namespace sandy_hip

using namespace sandy_hip;

extern "C" int sandy_hip_sample_workspace(const SandyTensor* logits, size_t* bytes, char* err, size_t err_cap) {
    Err e{err, err_cap};
    if (!bytes) return fail(e, SANDY_ERR_INVALID, "sample workspace needs a place for the size");
    if (int status = check_logits(logits, e)) return status;
    *bytes = logits->dims[0] ? static_cast<size_t>(plan_of(logits->dims[0], logits->dims[1]).bytes) : 0;
    return ok(e);
}

extern "C" int sandy_hip_sample(const SandyTensor* logits, const SandyTensor* temperature, const SandyTensor* top_k,
                                const SandyTensor* top_p, const SandyTensor* min_p, const SandyTensor* uniforms,
                                const SandyTensor* ids, const SandyTensor* probs, void* workspace, size_t workspace_bytes,
                                void* stream, char* err, size_t err_cap) {
    Err e{err, err_cap};
    if (int status = check_logits(logits, e)) return status;
    const int64_t rows = logits->dims[0], vocab = logits->dims[1];
    auto per_row = [&](const SandyTensor* t, bool index) {
        return valid_rank(t) && t->rank == 1 && t->dims[0] == rows && contiguous(*t) && (rows == 0 || t->data) &&
               (index ? is_index(t->dtype) : t->dtype == SANDY_F32);
    };
    for (const SandyTensor* t : {temperature, top_p, min_p})
        if (t && !per_row(t, false)) return fail(e, SANDY_ERR_INVALID, "sample temperature, top_p and min_p must be [rows] contiguous f32");
    if (top_k && !per_row(top_k, true)) return fail(e, SANDY_ERR_INVALID, "sample top_k must be [rows] contiguous i32 or i64");
    if (!per_row(uniforms, false)) return fail(e, SANDY_ERR_INVALID, "sample uniforms must be [rows] contiguous f32");
    if (!per_row(ids, true)) return fail(e, SANDY_ERR_INVALID, "sample ids must be [rows] contiguous i32 or i64");
    if (probs && !per_row(probs, false)) return fail(e, SANDY_ERR_INVALID, "sample probs must be [rows] contiguous f32");
    if (vocab > 1 && logits->strides[1] != 1) return fail(e, SANDY_ERR_INVALID, "sample logits must have unit inner stride");
    if (rows == 0) return ok(e);
    if (!logits->data) return fail(e, SANDY_ERR_INVALID, "sample logits are null");
    const Plan p = plan_of(rows, vocab);
    if (p.bytes && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 || workspace_bytes < static_cast<size_t>(p.bytes)))
        return fail(e, SANDY_ERR_INVALID, "sample needs a workspace of %lld bytes, 16-byte aligned", static_cast<long long>(p.bytes));
    SampleArgs a{};
    int status = 0;
    a.errw = device_error_word(e, &status);
    if (status) return status;
    auto f32 = [](const SandyTensor* t) { return t ? static_cast<const float*>(base_ptr(*t)) : nullptr; };
    a.logits = base_ptr(*logits);
    a.stride = rows > 1 ? logits->strides[0] : 0;
    a.temperature = f32(temperature);
    a.top_p = f32(top_p);
    a.min_p = f32(min_p);
    a.uniforms = f32(uniforms);
    a.top_k = top_k ? base_ptr(*top_k) : nullptr;
    a.top_k_dt = top_k ? top_k->dtype : SANDY_I32;
    a.ids = base_ptr(*ids);
    a.ids_dt = ids->dtype;
    a.probs = probs ? static_cast<float*>(base_ptr(*probs)) : nullptr;
    a.rows = static_cast<int32_t>(rows);
    a.vocab = static_cast<int32_t>(vocab);
    a.parts = p.parts;
    a.per = p.per;
    a.bits = 62 - (vocab > 1 ? 64 - __builtin_clzll(static_cast<uint64_t>(vocab - 1)) : 0);
    if (a.bits > 50) a.bits = 50;
    char* w = static_cast<char*>(workspace);
    a.peaks = reinterpret_cast<Peak*>(w + p.peaks);
    a.weights = reinterpret_cast<uint64_t*>(w + p.weights);
    a.counts = reinterpret_cast<uint32_t*>(w + p.counts);
    a.upto = reinterpret_cast<uint64_t*>(w + p.upto);
    a.settings = reinterpret_cast<Row*>(w + p.settings);
    a.cuts = reinterpret_cast<Cut*>(w + p.cuts);
    a.listed = reinterpret_cast<uint32_t*>(w + p.listed);
    a.list = reinterpret_cast<uint64_t*>(w + p.list);
    a.kept = reinterpret_cast<uint64_t*>(w + p.kept);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return logits->dtype == SANDY_BF16 ? launch_sample<BF16>(a, e, s) : launch_sample<F32>(a, e, s);
}
