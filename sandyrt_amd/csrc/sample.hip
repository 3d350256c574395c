// sample.hip -- one token a row drawn from its logits, on the device.  The reference samples on the host from logits it
// copies back (src/server/Sampler.cpp:69-79, 212).
//
//   w_i = exp((l_i - max) / T);  tokens ranked by logit, lowest id first among equals
//   K: the first top_k;  P: those of K before which less than top_p of K's weight lies;  M: those with w >= min_p
//   t = u * sum of the weights of P and M's common tokens;  the token where their running sum, in order of ids, passes t
//
// Weights are whole numbers: w_i rounded to 2^-s with s = 62 - log2(vocab) (44 bits of a 262144-token vocabulary).
// Sums of them are exact in any order, so that atomics, chunks and workgroups leave no trace in the result, and every
// comparison (top_p's and the draw's, whose factors have 24 bits) is exact too, in 128 bits.
//
// Ranks are never formed.  Logits fall into 1023 bins of equal width from the maximum down to where weights
// vanish; counts and weights of the bins say in which the cut of top_k and that of top_p lie, and only the tokens there
// (a list, or where it is too long the row again) are narrowed down, 1024 bins of (logit, id) at a time.  A small top_k
// needs counts alone: all it may keep is listed, and top_p looks at the list.  Five launches, the row read three
// times: peak, bins, cut, gather, draw.  Rows are cut into chunks of 4096 tokens, so that a single row fills many
// workgroups and the draw looks at one chunk.
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace sandy_hip {
namespace {

constexpr int kChunk = 4096;    // tokens whose kept weight is one number
constexpr int kBins = 1024;     // the last for tokens without weight
constexpr int kList = 8192;     // tokens of the bins that hold a cut
constexpr int kSmall = 4096;    // a top_k whose tokens are all listed
constexpr int kMaxVocab = 1 << 24;

struct Peak {
    float max, min;  // of the logits above -inf
    int32_t arg;     // lowest id of max; INT32_MAX: no token
    int32_t pad;
};

// A row's parameters and settings.
struct Row {
    double rate;        // log2(e) / temperature
    float max, scale;   // a logit's bin: (max - logit) * scale
    float top_p, least; // least: min_p
    float uniform;
    int32_t arg, bits;
    uint32_t top_k;     // 0: off
    bool greedy, bad;

    // top_k's tokens are all listed
    __device__ bool small() const { return top_k > 0 && top_k <= kSmall; }
    __device__ bool by_p() const { return top_p < 1.0f; }
};

struct Cut {
    Row row;
    // bins below `sure` are kept (as far as min_p goes); tokens of bins first .. last and k_bin are listed
    int32_t sure, first, last, k_bin;
    uint64_t weight;    // of top_k's tokens in bins below k_bin (k_bin < 0: of all of them)
    uint32_t rank;      // how many of the listed tokens from the first or k_bin on are in top_k
    uint32_t pad;
};

struct SampleArgs {
    const void* logits;
    const float *temperature, *top_p, *min_p, *uniforms;
    const void* top_k;
    void* ids;
    float* probs;
    uint32_t* errw;
    int64_t stride;
    int32_t top_k_dt, ids_dt;
    int32_t rows, vocab, chunks, parts, per;  // a part is `per` chunks, one workgroup
    int32_t bits;                             // s
    // workspace
    Peak* peaks;          // [rows, parts]
    uint64_t* weights;    // [rows, parts, kBins]; after the cut, part 0: weight up to and with each bin
    uint32_t* counts;     // [rows, parts, kBins]; likewise
    Cut* cuts;            // [rows]
    uint32_t* listed;     // [rows]
    uint64_t* list;       // [rows, kList]
    uint64_t* kept;       // [rows, chunks]
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

// Row parameters from its parts' peaks; every thread of the workgroup gets them.
__device__ __forceinline__ Row row_of(const SampleArgs& a, int row, Row* shared) {
    if (threadIdx.x < 64) {
        float mx = -__builtin_inff(), mn = __builtin_inff();
        int arg = INT32_MAX;
        const int p = threadIdx.x;  // at most 64 parts
        if (p < a.parts) {
            const Peak k = a.peaks[static_cast<int64_t>(row) * a.parts + p];
            mx = k.max, arg = k.arg, mn = k.min;
        }
        Row r;
        const float t = a.temperature ? a.temperature[row] : 1.0f;
        r.top_p = a.top_p ? a.top_p[row] : 1.0f;
        r.least = a.min_p ? a.min_p[row] : 0.0f;
        r.uniform = a.uniforms[row];
        const int64_t k = a.top_k ? load_index(a.top_k, a.top_k_dt, row) : 0;
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) {
            const float ox = __shfl_xor(mx, m, 64);
            const int oa = __shfl_xor(arg, m, 64);
            if (ox > mx || (ox == mx && oa < arg)) mx = ox, arg = oa;
            mn = fminf(mn, __shfl_xor(mn, m, 64));
        }
        if (threadIdx.x == 0) {
            r.max = mx;
            r.arg = arg;
            r.bits = a.bits;
            r.top_k = k > 0 && k < a.vocab ? static_cast<uint32_t>(k) : 0;
            r.greedy = t == 0.0f;
            r.bad = !(t >= 0.0f) || r.top_p != r.top_p || !(r.least <= 1.0f) || !(r.uniform >= 0.0f && r.uniform < 1.0f);
            r.rate = 1.4426950408889634074 / static_cast<double>(t);
            // bins reach to where weights vanish (2^-bits-1, and a little on), or to the lowest logit where that is nearer
            const double width = fmin(static_cast<double>(mx) - static_cast<double>(mn), (a.bits + 1.5) / r.rate);
            r.scale = width > 0.0 ? static_cast<float>(fmin((kBins - 2) / width, 3.0e38)) : 0.0f;
            *shared = r;
        }
    }
    __syncthreads();
    return *shared;
}

// exp((l - max) / T) = 2^f 2^k, 1 at the maximum: f in -1/2 .. 1/2 by the Taylor series of e^(f ln 2) to the 11th
// power (the next term is below 7e-15 of the sum).  Below 2^-200 it stays there, which weighs nothing.
struct Ratio {
    double p;
    int k;
    __device__ double value() const { return p * __longlong_as_double(static_cast<long long>(1023 + k) << 52); }
};
__device__ __forceinline__ Ratio ratio_of(const Row& r, float l) {
    if (l == r.max) return Ratio{1.0, 0};
    const double x = fmax((static_cast<double>(l) - static_cast<double>(r.max)) * r.rate, -200.0);  // (inf less inf: -200 too)
    const double k = __builtin_rint(x), f = x - k;
    double p = 4.44553827187081162e-10;  // (ln 2)^11 / 11!
    p = fma(p, f, 7.05491162080112336e-09);
    p = fma(p, f, 1.01780860092396999e-07);
    p = fma(p, f, 1.32154867901443095e-06);
    p = fma(p, f, 1.52527338040598411e-05);
    p = fma(p, f, 1.54035303933816088e-04);
    p = fma(p, f, 1.33335581464284433e-03);
    p = fma(p, f, 9.61812910762847688e-03);
    p = fma(p, f, 5.55041086648215831e-02);
    p = fma(p, f, 2.40226506959100722e-01);
    p = fma(p, f, 6.93147180559945286e-01);
    p = fma(p, f, 1.0);
    return Ratio{p, static_cast<int>(k)};
}
// to the nearest whole multiple of 2^-bits: 52 bits hold it behind 2^52
__device__ __forceinline__ uint64_t weight_of(const Row& r, const Ratio& ratio) {
    const double unit = __longlong_as_double(static_cast<long long>(1023 + r.bits + ratio.k) << 52);
    return static_cast<uint64_t>(__double_as_longlong(fma(ratio.p, unit, 4503599627370496.0))) - 0x4330000000000000ull;
}
__device__ __forceinline__ bool likely(const Row& r, const Ratio& ratio) {
    return r.least <= 0.0f || ratio.value() >= static_cast<double>(r.least);
}
// Non-decreasing as logits fall; the last bin holds no token that weighs anything (those end a ninetieth before it, or
// the lowest logit ends at kBins - 2).
__device__ __forceinline__ int bin_of(const Row& r, float l) {
    if (l == r.max) return 0;
    const float at = (r.max - l) * r.scale;
    return at >= static_cast<float>(kBins - 1) ? kBins - 1 : static_cast<int>(fminf(at, static_cast<float>(kBins - 2)));
}

// p * w rounded up or down, exactly; 0 <= p < 1
__device__ __forceinline__ uint64_t part_of(float p, uint64_t w, bool up) {
    const uint32_t u = __float_as_uint(p), e = u >> 23, m = e ? (u & 0x7fffffu) | 0x800000u : u & 0x7fffffu;
    const int shift = 150 - static_cast<int>(e ? e : 1);  // p = m * 2^-shift, shift >= 24
    const unsigned __int128 prod = static_cast<unsigned __int128>(m) * w;
    if (shift >= 100) return up && prod != 0 ? 1 : 0;
    const uint64_t q = static_cast<uint64_t>(prod >> shift);
    return q + (up && (prod & ((static_cast<unsigned __int128>(1) << shift) - 1)) != 0 ? 1 : 0);
}

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

// ------------------------------------------------------------------ peak
template <typename T>
__global__ __launch_bounds__(256) void sample_peak_kernel(SampleArgs a) {
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const int64_t at = row * a.stride;
    const int begin = part * a.per * kChunk, end = min(begin + a.per * kChunk, a.vocab);
    float mx = -__builtin_inff(), mn = __builtin_inff();
    int arg = INT32_MAX;
    for (int chunk = begin; chunk < end; chunk += kChunk) {
        float v[kChunk / 2048][8];  // requested together
#pragma unroll
        for (int h = 0; h < kChunk / 2048; h++) load_tokens<T>(a, at, chunk + h * 2048 + static_cast<int>(threadIdx.x) * 8, v[h]);
#pragma unroll
        for (int h = 0; h < kChunk / 2048; h++)
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (token(v[h][j])) {
                    if (v[h][j] > mx || arg == INT32_MAX) mx = v[h][j], arg = chunk + h * 2048 + static_cast<int>(threadIdx.x) * 8 + j;
                    mn = fminf(mn, v[h][j]);
                }
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const float ox = __shfl_xor(mx, m, 64);
        const int oa = __shfl_xor(arg, m, 64);
        if (ox > mx || (ox == mx && oa < arg)) mx = ox, arg = oa;
        mn = fminf(mn, __shfl_xor(mn, m, 64));
    }
    __shared__ Peak waves[4];
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = Peak{mx, mn, arg, 0};
    __syncthreads();
    if (threadIdx.x == 0) {
        Peak p = waves[0];
#pragma unroll
        for (int w = 1; w < 4; w++) {
            if (waves[w].max > p.max || (waves[w].max == p.max && waves[w].arg < p.arg)) p.max = waves[w].max, p.arg = waves[w].arg;
            p.min = fminf(p.min, waves[w].min);
        }
        a.peaks[blockIdx.x] = p;
    }
}

// ------------------------------------------------------------------ bins
// Counts where top_k asks for them, weights where top_p does and top_k's tokens are not all listed.
template <typename T>
__global__ __launch_bounds__(256) void sample_bins_kernel(SampleArgs a) {
    __shared__ uint64_t weights[kBins];
    __shared__ uint32_t counts[kBins];
    __shared__ Row shared;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    for (int i = threadIdx.x; i < kBins; i += 256) weights[i] = 0, counts[i] = 0;
    const Row r = row_of(a, row, &shared);
    if (r.greedy || r.bad || !(r.top_k || r.by_p())) return;
    const int64_t at = row * a.stride;
    const int begin = part * a.per * kChunk, end = min(begin + a.per * kChunk, a.vocab);
    auto fill = [&](auto count, auto weigh) {
        for (int i = begin + threadIdx.x * 8; i < end; i += 2048) {
            float v[8];
            load_tokens<T>(a, at, i, v);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (!token(v[j])) continue;
                const int b = bin_of(r, v[j]);
                if constexpr (decltype(count)::value) atomicAdd(&counts[b], 1u);
                if constexpr (decltype(weigh)::value)
                    atomicAdd(reinterpret_cast<unsigned long long*>(&weights[b]), static_cast<unsigned long long>(weight_of(r, ratio_of(r, v[j]))));
            }
        }
    };
    const bool weigh = r.by_p() && !r.small();
    if (!weigh) fill(std::true_type{}, std::false_type{});
    else if (r.top_k) fill(std::true_type{}, std::true_type{});
    else fill(std::false_type{}, std::true_type{});
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += 256) {
        a.weights[static_cast<int64_t>(blockIdx.x) * kBins + i] = weights[i];
        a.counts[static_cast<int64_t>(blockIdx.x) * kBins + i] = counts[i];
    }
}

// ------------------------------------------------------------------ sums over a workgroup of 1024
// Inclusive sums of v over the threads; `waves` holds 16 values, `total` all of them.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* waves, V* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const V o = __shfl_up(v, s, 64);
        if (lane >= s) v += o;
    }
    __syncthreads();  // the last use of `waves` is over
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        if (w < wave) before += waves[w];
        all += waves[w];
    }
    *total = all;
    return before + v;
}

// ------------------------------------------------------------------ cut
__global__ __launch_bounds__(1024) void sample_cut_kernel(SampleArgs a) {
    __shared__ Row shared;
    __shared__ uint64_t waves64[16];
    __shared__ uint32_t waves32[16];
    __shared__ int k_bin, k_last, p_first, p_last;
    __shared__ uint64_t low, high;
    __shared__ uint32_t rank;
    const int row = blockIdx.x, bin = threadIdx.x;
    const Row r = row_of(a, row, &shared);
    uint64_t w = 0, w_to = 0, all = 0;
    uint32_t c = 0, c_to = 0, tokens = 0;
    const bool cuts = !r.greedy && !r.bad && (r.top_k || r.by_p());
    if (cuts) {
        const int64_t first = static_cast<int64_t>(row) * a.parts * kBins + bin;
#pragma unroll 8
        for (int p = 0; p < a.parts; p++) {
            w += a.weights[first + p * kBins];
            c += a.counts[first + p * kBins];
        }
        w_to = block_scan(w, waves64, &all);
        c_to = block_scan(c, waves32, &tokens);
        a.weights[first] = w_to;  // part 0's, which no one else reads before the draw
    }
    if (bin == 0) k_bin = -1, k_last = p_first = p_last = kBins, low = high = all, rank = 0;
    __syncthreads();
    const uint32_t k = r.top_k;
    // the bin where top_k ends, if it ends inside one whose tokens weigh anything
    if (cuts && k && k < tokens && c_to >= k && c_to - c < k) {
        k_last = bin;
        if (c_to == k || bin == kBins - 1) {
            low = high = w_to;
        } else {
            k_bin = bin;
            low = w_to - w;
            high = w_to;
            rank = k - (c_to - c);
        }
    }
    __syncthreads();
    if (cuts && r.by_p() && !r.small()) {
        // top_p's cut lies where the sums reach its part of top_k's weight, which is between low and high
        const uint64_t from = r.top_p > 0.0f ? part_of(r.top_p, low, true) : 0, to = r.top_p > 0.0f ? part_of(r.top_p, high, true) : 0;
        const uint64_t before = w_to - w;
        if (w_to >= from && (bin == 0 || before < from)) p_first = bin;
        if (w_to >= to && (bin == 0 || before < to)) p_last = bin;
    }
    __syncthreads();
    if (bin == 0) {
        if (r.bad) atomicOr(a.errw, static_cast<uint32_t>(SANDY_DEVERR_SAMPLE));
        a.listed[row] = 0;
        Cut cut;
        cut.row = r;
        cut.weight = low;
        cut.rank = rank;
        cut.pad = 0;
        cut.k_bin = k_bin;
        cut.first = kBins;
        cut.last = -1;
        const int by_k = k_bin >= 0 ? k_bin : k_last < kBins ? k_last + 1 : kBins;
        cut.sure = by_k;
        if (cuts && r.small()) {
            // all that top_k may keep: to its last bin, or every token that weighs anything
            cut.sure = cut.first = 0;
            cut.last = min(k_last, kBins - 2);
            cut.rank = k < tokens && k_last < kBins - 1 ? k : 0;
        } else if (cuts && r.by_p()) {
            cut.first = p_first;
            cut.last = p_last;
            cut.sure = min(p_first, by_k);
        }
        a.cuts[row] = cut;
    }
}

__device__ __forceinline__ bool in_question(const Cut& c, int bin) { return bin == c.k_bin || (bin >= c.first && bin <= c.last); }

// ------------------------------------------------------------------ gather
template <typename T>
__global__ __launch_bounds__(256) void sample_gather_kernel(SampleArgs a) {
    __shared__ uint64_t waves[4], places[kChunk];
    __shared__ uint32_t found, to;
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const Cut cut = a.cuts[row];
    const Row& r = cut.row;
    if (r.greedy || r.bad) return;
    const int64_t at = row * a.stride;
    for (int chunk = part * a.per; chunk < min((part + 1) * a.per, a.chunks); chunk++) {
        if (threadIdx.x == 0) found = 0;
        __syncthreads();
        uint64_t sum = 0;
        float v[kChunk / 2048][8];
#pragma unroll
        for (int h = 0; h < kChunk / 2048; h++) load_tokens<T>(a, at, chunk * kChunk + h * 2048 + static_cast<int>(threadIdx.x) * 8, v[h]);
#pragma unroll
        for (int h = 0; h < kChunk / 2048; h++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (!token(v[h][j])) continue;
                const int b = bin_of(r, v[h][j]);
                if (b < cut.sure) {
                    const Ratio ratio = ratio_of(r, v[h][j]);
                    if (likely(r, ratio)) sum += weight_of(r, ratio);
                } else if (in_question(cut, b)) {
                    places[atomicAdd(&found, 1u)] = place_of(v[h][j], chunk * kChunk + h * 2048 + static_cast<int>(threadIdx.x) * 8 + j);
                }
            }
        sum = wave_sum(sum);
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            a.kept[static_cast<int64_t>(row) * a.chunks + chunk] = waves[0] + waves[1] + waves[2] + waves[3];
            if (found) to = atomicAdd(&a.listed[row], found);
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < found && to + i < kList; i += 256) a.list[static_cast<int64_t>(row) * kList + to + i] = places[i];
        __syncthreads();
    }
}

// ------------------------------------------------------------------ draw
// What the draw of a row keeps in LDS.
struct DrawShared {
    uint64_t places[kList], weights[kList];
    uint64_t bin_weights[kBins], waves64[16], lows[16], highs[16];
    uint32_t bin_counts[kBins], waves32[16];
    uint64_t lo, hi, weight_before;
    uint32_t count_before;
    int chosen;
};

// f(place, weight, bin) for every listed token, or (whole) every token of the row.
template <typename T, typename F>
__device__ __forceinline__ void each_token(const SampleArgs& a, const Row& r, const DrawShared& sh, int row, uint32_t listed, F f) {
    if (listed <= kList) {
        for (uint32_t i = threadIdx.x; i < listed; i += 1024) f(sh.places[i], sh.weights[i], bin_of(r, key_logit(static_cast<uint32_t>(sh.places[i] >> 24))));
        return;
    }
    for (int i = threadIdx.x * 8; i < a.vocab; i += 8192) {
        float v[8];
        load_tokens<T>(a, row * a.stride, i, v);
#pragma unroll 1
        for (int j = 0; j < 8; j++) {
            float l = v[0];
#pragma unroll
            for (int q = 1; q < 8; q++) l = j == q ? v[q] : l;
            if (token(l)) f(place_of(l, i + j), weight_of(r, ratio_of(r, l)), bin_of(r, l));
        }
    }
}

// Of the tokens of bins b0 .. b1, in rank order: the place of the one with which they become `rank`, or (rank 0) with
// which their weights reach `weight`; weight_before is then the sum up to and with it.  Places are told apart 1024
// equal steps at a time, each time among fewer than before.
template <typename T>
__device__ __attribute__((noinline)) uint64_t narrow(const SampleArgs& a, const Row& r, DrawShared& sh, int row, uint32_t listed, int b0, int b1,
                                                     uint32_t rank, uint64_t weight) {
    const int tid = threadIdx.x;
    // from the first to the last of them
    uint64_t low = ~uint64_t{0}, high = 0;
    each_token<T>(a, r, sh, row, listed, [&](uint64_t place, uint64_t, int b) {
        if (b < b0 || b > b1) return;
        low = min(low, place);
        high = max(high, place);
    });
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        low = min(low, static_cast<uint64_t>(__shfl_xor(low, m, 64)));
        high = max(high, static_cast<uint64_t>(__shfl_xor(high, m, 64)));
    }
    if ((tid & 63) == 0) sh.lows[tid >> 6] = low, sh.highs[tid >> 6] = high;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 16; w++) low = min(low, sh.lows[w]), high = max(high, sh.highs[w]);
        sh.lo = low;
        sh.hi = high;
        sh.weight_before = 0;
        sh.count_before = 0;
    }
    __syncthreads();
    for (;;) {
        const uint64_t from = sh.lo, to = sh.hi;
        const int shift = max(0, 54 - __builtin_clzll((to - from) | 1));  // at most 1024 steps
        sh.bin_weights[tid] = 0;
        sh.bin_counts[tid] = 0;
        __syncthreads();
        each_token<T>(a, r, sh, row, listed, [&](uint64_t place, uint64_t w, int b) {
            if (b < b0 || b > b1 || place < from || place > to) return;
            const int q = static_cast<int>((place - from) >> shift);
            atomicAdd(&sh.bin_counts[q], 1u);
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bin_weights[q]), static_cast<unsigned long long>(w));
        });
        __syncthreads();
        const uint64_t w = sh.bin_weights[tid];
        const uint32_t c = sh.bin_counts[tid];
        uint64_t all;
        uint32_t tokens;
        const uint64_t w_to = sh.weight_before + block_scan(w, sh.waves64, &all);
        const uint32_t c_to = sh.count_before + block_scan(c, sh.waves32, &tokens);
        // (a weight of 0 is reached by the first token)
        const bool here = c != 0 && (rank ? c_to >= rank && c_to - c < rank : w_to >= weight && (w_to - w < weight || c_to == c));
        if (!__syncthreads_or(here)) {  // fewer tokens, or less weight, than asked for: all of them
            if (tid == 0) sh.lo = to, sh.weight_before += all;
            __syncthreads();
            break;
        }
        if (here) {
            sh.lo = from + (static_cast<uint64_t>(tid) << shift);
            sh.hi = min(to, from + ((static_cast<uint64_t>(tid) + 1) << shift) - 1);
            sh.weight_before = shift == 0 ? w_to : w_to - w;
            sh.count_before = c_to - c;
        }
        __syncthreads();
        if (shift == 0) break;
    }
    return sh.lo;
}

template <typename T>
__global__ __launch_bounds__(1024) void sample_draw_kernel(SampleArgs a) {
    __shared__ DrawShared sh;
    const int tid = threadIdx.x, row = blockIdx.x;
    const Cut cut = a.cuts[row];
    const Row& r = cut.row;
    if (r.bad || r.greedy || r.arg == INT32_MAX) {
        if (tid == 0) {
            store_index(a.ids, a.ids_dt, row, r.bad || r.arg == INT32_MAX ? -1 : r.arg);
            if (a.probs) a.probs[row] = r.bad || r.arg == INT32_MAX ? 0.0f : 1.0f;
        }
        return;
    }
    const uint32_t listed = a.listed[row];  // above kList: the list does not hold them, the row again
    const int64_t at = row * a.stride;
    if (listed <= kList)
        for (uint32_t i = tid; i < listed; i += 1024) {
            const uint64_t place = a.list[static_cast<int64_t>(row) * kList + i];
            sh.places[i] = place;
            sh.weights[i] = weight_of(r, ratio_of(r, key_logit(static_cast<uint32_t>(place >> 24))));
        }
    __syncthreads();
    uint64_t last = ~uint64_t{0};  // the last place kept
    if (r.small()) {
        // ranks and weights from the first token on
        uint64_t kept = 0;
        if (cut.rank) {
            last = narrow<T>(a, r, sh, row, listed, 0, cut.last, cut.rank, 0);
            kept = sh.weight_before;
            __syncthreads();
        } else if (r.by_p()) {
            uint64_t mine = 0;
            each_token<T>(a, r, sh, row, listed, [&](uint64_t, uint64_t w, int b) { mine += b <= cut.last ? w : 0; });
            block_scan(mine, sh.waves64, &kept);
        }
        if (r.by_p()) {
            last = min(last, narrow<T>(a, r, sh, row, listed, 0, cut.last, 0, r.top_p > 0.0f ? part_of(r.top_p, kept, true) : 0));
            __syncthreads();
        }
    } else {
        uint64_t kept = cut.weight;  // top_k's
        if (cut.k_bin >= 0) {
            last = narrow<T>(a, r, sh, row, listed, cut.k_bin, cut.k_bin, cut.rank, 0);
            kept += sh.weight_before;
            __syncthreads();
        }
        if (cut.last >= 0) {
            const uint64_t upto = r.top_p > 0.0f ? part_of(r.top_p, kept, true) : 0;
            const uint64_t* to = a.weights + static_cast<int64_t>(row) * a.parts * kBins;
            int bin = cut.first;
            while (bin < cut.last && to[bin] < upto) bin++;
            const uint64_t before = bin > 0 ? to[bin - 1] : 0;
            last = min(last, narrow<T>(a, r, sh, row, listed, bin, bin, 0, upto > before ? upto - before : 0));
            __syncthreads();
        }
    }
    // the kept weight of each chunk: that of the bins below the cuts, and of the listed tokens up to `last`
    uint64_t* chunk_sums = a.kept + static_cast<int64_t>(row) * a.chunks;
    if (listed) {
        each_token<T>(a, r, sh, row, listed, [&](uint64_t place, uint64_t w, int b) {
            if (b < cut.sure || !in_question(cut, b) || place > last || w == 0) return;
            if (!likely(r, ratio_of(r, key_logit(static_cast<uint32_t>(place >> 24))))) return;
            atomicAdd(reinterpret_cast<unsigned long long*>(&chunk_sums[(place & 0xffffff) / kChunk]), static_cast<unsigned long long>(w));
        });
        __threadfence();
        __syncthreads();
    }
    auto chunk_sum = [&](int c) -> uint64_t { return __hip_atomic_load(&chunk_sums[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    uint64_t total = 0, mine = 0;
    for (int c = tid; c < a.chunks; c += 1024) mine += chunk_sum(c);
    block_scan(mine, sh.waves64, &total);
    const uint64_t target = part_of(r.uniform, total, false);
    uint64_t base = 0;
    if (tid == 0) sh.chosen = 0;
    __syncthreads();
    for (int c0 = 0; c0 < a.chunks; c0 += 1024) {
        const uint64_t w = c0 + tid < a.chunks ? chunk_sum(c0 + tid) : 0;
        uint64_t all;
        const uint64_t to = base + block_scan(w, sh.waves64, &all);
        if (to > target && to - w <= target) sh.chosen = c0 + tid, sh.weight_before = to - w;
        base += all;
    }
    __syncthreads();
    // the tokens of the chunk in which the sum passes the target, four a thread
    uint64_t w4[4], sum = 0;
    const int id0 = sh.chosen * kChunk + tid * 4;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float l = id0 + j < a.vocab ? Vec8<T>::load1(a.logits, at + id0 + j) : -__builtin_inff();
        w4[j] = 0;
        if (token(l)) {
            const Ratio ratio = ratio_of(r, l);
            const int b = bin_of(r, l);
            if ((b < cut.sure || (in_question(cut, b) && place_of(l, id0 + j) <= last)) && likely(r, ratio)) w4[j] = weight_of(r, ratio);
        }
        sum += w4[j];
    }
    uint64_t all;
    uint64_t to = sh.weight_before + block_scan(sum, sh.waves64, &all) - sum;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (to + w4[j] > target && to <= target) {
            store_index(a.ids, a.ids_dt, row, id0 + j);
            if (a.probs) a.probs[row] = static_cast<float>(static_cast<double>(w4[j]) / static_cast<double>(total));
        }
        to += w4[j];
    }
}

// How a call's rows are cut, and its workspace.
struct Plan {
    int32_t chunks, parts, per;
    int64_t peaks, weights, counts, cuts, listed, list, kept, bytes;
};

Plan plan_of(int64_t rows, int64_t vocab) {
    Plan p{};
    p.chunks = static_cast<int32_t>((vocab + kChunk - 1) / kChunk);
    // about four workgroups a CU, of at least two chunks, and no more parts than the cut sums up quickly
    const int64_t want = std::min<int64_t>({std::max<int64_t>((1024 + rows - 1) / rows, 1), (p.chunks + 1) / 2, 64});
    p.per = static_cast<int32_t>((p.chunks + want - 1) / want);
    p.parts = (p.chunks + p.per - 1) / p.per;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.peaks = take(rows * p.parts * static_cast<int64_t>(sizeof(Peak)));
    p.weights = take(rows * p.parts * kBins * 8);
    p.counts = take(rows * p.parts * kBins * 4);
    p.cuts = take(rows * static_cast<int64_t>(sizeof(Cut)));
    p.listed = take(rows * 4);
    p.list = take(rows * kList * 8);
    p.kept = take(rows * p.chunks * 8);
    p.bytes = at;
    return p;
}

int check_logits(const SandyTensor* logits, Err e) {
    if (!valid_rank(logits) || logits->rank != 2 || !is_float(logits->dtype) || logits->dims[0] < 0 || logits->dims[1] < 0)
        return fail(e, SANDY_ERR_INVALID, "sample logits must be [rows, vocab] f32 or bf16");
    if (logits->dims[0] > 0 && logits->dims[1] < 1) return fail(e, SANDY_ERR_INVALID, "sample logits must have a vocabulary");
    if (logits->dims[1] > kMaxVocab) return fail(e, SANDY_ERR_UNSUPPORTED, "sample vocabulary above 2^24 tokens");
    if (logits->dims[0] > (1 << 20)) return fail(e, SANDY_ERR_UNSUPPORTED, "sample of more than 2^20 rows");
    return SANDY_OK;
}

template <typename T>
int launch_sample(const SampleArgs& a, Err e, hipStream_t s) {
    const dim3 parts(static_cast<unsigned>(a.rows) * a.parts), rows(static_cast<unsigned>(a.rows));
    hipLaunchKernelGGL(sample_peak_kernel<T>, parts, dim3(256), 0, s, a);
    hipLaunchKernelGGL(sample_bins_kernel<T>, parts, dim3(256), 0, s, a);
    hipLaunchKernelGGL(sample_cut_kernel, rows, dim3(1024), 0, s, a);
    hipLaunchKernelGGL(sample_gather_kernel<T>, parts, dim3(256), 0, s, a);
    hipLaunchKernelGGL(sample_draw_kernel<T>, rows, dim3(1024), 0, s, a);
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
    if (rows * p.parts > (int64_t{1} << 23)) return fail(e, SANDY_ERR_UNSUPPORTED, "sample of too many rows");
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 || workspace_bytes < static_cast<size_t>(p.bytes))
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
    a.chunks = p.chunks;
    a.parts = p.parts;
    a.per = p.per;
    a.bits = 62 - (vocab > 1 ? 64 - __builtin_clzll(static_cast<uint64_t>(vocab - 1)) : 0);
    if (a.bits > 50) a.bits = 50;
    char* w = static_cast<char*>(workspace);
    a.peaks = reinterpret_cast<Peak*>(w + p.peaks);
    a.weights = reinterpret_cast<uint64_t*>(w + p.weights);
    a.counts = reinterpret_cast<uint32_t*>(w + p.counts);
    a.cuts = reinterpret_cast<Cut*>(w + p.cuts);
    a.listed = reinterpret_cast<uint32_t*>(w + p.listed);
    a.list = reinterpret_cast<uint64_t*>(w + p.list);
    a.kept = reinterpret_cast<uint64_t*>(w + p.kept);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return logits->dtype == SANDY_BF16 ? launch_sample<BF16>(a, e, s) : launch_sample<F32>(a, e, s);
}
