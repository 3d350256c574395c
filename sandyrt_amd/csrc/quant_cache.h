// quant_cache.h -- the paged K/V cache held in 8 bits: host checks shared by its
// entry points, and a block's scale and payload on the device.
#pragma once
#include "common.h"

namespace sandy_hip {

// What the kernels of this family share: the two caches, whose pages they are,
// and which rows of each sequence the call is about.
struct QuantPages {
    uint8_t* pool[2];    // K, V (V null where the call has none)
    uint8_t* scales[2];
    const int32_t* table;
    int64_t table_stride;
    int64_t num_pages;
    const void* pos;
    const void* counts;  // or null
    uint32_t* errw;
    int32_t pos_dt, counts_dt;
    int32_t batch, heads, dim;
    int32_t max_blocks, log2_page;
    int32_t tokens;  // T
};

// Checks caches, block table, positions and counts against `batch` sequences
// of `tokens` rows; fills everything of `p` but errw.  v_cache may be null.
int check_quant_pages(const SandyQuantCache* kc, const SandyQuantCache* vc, const SandyTensor* table,
                      const SandyTensor* pos, const SandyTensor* counts, int64_t batch, int64_t tokens, Err e,
                      QuantPages* p);

// Whether the counts of a [batch, heads, tokens, dim] call fit the kernels' 32-bit
// indices, and their product 64 bits with room (views that repeat memory can be any size).
inline bool quant_sizes_fit(int64_t batch, int64_t heads, int64_t tokens, int64_t dim) {
    constexpr int64_t kMost = int64_t{1} << 30;
    return batch <= INT32_MAX && heads <= kMost && tokens <= kMost && dim <= kMost &&
           static_cast<double>(batch) * static_cast<double>(heads) * static_cast<double>(tokens) * static_cast<double>(dim) <= 0x1p60;
}

template <int FORMAT>
struct Quant;

// Exponent field of the scale byte for a largest magnitude of these bits: with
// a = 1.m * 2^x and the largest payload 1.t * 2^s, x - s, or one more where m > t.
// The byte is biased like a float's exponent, so it is a's field less s.  One above
// 254 - s would let the payload stand for 2^128: such a magnitude is not held.
template <int FORMAT>
__device__ __forceinline__ int quant_code(uint32_t abs_bits) {
    if (abs_bits >= 0x7f800000u) return 255;
    const int code = static_cast<int>(abs_bits >> 23) - Quant<FORMAT>::kShift +
                     ((abs_bits & 0x7fffffu) > Quant<FORMAT>::kTop ? 1 : 0);
    return code > 254 - Quant<FORMAT>::kShift ? 255 : max(code, 1);
}

// 2^(code - 127); 255 gives NaN, 0 the subnormal 2^-127.
__device__ __forceinline__ float quant_scale(int code) {
    return __uint_as_float(code == 255 ? 0x7fc00000u : code == 0 ? 0x00400000u : static_cast<uint32_t>(code) << 23);
}

template <>
struct Quant<SANDY_QUANT_INT8> {
    static constexpr int kShift = 6;             // 127 = 1.984375 * 2^6
    static constexpr uint32_t kTop = 0x7e0000u;  // 0.984375
    // element J (0..3) of four payload bytes
    template <int J>
    __device__ __forceinline__ static float value(uint32_t w) {
        return static_cast<float>(static_cast<int8_t>(w >> (8 * J)));
    }
    // payloads of four values already divided by the scale: nearest, ties to even
    __device__ __forceinline__ static uint32_t pack(float a, float b, float c, float d) {
        auto byte = [](float f) { return static_cast<uint32_t>(static_cast<int>(__builtin_rintf(f))); };
        const uint32_t lo = __builtin_amdgcn_perm(byte(b), byte(a), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(byte(d), byte(c), 0x04000c0cu);
        return lo | hi;
    }
};

template <>
struct Quant<SANDY_QUANT_E4M3> {
    static constexpr int kShift = 8;             // 448 = 1.75 * 2^8
    static constexpr uint32_t kTop = 0x600000u;  // 0.75
    template <int J>
    __device__ __forceinline__ static float value(uint32_t w) {
        return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), J);
    }
    __device__ __forceinline__ static uint32_t pack(float a, float b, float c, float d) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
    }
};

template <int FORMAT>
__device__ __forceinline__ void quant_values(uint32_t w, float (&v)[4]) {
    v[0] = Quant<FORMAT>::template value<0>(w);
    v[1] = Quant<FORMAT>::template value<1>(w);
    v[2] = Quant<FORMAT>::template value<2>(w);
    v[3] = Quant<FORMAT>::template value<3>(w);
}

// Rows of sequence b in this call: counts[b] brought into 0..tokens.
__device__ __forceinline__ int quant_count(const QuantPages& p, int b) {
    if (!p.counts) return p.tokens;
    const int64_t n = load_index(p.counts, p.counts_dt, b);
    if (n < 0 || n > p.tokens) atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_QUANT_COUNT));
    return static_cast<int>(min<int64_t>(max<int64_t>(n, 0), p.tokens));
}

// Block id of page ordinal `page` of sequence b, or -1 (recorded) where the
// table names no page of the pool.
__device__ __forceinline__ int quant_block(const QuantPages& p, int b, int page) {
    const int id = p.table[b * p.table_stride + page];
    if (id >= 0 && id < p.num_pages) return id;
    atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_BLOCK));
    return -1;
}

} // namespace sandy_hip
