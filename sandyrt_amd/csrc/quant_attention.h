// quant_attention.h -- attention over the 8-bit paged K/V cache: the arguments
// its kernels share.
#pragma once
#include "quant_cache.h"

namespace sandy_hip {

struct QuantAttnArgs {
    QuantPages p;  // tokens = queries a sequence
    const void* q;
    void* out;
    int64_t qs[4], os[4];  // element strides over (b, h, t, d)
    int64_t window;
    float scale_log2;      // scale * log2(e)
    int32_t hq, group;     // q heads, of one kv head
    uint32_t group_magic;  // for divide() by group
    int32_t f32;           // q and out are f32, else bf16
};

// Keys [first, last] that a query sees (none: last < first).
struct KeyRange {
    int first, last;
};

// The positions of a sequence's queries in 32 bits: what lies past the block
// table (2^30 keys at most) or before the first key is brought to that border.
struct SeqKeys {
    int base;   // position of query 0
    int lower;  // its first key, or below 0
    int cap;    // keys the block table covers

    __device__ __forceinline__ KeyRange of(int t) const {
        return KeyRange{min(max(lower + t, 0), cap), min(base + t, cap - 1)};
    }
};

__device__ __forceinline__ SeqKeys quant_keys(const QuantAttnArgs& a, int64_t pos) {
    constexpr int64_t kFar = int64_t{1} << 30;
    SeqKeys s;
    s.cap = a.p.max_blocks << a.p.log2_page;
    s.base = static_cast<int>(min<int64_t>(max<int64_t>(pos, 0), kFar));
    // window <= INT64_MAX and pos >= 0: no overflow
    s.lower = a.window > 0 ? static_cast<int>(max<int64_t>(min<int64_t>(max<int64_t>(pos, 0) - a.window, kFar - 1), -kFar) + 1) : -static_cast<int>(kFar);
    return s;
}

// n / d with magic = 2^32 / d rounded down (2^32 - 1 for d = 1): at most one short.
__device__ __forceinline__ int divide(int n, int d, uint32_t magic) {
    const int q = static_cast<int>(__umulhi(static_cast<uint32_t>(n), magic));
    return q + (n - q * d >= d ? 1 : 0);
}

// Sums over V stay finite where V is next to 2^128: from the first block whose scale is
// 2^80 or more on ("loud"), a sum holds 2^-64 of itself.  A weight is below 2^8 and keys
// are at most 2^30, so a sum is below 2^126 before and below 2^104 after.  Values that
// 2^-64 takes below fp32's normal numbers are below 2^-62, 2^-148 of the loud block's
// largest.  The sum of weights, never negative, carries the mark as its sign.
constexpr int kLoudCode = 127 + 80;
constexpr uint32_t kLoudBits = static_cast<uint32_t>(kLoudCode) << 23;  // of such a scale; times 2^-64 none is
constexpr float kLoudDown = 0x1p-64f, kLoudUp = 0x1p64f;
__device__ __forceinline__ bool loud_code(int c) { return c >= kLoudCode && c != 255; }
__device__ __forceinline__ float mark_loud(float total, bool loud) {
    return __uint_as_float(__float_as_uint(total) | (loud ? 0x80000000u : 0u));
}
__device__ __forceinline__ bool is_loud(float total) { return __float_as_uint(total) >> 31; }

// Few queries a sequence (quant_decode.hip): whether the kernel takes the call,
// its workspace (whatever the call's strides), its launch.
bool quant_decode_takes(const QuantAttnArgs& a);
size_t quant_decode_workspace(int64_t batch, int64_t hq, int64_t heads, int64_t tokens, int64_t dim, int64_t page,
                              int64_t max_blocks, int64_t window);
int launch_quant_decode(const QuantAttnArgs& a, int32_t format, void* workspace, hipStream_t stream, Err e);

// Many queries a sequence (quant_prefill.hip), of the calls that quant_decode_takes; no workspace.
bool quant_prefill_takes(int64_t batch, int64_t hq, int64_t heads, int64_t tokens, int64_t dim, int64_t max_blocks,
                         bool f32);
int launch_quant_prefill(const QuantAttnArgs& a, int32_t format, hipStream_t stream, Err e);

} // namespace sandy_hip
