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
    int32_t f32;           // q and out are f32, else bf16
};

// Keys [first, last] that query t of a sequence at `pos` sees (none: last < first).
struct KeyRange {
    int first, last;
};

__device__ __forceinline__ KeyRange quant_keys(const QuantAttnArgs& a, int64_t pos, int t) {
    const int64_t at = min<int64_t>(pos, INT64_MAX - INT32_MAX) + t;
    const int64_t cap = static_cast<int64_t>(a.p.max_blocks) << a.p.log2_page;
    KeyRange r;
    r.last = static_cast<int>(min<int64_t>(at, cap - 1));
    r.first = a.window > 0 ? static_cast<int>(min<int64_t>(max<int64_t>(at - a.window + 1, 0), cap)) : 0;
    return r;
}

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
