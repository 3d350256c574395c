// quant_attention.hip -- causal attention over the 8-bit paged K/V cache.
//
// o = sum_k p_k v_k / sum_k p_k, p_k = 2^(s_k - m), s_k = scale log2(e) q . k_k,
// one pass over the keys with the running maximum m and sum.  A block's scale
// never touches its payload: K's multiplies the score, V's the weight p.
#include "quant_attention.h"

#include <algorithm>
#include <cmath>

namespace sandy_hip {
namespace {

constexpr int kMaxDim = 512;

// Any head dim, page size and stride: a workgroup per (sequence, q head, query), 256
// keys at a time.  A thread scores one key, W bytes of it a load; then groups of
// `lanes` threads (a thread a dim, two past 256 dims) weigh every groups-th key.  Bound
// by the one key a thread scores and the one workgroup a row: it serves what the MFMA
// kernels do not (pages under 16 rows, head dims that are no multiple of 16 or above
// 256, unaligned tensors).  32 sequences of 512 to 4096 keys of 32 / 4 heads of 64 take
// 352 us here (16 there), 2048 causal queries of them 1970 (54).
template <typename T, int FORMAT, int W>
__global__ __launch_bounds__(256) void quant_attention_general_kernel(QuantAttnArgs a) {
    constexpr int kDims = kMaxDim / 256;
    __shared__ float qf[kMaxDim];
    __shared__ float weight[256];
    __shared__ const uint8_t* row[256];
    __shared__ float part[4];
    __shared__ bool far[4];
    __shared__ double sums[4];
    const QuantPages& p = a.p;
    const int tid = threadIdx.x;
    uint32_t at = blockIdx.x;
    const int t = at % p.tokens;
    at /= p.tokens;
    const int h = at % a.hq;
    const int b = at / a.hq;
    const int kh = h / a.group;
    const int D = p.dim;
    const int64_t pos = load_index(p.pos, p.pos_dt, b);
    if (pos < 0 && tid == 0) atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_ATTN_POS));
    KeyRange keys = quant_keys(a, pos).of(t);
    if (pos < 0 || t >= quant_count(p, b)) keys = KeyRange{0, -1};
    const int64_t q0 = b * a.qs[0] + h * a.qs[1] + t * a.qs[2];
    for (int d = tid; d < D; d += 256) qf[d] = Vec8<T>::load1(a.q, q0 + d * a.qs[3]);
    __syncthreads();
    const int lanes = min(D, 256), groups = 256 / lanes, group = tid / lanes, dim0 = tid - group * lanes;
    float m = -INFINITY, acc[kDims];
    double l = 0.0;
    bool loud = false;
#pragma unroll
    for (int i = 0; i < kDims; i++) acc[i] = 0.0f;
    for (int k0 = keys.first; k0 <= keys.last; k0 += 256) {
        const int key = k0 + tid;
        float s = -INFINITY;
        int vc = 0;
        const uint8_t* vrow = nullptr;
        if (key <= keys.last) {
            const int id = quant_block(p, b, key >> p.log2_page);
            if (id >= 0) {
                const int64_t block = static_cast<int64_t>(id) * p.heads + kh;
                const int64_t from = ((block << p.log2_page) + (key & ((1 << p.log2_page) - 1))) * D;
                const uint8_t* krow = p.pool[0] + from;
                float dot = 0.0f;
                if constexpr (W == 4) {
#pragma unroll 4
                    for (int d = 0; d < D; d += 4) {
                        float k[4];
                        quant_values<FORMAT>(*reinterpret_cast<const uint32_t*>(krow + d), k);
#pragma unroll
                        for (int j = 0; j < 4; j++) dot = fmaf(qf[d + j], k[j], dot);
                    }
                } else {
                    for (int d = 0; d < D; d++) dot = fmaf(qf[d], Quant<FORMAT>::template value<0>(krow[d]), dot);
                }
                s = dot * quant_scale(p.scales[0][block]) * a.scale_log2;
                vc = p.scales[1][block];
                vrow = p.pool[1] + from;
            }
        }
        float mx = wave_max(s);
        const bool any = __any(loud_code(vc));
        __syncthreads();  // the sums over the chunk before have been read
        if ((tid & 63) == 0) part[tid >> 6] = mx, far[tid >> 6] = any;
        __syncthreads();
        mx = fmaxf(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), m);
        const float shift = mx == -INFINITY ? 0.0f : mx;
        const float alpha = __builtin_amdgcn_exp2f(m - shift);
        const float w = vrow ? __builtin_amdgcn_exp2f(s - shift) : 0.0f;
        l = l * static_cast<double>(alpha) + static_cast<double>(w);
        m = mx;
        if (!loud && (far[0] || far[1] || far[2] || far[3])) {
            loud = true;
#pragma unroll
            for (int i = 0; i < kDims; i++) acc[i] *= kLoudDown;
        }
        weight[tid] = vrow ? w * (quant_scale(vc) * (loud ? kLoudDown : 1.0f)) : 0.0f;
        row[tid] = vrow;
        __syncthreads();
        const int n = min(256, keys.last - k0 + 1);
#pragma unroll
        for (int i = 0; i < kDims; i++) {
            const int d = dim0 + 256 * i;
            acc[i] *= alpha;
            if (group >= groups || d >= D) continue;
#pragma unroll 4
            for (int j = group; j < n; j += groups)
                if (row[j]) acc[i] = fmaf(weight[j], Quant<FORMAT>::template value<0>(row[j][d]), acc[i]);
        }
    }
    l = wave_sum(l);
    if ((tid & 63) == 0) sums[tid >> 6] = l;
    __syncthreads();
    const double total = sums[0] + sums[1] + sums[2] + sums[3];
    const float inv = total == 0.0 ? 0.0f : 1.0f / static_cast<float>(total);
    const int64_t o0 = b * a.os[0] + h * a.os[1] + t * a.os[2];
    if (groups > 1) {  // one dim a thread
        weight[tid] = acc[0];
        __syncthreads();
        if (group == 0)
            for (int g = 1; g < groups; g++) acc[0] += weight[g * lanes + dim0];
    }
#pragma unroll
    for (int i = 0; i < kDims; i++) {
        const int d = dim0 + 256 * i;
        if (group == 0 && d < D) Vec8<T>::store1(a.out, o0 + d * a.os[3], acc[i] * inv * (loud ? kLoudUp : 1.0f));
    }
}

template <typename T, int FORMAT>
void launch_general(const QuantAttnArgs& a, unsigned wgs, hipStream_t stream) {
    const bool words = a.p.dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.p.pool[0]) % 4 == 0;
    if (words) hipLaunchKernelGGL((quant_attention_general_kernel<T, FORMAT, 4>), dim3(wgs), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((quant_attention_general_kernel<T, FORMAT, 1>), dim3(wgs), dim3(256), 0, stream, a);
}

// Whether a call of these sizes has rows enough for the prompt kernel.
bool is_prompt(const SandyTensor* q, const SandyQuantCache* kc, const SandyTensor* table) {
    return quant_prefill_takes(q->dims[0], q->dims[1], kc->prefix, q->dims[2], kc->inner, table->dims[1], q->dtype == SANDY_F32);
}

size_t workspace_of(const SandyTensor* q, const SandyQuantCache* kc, const SandyTensor* table, int64_t window) {
    const int64_t page = kc->page_size, D = kc->inner;
    if (D % 16 != 0 || D > 256 || page < 16 || numel(*q) == 0) return 0;
    if (is_prompt(q, kc, table)) return 0;
    return quant_decode_workspace(q->dims[0], q->dims[1], kc->prefix, q->dims[2], D, page, table->dims[1], window);
}

int check_quant_attention(const SandyTensor* q, const SandyQuantCache* kc, Err e) {
    if (!valid_rank(q) || !kc) return fail(e, SANDY_ERR_INVALID, "quant_paged attention requires q and caches");
    if (!is_float(q->dtype)) return fail(e, SANDY_ERR_INVALID, "attention q unsupported dtype");
    if (q->rank != 4) return fail(e, SANDY_ERR_INVALID, "quant_paged attention expects q [B, Hq, T, D]");
    if (kc->inner != q->dims[3]) return fail(e, SANDY_ERR_INVALID, "attention head dimension mismatch");
    if (kc->inner > kMaxDim) return fail(e, SANDY_ERR_UNSUPPORTED, "attention head dimension above 512");
    if (kc->prefix <= 0 || q->dims[1] <= 0 || q->dims[1] % kc->prefix != 0)
        return fail(e, SANDY_ERR_INVALID, "attention heads must be divisible by kv_heads");
    if (!quant_sizes_fit(q->dims[0], q->dims[1], q->dims[2], q->dims[3]))
        return fail(e, SANDY_ERR_UNSUPPORTED, "quant_paged batch or row count too large");
    return SANDY_OK;
}

} // namespace
} // namespace sandy_hip

using namespace sandy_hip;

extern "C" int sandy_hip_quant_paged_attention_workspace(const SandyTensor* q, const SandyQuantCache* kc,
                                                         const SandyTensor* table, int64_t window, size_t* bytes,
                                                         char* err, size_t err_cap) {
    Err e{err, err_cap};
    int status = check_quant_attention(q, kc, e);
    if (status) return status;
    if (!valid_rank(table) || table->rank != 2 || !bytes)
        return fail(e, SANDY_ERR_INVALID, "quant_paged attention requires a block table");
    *bytes = workspace_of(q, kc, table, window);
    return ok(e);
}

extern "C" int sandy_hip_quant_paged_attention(const SandyTensor* q, const SandyQuantCache* kc,
                                               const SandyQuantCache* vc, const SandyTensor* table,
                                               const SandyTensor* position_offsets, const SandyTensor* counts,
                                               int64_t window, double scale, const SandyTensor* out, void* workspace,
                                               size_t workspace_bytes, void* stream, char* err, size_t err_cap) {
    Err e{err, err_cap};
    int status = check_quant_attention(q, kc, e);
    if (status) return status;
    if (!vc || !valid_rank(out)) return fail(e, SANDY_ERR_INVALID, "quant_paged attention requires q and caches");
    if (!same_shape(*q, *out) || out->dtype != q->dtype) return fail(e, SANDY_ERR_INVALID, "attention output shape mismatch");
    for (int i = 0; i < 4; i++)
        if (out->dims[i] > 1 && out->strides[i] == 0) return fail(e, SANDY_ERR_INVALID, "attention output rows must not share memory");
    if (window < 0) return fail(e, SANDY_ERR_INVALID, "attention window must be >= 0");
    QuantAttnArgs a{};
    status = check_quant_pages(kc, vc, table, position_offsets, counts, q->dims[0], q->dims[2], e, &a.p);
    if (status) return status;
    if (numel(*q) == 0) return ok(e);
    a.q = base_ptr(*q);
    a.out = base_ptr(*out);
    for (int i = 0; i < 4; i++) {
        a.qs[i] = q->strides[i];
        a.os[i] = out->strides[i];
    }
    a.window = window;
    // rounded once: what it is off by goes into every exponent times its score
    a.scale_log2 = static_cast<float>((scale <= 0.0 ? 1.0 / std::sqrt(static_cast<double>(a.p.dim)) : scale) * 1.4426950408889634074);
    a.hq = static_cast<int32_t>(q->dims[1]);
    a.group = a.hq / a.p.heads;
    a.group_magic = a.group == 1 ? UINT32_MAX : static_cast<uint32_t>((uint64_t{1} << 32) / static_cast<uint32_t>(a.group));
    a.f32 = q->dtype == SANDY_F32;
    const bool tiles = quant_decode_takes(a);
    const size_t need = tiles ? workspace_of(q, kc, table, window) : 0;
    if (workspace_bytes < need || (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)))
        return fail(e, SANDY_ERR_INVALID, "quant_paged attention needs a 16-byte aligned workspace of %zu bytes", need);
    const int64_t wgs = q->dims[0] * q->dims[1] * q->dims[2];
    if (!tiles && wgs > UINT32_MAX / 256) return fail(e, SANDY_ERR_UNSUPPORTED, "quant_paged attention of too many queries");
    a.p.errw = device_error_word(e, &status);
    if (status) return status;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (tiles) {
        if (is_prompt(q, kc, table)) return launch_quant_prefill(a, kc->format, s, e);
        return launch_quant_decode(a, kc->format, workspace, s, e);
    }
    const unsigned n = static_cast<unsigned>(wgs);
    if (kc->format == SANDY_QUANT_INT8) a.f32 ? launch_general<F32, SANDY_QUANT_INT8>(a, n, s) : launch_general<BF16, SANDY_QUANT_INT8>(a, n, s);
    else a.f32 ? launch_general<F32, SANDY_QUANT_E4M3>(a, n, s) : launch_general<BF16, SANDY_QUANT_E4M3>(a, n, s);
    SANDY_HIP_TRY(hipGetLastError(), e, "quant_paged attention launch");
    return ok(e);
}
