// quant_cache.hip -- writing the 8-bit paged K/V cache (quantised as rows
// arrive) and reading it back.  The reference keeps pages in the model's type
// (src/device/cuda/CudaPagedTensor.cpp:187-226, 345-447); page layout and block
// tables are the same here.
//
// A block (one page of one head) has one scale, a power of two c chosen from
// the largest magnitude a: the smallest with a / c <= 127 (448 for e4m3), read
// off a's exponent and mantissa bits.  Appending to a block that has rows takes
// c' = max(c, c_new) and, where c' > c, rounds the rows there again:
// q' = rne(q c / c').  The factors are powers of two, so a payload's error after
// any number of such steps is at most 1/2 + 1/4 + 1/8 + ... < 1 final step.  A
// free scale (a / 127) would give up to one bit more and cost that: each growth
// re-rounds by another half step, and bf16 no longer holds the values.
//
// Both directions are memory streams: 8 sequences of 4096 rows of 8 heads of 128, K
// and V (201 MB with 16-bit rows), are written in 41.5 us (4.8 TB/s) and read back in
// 29.6 us (6.8 TB/s, the writes left part of them in the 256 MB cache); 172 MB of mixed
// contexts are read in 29.5 us.  Single rows are a chain of memory latencies (position,
// block table, scale or payload): 3.4 us a step of one sequence, 3.7 of 64, a read of
// 100 rows 3.1 us.
#include "quant_cache.h"

#include <algorithm>
#include <type_traits>

namespace sandy_hip {

int check_quant_pages(const SandyQuantCache* kc, const SandyQuantCache* vc, const SandyTensor* table,
                      const SandyTensor* pos, const SandyTensor* counts, int64_t batch, int64_t tokens, Err e,
                      QuantPages* p) {
    if (!kc || !valid_rank(table) || !valid_rank(pos) || (counts && !valid_rank(counts)))
        return fail(e, SANDY_ERR_INVALID, "quant_paged requires a cache, a block table and positions");
    for (const SandyQuantCache* c : {kc, vc}) {
        if (!c) continue;
        if (c->format != SANDY_QUANT_INT8 && c->format != SANDY_QUANT_E4M3)
            return fail(e, SANDY_ERR_INVALID, "quant_paged cache format must be int8 or e4m3");
        if (c->page_size <= 0 || (c->page_size & (c->page_size - 1)) != 0)
            return fail(e, SANDY_ERR_INVALID, "paged tensor pool page_size must be a power of two");
        if (c->prefix <= 0 || c->inner <= 0 || c->num_pages <= 0)
            return fail(e, SANDY_ERR_INVALID, "quant_paged cache must have pages, heads and a head dim");
        if (!c->pool || !c->scales) return fail(e, SANDY_ERR_INVALID, "quant_paged cache pool or scales is null");
        if (c->page_size > (int64_t{1} << 30) || c->inner > (int64_t{1} << 30) || c->prefix > (int64_t{1} << 30) ||
            c->page_size * c->inner > (int64_t{1} << 30) || c->num_pages > INT32_MAX ||
            c->num_pages * c->prefix > INT64_MAX / (c->page_size * c->inner))
            return fail(e, SANDY_ERR_UNSUPPORTED, "quant_paged page of one head above 2^30 elements, or too many pages");
    }
    if (vc && (vc->format != kc->format || vc->page_size != kc->page_size || vc->prefix != kc->prefix ||
               vc->inner != kc->inner || vc->num_pages != kc->num_pages))
        return fail(e, SANDY_ERR_INVALID, "quant_paged k and v caches must have the same format and shape");
    if (table->dtype != SANDY_I32 || table->rank != 2 || table->dims[0] != batch ||
        (table->dims[1] > 1 && table->strides[1] != 1))
        return fail(e, SANDY_ERR_INVALID, "quant_paged block table must be [B, max_blocks] int32 with unit inner stride");
    if (!is_index(pos->dtype) || numel(*pos) != batch || !contiguous(*pos))
        return fail(e, SANDY_ERR_INVALID, "quant_paged position_offsets must be B contiguous i32 or i64 values");
    if (counts && (!is_index(counts->dtype) || numel(*counts) != batch || !contiguous(*counts)))
        return fail(e, SANDY_ERR_INVALID, "quant_paged counts must be B contiguous i32 or i64 values");
    if (table->dims[1] > (int64_t{1} << 30) || table->dims[1] * kc->page_size > (int64_t{1} << 30))
        return fail(e, SANDY_ERR_UNSUPPORTED, "quant_paged block table covers more than 2^30 rows");
    if (!quant_sizes_fit(batch, kc->prefix, tokens, kc->inner))
        return fail(e, SANDY_ERR_UNSUPPORTED, "quant_paged batch or row count too large");
    *p = QuantPages{};
    p->pool[0] = static_cast<uint8_t*>(kc->pool);
    p->scales[0] = static_cast<uint8_t*>(kc->scales);
    if (vc) {
        p->pool[1] = static_cast<uint8_t*>(vc->pool);
        p->scales[1] = static_cast<uint8_t*>(vc->scales);
    }
    p->table = static_cast<const int32_t*>(base_ptr(*table));
    p->table_stride = table->strides[0];
    p->num_pages = kc->num_pages;
    p->pos = base_ptr(*pos);
    p->pos_dt = pos->dtype;
    p->counts = counts ? base_ptr(*counts) : nullptr;
    p->counts_dt = counts ? counts->dtype : SANDY_I64;
    p->batch = static_cast<int32_t>(batch);
    p->heads = static_cast<int32_t>(kc->prefix);
    p->dim = static_cast<int32_t>(kc->inner);
    p->max_blocks = static_cast<int32_t>(table->dims[1]);
    p->log2_page = __builtin_ctzll(static_cast<uint64_t>(kc->page_size));
    p->tokens = static_cast<int32_t>(tokens);
    return SANDY_OK;
}

namespace {

struct AppendArgs {
    QuantPages p;
    const void* x[2];
    int64_t xs[2][4];  // element strides over (b, h, t, d)
    int32_t ordinals;  // pages a sequence's rows can touch
};

// A workgroup per (sequence, touched page, head) and cache.  N elements a piece:
// 8 where rows of x and of the pool allow 16- and 8-byte accesses, else 1.  The
// first kHeld pieces of a thread stay in registers between the maximum and the
// rounding; a block with more reads the others twice.  A block is what one maximum
// and one scale are for, so nothing crosses workgroups and one launch does all.
template <typename T, int FORMAT, int N, int THREADS>
__global__ __launch_bounds__(THREADS) void quant_append_kernel(AppendArgs a) {
    constexpr int kHeld = 4;
    const QuantPages& p = a.p;
    const int tid = threadIdx.x;
    uint32_t at = blockIdx.x;
    const int h = at % p.heads;
    at /= p.heads;
    const int ord = at % a.ordinals;
    at /= a.ordinals;
    const int b = at % p.batch;
    const int c = at / p.batch;
    const int page_rows = 1 << p.log2_page;
    const int64_t pos = load_index(p.pos, p.pos_dt, b);
    const int count = quant_count(p, b);
    if (count == 0) return;
    if (pos < 0 || pos > (static_cast<int64_t>(p.max_blocks) << p.log2_page) - count) {
        if (tid == 0) atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_QUANT_ROWS));
        return;
    }
    const int page = static_cast<int>(pos >> p.log2_page) + ord;
    const int64_t begin = static_cast<int64_t>(page) << p.log2_page;
    // rows r0 .. r1 - 1 of the page are new, rows before them were there
    const int r0 = static_cast<int>(max<int64_t>(pos - begin, 0));
    const int r1 = static_cast<int>(min<int64_t>(pos + count - begin, page_rows));
    if (r0 >= r1) return;
    const int per_row = p.dim / N;
    const int pieces = (r1 - r0) * per_row;
    const int64_t t0 = begin + r0 - pos;
    const int64_t x0 = b * a.xs[c][0] + h * a.xs[c][1] + t0 * a.xs[c][2];
    auto from = [&](int i) -> int64_t {
        const int r = i / per_row, d = (i - r * per_row) * N;
        return x0 + r * a.xs[c][2] + d * a.xs[c][3];
    };
    auto load = [&](int i, float (&v)[N]) {
        if constexpr (N == 8) Vec8<T>::load(a.x[c], from(i), v);
        else v[0] = Vec8<T>::load1(a.x[c], from(i));
    };
    // the first pieces are on their way, unconverted, while the block table and the
    // scale are read (past the last: the last again, which changes no maximum)
    std::conditional_t<N == 8, typename Vec8<T>::raw, float> held[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; u++) {
        if (u > 0 && u * THREADS >= pieces) break;  // the same for every thread
        const int64_t at = from(min(tid + u * THREADS, pieces - 1));
        if constexpr (N == 8) held[u] = Vec8<T>::load_raw_nt(a.x[c], at);
        else held[u] = Vec8<T>::load1(a.x[c], at);
    }
    auto value = [&](int u, float (&v)[N]) {
        if constexpr (N == 8) Vec8<T>::unpack(held[u], v);
        else v[0] = held[u];
    };
    const int id = quant_block(p, b, page);
    if (id < 0) return;
    const int64_t block = static_cast<int64_t>(id) * p.heads + h;
    uint8_t* scale_at = p.scales[c] + block;
    uint8_t* out = p.pool[c] + (block << p.log2_page) * p.dim;
    const int was = r0 > 0 ? *scale_at : 0;
    uint32_t top = 0;
    auto see = [&](const float (&v)[N]) {
#pragma unroll
        for (int j = 0; j < N; j++) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    };
#pragma unroll
    for (int u = 0; u < kHeld; u++) {
        if (u > 0 && u * THREADS >= pieces) break;
        float v[N];
        value(u, v);
        see(v);
    }
    for (int i = tid + kHeld * THREADS; i < pieces; i += THREADS) {
        float v[N];
        load(i, v);
        see(v);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, 64)));
    if constexpr (THREADS > 64) {
        __shared__ uint32_t tops[THREADS / 64];
        if ((tid & 63) == 0) tops[tid >> 6] = top;
        __syncthreads();  // also: every thread has read the scale before it is written
#pragma unroll
        for (int w = 0; w < THREADS / 64; w++) top = max(top, tops[w]);
    }
    const int code = max(quant_code<FORMAT>(top), was);
    if (tid == 0) *scale_at = static_cast<uint8_t>(code);
    const float inv = quant_scale(254 - min(code, 254));
    auto put = [&](int i, const float (&v)[N]) {
        if constexpr (N == 8) {
            uint2 w = make_uint2(0, 0);
            if (code != 255) {
                w.x = Quant<FORMAT>::pack(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                w.y = Quant<FORMAT>::pack(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
            }
            *reinterpret_cast<uint2*>(out + static_cast<int64_t>(r0) * p.dim + static_cast<int64_t>(i) * 8) = w;
        } else {
            out[static_cast<int64_t>(r0) * p.dim + i] =
                code == 255 ? 0 : static_cast<uint8_t>(Quant<FORMAT>::pack(v[0] * inv, 0.0f, 0.0f, 0.0f));
        }
    };
#pragma unroll
    for (int u = 0; u < kHeld; u++)
        if (tid + u * THREADS < pieces) {
            float v[N];
            value(u, v);
            put(tid + u * THREADS, v);
        }
    for (int i = tid + kHeld * THREADS; i < pieces; i += THREADS) {
        float v[N];
        load(i, v);
        put(i, v);
    }
    if (r0 > 0 && code > was && code != 255) {
        // rows that were there: below 2^-126 a factor leaves nothing of a payload
        const float f = quant_scale(max(127 + was - code, 1));
        for (int i = tid; i < r0 * per_row; i += THREADS) {
            if constexpr (N == 8) {
                uint2* q = reinterpret_cast<uint2*>(out) + i;
                float lo[4], hi[4];
                quant_values<FORMAT>(q->x, lo);
                quant_values<FORMAT>(q->y, hi);
                *q = make_uint2(Quant<FORMAT>::pack(lo[0] * f, lo[1] * f, lo[2] * f, lo[3] * f),
                                Quant<FORMAT>::pack(hi[0] * f, hi[1] * f, hi[2] * f, hi[3] * f));
            } else {
                out[i] = static_cast<uint8_t>(
                    Quant<FORMAT>::pack(Quant<FORMAT>::template value<0>(out[i]) * f, 0.0f, 0.0f, 0.0f));
            }
        }
    }
}

struct ReadArgs {
    QuantPages p;
    void* out[2];
    int32_t chunks;  // workgroups per (cache, sequence, head)
};

// A piece is N elements of a row (8, or 1 where rows are no multiples of 8 bytes);
// a thread takes U of them, 256 apart, each step of the chain block table ->
// payload and scale -> store for all of them at once.
template <typename T, int FORMAT, int N, int U>
__global__ __launch_bounds__(256) void quant_read_kernel(ReadArgs a) {
    const QuantPages& p = a.p;
    uint32_t at = blockIdx.x;
    const int chunk = at % a.chunks;
    at /= a.chunks;
    const int h = at % p.heads;
    at /= p.heads;
    const int b = at % p.batch;
    const int c = at / p.batch;
    const int per_row = p.dim / N;
    const int64_t total = static_cast<int64_t>(p.tokens) * per_row;
    const int64_t first = static_cast<int64_t>(chunk) * 256 * U + threadIdx.x;
    const int64_t pos = load_index(p.pos, p.pos_dt, b);
    const int count = quant_count(p, b);
    const int64_t cap = static_cast<int64_t>(p.max_blocks) << p.log2_page;
    bool there[U];
    int64_t row[U];
    int id[U], d[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t i = min(first + 256 * u, total - 1);
        const int t = static_cast<int>(i / per_row);
        d[u] = static_cast<int>(i - static_cast<int64_t>(t) * per_row) * N;
        row[u] = pos + t;
        there[u] = t < count;
        if (there[u] && (row[u] < 0 || row[u] >= cap)) {
            atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_QUANT_ROWS));
            there[u] = false;
        }
        id[u] = there[u] ? p.table[b * p.table_stride + (row[u] >> p.log2_page)] : 0;
    }
    uint2 w[U];
    int code[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (id[u] < 0 || id[u] >= p.num_pages) {
            atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_BLOCK));
            there[u] = false;
        }
        const int64_t block = static_cast<int64_t>(there[u] ? id[u] : 0) * p.heads + h;
        const uint8_t* from = p.pool[c] + ((block << p.log2_page) + (there[u] ? row[u] & ((1 << p.log2_page) - 1) : 0)) * p.dim + d[u];
        code[u] = p.scales[c][block];
        if constexpr (N == 8) w[u] = *reinterpret_cast<const uint2*>(from);
        else w[u].x = *from;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        if (!there[u]) w[u] = make_uint2(0, 0), code[u] = 0;
    const int64_t to = (static_cast<int64_t>(b) * p.heads + h) * p.tokens * p.dim;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t i = first + 256 * u;
        if (i >= total) continue;
        const float s = quant_scale(code[u]);
        float lo[4], hi[4];
        quant_values<FORMAT>(w[u].x, lo);
        if constexpr (N == 8) {
            quant_values<FORMAT>(w[u].y, hi);
            const float v[8] = {lo[0] * s, lo[1] * s, lo[2] * s, lo[3] * s, hi[0] * s, hi[1] * s, hi[2] * s, hi[3] * s};
            Vec8<T>::store(a.out[c], to + i * 8, v);
        } else {
            Vec8<T>::store1(a.out[c], to + i, lo[0] * s);
        }
    }
}

bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T, int FORMAT>
int launch_append(const AppendArgs& a, int64_t wgs, bool vec, bool small, Err e, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(wgs));
    if (!vec) hipLaunchKernelGGL((quant_append_kernel<T, FORMAT, 1, 256>), grid, dim3(256), 0, stream, a);
    else if (small) hipLaunchKernelGGL((quant_append_kernel<T, FORMAT, 8, 64>), grid, dim3(64), 0, stream, a);
    else hipLaunchKernelGGL((quant_append_kernel<T, FORMAT, 8, 256>), grid, dim3(256), 0, stream, a);
    SANDY_HIP_TRY(hipGetLastError(), e, "quant_paged append launch");
    return ok(e);
}

template <typename T, int FORMAT>
int launch_read(const ReadArgs& a, int64_t wgs, int pieces, bool vec, Err e, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(wgs));
    if (!vec) hipLaunchKernelGGL((quant_read_kernel<T, FORMAT, 1, 1>), grid, dim3(256), 0, stream, a);
    else if (pieces == 1) hipLaunchKernelGGL((quant_read_kernel<T, FORMAT, 8, 1>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((quant_read_kernel<T, FORMAT, 8, 4>), grid, dim3(256), 0, stream, a);
    SANDY_HIP_TRY(hipGetLastError(), e, "quant_paged read launch");
    return ok(e);
}

} // namespace
} // namespace sandy_hip

using namespace sandy_hip;

extern "C" int sandy_hip_quant_paged_append(const SandyTensor* k, const SandyTensor* v, const SandyQuantCache* kc,
                                            const SandyQuantCache* vc, const SandyTensor* table,
                                            const SandyTensor* position_offsets, const SandyTensor* counts,
                                            void* stream, char* err, size_t err_cap) {
    Err e{err, err_cap};
    if (!valid_rank(k) || (v && !valid_rank(v)) || !kc || !v != !vc)
        return fail(e, SANDY_ERR_INVALID, "quant_paged append takes k with its cache, and v and its cache or neither");
    if (k->rank != 4 || !is_float(k->dtype)) return fail(e, SANDY_ERR_INVALID, "quant_paged append rows must be [B, heads, T, D] f32 or bf16");
    if (v && (!same_shape(*k, *v) || v->dtype != k->dtype))
        return fail(e, SANDY_ERR_INVALID, "quant_paged append k and v must have the same shape and dtype");
    AppendArgs a{};
    int status = check_quant_pages(kc, vc, table, position_offsets, counts, k->dims[0], k->dims[2], e, &a.p);
    if (status) return status;
    if (k->dims[1] != kc->prefix || k->dims[3] != kc->inner)
        return fail(e, SANDY_ERR_INVALID, "quant_paged append rows must have the cache's heads and head dim");
    auto overlap = [](const void* x, const void* y, int64_t bytes) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
        return (a < b ? b - a : a - b) < static_cast<uintptr_t>(bytes);
    };
    const int64_t blocks = kc->num_pages * kc->prefix;
    if (vc && (overlap(kc->pool, vc->pool, blocks * kc->page_size * kc->inner) || overlap(kc->scales, vc->scales, blocks)))
        return fail(e, SANDY_ERR_INVALID, "quant_paged append k and v caches must not share memory");
    if (numel(*k) == 0) return ok(e);
    a.p.errw = device_error_word(e, &status);
    if (status) return status;
    bool vec = a.p.dim % 8 == 0;
    for (int c = 0; c < (v ? 2 : 1); c++) {
        const SandyTensor& x = c ? *v : *k;
        a.x[c] = base_ptr(x);
        int64_t all = 0;
        for (int i = 0; i < 4; i++) {
            a.xs[c][i] = x.strides[i];
            if (i < 3 && x.dims[i] > 1) all |= x.strides[i];
        }
        vec = vec && x.strides[3] == 1 && aligned_to(a.x[c], 16) && all % (x.dtype == SANDY_BF16 ? 8 : 4) == 0 &&
              aligned_to(a.p.pool[c], 8);
    }
    const int64_t page = int64_t{1} << a.p.log2_page;
    const int64_t ordinals = (a.p.tokens + page - 2) / page + 1;
    const int64_t wgs = ordinals * a.p.heads * a.p.batch * (v ? 2 : 1);
    // a wave for a block of up to 256 pieces (all held in its registers), else four: with
    // the reads after them, 128 pieces 13.1 us so and 16.3 by four waves, 512 pieces 75.2
    // by four and 85.7 by one
    const bool small = vec && std::min<int64_t>(a.p.tokens, page) * a.p.dim <= 256 * 8;
    if (wgs > UINT32_MAX / (small ? 64 : 256)) return fail(e, SANDY_ERR_UNSUPPORTED, "quant_paged append of too many blocks");
    a.ordinals = static_cast<int32_t>(ordinals);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (k->dtype == SANDY_BF16)
        return kc->format == SANDY_QUANT_INT8 ? launch_append<BF16, SANDY_QUANT_INT8>(a, wgs, vec, small, e, s)
                                              : launch_append<BF16, SANDY_QUANT_E4M3>(a, wgs, vec, small, e, s);
    return kc->format == SANDY_QUANT_INT8 ? launch_append<F32, SANDY_QUANT_INT8>(a, wgs, vec, small, e, s)
                                          : launch_append<F32, SANDY_QUANT_E4M3>(a, wgs, vec, small, e, s);
}

extern "C" int sandy_hip_quant_paged_read(const SandyQuantCache* kc, const SandyQuantCache* vc,
                                          const SandyTensor* table, const SandyTensor* position_offsets,
                                          const SandyTensor* counts, const SandyTensor* k_out,
                                          const SandyTensor* v_out, void* stream, char* err, size_t err_cap) {
    Err e{err, err_cap};
    if (!valid_rank(k_out) || (v_out && !valid_rank(v_out)) || !kc || !v_out != !vc)
        return fail(e, SANDY_ERR_INVALID, "quant_paged read takes a cache with its output, and v's or neither");
    if (k_out->rank != 4 || !is_float(k_out->dtype) || !contiguous(*k_out) || (v_out && !contiguous(*v_out)))
        return fail(e, SANDY_ERR_INVALID, "quant_paged read outputs must be contiguous [B, heads, T, D] f32 or bf16");
    if (v_out && (!same_shape(*k_out, *v_out) || v_out->dtype != k_out->dtype))
        return fail(e, SANDY_ERR_INVALID, "quant_paged read k and v outputs must have the same shape and dtype");
    ReadArgs a{};
    int status = check_quant_pages(kc, vc, table, position_offsets, counts, k_out->dims[0], k_out->dims[2], e, &a.p);
    if (status) return status;
    if (k_out->dims[1] != kc->prefix || k_out->dims[3] != kc->inner)
        return fail(e, SANDY_ERR_INVALID, "quant_paged read outputs must have the cache's heads and head dim");
    if (numel(*k_out) == 0) return ok(e);
    a.p.errw = device_error_word(e, &status);
    if (status) return status;
    bool vec = a.p.dim % 8 == 0;
    for (int c = 0; c < (v_out ? 2 : 1); c++) {
        a.out[c] = base_ptr(c ? *v_out : *k_out);
        vec = vec && aligned_to(a.out[c], 16) && aligned_to(a.p.pool[c], 8);
    }
    // four pieces a thread once that leaves 8 workgroups a CU: 270 MB 43.9 -> 32.1 us;
    // 0.2 MB 3.4 us with one, 6.1 with four
    const int64_t per_head = static_cast<int64_t>(a.p.tokens) * (a.p.dim / (vec ? 8 : 1));
    const int64_t units = static_cast<int64_t>(a.p.heads) * a.p.batch * (v_out ? 2 : 1);
    const int pieces = vec && (per_head + 1023) / 1024 * units >= 2048 ? 4 : 1;
    const int64_t chunks = (per_head + 256 * pieces - 1) / (256 * pieces);
    const int64_t wgs = chunks * units;
    if (wgs * 256 > UINT32_MAX) return fail(e, SANDY_ERR_UNSUPPORTED, "quant_paged read of too many rows");
    a.chunks = static_cast<int32_t>(chunks);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (k_out->dtype == SANDY_BF16)
        return kc->format == SANDY_QUANT_INT8 ? launch_read<BF16, SANDY_QUANT_INT8>(a, wgs, pieces, vec, e, s)
                                              : launch_read<BF16, SANDY_QUANT_E4M3>(a, wgs, pieces, vec, e, s);
    return kc->format == SANDY_QUANT_INT8 ? launch_read<F32, SANDY_QUANT_INT8>(a, wgs, pieces, vec, e, s)
                                          : launch_read<F32, SANDY_QUANT_E4M3>(a, wgs, pieces, vec, e, s);
}
