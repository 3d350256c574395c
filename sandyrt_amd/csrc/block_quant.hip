// block_quant.hip -- rows and weights into 8 bits and back.  No counterpart in the reference, which keeps
// every operand in the model's type.
//
// A block is 128 columns of one row (activations: every row gets its own range) or of 128 rows (weights).  With
// a its largest magnitude, its scale is the smallest power of two with a / 2^s <= 448, read off a's exponent and
// mantissa bits as the 8-bit K/V cache does, and a payload is rne(x / 2^s): the division is exact, so each value
// is rounded once.  e4m3 is a floating format: a free scale (a / 448) would round no value better, only move
// where its subnormals begin, and the matrix instructions of gfx950 apply powers of two by themselves.
//
// Both directions are memory streams: a thread takes eight elements, sixteen threads a row of a block, whose
// largest magnitude crosses lanes with DPP moves (and LDS for the 128 rows of a weight's block).
#include "block_quant.h"

namespace sandy_hip {
namespace {

struct BlockArgs {
    const void* x;
    void* out;
    uint8_t* payload;
    uint8_t* scales;
    int64_t xs[3];  // element strides of x over (batch, row, column)
    int64_t pitch, batch_pitch;
    int32_t rows, k, blocks, scale_rows, shift;
    uint32_t units;
};

// Columns d .. d + 7 of a row at `at`, those from k on as 0.
template <typename T, bool UNIT>
__device__ __forceinline__ void load_piece(const BlockArgs& a, int64_t at, int d, float (&v)[8]) {
    if (UNIT && d + 8 <= a.k) {
        load8_unaligned<T>(a.x, at + d, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = d + j < a.k ? Vec8<T>::load1(a.x, at + (d + j) * (UNIT ? 1 : a.xs[2])) : 0.0f;
}

__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    return top;
}

// the largest of 16 lanes in each of them
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    auto move = [](uint32_t u, auto ctrl) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(u), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    v = max(v, move(v, std::integral_constant<int, 0xB1>{}));   // lane ^ 1
    v = max(v, move(v, std::integral_constant<int, 0x4E>{}));   // lane ^ 2
    v = max(v, move(v, std::integral_constant<int, 0x141>{}));  // row_half_mirror
    return max(v, move(v, std::integral_constant<int, 0x140>{}));  // row_mirror
}

__device__ __forceinline__ void store_piece(const BlockArgs& a, int64_t at, int d, int code, const float (&v)[8]) {
    using Q = Quant<SANDY_QUANT_E4M3>;
    const float inv = quant_scale(254 - min(code, 253));
    uint2 w = make_uint2(0, 0);
    if (code != 255) {
        w.x = Q::pack(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        w.y = Q::pack(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    }
    uint8_t* to = a.payload + at + d;
    if (d + 8 <= a.k) {
        __builtin_memcpy(to, &w, 8);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (d + j < a.k) to[j] = static_cast<uint8_t>((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
}

// Sixteen threads a block of one row.  4096 x 5632 bf16, 70 MB in all: 13 us a call among others, whose inputs the cache holds
// in part, 13 to 20, 16 on average, where each is waited for, 4.3 TB/s (a large copy's rate: 5.2).
// Rows of another inner stride (UNIT false, here and below) are read element by element: a transposed 4096 x 5632 bf16
// takes 100 us, in blocks of 128 rows 51 for 15, 2999 x 4133 f32 32 for 17.
template <typename T, bool UNIT>
__global__ __launch_bounds__(256) void quant_row_blocks_kernel(BlockArgs a) {
    const uint32_t unit = blockIdx.x * 16u + (threadIdx.x >> 4);
    if (unit >= a.units) return;  // all sixteen
    const uint32_t line = unit / a.blocks;
    const int block = static_cast<int>(unit - line * a.blocks);
    const uint32_t b = line / a.rows, r = line - b * a.rows;
    const int d = block * kQuantBlock + (threadIdx.x & 15) * 8;
    float v[8];
    load_piece<T, UNIT>(a, b * a.xs[0] + r * a.xs[1], d, v);
    const int code = quant_code<SANDY_QUANT_E4M3>(max16(top_of(v)));
    if ((threadIdx.x & 15) == 0) a.scales[unit] = static_cast<uint8_t>(code);
    if (d < a.k) store_piece(a, b * a.batch_pitch + r * a.pitch, d, code, v);
}

// A workgroup a block of 128 rows, held in registers between the maximum and the rounding.  2999 x 4133 f32, 62 MB: 17.3 us,
// 3.6 TB/s: 792 workgroups are one round, which reads, meets and writes.
template <typename T, bool UNIT>
__global__ __launch_bounds__(256) void quant_tile_blocks_kernel(BlockArgs a) {
    const uint32_t unit = blockIdx.x;
    const uint32_t line = unit / a.blocks;
    const int block = static_cast<int>(unit - line * a.blocks);
    const uint32_t b = line / a.scale_rows;
    const int r0 = static_cast<int>(line - b * a.scale_rows) * kQuantBlock + (threadIdx.x >> 4);
    const int d = block * kQuantBlock + (threadIdx.x & 15) * 8;
    float v[8][8];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < 8; u++) {
        const int r = min(r0 + 16 * u, a.rows - 1);  // the last row again changes no maximum
        load_piece<T, UNIT>(a, b * a.xs[0] + r * a.xs[1], d, v[u]);
    }
#pragma unroll
    for (int u = 0; u < 8; u++) top = max(top, top_of(v[u]));
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, 64)));
    __shared__ uint32_t tops[4];
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    const int code = quant_code<SANDY_QUANT_E4M3>(top);
    if (threadIdx.x == 0) a.scales[unit] = static_cast<uint8_t>(code);
    if (d >= a.k) return;
#pragma unroll
    for (int u = 0; u < 8; u++)
        if (r0 + 16 * u < a.rows) store_piece(a, b * a.batch_pitch + static_cast<int64_t>(r0 + 16 * u) * a.pitch, d, code, v[u]);
}

// Eight elements a thread; `units` are the sixteenths of blocks, row by row.  4096 x 5632 to bf16 14 us, 5.0 TB/s;
// 2999 x 4133 to f32 13 us, 4.7 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void block_dequant_kernel(BlockArgs a) {
    const uint32_t unit = blockIdx.x * 16u + (threadIdx.x >> 4);
    if (unit >= a.units) return;
    const uint32_t line = unit / a.blocks;
    const int block = static_cast<int>(unit - line * a.blocks);
    const uint32_t b = line / a.rows, r = line - b * a.rows;
    const int d = block * kQuantBlock + (threadIdx.x & 15) * 8;
    if (d >= a.k) return;
    const uint8_t* from = a.payload + b * a.batch_pitch + r * a.pitch + d;
    const float s = quant_scale(a.scales[(static_cast<int64_t>(b) * a.scale_rows + (r >> a.shift)) * a.blocks + block]);
    const int64_t to = static_cast<int64_t>(line) * a.k + d;
    uint2 w = make_uint2(0, 0);
    const int n = min(8, a.k - d);
    if (n == 8) {
        __builtin_memcpy(&w, from, 8);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < n) (j < 4 ? w.x : w.y) |= static_cast<uint32_t>(from[j]) << (8 * (j & 3));
    }
    float lo[4], hi[4];
    quant_values<SANDY_QUANT_E4M3>(w.x, lo);
    quant_values<SANDY_QUANT_E4M3>(w.y, hi);
    const float v[8] = {lo[0] * s, lo[1] * s, lo[2] * s, lo[3] * s, hi[0] * s, hi[1] * s, hi[2] * s, hi[3] * s};
    if (n == 8) {
        if constexpr (std::is_same_v<T, BF16>) {
            const uint4 o = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                       pack_bf16x2(v[6], v[7]));
            __builtin_memcpy(static_cast<uint16_t*>(a.out) + to, &o, 16);
        } else {
            __builtin_memcpy(static_cast<float*>(a.out) + to, v, 32);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j < n) Vec8<T>::store1(a.out, to + j, v[j]);
}

template <typename T>
int launch_quant(const BlockArgs& a, bool unit_stride, Err e, hipStream_t s) {
    if (a.shift) {
        if (unit_stride) hipLaunchKernelGGL((quant_tile_blocks_kernel<T, true>), dim3(a.units), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((quant_tile_blocks_kernel<T, false>), dim3(a.units), dim3(256), 0, s, a);
    } else {
        const dim3 grid((a.units + 15) / 16);
        if (unit_stride) hipLaunchKernelGGL((quant_row_blocks_kernel<T, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((quant_row_blocks_kernel<T, false>), grid, dim3(256), 0, s, a);
    }
    SANDY_HIP_TRY(hipGetLastError(), e, "block_quant launch");
    return ok(e);
}

BlockArgs block_args(const QuantMat& m) {
    BlockArgs a{};
    a.payload = m.payload;
    a.scales = m.scales;
    a.pitch = m.pitch;
    a.batch_pitch = m.batch_pitch;
    a.rows = static_cast<int32_t>(m.rows);
    a.k = static_cast<int32_t>(m.k);
    a.blocks = static_cast<int32_t>(m.blocks);
    a.scale_rows = static_cast<int32_t>(m.scale_rows);
    a.shift = m.shift;
    return a;
}

} // namespace
} // namespace sandy_hip

using namespace sandy_hip;

extern "C" int sandy_hip_block_quant(const SandyTensor* x, int64_t block_rows, const SandyTensor* payload,
                                     const SandyTensor* scales, void* stream, char* err, size_t err_cap) {
    Err e{err, err_cap};
    if (block_rows != 1 && block_rows != kQuantBlock) return fail(e, SANDY_ERR_INVALID, "block_quant block_rows must be 1 or 128");
    if (!valid_rank(x) || !is_float(x->dtype) || (x->rank != 2 && x->rank != 3))
        return fail(e, SANDY_ERR_INVALID, "block_quant x must be f32 or bf16 of rank 2 or 3");
    QuantMat m;
    if (int status = check_quant_matrix(payload, scales, "block_quant", e, &m)) return status;
    if (!same_shape(*x, *payload)) return fail(e, SANDY_ERR_INVALID, "block_quant payloads must have x's shape");
    const int64_t scale_rows = (m.rows + block_rows - 1) / block_rows;
    if (m.scale_rows != scale_rows) return fail(e, SANDY_ERR_INVALID, "block_quant scales must be [.., ceil(rows / block_rows), ceil(k / 128)]");
    if (numel(*x) == 0) return ok(e);
    if (!x->data) return fail(e, SANDY_ERR_INVALID, "block_quant x is null");
    const int64_t units = m.batch * scale_rows * m.blocks;
    if (units > UINT32_MAX / (block_rows == 1 ? 16 : 256)) return fail(e, SANDY_ERR_UNSUPPORTED, "block_quant of too many blocks");
    BlockArgs a = block_args(m);
    a.x = base_ptr(*x);
    const int r = x->rank;
    a.xs[0] = r == 3 ? x->strides[0] : 0;
    a.xs[1] = x->strides[r - 2];
    a.xs[2] = x->strides[r - 1];
    a.shift = block_rows == 1 ? 0 : 7;
    a.units = static_cast<uint32_t>(units);
    const bool unit_stride = m.k == 1 || a.xs[2] == 1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return x->dtype == SANDY_BF16 ? launch_quant<BF16>(a, unit_stride, e, s) : launch_quant<F32>(a, unit_stride, e, s);
}

extern "C" int sandy_hip_block_dequant(const SandyTensor* payload, const SandyTensor* scales, const SandyTensor* out,
                                       void* stream, char* err, size_t err_cap) {
    Err e{err, err_cap};
    QuantMat m;
    if (int status = check_quant_matrix(payload, scales, "block_dequant", e, &m)) return status;
    if (!valid_rank(out) || !is_float(out->dtype) || !same_shape(*out, *payload) || !contiguous(*out))
        return fail(e, SANDY_ERR_INVALID, "block_dequant out must be contiguous f32 or bf16 of the payloads' shape");
    if (numel(*out) == 0) return ok(e);
    if (!out->data) return fail(e, SANDY_ERR_INVALID, "block_dequant out is null");
    const int64_t units = m.batch * m.rows * m.blocks;
    if (units > UINT32_MAX / 16) return fail(e, SANDY_ERR_UNSUPPORTED, "block_dequant of too many blocks");
    BlockArgs a = block_args(m);
    a.out = base_ptr(*out);
    a.units = static_cast<uint32_t>(units);
    const dim3 grid((a.units + 15) / 16);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (out->dtype == SANDY_BF16) hipLaunchKernelGGL((block_dequant_kernel<BF16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((block_dequant_kernel<F32>), grid, dim3(256), 0, s, a);
    SANDY_HIP_TRY(hipGetLastError(), e, "block_dequant launch");
    return ok(e);
}
