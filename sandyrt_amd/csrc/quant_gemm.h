// quant_gemm.h -- products of two matrices in 8 bits (block_quant.h): what their kernels share.
#pragma once
#include "block_quant.h"

#include <type_traits>

namespace sandy_hip {

// x [rows, k] . w [groups][n, k]^T; rows offsets[g] .. offsets[g + 1] - 1 of x belong to group g (no
// offsets: all rows to the one group).
struct QuantGemm {
    const uint8_t* x;
    const uint8_t* xs;   // [rows, blocks]
    const uint8_t* w;
    const uint8_t* ws;   // [groups, w_scale_rows, blocks]
    const void* offsets; // or null
    const void* bias;    // [n] of out's type, or null
    void* out;           // rows out_pitch elements apart
    uint32_t* errw;
    int64_t x_pitch, w_pitch, w_group, out_pitch;
    int32_t offsets_dt;
    int32_t rows, groups, n, k, blocks, w_scale_rows, w_shift;
};

typedef int32_t i32x8_t __attribute__((ext_vector_type(8)));
typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// 32 payloads as they stand for, in four operands of the bf16 matrix instructions: exact (4 bits), but for values
// below 2^-126.  The conversion applies the scale.
struct Widened {
    bf16x8_t v[4];
};
__device__ __forceinline__ Widened widen(i32x8_t p, float scale) {
    Widened r;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(p[i], scale, false);
        const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(p[i], scale, true);
        r.v[i >> 1][4 * (i & 1)] = lo[0];
        r.v[i >> 1][4 * (i & 1) + 1] = lo[1];
        r.v[i >> 1][4 * (i & 1) + 2] = hi[0];
        r.v[i >> 1][4 * (i & 1) + 3] = hi[1];
    }
    return r;
}

// Rows of group g, or none where its offsets are out of order (recorded).
__device__ __forceinline__ void quant_group_rows(const QuantGemm& a, int g, int* begin, int* end) {
    *begin = 0;
    *end = a.rows;
    if (!a.offsets) return;
    const int64_t b = load_index(a.offsets, a.offsets_dt, g), e = load_index(a.offsets, a.offsets_dt, g + 1);
    if (b < 0 || e < b || e > a.rows) {
        if (threadIdx.x == 0) atomicOr(a.errw, static_cast<uint32_t>(SANDY_DEVERR_OFFSETS));
        *end = 0;
        return;
    }
    *begin = static_cast<int>(b);
    *end = static_cast<int>(e);
}

// The kernel for few rows (quant_linear.hip), or that for many (quant_tile.h) in one of its tile forms.
enum class QuantForm { kStream, k32x32Split, k64x64Split, k64x128Split, k128x128Split, k64x128, k128x128, k192x256, k256x256 };
int launch_quant_tiles(const QuantGemm& a, bool bf16, QuantForm form, Err e, hipStream_t s);

// The bits of a dword that hold the first n bytes.
__device__ __forceinline__ uint32_t first_bytes(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u; }

// Four neighbouring columns c .. c + 3 of an output row, those from n on left out.
template <typename T>
__device__ __forceinline__ void store_columns(const QuantGemm& a, int64_t row, int c, f32x4_t v) {
    if (a.bias) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] += Vec8<T>::load1(a.bias, min(c + i, a.n - 1));
    }
    const int64_t to = row * a.out_pitch + c;
    if (c + 4 <= a.n && (a.out_pitch & 3) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0) {
        if constexpr (std::is_same_v<T, BF16>)
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + to) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        else
            *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + to) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (c + i < a.n) Vec8<T>::store1(a.out, to + i, v[i]);
}

} // namespace sandy_hip
