// quant_mfma.h -- what the MFMA kernels over the 8-bit cache share: payloads and
// floats as bf16 operands.
#pragma once
#include <type_traits>

#include "quant_attention.h"

namespace sandy_hip {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef int i32x2_t __attribute__((ext_vector_type(2)));

constexpr int kRsrcWord3 = 0x00020000;  // gfx9 buffer resource word 3: raw dword access

// Four payloads as four bf16, times `scale` (e4m3 only; a power of two).
template <int FORMAT>
__device__ __forceinline__ void payload_bf16(uint32_t w, float scale, uint32_t& lo, uint32_t& hi) {
    if constexpr (FORMAT == SANDY_QUANT_E4M3) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
    } else {  // at most 8 bits: the upper halves of the floats
        float v[4];
        quant_values<FORMAT>(w, v);
        lo = __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x07060302u);
        hi = __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x07060302u);
    }
}

template <int FORMAT>
__device__ __forceinline__ bf16x8_t payload_operand(uint32_t w0, uint32_t w1, float s0, float s1) {
    u32x4_t r;
    uint32_t a, b;
    payload_bf16<FORMAT>(w0, s0, a, b);
    r[0] = a, r[1] = b;
    payload_bf16<FORMAT>(w1, s1, a, b);
    r[2] = a, r[3] = b;
    return __builtin_bit_cast(bf16x8_t, r);
}

// x and y as three bf16 parts each, packed in pairs: 8 of a float's 24 bits a part, so
// that together they are the float (a finite one)
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&part)[3]) {
#pragma unroll
    for (int n = 0; n < 2; n++) {
        const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
        part[n] = __builtin_amdgcn_perm(yb, xb, 0x07060302u);  // the upper halves
        x -= __uint_as_float(xb & 0xffff0000u);
        y -= __uint_as_float(yb & 0xffff0000u);
    }
    part[2] = __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(x), static_cast<__bf16>(y)});
}

template <typename T>
__device__ __forceinline__ void store4(void* p, int64_t at, f32x4_t v) {
    if constexpr (std::is_same_v<T, F32>) *reinterpret_cast<f32x4_t*>(static_cast<float*>(p) + at) = v;
    else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

} // namespace sandy_hip
