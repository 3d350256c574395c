// sample_parts.h -- parts of whole weights by floats, exactly.  Plain C++ (constexpr functions are the
// device's too), so that they can be checked on the host alone.
#pragma once
#include <cstdint>

namespace sandy_hip {

// p * w rounded up or down; 0 <= p < 1, -0.0 among them: the sign is no part of the exponent
constexpr uint64_t part_of(float p, uint64_t w, bool up) {
    const uint32_t u = __builtin_bit_cast(uint32_t, p), e = u >> 23 & 0xffu, m = e ? (u & 0x7fffffu) | 0x800000u : u & 0x7fffffu;
    const int shift = 150 - static_cast<int>(e ? e : 1);  // p = m * 2^-shift, shift >= 24
    const unsigned __int128 prod = static_cast<unsigned __int128>(m) * w;
    if (shift >= 100) return up && prod != 0 ? 1 : 0;
    const uint64_t q = static_cast<uint64_t>(prod >> shift);
    return q + (up && (prod & ((static_cast<unsigned __int128>(1) << shift) - 1)) != 0 ? 1 : 0);
}

} // namespace sandy_hip
