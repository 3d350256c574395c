// quant_tile.hip -- launches of the kernel for many rows of the products of matrices in 8 bits.
#include "quant_tile.h"

#include <algorithm>

namespace sandy_hip {

namespace {

template <typename T, int WM, int WN, int PM, int PN, int STAGES, int SPLIT>
int launch(const QuantGemm& a, Err e, hipStream_t s) {
    using G = QuantTile<WM, WN, PM, PN, STAGES, SPLIT>;
    constexpr int kBytes = G::template lds<T>();
    // row tiles: of the experts, not known here, at most one each that has a row and one more for every BM further rows
    const int64_t some = std::min<int64_t>(a.rows, a.groups), n = (a.n + G::BN - 1) / G::BN;
    const int64_t m = a.offsets ? some + (a.rows - some) / G::BM : (a.rows + G::BM - 1) / G::BM;
    if (m * n + 7 > UINT32_MAX / (SPLIT * G::kThreads)) return fail(e, SANDY_ERR_UNSUPPORTED, "quant product of too many tiles");
    const uint64_t row_bytes = static_cast<uint64_t>(a.out_pitch) * sizeof(typename Vec8<T>::elem);
    const auto kernel = ((reinterpret_cast<uintptr_t>(a.out) | row_bytes) & 15) == 0 ? quant_tile_kernel<T, true, WM, WN, PM, PN, STAGES, SPLIT>
                                                                                    : quant_tile_kernel<T, false, WM, WN, PM, PN, STAGES, SPLIT>;
    SANDY_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kBytes), e, "quant tile");
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((m * n + 7) / 8 * 8)), dim3(SPLIT * G::kThreads), kBytes, s, a, static_cast<int>(m), static_cast<int>(n));
    SANDY_HIP_TRY(hipGetLastError(), e, "quant tile launch");
    return ok(e);
}

template <typename T>
int launch(const QuantGemm& a, QuantForm form, Err e, hipStream_t s) {
    switch (form) {
        case QuantForm::k32x32Split: return launch<T, 1, 1, 1, 1, 2, 4>(a, e, s);
        case QuantForm::k64x64Split: return launch<T, 1, 1, 2, 2, 2, 2>(a, e, s);
        case QuantForm::k64x128Split: return launch<T, 1, 2, 2, 2, 2, 2>(a, e, s);
        case QuantForm::k128x128Split: return launch<T, 2, 2, 2, 2, 2, 2>(a, e, s);
        case QuantForm::k64x128: return launch<T, 1, 2, 2, 2, 2, 1>(a, e, s);
        case QuantForm::k128x128: return launch<T, 2, 2, 2, 2, 2, 1>(a, e, s);
        case QuantForm::k192x256:
            if constexpr (std::is_same_v<T, BF16>) return launch<T, 3, 4, 2, 2, 2, 1>(a, e, s);
            [[fallthrough]];
        default: return launch<T, 4, 4, 2, 2, 2, 1>(a, e, s);
    }
}

} // namespace

int launch_quant_tiles(const QuantGemm& a, bool bf16, QuantForm form, Err e, hipStream_t s) {
    return bf16 ? launch<BF16>(a, form, e, s) : launch<F32>(a, form, e, s);
}

} // namespace sandy_hip
