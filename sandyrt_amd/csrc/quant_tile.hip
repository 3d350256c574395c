// quant_tile.hip -- launches of the kernel for many rows of the products of matrices in 8 bits.
#include "quant_tile.h"

namespace sandy_hip {

namespace {

template <typename T, int WM, int WN, int PN, int STAGES>
int launch(const QuantGemm& a, Err e, hipStream_t s) {
    using G = QuantTile<WM, WN, PN, STAGES>;
    constexpr int kBytes = G::template lds<T>();
    // row tiles: those of the experts are not known here, at most one more each than their rows fill
    const int64_t m = (a.rows + G::BM - 1) / G::BM + (a.offsets ? a.groups - 1 : 0), n = (a.n + G::BN - 1) / G::BN;
    if (m * n > (int64_t{1} << 28)) return fail(e, SANDY_ERR_UNSUPPORTED, "quant product of too many tiles");
    const auto kernel = quant_tile_kernel<T, WM, WN, PN, STAGES>;
    SANDY_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kBytes), e, "quant tile");
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((m * n + 7) / 8 * 8)), dim3(G::kThreads), kBytes, s, a, static_cast<int>(m), static_cast<int>(n));
    SANDY_HIP_TRY(hipGetLastError(), e, "quant tile launch");
    return ok(e);
}

} // namespace

int launch_quant_tiles(const QuantGemm& a, bool bf16, int form, Err e, hipStream_t s) {
    if (bf16) {
        switch (form) {
            case 0: return launch<BF16, 4, 4, 2, 2>(a, e, s);
            case 1: return launch<BF16, 2, 2, 2, 4>(a, e, s);
            case 2: return launch<BF16, 2, 2, 2, 2>(a, e, s);
            case 3: return launch<BF16, 1, 1, 2, 4>(a, e, s);
            case 4: return launch<BF16, 4, 2, 2, 2>(a, e, s);
            case 6: return launch<BF16, 4, 2, 4, 2>(a, e, s);
            case 7: return launch<BF16, 2, 2, 4, 2>(a, e, s);
            default: return launch<BF16, 1, 2, 2, 4>(a, e, s);
        }
    }
    switch (form) {
        case 0: return launch<F32, 4, 4, 2, 2>(a, e, s);
        case 3: return launch<F32, 1, 1, 2, 4>(a, e, s);
        default: return launch<F32, 2, 2, 2, 2>(a, e, s);
    }
}

} // namespace sandy_hip
