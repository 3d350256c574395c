// quant_linear.hip -- products of rows in 8 bits with weights in 8 bits, dense and by expert: entry points
// and the kernel for few rows.  No counterpart in the reference, whose products keep the model's type
// (src/device/cuda/CudaMatMulKernels.cu:173-616).
//
//   y[m, n] = bias[n] + sum over blocks j of 2^(cx[m, j] + cw[n, j] - 254) sum over i in j of px[m, i] pw[n, i]
//
// bf16 outputs: v_mfma_scale_f32_{16x16x128, 32x32x64}_f8f6f4 multiplies its sums by both scale bytes as it adds them
// to f32, so the scales cost an operand and no instruction.  Within eight neighbouring columns it cuts products off
// 13 bits below the largest of them (measured: a product of 2^-13 of its neighbour's counts, one of 2^-14 does not;
// the eights are added in f32).  That is 2^9 below the rounding the operands themselves carry and, over whole
// outputs, 1.5e-5 of their norm for normal values and 5e-5 for random payloads, where rounding to bf16 is 1.7e-3.
// f32 outputs, where that would show, are formed by the bf16 instructions from payloads widened on their way into
// the operands (exact; the conversion applies the scale), at half the rate: 1e-8 to 8e-8.
#include "quant_gemm.h"

#include <algorithm>

namespace sandy_hip {
namespace {

// Few rows: a stream of the weight.  A workgroup takes 16 weight rows, a wave every WAVES-th block of 128 columns; a lane
// loads 32 bytes of its weight row (16 rows of whole 128-byte lines a wave) and of its x row straight into the operand
// registers, DEPTH blocks ahead.  The waves' sums meet in LDS, in their order.  More than 16 rows go round again, the
// weights then coming from L2.
// One row of 28672 x 8192: 52 us, 4.5 TB/s of HBM; of 11264 x 2048 7.2 us, 3.2 TB/s, where a call that does nothing takes 2.
template <typename T, int WAVES, int DEPTH>
__global__ __launch_bounds__(64 * WAVES) void quant_stream_kernel(QuantGemm a) {
    __shared__ float red[WAVES][4][64];
    const int lane = threadIdx.x & 63, row = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int g = blockIdx.y, n0 = static_cast<int>(blockIdx.x) * 16;
    int begin, end;
    quant_group_rows(a, g, &begin, &end);
    if (begin >= end) return;
    const int last = a.blocks - 1, rest = a.k - last * kQuantBlock;  // columns of the last block
    const int n = min(n0 + row, a.n - 1);
    const uint8_t* wp = a.w + g * a.w_group + n * a.w_pitch + 32 * quarter;
    const uint8_t* wsp = a.ws + (static_cast<int64_t>(g) * a.w_scale_rows + (n >> a.w_shift)) * a.blocks;
    // a block's 32 bytes of a row, those past k as 0 (a piece that begins there is not read)
    auto load = [&](const uint8_t* p, int j) -> i32x8_t {
        const uint8_t* at = p + static_cast<int64_t>(j) * kQuantBlock;
        i32x4_t lo, hi;
        if (j < last || rest == kQuantBlock) {
            lo = *reinterpret_cast<const i32x4_t*>(at);
            hi = *reinterpret_cast<const i32x4_t*>(at + 16);
        } else {
            lo = hi = i32x4_t{0, 0, 0, 0};
            const int left = rest - 32 * quarter;
            if (left > 0) lo = *reinterpret_cast<const i32x4_t*>(at);
            if (left > 16) hi = *reinterpret_cast<const i32x4_t*>(at + 16);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                lo[i] &= static_cast<int>(first_bytes(left - 4 * i));
                hi[i] &= static_cast<int>(first_bytes(left - 16 - 4 * i));
            }
        }
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    for (int r0 = begin; r0 < end; r0 += 16) {
        const int r = min(r0 + row, end - 1);
        const uint8_t* xp = a.x + r * a.x_pitch + 32 * quarter;
        const uint8_t* xsp = a.xs + static_cast<int64_t>(r) * a.blocks;
        i32x8_t wf[DEPTH], xf[DEPTH];
        int wsf[DEPTH], xsf[DEPTH];
        auto request = [&](int d, int j) {
            wf[d] = load(wp, j), wsf[d] = wsp[j];
            xf[d] = load(xp, j), xsf[d] = xsp[j];
        };
        f32x4_t acc{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (wave + d * WAVES <= last) request(d, wave + d * WAVES);
        for (int j0 = wave; j0 <= last; j0 += DEPTH * WAVES) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                const int j = j0 + d * WAVES;
                if (j > last) break;
                if constexpr (std::is_same_v<T, BF16>) {
                    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[d], xf[d], acc, 0, 0, 0, wsf[d], 0, xsf[d]);
                } else {
                    const Widened xw = widen(xf[d], quant_scale(xsf[d])), ww = widen(wf[d], quant_scale(wsf[d]));
#pragma unroll
                    for (int s = 0; s < 4; s++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww.v[s], xw.v[s], acc, 0, 0, 0);
                }
                if (j + DEPTH * WAVES <= last) request(d, j + DEPTH * WAVES);
            }
        }
        // acc[i]: x row lane % 16, column 4 (lane / 16) + i
#pragma unroll
        for (int i = 0; i < 4; i++) red[wave][i][lane] = acc[i];
        __syncthreads();
        if (wave == 0) {
            f32x4_t v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < WAVES; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] += red[s][i][lane];
            if (r0 + row < end) store_columns<T>(a, r0 + row, n0 + 4 * quarter, v);
        }
        __syncthreads();
    }
}

// Which kernel, from how many tiles there are for 256 CUs (us, bf16 outputs, rows x columns x k).  One workgroup a CU leaves
// most of it idle, so few tiles are made smaller and their k is split between two groups of waves, or four:
//   64 x 4096 x 4096     32 x 32 split 8.2, 64 x 64 split 11     64 x 1024 x 8192  10.5 against 18    64 x 2048 x 5632  9.1, 14
//   128 x 4096 x 4096    32 x 32 split 10.8, 64 x 64 split 11.2  16 x 11264 x 2048  9.3 against 8.8   64 x 11264 x 2048  14.5, 9.6
//   333 x 1999 x 5617    64 x 64 split 15.8, 64 x 128 whole 26, 128 x 128 whole 34, 256 x 256 84
//   128 x 11264 x 2048   64 x 128 split 11.9, whole 13.5, 64 x 64 split 14
//   1024 x 4096 x 4096   128 x 128 split 23.5, whole 27, 256 x 256 46
// Many tiles: 256 x 256 has half the traffic of 128 x 128, which two a CU come in smaller rounds; 192 x 256 (bf16 outputs,
// for f32's double products it gains nothing) fills rounds that 256 x 256 does not:
//   128 x 128, 192 x 256, 256 x 256    1024 x 11264 x 2048  36, 48, 30      2048 x 11264 x 2048  55, 52, 60
//   4096 x 2560 x 2048   31, 26, 30    8192 x 2816 x 2816   71, 65, 77      4096 x 11264 x 2048  99, 102, 96
//   1500 x 8192 x 4096   61, 47, 50    4096 x 4096 x 4096   70, 81, 57      4096 x 8192 x 8192   266, 237, 204
// A short k, mostly output: 64 x 128, of which there are three a CU (128 x 128, 192 x 256 behind it):
//   4096 x 2560 x 64     8.0, 9.8, 10.7    1000 x 5632 x 256    7.7, 8.1, 12.7    561 x 17025 x 23    15, 21, 31
//   83 x 32000 x 704     11.2, 11.4, 17.5  634 x 11264 x 768    17.7, 13.8, 21.6
// Few rows: the stream of the weight.  Every workgroup reads x for 16 columns, so that more rows and many columns are for tiles:
//   1 x 11264 x 2048     7.2, 64 x 64 split 8.7      16 x 2048 x 2048  5.4, 32 x 32 split 5.9    16 x 8192 x 8192  24 against 16
//   1 x 28672 x 8192     52, 64 x 128 split 62       4 x 16384 x 4096   19 against 17       1 x 32000 x 2048  18.3, 64 x 128 15.2
// Many columns for a row of tiles, split where k is long: 64 x 128 split and whole
//   8 x 65536 x 2048     32 and 28                   8 x 152064 x 4096  116 and 138
// Experts: as if the rows were spread evenly over as many as may have one, but that their unevenness wants room for more
// tiles.  A stream has workgroups for the empty ones as well, which cost it from some thousands on (us, experts x columns x k):
//   2 rows, 8 x 1024 x 4096     stream 6.9, 64 x 64 split 12.4     8 rows, 256 x 2048 x 256    16.7 against 6.7
//   8 rows, 128 x 2816 x 704    stream 18.6, 64 x 128 11           128 rows, 128 x 2816 x 704  58 against 31
//   64 rows, 8 x 14336 x 4096   64 x 128 split 106, whole 116      2 times 64 rows, 8 x 4096 x 1024  split 18.7, whole 13.8
//   64 rows each, 128 x 1408 x 2816 and 2816 x 704   64 x 128 136 and 95, 128 x 128 140 and 97
//   256 rows each, the same     64 x 128 262 and 224, 128 x 128 232 and 196
QuantForm form_of(const QuantGemm& a, bool bf16) {
    const int64_t some = std::min<int64_t>(a.groups, a.rows), rows = (a.rows + some - 1) / some;
    auto tiles = [&](int64_t m, int64_t n) { return (rows + m - 1) / m * some * ((a.n + n - 1) / n); };
    const int64_t least = tiles(64, 64), streams = int64_t{a.groups} * ((a.n + 15) / 16);
    const bool brief = a.blocks <= 6;
    const int64_t alone = least <= 128 ? (brief ? 32 : a.blocks < 64 ? 16 : 4) : least < 256 && brief ? 16 : least < 256 || a.blocks >= 64 ? 4 : 0;
    const int64_t few = !a.offsets ? alone : streams <= 1024 ? (brief ? 16 : 8) : streams <= 4096 ? 2 : 0;
    if (rows <= few) return QuantForm::kStream;
    if (tiles(32, 32) <= (a.blocks >= (bf16 ? 32 : 16) ? 512 : 256)) return QuantForm::k32x32Split;
    if (least <= 256 || a.n <= 64) return QuantForm::k64x64Split;
    if (a.offsets && rows <= 64) return tiles(64, 128) <= 128 || a.blocks >= 32 ? QuantForm::k64x128Split : QuantForm::k64x128;
    if (tiles(64, 128) <= 256 || (rows <= 64 && a.blocks >= 32)) return QuantForm::k64x128Split;
    if (rows <= 64 || a.blocks <= 4 || (a.blocks <= 8 && tiles(128, 128) <= 256)) return QuantForm::k64x128;
    if (tiles(128, 128) <= 256 && a.blocks >= 24) return QuantForm::k128x128Split;
    // rounds, of 512 tiles of 128 x 128 and 256 larger ones, in times of the former (36, 47 and 57 us at k = 4096; 13.5 and 27 at
    // k = 704; f32 outputs 60 and 113 at k = 4096).
    auto rounds = [&](int64_t m, int64_t n, int64_t at_once) { return static_cast<double>((tiles(m, n) + at_once - 1) / at_once); };
    const double small = rounds(128, 128, 512), middle = (1.25 + 2.0 / a.blocks) * rounds(192, 256, 256);
    const double large = ((bf16 ? 1.55 : 1.85) + 3.0 / a.blocks) * rounds(256, 256, 256);
    if (bf16 && middle < std::min(small, large)) return QuantForm::k192x256;
    return large < small ? QuantForm::k256x256 : QuantForm::k128x128;
}

template <typename T>
int launch_products(const QuantGemm& a, const char* what, Err e, hipStream_t s) {
    const QuantForm form = static_cast<QuantForm>(env_int("SANDY_QUANT_FORM", static_cast<int>(form_of(a, std::is_same_v<T, BF16>))));
    if (form != QuantForm::kStream) return launch_quant_tiles(a, std::is_same_v<T, BF16>, form, e, s);
    const dim3 grid(static_cast<unsigned>((a.n + 15) / 16), static_cast<unsigned>(a.groups));
    // eight waves where each still has four blocks (1 x 1024 x 8192: 7.6 us against 11.1; 1 x 11264 x 2048: 8.2 against 7.3)
    if (a.blocks >= 32) hipLaunchKernelGGL((quant_stream_kernel<T, 8, 2>), grid, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((quant_stream_kernel<T, 4, 4>), grid, dim3(256), 0, s, a);
    SANDY_HIP_TRY(hipGetLastError(), e, what);
    return ok(e);
}

// What both products check of their operands; x and out are taken as one run of rows.
int check_products(const SandyTensor* x, const SandyTensor* x_scales, const SandyTensor* w, const SandyTensor* w_scales,
                   const SandyTensor* out, const char* what, Err e, QuantGemm* a) {
    QuantMat xm, wm;
    if (int status = check_quant_matrix(x, x_scales, what, e, &xm)) return status;
    if (int status = check_quant_matrix(w, w_scales, what, e, &wm)) return status;
    if (xm.k <= 0 || wm.k <= 0 || wm.rows <= 0 || wm.batch <= 0) return fail(e, SANDY_ERR_INVALID, "%s expects static positive dimensions", what);
    if (xm.k != wm.k) return fail(e, SANDY_ERR_INVALID, "%s contracting dimension mismatch", what);
    if (xm.shift) return fail(e, SANDY_ERR_INVALID, "%s x must have a scale for every row", what);
    if (!valid_rank(out) || !is_float(out->dtype)) return fail(e, SANDY_ERR_INVALID, "%s out must be f32 or bf16", what);
    const int r = x->rank;
    if (out->rank != r || out->dims[r - 1] != wm.rows) return fail(e, SANDY_ERR_INVALID, "%s output shape mismatch", what);
    for (int i = 0; i + 1 < r; i++)
        if (out->dims[i] != x->dims[i]) return fail(e, SANDY_ERR_INVALID, "%s output shape mismatch", what);
    *a = QuantGemm{};
    const int64_t rows = xm.batch * xm.rows;
    a->rows = static_cast<int32_t>(rows);
    a->groups = static_cast<int32_t>(wm.batch);
    a->n = static_cast<int32_t>(wm.rows);
    a->k = static_cast<int32_t>(xm.k);
    a->blocks = static_cast<int32_t>(xm.blocks);
    if (rows == 0) return SANDY_OK;
    if (rows > (int64_t{1} << 30) || wm.rows > (int64_t{1} << 30)) return fail(e, SANDY_ERR_UNSUPPORTED, "%s of too many rows", what);
    if (!quant_rows_aligned(xm) || !quant_rows_aligned(wm))
        return fail(e, SANDY_ERR_UNSUPPORTED, "%s payload rows must begin on 16-byte boundaries", what);
    // rows of [B, M, ..] as one run: one pitch between all of them
    a->x_pitch = xm.rows > 1 ? xm.pitch : xm.batch > 1 ? xm.batch_pitch : xm.pitch;
    if (xm.batch > 1 && xm.rows > 1 && xm.batch_pitch != xm.rows * xm.pitch)
        return fail(e, SANDY_ERR_UNSUPPORTED, "%s rows of x must be evenly spaced", what);
    const int64_t ro = out->strides[r - 2], bo = r == 3 ? out->strides[0] : 0;
    a->out_pitch = xm.rows > 1 ? ro : xm.batch > 1 ? bo : wm.rows;
    if ((wm.rows > 1 && out->strides[r - 1] != 1) || (rows > 1 && a->out_pitch < wm.rows) ||
        (xm.batch > 1 && xm.rows > 1 && bo != xm.rows * ro))
        return fail(e, SANDY_ERR_UNSUPPORTED, "%s rows of out must have unit inner stride and be evenly spaced", what);
    constexpr int64_t kFar = int64_t{1} << 22;
    if (xm.pitch > kFar || a->x_pitch > kFar || wm.pitch > kFar)
        return fail(e, SANDY_ERR_UNSUPPORTED, "%s payload rows more than 2^22 bytes apart", what);
    if (!out->data) return fail(e, SANDY_ERR_INVALID, "%s out is null", what);
    a->x = xm.payload;
    a->xs = xm.scales;
    a->w = wm.payload;
    a->ws = wm.scales;
    a->w_pitch = wm.pitch;
    a->w_group = wm.batch_pitch;
    a->w_scale_rows = static_cast<int32_t>(wm.scale_rows);
    a->w_shift = wm.shift;
    a->out = base_ptr(*out);
    return SANDY_OK;
}

} // namespace
} // namespace sandy_hip

using namespace sandy_hip;

extern "C" int sandy_hip_quant_linear(const SandyTensor* x, const SandyTensor* x_scales, const SandyTensor* weight,
                                      const SandyTensor* weight_scales, const SandyTensor* bias, const SandyTensor* out,
                                      void* stream, char* err, size_t err_cap) {
    Err e{err, err_cap};
    QuantGemm a;
    if (int status = check_products(x, x_scales, weight, weight_scales, out, "quant_linear", e, &a)) return status;
    if (weight->rank != 2) return fail(e, SANDY_ERR_INVALID, "quant_linear weight must be rank 2");
    if (bias) {
        if (!valid_rank(bias) || bias->dtype != out->dtype || bias->rank != 1 || bias->dims[0] != a.n || !contiguous(*bias) || !bias->data)
            return fail(e, SANDY_ERR_INVALID, "quant_linear bias must be [out_features] of the output's type");
        a.bias = base_ptr(*bias);
    }
    if (a.rows == 0) return ok(e);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return out->dtype == SANDY_BF16 ? launch_products<BF16>(a, "quant_linear launch", e, s) : launch_products<F32>(a, "quant_linear launch", e, s);
}

extern "C" int sandy_hip_quant_moe_matmul(const SandyTensor* x, const SandyTensor* x_scales, const SandyTensor* expert_offsets,
                                          const SandyTensor* weight, const SandyTensor* weight_scales, const SandyTensor* out,
                                          void* stream, char* err, size_t err_cap) {
    Err e{err, err_cap};
    QuantGemm a;
    if (int status = check_products(x, x_scales, weight, weight_scales, out, "quant_moe_matmul", e, &a)) return status;
    if (x->rank != 2 || weight->rank != 3) return fail(e, SANDY_ERR_INVALID, "quant_moe_matmul expects ranks [N,K], [E+1], [E,M,K]");
    if (!valid_rank(expert_offsets) || !is_index(expert_offsets->dtype) || expert_offsets->rank != 1 ||
        expert_offsets->dims[0] != a.groups + int64_t{1} || !contiguous(*expert_offsets) || !expert_offsets->data)
        return fail(e, SANDY_ERR_INVALID, "quant_moe_matmul expert_offsets must be E + 1 contiguous i32 or i64 values");
    if (a.rows == 0) return ok(e);
    if (a.groups > 65535) return fail(e, SANDY_ERR_UNSUPPORTED, "quant_moe_matmul of more than 65535 experts");
    a.offsets = base_ptr(*expert_offsets);
    a.offsets_dt = expert_offsets->dtype;
    int status = 0;
    a.errw = device_error_word(e, &status);
    if (status) return status;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return out->dtype == SANDY_BF16 ? launch_products<BF16>(a, "quant_moe_matmul launch", e, s)
                                    : launch_products<F32>(a, "quant_moe_matmul launch", e, s);
}
