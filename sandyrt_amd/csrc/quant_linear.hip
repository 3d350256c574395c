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

// Few rows: a stream of the weight.  A workgroup takes 16 NW weight rows and every WAVES-th block of 128 columns
// per wave; a lane loads 32 bytes of its weight row (16 rows of whole 128-byte lines a wave) and of its x
// row straight into the operand registers, DEPTH blocks ahead.  The waves' sums meet in LDS, in their order.
// More than 16 RT rows go round again, the weights then coming from L2.
template <typename T, int RT, int NW, int WAVES, int DEPTH>
__global__ __launch_bounds__(64 * WAVES) void quant_stream_kernel(QuantGemm a) {
    constexpr bool kScaled = std::is_same_v<T, BF16>;
    __shared__ float red[WAVES][RT * NW][4][64];
    const int lane = threadIdx.x & 63, row = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int g = blockIdx.y, n0 = static_cast<int>(blockIdx.x) * 16 * NW;
    int begin, end;
    quant_group_rows(a, g, &begin, &end);
    if (begin >= end) return;
    const int last = a.blocks - 1, rest = a.k - last * kQuantBlock;  // columns of the last block
    const uint8_t* wp[NW];
    const uint8_t* wsp[NW];
#pragma unroll
    for (int c = 0; c < NW; c++) {
        const int n = min(n0 + 16 * c + row, a.n - 1);
        wp[c] = a.w + g * a.w_group + n * a.w_pitch + 32 * quarter;
        wsp[c] = a.ws + (static_cast<int64_t>(g) * a.w_scale_rows + (n >> a.w_shift)) * a.blocks;
    }
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
    for (int r0 = begin; r0 < end; r0 += 16 * RT) {
        const uint8_t* xp[RT];
        const uint8_t* xsp[RT];
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int r = min(r0 + 16 * t + row, end - 1);
            xp[t] = a.x + r * a.x_pitch + 32 * quarter;
            xsp[t] = a.xs + static_cast<int64_t>(r) * a.blocks;
        }
        i32x8_t wf[DEPTH][NW], xf[DEPTH][RT];
        int wsf[DEPTH][NW], xsf[DEPTH][RT];
        auto request = [&](int d, int j) {
#pragma unroll
            for (int c = 0; c < NW; c++) wf[d][c] = load(wp[c], j), wsf[d][c] = wsp[c][j];
#pragma unroll
            for (int t = 0; t < RT; t++) xf[d][t] = load(xp[t], j), xsf[d][t] = xsp[t][j];
        };
        f32x4_t acc[RT][NW];
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int c = 0; c < NW; c++) acc[t][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (wave + d * WAVES <= last) request(d, wave + d * WAVES);
        for (int j0 = wave; j0 <= last; j0 += DEPTH * WAVES) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                const int j = j0 + d * WAVES;
                if (j > last) break;
#pragma unroll
                for (int c = 0; c < NW; c++)
#pragma unroll
                    for (int t = 0; t < RT && kScaled; t++)
                        acc[t][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[d][c], xf[d][t], acc[t][c], 0, 0, 0, wsf[d][c],
                                                                                    0, xsf[d][t]);
                if constexpr (!kScaled) {
                    Widened xw[RT];
#pragma unroll
                    for (int t = 0; t < RT; t++) xw[t] = widen(xf[d][t], quant_scale(xsf[d][t]));
#pragma unroll
                    for (int c = 0; c < NW; c++) {
                        const Widened ww = widen(wf[d][c], quant_scale(wsf[d][c]));
#pragma unroll
                        for (int s = 0; s < 4; s++)
#pragma unroll
                            for (int t = 0; t < RT; t++)
                                acc[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww.v[s], xw[t].v[s], acc[t][c], 0, 0, 0);
                    }
                }
                if (j + DEPTH * WAVES <= last) request(d, j + DEPTH * WAVES);
            }
        }
        // acc[t][c][i]: x row 16 t + lane % 16, column 16 c + 4 (lane / 16) + i
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int c = 0; c < NW; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) red[wave][t * NW + c][i][lane] = acc[t][c][i];
        __syncthreads();
        for (int q = wave; q < RT * NW; q += WAVES) {
            const int t = q / NW, c = q % NW;
            f32x4_t v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < WAVES; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] += red[s][q][i][lane];
            const int r = r0 + 16 * t + row;
            if (r < end) store_columns<T>(a, r, n0 + 16 * c + 4 * quarter, v);
        }
        __syncthreads();
    }
}

template <typename T>
int launch_products(const QuantGemm& a, const char* what, Err e, hipStream_t s) {
    const int64_t rows = a.offsets ? (a.rows + a.groups - 1) / a.groups : a.rows;
    auto grid = [&](int nw) { return dim3(static_cast<unsigned>((a.n + 16 * nw - 1) / (16 * nw)), static_cast<unsigned>(a.groups)); };
    auto tiles = [&](int64_t edge) { return (rows + edge - 1) / edge * a.groups * ((a.n + edge - 1) / edge); };
    const int form = env_int("SANDY_QUANT_TILE", rows <= 32 ? -1 : tiles(256) >= 512 && !a.offsets ? 0 : tiles(128) >= 256 ? 2 : 3);
    if (form >= 0) return launch_quant_tiles(a, std::is_same_v<T, BF16>, form, e, s);
    if (rows <= 16) hipLaunchKernelGGL((quant_stream_kernel<T, 1, 1, 4, 4>), grid(1), dim3(256), 0, s, a);
    else if (rows <= 32) hipLaunchKernelGGL((quant_stream_kernel<T, 2, 2, 4, 2>), grid(2), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((quant_stream_kernel<T, 4, 2, 4, 2>), grid(2), dim3(256), 0, s, a);
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
