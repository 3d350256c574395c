// quant_prefill.hip -- attention of many queries a sequence (prompts and prompt
// chunks) over the 8-bit paged cache on v_mfma_f32_32x32x16_bf16.
//
// The rows of a kv head are its (query, head of the group) pairs, query major,
// so a workgroup's 32 CT rows are a few neighbouring queries of the whole group.
// Its four waves take the key pairs of tiles in turn, each by itself (no barrier
// in the loop), and are merged at the end.  As in quant_decode.hip payloads go to
// the matrix unit as they are: S^T = K Q^T straight from 16-byte loads, O^T += V^T
// P^T with V through the wave's own LDS rows and ds_read_b64_tr_b8; K's scale
// multiplies the scores in the multiply-add of their exponents, V's the weights
// (int8) or the conversion (e4m3).  Converted keys serve CT tiles of rows.  bf16
// queries' weights enter as two bf16 numbers (2^-15), f32 queries and weights as
// three (exact).
#include "quant_mfma.h"

#include <algorithm>

namespace sandy_hip {
namespace {

struct PromptArgs {
    QuantAttnArgs a;
    int32_t row_blocks;
};

template <typename T, int FORMAT, int DP, int CT>
struct PromptGeo {
    static constexpr bool kF32 = std::is_same_v<T, F32>;
    static constexpr int KP = DP / 32;  // 16-byte pieces of K a lane holds of a pair of tiles
    static constexpr int VP = DP + 16;  // bytes of a V row in LDS
    static constexpr int NV = DP / 64;  // 16-byte pieces of V a lane holds of a tile
    static constexpr int DT = DP / 32;  // 32-dim tiles of O^T
    static constexpr int kV = 32 * VP;
    static constexpr int kMerge = 4 * CT * 16 * 64 * 4;  // one 32-dim tile of every wave
    static constexpr int kBytes = std::max(4 * kV, kMerge) + 4 * CT * 32 * 8;
    static constexpr int kWaves = DP == 64 ? (CT == 2 || kF32 ? 2 : 3) : DP == 128 && CT == 1 ? 2 : 1;  // a SIMD
};

template <typename T, int FORMAT, int DP, int CT>
__global__ __launch_bounds__(256, (PromptGeo<T, FORMAT, DP, CT>::kWaves)) void quant_prompt_kernel(PromptArgs pa) {
    using G = PromptGeo<T, FORMAT, DP, CT>;
    constexpr bool kF32 = G::kF32;
    constexpr int NQ = kF32 ? 3 : 1, NP = kF32 ? 3 : 2, KS = DP / 16, DT = G::DT;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const QuantAttnArgs& a = pa.a;
    const QuantPages& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int D = p.dim;
    // heads vary fastest (an XCD serves few), the longest row blocks start first
    const int heads = p.batch * p.heads;
    const int bh = static_cast<int>(blockIdx.x) % heads;
    const int rb = pa.row_blocks - 1 - static_cast<int>(blockIdx.x) / heads;
    const int b = bh / p.heads, kh = bh % p.heads;
    const int rows = a.group * p.tokens;
    const int64_t pos = load_index(p.pos, p.pos_dt, b);
    const int count = pos < 0 ? 0 : quant_count(p, b);
    if (pos < 0 && tid == 0) atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_ATTN_POS));
    // the rows' queries, those of the padding aside
    const int r0 = rb * 32 * CT;
    const SeqKeys seq = quant_keys(a, pos);
    const int t_lo = divide(r0, a.group, a.group_magic), t_hi = divide(min(rows - 1, r0 + 32 * CT - 1), a.group, a.group_magic);
    const int t_end = min(t_hi, count - 1);
    const int begin = seq.of(t_lo).first & ~15;
    const int last = t_lo <= t_end ? seq.of(t_end).last : -1;
    const int pairs = last >= begin ? (last - begin + 32) >> 5 : 0;
    // keys that every row sees
    const int all_first = seq.of(t_hi).first;
    const int all_last = t_hi < count ? seq.of(t_lo).last : -1;

    // this lane's rows (past the end: the last one, not stored) and their keys
    int row[CT], qt[CT], qg[CT];
    KeyRange mine[CT];
    // B operands of Q^T: row, dims 32 (s / 2) + 16 half + 8 (s & 1) .. + 7 in step s, zeros past D
    u32x4_t qv[CT][NQ][KS];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        row[c] = r0 + 32 * c + col;
        const int rc = min(row[c], rows - 1);
        qt[c] = divide(rc, a.group, a.group_magic), qg[c] = rc - qt[c] * a.group;
        mine[c] = seq.of(qt[c]);
        if (qt[c] >= count) mine[c].last = -1;
        const int64_t q0 = b * a.qs[0] + (kh * a.group + qg[c]) * a.qs[1] + qt[c] * a.qs[2];
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int d = 32 * (s >> 1) + 16 * half + 8 * (s & 1);
            if constexpr (kF32) {
                float x[8];
                Vec8<F32>::load(a.q, q0 + (d < D ? d : 0), x);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t part[3];
                    split_pair<3>(d < D ? x[2 * i] : 0.0f, d < D ? x[2 * i + 1] : 0.0f, part);
#pragma unroll
                    for (int n = 0; n < 3; n++) qv[c][n][s][i] = part[n];
                }
            } else {
                qv[c][0][s] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.q) + q0 + (d < D ? d : 0));
                if (d >= D) qv[c][0][s] = u32x4_t{0, 0, 0, 0};
            }
        }
    }

    f32x16_t acc[CT][DT];
    float m[CT], l[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        m[c] = -INFINITY;
        l[c] = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[c][t][i] = 0.0f;
    }

    unsigned char* vrows = lds + wave * G::kV;
    int k_off[G::KP], v_to[G::NV];
#pragma unroll
    for (int j = 0; j < G::KP; j++) k_off[j] = (lane & 15) * D + (32 * j + 16 * half < D ? 32 * j + 16 * half : 0);
#pragma unroll
    for (int j = 0; j < G::NV; j++) {
        const int piece = lane + 64 * j, per_row = D / 16;
        const int r = piece / per_row;
        v_to[j] = r < 16 ? r * G::VP + 16 * (piece - r * per_row) : DP;  // none: the padding of the first row
    }
    // ds_read_b64_tr_b8: lanes 2 n and 2 n + 1 of 16 address row n's 16 bytes, lane i
    // gets byte i of the 8 rows: keys 4 half + n and 8 + 4 half + n - 4 of a tile
    const int trow = (lane & 15) >> 1;
    const unsigned char* v_from = vrows + (trow < 4 ? 4 * half + trow : 8 + 4 * half + trow - 4) * G::VP + 16 * ((lane >> 4) & 1) + 8 * (lane & 1);

    // a wave takes every fourth pair, 32 of them (64 tiles) a round: lane i holds
    // tile i & 1 of pair i / 2, its bytes' offset, its rows (none: 0) and factors
    int bytes_in = 0;
    uint64_t offset = 0;
    float kf = 0.0f, vf = 1.0f;
    u32x4_t kr[G::KP], vr[2][G::NV];
    auto load = [&](int n) {
        uint64_t off[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int tile = (2 * n + h) & 63;
            // rows past the last key and tiles without a page: an empty range reads zeros
            const int bytes = n < 32 ? __builtin_amdgcn_readlane(bytes_in, tile) : 0;
            off[h] = static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(offset >> 32), tile)) << 32 |
                     static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(offset), tile));
            const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(p.pool[1] + off[h], 0, bytes, kRsrcWord3);
#pragma unroll
            for (int j = 0; j < G::NV; j++) vr[h][j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rv, 16 * (lane + 64 * j), 0, 0));
        }
        // K: a lane's key is in the first or the second tile (one without a page: page 0's
        // bytes, masked)
        const uint8_t* kp = p.pool[0] + ((lane & 16) ? off[1] : off[0]);
#pragma unroll
        for (int j = 0; j < G::KP; j++) kr[j] = *reinterpret_cast<const u32x4_t*>(kp + k_off[j]);
    };
    auto begin_round = [&](int round0) {
        const int pair = round0 + 4 * (lane >> 1);
        const int key0 = begin + 32 * pair + 16 * (lane & 1);
        const int id = pair < pairs && key0 <= last ? quant_block(p, b, key0 >> p.log2_page) : -1;
        bytes_in = id < 0 ? 0 : min(16, last - key0 + 1) * D;
        const int64_t block = static_cast<int64_t>(max(id, 0)) * p.heads + kh;
        offset = id < 0 ? 0 : static_cast<uint64_t>((block << p.log2_page) + (key0 & ((1 << p.log2_page) - 1))) * D;
        const int kc = p.scales[0][block], vc = p.scales[1][block];
        load(0);
        // a NaN block: NaN scores for whoever sees it, V's own factor aside
        kf = vc == 255 || kc == 255 ? quant_scale(255) : fmaxf(quant_scale(kc) * a.scale_log2, 0x1p-126f);
        vf = quant_scale(vc == 255 ? 127 : vc);
    };
    auto attend = [&](int round0, int n) {
        f32x16_t sc[CT];
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) sc[c][i] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const bf16x8_t ka = payload_operand<FORMAT>(kr[s >> 1][2 * (s & 1)], kr[s >> 1][2 * (s & 1) + 1], 1.0f, 1.0f);
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int i = NQ - 1; i >= 0; i--)
                    sc[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka, __builtin_bit_cast(bf16x8_t, qv[c][i][s]), sc[c], 0, 0, 0);
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < G::NV; j++) *reinterpret_cast<u32x4_t*>(vrows + 16 * h * G::VP + v_to[j]) = vr[h][j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        load(n + 1);
        float f[2], v[2];
        bool none[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f[h] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kf), 2 * n + h));
            v[h] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vf), 2 * n + h));
            none[h] = __builtin_amdgcn_readlane(bytes_in, 2 * n + h) == 0;
        }
        const int k0 = begin + 32 * (round0 + 4 * n);
        // element i: key k0 + 8 (i / 4) + 4 half + i % 4, in the first tile for i < 8
        if ((k0 < all_first) | (k0 + 31 > all_last) | none[0] | none[1] | (f[0] != f[0]) | (f[1] != f[1])) {
            int key0 = k0 + 4 * half;
            asm volatile("" : "+v"(key0));  // keeps the compares out of whole tiles
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const bool nan = f[h] != f[h];
                if (nan) f[h] = 1.0f;  // into the scores themselves
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    const int end = none[h] ? -1 : mine[c].last;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int key = key0 + 16 * h + 8 * (i >> 2) + (i & 3);
                        const float s = nan ? quant_scale(255) : sc[c][8 * h + i];
                        sc[c][8 * h + i] = (key < mine[c].first) | (key > end) ? -INFINITY : s;
                    }
                }
            }
        }
        // V^T operands (dims past D: bytes of earlier tiles, in accumulators that nothing
        // stores), kept where they serve two tiles of rows
        bf16x8_t va[2][DT];
        auto v_operand = [&](int h, int t) {
            const i32x2_t eight = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (i32x2_t __attribute__((address_space(3)))*)((unsigned char __attribute__((address_space(3)))*)(v_from + 16 * h * G::VP + 32 * t)));
            return payload_operand<FORMAT>(static_cast<uint32_t>(eight[0]), static_cast<uint32_t>(eight[1]), v[h], v[h]);
        };
        if constexpr (CT > 1)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int t = 0; t < DT; t++) va[h][t] = v_operand(h, t);
#pragma unroll
        for (int c = 0; c < CT; c++) {
            float top[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                top[h] = sc[c][8 * h];
#pragma unroll
                for (int i = 1; i < 8; i++) top[h] = fmaxf(top[h], sc[c][8 * h + i]);
            }
            float mx = fmaxf(top[0] * f[0], top[1] * f[1]);
            // a row's reference m moves only once its maximum has grown by 2^8
            if (__any(mx > m[c] + 8.0f)) {
                mx = max_xor32(mx);
                const float m_new = fmaxf(m[c], mx);
                const float alpha = m[c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[c] - m_new);
                l[c] *= alpha;
#pragma unroll
                for (int t = 0; t < DT; t++) acc[c][t] *= alpha;
                m[c] = m_new;
            }
            const float shift = m[c] == -INFINITY ? 0.0f : m[c];
            float w[16];
#pragma unroll
            for (int i = 0; i < 16; i++) w[i] = __builtin_amdgcn_exp2f(fmaf(sc[c][i], f[i >> 3], -shift));
            float rs[8];
#pragma unroll
            for (int i = 0; i < 8; i++) rs[i] = w[2 * i] + w[2 * i + 1];
            l[c] += ((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7]));
            if constexpr (FORMAT == SANDY_QUANT_INT8)
#pragma unroll
                for (int i = 0; i < 16; i++) w[i] *= v[i >> 3];
            // contraction slot 8 half + j of step h: this lane's element 8 h + j
#pragma unroll
            for (int h = 0; h < 2; h++) {
                u32x4_t parts[NP];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    uint32_t part[NP];
                    split_pair<NP>(w[8 * h + j], w[8 * h + j + 1], part);
#pragma unroll
                    for (int n2 = 0; n2 < NP; n2++) parts[n2][j / 2] = part[n2];
                }
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    if constexpr (CT == 1) va[h][t] = v_operand(h, t);
#pragma unroll
                    for (int n2 = NP - 1; n2 >= 0; n2--)
                        acc[c][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[h][t], __builtin_bit_cast(bf16x8_t, parts[n2]), acc[c][t], 0, 0, 0);
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    };
    for (int round0 = wave; round0 < pairs; round0 += 4 * 32) {
        begin_round(round0);
        const int n_pairs = min(32, (pairs - round0 + 3) / 4);
        for (int n = 0; n < n_pairs; n++) attend(round0, n);
    }

    // the four waves' maxima and sums, then their accumulators, 32 dims at a time
    float2* ml = reinterpret_cast<float2*>(lds + std::max(4 * G::kV, G::kMerge));  // [wave][CT][32]
    float f[CT], inv[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        l[c] = sum_xor32(l[c]);
        if (half == 0) ml[(wave * CT + c) * 32 + col] = make_float2(m[c], l[c]);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CT; c++) {
        float mm = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) mm = fmaxf(mm, ml[(w * CT + c) * 32 + col].x);
        const float shift = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float2 e = ml[(w * CT + c) * 32 + col];
            total += e.y * __builtin_amdgcn_exp2f(e.x - shift);
        }
        f[c] = __builtin_amdgcn_exp2f(m[c] - shift);
        inv[c] = total == 0.0f ? 0.0f : 1.0f / total;
    }
    float* red = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int t = 0; t < DT; t++) {
        if (t > 0) __syncthreads();
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) red[((wave * CT + c) * 16 + i) * 64 + lane] = acc[c][t][i] * f[c];
        __syncthreads();
        // this wave's elements 4 wave .. + 3: dims 32 t + 8 wave + 4 half + 0 .. 3
        const int d = 32 * t + 8 * wave + 4 * half;
#pragma unroll
        for (int c = 0; c < CT; c++) {
            if (row[c] >= rows || d >= D) continue;
            f32x4_t o;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float* e = red + (c * 16 + 4 * wave + i) * 64 + lane;
                o[i] = ((e[0] + e[CT * 1024]) + (e[2 * CT * 1024] + e[3 * CT * 1024])) * inv[c];
            }
            store4<T>(a.out, b * a.os[0] + (kh * a.group + qg[c]) * a.os[1] + qt[c] * a.os[2] + d, o);
        }
    }
}

template <typename T, int FORMAT, int DP, int CT>
int launch_rows(const QuantAttnArgs& a, hipStream_t stream, Err e) {
    using G = PromptGeo<T, FORMAT, DP, CT>;
    static_assert(G::kBytes <= 64 * 1024, "LDS of a workgroup");
    PromptArgs pa{};
    pa.a = a;
    const int64_t rows = static_cast<int64_t>(a.group) * a.p.tokens;
    pa.row_blocks = static_cast<int32_t>((rows + 32 * CT - 1) / (32 * CT));
    const int64_t wgs = static_cast<int64_t>(pa.row_blocks) * a.p.batch * a.p.heads;
    void* params[] = {&pa};
    SANDY_HIP_TRY(hipLaunchKernel(reinterpret_cast<const void*>(&quant_prompt_kernel<T, FORMAT, DP, CT>),
                                  dim3(static_cast<unsigned>(wgs)), dim3(256), params, G::kBytes, stream), e,
                  "quant_paged attention launch");
    return ok(e);
}

template <typename T, int FORMAT, int DP>
int launch_dim(const QuantAttnArgs& a, hipStream_t stream, Err e) {
    const int64_t rows = static_cast<int64_t>(a.group) * a.p.tokens;
    const int64_t wgs = (rows + 63) / 64 * a.p.batch * a.p.heads;
    const int ct = env_int("SANDY_QUANT_CT", wgs >= 512 ? 2 : 1);
    if constexpr (DP <= 128 && !(DP == 128 && std::is_same_v<T, F32>))
        if (ct == 2) return launch_rows<T, FORMAT, DP, 2>(a, stream, e);
    return launch_rows<T, FORMAT, DP, 1>(a, stream, e);
}

template <typename T, int FORMAT>
int launch_format(const QuantAttnArgs& a, hipStream_t stream, Err e) {
    if (a.p.dim <= 64) return launch_dim<T, FORMAT, 64>(a, stream, e);
    if constexpr (!std::is_same_v<T, F32>)
        if (a.p.dim > 128) return launch_dim<T, FORMAT, 256>(a, stream, e);
    return launch_dim<T, FORMAT, 128>(a, stream, e);
}

} // namespace

bool quant_prefill_takes(int64_t batch, int64_t hq, int64_t heads, int64_t tokens, int64_t dim, int64_t max_blocks, bool f32) {
    const int64_t rows = hq / heads * tokens;
    return tokens > 1 && rows >= env_int("SANDY_QUANT_PREFILL_ROWS", 64) && (!f32 || dim <= 128) && max_blocks > 0 &&
           (rows + 31) / 32 * batch * heads <= UINT32_MAX / 256;
}

int launch_quant_prefill(const QuantAttnArgs& a, int32_t format, hipStream_t stream, Err e) {
    if (format == SANDY_QUANT_INT8)
        return a.f32 ? launch_format<F32, SANDY_QUANT_INT8>(a, stream, e) : launch_format<BF16, SANDY_QUANT_INT8>(a, stream, e);
    return a.f32 ? launch_format<F32, SANDY_QUANT_E4M3>(a, stream, e) : launch_format<BF16, SANDY_QUANT_E4M3>(a, stream, e);
}

} // namespace sandy_hip
