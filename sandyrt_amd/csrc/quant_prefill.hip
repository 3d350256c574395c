// quant_prefill.hip -- attention of many queries a sequence (prompts and prompt
// chunks) over the 8-bit paged cache on v_mfma_f32_32x32x16_bf16.
//
// The rows of a kv head are its (query, head of the group) pairs, query major,
// so a workgroup's 32 rows are a few neighbouring queries of the whole group.  Its
// four waves take the pairs of key tiles in turn, each by itself (no barrier in the
// loop), and are merged at the end.  As in quant_decode.hip payloads go to
// the matrix unit as they are: S^T = K Q^T straight from 16-byte loads, O^T += V^T
// P^T with V through the wave's own LDS rows and ds_read_b64_tr_b8; K's scale
// multiplies the scores in the multiply-add of their exponents, V's the weights
// (int8) or the conversion (e4m3).  f32 queries and all weights enter as three bf16
// numbers (exact).
//
// 2048 queries of 32 / 4 heads of 64 (e4m3, causal) take 48 to 54 us, 318 to 358 TFLOP/s;
// int8 62 where e4m3 takes 54 (three instructions convert two payloads, one of e4m3's),
// f32 68.  No single unit bounds it: vector instructions issue in 65 % of the cycles, MFMA
// in 27 %.  bf16 queries' weights in two parts took 40 to 49 us, but kept 16 of 24 bits;
// beside those, other layouts were slower: K in LDS tiles for several waves (52 to 57),
// two row tiles a wave (D 128 34 against 20), the keys split over workgroups (69 against 45).
#include "quant_mfma.h"

#include <algorithm>

namespace sandy_hip {
namespace {

struct PromptArgs {
    QuantAttnArgs a;
    int32_t row_blocks;  // workgroups of a kv head
};

constexpr int kRows = 32;  // of a workgroup

template <typename T, int FORMAT, int DP>
struct PromptGeo {
    static constexpr bool kF32 = std::is_same_v<T, F32>;
    static constexpr int KP = DP / 32;  // 16-byte pieces of K a lane holds of a pair of tiles
    static constexpr int VP = DP + 16;  // bytes of a V row in LDS
    static constexpr int NV = DP / 64;  // 16-byte pieces of V a lane holds of a tile
    static constexpr int DT = DP / 32;  // 32-dim tiles of O^T
    static constexpr int kV = 32 * VP;
    static constexpr int kMerge = 4 * 16 * 64 * 4;  // one 32-dim tile of every wave
    static constexpr int NQ = kF32 ? 3 : 1, KS = DP / 16;
    // Q in LDS, once for the four waves: two waves a SIMD then hold the rest in their 256
    // registers (3000 queries of 8 / 2 heads: 87 us, with Q in one wave's 512 114)
    static constexpr bool kQLds = DP == 256;
    static constexpr int kQ = kQLds ? NQ * KS * 64 * 16 : 0;
    static constexpr int kBytes = std::max(4 * kV, kMerge) + 4 * 32 * 8 + kQ;
    static constexpr int kWaves = DP == 64 ? (kF32 ? 3 : 4) : 2;  // a SIMD
};

// Workgroup i's place in the list by falling length: every second round of the
// 256 CUs backwards, so that the workgroups a CU gets add up to about the same (1024
// queries 19.2 us so and 22.3 in order, 8 chunks of 300 of D 128 behind 100 to 2000 keys
// 62 and 69, 4 of 700 without a context 39 and 37).
__device__ __forceinline__ uint32_t snake(uint32_t i, uint32_t n) {
    const uint32_t round = i & ~255u;
    return (i & 256) ? round + min(256u, n - round) - 1 - (i - round) : i;
}

// EXACT: the head dim is DP itself, so that K's addresses are one and constants (D 256:
// registers again)
template <typename T, int FORMAT, int DP, bool EXACT>
__global__ __launch_bounds__(256, (PromptGeo<T, FORMAT, DP>::kWaves)) void quant_prompt_kernel(PromptArgs pa) {
    using G = PromptGeo<T, FORMAT, DP>;
    constexpr bool kF32 = G::kF32;
    constexpr int NQ = G::NQ, KS = G::KS, DT = G::DT;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const QuantAttnArgs& a = pa.a;
    const QuantPages& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int D = EXACT ? DP : p.dim;
    // heads vary fastest (an XCD serves few), the longest row blocks come first
    uint32_t at = snake(blockIdx.x, gridDim.x);
    const int kh = at % p.heads;
    at /= p.heads;
    const int b = at % p.batch;
    const int rows = a.group * p.tokens;
    const int r0 = kRows * (pa.row_blocks - 1 - static_cast<int>(at / p.batch));
    const int64_t pos = load_index(p.pos, p.pos_dt, b);
    const int count = pos < 0 ? 0 : quant_count(p, b);
    if (pos < 0 && tid == 0) atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_ATTN_POS));
    const SeqKeys seq = quant_keys(a, pos);
    // the rows' queries, those of the padding aside, and their keys
    const int t_lo = divide(r0, a.group, a.group_magic), t_hi = divide(min(rows - 1, r0 + 31), a.group, a.group_magic);
    const int begin = seq.of(t_lo).first & ~15;
    const int last = t_lo < count ? seq.of(min(t_hi, count - 1)).last : -1;
    const int pairs = last >= begin ? (last - begin + 32) >> 5 : 0;
    // keys that every row sees
    const int all_first = seq.of(t_hi).first;
    const int all_last = t_hi < count ? seq.of(t_lo).last : -1;

    // this lane's row (past the end: the last one, not stored) and its keys
    const int row = min(r0 + col, rows - 1);
    const int qt = divide(row, a.group, a.group_magic), qg = row - qt * a.group;
    KeyRange mine = seq.of(qt);
    if (qt >= count) mine.last = -1;
    // B operands of Q^T: row, dims 32 (s / 2) + 16 half + 8 (s & 1) .. + 7 in step s, zeros past D
    u32x4_t qv[G::kQLds ? 1 : NQ][G::kQLds ? 1 : KS];
    u32x4_t* q_lds = reinterpret_cast<u32x4_t*>(lds + G::kBytes - G::kQ);  // [NQ][KS][lane]
    const int64_t q0 = b * a.qs[0] + (kh * a.group + qg) * a.qs[1] + qt * a.qs[2];
    auto query = [&](int s, u32x4_t (&v)[NQ]) {
        const int d = 32 * (s >> 1) + 16 * half + 8 * (s & 1);
        if constexpr (kF32) {
            float x[8];
            Vec8<F32>::load(a.q, q0 + (d < D ? d : 0), x);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t part[3];
                split_pair(d < D ? x[2 * i] : 0.0f, d < D ? x[2 * i + 1] : 0.0f, part);
#pragma unroll
                for (int n = 0; n < 3; n++) v[n][i] = part[n];
            }
        } else {
            v[0] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.q) + q0 + (d < D ? d : 0));
            if (d >= D) v[0] = u32x4_t{0, 0, 0, 0};
        }
    };
    if constexpr (G::kQLds) {  // the same for the four waves: each fetches a quarter
#pragma unroll
        for (int s = 0; s < KS / 4; s++) {
            u32x4_t v[NQ];
            query(4 * s + wave, v);
#pragma unroll
            for (int n = 0; n < NQ; n++) q_lds[(n * KS + 4 * s + wave) * 64 + lane] = v[n];
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int s = 0; s < KS; s++) {
            u32x4_t v[NQ];
            query(s, v);
#pragma unroll
            for (int n = 0; n < NQ; n++) qv[n][s] = v[n];
        }
    }

    f32x16_t acc[DT];
    float m = -INFINITY, l = 0.0f;
    bool loud = false;  // the same for the wave
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[t][i] = 0.0f;

    unsigned char* vrows = lds + wave * G::kV;
    int k_off[G::KP], v_to[G::NV];
#pragma unroll
    for (int j = 0; j < G::KP; j++) k_off[j] = EXACT || 32 * j + 16 * half < D ? 32 * j : -16 * half;
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
    uint64_t odd = 0;  // the tiles without a page, that are NaN, or that make the sums loud
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
        const uint8_t* kp = p.pool[0] + ((lane & 16) ? off[1] : off[0]) + ((lane & 15) * D + 16 * half);
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
        // a NaN block: NaN scores for whoever sees it, V's own factor aside (and none is 0,
        // which would make masked scores NaN)
        kf = quant_scale(vc == 255 ? 255 : kc) * a.scale_log2;
        if (kf == 0.0f) kf = 0x1p-149f;
        vf = quant_scale(vc == 255 || id < 0 ? 127 : vc);
        if (loud) vf = fmaxf(vf * kLoudDown, 0x1p-126f);
        odd = __ballot((id < 0) | (kf != kf) | (__float_as_uint(vf) >= kLoudBits));
    };
    // before such a block's values first enter the sums
    auto get_loud = [&]() {
        loud = true;
        vf = fmaxf(vf * kLoudDown, 0x1p-126f);
#pragma unroll
        for (int t = 0; t < DT; t++) acc[t] *= kLoudDown;
    };
    auto attend = [&](int round0, int n) {
        f32x16_t sc;
#pragma unroll
        for (int i = 0; i < 16; i++) sc[i] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const bf16x8_t ka = payload_operand<FORMAT>(kr[s >> 1][2 * (s & 1)], kr[s >> 1][2 * (s & 1) + 1], 1.0f, 1.0f);
#pragma unroll
            for (int i = NQ - 1; i >= 0; i--) {
                u32x4_t qi;
                if constexpr (G::kQLds) qi = q_lds[(i * KS + s) * 64 + lane];
                else qi = qv[i][s];
                sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka, __builtin_bit_cast(bf16x8_t, qi), sc, 0, 0, 0);
            }
            // int8's conversions all at once would not leave registers for two waves (1500 queries 42 us, 59)
            if (DP == 256 && s % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < G::NV; j++) *reinterpret_cast<u32x4_t*>(vrows + 16 * h * G::VP + v_to[j]) = vr[h][j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        load(n + 1);
        float f[2];
        uint32_t v[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f[h] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kf), 2 * n + h));
            v[h] = __builtin_amdgcn_readlane(__float_as_uint(vf), 2 * n + h);
        }
        const int k0 = begin + 32 * (round0 + 4 * n);
        // element i: key k0 + 8 (i / 4) + 4 half + i % 4, in the first tile for i < 8
        if ((k0 < all_first) | (k0 + 31 > all_last) | ((odd >> (2 * n) & 3) != 0)) {
            if (max(v[0], v[1]) >= kLoudBits) {
                get_loud();
#pragma unroll
                for (int h = 0; h < 2; h++) v[h] = __builtin_amdgcn_readlane(__float_as_uint(vf), 2 * n + h);
            }
            int key0 = k0 + 4 * half;
            asm volatile("" : "+v"(key0));  // keeps the compares out of whole tiles
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const bool nan = f[h] != f[h];
                if (nan) f[h] = 1.0f;  // into the scores themselves
                const int end = __builtin_amdgcn_readlane(bytes_in, 2 * n + h) == 0 ? -1 : mine.last;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = key0 + 16 * h + 8 * (i >> 2) + (i & 3);
                    const float s = nan ? quant_scale(255) : sc[8 * h + i];
                    sc[8 * h + i] = (key < mine.first) | (key > end) ? -INFINITY : s;
                }
            }
        }
        float top[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            top[h] = sc[8 * h];
#pragma unroll
            for (int i = 1; i < 8; i++) top[h] = fmaxf(top[h], sc[8 * h + i]);
        }
        float mx = fmaxf(top[0] * f[0], top[1] * f[1]);
        // a row's reference m moves only once its maximum has grown by 2^8
        if (__any(mx > m + 8.0f)) {
            mx = max_xor32(mx);
            const float m_new = fmaxf(m, mx);
            const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
            l *= alpha;
#pragma unroll
            for (int t = 0; t < DT; t++) acc[t] *= alpha;
            m = m_new;
        }
        const float shift = m == -INFINITY ? 0.0f : m;
        float w[16];
#pragma unroll
        for (int i = 0; i < 16; i++) w[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], f[i >> 3], -shift));
        float rs[8];
#pragma unroll
        for (int i = 0; i < 8; i++) rs[i] = w[2 * i] + w[2 * i + 1];
        l += ((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7]));
        if constexpr (FORMAT == SANDY_QUANT_INT8)
#pragma unroll
            for (int i = 0; i < 16; i++) w[i] *= __uint_as_float(v[i >> 3]);
        // contraction slot 8 half + j of step h: this lane's element 8 h + j (dims past D:
        // bytes of earlier tiles, in accumulators that nothing stores)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            u32x4_t parts[3];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                uint32_t part[3];
                split_pair(w[8 * h + j], w[8 * h + j + 1], part);
#pragma unroll
                for (int i = 0; i < 3; i++) parts[i][j / 2] = part[i];
            }
#pragma unroll
            for (int t = 0; t < DT; t++) {
                const i32x2_t eight = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (i32x2_t __attribute__((address_space(3)))*)((unsigned char __attribute__((address_space(3)))*)(v_from + 16 * h * G::VP + 32 * t)));
                const bf16x8_t va = payload_operand<FORMAT>(static_cast<uint32_t>(eight[0]), static_cast<uint32_t>(eight[1]), __uint_as_float(v[h]), __uint_as_float(v[h]));
#pragma unroll
                for (int i = 2; i >= 0; i--)
                    acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, __builtin_bit_cast(bf16x8_t, parts[i]), acc[t], 0, 0, 0);
                if (DP == 256 && t % 4 == 3) __builtin_amdgcn_sched_barrier(0);
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
    float2* ml = reinterpret_cast<float2*>(lds + std::max(4 * G::kV, G::kMerge));  // [wave][32]
    l = sum_xor32(l);
    if (half == 0) ml[wave * 32 + col] = make_float2(m, mark_loud(l, loud));
    __syncthreads();
    float mm = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) mm = fmaxf(mm, ml[w * 32 + col].x);
    const float shift = mm == -INFINITY ? 0.0f : mm;
    bool any_loud = false;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float2 e = ml[w * 32 + col];
        total += fabsf(e.y) * __builtin_amdgcn_exp2f(e.x - shift);
        any_loud |= is_loud(e.y);
    }
    const float down = any_loud && !loud ? kLoudDown : 1.0f, up = any_loud ? kLoudUp : 1.0f;
    const float f = __builtin_amdgcn_exp2f(m - shift);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int64_t o0 = b * a.os[0] + (kh * a.group + qg) * a.os[1] + qt * a.os[2] + 4 * half;
    f32x4_t* red = reinterpret_cast<f32x4_t*>(lds);  // [wave][4][64]: elements 4 i .. + 3
#pragma unroll
    for (int t = 0; t < DT; t++) {
        if (t > 0) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++)
            red[(wave * 4 + i) * 64 + lane] = f32x4_t{acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]} * down * f;
        __syncthreads();
        // this wave's elements 4 wave .. + 3: dims 32 t + 8 wave + 4 half + 0 .. 3
        const int d = 32 * t + 8 * wave;
        if (r0 + col >= rows || d >= D) continue;
        const f32x4_t o = (red[wave * 64 + lane] + red[(4 + wave) * 64 + lane]) + (red[(8 + wave) * 64 + lane] + red[(12 + wave) * 64 + lane]);
        store4<T>(a.out, o0 + d, o * inv * up);
    }
}

template <typename T, int FORMAT, int DP>
int launch_dim(const QuantAttnArgs& a, hipStream_t stream, Err e) {
    using G = PromptGeo<T, FORMAT, DP>;
    static_assert(G::kBytes <= 64 * 1024, "LDS of a workgroup");
    PromptArgs pa{};
    pa.a = a;
    pa.row_blocks = static_cast<int32_t>((static_cast<int64_t>(a.group) * a.p.tokens + kRows - 1) / kRows);
    const int64_t wgs = static_cast<int64_t>(pa.row_blocks) * a.p.batch * a.p.heads;
    void* params[] = {&pa};
    const void* kernel = a.p.dim == DP ? reinterpret_cast<const void*>(&quant_prompt_kernel<T, FORMAT, DP, true>)
                                       : reinterpret_cast<const void*>(&quant_prompt_kernel<T, FORMAT, DP, false>);
    SANDY_HIP_TRY(hipLaunchKernel(kernel, dim3(static_cast<unsigned>(wgs)), dim3(256), params, G::kBytes, stream), e,
                  "quant_paged attention launch");
    return ok(e);
}

template <typename T, int FORMAT>
int launch_format(const QuantAttnArgs& a, hipStream_t stream, Err e) {
    if (a.p.dim <= 64) return launch_dim<T, FORMAT, 64>(a, stream, e);
    if constexpr (!std::is_same_v<T, F32>)
        if (a.p.dim > 128) return launch_dim<T, FORMAT, 256>(a, stream, e);
    return launch_dim<T, FORMAT, 128>(a, stream, e);
}

} // namespace

// Rows for more than one 16-row tile, and about a workgroup a CU; fewer leave the chip to
// those tiles, which fill with half the rows and split their keys.  us, 16-row tiles / here:
// - one sequence, no / 1000 / 4000 keys before the chunk, by the number of workgroups: D 64
//   192 6.4 / 6.6, 14.7 / 13.4, 28.9 / 32.9, 256 6.7 / 6.8, 16.0 / 14.2, 35.6 / 34.7; D 128
//   160 8.9 / 9.6, 20.8 / 18.5, 48.1 / 43.2, 192 9.7 / 9.7, 21.1 / 18.7, 47.7 / 42.9; D 256
//   192 19.7 / 21.8, 38.8 / 37.4, 84 / 80, 256 23.3 / 24.6, 41.7 / 40.7, 105 / 89; f32 D 128
//   192 10.7 / 12.0, 23.1 / 24.0, 55 / 58, 256 12.5 / 13.6, 24.7 / 25.7, 68 / 61.
// - batches of mixed contexts of 500 to 8000 keys, where one sequence's workgroups take longest:
//   D 64 of 32 rows 192 50.7 / 76.5, 384 84 / 98, 768 172 / 131; D 128 of 32 to 64 rows 192
//   76 to 93 / 89 to 91, 384 138 to 162 / 107 to 109; D 256 192 140 / 147, 384 254 / 201.
// - the same of 16 rows: D 64 192 34 / 58, 384 57 / 82, 768 97 / 116; D 128 384 99 to 108 / 98 to
//   103, 768 171 to 202 / 200 to 210; D 256 768 371 / 406.  Short contexts: 8.1 / 8.8, 9.5 / 11.1.
bool quant_prefill_takes(int64_t batch, int64_t hq, int64_t heads, int64_t tokens, int64_t dim, int64_t max_blocks, bool f32) {
    const int64_t rows = hq / heads * tokens, wgs = (rows + kRows - 1) / kRows * batch * heads;
    if (tokens < 2 || (f32 && dim > 128) || max_blocks == 0) return false;
    const int forced = env_int("SANDY_QUANT_PROMPT_WGS", 0);
    if (forced > 0) return wgs >= forced;
    return rows > 16 && wgs >= (dim > 64 && dim <= 128 && !f32 ? 192 : 256);
}

int launch_quant_prefill(const QuantAttnArgs& a, int32_t format, hipStream_t stream, Err e) {
    if (format == SANDY_QUANT_INT8)
        return a.f32 ? launch_format<F32, SANDY_QUANT_INT8>(a, stream, e) : launch_format<BF16, SANDY_QUANT_INT8>(a, stream, e);
    return a.f32 ? launch_format<F32, SANDY_QUANT_E4M3>(a, stream, e) : launch_format<BF16, SANDY_QUANT_E4M3>(a, stream, e);
}

} // namespace sandy_hip
