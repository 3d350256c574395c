// quant_prefill.hip -- attention of many queries a sequence (prompts and prompt
// chunks) over the 8-bit paged cache on v_mfma_f32_32x32x16_bf16.
//
// The rows of a kv head are its (query, head of the group) pairs, query major,
// so a workgroup's rows are a few neighbouring queries of the whole group.
// S^T = K Q^T (a lane holds the scores of one row), O^T += V^T P^T with P^T as it
// leaves the softmax.  Payloads become bf16 (exactly) once a workgroup, on their
// way into LDS; scales never touch them: with K's factor f (scale log2(e) times
// the block's) and V's scale 2^e, a weight enters as 2^(s f - m + e), which costs
// the multiply-add that the exponent takes anyway, and the row sum takes the
// block's partial sum times 2^-e.  bf16 queries' weights enter as two bf16
// numbers (2^-15), f32 queries and weights as three (exact).
// A table in LDS holds the blocks' byte offsets and factors, read from the block
// table and scales once (a segment of kTable pages at a time): a chunk's loads
// depend on LDS alone.
// Four waves a workgroup: RW of them own 32 rows each, KW = 4 / RW share the keys
// of a chunk and are merged at the end; at D 256 twice as many, each with half of
// the head dims of O.
#include "quant_attention.h"

#include <algorithm>
#include <type_traits>

namespace sandy_hip {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTable = 512;              // pages of a segment
constexpr uint32_t kNoPage = 0xffffffffu;  // upper half of the offset of a page that is not there

struct PrefillQArgs {
    QuantAttnArgs a;
    int32_t row_blocks;
    int32_t table;  // entries of the LDS table: pages of a segment
};

template <typename T, int FORMAT, int DP, int RW>
struct QGeo {
    static constexpr bool kF32 = std::is_same_v<T, F32>;
    static constexpr int DS = DP == 256 ? 2 : 1;
    static constexpr int THREADS = 256 * DS;
    static constexpr int DT = DP / 32 / DS;  // 32-dim tiles of O^T a wave owns
    static constexpr int KW = 4 / RW;
    static constexpr int SUB = RW == 4 ? 2 : 1;  // 32-key blocks of a chunk a wave takes
    static constexpr int CK = 32 * SUB * KW;     // keys of a chunk
    static constexpr int KP = 2 * DP + 16;   // bytes of a K row in LDS: reads down a column touch every bank once
    static constexpr int VP = 2 * DP + 64;   // of a V row: 4 rows x 64 bytes a transposing read
    static constexpr int kBuf = CK * (KP + VP);
    static constexpr int NB = 2 * kBuf <= 144 * 1024 ? 2 : 1;
    static constexpr int NPC = CK * DP / 16 / THREADS;  // 16-byte pieces of K (of V) a thread stages
    static constexpr int kMerge = KW == 1 ? 0 : (KW - 1) * RW * DP * 32 * 4 + 4 * 32 * 8;
    static constexpr int kBytes = std::max(NB * kBuf, kMerge);
};

// Four payloads times `scale`, a power of two, as bf16 (exact).
template <int FORMAT, bool SCALED>
__device__ __forceinline__ void to_bf16(uint32_t w, float scale, uint32_t& lo, uint32_t& hi) {
    if constexpr (FORMAT == SANDY_QUANT_E4M3) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, SCALED ? scale : 1.0f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, SCALED ? scale : 1.0f, true));
    } else {
        float v[4];
        quant_values<FORMAT>(w, v);
        if constexpr (SCALED)
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] *= scale;
        lo = __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x07060302u);
        hi = __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x07060302u);
    }
}

// x and y as NS bf16 parts each, packed in pairs: the first ones cut, the last rounded
template <int NS>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&part)[NS]) {
#pragma unroll
    for (int n = 0; n < NS - 1; n++) {
        const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
        part[n] = __builtin_amdgcn_perm(yb, xb, 0x07060302u);
        x -= __uint_as_float(xb & 0xffff0000u);
        y -= __uint_as_float(yb & 0xffff0000u);
    }
    part[NS - 1] = __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(x), static_cast<__bf16>(y)});
}

// Workgroup i's place in the list by falling length: every second round of the
// 256 CUs backwards, so that the workgroups a CU gets add up to about the same.
__device__ __forceinline__ int snake(int i, int n) {
    const int round = i & ~255;
    return (i & 256) ? round + min(256, n - round) - 1 - (i - round) : i;
}

template <typename T, int FORMAT, int DP, int RW>
__global__ __launch_bounds__((QGeo<T, FORMAT, DP, RW>::THREADS), 2) void quant_prefill_kernel(PrefillQArgs pa) {
    using G = QGeo<T, FORMAT, DP, RW>;
    constexpr bool kF32 = G::kF32;
    constexpr int KW = G::KW, CK = G::CK, KP = G::KP, VP = G::VP, NPC = G::NPC, DT = G::DT, NB = G::NB;
    constexpr int NQ = kF32 ? 3 : 1, NP = kF32 ? 3 : 2, KS = DP / 16;  // MFMA steps over the head dim
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const QuantAttnArgs& a = pa.a;
    const QuantPages& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave % RW, kw = (wave & 3) / RW, ds = wave >> 2;
    const int col = lane & 31, half = lane >> 5;
    const int D = p.dim;
    // heads vary fastest (an XCD serves few), the longest row blocks first
    const int heads = p.batch * p.heads;
    const int at = snake(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
    const int bh = at % heads;
    const int rb = pa.row_blocks - 1 - at / heads;
    const int b = bh / p.heads, kh = bh % p.heads;
    const int rows = a.group * p.tokens;
    const int64_t pos = load_index(p.pos, p.pos_dt, b);
    const int count = pos < 0 ? 0 : quant_count(p, b);
    if (pos < 0 && tid == 0) atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_ATTN_POS));
    const int r0 = rb * 32 * RW;
    // the workgroup's keys: those of its first query that is none of the padding to its last
    int k_begin = 0, k_end = 0;
    {
        const int t0 = r0 / a.group, t1 = min(min(rows - 1, r0 + 32 * RW - 1) / a.group, count - 1);
        if (t0 <= t1) {
            k_begin = quant_keys(a, pos, t0).first & ~15;
            k_end = quant_keys(a, pos, t1).last + 1;
        }
    }
    // this lane's row (past the end: the last one, not stored)
    const int row = r0 + 32 * rw + col;
    const int rc = min(row, rows - 1);
    const int qt = rc / a.group, qg = rc - qt * a.group;
    KeyRange mine = quant_keys(a, pos, qt);
    if (qt >= count) mine.last = -1;
    // keys that every row of the wave sees, and keys that some row sees
    const int t_lo = min(rows - 1, r0 + 32 * rw) / a.group, t_hi = min(rows - 1, r0 + 32 * rw + 31) / a.group;
    const int any_first = quant_keys(a, pos, t_lo).first;
    const int any_last = t_lo < count ? quant_keys(a, pos, min(t_hi, count - 1)).last : -1;
    const int all_first = quant_keys(a, pos, t_hi).first;
    const int all_last = t_hi < count ? quant_keys(a, pos, t_lo).last : -1;

    // B operands of Q^T: row, dims 16 s + 8 half .. + 7 in step s (past D zeros: so are K's)
    u32x4_t qv[NQ][KS];
    {
        const int64_t q0 = b * a.qs[0] + (kh * a.group + qg) * a.qs[1] + qt * a.qs[2] + 8 * half;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int64_t from = q0 + (16 * s < D ? 16 * s : 0);
            if constexpr (kF32) {
                float x[8];
                Vec8<F32>::load(a.q, from, x);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t part[3];
                    split_pair<3>(x[2 * i], x[2 * i + 1], part);
#pragma unroll
                    for (int c = 0; c < 3; c++) qv[c][s][i] = part[c];
                }
            } else {
                qv[0][s] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.q) + from);
            }
        }
    }

    u32x4_t* table = reinterpret_cast<u32x4_t*>(lds + G::kBytes);
    // thread piece i: chunk row prow + i * kRowStep, dims 16 ppc .. + 15
    constexpr int kRowStep = G::THREADS / (DP / 16);
    const int prow = tid / (DP / 16), ppc = tid % (DP / 16);
    const bool in_dim = 16 * ppc < D;
    const int page_mask = (1 << p.log2_page) - 1;
    u32x4_t kr[NPC], vr[NPC];
    bool there[NPC];
    float vs[NPC];
    auto load = [&](int c0, int page0) {
#pragma unroll
        for (int i = 0; i < NPC; i++) {
            const int key = min(c0 + prow + i * kRowStep, k_end - 1);
            const u32x4_t e = table[(key >> p.log2_page) - page0];
            const bool page = e[1] != kNoPage && in_dim;
            vs[i] = __uint_as_float(e[3]);
            there[i] = page && c0 + prow + i * kRowStep < k_end;
            const uint64_t off = page ? (static_cast<uint64_t>(e[1]) << 32 | e[0]) + static_cast<uint32_t>(key & page_mask) * static_cast<uint32_t>(D) + 16 * ppc : 0;
            kr[i] = *reinterpret_cast<const u32x4_t*>(p.pool[0] + off);
            vr[i] = *reinterpret_cast<const u32x4_t*>(p.pool[1] + off);
        }
    };
    auto store = [&](int buf) {
        unsigned char* kt = lds + buf * G::kBuf;
        unsigned char* vt = kt + CK * KP;
#pragma unroll
        for (int i = 0; i < NPC; i++) {
            const int r = prow + i * kRowStep;
            u32x4_t k = kr[i], v = vr[i];
            // rows past the last key and missing pages: zeros (their weights are 0)
            if (!there[i]) k = v = u32x4_t{0, 0, 0, 0};
            u32x4_t o[2];
#pragma unroll
            for (int w = 0; w < 4; w++) {
                uint32_t lo, hi;
                to_bf16<FORMAT, false>(k[w], 1.0f, lo, hi);
                o[w >> 1][2 * (w & 1)] = lo, o[w >> 1][2 * (w & 1) + 1] = hi;
            }
            *reinterpret_cast<u32x4_t*>(kt + r * KP + 32 * ppc) = o[0];
            *reinterpret_cast<u32x4_t*>(kt + r * KP + 32 * ppc + 16) = o[1];
#pragma unroll
            for (int w = 0; w < 4; w++) {
                uint32_t lo, hi;
                to_bf16<FORMAT, true>(v[w], vs[i], lo, hi);
                o[w >> 1][2 * (w & 1)] = lo, o[w >> 1][2 * (w & 1) + 1] = hi;
            }
            *reinterpret_cast<u32x4_t*>(vt + r * VP + 32 * ppc) = o[0];
            *reinterpret_cast<u32x4_t*>(vt + r * VP + 32 * ppc + 16) = o[1];
        }
    };

    f32x16_t acc[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[t][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int buf = 0;

    // segments of whole pages that the table holds (k_end at the last)
    for (int seg = k_begin; seg < k_end;) {
        const int page0 = seg >> p.log2_page;
        const int64_t seg_last = (static_cast<int64_t>(page0) + pa.table) << p.log2_page;
        // chunks start at k_begin + a multiple of CK: a segment ends where one does
        const int seg_end = seg_last >= k_end ? k_end : k_begin + (static_cast<int>(seg_last) - k_begin) / CK * CK;
        __syncthreads();  // the segment before has been read
        for (int i = tid; i < pa.table && page0 + i <= (seg_end - 1) >> p.log2_page; i += G::THREADS) {
            const int id = quant_block(p, b, page0 + i);
            u32x4_t e{0, kNoPage, 0, 0};
            if (id >= 0) {
                const int64_t block = static_cast<int64_t>(id) * p.heads + kh;
                const uint64_t off = static_cast<uint64_t>(block << p.log2_page) * D;
                const int kc = p.scales[0][block], vc = p.scales[1][block];
                // a NaN block: NaN scores for the rows that see it, V's own factor aside
                const float f = kc == 255 || vc == 255 ? quant_scale(255) : fmaxf(quant_scale(kc) * a.scale_log2, 0x1p-126f);
                e = u32x4_t{static_cast<uint32_t>(off), static_cast<uint32_t>(off >> 32), __float_as_uint(f),
                            __float_as_uint(quant_scale(vc == 255 ? 127 : vc))};
            }
            table[i] = e;
        }
        __syncthreads();
        load(seg, page0);
        for (int c0 = seg; c0 < seg_end; c0 += CK, buf ^= NB - 1) {
            if (NB == 1 && c0 > seg) __syncthreads();  // the chunk before has been read
            store(buf);
            __syncthreads();
            if (c0 + CK < seg_end) load(c0 + CK, page0);
            const int k0 = c0 + 32 * G::SUB * kw;
            if (k0 > any_last || k0 + 32 * G::SUB - 1 < any_first) continue;  // wave-uniform
            const unsigned char* kt = lds + buf * G::kBuf + (32 * G::SUB * kw + col) * KP + 16 * half;
            const unsigned char* vt = lds + buf * G::kBuf + CK * KP + 32 * G::SUB * kw * VP;
            f32x16_t sc[G::SUB];
#pragma unroll
            for (int u = 0; u < G::SUB; u++) {
#pragma unroll
                for (int i = 0; i < 16; i++) sc[u][i] = 0.0f;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    const bf16x8_t ka = *reinterpret_cast<const bf16x8_t*>(kt + 32 * u * KP + 32 * s);
#pragma unroll
                    for (int c = NQ - 1; c >= 0; c--)
                        sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka, __builtin_bit_cast(bf16x8_t, qv[c][s]), sc[u], 0, 0, 0);
                }
            }
            // factors of the 16-key tiles (the last ones may lie past the last key)
            float f[2 * G::SUB];
            bool plain = k0 + 32 * G::SUB - 1 <= all_last && k0 >= all_first;
#pragma unroll
            for (int h = 0; h < 2 * G::SUB; h++) {
                const u32x4_t e = table[(min(k0 + 16 * h, k_end - 1) >> p.log2_page) - page0];
                f[h] = __uint_as_float(e[2]);  // 0 without a page, or NaN
                plain = plain && __any(f[h] > 0.0f);
            }
            // element i of block u: key k0 + 32 u + 8 (i / 4) + 4 half + i % 4
            if (!plain) {
                int key0 = k0 + 4 * half;
                asm volatile("" : "+v"(key0));  // keeps the compares out of whole tiles
#pragma unroll
                for (int h = 0; h < 2 * G::SUB; h++) {
                    const bool none = f[h] == 0.0f, nan = f[h] != f[h];
                    const int end = none ? -1 : mine.last;
                    if (none | nan) f[h] = 1.0f;  // the factor goes into the scores themselves
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int key = key0 + 16 * h + 8 * (i >> 2) + (i & 3);
                        const float s = nan ? quant_scale(255) : sc[h >> 1][8 * (h & 1) + i];
                        sc[h >> 1][8 * (h & 1) + i] = (key < mine.first) | (key > end) ? -INFINITY : s;
                    }
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2 * G::SUB; h++) {
                float top = sc[h >> 1][8 * (h & 1)];
#pragma unroll
                for (int i = 1; i < 8; i++) top = fmaxf(top, sc[h >> 1][8 * (h & 1) + i]);
                mx = fmaxf(mx, top * f[h]);
            }
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
#pragma unroll
            for (int u = 0; u < G::SUB; u++) {
#pragma unroll
                for (int i = 0; i < 16; i++) sc[u][i] = __builtin_amdgcn_exp2f(fmaf(sc[u][i], f[2 * u + (i >> 3)], -shift));
                {
                    float rs[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) rs[i] = sc[u][2 * i] + sc[u][2 * i + 1];
                    l += ((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7]));
                }
                // contraction slot 8 half + j of step s2: key 16 s2 + 4 half + j (j < 4) or + 8 + j - 4
#pragma unroll
                for (int s2 = 0; s2 < 2; s2++) {
                    u32x4_t pw[NP];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        uint32_t part[NP];
                        split_pair<NP>(sc[u][8 * s2 + j], sc[u][8 * s2 + j + 1], part);
#pragma unroll
                        for (int c = 0; c < NP; c++) pw[c][j / 2] = part[c];
                    }
                    // ds_read_b64_tr_b16: in each 16-lane group, lane i gets element i % 4 of
                    // the 8-byte pieces addressed by lanes 4 n + i / 4 (n = 0..3)
                    const int i16 = lane & 15;
                    const unsigned char* src = vt + (32 * u + 16 * s2 + 4 * half + (i16 >> 2)) * VP + 2 * (16 * ((lane >> 4) & 1) + 4 * (i16 & 3));
#pragma unroll
                    for (int t = 0; t < DT; t++) {
                        const unsigned char* s0 = src + 64 * (DT * ds + t);
                        const short4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (short4_t __attribute__((address_space(3)))*)((unsigned char __attribute__((address_space(3)))*)s0));
                        const short4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (short4_t __attribute__((address_space(3)))*)((unsigned char __attribute__((address_space(3)))*)(s0 + 8 * VP)));
                        const bf16x8_t va = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                        for (int c = NP - 1; c >= 0; c--)
                            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, __builtin_bit_cast(bf16x8_t, pw[c]), acc[t], 0, 0, 0);
                    }
                }
            }
        }
        seg = seg_end;
    }

    // the two halves of a row's sum; then the key shares of the KW waves
    l = sum_xor32(l);
    if constexpr (KW > 1) {
        __syncthreads();
        float* red = reinterpret_cast<float*>(lds);
        float2* ml = reinterpret_cast<float2*>(lds + (KW - 1) * RW * DP * 32 * 4);  // [wave of the first half][32]
        if (half == 0 && ds == 0) ml[(wave & 3) * 32 + col] = make_float2(m, l);
        __syncthreads();
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < KW; w++) mm = fmaxf(mm, ml[(w * RW + rw) * 32 + col].x);
        const float shift = mm == -INFINITY ? 0.0f : mm;
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; w++) {
            const float2 e = ml[(w * RW + rw) * 32 + col];
            l += e.y * __builtin_amdgcn_exp2f(e.x - shift);
        }
        const float f = __builtin_amdgcn_exp2f(m - shift);
#pragma unroll
        for (int t = 0; t < DT; t++) acc[t] *= f;
        if (kw > 0) {
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) red[(((kw - 1) * RW + rw) * (DP / 2) + 16 * (DT * ds + t) + i) * 64 + lane] = acc[t][i];
        }
        __syncthreads();
        if (kw > 0) return;
#pragma unroll
        for (int w = 0; w < KW - 1; w++)
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[t][i] += red[((w * RW + rw) * (DP / 2) + 16 * (DT * ds + t) + i) * 64 + lane];
    }
    if (row >= rows) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t o0 = b * a.os[0] + (kh * a.group + qg) * a.os[1] + qt * a.os[2] + 4 * half;
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = 32 * (DT * ds + t) + 8 * i;
            if (d >= D) continue;
            const f32x4_t o = f32x4_t{acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]} * inv;
            if constexpr (kF32) *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + o0 + d) = o;
            else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + o0 + d) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
        }
}

template <typename T, int FORMAT, int DP, int RW>
int launch_rows(const QuantAttnArgs& a, hipStream_t stream, Err e) {
    using G = QGeo<T, FORMAT, DP, RW>;
    static_assert(G::kBytes + kTable * 16 <= 160 * 1024 - 256, "LDS of a workgroup");
    PrefillQArgs pa{};
    pa.a = a;
    const int64_t rows = static_cast<int64_t>(a.group) * a.p.tokens;
    pa.row_blocks = static_cast<int32_t>((rows + 32 * RW - 1) / (32 * RW));
    pa.table = std::min(kTable, a.p.max_blocks);
    const size_t bytes = G::kBytes + static_cast<size_t>(pa.table) * 16;
    const void* fn = reinterpret_cast<const void*>(&quant_prefill_kernel<T, FORMAT, DP, RW>);
    if (bytes > 64 * 1024)
        SANDY_HIP_TRY(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)), e,
                      "quant_paged attention launch");
    const int64_t wgs = static_cast<int64_t>(pa.row_blocks) * a.p.batch * a.p.heads;
    void* params[] = {&pa};
    SANDY_HIP_TRY(hipLaunchKernel(fn, dim3(static_cast<unsigned>(wgs)), dim3(G::THREADS), params, bytes, stream), e,
                  "quant_paged attention launch");
    return ok(e);
}

template <typename T, int FORMAT, int DP>
int launch_dim(const QuantAttnArgs& a, hipStream_t stream, Err e) {
    const int64_t rows = static_cast<int64_t>(a.group) * a.p.tokens;
    const int64_t wgs = (rows + 63) / 64 * a.p.batch * a.p.heads;
    const int rw = env_int("SANDY_QUANT_RW", wgs >= 224 ? 2 : 1);
    if (rw == 4) return launch_rows<T, FORMAT, DP, 4>(a, stream, e);
    if (rw == 2) return launch_rows<T, FORMAT, DP, 2>(a, stream, e);
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
           (rows + 31) / 32 * batch * heads <= UINT32_MAX / 512;
}

int launch_quant_prefill(const QuantAttnArgs& a, int32_t format, hipStream_t stream, Err e) {
    if (format == SANDY_QUANT_INT8)
        return a.f32 ? launch_format<F32, SANDY_QUANT_INT8>(a, stream, e) : launch_format<BF16, SANDY_QUANT_INT8>(a, stream, e);
    return a.f32 ? launch_format<F32, SANDY_QUANT_E4M3>(a, stream, e) : launch_format<BF16, SANDY_QUANT_E4M3>(a, stream, e);
}

} // namespace sandy_hip
