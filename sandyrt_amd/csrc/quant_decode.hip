// quant_decode.hip -- attention of few queries a sequence over the 8-bit paged
// cache on bf16 MFMA, the keys split over workgroups.
//
// Both payload types are exact in bf16, so a payload goes to the matrix unit as
// it is: S^T = K Q^T with K's scale applied to the scores, O^T += V^T P^T with
// V's applied to the weights (int8) or in the conversion itself (e4m3: exact,
// the scale is a power of two).  f32 queries and all weights enter as three bf16
// operands that hold them exactly.  Tiles are 16 keys; a wave takes
// two at a time:
//   - K straight into the A operand: a lane holds 16 consecutive dims of its key,
//     the first 8 for one MFMA step and the others for the next (the order of the
//     contraction is free as long as Q has the same);
//   - V through the wave's own LDS rows, back by ds_read_b64_tr_b8, which gives a
//     lane one dim of 8 keys -- the A operand of O^T in the order that P leaves S^T.
//
// In a graph, 32 sequences of 512 to 4096 keys, 32 / 4 heads of 64: 37 MB in 15.7 us (2.4
// TB/s; a copy would take 7.2); one sequence of 32749 keys 13.8 us; 64 with a window of
// 1024, 8 / 2 heads of 256: 20.2 us; 32 of 8000 keys 32.3 us (4.1 TB/s).  Vector
// instructions issue in 11 to 20 % of these cycles, MFMA in 2 to 6 %.  Short contexts are
// latency: a call of up to 128 keys takes 4.7 us, of 600 7.3, the chain position, block
// table, payload, join.
#include "quant_split.h"

namespace sandy_hip {
namespace {

template <typename T, int FORMAT, int DP>
struct DecodeGeo {
    static constexpr int kChunks = DP / 64;  // 16-byte pieces a lane holds of a K (V) tile
    static constexpr int kRing = DP == 256 ? 1 : 2;  // pairs in flight (D 256 with two: 38 us to 20)
    static constexpr int kWaves = DP == 64 ? 3 : DP == 256 && std::is_same_v<T, F32> ? 1 : 2;  // a SIMD
    static constexpr int VP = DP + 16;       // bytes of a V row in LDS: column reads spread over the banks
    static constexpr int kV = 32 * VP;       // a wave's V rows
    static constexpr int kSet = DP == 256 ? 8 : DP / 16;  // accumulator tiles the waves exchange at a time
    static constexpr int kMerge = 4 * kSet * 64 * 16;
    static constexpr int kBytes = std::max(4 * kV, kMerge) + 4 * 16 * 2 * 4;
};

template <typename T, int FORMAT, int DP>
__global__ __launch_bounds__(256, (DecodeGeo<T, FORMAT, DP>::kWaves)) void quant_decode_kernel(SplitArgs da) {
    using G = DecodeGeo<T, FORMAT, DP>;
    constexpr bool kF32 = std::is_same_v<T, F32>;
    constexpr int NQ = kF32 ? 3 : 1, NCH = G::kChunks, NT = DP / 16, RING = G::kRing;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const QuantAttnArgs& a = da.a;
    const QuantPages& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int D = p.dim;
    // heads vary fastest, then sequences, column tiles, splits: those without keys come last,
    // not between the others on the same XCDs
    uint32_t at = blockIdx.x;
    const int kh = at % p.heads;
    at /= p.heads;
    const int b = at % p.batch;
    at /= p.batch;
    const int ct = at % da.col_tiles;
    const int split = at / da.col_tiles;
    const int rows = a.group * p.tokens;
    const int64_t pos = load_index(p.pos, p.pos_dt, b);
    const int count = pos < 0 ? 0 : quant_count(p, b);
    const SeqKeys seq = quant_keys(a, pos);
    const int t_lo = divide(16 * ct, a.group, a.group_magic), t_hi = divide(min(rows - 1, 16 * ct + 15), a.group, a.group_magic);
    const TileKeys tk = tile_keys(da, seq, count, t_lo, t_hi);
    if (split >= tk.active) return;
    if (pos < 0 && tid == 0) atomicOr(p.errw, static_cast<uint32_t>(SANDY_DEVERR_ATTN_POS));

    // this lane's column: query qt, head qg of the group (past the rows: the last one, not stored)
    const int row = min(16 * ct + col, rows - 1);
    const int qt = divide(row, a.group, a.group_magic), qg = row - qt * a.group;
    KeyRange mine = seq.of(qt);
    if (qt >= count) mine.last = -1;
    // keys that every column sees
    const int all_first = seq.of(t_hi).first;
    const int all_last = t_hi < count ? seq.of(t_lo).last : -1;

    // B operands of Q^T: column, dims 64 j + 16 g + 8 s .. + 7 in step 2 j + s
    // (past D any of the row's: K is zero there)
    u32x4_t raw[kF32 ? 2 : 1][2 * NCH], qv[NQ][2 * NCH];
    {
        const int64_t q0 = b * a.qs[0] + (kh * a.group + qg) * a.qs[1] + qt * a.qs[2];
#pragma unroll
        for (int s = 0; s < 2 * NCH; s++) {
            const int d = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
            const char* from = static_cast<const char*>(a.q) + (q0 + (d < D ? d : 0)) * (kF32 ? 4 : 2);
#pragma unroll
            for (int i = 0; i < (kF32 ? 2 : 1); i++) raw[i][s] = *reinterpret_cast<const u32x4_t*>(from + 16 * i);
        }
    }

    f32x4_t acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    bool loud = false;  // the same for the wave

    unsigned char* vrows = lds + wave * G::kV;
    int k_off[NCH], v_to[NCH];  // this lane's bytes of a tile; its V pieces' places in LDS
#pragma unroll
    for (int j = 0; j < NCH; j++) {
        const int d = 64 * j + 16 * g;
        k_off[j] = d < D ? col * D + d : 0x7ffffff0;  // past every tile: zeros
        const int piece = lane + 64 * j, per_row = D / 16;
        const int r = piece / per_row;
        v_to[j] = r < 16 ? r * G::VP + 16 * (piece - r * per_row) : DP;  // none: the padding of the first row
    }
    // ds_read_b64_tr_b8: lanes 2 n and 2 n + 1 of 16 address row n's 16 bytes, lane i
    // gets byte i of the 8 rows: keys 4 g + n of the first tile, then of the second
    const int trow = (lane & 15) >> 1;
    const unsigned char* v_from = vrows + (trow < 4 ? 4 * g + trow : 16 + 4 * g + trow - 4) * G::VP + 8 * (lane & 1);

    const int last_pair = min((split + 1) * tk.per, tk.pairs);
    // a wave takes every fourth pair, 32 of them (64 tiles) a round: lane i holds
    // tile i & 1 of pair i / 2, its bytes' offset, its rows (none: 0) and factors
    int bytes_in = 0;
    uint64_t offset = 0;
    float kf = 0.0f, vf = 1.0f;
    uint64_t odd = 0;  // the tiles without a page, or that make the sums loud
    u32x4_t kr[RING][2][NCH], vr[RING][2][NCH];
    auto load = [&](int n, u32x4_t (&k)[2][NCH], u32x4_t (&v)[2][NCH]) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int tile = (2 * n + h) & 63;
            // rows past the last key and tiles without a page: an empty range reads zeros
            const int bytes = n < 32 ? __builtin_amdgcn_readlane(bytes_in, tile) : 0;
            const uint64_t off = static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(offset >> 32), tile)) << 32 |
                                 static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(offset), tile));
            const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(p.pool[0] + off, 0, bytes, kRsrcWord3);
            const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(p.pool[1] + off, 0, bytes, kRsrcWord3);
#pragma unroll
            for (int j = 0; j < NCH; j++) k[h][j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off[j], 0, 0));
#pragma unroll
            for (int j = 0; j < NCH; j++) v[h][j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rv, 16 * (lane + 64 * j), 0, 0));
        }
    };
    auto begin_round = [&](int round0) {
        const int pair = round0 + 4 * (lane >> 1);
        const int key0 = tk.begin + 32 * pair + 16 * (lane & 1);
        const bool mine_in = pair < last_pair && key0 <= tk.last;
        const int id = mine_in ? quant_block(p, b, key0 >> p.log2_page) : -1;
        bytes_in = id < 0 ? 0 : min(16, tk.last - key0 + 1) * D;
        const int64_t block = static_cast<int64_t>(max(id, 0)) * p.heads + kh;
        offset = id < 0 ? 0 : static_cast<uint64_t>((block << p.log2_page) + (key0 & ((1 << p.log2_page) - 1))) * D;
        const int kc = p.scales[0][block], vc = p.scales[1][block];
#pragma unroll
        for (int i = 0; i < RING; i++) load(i, kr[i], vr[i]);
        // a NaN block: NaN scores for whoever sees it, V's own factor aside
        kf = quant_scale(vc == 255 ? 255 : kc) * a.scale_log2;
        vf = quant_scale(vc == 255 || id < 0 ? 127 : vc);
        if (loud) vf = fmaxf(vf * kLoudDown, 0x1p-126f);
        odd = __ballot((id < 0) | (__float_as_uint(vf) >= kLoudBits));
    };
    // before such a block's values first enter the sums
    auto get_loud = [&]() {
        loud = true;
        vf = fmaxf(vf * kLoudDown, 0x1p-126f);
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] *= kLoudDown;
    };
    auto attend = [&](int round0, int n, u32x4_t (&k)[2][NCH], u32x4_t (&v)[2][NCH]) {
        f32x4_t sc[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            sc[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < NCH; j++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const bf16x8_t ka = payload_operand<FORMAT>(k[h][j][2 * s], k[h][j][2 * s + 1], 1.0f, 1.0f);
#pragma unroll
                    for (int c = NQ - 1; c >= 0; c--)
                        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, __builtin_bit_cast(bf16x8_t, qv[c][2 * j + s]), sc[h], 0, 0, 0);
                }
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < NCH; j++) *reinterpret_cast<u32x4_t*>(vrows + 16 * h * G::VP + v_to[j]) = v[h][j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        load(n + RING, k, v);
        const float kf0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kf), 2 * n));
        const float kf1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kf), 2 * n + 1));
        uint32_t vf0 = __builtin_amdgcn_readlane(__float_as_uint(vf), 2 * n);
        uint32_t vf1 = __builtin_amdgcn_readlane(__float_as_uint(vf), 2 * n + 1);
        const int k0 = tk.begin + 32 * (round0 + 4 * n);
        sc[0] *= kf0;
        sc[1] *= kf1;
        if ((k0 < all_first) | (k0 + 31 > all_last) | ((odd >> (2 * n) & 3) != 0)) {
            if (max(vf0, vf1) >= kLoudBits) {
                get_loud();
                vf0 = __builtin_amdgcn_readlane(__float_as_uint(vf), 2 * n);
                vf1 = __builtin_amdgcn_readlane(__float_as_uint(vf), 2 * n + 1);
            }
            // element i of tile h: key k0 + 16 h + 4 g + i
            const int end0 = __builtin_amdgcn_readlane(bytes_in, 2 * n) == 0 ? -1 : mine.last;
            const int end1 = __builtin_amdgcn_readlane(bytes_in, 2 * n + 1) == 0 ? -1 : mine.last;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int key = k0 + 4 * g + i;
                sc[0][i] = (key < mine.first) | (key > end0) ? -INFINITY : sc[0][i];
                sc[1][i] = (key + 16 < mine.first) | (key + 16 > end1) ? -INFINITY : sc[1][i];
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                         fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
        // a column's reference m moves only once its maximum has grown by 2^8:
        // weights stay below that, at the same relative precision
        if (__any(mx > m + 8.0f)) {
            mx = max_xor32(max_xor16(mx));
            const float m_new = fmaxf(m, mx);
            const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
            l *= alpha;
#pragma unroll
            for (int t = 0; t < NT; t++) acc[t] *= alpha;
            m = m_new;
        }
        const float shift = m == -INFINITY ? 0.0f : m;
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = __builtin_amdgcn_exp2f(sc[i >> 2][i & 3] - shift);
        l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        if constexpr (FORMAT == SANDY_QUANT_INT8)
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] *= __uint_as_float(i < 4 ? vf0 : vf1);
        bf16x8_t pw[3];
        {
            u32x4_t parts[3];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                uint32_t part[3];
                split_pair(w[i], w[i + 1], part);
#pragma unroll
                for (int c = 0; c < 3; c++) parts[c][i / 2] = part[c];
            }
#pragma unroll
            for (int c = 0; c < 3; c++) pw[c] = __builtin_bit_cast(bf16x8_t, parts[c]);
        }
        // (dims past D: bytes of earlier tiles, in accumulators that nothing stores)
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const i32x2_t eight = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (i32x2_t __attribute__((address_space(3)))*)((unsigned char __attribute__((address_space(3)))*)(v_from + 16 * t)));
            const bf16x8_t va = payload_operand<FORMAT>(static_cast<uint32_t>(eight[0]), static_cast<uint32_t>(eight[1]), __uint_as_float(vf0), __uint_as_float(vf1));
#pragma unroll
            for (int c = 2; c >= 0; c--) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pw[c], acc[t], 0, 0, 0);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    };
    int round0 = split * tk.per + wave;
    if (round0 < last_pair) {
        begin_round(round0);
#pragma unroll
        for (int s = 0; s < 2 * NCH; s++) {
            if constexpr (kF32) {
                // an infinity leaves inf - inf for its later parts: NaN scores, as an
                // infinite score's weight has
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t part[3];
                    split_pair(__uint_as_float(raw[i >> 1][s][2 * (i & 1)]), __uint_as_float(raw[i >> 1][s][2 * (i & 1) + 1]), part);
#pragma unroll
                    for (int c = 0; c < 3; c++) qv[c][s][i] = part[c];
                }
            } else {
                qv[0][s] = raw[0][s];
            }
        }
        for (;;) {
            // no branch around a load: the waits stay exact and later loads in flight
            const int n_pairs = min(32, (last_pair - round0 + 3) / 4);
            int n = 0;
            for (; n + RING <= n_pairs; n += RING)
#pragma unroll
                for (int i = 0; i < RING; i++) attend(round0, n + i, kr[i], vr[i]);
            if (n < n_pairs) attend(round0, n, kr[0], vr[0]);
            round0 += 4 * 32;
            if (round0 >= last_pair) break;
            begin_round(round0);
        }
    }

    // the four waves' maxima and sums, then their accumulators
    l = sum_xor32(sum_xor16(l));
    float* ml = reinterpret_cast<float*>(lds + std::max(4 * G::kV, G::kMerge));
    if (g == 0) {
        ml[(wave * 16 + col) * 2] = m;
        ml[(wave * 16 + col) * 2 + 1] = mark_loud(l, loud);
    }
    __syncthreads();
    float mm = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) mm = fmaxf(mm, ml[(w * 16 + col) * 2]);
    const float shift = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
    for (int w = 0; w < 4; w++) total += fabsf(ml[(w * 16 + col) * 2 + 1]) * __builtin_amdgcn_exp2f(ml[(w * 16 + col) * 2] - shift);
    bool any_loud = false;
#pragma unroll
    for (int w = 0; w < 4; w++) any_loud |= is_loud(ml[(w * 16 + col) * 2 + 1]);
    const float down = any_loud && !loud ? kLoudDown : 1.0f, up = any_loud ? kLoudUp : 1.0f;
    const float f = __builtin_amdgcn_exp2f(m - shift);
    f32x4_t* red = reinterpret_cast<f32x4_t*>(lds);
    const bool final_out = tk.active == 1;
    const int64_t unit = (static_cast<int64_t>(ct) * p.batch + b) * p.heads + kh;
    const int64_t slot = unit * da.splits + split;
    const Through po(da.part_o + slot * 16 * D);
    const bool stored = 16 * ct + col < rows;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int64_t o0 = b * a.os[0] + (kh * a.group + qg) * a.os[1] + qt * a.os[2];
    constexpr int SET = G::kSet;
#pragma unroll
    for (int s0 = 0; s0 < NT; s0 += SET) {
        if (s0 > 0) __syncthreads();
#pragma unroll
        for (int t = 0; t < SET; t++) red[(wave * SET + t) * 64 + lane] = acc[s0 + t] * down * f;
        __syncthreads();
#pragma unroll
        for (int t4 = 0; t4 < SET; t4 += 4) {
            const int t = t4 + wave;
            const int d = 16 * (s0 + t) + 4 * g;
            if (d >= D || !stored) continue;
            const f32x4_t o = (red[t * 64 + lane] + red[(SET + t) * 64 + lane]) +
                              (red[(2 * SET + t) * 64 + lane] + red[(3 * SET + t) * 64 + lane]);
            if (final_out) store4<T>(a.out, o0 + d, o * inv * up);
            else po.put(col * D + d, o);
        }
    }
    if (final_out) return;
    if (tid < 16 && stored) Through(da.part_ml + slot * 32).put(2 * col, mm, mark_loud(total, any_loud));
    finish_split<T, 16>(da, unit, split, tk.active, ct, kh, b);
}

template <typename T, int FORMAT, int DP>
int launch_dim(const SplitArgs& d, hipStream_t stream, Err e) {
    using G = DecodeGeo<T, FORMAT, DP>;
    static_assert(G::kBytes <= 64 * 1024, "LDS of a workgroup");
    return launch_split<T, 16>(reinterpret_cast<const void*>(&quant_decode_kernel<T, FORMAT, DP>), d, G::kBytes, stream, e);
}

template <typename T, int FORMAT>
int launch_format(const SplitArgs& d, hipStream_t stream, Err e) {
    if (d.a.p.dim <= 64) return launch_dim<T, FORMAT, 64>(d, stream, e);
    if (d.a.p.dim <= 128) return launch_dim<T, FORMAT, 128>(d, stream, e);
    return launch_dim<T, FORMAT, 256>(d, stream, e);
}

} // namespace

bool quant_decode_takes(const QuantAttnArgs& a) {
    const QuantPages& p = a.p;
    const int64_t es = a.f32 ? 4 : 2;
    if (p.dim % 16 != 0 || p.dim > 256 || p.log2_page < 4) return false;
    auto aligned = [](const void* ptr, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; };
    if (!aligned(p.pool[0], 16) || !aligned(p.pool[1], 16)) return false;
    // q read and out written in pieces of 16 bytes (out bf16: 8)
    const int64_t in[3] = {p.batch > 1 ? a.qs[0] : 0, a.hq > 1 ? a.qs[1] : 0, p.tokens > 1 ? a.qs[2] : 0};
    const int64_t to[3] = {p.batch > 1 ? a.os[0] : 0, a.hq > 1 ? a.os[1] : 0, p.tokens > 1 ? a.os[2] : 0};
    if (!aligned(a.q, 16) || ((in[0] | in[1] | in[2]) & (16 / es - 1)) || a.qs[3] != 1) return false;
    if (!aligned(a.out, 4 * es) || ((to[0] | to[1] | to[2]) & 3) || a.os[3] != 1) return false;
    const int64_t rows = static_cast<int64_t>(a.group) * p.tokens;
    const int64_t col_tiles = (rows + 15) / 16;
    // threads of a launch below 2^32, splits (of fewer tiles than wanted) included
    return rows < (1 << 30) && col_tiles * p.batch * p.heads <= UINT32_MAX / 256 - 2048;
}

size_t quant_decode_workspace(int64_t batch, int64_t hq, int64_t heads, int64_t tokens, int64_t dim, int64_t page,
                              int64_t max_blocks, int64_t window) {
    const int64_t units = (hq / heads * tokens + 15) / 16 * batch * heads;
    SplitArgs d{};
    set_splits(&d, units, dim, max_blocks * page, window, tokens);
    return d.splits == 1 ? 0 : static_cast<size_t>(units * d.splits * 16 * (dim + 2)) * sizeof(float);
}

int launch_quant_decode(const QuantAttnArgs& a, int32_t format, void* workspace, hipStream_t stream, Err e) {
    const QuantPages& p = a.p;
    SplitArgs d{};
    d.a = a;
    d.col_tiles = (a.group * p.tokens + 15) / 16;
    set_splits(&d, static_cast<int64_t>(p.batch) * p.heads * d.col_tiles, p.dim,
               static_cast<int64_t>(p.max_blocks) << p.log2_page, a.window, p.tokens);
    const int status = split_memory<16>(&d, workspace, stream, e);
    if (status) return status;
    if (format == SANDY_QUANT_INT8)
        return a.f32 ? launch_format<F32, SANDY_QUANT_INT8>(d, stream, e) : launch_format<BF16, SANDY_QUANT_INT8>(d, stream, e);
    return a.f32 ? launch_format<F32, SANDY_QUANT_E4M3>(d, stream, e) : launch_format<BF16, SANDY_QUANT_E4M3>(d, stream, e);
}

} // namespace sandy_hip
