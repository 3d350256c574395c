// quant_tile.h -- the kernel for many rows of the products of matrices in 8 bits (quant_gemm.h).
#pragma once
#include "quant_gemm.h"

#include <algorithm>

namespace sandy_hip {

// Workgroup tile 32 PM WM x 32 PN WN of rows x columns, PM x PN waves of 32 WM x 32 WN on 32 x 32 instructions, 128 columns
// of k (a block, a whole 128-byte line of every row) a chunk, STAGES chunks in LDS.  SPLIT groups of so many waves share the
// chunks, a run each, and add up their sums at the end.
//
// What it is up against: a CU's copies into LDS came to no more than 35 bytes a cycle (83 KB/us) in any form, also with 4 and
// 8 chunks under way and one meeting a chunk in place of two.  A chunk of a 64 x 64 tile takes them 480 cycles for 64 a wave
// of products, one of 128 x 128 960 for 512 of two workgroups, one of 256 x 256 1900 for 2048, so that large tiles are bound
// by both (2720 TFLOP/s at 4096 x 8192 x 8192) and small ones by copies: 333 x 1999 x 5617 in 22 us, where each workgroup
// waits at every meeting, and 15.8 with SPLIT 2, whose groups wait for each other's copies; 4 gain nothing there.
template <int WM, int WN, int PM, int PN, int STAGES, int SPLIT>
struct QuantTile {
    static constexpr int BM = 32 * PM * WM, BN = 32 * PN * WN, kThreads = 64 * PM * PN;
    static constexpr int kX = BM * 128, kStage = (BM + BN) * 128;
    // the scale bytes of kRun blocks of every row, twice, behind the stages: 8 for small tiles, so that three workgroups of
    // 64 x 128 fit a CU (128 rows of 128 experts of 1408 x 2816: 62 us to 53), 16 for large ones (4096 x 8192 x 8192: 212 to 203)
    static constexpr int kRun = WM * WN < 16 ? 8 : 16, kScales = STAGES * kStage, kScaleBytes = (BM + BN) * kRun;
    static constexpr int kStep = kThreads / 8, kXLoads = BM / kStep, kLoads = (BM + BN) / kStep;  // 16-byte pieces a thread moves a chunk
    template <typename T>
    static constexpr int row_bytes() { return 32 * WN * static_cast<int>(sizeof(typename Vec8<T>::elem)) + 16; }
    template <typename T>
    static constexpr int group_lds() {
        const int out = kThreads / 64 * 32 * row_bytes<T>();
        constexpr int loop = kScales + 2 * kScaleBytes, sums = SPLIT > 1 ? BM * BN * 4 : 0;
        return std::max({loop, sums, (out + 1023) / 1024 * 1024});
    }
    template <typename T>
    static constexpr int lds() { return SPLIT * group_lds<T>(); }
};

// N scale bytes from j on of a row, the last for those past it.
template <int N>
__device__ __forceinline__ auto some_scales(const uint8_t* row, int j, int blocks) {
    int32_t __attribute__((ext_vector_type(N / 4))) v = 0;
    if (j + N <= blocks) {
        __builtin_memcpy(&v, row + j, N);
    } else {  // (all at once: loads under a condition each would wait for one another)
#pragma unroll
        for (int i = 0; i < N; i++) v[i >> 2] |= row[min(j + i, blocks - 1)] << (8 * (i & 3));
    }
    return v;
}

// 16 bytes a lane from a buffer straight into LDS, the wave's 1024 bytes in a row from `lds` on.  In flight until
// a wait on vmcnt; the compiler does not count it (its own waits only become stricter).  (s_nop: a vector
// instruction may just have written one of the scalars.)  m0 is named as overwritten, so that no value the compiler puts
// there is taken to live across it; the warning that m0 is a reserved register is no news.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy_to_lds(i32x4_t buffer, int offset, int more, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(offset), "s"(buffer), "s"(more)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// WHOLE: rows of out begin on 16-byte boundaries.
template <typename T, bool WHOLE, int WM, int WN, int PM, int PN, int STAGES, int SPLIT>
__global__ __launch_bounds__(64 * PM * PN * SPLIT, 1) void quant_tile_kernel(QuantGemm a, int m_tiles, int n_tiles) {
    using G = QuantTile<WM, WN, PM, PN, STAGES, SPLIT>;
    constexpr bool kScaled = std::is_same_v<T, BF16>;
    extern __shared__ __align__(1024) unsigned char all_lds[];
    const int lane = threadIdx.x & 63, waves = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int group = waves / (PM * PN), wave = waves - group * PM * PN, tid = 64 * wave + lane;
    unsigned char* const lds = all_lds + group * G::template group_lds<T>();
    const int wm = wave % PM, wn = wave / PM;
    const int col = lane & 31, half = lane >> 5;

    // experts' row tiles: a lane takes four experts from `base` on, up to whose end there are `upto` more than before base
    int64_t edge[5];
    int tiles[4], mine_tiles = 0;
    auto count = [&](int base) {
        const int e0 = base + 4 * lane;
        if (a.offsets_dt == SANDY_I32) {
#pragma unroll
            for (int i = 0; i < 5; i++) edge[i] = static_cast<const int32_t*>(a.offsets)[min(e0 + i, a.groups)];
        } else {
#pragma unroll
            for (int i = 0; i < 5; i++) edge[i] = static_cast<const int64_t*>(a.offsets)[min(e0 + i, a.groups)];
        }
        bool bad = false;
        mine_tiles = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool in_order = edge[i] >= 0 && edge[i + 1] >= edge[i] && edge[i + 1] <= a.rows;
            bad |= !in_order;
            mine_tiles += tiles[i] = in_order ? static_cast<int>((edge[i + 1] - edge[i] + G::BM - 1) / G::BM) : 0;
        }
        if (bad) atomicOr(a.errw, static_cast<uint32_t>(SANDY_DEVERR_OFFSETS));
        int upto = mine_tiles;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int below = __shfl_up(upto, s, 64);
            if (lane >= s) upto += below;
        }
        return upto;
    };
    int upto = 0;
    if (a.offsets) {
        // the grid has room for the most there can be; the XCDs share what there is (1024 tokens to 8 of 128 experts of
        // 2816 x 704: 118 us where the last XCDs had the empty ones, 98 so)
        int all = 0;
        for (int base = 0; base < a.groups; base += 256) all += __shfl(upto = count(base), 63, 64);
        m_tiles = min(__builtin_amdgcn_readfirstlane(all), m_tiles);
        if (m_tiles <= 0) return;
    }
    // workgroups go to the eight XCDs in turn: each takes a run of tiles, eight rows of tiles high, whose operands
    // its L2 then holds
    const uint32_t total = static_cast<uint32_t>(m_tiles) * n_tiles, per = (total + 7) / 8;
    const uint32_t tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (blockIdx.x >> 3 >= per || tile >= total) return;
    const uint32_t band = tile / (8u * n_tiles), high = min(8u, m_tiles - 8u * band), in = tile - band * 8u * n_tiles;
    const int m_tile = static_cast<int>(8u * band + in % high), n_tile = static_cast<int>(in / high);
    int g = 0, r0 = m_tile * G::BM, end = a.rows;
    if (a.offsets) {
        // the expert of the m_tile-th
        int before = 0;
        g = -1;
        for (int base = 0; base < a.groups && g < 0; base += 256) {
            if (a.groups > 256) upto = count(base);
            const uint64_t here = __ballot(before + upto > m_tile);
            if (here) {
                const int l = __builtin_ctzll(here);
                int at = before + upto - mine_tiles, found = 0, first = 0, past = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool in = m_tile >= at && m_tile < at + tiles[i];
                    found = in ? base + 4 * lane + i : found;
                    first = in ? static_cast<int>(edge[i]) + (m_tile - at) * G::BM : first;
                    past = in ? static_cast<int>(edge[i + 1]) : past;
                    at += tiles[i];
                }
                g = __shfl(found, l, 64);
                r0 = __shfl(first, l, 64);
                end = __shfl(past, l, 64);
            }
            before += __shfl(upto, 63, 64);
        }
        if (g < 0 || r0 < 0 || r0 >= end) return;  // (the latter where offsets are out of order)
        g = __builtin_amdgcn_readfirstlane(g);
        r0 = __builtin_amdgcn_readfirstlane(r0);
        end = __builtin_amdgcn_readfirstlane(end);
    }
    const int n0 = n_tile * G::BN;
    const int xrows = min(G::BM, end - r0), wrows = min(G::BN, a.n - n0);

    // piece i of a thread: 16 bytes of tile row kStep i + tid / 8, x's rows first; rows past the tile's end repeat the last
    // (never stored).  LDS slot p of row r holds the line's piece p ^ (r / 2) % 8: reads of 16 rows meet no bank twice.
    const uint8_t* xbase = a.x + r0 * a.x_pitch;
    const uint8_t* wbase = a.w + g * a.w_group + n0 * a.w_pitch;
    const int k16 = (a.k + 15) & ~15;
    auto buffer = [](const uint8_t* p, int64_t bytes) {
        const uint64_t v = reinterpret_cast<uint64_t>(p);
        i32x4_t r;
        r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(v));
        r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32) & 0xffff);
        r[2] = __builtin_amdgcn_readfirstlane(static_cast<int>(bytes));
        r[3] = 0x00020000;
        return r;
    };
    const i32x4_t xres = buffer(xbase, (xrows - 1) * a.x_pitch + k16), wres = buffer(wbase, (wrows - 1) * a.w_pitch + k16);
    const int prow = tid >> 3, slot = tid & 7;
    auto piece = [&](int i) { return slot ^ (((G::kStep * i + prow) >> 1) & 7); };  // (the same for all i from 16 rows a step on)
    int from[G::kLoads];
#pragma unroll
    for (int i = 0; i < G::kLoads; i++) {
        const bool is_x = i < G::kXLoads;
        const int r = G::kStep * (is_x ? i : i - G::kXLoads) + prow;
        from[i] = static_cast<int>(min(r, (is_x ? xrows : wrows) - 1) * (is_x ? a.x_pitch : a.w_pitch)) + 16 * piece(i);
    }
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)lds));
    auto copy = [&](int c, int stage, int i) {
        const uint32_t to = lds0 + stage * G::kStage + wave * 1024 + i * (16 * G::kThreads);
        copy_to_lds(i < G::kXLoads ? xres : wres, from[i], __builtin_amdgcn_readfirstlane(c * 128), __builtin_amdgcn_readfirstlane(to));
    };
    // The group's whole blocks are first .. first + mine - 1, of all groups' `turns` turns; those past the last are the last
    // again, copied and never read: every round waits for the same number.
    const int chunks = a.k / kQuantBlock, rest = a.k - chunks * kQuantBlock;
    const int turns = (chunks + SPLIT - 1) / SPLIT, first = min(group * turns, max(chunks - 1, 0));
    const int mine = min(turns, chunks - group * turns), last = max(first + mine - 1, first);
    auto issue = [&](int c, int stage) {
#pragma unroll
        for (int i = 0; i < G::kLoads; i++) copy(min(first + c, last), stage, i);
    };
    const int sw = (col >> 1) & 7;
    const int xat = (32 * WM * wm + col) * 128, wat = G::kX + (32 * WN * wn + col) * 128;
    // half i & 1 of operand i / 2 (the weight's first) of the chunk's columns 64 s ..
    auto read1 = [&](int stage, int s, int i, i32x4_t (&xf)[WM][2], i32x4_t (&wf)[WN][2]) {
        const int at = stage * G::kStage + (((4 * s + 2 * half + (i & 1)) ^ sw) << 4);
        if (i < 2 * WN) wf[i / 2][i & 1] = *reinterpret_cast<const i32x4_t*>(lds + wat + 4096 * (i / 2) + at);
        else xf[i / 2 - WN][i & 1] = *reinterpret_cast<const i32x4_t*>(lds + xat + 4096 * (i / 2 - WN) + at);
    };
    constexpr int kReads = 2 * (WM + WN);
    auto frags = [&](int stage, int s, i32x4_t (&xf)[WM][2], i32x4_t (&wf)[WN][2]) {
#pragma unroll
        for (int i = 0; i < kReads; i++) read1(stage, s, i, xf, wf);
    };
    f32x16_t acc[WM][WN];
#pragma unroll
    for (int t = 0; t < WM; t++)
#pragma unroll
        for (int c = 0; c < WN; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[t][c][i] = 0.0f;

    // scale bytes come a run of blocks at a time: a row a thread (or two) from memory, half a segment ahead, through LDS to the
    // lanes that multiply with them
    const uint8_t* xsbase = a.xs + static_cast<int64_t>(r0) * a.blocks;
    const uint8_t* wsbase = a.ws + static_cast<int64_t>(g) * a.w_scale_rows * a.blocks;
    auto scale_row = [&](int r) {
        return r < G::BM ? xsbase + static_cast<int64_t>(min(r, xrows - 1)) * a.blocks
                         : wsbase + static_cast<int64_t>((n0 + min(r - G::BM, wrows - 1)) >> a.w_shift) * a.blocks;
    };
    constexpr int kScaleRows = (G::BM + G::BN + G::kThreads - 1) / G::kThreads;
    constexpr int kRun = G::kRun;
    decltype(some_scales<kRun>(nullptr, 0, 0)) held[kScaleRows];
    auto load_scales = [&](int at) {
#pragma unroll
        for (int u = 0; u < kScaleRows; u++)
            if (G::kThreads * u + tid < G::BM + G::BN) held[u] = some_scales<kRun>(scale_row(G::kThreads * u + tid), first + at, a.blocks);
    };
    auto store_scales = [&](int at) {
#pragma unroll
        for (int u = 0; u < kScaleRows; u++)
            if (G::kThreads * u + tid < G::BM + G::BN)
                *reinterpret_cast<decltype(&held[0])>(lds + G::kScales + (at / kRun & 1) * G::kScaleBytes + (G::kThreads * u + tid) * kRun) = held[u];
    };
    int xs[WM], ws[WN], xs_next[WM], ws_next[WN];
    auto scales = [&](int c) {  // of chunks c .. c + 3, c a multiple of 4
        const unsigned char* at = lds + G::kScales + (c / kRun & 1) * G::kScaleBytes + (c & (kRun - 4));
#pragma unroll
        for (int t = 0; t < WM; t++) xs_next[t] = *reinterpret_cast<const int*>(at + (32 * (WM * wm + t) + col) * kRun);
#pragma unroll
        for (int q = 0; q < WN; q++) ws_next[q] = *reinterpret_cast<const int*>(at + (G::BM + 32 * (WN * wn + q) + col) * kRun);
    };
    auto use_scales = [&] {
#pragma unroll
        for (int t = 0; t < WM; t++) xs[t] = xs_next[t];
#pragma unroll
        for (int c = 0; c < WN; c++) ws[c] = ws_next[c];
    };
    // all products of 64 columns, other(i) before the i-th of WM WN
    auto multiply = [&](const i32x4_t (&xf)[WM][2], const i32x4_t (&wf)[WN][2], auto other) {
        auto both = [](const i32x4_t (&h)[2]) { return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7); };
        if constexpr (kScaled) {
#pragma unroll
            for (int c = 0; c < WN; c++)
#pragma unroll
                for (int t = 0; t < WM; t++) {
                    other(c * WM + t);
                    acc[t][c] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(both(wf[c]), both(xf[t]), acc[t][c], 0, 0, 0, ws[c], 0, xs[t]);
                    __builtin_amdgcn_sched_barrier(0);
                }
        } else {
            Widened xw[WM];
#pragma unroll
            for (int t = 0; t < WM; t++) xw[t] = widen(both(xf[t]), quant_scale(xs[t] & 255));
#pragma unroll
            for (int c = 0; c < WN; c++) {
                const Widened ww = widen(both(wf[c]), quant_scale(ws[c] & 255));
#pragma unroll
                for (int t = 0; t < WM; t++) other(c * WM + t);
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int t = 0; t < WM; t++) acc[t][c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ww.v[s], xw[t].v[s], acc[t][c], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // LDS reads and writes of this wave done, copies but the youngest `left` arrived, then every wave's
    auto meet = [&](auto left) {
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        wait_copies<decltype(left)::value>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // The 2 kTimes products of a chunk c are the clock.  First its second half is read; at kFree it is in every wave's
    // registers, and copies of chunk c + STAGES into its place begin, spread over what is left; at kLand the next chunk
    // has to be in LDS, and its first half is read.
    constexpr int kTimes = WM * WN, kFree = 7 * kTimes / 16, kLand = kTimes + 9 * kTimes / 16;
    constexpr auto when = [](int q) { return kFree + q * (2 * kTimes - kFree) / G::kLoads; };
    constexpr int kIssued = [when] {
        int n = 0;
        while (n < G::kLoads && when(n) <= kLand) n++;
        return n;
    }();
    using Left = std::integral_constant<int, (STAGES - 2) * G::kLoads + kIssued>;
    using First = std::integral_constant<int, (STAGES - 1) * G::kLoads>;

    i32x4_t xf[2][WM][2], wf[2][WN][2];
    if (chunks) {
#pragma unroll
        for (int s = 0; s < STAGES - 1; s++) issue(s, s);
    }
    if (rest) {
        // the last block of a k that is no multiple of 128 goes first, through registers: bytes past k are 0 (all of them
        // for groups but the first)
        const int left = group ? 0 : rest;
        i32x4_t v[G::kLoads];
#pragma unroll
        for (int i = 0; i < G::kLoads; i++) {
            v[i] = i32x4_t{0, 0, 0, 0};
            if (left > 16 * piece(i)) v[i] = *reinterpret_cast<const i32x4_t*>((i < G::kXLoads ? xbase : wbase) + (static_cast<uint32_t>(from[i]) + chunks * 128));
        }
#pragma unroll
        for (int i = 0; i < G::kLoads; i++) {
#pragma unroll
            for (int j = 0; j < 4; j++) v[i][j] &= static_cast<int>(first_bytes(left - 16 * piece(i) - 4 * j));
            *reinterpret_cast<i32x4_t*>(lds + (STAGES - 1) * G::kStage + i * (16 * G::kThreads) + tid * 16) = v[i];
        }
#pragma unroll
        for (int t = 0; t < WM; t++) xs[t] = scale_row(32 * (WM * wm + t) + col)[chunks];
#pragma unroll
        for (int c = 0; c < WN; c++) ws[c] = scale_row(G::BM + 32 * (WN * wn + c) + col)[chunks];
        __syncthreads();
        frags(STAGES - 1, 0, xf[0], wf[0]);
        frags(STAGES - 1, 1, xf[1], wf[1]);
        multiply(xf[0], wf[0], [](int) {});
        multiply(xf[1], wf[1], [](int) {});
        __syncthreads();
    }
    if (chunks) {
        load_scales(0);
        store_scales(0);
        issue(STAGES - 1, STAGES - 1);
        meet(First{});
        frags(0, 0, xf[0], wf[0]);
        scales(0);
        use_scales();
    }
    for (int c = 0, stage = 0; c < mine; c++) {
        const int next = stage + 1 == STAGES ? 0 : stage + 1, then = min(first + c + STAGES, last);
        auto at_slot = [&](int slot) {
            constexpr int kRead = (4 * kReads + kTimes - 1) / kTimes;
#pragma unroll
            for (int q = slot * kRead; q < min((slot + 1) * kRead, kReads); q++) read1(stage, 1, q, xf[1], wf[1]);
            if (slot == kFree) {
                __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
#pragma unroll
            for (int q = 0; q < G::kLoads; q++)
                if (when(q) == slot) copy(then, stage, q);
            if (slot == kLand) meet(Left{});
            if (slot >= kLand)
#pragma unroll
                for (int q = (slot - kLand) * kRead; q < min((slot - kLand + 1) * kRead, kReads); q++) read1(next, 0, q, xf[0], wf[0]);
        };
        multiply(xf[0], wf[0], at_slot);
        constexpr int kLoad = kRun == 8 ? 1 : 6, kStore = kRun == 8 ? 5 : 7;
        if ((c & (kRun - 1)) == kStore) store_scales(c + kRun - kStore);
        if ((c & (kRun - 1)) == kLoad && first + c + kRun - kLoad <= last) load_scales(c + kRun - kLoad);
        if ((c & 3) == 3) scales(c + 1);
        multiply(xf[1], wf[1], [&](int i) { at_slot(kTimes + i); });
        stage = next;
        if ((c & 3) == 3) {
            use_scales();
        } else {
#pragma unroll
            for (int t = 0; t < WM; t++) xs[t] = static_cast<int>(static_cast<uint32_t>(xs[t]) >> 8);
#pragma unroll
            for (int q = 0; q < WN; q++) ws[q] = static_cast<int>(static_cast<uint32_t>(ws[q]) >> 8);
        }
    }
    for (int c = max(mine, 0); c < turns; c++) {  // the other groups' meetings
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_s_barrier();
    }
    wait_copies<0>();  // LDS is used again
    __syncthreads();
    if constexpr (SPLIT > 1) {
        // the groups' sums, in their order
        auto at = [&](int g, int t, int c, int q) {
            return reinterpret_cast<f32x4_t*>(all_lds + g * G::template group_lds<T>()) + ((wave * WM + t) * WN + c) * 256 + 64 * q + lane;
        };
#pragma unroll
        for (int t = 0; t < WM && group; t++)
#pragma unroll
            for (int c = 0; c < WN; c++)
#pragma unroll
                for (int q = 0; q < 4; q++) *at(group, t, c, q) = f32x4_t{acc[t][c][4 * q], acc[t][c][4 * q + 1], acc[t][c][4 * q + 2], acc[t][c][4 * q + 3]};
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int g = 1; g < SPLIT; g++)
#pragma unroll
            for (int t = 0; t < WM; t++)
#pragma unroll
                for (int c = 0; c < WN; c++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const f32x4_t v = *at(g, t, c, q);
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[t][c][4 * q + i] += v[i];
                    }
    }

    // acc[t][c][i]: row 32 t + col, column 32 c + 8 (i / 4) + 4 half + i % 4 of the wave's part: 32 rows at a time through
    // LDS (wave-private) into whole row segments
    using E = typename Vec8<T>::elem;
    constexpr int kRow = G::template row_bytes<T>(), kLanes = 32 * WN * static_cast<int>(sizeof(E)) / 16, kEach = 16 / static_cast<int>(sizeof(E));
    unsigned char* part = lds + wave * 32 * kRow;
    const int mw = 32 * WM * wm, nw = 32 * WN * wn;
    E* out = static_cast<E*>(a.out) + r0 * a.out_pitch + n0;
#pragma unroll
    for (int t = 0; t < WM; t++) {
        if (mw + 32 * t >= xrows) break;
#pragma unroll
        for (int c = 0; c < WN; c++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int at = 32 * c + 8 * q + 4 * half;
                f32x4_t v{acc[t][c][4 * q], acc[t][c][4 * q + 1], acc[t][c][4 * q + 2], acc[t][c][4 * q + 3]};
                if (a.bias)
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] += Vec8<T>::load1(a.bias, min(n0 + nw + at + j, a.n - 1));
                if constexpr (kScaled)
                    *reinterpret_cast<uint2*>(part + col * kRow + 2 * at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
                else
                    *reinterpret_cast<f32x4_t*>(part + col * kRow + 4 * at) = v;
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if constexpr (WHOLE) {
#pragma unroll
            for (int i = 0; i < 32 * kLanes / 64; i++) {
                const int at = 64 * i + lane, r = mw + 32 * t + at / kLanes, n = nw + kEach * (at % kLanes);
                const unsigned char* p = part + at / kLanes * kRow + 16 * (at % kLanes);
                if (r >= xrows || n >= wrows) continue;
                if (n + kEach <= wrows) {
                    __builtin_nontemporal_store(*reinterpret_cast<const i32x4_t*>(p), reinterpret_cast<i32x4_t*>(out + r * a.out_pitch + n));
                } else {
                    for (int j = 0; j < kEach && n + j < wrows; j++) out[r * a.out_pitch + n + j] = reinterpret_cast<const E*>(p)[j];
                }
            }
        } else {
            // rows of other alignments: the 16-byte pieces that memory has, put together from LDS, then what is left of every
            // row on either side, in halves of a piece and so on (2048 x 11263 x 2048: 92 us with stores of one column, 75 so)
            const int most = min(32 * WN, wrows - nw);
            // of a row: where it goes, how far its first boundary is, how many whole pieces follow
            auto pieces = [&](int row, int* lead, int* full) {
                E* const to = out + static_cast<int64_t>(mw + 32 * t + row) * a.out_pitch + nw;
                *lead = static_cast<int>(-(reinterpret_cast<uintptr_t>(to) / sizeof(E)) & (kEach - 1));
                *full = max(most - *lead, 0) / kEach;
                return to;
            };
            int lead, full;
#pragma unroll 1
            for (int at = lane; at < 32 * kLanes; at += 64) {
                const int row = at / kLanes, p = at % kLanes;
                if (mw + 32 * t + row >= xrows) break;
                E* const to = pieces(row, &lead, &full);
                if (p >= full) continue;
                const int e0 = lead + kEach * p;
                const uint32_t* w = reinterpret_cast<const uint32_t*>(part + row * kRow + (e0 * static_cast<int>(sizeof(E)) & ~3));
                i32x4_t v;
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = static_cast<int>(sizeof(E) == 2 && (e0 & 1) ? __builtin_amdgcn_alignbit(w[j + 1], w[j], 16) : w[j]);
                *reinterpret_cast<i32x4_t*>(to + e0) = v;
            }
            if (mw + 32 * t + col < xrows) {  // a lane the near side of a row, another the far
                E* const to = pieces(col, &lead, &full);
                const E* row = reinterpret_cast<const E*>(part + col * kRow);
                if (lead >= most) {
                    for (int e = half; e < most; e += 2) to[e] = row[e];
                } else {
                    int e = half ? lead + full * kEach : 0;
                    const int left = half ? most - e : lead;
#pragma unroll
                    for (int s = 1; s < kEach; s <<= 1) {
                        const int size = half ? kEach / 2 / s : s;  // up to a boundary growing, behind it shrinking
                        if (!(left & size)) continue;
                        if (size == 1) {
                            to[e] = row[e];
                        } else if (size == 2) {
                            const E v[2] = {row[e], row[e + 1]};
                            __builtin_memcpy(__builtin_assume_aligned(to + e, sizeof(v)), v, sizeof(v));
                        } else {
                            const E v[4] = {row[e], row[e + 1], row[e + 2], row[e + 3]};
                            __builtin_memcpy(__builtin_assume_aligned(to + e, sizeof(v)), v, sizeof(v));
                        }
                        e += size;
                    }
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

} // namespace sandy_hip
