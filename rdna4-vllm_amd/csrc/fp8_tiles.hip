// Block-scaled fp8 products of many rows (gfx950 MFMA), dense or grouped.
//
// A work-group owns BT rows by BN weight rows (columns); per group of 128 k both come straight from
// memory to LDS (16 bytes a lane, no registers), S slots deep. Weights are the first MFMA operand: a
// lane ends up with four adjacent columns of one row, so the scale xs[row, g] * ws[block, g] is one
// number a row fragment, lane and group (a wave's columns lie in one 128-block of the weights).
#include <algorithm>
#include <type_traits>

#include "fp8_block.h"
#include "fp8_mfma.h"

namespace w4a8 {
namespace {

using lds_void_ptr = __attribute__((address_space(3))) void*;
using global_cvoid_ptr = const __attribute__((address_space(1))) void*;

constexpr int kTileXcds = 8;
constexpr int kRunRows = 8;       // row tiles of an XCD's run

// What pieces past the end of K are read from.
__device__ __attribute__((aligned(16))) uint32_t g_zero_piece[4];

// s_waitcnt operand: at most n vector-memory loads in flight, the other counters ignored.
constexpr int wait_vm(int n) { return 0x0F70 | (n & 0xF) | ((n >> 4) << 14); }

// Work-group barrier that no load or store may be moved across and that waits for none of them.
__device__ __forceinline__ void group_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

template <int WT_, int WN_, int FT_, int FN_, int S_>
struct TileCfg {
    static constexpr int WT = WT_, WN = WN_, FT = FT_, FN = FN_, S = S_;
    static constexpr int kWaves = WT * WN, kThreads = 64 * kWaves;
    static constexpr int BT = WT * FT * 16, BN = WN * FN * 16;
    static constexpr int kSlot = (BT + BN) * kBlk + BT * 4;      // rows, weights, row scales
    static constexpr int PX = BT * 8 / kThreads, PW = BN * 8 / kThreads;   // 16-byte pieces a thread
    static_assert(PX * kThreads == BT * 8 && PW * kThreads == BN * 8, "pieces divide");
    static_assert(FN * 16 <= kBlk && kBlk % (FN * 16) == 0, "a wave's columns lie in one block");
    static_assert(BT % 64 == 0, "row scales come 64 at a time");
};

template <typename C, Dst DST, bool EXACT>
__global__ void __launch_bounds__(C::kThreads) block_tiles_kernel(BlockParams p, int mtiles, int ntiles) {
    constexpr int FT = C::FT, FN = C::FN, BT = C::BT, BN = C::BN;
    __shared__ __attribute__((aligned(1024))) uint8_t slot0[C::kSlot];
    __shared__ __attribute__((aligned(1024))) uint8_t slot1[C::kSlot];
    __shared__ __attribute__((aligned(1024))) uint8_t slot2[C::S > 2 ? C::kSlot : 16];

    // ---- the tile: an XCD takes a contiguous run, eight row tiles by all column tiles ----
    const int items = mtiles * ntiles, perx = (items + kTileXcds - 1) / kTileXcds;
    const int jx = blockIdx.x / kTileXcds, item = (int)(blockIdx.x % kTileXcds) * perx + jx;
    if (jx >= perx || item >= items) return;
    const int run_items = kRunRows * ntiles;
    const int m0 = item / run_items * kRunRows, rem = item % run_items;
    const int rows_here = min(kRunRows, mtiles - m0);
    const int row0 = (m0 + rem % rows_here) * BT, col0 = rem / rows_here * BN;

    int e = 0, end = p.P;
    if (p.sorted_ids != nullptr) {
        end = min(p.ntp[0], p.P);
        if (row0 >= end) return;
        e = __builtin_amdgcn_readfirstlane(p.expert_ids[row0 / p.block_m]);
        if (e < 0 || e >= p.E) return;
        end = min(end, (row0 / p.block_m + 1) * p.block_m);     // (a tile of rows lies in one block)
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wt = wave / C::WN, wn = wave % C::WN;
    const int q = lane >> 4, c = lane & 15;
    const int K = p.K, G = p.G, N = p.N;

    // ---- staging: piece i of a thread is row (tid + i kThreads) / 8 of the slot, slot piece tid % 8.
    // Row r lies at place r ^ ((r >> 3) & 1), its piece j at j ^ (r & 7): equal pieces of sixteen rows
    // in different banks.
    const uint8_t* xb = reinterpret_cast<const uint8_t*>(p.x);
    const uint8_t* wb = p.w + ((int64_t)e * N + col0) * K;
    uint32_t xoff[C::PX], woff[C::PW];
    int kx[C::PX], kw[C::PW];                                  // the piece's first k within a group
#pragma unroll
    for (int i = 0; i < C::PX; ++i) {
        const int pr = (tid + i * C::kThreads) >> 3, r = pr ^ ((pr >> 3) & 1);
        int xrow;
        block_slot(p, row0 + r, end, xrow);
        kx[i] = ((tid & 7) ^ (r & 7)) * 16;
        xoff[i] = (uint32_t)xrow * (uint32_t)p.ldx + (uint32_t)kx[i];
    }
#pragma unroll
    for (int i = 0; i < C::PW; ++i) {
        const int pr = (tid + i * C::kThreads) >> 3, r = pr ^ ((pr >> 3) & 1);
        kw[i] = ((tid & 7) ^ (r & 7)) * 16;
        woff[i] = (uint32_t)min(r, N - 1 - col0) * (uint32_t)K + (uint32_t)kw[i];
    }
    int srow;
    block_slot(p, row0 + (wave * 64 + lane) % BT, end, srow);
    const uint32_t soff = (uint32_t)srow * (uint32_t)G * 4u;
    auto put = [&](const uint8_t* src, uint8_t* dst) __attribute__((always_inline)) {
        __builtin_amdgcn_global_load_lds((global_cvoid_ptr)src, (lds_void_ptr)dst, 16, 0, 0);
    };
    // whole: the group is not the last one
    auto issue = [&](uint8_t* slot, int g, auto whole) __attribute__((always_inline)) {
        const uint8_t *xg = xb + g * kBlk, *wg = wb + g * kBlk;
        if (decltype(whole)::value || (g + 1) * kBlk <= K) {
#pragma unroll
            for (int i = 0; i < C::PX; ++i) put(xg + opaque_u32(xoff[i]), slot + (wave * 64 + i * C::kThreads) * 16);
#pragma unroll
            for (int i = 0; i < C::PW; ++i) put(wg + opaque_u32(woff[i]), slot + BT * kBlk + (wave * 64 + i * C::kThreads) * 16);
        } else {
            // the last, partial group: pieces past the end are zero in both operands
            const uint8_t* zero = reinterpret_cast<const uint8_t*>(g_zero_piece);
#pragma unroll
            for (int i = 0; i < C::PX; ++i) put(g * kBlk + kx[i] < K ? xg + xoff[i] : zero, slot + (wave * 64 + i * C::kThreads) * 16);
#pragma unroll
            for (int i = 0; i < C::PW; ++i)
                put(g * kBlk + kw[i] < K ? wg + woff[i] : zero, slot + BT * kBlk + (wave * 64 + i * C::kThreads) * 16);
        }
        // (waves past BT / 64 write what another one writes: every wave has the same count in flight)
        __builtin_amdgcn_global_load_lds((global_cvoid_ptr)(reinterpret_cast<const uint8_t*>(p.xs + g) + opaque_u32(soff)),
                                         (lds_void_ptr)(slot + (BT + BN) * kBlk + (wave * 64 % BT) * 4), 4, 0, 0);
    };
    constexpr int kOps = C::PX + C::PW + 1;

    const float* wsb = p.ws + ((int64_t)e * p.NB + min(col0 + wn * FN * 16, N - 1) / kBlk) * G;

    v4f run[FT][FN];
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) run[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

    const int cr = c ^ (c >> 3);
    const int p0 = (q ^ (c & 7)) << 4, p1 = ((q + 4) ^ (c & 7)) << 4;
    const int x_lane = (wt * FT * 16 + cr) * kBlk, w_lane = BT * kBlk + (wn * FN * 16 + cr) * kBlk;
    const int s_lane = (BT + BN) * kBlk + (wt * FT * 16 + c) * 4;
    auto compute = [&](const uint8_t* slot, float ws) __attribute__((always_inline)) {
        GroupOp<EXACT> xf[FT];
        float s[FT];
#pragma unroll
        for (int i = 0; i < FT; ++i) {
            xf[i] = group_op<EXACT>(*reinterpret_cast<const u32x4*>(slot + x_lane + i * 16 * kBlk + p0),
                                    *reinterpret_cast<const u32x4*>(slot + x_lane + i * 16 * kBlk + p1));
            s[i] = *reinterpret_cast<const float*>(slot + s_lane + i * 64) * ws;
        }
        v4f pend[2][FT];
        auto fold = [&](int j) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < FT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) run[i][j][r] = fmaf(pend[j & 1][i][r], s[i], run[i][j][r]);
        };
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const GroupOp<EXACT> wf = group_op<EXACT>(*reinterpret_cast<const u32x4*>(slot + w_lane + j * 16 * kBlk + p0),
                                                      *reinterpret_cast<const u32x4*>(slot + w_lane + j * 16 * kBlk + p1));
#pragma unroll
            for (int i = 0; i < FT; ++i) pend[j & 1][i] = group_mfma<EXACT>(wf, xf[i]);
            if (j > 0) fold(j - 1);
        }
        fold(FN - 1);
    };
    // One group. Its stage has landed for this wave when no more than the later ones' loads are in
    // flight, and for all waves behind the barrier. With three slots the barrier also says that
    // nobody reads the slot of the group before, which the next loads go to; with two a second one does.
    // LAST: the loads may end before the group does (the compiler counts loads in flight along every
    // path: with the branches in the main loop it would wait for all of them in each round).
    constexpr int kAhead = C::S == 2 ? 1 : C::S - 2;           // later stages in flight at the wait
    auto step = [&](uint8_t* slot, uint8_t* next, int g, float ws, auto last) __attribute__((always_inline)) {
        constexpr bool LAST = decltype(last)::value;
        if (!LAST || g + kAhead < G) __builtin_amdgcn_s_waitcnt(wait_vm(kAhead * kOps));
        else __builtin_amdgcn_s_waitcnt(wait_vm(0));
        group_barrier();
        if constexpr (C::S > 2)
            if (!LAST || g + C::S - 1 < G) issue(next, g + C::S - 1, std::integral_constant<bool, !LAST>{});
        __builtin_amdgcn_sched_barrier(0);
        compute(slot, ws);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (C::S == 2) {
            group_barrier();
            if (!LAST || g + 2 < G) issue(slot, g + 2, std::integral_constant<bool, !LAST>{});
        }
    };
    issue(slot0, 0, std::false_type{});
    if (G > 1) issue(slot1, 1, std::false_type{});
    constexpr int kIssued = C::S == 2 ? 2 : C::S - 1;          // a step issues the group this far on
    constexpr int kSpan = 62 * C::S;                           // groups of a table of weight scales
    int g = 0;
    float wsv[C::S];                                           // lane l: groups base + l S + t
    auto round = [&](int l, auto last) __attribute__((always_inline)) {
        constexpr bool LAST = decltype(last)::value;
        auto ws_of = [&](int t) __attribute__((always_inline)) {
            return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(wsv[t]), l));
        };
        step(slot0, C::S > 2 ? slot2 : slot0, g, ws_of(0), last);
        if (!LAST || g + 1 < G) step(slot1, slot0, g + 1, ws_of(1), last);
        if constexpr (C::S > 2)
            if (!LAST || g + 2 < G) step(slot2, slot1, g + 2, ws_of(2), last);
    };
    int base;
    do {
        base = g;
#pragma unroll
        for (int t = 0; t < C::S; ++t) wsv[t] = wsb[min(base + lane * C::S + t, G - 1)];
        for (; g + C::S + kIssued < G && g < base + kSpan; g += C::S) round((g - base) / C::S, std::false_type{});
    } while (g + C::S + kIssued < G);
    // (at most two rounds are left, and the table reaches two past its span)
    for (; g < G; g += C::S) round((g - base) / C::S, std::true_type{});

    // ---- epilogue: lane (q, c) holds row 16 i + c, columns 4 q .. 4 q + 3 of each fragment ----
#pragma unroll
    for (int i = 0; i < FT; ++i) {
        const int row = row0 + (wt * FT + i) * 16 + c;
        int xrow;
        const int sl = block_slot(p, row, end, xrow);
        if (sl < 0) continue;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int col = col0 + (wn * FN + j) * 16 + 4 * q;
            if (col >= N) continue;
            store4<DST>(p, row, col, N, run[i][j]);
        }
    }
}

template <typename C, Dst DST, bool EXACT>
int tiles_go(const BlockParams& p, hipStream_t s) {
    const int ntiles = (p.N + C::BN - 1) / C::BN, mtiles = (p.P + C::BT - 1) / C::BT;
    const int64_t items = (int64_t)mtiles * ntiles;
    if (items >= (int64_t)1 << 30) {
        set_error("fp8 block product: too many tiles");
        return W4A8_ERR_INVALID;
    }
    launch_kernel(&block_tiles_kernel<C, DST, EXACT>, dim3((unsigned)((items + kTileXcds - 1) / kTileXcds * kTileXcds)),
                  dim3(C::kThreads), 0, s, p, mtiles, ntiles);
    return check_launch("block_tiles_kernel");
}

#ifndef TILE
#define TILE 4, 1, 4, 8, 3
#endif
using Tile256x256 = TileCfg<TILE>;

}  // namespace

int launch_block_tiles(const BlockArgs& a, hipStream_t s) {
    const BlockParams p = block_params(a);
    if (p.P == 0) return W4A8_OK;
    return a.dst == Dst::kBf16 ? tiles_go<Tile256x256, Dst::kBf16, false>(p, s) : tiles_go<Tile256x256, Dst::kF16, false>(p, s);
}

}  // namespace w4a8
