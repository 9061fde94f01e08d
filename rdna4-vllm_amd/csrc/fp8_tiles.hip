// Block-scaled fp8 products of many rows (gfx950 MFMA), dense or grouped.
//
// A work-group owns BT rows by BN weight rows (columns); per group of 128 k both come straight from
// memory to LDS (16 bytes a lane, no registers), three groups deep. Weights are the first MFMA operand: a
// lane ends up with four adjacent columns of one row, so the scale xs[row, g] * ws[block, g] is one
// number a row fragment, lane and group (a wave's columns lie in one 128-block of the weights).
//
// A tile takes any rows of the padded layout: it passes over the experts of its 16-row fragments one
// by one, so blocks of any multiple of 16 rows do.
#include <algorithm>
#include <type_traits>

#include "fp8_mfma.h"

namespace w4a8 {
namespace {

using lds_void_ptr = __attribute__((address_space(3))) void*;
using global_cvoid_ptr = const __attribute__((address_space(1))) void*;

constexpr int kTileXcds = 8;
constexpr int kRunRows = 4;       // row tiles of an XCD's run

// What pieces past the end of K are read from.
__device__ __attribute__((aligned(16))) uint32_t g_zero_piece[4];

// s_waitcnt operand: at most n vector-memory loads and no LDS operation in flight.
constexpr int wait_vm(int n) { return 0x0070 | (n & 0xF) | ((n >> 4) << 14); }

// Work-group barrier that no load or store may be moved across and that waits for none of them.
__device__ __forceinline__ void group_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

constexpr int kSlots = 3;         // groups of k in LDS

// WT x WN waves of FT row fragments x FN column fragments of 16, three groups in LDS; KS such parts of
// a work-group share K, each with slots of its own, and add their sums at the end.
// XB: bytes of a row's value (2: bf16 numbers that hold e4m3 values).
template <int WT_, int WN_, int FT_, int FN_, int KS_ = 1, int XB_ = 1>
struct TileCfg {
    static constexpr int WT = WT_, WN = WN_, FT = FT_, FN = FN_, KS = KS_, XB = XB_;
    static constexpr int kWaves = WT * WN, kThreads = 64 * kWaves;   // of a part
    static constexpr int BT = WT * FT * 16, BN = WN * FN * 16;
    static constexpr int kW = BT * kBlk * XB;                    // weights behind the rows
    static constexpr int kSlot = kW + BN * kBlk;
    static constexpr int PX = BT * 8 * XB / kThreads, PW = BN * 8 / kThreads;   // 16-byte pieces a thread
    static constexpr int kLoads = PX + PW;                       // of a wave and group
    static constexpr int kChunk = 6;                             // groups whose row scales are loaded at once
    static constexpr int PT = (BT * kChunk + kThreads - 1) / kThreads;   // entries a thread
    static_assert(PX * kThreads == BT * 8 * XB && PW * kThreads == BN * 8, "pieces divide");
    static_assert(FN * 16 <= kBlk && kBlk % (FN * 16) == 0, "a wave's columns lie in one block");
    static_assert(kChunk == 2 * kSlots, "two rounds a chunk");
    static_assert(kLoads < 64, "loads in flight can be counted");
};

template <typename C, Dst DST, bool EXACT, bool TAIL, bool GROUPED>
__global__ void __launch_bounds__(C::kThreads * C::KS, 2) block_tiles_kernel(BlockParams p, int ntiles, int run_rows, int cts) {
    constexpr int FT = C::FT, FN = C::FN, BT = C::BT, BN = C::BN;
    constexpr bool kSilu = DST == Dst::kSiluFp8;
    constexpr int KS = C::KS;
    static_assert(!kSilu || BN == 256, "SiLU tiles hold 128 gate and 128 up columns");
    static_assert(C::XB == 1 || (C::XB == 2 && EXACT && !TAIL), "wide rows are for the bf16 matrix cores");
    static_assert(KS == 1 || (DST == Dst::kF16 && !GROUPED), "a divided K is for dense products");
    // arrays of their own: the compiler then sees that reads of one do not wait for loads into another
    __shared__ __attribute__((aligned(1024))) uint8_t slots0[KS * C::kSlot];
    __shared__ __attribute__((aligned(1024))) uint8_t slots1[KS * C::kSlot];
    __shared__ __attribute__((aligned(1024))) uint8_t slots2[KS * C::kSlot];
    __shared__ float s_xs[KS * 2 * C::kChunk * BT];              // row scales [group][row] of two chunks
    __shared__ float s_max[kSilu ? C::WN * BT : 1];              // rows' absmax of a wave's columns

    // ---- the tile. Dense: an XCD takes a contiguous run of them, run_rows row tiles by all columns.
    // Grouped: XCDs take such runs in turn (how many row tiles are in use is known on the device only;
    // a tile finds its rows before it knows, so that the loads below go out together), and a work-group
    // cts column tiles, one after the other: the next one's first loads are under way while it writes. ----
    const int xcd = blockIdx.x % kTileXcds, jx = blockIdx.x / kTileXcds;
    const int mall = (p.P + BT - 1) / BT;
    int m_tile, ct_first;
    if constexpr (GROUPED) {
        const int run_items = run_rows * ((ntiles + cts - 1) / cts), rem = jx % run_items;
        m_tile = (jx / run_items * kTileXcds + xcd) * run_rows + rem % run_rows;
        ct_first = rem / run_rows * cts;
        if (m_tile >= mall) return;
    } else {
        const int run_items = run_rows * ntiles;
        const int items = mall * ntiles, perx = (items + kTileXcds - 1) / kTileXcds, item = xcd * perx + jx;
        if (jx >= perx || item >= items) return;
        const int m0 = item / run_items * run_rows, rem = item % run_items;
        const int rows_here = min(run_rows, mall - m0);
        m_tile = m0 + rem % rows_here;
        ct_first = rem / rows_here;
    }
    const int ct_end = GROUPED ? min(ct_first + cts, ntiles) : ct_first + 1;
    const int row0 = m_tile * BT;
    const int part = KS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / C::kThreads) : 0;
    const int tid = KS > 1 ? threadIdx.x % C::kThreads : threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, c = lane & 15;
    const int K = p.K, G = p.G, N = p.N;
    const int G1 = (G + KS - 1) / KS, g_first = part * G1;       // groups of a part, the first of them
    uint8_t *const slot0 = slots0 + part * C::kSlot, *const slot1 = slots1 + part * C::kSlot;
    uint8_t* const slot2 = slots2 + part * C::kSlot;

    // the expert of fragment `lane`'s rows (-1: none)
    int fe = 0;
    if constexpr (GROUPED) fe = p.expert_ids[min(row0 + 16 * (lane % (BT / 16)), p.P - 1) / p.block_m];
    // row r of the tile: the row of x it reads (a row that exists, for rows of no use)
    auto xrow_of = [&](int r) __attribute__((always_inline)) {
        const int row = min(row0 + r, p.P - 1);
        if constexpr (!GROUPED) return (uint32_t)row;
        if (!p.gather) return (uint32_t)min(row, p.x_rows - 1);
        const int s = p.sorted_ids[row];
        return (uint32_t)(s >= 0 && s < p.num_valid ? min(s / p.top_k, p.x_rows - 1) : 0);
    };
    auto piece_k = [&](int r) __attribute__((always_inline)) {         // the piece's first k within a group
        const int j = (tid & 7) ^ (r & 7);
        return ((j >> 1) | (j & 1) << 2) * 16;
    };
    auto piece_row = [&](int i) __attribute__((always_inline)) {
        const int pr = (tid + i * C::kThreads) >> 3;
        return pr ^ ((pr >> 3) & 1);
    };
    // (entries of a table of row scales past the last one are the last one again)
    auto entry = [&](int i) __attribute__((always_inline)) { return min(tid + i * C::kThreads, BT * C::kChunk - 1); };
    // (rows of two bytes a value: sixteen pieces, piece j of row r at j ^ (r & 15))
    auto xpiece_row = [&](int i) __attribute__((always_inline)) {
        return C::XB == 2 ? (tid + i * C::kThreads) >> 4 : piece_row(i);
    };
    auto xpiece_at = [&](int i) __attribute__((always_inline)) {
        return C::XB == 2 ? ((tid & 15) ^ (xpiece_row(i) & 15)) * 16 : piece_k(piece_row(i));
    };
    uint32_t xoff[C::PX], toff[C::PT];
#pragma unroll
    for (int i = 0; i < C::PX; ++i) xoff[i] = xrow_of(xpiece_row(i));
#pragma unroll
    for (int i = 0; i < C::PT; ++i) toff[i] = xrow_of(entry(i) / C::kChunk);
    const int end = GROUPED ? min(p.ntp[0], p.P) : p.P;
    if (row0 >= end) return;
#pragma unroll
    for (int i = 0; i < C::PX; ++i) xoff[i] = xoff[i] * (uint32_t)p.ldx * C::XB + (uint32_t)xpiece_at(i);
#pragma unroll
    for (int i = 0; i < C::PT; ++i) toff[i] *= (uint32_t)G;
    if (lane >= BT / 16 || row0 + 16 * lane >= end || fe >= p.E) fe = -1;
    const int wt = wave / C::WN, wn = wave % C::WN;
    // the weight row behind row r of the slot's BN: fragment r / 16 belongs to wave r / (16 FN); kSilu
    // takes FN / 2 fragments of the gate half and the same of the up half
    const int half = N / 2;
    auto col_of = [&](int ct, int r) __attribute__((always_inline)) {
        if constexpr (kSilu) {
            const int w = r / (FN * 16), j = r / 16 % FN;
            return ct * kBlk + (w * (FN / 2) + j % (FN / 2)) * 16 + r % 16 + (j >= FN / 2 ? half : 0);
        } else if constexpr (FN % 2 == 0) {
            // (a lane's four columns of two fragments are eight adjacent ones)
            return ct * BN + (r & ~31) + (r % 16 / 4) * 8 + (r / 16 % 2) * 4 + r % 4;
        } else {
            return ct * BN + r;
        }
    };

    uint32_t todo = (uint32_t)__ballot(fe >= 0);                 // row fragments not yet done
    while (todo != 0) {
        const int e = __builtin_amdgcn_readlane(fe, __builtin_ctz(todo));
        const uint32_t now = (uint32_t)__ballot(fe == e) & todo;
        todo &= ~now;

        // ---- staging: piece i of a thread is row (tid + i kThreads) / 8 of the slot, slot piece tid % 8.
        // Row r lies at place r ^ ((r >> 3) & 1), its piece j at (2 (j % 4) + j / 4) ^ (r & 7): the sixteen
        // lanes that a 16-byte LDS read serves at once then read different banks.
        const uint8_t* xb = reinterpret_cast<const uint8_t*>(p.x);
        const uint8_t* wb = p.w + (int64_t)e * N * K;
        uint32_t woff[C::PW];
        auto dma = [&](const uint8_t* src, uint8_t* dst) __attribute__((always_inline)) {
            __builtin_amdgcn_global_load_lds((global_cvoid_ptr)src, (lds_void_ptr)dst, 16, 0, 0);
        };
        int ct = ct_first, turn = 0;
        // The group of k of step g (one that exists, past the last step too). Grouped, rows of a multiple of 4096
        // bytes: column tiles start at groups of their own. In step, work-groups would read the same few memory
        // channels (64 experts, 32 slots each, 4096 -> 2048: 165 us, 3.3 TB/s of weights; 109 so; 2048 -> 1024: 112
        // and 111; a layer of 2048 x 512, 4096 tokens: 471, 478 so). Dense weights are shared by more work-groups,
        // which that would keep apart (2048 x 4096 x 12288: 110 us, 130 so).
        auto group_at = [&](int g) __attribute__((always_inline)) {
            if constexpr (!GROUPED) return min(g_first + g, G - 1);
            const int at = min(g, G - 1) + turn;
            return at < G ? at : at - G;
        };
        // Past the last group every lane reads one piece (nobody reads the slot). TAIL: absent pieces of
        // the last, partial group are zero in both operands.
        auto issue_some = [&](uint8_t* slot, int g, int some, int parts) __attribute__((always_inline)) {
            const uint32_t on = g < G1 && g_first + g < G ? ~0u : 0u;
            const int gg = group_at(g);
            const uint8_t *xg = xb + (int64_t)gg * kBlk * C::XB, *wg = wb + (int64_t)gg * kBlk;
            asm volatile("" : "+s"(xg), "+s"(wg));               // (scalar bases, 32-bit offsets)
            uint8_t *xd = slot + wave * 1024, *wd = slot + C::kW + wave * 1024;
            auto src = [&](const uint8_t* base, uint32_t off, int i) __attribute__((always_inline)) {
                const uint8_t* at = base + opaque_u32(off & on);
                if constexpr (TAIL)
                    if (gg * kBlk + piece_k(piece_row(i)) >= K) at = reinterpret_cast<const uint8_t*>(g_zero_piece);
                return at;
            };
#pragma unroll
            for (int i = 0; i < C::PX; ++i)
                if (i * parts / C::kLoads == some) dma(src(xg, xoff[i], i), xd + i * C::kThreads * 16);
#pragma unroll
            for (int i = 0; i < C::PW; ++i)
                if ((C::PX + i) * parts / C::kLoads == some) dma(src(wg, woff[i], i), wd + i * C::kThreads * 16);
        };
        auto issue = [&](uint8_t* slot, int g) __attribute__((always_inline)) { issue_some(slot, g, 0, 1); };
        // Row scales: kChunk groups at a time, through registers to a table (read group by group, each
        // row's scale is a request of its own: more of them than the rows and weights make together).
        float tv[C::PT];
        auto load_scales = [&](int g0) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < C::PT; ++i)
                tv[i] = p.xs[toff[i] + (uint32_t)group_at(g0 + entry(i) % C::kChunk)];
        };
        auto store_scales = [&](int at) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < C::PT; ++i) s_xs[part * 2 * C::kChunk * BT + at + entry(i) % C::kChunk * BT + entry(i) / C::kChunk] = tv[i];
        };
        const float* wsb = p.ws + (int64_t)e * p.NB * G;
        const float *wsg = wsb, *wsu = wsb;
        auto set_columns = [&]() __attribute__((always_inline)) {
            if (GROUPED && K % 4096 == 0) turn = ct * 5 % G;
#pragma unroll
            for (int i = 0; i < C::PW; ++i)
                woff[i] = (uint32_t)min(col_of(ct, piece_row(i)), N - 1) * (uint32_t)K + (uint32_t)piece_k(piece_row(i));
            wsg = wsb + (int64_t)(min(col_of(ct, wn * FN * 16), N - 1) / kBlk) * G;
            if (kSilu) wsu = wsb + (int64_t)(min(col_of(ct, (wn * FN + FN - 1) * 16), N - 1) / kBlk) * G;
        };
        v4f run[FT][FN];

        const int cr = (c ^ (c >> 3)) * kBlk;
        const int p0 = cr + (((2 * q) ^ (c & 7)) << 4), p1 = cr + (((2 * q + 1) ^ (c & 7)) << 4);
        const int px = c * kBlk * 2 + (((2 * q) ^ c) << 4);      // (wide rows)
        // One group: the rows' fragments against the columns', of which the next is read while one is
        // multiplied and the one before is folded. The loads of group g + 2 are issued between the fragments, into
        // `next`, so that no wave waits for the address unit to take all of them (2048 x 4096 x 12288: 132 -> 102 us).
        // A part's groups past the last one are read as anything and not folded.
        auto compute = [&](const uint8_t* slot, uint8_t* next, int g, int xs_at, float wg, float wu) __attribute__((always_inline)) {
            auto frag = [&](int at, u32x4 (&f)[2]) __attribute__((always_inline)) {
                f[0] = *reinterpret_cast<const u32x4*>(slot + at + p0);
                f[1] = *reinterpret_cast<const u32x4*>(slot + at + p1);
            };
            u32x4 wf[2][2];
            float xs[FT];
            GroupOp<EXACT> xf[FT];
            v4f pend[2][FT];
            const bool on = KS == 1 || g_first + g < G;
            auto fold = [&](int j) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < FT; ++i) {
                    const float s = xs[i] * (kSilu && j >= FN / 2 ? wu : wg);
#pragma unroll
                    for (int r = 0; r < 4; ++r) run[i][j][r] = fmaf(pend[j & 1][i][r], s, run[i][j][r]);
                }
            };
            frag(C::kW + wn * FN * 16 * kBlk, wf[0]);
            if constexpr (C::XB == 2) {
#pragma unroll
                for (int i = 0; i < FT; ++i)
#pragma unroll
                    for (int h = 0; h < 4; ++h)              // pieces 2 q, 2 q + 1, 2 q + 8, 2 q + 9 of the row
                        xf[i].h[h] = *reinterpret_cast<const v8bf*>(slot + (wt * FT + i) * 16 * kBlk * 2 +
                                                                    (px ^ ((h & 1) * 16 + (h >> 1) * 128)));
#pragma unroll
                for (int i = 0; i < FT; ++i) xs[i] = s_xs[xs_at + i * 16];
            } else {
                u32x4 xr[FT][2];
#pragma unroll
                for (int i = 0; i < FT; ++i) frag((wt * FT + i) * 16 * kBlk, xr[i]);
#pragma unroll
                for (int i = 0; i < FT; ++i) xs[i] = s_xs[xs_at + i * 16];
#pragma unroll
                for (int i = 0; i < FT; ++i) xf[i] = group_op<EXACT>(xr[i][0], xr[i][1]);
            }
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if (j + 1 < FN) frag(C::kW + (wn * FN + j + 1) * 16 * kBlk, wf[(j + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
                const GroupOp<EXACT> w = group_op<EXACT>(wf[j & 1][0], wf[j & 1][1]);
#pragma unroll
                for (int i = 0; i < FT; ++i) pend[j & 1][i] = group_mfma<EXACT>(w, xf[i]);
                issue_some(next, g + 2, j, FN);
                if (j > 0 && on) fold(j - 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (on) fold(FN - 1);
        };

        // Group g. Its stage has landed for this wave when no more than the next one's loads are in flight, and
        // for all waves behind the barrier, which also says that nobody reads group g - 1's slot any more, where
        // the next loads go. Loads are issued in every step, past the last group too: the compiler counts those
        // in flight along every path, and would wait for all of them where some path issues none.
        auto step = [&](uint8_t* slot, uint8_t* next, int g, int xs_at, float wg, float wu) __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(wait_vm(C::kLoads));
            group_barrier();
            compute(slot, next, g, xs_at, wg, wu);
            __builtin_amdgcn_sched_barrier(0);
        };
        constexpr int kSpan = 64 * kSlots;                       // groups of a table of weight scales
        float wgv[kSlots], wuv[kSlots];                          // lane l: groups base + l kSlots + t
        auto load_ws = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < kSlots; ++t) {
                const int k = group_at(base + lane * kSlots + t);
                wgv[t] = wsg[k];
                wuv[t] = kSilu ? wsu[k] : 0.f;
            }
        };
        auto hold_ws = [&]() __attribute__((always_inline)) {
            // (waited for here: at their first use, in the loop, the wait would be every round's)
#pragma unroll
            for (int t = 0; t < kSlots; ++t) asm volatile("" : "+v"(wgv[t]), "+v"(wuv[t]));
        };
        const int xs_lane = part * 2 * C::kChunk * BT + wt * FT * 16 + c;
        // A chunk's table is written behind the first round of the chunk before: its last readers are past
        // a barrier by then, and the chunk's own first barrier shows it to everybody.
        set_columns();
        load_scales(0);
        load_ws(0);
        issue(slot0, 0);
        issue(slot1, 1);
      for (;;) {                                                 // column tiles
        hold_ws();
        store_scales(0);
        load_scales(C::kChunk);
#pragma unroll
        for (int i = 0; i < FT; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) run[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
        int g = 0, base = 0;
        // (the ways out of the loop are jumps: with a flag the compiler counts loads in flight along paths
        // from there back into the loop)
        for (int at = 0;; at ^= C::kChunk * BT) {
            if (g - base >= kSpan) {
                base = g;
                load_ws(base);
                hold_ws();
            }
            int l = (g - base) / kSlots, xa = at + xs_lane;
            auto pick = [&](float v) __attribute__((always_inline)) {
                return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), l));
            };
            // three groups
            auto round0 = [&]() __attribute__((always_inline)) { step(slot0, slot2, g, xa, pick(wgv[0]), pick(wuv[0])); };
            auto round1 = [&]() __attribute__((always_inline)) { step(slot1, slot0, g, xa + BT, pick(wgv[1]), pick(wuv[1])); };
            auto round2 = [&]() __attribute__((always_inline)) { step(slot2, slot1, g, xa + 2 * BT, pick(wgv[2]), pick(wuv[2])); };
            round0();
            if (++g == G1) goto summed;
            round1();
            if (++g == G1) goto summed;
            round2();
            if (++g == G1) goto summed;
            store_scales(at ^ (C::kChunk * BT));
            load_scales(g - kSlots + 2 * C::kChunk);
            ++l;
            xa += kSlots * BT;
            round0();
            if (++g == G1) goto summed;
            round1();
            if (++g == G1) goto summed;
            round2();
            if (++g == G1) goto summed;
        }
    summed:
        __builtin_amdgcn_s_waitcnt(wait_vm(0));                  // (the loads past the last group)
        if constexpr (KS > 1) {
            v4f* sums = reinterpret_cast<v4f*>(slots0);          // [KS - 1][FT FN][kThreads]
            static_assert((KS - 1) * FT * FN * C::kThreads * sizeof(v4f) <= C::kSlot * KS, "sums fit");
            group_barrier();                                     // nobody reads or loads a slot any more
#pragma unroll
            for (int i = 0; i < FT * FN; ++i)
                if (part > 0) sums[((part - 1) * FT * FN + i) * C::kThreads + tid] = run[i / FN][i % FN];
            lds_barrier();
            if (part > 0) return;
#pragma unroll
            for (int w = 0; w < KS - 1; ++w)
#pragma unroll
                for (int i = 0; i < FT * FN; ++i) run[i / FN][i % FN] += sums[(w * FT * FN + i) * C::kThreads + tid];
        }

        // ---- the next column tile's first loads, and this one's epilogue: lane (q, c) holds row 16 i + c,
        // columns 4 q .. 4 q + 3 of each fragment ----
        const int at_ct = ct;
        const bool more = GROUPED && ++ct < ct_end;
        if (GROUPED) group_barrier();                            // nobody reads the slots or the tables any more
        if (more) {
            set_columns();
            load_scales(0);
            load_ws(0);
            issue(slot0, 0);
            issue(slot1, 1);
        }
        auto live = [&](int i, int& row) __attribute__((always_inline)) {
            const int f = wt * FT + i;
            row = row0 + f * 16 + c;
            if (!(now >> f & 1) || row >= end) return false;
            if (!GROUPED || p.all_rows) return true;
            const int s = p.sorted_ids[row];
            return s >= 0 && s < p.num_valid && (p.gather ? s / p.top_k : row) < p.x_rows;
        };
        if constexpr (kSilu) {
            // h of this wave's columns; a row's absmax over the 128 is joined over the waves in LDS
            float top[FT];
#pragma unroll
            for (int i = 0; i < FT; ++i) {
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < FN / 2; ++j) {
                    run[i][j] = silu_mul_f32(run[i][j], run[i][j + FN / 2]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(run[i][j][r]));
                }
                top[i] = rows4_max(m);
            }
#pragma unroll
            for (int i = 0; i < FT; ++i)
                if (q == 0) s_max[wn * BT + (wt * FT + i) * 16 + c] = top[i];
            lds_barrier();
#pragma unroll
            for (int i = 0; i < FT; ++i) {
                float m = s_max[(wt * FT + i) * 16 + c];
#pragma unroll
                for (int w = 1; w < C::WN; ++w) m = fmaxf(m, s_max[w * BT + (wt * FT + i) * 16 + c]);
                const float sc = act_scale_from_absmax(m), inv = 1.0f / sc;
                int row;
                if (!live(i, row)) continue;
#pragma unroll
                for (int j = 0; j < FN / 2; ++j)
                    *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out) + (int64_t)row * p.ldo +
                                                 col_of(at_ct, (wn * FN + j) * 16 + 4 * q)) =
                        pack4_e4m3(run[i][j][0] * inv, run[i][j][1] * inv, run[i][j][2] * inv, run[i][j][3] * inv);
                if (wn == 0 && q == 0) p.out_scales[(int64_t)row * (half / kBlk) + at_ct] = sc;
            }
        } else if constexpr (DST == Dst::kRowF16) {
            // a row's largest finite value of this wave's columns to [2^14, 2^15): infinities, NaN and zeros as they are
#pragma unroll
            for (int i = 0; i < FT; ++i) {
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v = fabsf(run[i][j][r]);
                        m = fmaxf(m, v < INFINITY ? v : 0.f);
                    }
                const uint32_t eb = __float_as_uint(rows4_max(m)) >> 23;
                const uint32_t sb = eb == 0 ? 127u : eb > 15 ? eb - 14 : 1u;
                const float inv = __uint_as_float((254u - sb) << 23);
                int row;
                if (!live(i, row)) continue;
#pragma unroll
                for (int j = 0; j < FN; ++j) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) run[i][j][r] *= inv;
                    if (j % 2 == 0) continue;
                    const int col = col_of(at_ct, (wn * FN + j - 1) * 16 + 4 * q);  // (whole tiles: N % 128 == 0)
                    store16x8(p, row, col, run[i][j - 1], run[i][j], false);
                    if (q == 0) p.out_scales[(int64_t)row * (N / 32) + col / 32] = __uint_as_float(sb << 23);
                }
            }
        } else if constexpr (DST == Dst::kSlotF32) {
#pragma unroll
            for (int i = 0; i < FT; ++i) {
                int row;
                if (!live(i, row)) continue;                     // (padding has no slot)
                const int slot = p.sorted_ids[row];
#pragma unroll
                for (int j = 0; j < FN; ++j)                     // (whole tiles: N % 128 == 0)
                    store4<DST>(p, slot, col_of(at_ct, (wn * FN + j) * 16 + 4 * q), N, run[i][j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < FT; ++i) {
                int row;
                if (!live(i, row)) continue;
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    const int col = col_of(at_ct, (wn * FN + j) * 16 + 4 * q);
                    if (FN % 2 == 0 && p.out16 && p.ldo % 8 == 0) {
                        if (j % 2 == 1 && col < N) store16x8(p, row, col - 4, run[i][j - 1], run[i][j], p.out_bf16 != 0);
                    } else if (col < N) {
                        store16(p, row, col, N, run[i][j], p.out_bf16 != 0);
                    }
                }
            }
        }
        if (!more) break;
      }
    }
}

template <typename C, Dst DST, bool GROUPED>
int tiles_go(const BlockParams& p, hipStream_t s) {
    constexpr bool silu = DST == Dst::kSiluFp8;
    const int ntiles = silu ? p.N / 2 / kBlk : (p.N + C::BN - 1) / C::BN, mtiles = (p.P + C::BT - 1) / C::BT;
    const int run_rows = std::min(kRunRows, mtiles);
    const int64_t runs = (mtiles + run_rows - 1) / run_rows;
    // Grouped: two column tiles a work-group where that leaves four rounds or more of them (a layer's
    // products of 4096 tokens x 8, 256 experts: 260 -> 247 and 180 -> 162 us; four tiles: 279 and 167; 256 x 8
    // slots of 8 experts, one round: 79 -> 83).
    const int64_t passes = p.num_valid / C::BT + std::min(p.E, p.num_valid);
    const int cts = GROUPED && ntiles > 1 && passes * ntiles >= 4 * (int64_t)device_cu_count() * (512 / C::kThreads) ? 2 : 1;
    const int sets = (ntiles + cts - 1) / cts;
    const int64_t items = GROUPED ? (runs + kTileXcds - 1) / kTileXcds * kTileXcds * run_rows * sets
                                  : ((int64_t)mtiles * ntiles + kTileXcds - 1) / kTileXcds * kTileXcds;
    if (!grid_fits(items, C::kThreads * C::KS)) {
        set_error("fp8 block product: too many tiles");
        return W4A8_ERR_INVALID;
    }
    const dim3 grid((unsigned)items);
    if constexpr (DST == Dst::kF16)
        if (p.K % kBlk != 0) {
            launch_kernel(&block_tiles_kernel<C, DST, silu, true, GROUPED>, grid, dim3(C::kThreads * C::KS), 0, s, p, ntiles, run_rows, cts);
            return check_launch("block_tiles_kernel");
        }
    launch_kernel(&block_tiles_kernel<C, DST, silu, false, GROUPED>, grid, dim3(C::kThreads * C::KS), 0, s, p, ntiles, run_rows, cts);
    return check_launch("block_tiles_kernel");
}

using Tile64x32K4 = TileCfg<2, 2, 2, 1, 4>;  // sixteen waves, one work-group a CU
using Tile64x32K2 = TileCfg<2, 2, 2, 1, 2>;  // eight waves, two work-groups a CU
using Tile64x64K2 = TileCfg<1, 4, 4, 1, 2>;  // eight waves, one work-group a CU
using Tile64x64 = TileCfg<1, 4, 4, 1>;       // four, three
using Tile64x128 = TileCfg<1, 4, 4, 2>;      // four, two
using Tile256x128 = TileCfg<4, 2, 4, 4>;     // eight, one
// Rows in bf16: converting them in each of the eight waves takes two thirds of the conversions (layer of 4096
// tokens, 256 experts: first product 247 -> 231 us; 1111 tokens x 6, 64 experts, the whole layer: 150 -> 142).
using TileSilu = TileCfg<1, 8, 4, 2, 1, 2>;  // 64 x 256: eight, one

// The dense tile of least cost. us as measured at K = 4096 (the rule compares tiles at one K, as if all their
// costs grew with it alike; other K were timed for the chosen tiles only):
//   work-groups a CU:    <= 1     2     3     4     8
//   64 x 64, K in two     12    24
//   64 x 64               14    19    29    36    64
//   64 x 128              20    28    52    54
//   256 x 128          34-42    84
// 64 rows x 64 columns alone are bound by what one CU has under way (45 GB/s), so where they leave CUs idle half
// the columns and K in two or four parts: 64 x 4096 x 4096 64 x 64 14.7, K in two 12.2, 64 x 32 in two 10.8, in four
// 9.6; 17 x 2048 x 12288 35 / 26 / 23 / 16; 48 x 1024 x 1024 (8 groups) 5.3 / 5.3 / 4.6 / 5.3. The largest tile is
// bound by what LDS gives the matrix cores (2048 x 4096 x 12288: 2.0 PFLOP/s).
int dense_go(const BlockParams& p, hipStream_t s) {
    const int64_t cus = device_cu_count();
    auto tiles = [&](int bt, int bn) { return (int64_t)((p.P + bt - 1) / bt) * ((p.N + bn - 1) / bn); };
    const int64_t n64 = tiles(64, 64), n128 = tiles(64, 128), n256 = tiles(256, 128);
    if (tiles(64, 32) <= cus)
        return p.G > 16 ? tiles_go<Tile64x32K4, Dst::kF16, false>(p, s) : tiles_go<Tile64x32K2, Dst::kF16, false>(p, s);
    if (n64 <= cus) return tiles_go<Tile64x64K2, Dst::kF16, false>(p, s);
    const int64_t t64 = std::max<int64_t>(14 * cus, 9 * n64);
    const int64_t t128 = n128 <= cus ? 20 * cus : (n128 + 2 * cus - 1) / (2 * cus) * 27 * cus;
    const int64_t t256 = n256 <= cus ? 34 * cus + 8 * n256 : (n256 + cus - 1) / cus * 42 * cus;
    if (t256 <= std::min(t64, t128)) return tiles_go<Tile256x128, Dst::kF16, false>(p, s);
    if (t128 <= t64) return tiles_go<Tile64x128, Dst::kF16, false>(p, s);
    return tiles_go<Tile64x64, Dst::kF16, false>(p, s);
}

}  // namespace

bool block_tiles_supported(const BlockArgs& a) {
    // rows, scales and an expert's weights are addressed in 32 bits
    const int64_t lim = (int64_t)1 << 32;
    const bool silu = a.dst == Dst::kSiluFp8;
    return a.src == (silu ? Src::kWide : Src::kFp8) && a.x_rows * a.ldx * (silu ? 2 : 1) < lim && a.x_rows * blk_groups(a.K) * 4 < lim && a.N * a.K < lim &&
           (a.dst == Dst::kF16 || a.dst == Dst::kBf16 ||
            ((a.dst == Dst::kRowF16 || (a.dst == Dst::kSlotF32 && !a.all_rows)) && a.sorted_ids != nullptr &&
             a.K % kBlk == 0 && a.N % kBlk == 0) ||
            (silu && a.sorted_ids != nullptr && a.K % kBlk == 0 && a.N % (2 * kBlk) == 0));
}

int launch_block_tiles(const BlockArgs& a, hipStream_t s) {
    const BlockParams p = block_params(a);
    if (p.P == 0) return W4A8_OK;
    if (!block_tiles_supported(a)) {
        set_error("fp8 block product: sizes not taken by the tiles");
        return W4A8_ERR_INVALID;
    }
    if (a.dst == Dst::kSiluFp8) return tiles_go<TileSilu, Dst::kSiluFp8, true>(p, s);
    if (a.dst == Dst::kRowF16) return tiles_go<Tile64x128, Dst::kRowF16, true>(p, s);
    if (a.dst == Dst::kSlotF32) return tiles_go<Tile64x128, Dst::kSlotF32, true>(p, s);
    if (a.sorted_ids != nullptr) return tiles_go<Tile64x128, Dst::kF16, true>(p, s);
    return dense_go(p, s);
}

}  // namespace w4a8
