// int8 products of many rows (gfx950 MFMA), dense or grouped.
//
// A work-group owns BT rows by BN weight rows (columns); per step of 128 k both come straight from memory to LDS
// (16 bytes a lane, no registers), S steps deep. Weights are the first MFMA operand (32 x 32 x 32, whole numbers): a lane
// ends up with sixteen values of one row, which are sixteen adjacent columns, as the weight rows of 32 lie in LDS in an
// order that makes them so.
//
// Work-groups are persistent: a tile's ids are read under the one before, its first steps are loaded under the one
// before's epilogue.
//
// Bound: of few rows HBM (77 rows of 12288 x 4096: 13.6 us, 4 TB/s), of many the matrix cores' power (see dense_go). Of a
// layer's 32768 slots over 256 experts (2048 x 512, rows skewed) the first product takes 173 us (537 MB of weights at
// 3.1 TB/s, x and h beside them), the second 135 (268 MB, and 268 MB of slots' rows written: 4 TB/s).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "int8.h"

namespace w4a8 {
namespace {

using lds_void_ptr = __attribute__((address_space(3))) void*;
using global_cvoid_ptr = const __attribute__((address_space(1))) void*;

constexpr int kTileXcds = 8;
constexpr int kRunRows = 4;       // row tiles of a run: they share its columns' weights

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

__device__ __forceinline__ v16i mfma_i8_32(const u32x4& a, const u32x4& b, const v16i& c) {
    const v4i x{(int)a[0], (int)a[1], (int)a[2], (int)a[3]}, y{(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(x, y, c, 0, 0, 0);
}

// WT x WN waves of FT row fragments x FN column fragments of 32, S steps in LDS; KS such parts of a work-group share
// K, each with slots of its own, and add their sums at the end. EU: waves a SIMD. DEEP: a step's fragments are read
// during the step before (small wave tiles, whose MFMAs of a quarter step take less than an LDS read).
template <int WT_, int WN_, int FT_, int FN_, int S_, int KS_, int EU_, bool DEEP_ = false>
struct Tile {
    static constexpr bool DEEP = DEEP_;
    static constexpr int WT = WT_, WN = WN_, FT = FT_, FN = FN_, S = S_, KS = KS_, EU = EU_;
    static constexpr int kWaves = WT * WN, kThreads = 64 * kWaves;   // of a part
    static constexpr int BT = WT * FT * 32, BN = WN * FN * 32;
    static constexpr int kW = BT * kStep;                        // weights behind the rows
    static constexpr int kSlot = kW + BN * kStep;
    static constexpr int PX = BT * 8 / kThreads, PW = BN * 8 / kThreads;   // 16-byte pieces a thread
    static constexpr int kLoads = PX + PW;                       // of a wave and step
    static_assert(PX * kThreads == BT * 8 && PW * kThreads == BN * 8, "pieces divide");
    static_assert(S >= 2 && S <= 4 && (!DEEP || S % 2 == 0), "two to four slots, for two sets of fragments in turn");
    static_assert(kLoads * (S - 1) < 64, "loads in flight can be counted");
};

template <typename C, Out8 DST, bool TAIL, bool GROUPED>
__global__ void __launch_bounds__(C::kThreads * C::KS, C::EU) int8_tiles_kernel(Int8Params p, int ntiles) {
    constexpr int FT = C::FT, FN = C::FN, BT = C::BT, BN = C::BN, KS = C::KS, S = C::S;
    constexpr bool kSilu = DST == Out8::kSiluF32;
    static_assert(!kSilu || FN % 2 == 0, "gate and up fragments of a wave go together");
    // arrays of their own: the compiler then sees that reads of one do not wait for loads into another
    __shared__ __attribute__((aligned(1024))) int8_t slots0[KS * C::kSlot];
    __shared__ __attribute__((aligned(1024))) int8_t slots1[KS * C::kSlot];
    __shared__ __attribute__((aligned(1024))) int8_t slots2[S > 2 ? KS * C::kSlot : 16];
    __shared__ __attribute__((aligned(1024))) int8_t slots3[S > 3 ? KS * C::kSlot : 16];
    // Tables for the epilogue, in the last slot between a tile's last step and the next one's loads into it.
    int8_t* const aside = S == 2 ? slots1 : S == 3 ? slots2 : slots3;
    float *const s_xs = reinterpret_cast<float*>(aside), *const s_ws = s_xs + BT, *const s_bias = s_ws + BN;
    int* const s_slot = reinterpret_cast<int*>(s_bias + BN);

    // ---- the tiles of this work-group: an XCD takes a contiguous run of them, kRunRows row tiles by all columns
    // each; its work-groups take its tiles in turn ----
    const int xcd = blockIdx.x % kTileXcds, jx = blockIdx.x / kTileXcds, step_items = gridDim.x / kTileXcds;
    const int end = GROUPED ? min(p.ntp[0], p.P) : p.P;
    const int mall = (end + BT - 1) / BT;
    const int items = mall * ntiles, perx = (items + kTileXcds - 1) / kTileXcds;
    const int last = min((xcd + 1) * perx, items);
    int item = xcd * perx + jx;
    if (item >= last) return;

    const int part = KS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / C::kThreads) : 0;
    const int tid = KS > 1 ? threadIdx.x % C::kThreads : threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, c = lane & 31;
    const int wt = wave / C::WN, wn = wave % C::WN;
    const int K = p.K, N = p.N, G = (K + kStep - 1) / kStep;
    const int G1 = (G + KS - 1) / KS, g_first = part * G1;       // steps of a part, the first of them
    auto slot_of = [&](auto i) __attribute__((always_inline)) {      // slot i % S
        constexpr int n = decltype(i)::value % S;
        int8_t* const all = n == 0 ? slots0 : n == 1 ? slots1 : n == 2 ? slots2 : slots3;
        return all + part * C::kSlot;
    };

    // Piece i of a thread is the slot's piece tid + i kThreads: place / 8 and piece % 8. Row r lies at place
    // r ^ ((r >> 3) & 1), its piece j at j ^ (r & 7): the sixteen lanes that a 16-byte LDS read serves at once then read
    // different banks.
    auto piece_row = [&](int i) __attribute__((always_inline)) {
        const int pl = (tid + i * C::kThreads) >> 3;
        return pl ^ ((pl >> 3) & 1);
    };
    auto piece_k = [&](int i) __attribute__((always_inline)) { return ((tid & 7) ^ (piece_row(i) & 7)) * 16; };
    // The column behind row r of the slot's BN: of each 32, MFMA row 8 a + 4 b + d is column 16 b + 4 a + d. kSilu takes
    // FN / 2 fragments of the gate half and the same of the up half.
    const int half = N / 2;
    auto col_of = [&](int ct, int r) __attribute__((always_inline)) {
        const int f = r >> 5, in = (r & 4) * 4 + (r >> 3 & 3) * 4 + (r & 3);
        if constexpr (kSilu) {
            const int w = f / FN, j = f % FN;
            return min(ct * (BN / 2) + (w * (FN / 2) + j % (FN / 2)) * 32 + in, half - 1) + (j >= FN / 2 ? half : 0);
        } else {
            return min(ct * BN + f * 32 + in, N - 1);
        }
    };
    auto place_of = [&](int it, int& row0, int& ct) __attribute__((always_inline)) {
        const int run_items = kRunRows * ntiles, m0 = it / run_items * kRunRows, rem = it % run_items;
        const int rows_here = min(kRunRows, mall - m0);
        row0 = (m0 + rem % rows_here) * BT;
        ct = rem / rows_here;
    };

    // ---- a tile's addresses ----
    int row0, ct, e = 0;
    const int8_t* we = p.w;                                      // the expert's weights
    uint32_t xoff[C::PX], woff[C::PW];
    constexpr int NX = (BT + C::kThreads - 1) / C::kThreads, NW = (BN + C::kThreads - 1) / C::kThreads;
    int ids[C::PX], eid = 0, tids[NX];                           // tids: of the tables' rows
    auto read_ids = [&](int r0) __attribute__((always_inline)) {
        if constexpr (GROUPED) {
            eid = p.expert_ids[r0 / p.block_m];
#pragma unroll
            for (int i = 0; i < C::PX; ++i) ids[i] = p.sorted_ids[min(r0 + piece_row(i), p.P - 1)];
#pragma unroll
            for (int i = 0; i < NX; ++i) tids[i] = p.sorted_ids[min(r0 + tid + i * C::kThreads, p.P - 1)];
        }
    };
    // row r of the tile: the row of x it reads (a row that exists, for rows of no use)
    auto xrow_of = [&](int r, int s) __attribute__((always_inline)) {
        if constexpr (!GROUPED) return (uint32_t)min(r, p.P - 1);
        if (!p.gather) return (uint32_t)min(r, p.x_rows - 1);
        return (uint32_t)(s >= 0 && s < p.num_valid ? s / p.top_k : 0);
    };
    float xs_v[NX], ws_v[NW], bias_v[NW];
    int slot_v[NX];
    auto set_tile = [&]() __attribute__((always_inline)) {
        e = GROUPED ? min(max(__builtin_amdgcn_readfirstlane(eid), 0), p.E - 1) : 0;
        we = p.w + (int64_t)e * N * K;
#pragma unroll
        for (int i = 0; i < C::PX; ++i)
            xoff[i] = xrow_of(row0 + piece_row(i), GROUPED ? ids[i] : 0) * (uint32_t)p.ldx + (uint32_t)piece_k(i);
#pragma unroll
        for (int i = 0; i < C::PW; ++i) woff[i] = (uint32_t)col_of(ct, piece_row(i)) * (uint32_t)K + (uint32_t)piece_k(i);
        // the tile's scales, for its epilogue
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const int row = row0 + tid + i * C::kThreads, s = GROUPED ? tids[i] : row;
            xs_v[i] = p.xs[xrow_of(row, s)];
            slot_v[i] = row < end && s >= 0 && s < p.num_valid ? s : -1;
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int r = (tid + i * C::kThreads) % BN;
            // (column 32 f + n of the tile, not the MFMA row)
            const int n = kSilu ? (r >> 5) % FN : 0;
            const int col = kSilu ? min(ct * (BN / 2) + ((r >> 5) / FN * (FN / 2) + n % (FN / 2)) * 32 + (r & 31), half - 1) +
                                        (n >= FN / 2 ? half : 0)
                                  : min(ct * BN + r, N - 1);
            ws_v[i] = p.ws[(int64_t)e * N + col];
            bias_v[i] = DST == Out8::k16 ? w4a8::bias_at(p, col) : 0.f;
        }
    };

    auto dma = [&](const int8_t* src, int8_t* dst) __attribute__((always_inline)) {
        __builtin_amdgcn_global_load_lds((global_cvoid_ptr)src, (lds_void_ptr)dst, 16, 0, 0);
    };
    // Past the last step every lane reads zeros. TAIL: absent pieces of the last, partial step are zero in both
    // operands. Loads some of parts.
    const int8_t* const zeros = reinterpret_cast<const int8_t*>(g_zero_piece);
    auto issue = [&](int8_t* slot, int g, int some, int parts) __attribute__((always_inline)) {
        const bool is = g < G1 && g_first + g < G;
        const uint32_t on = is ? ~0u : 0u;
        const int gg = g_first + g;
        const uint64_t at = (uint64_t)(uint32_t)gg * kStep;
        const uint64_t far = is ? ~0ull : 0ull, z = reinterpret_cast<uint64_t>(zeros) & ~far;
        const int8_t* xg = reinterpret_cast<const int8_t*>(((reinterpret_cast<uint64_t>(p.x) + at) & far) | z);
        const int8_t* wg = reinterpret_cast<const int8_t*>(((reinterpret_cast<uint64_t>(we) + at) & far) | z);
        asm volatile("" : "+s"(xg), "+s"(wg));                   // (scalar bases, 32-bit offsets)
        int8_t *xd = slot + wave * 1024, *wd = slot + C::kW + wave * 1024;
        auto src = [&](const int8_t* base, uint32_t off, int i) __attribute__((always_inline)) {
            const int8_t* at = base + opaque_u32(off & on);
            if constexpr (TAIL)
                if (gg * kStep + piece_k(i) >= K) at = zeros;
            return at;
        };
#pragma unroll
        for (int i = 0; i < C::PX; ++i)
            if (i * parts / C::kLoads == some) dma(src(xg, xoff[i], i), xd + i * C::kThreads * 16);
#pragma unroll
        for (int i = 0; i < C::PW; ++i)
            if ((C::PX + i) * parts / C::kLoads == some) dma(src(wg, woff[i], i), wd + i * C::kThreads * 16);
    };

    // ---- fragments: lane (h, c) reads piece 2 s + h of row c of each 32, sub-step s of four ----
    const int at0 = (c ^ ((c >> 3) & 1)) * kStep + ((h ^ (c & 7)) << 4);
    constexpr bool DEEP = C::DEEP;
    constexpr int kSets = DEEP ? 8 : 2;                          // sub-steps in registers
    u32x4 xf[kSets][FT], wf[kSets][FN];
    auto frags = [&](const int8_t* slot, int s, int set) __attribute__((always_inline)) {
        const int8_t* b = slot + (at0 ^ (s << 5));
#pragma unroll
        for (int j = 0; j < FN; ++j) wf[set][j] = *reinterpret_cast<const u32x4*>(b + C::kW + (wn * FN + j) * 32 * kStep);
#pragma unroll
        for (int i = 0; i < FT; ++i) xf[set][i] = *reinterpret_cast<const u32x4*>(b + (wt * FT + i) * 32 * kStep);
    };
    v16i run[FT][FN];
    auto multiply = [&](int set, int i0, int i1) __attribute__((always_inline)) {
#pragma unroll
        for (int i = i0; i < i1; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) run[i][j] = mfma_i8_32(wf[set][j], xf[set][i], run[i][j]);
    };
    // Step g from `slot`. Loads are issued in every step, past the last one too, so that those in flight can be
    // counted: the next step's stage has landed for this wave when those of S - 2 later ones are in flight, and for all
    // waves behind the barrier, which also says that none reads `slot` any more. There the loads of step g + S go.
    auto step = [&](int8_t* slot, const int8_t* next, int g, auto odd) __attribute__((always_inline)) {
        if constexpr (DEEP) {
            // its fragments are in registers
            constexpr int now = decltype(odd)::value % 2 * 4, then = 4 - now;
            __builtin_amdgcn_s_waitcnt(wait_vm(C::kLoads * (S - 2)));
            group_barrier();
#pragma unroll
            for (int s = 0; s < 4; ++s) frags(next, s, then + s);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                issue(slot, g + S, s, 4);
                multiply(now + s, 0, FT);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // its first quarter's fragments are in registers
#pragma unroll
            for (int s = 0; s < 3; ++s) {
                frags(slot, s + 1, (s + 1) & 1);
                __builtin_amdgcn_sched_barrier(0);
                multiply(s & 1, 0, FT);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_waitcnt(wait_vm(C::kLoads * (S - 2)));
            group_barrier();
            frags(next, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < FT; ++i) {
                issue(slot, g + S, i, FT);
                multiply(1, i, i + 1);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    place_of(item, row0, ct);
    read_ids(row0);
    set_tile();
    auto each_slot = [&](auto&& f) __attribute__((always_inline)) {
        f(std::integral_constant<int, 0>{});
        f(std::integral_constant<int, 1>{});
        if constexpr (S > 2) f(std::integral_constant<int, 2>{});
        if constexpr (S > 3) f(std::integral_constant<int, 3>{});
    };
    each_slot([&](auto i) __attribute__((always_inline)) { issue(slot_of(i), decltype(i)::value, 0, 1); });
    for (;;) {
        const int r0_now = row0, ct_now = ct, next_item = item + step_items;
        const bool more = next_item < last;
        int row0_next = 0, ct_next = 0;
        if (more) {
            place_of(next_item, row0_next, ct_next);
            read_ids(row0_next);
        }
#pragma unroll
        for (int i = 0; i < FT; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) run[i][j][r] = 0;
        __builtin_amdgcn_s_waitcnt(wait_vm(C::kLoads * (S - 1)));
        group_barrier();
#pragma unroll
        for (int s = 0; s < (DEEP ? 4 : 1); ++s) frags(slot_of(std::integral_constant<int, 0>{}), s, s);
        // (whole rounds of S steps: those past the last one multiply zeros)
        for (int g = 0; g < G1; g += S)
            each_slot([&](auto i) __attribute__((always_inline)) {
                constexpr int n = decltype(i)::value;
                step(slot_of(i), slot_of(std::integral_constant<int, n + 1>{}), g + n, i);
            });
        __builtin_amdgcn_s_waitcnt(wait_vm(0));                  // (the loads past the last step)
        group_barrier();                                         // nobody reads or loads a slot any more
        if constexpr (KS > 1) {
            v4i* sums = reinterpret_cast<v4i*>(slots0);          // [KS - 1][FT FN 4][kThreads]
            static_assert(KS == 1 || (KS - 1) * FT * FN * 4 * C::kThreads * sizeof(v4i) <= C::kSlot * KS, "sums fit");
            if (part > 0)
#pragma unroll
                for (int i = 0; i < FT * FN * 4; ++i) {
                    const v16i& v = run[i / 4 / FN][i / 4 % FN];
                    sums[((part - 1) * FT * FN * 4 + i) * C::kThreads + tid] =
                        v4i{v[i % 4 * 4], v[i % 4 * 4 + 1], v[i % 4 * 4 + 2], v[i % 4 * 4 + 3]};
                }
            lds_barrier();
            if (part == 0)
#pragma unroll
                for (int w = 0; w < KS - 1; ++w)
#pragma unroll
                    for (int i = 0; i < FT * FN * 4; ++i) {
                        const v4i v = sums[(w * FT * FN * 4 + i) * C::kThreads + tid];
#pragma unroll
                        for (int r = 0; r < 4; ++r) run[i / 4 / FN][i / 4 % FN][i % 4 * 4 + r] += v[r];
                    }
            lds_barrier();
        }

        // ---- the next tile's first loads, and this one's epilogue: lane (h, c) holds row 32 i + c, columns 16 h .. 16 h +
        // 15 of each fragment ----
        if (part == 0) {
#pragma unroll
            for (int i = 0; i < NX; ++i) {
                const int r = tid + i * C::kThreads;
                if (r < BT) {
                    s_xs[r] = xs_v[i];
                    s_slot[r] = slot_v[i];
                }
            }
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const int r = tid + i * C::kThreads;
                if (r < BN) {
                    s_ws[r] = ws_v[i];
                    if (DST == Out8::k16) s_bias[r] = bias_v[i];
                }
            }
        }
        if (more) {
            row0 = row0_next;
            ct = ct_next;
            set_tile();
            each_slot([&](auto i) __attribute__((always_inline)) {
                if (decltype(i)::value != S - 1) issue(slot_of(i), decltype(i)::value, 0, 1);
            });
        }
        lds_barrier();
        // A wave turns 32 rows at a time through LDS, so that its stores are whole lines: a row's values lie in
        // chunks of 16 bytes, chunk i of row r at i ^ (r & 15) (rows of 256 bytes or more), i ^ (r / 2 & 7) (of 128) or
        // i ^ (r / 4 & 3) (of 64): sixteen lanes then write to different banks.
        // 16-bit rows of all the wave's columns, fp32 rows of a fragment's.
        constexpr bool k2 = DST == Out8::k16;
        constexpr int kFrags = kSilu ? FN / 2 : FN, kAt = k2 ? kFrags : 1, kSize = k2 ? 2 : 4;
        constexpr int kRowBytes = kAt * 32 * kSize, kChunks = kRowBytes / 16;
        static_assert(kChunks >= 4, "a row is 64 bytes or more");
        static_assert(KS * C::kSlot >= 4 * (2 * BT + 2 * BN) + C::kWaves * 32 * kRowBytes, "tables and rows fit");
        int8_t* const strip = aside + 4 * (2 * BT + 2 * BN) + wave * 32 * kRowBytes;
        auto chunk_at = [&](int row, int i) __attribute__((always_inline)) {
            return row * kRowBytes + ((i ^ (kChunks >= 16 ? row & 15 : kChunks == 8 ? row >> 1 & 7 : row >> 2 & 3)) << 4);
        };
        const int col0 = (ct_now * C::WN + wn) * kFrags * 32;
        // (scales and bias of the lane's columns: held where registers allow, else read again for each 32 rows)
        constexpr bool kHeld = FT <= 2;
        float ws[kHeld ? FN : 1][16], bias[kHeld && DST == Out8::k16 ? FN : 1][16];
        if constexpr (kHeld)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    ws[j][r] = s_ws[(wn * FN + j) * 32 + 16 * h + r];
                    if constexpr (DST == Out8::k16) bias[j][r] = s_bias[(wn * FN + j) * 32 + 16 * h + r];
                }
        auto ws_at = [&](int j, int r) __attribute__((always_inline)) {
            return kHeld ? ws[kHeld ? j : 0][r] : s_ws[(wn * FN + j) * 32 + 16 * h + r];
        };
        auto bias_at = [&](int j, int r) __attribute__((always_inline)) {
            return kHeld ? bias[kHeld && DST == Out8::k16 ? j : 0][r] : s_bias[(wn * FN + j) * 32 + 16 * h + r];
        };
        auto turn_rows = [&](int i, int j0, auto bf16) __attribute__((always_inline)) {
            const float xs = s_xs[(wt * FT + i) * 32 + c];
#pragma unroll
            for (int j = j0; j < j0 + kAt; ++j) {
                float t[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float v = (float)run[i][j][r];
                    if constexpr (kSilu)
                        t[r] = silu_mul(v * (xs * ws_at(j, r)), (float)run[i][j + FN / 2][r] * (xs * ws_at(j + FN / 2, r)));
                    else if constexpr (DST == Out8::k16) t[r] = fmaf(v, xs * ws_at(j, r), bias_at(j, r));
                    else t[r] = v * (xs * ws_at(j, r));
                }
                const int chunk = ((j - j0) * 32 + 16 * h) * kSize / 16;
                if constexpr (k2) {
                    constexpr bool b = decltype(bf16)::value;
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        *reinterpret_cast<u32x4*>(strip + chunk_at(c, chunk + q)) =
                            u32x4{pack16<b>(t[8 * q], t[8 * q + 1]), pack16<b>(t[8 * q + 2], t[8 * q + 3]),
                                  pack16<b>(t[8 * q + 4], t[8 * q + 5]), pack16<b>(t[8 * q + 6], t[8 * q + 7])};
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<v4f*>(strip + chunk_at(c, chunk + q)) =
                            v4f{t[4 * q], t[4 * q + 1], t[4 * q + 2], t[4 * q + 3]};
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto put = [&](int i, int j0) __attribute__((always_inline)) {
            constexpr int kRows = 64 / kChunks;                  // rows of one store
            static_assert(kChunks <= 64 && 32 % kRows == 0, "a store takes whole rows");
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += kRows) {
                const int r = r0 + lane / kChunks, chunk = lane % kChunks;
                const u32x4 v = *reinterpret_cast<const u32x4*>(strip + chunk_at(r, chunk));
                const int slot = s_slot[(wt * FT + i) * 32 + r];
                const int64_t row = DST == Out8::kSlotF32 ? slot : r0_now + (wt * FT + i) * 32 + r;
                const int col = col0 + j0 * 32 + chunk * 16 / kSize;
                if (slot < 0 || col >= (kSilu ? half : N)) continue;
                if constexpr (k2) {
                    if (p.out16 && col + 8 <= N) {
                        *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(p.out) + row * p.ldo + col) = v;
                    } else {
                        const uint32_t w[4] = {v[0], v[1], v[2], v[3]};
                        store16_some<8>(p, row, col, w);
                    }
                } else {                                         // (whole layers: multiples of 64 columns)
                    *reinterpret_cast<u32x4*>(reinterpret_cast<float*>(p.out) + row * p.ldo + col) = v;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
        };
        if (KS == 1 || part == 0) {
#pragma unroll
            for (int i = 0; i < FT; ++i)
#pragma unroll
                for (int j = 0; j < kFrags; j += kAt) {
                    if (DST == Out8::k16 && p.bf16) turn_rows(i, j, std::true_type{});
                    else turn_rows(i, j, std::false_type{});
                    put(i, j);
                }
        }
        if (!more) break;
        item = next_item;
        lds_barrier();                                           // nobody reads the tables any more
        issue(slot_of(std::integral_constant<int, S - 1>{}), S - 1, 0, 1);
    }
}

template <typename C, Out8 DST, bool GROUPED>
int tiles_go(const Int8Params& p, hipStream_t s) {
    constexpr bool silu = DST == Out8::kSiluF32;
    const int cols = silu ? p.N / 2 : p.N, per = silu ? C::BN / 2 : C::BN;
    const int ntiles = (cols + per - 1) / per;
    const int64_t mtiles = (p.P + C::BT - 1) / C::BT;
    if (mtiles * ntiles >= ((int64_t)1 << 30)) {
        set_error("int8 product: too many tiles");
        return W4A8_ERR_INVALID;
    }
    const auto whole = &int8_tiles_kernel<C, DST, false, GROUPED>;
    const auto tail = &int8_tiles_kernel<C, DST, true, GROUPED>;
    const auto kernel = p.K % kStep != 0 ? tail : whole;
    const int threads = C::kThreads * C::KS;
    const int64_t each = std::max(1, blocks_per_cu(reinterpret_cast<const void*>(kernel), threads, 0));
    const int64_t perx = (mtiles * ntiles + kTileXcds - 1) / kTileXcds;
    const int64_t grid = kTileXcds * std::min<int64_t>(perx, std::max<int64_t>(1, each * device_cu_count() / kTileXcds));
    launch_kernel(kernel, dim3((unsigned)grid), dim3(threads), 0, s, p, ntiles);
    return check_launch("int8_tiles_kernel");
}

//                      WT WN FT FN S KS EU
using Tile32x32K4 = Tile<1, 1, 1, 1, 4, 4, 1, true>;
using Tile64x32K2 = Tile<2, 1, 1, 1, 4, 2, 1, true>;
using Tile64x64 = Tile<2, 2, 1, 1, 4, 1, 2, true>;       // two work-groups a CU, the others one
using Tile128x64 = Tile<4, 2, 1, 1, 4, 1, 2, true>;
using Tile128x128 = Tile<2, 4, 2, 1, 4, 1, 2, true>;
using Tile256x128 = Tile<4, 2, 2, 2, 3, 1, 2>;
using Tile256x256 = Tile<2, 4, 4, 2, 2, 1, 2>;
// grouped: the layer's first and second product, blocks of 64 and 128 rows. The first product's waves hold gate and up
// fragments of the same columns; the second one's steps are few, so that waves (eight, two work-groups a CU) hide its
// prologue and stores (with four a layer of 4096 tokens, 256 experts of 2048 x 512, takes as long, 371 us).
using First64 = Tile<1, 4, 2, 2, 2, 1, 2>;
using Second64 = Tile<2, 4, 1, 2, 2, 1, 4>;
using First128 = Tile<2, 4, 2, 2, 3, 1, 2>;
using Second128 = Tile<2, 4, 2, 2, 3, 1, 2>;

// The dense tile of least cost. us as measured at N = K = 4096 (the rule compares tiles at one K, as if all their costs
// grew with it alike), by the tiles a CU has to take:
//                            1/4   1/2   3/4     1   1.5     2     3     4
//   32 x 32, K in four             7.0         14.3*
//   64 x 32, K in two        8.3   8.4         14.7*
//   64 x 64                  9.3   9.4  ...    10.0  14.8  15.6  21.8  28.5
//   128 x 64                10.2  11.5  12.1   13.7  23.4  25.5  36.8  49.8
//   128 x 128               15.0  15.8  18.1   21.2  35.3  40.7        79.2
//   256 x 128               25.5  27.3  30.4   35.9        71.7       218 (6)
//   256 x 256               42.9  44.5         59.0       190.7 (3)
// (* two a CU do not run beside each other.) 8 rows of K = 12288, N = 4096: 32 x 32 11.8, 64 x 32 13.7. What a CU loads into
// LDS bounds the small ones: about 95 bytes a nanosecond with all CUs at it, 120 with few. The largest does 2.25e15
// operations a second (4096 x 12288 x 4096: 183 us), where MFMAs alone on such data, by the card's power, do 3.4e15.
int dense_go(const Int8Params& p, hipStream_t s) {
    const float cus = (float)device_cu_count();
    auto share = [&](int bt, int bn) { return (float)((int64_t)((p.P + bt - 1) / bt) * ((p.N + bn - 1) / bn)) / cus; };
    auto cost = [](float f, float base, float slope, float least, float each) {   // f: tiles a CU
        return f <= 1.f ? std::max(least, base + slope * f) : each * std::ceil(f);
    };
    const float f32x32 = share(32, 32), f32 = share(64, 32), f64 = share(64, 64);
    const float c32x32 = f32x32 <= 1.f ? 7.4f : 1e9f;
    const float c32 = f32 <= 1.f ? 8.4f : 1e9f;
    const float c64 = f64 <= 1.f ? 9.7f : 2.2f + 6.7f * std::ceil(f64);
    const float c128x64 = cost(share(128, 64), 10.4f, 3.2f, 0.f, 12.5f);
    const float c128 = cost(share(128, 128), 10.4f, 10.8f, 15.2f, 20.f);
    const float c256x128 = cost(share(256, 128), 18.f, 18.f, 26.5f, 36.f);
    const float c256 = cost(share(256, 256), 30.f, 29.f, 43.f, 62.f);
    const float best = std::min({c32x32, c32, c64, c128x64, c128, c256x128, c256});
    if (c256 == best) return tiles_go<Tile256x256, Out8::k16, false>(p, s);
    if (c256x128 == best) return tiles_go<Tile256x128, Out8::k16, false>(p, s);
    if (c128 == best) return tiles_go<Tile128x128, Out8::k16, false>(p, s);
    if (c128x64 == best) return tiles_go<Tile128x64, Out8::k16, false>(p, s);
    if (c64 == best) return tiles_go<Tile64x64, Out8::k16, false>(p, s);
    if (c32x32 == best) return tiles_go<Tile32x32K4, Out8::k16, false>(p, s);
    return tiles_go<Tile64x32K2, Out8::k16, false>(p, s);
}

}  // namespace

int launch_int8_tiles(const Int8Args& a, hipStream_t s) {
    const Int8Params p = int8_params(a);
    if (p.P == 0) return W4A8_OK;
    auto grouped = [&](auto first, auto second) -> int {
        if (a.dst == Out8::kSiluF32) return tiles_go<decltype(first), Out8::kSiluF32, true>(p, s);
        return tiles_go<decltype(second), Out8::kSlotF32, true>(p, s);
    };
    if (a.sorted_ids != nullptr) return a.block_m == 128 ? grouped(First128{}, Second128{}) : grouped(First64{}, Second64{});
    return dense_go(p, s);
}

}  // namespace w4a8
