// Block-scaled fp8 products of few rows (gfx950): the weights are streamed once, dense or grouped.
//
// Bound: HBM, every weight once per 16 rows. Weights go from memory to the MFMA operands' registers
// with no detour: of each group of 128 values, lane (q, c) = (lane / 16, lane % 16) holds the 16-byte
// pieces q and q + 4 of row c, for rows and weights alike, so a load instruction touches 64 contiguous
// bytes of sixteen rows. Weights are the first operand: a lane ends up with four adjacent columns of
// one row, and the scale xs[row, g] * ws[block, g] is one number a lane and group.
//
// block_rows_kernel holds its rows in registers (16 rows by GPW groups a wave, quantised there
// where they come in 16 or 32 bits) and walks over column fragments with D of them in flight; KS
// waves share K and add their sums in LDS, one barrier per D fragments. block_stream_kernel takes any
// K and reads the rows again for each column fragment. Measured: 1 x 4096 x 4096 8.0 us (2.1 TB/s: one
// work-group a CU, a load's and a join's latency), 24 tokens x 8 of 256 experts, 2048 -> 1024, 65 us (4.4 TB/s);
// a layer's products of 32 tokens x 8, 2048 x 512: 79 us (4.4 TB/s) and 54 us (3.2 TB/s: 128 KB of weights a
// wave, behind the ids, the rows and their quantisation).
#include <algorithm>
#include <type_traits>

#include "fp8_mfma.h"

namespace w4a8 {
namespace {

// Raw bytes of a row's 32 values of one group, as loaded.
template <Src SRC>
constexpr int kSrcBytes = SRC == Src::kFp8 ? 1 : SRC == Src::kF32 ? 4 : 2;
template <Src SRC>
struct RowRaw {
    u32x4 v[2 * kSrcBytes<SRC>];
};
// xp: the lane's row; absent pieces read the last one and are zeroed in row_operand.
template <Src SRC>
__device__ __forceinline__ void row_load(RowRaw<SRC>& r, const uint8_t* xp, int g, int q, int K) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = min(g * kBlk + h * 64 + q * 16, K - 16);
#pragma unroll
        for (int b = 0; b < kSrcBytes<SRC>; ++b)
            r.v[h * kSrcBytes<SRC> + b] = *reinterpret_cast<const u32x4*>(xp + (int64_t)k * kSrcBytes<SRC> + 16 * b);
    }
}
// The MFMA operand; rows in 16 or 32 bits are quantised (the group's absmax lies in four lanes).
template <Src SRC, bool EXACT>
__device__ __forceinline__ GroupOp<EXACT> row_operand(const RowRaw<SRC>& r, int g, int q, int K, float& xs) {
    const bool in[2] = {g * kBlk + q * 16 < K, g * kBlk + 64 + q * 16 < K};
    uint32_t o[8];
    if constexpr (SRC == Src::kFp8) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int d = 0; d < 4; ++d) o[4 * h + d] = in[h] ? r.v[h][d] : 0u;
    } else {
        float f[2][16];
        float m = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                if constexpr (SRC == Src::kF32) {
                    f[h][t] = __uint_as_float(r.v[h * 4 + t / 4][t % 4]);
                } else {
                    const uint32_t u = r.v[h * 2 + t / 8][(t / 2) % 4];
                    if constexpr (SRC == Src::kBf16)
                        f[h][t] = __uint_as_float((t & 1) ? u & 0xFFFF0000u : u << 16);
                    else
                        f[h][t] = __half2float(__ushort_as_half((uint16_t)((t & 1) ? u >> 16 : u & 0xFFFF)));
                }
                f[h][t] = in[h] ? f[h][t] : 0.f;
                m = fmaxf(m, fabsf(f[h][t]));
            }
        }
        xs = act_scale_from_absmax(rows4_max(m));
        const float inv = 1.0f / xs;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int d = 0; d < 4; ++d)
                o[4 * h + d] = pack4_e4m3(f[h][4 * d] * inv, f[h][4 * d + 1] * inv, f[h][4 * d + 2] * inv,
                                               f[h][4 * d + 3] * inv);
    }
    return group_op<EXACT>(u32x4{o[0], o[1], o[2], o[3]}, u32x4{o[4], o[5], o[6], o[7]});
}

// The expert and the end of the rows in use of the 16 rows from row0, c of them this lane's; false:
// nothing to do (blocks of more rows end in whole fragments of padding).
__device__ __forceinline__ bool block_expert(const BlockParams& p, int row0, int c, int& e, int& end) {
    e = 0;
    end = p.P;
    if (p.sorted_ids != nullptr) {
        const int s = p.sorted_ids[min(row0 + c, p.P - 1)];
        e = __builtin_amdgcn_readfirstlane(p.expert_ids[row0 / p.block_m]);
        end = min(p.ntp[0], p.P);
        if (row0 >= end || e < 0 || e >= p.E) return false;
        if (__ballot(row0 + c < end && s >= 0 && s < p.num_valid) == 0) return false;
    }
    return true;
}

// CG groups of KS waves; a group walks over its own `per` column fragments (kSiluF32: fragments of
// the gate half, each with its up fragment), D in flight. part: [2][CG][D][KS][64] v4f in LDS.
template <int GPW, int KS, int CG, int D, Src SRC, Dst DST>
__global__ void __launch_bounds__(64 * KS * CG) block_rows_kernel(BlockParams p, int slices, int per) {
    constexpr bool kSilu = DST == Dst::kSiluF32;
    constexpr bool EXACT = kSilu;
    constexpr int kPair = kSilu ? 2 : 1;                       // fragments of one output fragment
    static_assert(D % kPair == 0, "an output fragment's parts are in flight together");
    constexpr int kUnits = D / kPair;                     // output fragments of one round
    __shared__ __attribute__((aligned(16))) v4f part[KS > 1 ? 2 : 1][KS > 1 ? CG : 1][KS > 1 ? D : 1]
                                                    [KS > 1 ? KS : 1][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = wave % KS, cg = wave / KS;
    const int q = lane >> 4, c = lane & 15;
    const int tb = blockIdx.x / slices, sl = blockIdx.x % slices;
    const int row0 = tb * 16;
    int e, end;
    if (!block_expert(p, row0, c, e, end)) return;
    const int half = p.N / 2;
    const int cols = kSilu ? half : p.N;
    const int K = p.K, G = p.G;
    const int frags = (cols + 15) / 16;
    const int f0 = (sl * CG + cg) * per;                       // first output fragment of this group
    const int g0 = ks * GPW;                                   // first K group of this wave

    // ---- weights: step i is fragment f0 + i / kPair of the gate (i even) or the up half ----
    const uint8_t* we = p.w + (int64_t)e * p.N * K;
    const float* wse = p.ws + (int64_t)e * p.NB * G;
    struct Stage {
        u32x4 w[GPW][2];
        float ws[GPW];
    };
    auto load = [&](Stage& s, int i) __attribute__((always_inline)) {
        const int f = min(f0 + min(i / kPair, per - 1), frags - 1);
        const int up = kSilu && (i & 1) ? half : 0;
        // (columns past the end read the last one; never stored)
        const uint8_t* wr = we + (int64_t)(up + min(f * 16 + c, cols - 1)) * K;
        const float* sr = wse + (int64_t)((up + f * 16) / kBlk) * G;
#pragma unroll
        for (int i = 0; i < GPW; ++i) {
            const int g = min(g0 + i, G - 1);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                s.w[i][h] = *reinterpret_cast<const u32x4*>(wr + min(g * kBlk + h * 64 + q * 16, K - 16));
            s.ws[i] = sr[g];
        }
    };
    Stage ring[D];
#pragma unroll
    for (int d = 0; d < D; ++d) load(ring[d], d);
    __builtin_amdgcn_sched_barrier(0);

    // ---- rows, held ----
    GroupOp<EXACT> x[GPW];
    float xs[GPW];
    int xrow;
    const int slot = block_slot(p, row0 + c, end, xrow);
    const uint8_t* xp = reinterpret_cast<const uint8_t*>(p.x) + (int64_t)xrow * p.ldx * kSrcBytes<SRC>;
    // (some groups' raw bytes at a time: all of them beside the ring would not fit the registers)
    constexpr int kAt = SRC == Src::kF32 ? (GPW < 2 ? GPW : 2) : GPW < 4 ? GPW : 4;
    static_assert(GPW % kAt == 0, "groups divide");
#pragma unroll
    for (int j0 = 0; j0 < GPW; j0 += kAt) {
        RowRaw<SRC> raw[kAt];
#pragma unroll
        for (int j = 0; j < kAt; ++j) {
            const int g = min(g0 + j0 + j, G - 1);
            row_load(raw[j], xp, g, q, K);
            xs[j0 + j] = 0.f;
            if constexpr (SRC == Src::kFp8) xs[j0 + j] = p.xs[(int64_t)xrow * G + g];
        }
#pragma unroll
        for (int j = 0; j < kAt; ++j) {
            // groups past the end: zero rows and a zero scale (what the clamped addresses hold
            // counts in its own group)
            const int g = g0 + j0 + j;
            x[j0 + j] = row_operand<SRC, EXACT>(raw[j], g, q, K, xs[j0 + j]);
            if (g >= G) xs[j0 + j] = 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
    }

    const int mine = min(per, frags - f0);                     // output fragments of this group (may be <= 0)
    const int rounds = (per * kPair + D - 1) / D;              // of the work-group: the barriers agree
    for (int it = 0; it < rounds; ++it) {
        v4f run[D];
#pragma unroll
        for (int d = 0; d < D; ++d) {
            run[d] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < GPW; ++j) {
                const v4f t = group_mfma<EXACT>(group_op<EXACT>(ring[d].w[j][0], ring[d].w[j][1]), x[j]);
                const float s = xs[j] * ring[d].ws[j];
#pragma unroll
                for (int r = 0; r < 4; ++r) run[d][r] = fmaf(t[r], s, run[d][r]);
            }
            __builtin_amdgcn_sched_barrier(0);
            load(ring[d], (it + 1) * D + d);
            __builtin_amdgcn_sched_barrier(0);
        }
        // unit u of the round: an output fragment
        auto put = [&](int u, v4f t, const v4f& up) __attribute__((always_inline)) {
            const int of = it * kUnits + u;
            const int col = (f0 + of) * 16 + 4 * q;
            if constexpr (kSilu) t = silu_mul_f32(t, up);
            if (of >= mine || slot < 0 || col >= cols) return;
            store4<DST>(p, DST == Dst::kSlotF32 ? slot : row0 + c, col, cols, t);
        };
        if constexpr (KS == 1) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) put(u, run[u * kPair], run[u * kPair + kPair - 1]);
        } else {
            auto& buf = part[it & 1][cg];
#pragma unroll
            for (int d = 0; d < D; ++d) buf[d][ks][lane] = run[d];
            lds_barrier();
            // (the next round writes the other buffer; this one is written again behind its barrier)
#pragma unroll
            for (int u0 = 0; u0 < kUnits; u0 += KS) {
                const int u = u0 + ks;
                if (kUnits % KS != 0 && u >= kUnits) break;
                auto total = [&](int d) __attribute__((always_inline)) {
                    v4f t = buf[d][0][lane];
#pragma unroll
                    for (int w = 1; w < KS; ++w) t += buf[d][w][lane];
                    return t;
                };
                const v4f t = total(u * kPair);
                if constexpr (kSilu) put(u, t, total(u * kPair + 1));
                else put(u, t, t);
            }
        }
    }
}

// Any K: KS waves take the K groups in turn (what they read at one time is contiguous along K).
constexpr int kRing = 3;          // groups of a wave in flight
template <int FN, int KS, Src SRC, Dst DST>
__global__ void __launch_bounds__(64 * KS) block_stream_kernel(BlockParams p, int slices) {
    constexpr bool kSilu = DST == Dst::kSiluF32;
    constexpr bool EXACT = kSilu;
    constexpr int kCols = kSilu ? FN / 2 : FN;                 // column fragments of the output
    __shared__ __attribute__((aligned(16))) v4f part[KS][FN][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, c = lane & 15;
    const int tb = blockIdx.x / slices, sl = blockIdx.x % slices;
    const int row0 = tb * 16;
    int e, end;
    if (!block_expert(p, row0, c, e, end)) return;
    const int half = p.N / 2;
    const int cols = kSilu ? half : p.N;
    const int K = p.K, G = p.G;

    const uint8_t* wp[FN];
    const float* wsp[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int f = (sl * kCols + j % kCols) * 16, up = kSilu && j >= kCols ? half : 0;
        wp[j] = p.w + ((int64_t)e * p.N + up + min(f + c, cols - 1)) * K;
        wsp[j] = p.ws + ((int64_t)e * p.NB + (up + min(f, cols - 1)) / kBlk) * G;
    }
    int xrow;
    const int slot = block_slot(p, row0 + c, end, xrow);
    const uint8_t* xp = reinterpret_cast<const uint8_t*>(p.x) + (int64_t)xrow * p.ldx * kSrcBytes<SRC>;
    const float* xsp = p.xs + (SRC == Src::kFp8 ? (int64_t)xrow * G : 0);
    struct Stage {
        u32x4 w[FN][2];
        RowRaw<SRC> x;
        float ws[FN];
        float xs;
    };
    auto load = [&](Stage& s, int step) __attribute__((always_inline)) {
        const int g = min(step * KS + wave, G - 1);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                s.w[j][h] = *reinterpret_cast<const u32x4*>(wp[j] + min(g * kBlk + h * 64 + q * 16, K - 16));
            s.ws[j] = wsp[j][g];
        }
        row_load(s.x, xp, g, q, K);
        if constexpr (SRC == Src::kFp8) s.xs = xsp[g];
    };
    v4f run[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) run[j] = v4f{0.f, 0.f, 0.f, 0.f};
    auto consume = [&](const Stage& s, int step) __attribute__((always_inline)) {
        const int g = step * KS + wave;
        float xs = s.xs;
        const GroupOp<EXACT> xv = row_operand<SRC, EXACT>(s.x, g, q, K, xs);   // zero past the end
        if (g >= G) xs = 0.f;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const v4f t = group_mfma<EXACT>(group_op<EXACT>(s.w[j][0], s.w[j][1]), xv);
            const float sc = xs * s.ws[j];
#pragma unroll
            for (int r = 0; r < 4; ++r) run[j][r] = fmaf(t[r], sc, run[j][r]);
        }
    };
    const int steps = (G + KS - 1) / KS;
    Stage ring[kRing];
#pragma unroll
    for (int d = 0; d < kRing; ++d) load(ring[d], d);
    for (int s0 = 0; s0 < steps; s0 += kRing) {
#pragma unroll
        for (int d = 0; d < kRing; ++d) {
            consume(ring[d], s0 + d);
            __builtin_amdgcn_sched_barrier(0);
            load(ring[d], s0 + d + kRing);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) part[wave][j][lane] = run[j];
    __syncthreads();
    // wave j joins column fragment j (four adjacent columns of a row a lane)
    static_assert(kCols <= KS, "a wave a fragment");
    if (wave >= kCols) return;
    auto total = [&](int f) __attribute__((always_inline)) {
        v4f t = part[0][f][lane];
#pragma unroll
        for (int w = 1; w < KS; ++w) t += part[w][f][lane];
        return t;
    };
    v4f t = total(wave);
    if constexpr (kSilu) t = silu_mul_f32(t, total(kCols + wave));
    const int col = (sl * kCols + wave) * 16 + 4 * q;
    if (slot >= 0 && col < cols) store4<DST>(p, DST == Dst::kSlotF32 ? slot : row0 + c, col, cols, t);
}

int too_many() {
    set_error("fp8 block product: too many tiles");
    return W4A8_ERR_INVALID;
}

template <int FN, int KS, Src SRC, Dst DST>
int go_any(const BlockParams& p, hipStream_t s) {
    constexpr bool silu = DST == Dst::kSiluF32;
    const int cols = silu ? p.N / 2 : p.N, per = 16 * (silu ? FN / 2 : FN);
    const int slices = (cols + per - 1) / per;
    const int64_t grid = (int64_t)((p.P + 15) / 16) * slices;
    if (!grid_fits(grid, 64 * KS)) return too_many();
    launch_kernel(&block_stream_kernel<FN, KS, SRC, DST>, dim3((unsigned)grid), dim3(64 * KS), 0, s, p, slices);
    return check_launch("block_stream_kernel");
}

// per: output fragments a group of waves walks over. The kernel loads D fragments beforehand whatever
// `per` is, so few of them take a variant with a smaller D.
template <int GPW, int KS, int CG, int D, Src SRC, Dst DST>
int launch_rows(const BlockParams& p, int frags, int64_t per, hipStream_t s) {
    constexpr int pair = DST == Dst::kSiluF32 ? 2 : 1;
    if constexpr (D > pair)
        if (per * pair <= D / 2) return launch_rows<GPW, KS, CG, D / 2, SRC, DST>(p, frags, per, s);
    const int slices = (int)((frags + per * CG - 1) / (per * CG));
    const int64_t grid = (int64_t)((p.P + 15) / 16) * slices;
    if (!grid_fits(grid, 64 * KS * CG)) return too_many();
    launch_kernel(&block_rows_kernel<GPW, KS, CG, D, SRC, DST>, dim3((unsigned)grid), dim3(64 * KS * CG), 0, s, p, slices,
                  (int)per);
    return check_launch("block_rows_kernel");
}

// blocks: row blocks expected to hold rows
template <int GPW, int KS, int CG, int D, Src SRC, Dst DST>
int go_rows(const BlockParams& p, int64_t blocks, hipStream_t s) {
    constexpr int unit = D / (DST == Dst::kSiluF32 ? 2 : 1);
    const int frags = ((DST == Dst::kSiluF32 ? p.N / 2 : p.N) + 15) / 16;
    // One round of work-groups (eight waves a CU), each walking over what that leaves it, up to eight
    // rings' worth. us at most 8 / at most 4 / three rounds or more instead of one:
    // 64 experts, 64 rows x 8, 4096 -> 2048: 110 / 118 / 126; layer of 256 experts, 128 tokens x 8: 187 / 208 / 211,
    // 32 tokens: 142 / 140 / 150; 256 experts, 24 tokens x 8, 2048 -> 1024: 61 / 57 / 57.
    const int64_t groups = (int64_t)device_cu_count() * std::max(1, 8 / (KS * CG)) * CG;
    int64_t per = (blocks * frags + groups - 1) / groups;
    if (per > unit) per = std::min<int64_t>((per + unit - 1) / unit, 8) * unit;
    return launch_rows<GPW, KS, CG, D, SRC, DST>(p, frags, std::max<int64_t>(1, per), s);
}

// The wave split by the number of K groups: a wave holds the rows' values of up to four of them (two
// weight fragments of four groups in flight are 64 registers), up to eight waves share K. Beyond 32
// groups (4096 values) rows are read again: 4 x 4096 x 12288 in 15 us, 3.3 TB/s.
template <Src SRC, Dst DST>
int rows16(const BlockParams& p, int64_t blocks, hipStream_t s) {
    if (p.G <= 1) return go_rows<1, 1, 4, 4, SRC, DST>(p, blocks, s);
    if (p.G <= 2) return go_rows<2, 1, 4, 4, SRC, DST>(p, blocks, s);
    if (p.G <= 4) return go_rows<4, 1, 4, 2, SRC, DST>(p, blocks, s);
    if (p.G <= 8) return go_rows<2, 4, 1, 4, SRC, DST>(p, blocks, s);
    if (p.G <= 16) return go_rows<4, 4, 1, 2, SRC, DST>(p, blocks, s);
    if (p.G <= 32) return go_rows<4, 8, 1, 2, SRC, DST>(p, blocks, s);
    return go_any<DST == Dst::kSiluF32 ? 2 : 1, 8, SRC, DST>(p, s);
}

}  // namespace

int launch_block_stream(const BlockArgs& a, hipStream_t s) {
    const BlockParams p = block_params(a);
    if (p.P == 0) return W4A8_OK;
    const int64_t blocks = a.sorted_ids != nullptr ? std::min<int64_t>(std::min(a.P / 16, a.num_valid), a.E + a.num_valid / 16)
                                                   : (a.P + 15) / 16;
    auto out16 = [&](auto src) -> int {
        constexpr Src S = decltype(src)::value;
        if (a.dst == Dst::kF16 || a.dst == Dst::kBf16) return rows16<S, Dst::kF16>(p, blocks, s);
        if (a.dst == Dst::kSiluF32) return rows16<S, Dst::kSiluF32>(p, blocks, s);
        set_error("fp8 block product: output form not taken by the streaming kernel");
        return W4A8_ERR_INVALID;
    };
    switch (a.src) {
        case Src::kFp8: return out16(std::integral_constant<Src, Src::kFp8>{});
        case Src::kF16: return out16(std::integral_constant<Src, Src::kF16>{});
        case Src::kBf16: return out16(std::integral_constant<Src, Src::kBf16>{});
        default: break;
    }
    if (a.dst == Dst::kSlotF32) return rows16<Src::kF32, Dst::kSlotF32>(p, blocks, s);
    set_error("fp8 block product: fp32 rows are the layer's second product's");
    return W4A8_ERR_INVALID;
}

}  // namespace w4a8
