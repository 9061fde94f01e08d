// Block-scaled fp8 products of few rows (gfx950): the weights are streamed once, dense or grouped.
//
// Bound: HBM, every weight once per 16 FT rows. Weights go from memory to the MFMA operands' registers
// with no detour: of each group of 128 values, lane (q, c) = (lane / 16, lane % 16) holds the 16-byte
// pieces q and q + 4 of row c, for rows and weights alike, so a load instruction touches 64 contiguous
// bytes of sixteen rows. Weights are the first operand: a lane ends up with four adjacent columns of
// one row, and the scale xs[row, g] * ws[block, g] is one number a lane and group.
//
// block_rows_kernel holds its rows in registers (16 FT rows by GPW groups a wave, quantised there
// where they come in 16 or 32 bits) and walks over column fragments with D of them in flight; KS
// waves share K and add their sums in LDS, one barrier per D fragments. block_stream_kernel takes any
// K and reads the rows again for each column fragment.
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

// The expert and the end of the rows in use of the rows from row0; false: nothing to do.
__device__ __forceinline__ bool block_expert(const BlockParams& p, int row0, int& e, int& end) {
    e = 0;
    end = p.P;
    if (p.sorted_ids != nullptr) {
        end = min(p.ntp[0], p.P);
        if (row0 >= end) return false;
        e = __builtin_amdgcn_readfirstlane(p.expert_ids[row0 / p.block_m]);
        if (e < 0 || e >= p.E) return false;
    }
    return true;
}

// CG groups of KS waves; a group walks over its own `per` column fragments (kSiluF32: fragments of
// the gate half, each with its up fragment), D in flight. part: [2][CG][D][FT][KS][64] v4f in LDS.
template <int FT, int GPW, int KS, int CG, int D, Src SRC, Dst DST>
__global__ void __launch_bounds__(64 * KS * CG) block_rows_kernel(BlockParams p, int slices, int per) {
    constexpr bool kSilu = DST == Dst::kSiluF32;
    constexpr bool EXACT = kSilu;
    constexpr int kPair = kSilu ? 2 : 1;                       // fragments of one output fragment
    static_assert(D % kPair == 0, "an output fragment's parts are in flight together");
    constexpr int kUnits = D / kPair * FT;                     // output fragments of one round
    __shared__ __attribute__((aligned(16))) v4f part[KS > 1 ? 2 : 1][KS > 1 ? CG : 1][KS > 1 ? D * FT : 1]
                                                    [KS > 1 ? KS : 1][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = wave % KS, cg = wave / KS;
    const int q = lane >> 4, c = lane & 15;
    const int tb = blockIdx.x / slices, sl = blockIdx.x % slices;
    const int row0 = tb * (16 * FT);
    int e, end;
    if (!block_expert(p, row0, e, end)) return;
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
        const int f = min(f0 + i / kPair, frags - 1);
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
    int slot[FT];
    GroupOp<EXACT> x[FT][GPW];
    float xs[FT][GPW];
#pragma unroll
    for (int i = 0; i < FT; ++i) {
        int xrow;
        slot[i] = block_slot(p, row0 + 16 * i + c, end, xrow);
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
                xs[i][j0 + j] = 0.f;
                if constexpr (SRC == Src::kFp8) xs[i][j0 + j] = p.xs[(int64_t)xrow * G + g];
            }
#pragma unroll
            for (int j = 0; j < kAt; ++j) {
                // groups past the end: zero rows and a zero scale (what the clamped addresses hold
                // counts in its own group)
                const int g = g0 + j0 + j;
                x[i][j0 + j] = row_operand<SRC, EXACT>(raw[j], g, q, K, xs[i][j0 + j]);
                if (g >= G) xs[i][j0 + j] = 0.f;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    const int mine = min(per, frags - f0);                     // output fragments of this group (may be <= 0)
    const int rounds = (per * kPair + D - 1) / D;              // of the work-group: the barriers agree
    for (int it = 0; it < rounds; ++it) {
        v4f run[D][FT];
#pragma unroll
        for (int d = 0; d < D; ++d) {
#pragma unroll
            for (int i = 0; i < FT; ++i) {
                run[d][i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < GPW; ++j) {
                    const v4f t = group_mfma<EXACT>(group_op<EXACT>(ring[d].w[j][0], ring[d].w[j][1]), x[i][j]);
                    const float s = xs[i][j] * ring[d].ws[j];
#pragma unroll
                    for (int r = 0; r < 4; ++r) run[d][i][r] = fmaf(t[r], s, run[d][i][r]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load(ring[d], (it + 1) * D + d);
            __builtin_amdgcn_sched_barrier(0);
        }
        // unit u of the round: output fragment u / FT, row fragment u % FT
        auto put = [&](int u, v4f t, const v4f& up, int sl_id) __attribute__((always_inline)) {
            const int of = it * (D / kPair) + u / FT;
            const int col = (f0 + of) * 16 + 4 * q;
            if constexpr (kSilu) {
#pragma unroll
                for (int r = 0; r < 4; ++r) t[r] = silu_mul_f32(t[r], up[r]);
            }
            if (of >= mine || sl_id < 0 || col >= cols) return;
            store4<DST>(p, DST == Dst::kSlotF32 ? sl_id : row0 + 16 * (u % FT) + c, col, cols, t);
        };
        if constexpr (KS == 1) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u)
                put(u, run[u / FT * kPair][u % FT], run[u / FT * kPair + kPair - 1][u % FT], slot[u % FT]);
        } else {
            auto& buf = part[it & 1][cg];
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int i = 0; i < FT; ++i) buf[d * FT + i][ks][lane] = run[d][i];
            lds_barrier();
            // (the next round writes the other buffer; this one is written again behind its barrier)
#pragma unroll
            for (int u0 = 0; u0 < kUnits; u0 += KS) {
                const int u = u0 + ks;
                if (kUnits % KS != 0 && u >= kUnits) break;
                auto total = [&](int d) __attribute__((always_inline)) {
                    v4f t = buf[d * FT + u % FT][0][lane];
#pragma unroll
                    for (int w = 1; w < KS; ++w) t += buf[d * FT + u % FT][w][lane];
                    return t;
                };
                const v4f t = total(u / FT * kPair);
                int sl_id = slot[0];
#pragma unroll
                for (int i = 1; i < FT; ++i)
                    if (u % FT == i) sl_id = slot[i];
                if constexpr (kSilu) put(u, t, total(u / FT * kPair + 1), sl_id);
                else put(u, t, t, sl_id);
            }
        }
    }
}

// Any K: KS waves take the K groups in turn (what they read at one time is contiguous along K).
constexpr int kRing = 3;          // groups of a wave in flight
template <int FT, int FN, int KS, Src SRC, Dst DST>
__global__ void __launch_bounds__(64 * KS) block_stream_kernel(BlockParams p, int slices) {
    constexpr bool kSilu = DST == Dst::kSiluF32;
    constexpr bool EXACT = kSilu;
    constexpr int kCols = kSilu ? FN / 2 : FN;                 // column fragments of the output
    __shared__ __attribute__((aligned(16))) v4f part[KS][FT * FN][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, c = lane & 15;
    const int tb = blockIdx.x / slices, sl = blockIdx.x % slices;
    const int row0 = tb * (16 * FT);
    int e, end;
    if (!block_expert(p, row0, e, end)) return;
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
    const uint8_t* xp[FT];
    const float* xsp[FT];
#pragma unroll
    for (int i = 0; i < FT; ++i) {
        int xrow;
        block_slot(p, row0 + 16 * i + c, end, xrow);
        xp[i] = reinterpret_cast<const uint8_t*>(p.x) + (int64_t)xrow * p.ldx * kSrcBytes<SRC>;
        xsp[i] = p.xs + (SRC == Src::kFp8 ? (int64_t)xrow * G : 0);
    }
    struct Stage {
        u32x4 w[FN][2];
        RowRaw<SRC> x[FT];
        float ws[FN];
        float xs[FT];
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
#pragma unroll
        for (int i = 0; i < FT; ++i) {
            row_load(s.x[i], xp[i], g, q, K);
            if constexpr (SRC == Src::kFp8) s.xs[i] = xsp[i][g];
        }
    };
    v4f run[FT][FN];
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) run[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    auto consume = [&](const Stage& s, int step) __attribute__((always_inline)) {
        const int g = step * KS + wave;
#pragma unroll
        for (int i = 0; i < FT; ++i) {
            float xs = s.xs[i];
            const GroupOp<EXACT> xv = row_operand<SRC, EXACT>(s.x[i], g, q, K, xs);   // zero past the end
            if (g >= G) xs = 0.f;
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const v4f t = group_mfma<EXACT>(group_op<EXACT>(s.w[j][0], s.w[j][1]), xv);
                const float sc = xs * s.ws[j];
#pragma unroll
                for (int r = 0; r < 4; ++r) run[i][j][r] = fmaf(t[r], sc, run[i][j][r]);
            }
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
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) part[wave][i * FN + j][lane] = run[i][j];
    __syncthreads();
    for (int u = tid; u < FT * kCols * 64; u += 64 * KS) {     // four adjacent columns of a row
        const int ln = u & 63, f = u >> 6, i = f / kCols, j = f % kCols;
        auto total = [&](int frag) __attribute__((always_inline)) {
            v4f t = part[0][frag][ln];
#pragma unroll
            for (int w = 1; w < KS; ++w) t += part[w][frag][ln];
            return t;
        };
        v4f t = total(i * FN + j);
        if constexpr (kSilu) {
            const v4f up = total(i * FN + kCols + j);
#pragma unroll
            for (int r = 0; r < 4; ++r) t[r] = silu_mul_f32(t[r], up[r]);
        }
        int xrow;
        const int row = row0 + 16 * i + (ln & 15);
        const int sl_id = block_slot(p, row, end, xrow);
        const int col = (sl * kCols + j) * 16 + 4 * (ln >> 4);
        if (sl_id < 0 || col >= cols) continue;
        store4<DST>(p, DST == Dst::kSlotF32 ? sl_id : row, col, cols, t);
    }
}

int too_many() {
    set_error("fp8 block product: too many tiles");
    return W4A8_ERR_INVALID;
}

template <int FT, int FN, int KS, Src SRC, Dst DST>
int go_any(const BlockParams& p, hipStream_t s) {
    constexpr bool silu = DST == Dst::kSiluF32;
    const int cols = silu ? p.N / 2 : p.N, per = 16 * (silu ? FN / 2 : FN);
    const int slices = (cols + per - 1) / per;
    const int64_t grid = (int64_t)((p.P + 16 * FT - 1) / (16 * FT)) * slices;
    if (grid >= (int64_t)1 << 31) return too_many();
    launch_kernel(&block_stream_kernel<FT, FN, KS, SRC, DST>, dim3((unsigned)grid), dim3(64 * KS), 0, s, p, slices);
    return check_launch("block_stream_kernel");
}

// blocks: row blocks expected to hold rows
template <int FT, int GPW, int KS, int CG, int D, Src SRC, Dst DST>
int go_rows(const BlockParams& p, int64_t blocks, hipStream_t s) {
    constexpr bool silu = DST == Dst::kSiluF32;
    const int frags = ((silu ? p.N / 2 : p.N) + 15) / 16;
    // a work-group a CU and round where there are fewer fragments than that, else some rounds' worth
    // of groups, each with whole rounds of D
    constexpr int unit = D / (silu ? 2 : 1);
    const int64_t want = (int64_t)device_cu_count() * (8 / (KS * CG) > 0 ? 8 / (KS * CG) : 1) * 2;
    int64_t per = (blocks * frags + want * CG - 1) / (want * CG);
    per = std::max<int64_t>(unit, std::min<int64_t>((per + unit - 1) / unit * unit, 4 * unit));
    const int slices = (int)((frags + per * CG - 1) / (per * CG));
    const int64_t grid = (int64_t)((p.P + 16 * FT - 1) / (16 * FT)) * slices;
    if (grid >= (int64_t)1 << 31) return too_many();
    launch_kernel(&block_rows_kernel<FT, GPW, KS, CG, D, SRC, DST>, dim3((unsigned)grid), dim3(64 * KS * CG), 0, s, p,
                  slices, (int)per);
    return check_launch("block_rows_kernel");
}

// FT row fragments: the wave split by the number of K groups.
template <Src SRC, Dst DST>
int rows1(const BlockParams& p, int64_t blocks, hipStream_t s) {
    if (p.G <= 1) return go_rows<1, 1, 1, 4, 4, SRC, DST>(p, blocks, s);
    if (p.G <= 2) return go_rows<1, 2, 1, 4, 4, SRC, DST>(p, blocks, s);
    if (p.G <= 4) return go_rows<1, 4, 1, 4, 2, SRC, DST>(p, blocks, s);
    if (p.G <= 8) return go_rows<1, 2, 4, 1, 4, SRC, DST>(p, blocks, s);
    if (p.G <= 16) return go_rows<1, 4, 4, 1, 2, SRC, DST>(p, blocks, s);
    if (p.G <= 32) return go_rows<1, 4, 8, 1, 2, SRC, DST>(p, blocks, s);
    if constexpr (DST != Dst::kSiluF32)
        if (p.G <= 64) return go_rows<1, 8, 8, 1, 1, SRC, DST>(p, blocks, s);
    return go_any<1, 2, 4, SRC, DST>(p, s);
}

}  // namespace

int launch_block_stream(const BlockArgs& a, hipStream_t s) {
    const BlockParams p = block_params(a);
    if (p.P == 0) return W4A8_OK;
    const int64_t blocks = a.sorted_ids != nullptr ? std::min<int64_t>(std::min(a.P / 16, a.num_valid), a.E + a.num_valid / 16)
                                                   : (a.P + 15) / 16;
    auto out16 = [&](auto src) -> int {
        constexpr Src S = decltype(src)::value;
        if (a.dst == Dst::kF16) return rows1<S, Dst::kF16>(p, blocks, s);
        if (a.dst == Dst::kBf16) return rows1<S, Dst::kBf16>(p, blocks, s);
        if (a.dst == Dst::kSiluF32) return rows1<S, Dst::kSiluF32>(p, blocks, s);
        set_error("fp8 block product: output form not taken by the streaming kernel");
        return W4A8_ERR_INVALID;
    };
    switch (a.src) {
        case Src::kFp8: return out16(std::integral_constant<Src, Src::kFp8>{});
        case Src::kF16: return out16(std::integral_constant<Src, Src::kF16>{});
        case Src::kBf16: return out16(std::integral_constant<Src, Src::kBf16>{});
        default: break;
    }
    if (a.dst == Dst::kSlotF32) return rows1<Src::kF32, Dst::kSlotF32>(p, blocks, s);
    set_error("fp8 block product: fp32 rows are the layer's second product's");
    return W4A8_ERR_INVALID;
}

}  // namespace w4a8
