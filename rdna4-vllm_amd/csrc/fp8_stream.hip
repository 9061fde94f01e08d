// Block-scaled fp8 products that stream the weights (gfx950 fp8 MFMA): few rows, dense or grouped.
//
// A work-group owns 16 FT rows and 16 FN columns; its waves take the K groups in turn (wave w the
// groups w, w + waves, ...: what they read at one time is contiguous along K) and add their sums in
// LDS, in wave order. Weights and e4m3 rows go from memory to the MFMA operands' registers with no
// detour: of each group of 128 values, lane (q, c) = (lane / 16, lane % 16) holds the 16-byte pieces
// q and q + 4 of row c, for rows and weights alike, so a load instruction touches 64 contiguous bytes
// of sixteen rows. Weights are the first operand: a lane ends up with four adjacent columns of one row,
// and the scale xs[row, g] * ws[block, g] is one number a lane and group.
// Bound: HBM (every weight once per 16 FT rows).
#include <algorithm>
#include <type_traits>

#include "fp8_block.h"

namespace w4a8 {
namespace {

constexpr int kRing = 3;          // groups of a wave in flight

template <int FT, int FN, int KS, Src SRC, Dst DST, bool TAIL>
__global__ void __launch_bounds__(64 * KS) block_stream_kernel(BlockParams p, int slices) {
    // kSiluF32: the column fragments are FN / 2 of the gate half and the matching ones of the up half
    constexpr bool kSilu = DST == Dst::kSiluF32;
    constexpr int kCols = kSilu ? FN / 2 : FN;                 // column fragments of the output
    __shared__ __attribute__((aligned(16))) v4f part[KS][FT * FN][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, c = lane & 15;
    const int tb = blockIdx.x / slices, sl = blockIdx.x % slices;
    const int row0 = tb * (16 * FT);
    int e = 0, end = p.P;
    if (p.sorted_ids != nullptr) {
        end = min(p.ntp[0], p.P);
        if (row0 >= end) return;
        e = p.expert_ids[row0 / p.block_m];
        if (e < 0 || e >= p.E) return;
    }
    const int half = p.N / 2;
    const int cols = kSilu ? half : p.N;
    const int K = p.K, G = p.G;

    const uint8_t* wp[FN];
    const float* wsp[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        // columns past the end read the last one (never stored)
        const int col = min((sl * kCols + j % kCols) * 16 + c, cols - 1) + (kSilu && j >= kCols ? half : 0);
        const int blk = min((sl * kCols + j % kCols) * 16, cols - 1) + (kSilu && j >= kCols ? half : 0);
        wp[j] = p.w + ((int64_t)e * p.N + col) * K;
        // (kSiluF32 takes halves of whole blocks, and blocks are a multiple of 16 columns)
        wsp[j] = p.ws + ((int64_t)e * p.NB + blk / kBlk) * G;
    }
    int slot[FT];
    const uint8_t* xp[FT];
    const float* xsp[FT];
    constexpr int kBytes = SRC == Src::kFp8 ? 1 : SRC == Src::kF32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < FT; ++i) {
        int xrow;
        slot[i] = block_slot(p, row0 + 16 * i + c, end, xrow);
        xp[i] = reinterpret_cast<const uint8_t*>(p.x) + (int64_t)xrow * p.ldx * kBytes;
        xsp[i] = p.xs + (SRC == Src::kFp8 ? (int64_t)xrow * G : 0);
    }

    struct Stage {
        u32x4 w[FN][2];
        u32x4 x[FT][2 * kBytes];
        float ws[FN];
        float xs[FT];
    };
    // the group of step i; past the end the last one, whose result is scaled by 0
    auto load = [&](Stage& s, int step) __attribute__((always_inline)) {
        const int g = min(step * KS + wave, G - 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int k = g * kBlk + h * 64 + q * 16;
            if constexpr (TAIL) k = min(k, K - 16);
#pragma unroll
            for (int j = 0; j < FN; ++j) s.w[j][h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp[j] + k));
#pragma unroll
            for (int i = 0; i < FT; ++i)
#pragma unroll
                for (int b = 0; b < kBytes; ++b)
                    s.x[i][h * kBytes + b] = *reinterpret_cast<const u32x4*>(xp[i] + (int64_t)k * kBytes + 16 * b);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) s.ws[j] = wsp[j][g];
        if constexpr (SRC == Src::kFp8) {
#pragma unroll
            for (int i = 0; i < FT; ++i) s.xs[i] = xsp[i][g];
        }
    };
    // a row's 32 values of this lane as an MFMA operand, and their scale
    auto operand = [&](const Stage& s, int i, int g, float& xs) __attribute__((always_inline)) {
        bool in[2] = {true, true};
        if constexpr (TAIL) {
            in[0] = g * kBlk + q * 16 < K;
            in[1] = g * kBlk + 64 + q * 16 < K;
        }
        v8i o;
        if constexpr (SRC == Src::kFp8) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int d = 0; d < 4; ++d) o[4 * h + d] = in[h] ? (int)s.x[i][h][d] : 0;
            xs = s.xs[i];
        } else {
            float f[2][16];
            float m = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int t = 0; t < 16; ++t) {
                    if constexpr (SRC == Src::kF32) {
                        f[h][t] = __uint_as_float(s.x[i][h * 4 + t / 4][t % 4]);
                    } else {
                        const uint32_t u = s.x[i][h * 2 + t / 8][(t / 2) % 4];
                        if constexpr (SRC == Src::kBf16)
                            f[h][t] = __uint_as_float((t & 1) ? u & 0xFFFF0000u : u << 16);
                        else
                            f[h][t] = __half2float(__ushort_as_half((uint16_t)((t & 1) ? u >> 16 : u & 0xFFFF)));
                    }
                    if constexpr (TAIL) f[h][t] = in[h] ? f[h][t] : 0.f;
                    m = fmaxf(m, fabsf(f[h][t]));
                }
            }
            xs = act_scale_from_absmax(rows4_max(m));
            const float inv = 1.0f / xs;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    o[4 * h + d] = (int)pack4_e4m3(as_f32(f[h][4 * d] * inv), as_f32(f[h][4 * d + 1] * inv),
                                                   as_f32(f[h][4 * d + 2] * inv), as_f32(f[h][4 * d + 3] * inv));
        }
        return o;
    };

    v4f run[FT][FN];
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) run[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    auto consume = [&](const Stage& s, int step) __attribute__((always_inline)) {
        const int g = step * KS + wave;
        v8i wv[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                wv[j][d] = (int)s.w[j][d / 4][d % 4];
                // both operands of absent pieces are zero: what the clamped address holds may be NaN
                if constexpr (TAIL) wv[j][d] = g * kBlk + (d / 4) * 64 + q * 16 < K ? wv[j][d] : 0;
            }
#pragma unroll
        for (int i = 0; i < FT; ++i) {
            float xs;
            const v8i xv = operand(s, i, g, xs);
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const v4f t = mfma_16x16x128(wv[j], xv, v4f{0.f, 0.f, 0.f, 0.f});
                const float sc = g < G ? xs * s.ws[j] : 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r) run[i][j][r] = g < G ? fmaf(t[r], sc, run[i][j][r]) : run[i][j][r];
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
    // one unit: four adjacent columns of a row
    for (int u = tid; u < FT * kCols * 64; u += 64 * KS) {
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
        // the lane that holds row 16 i + ln % 16 in every wave knows its slot
        int xrow;
        const int row = row0 + 16 * i + (ln & 15);
        const int sl_id = block_slot(p, row, end, xrow);
        if (sl_id < 0) continue;
        const int col = (sl * kCols + j) * 16 + 4 * (ln >> 4);
        if (col >= cols) continue;
        const int64_t orow = DST == Dst::kSlotF32 ? sl_id : row;
        if constexpr (DST == Dst::kSlotF32 || kSilu) {
            float* o = reinterpret_cast<float*>(p.out) + orow * p.ldo + col;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (col + r < cols) o[r] = t[r];
        } else {
            uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + orow * p.ldo + col;
            constexpr bool bf16 = DST == Dst::kBf16;
            const uint32_t a = pack_out16(t[0], t[1], bf16), b = pack_out16(t[2], t[3], bf16);
            if (col + 3 < cols && p.ldo % 4 == 0) {
                *reinterpret_cast<uint2*>(o) = make_uint2(a, b);
            } else {
                const uint32_t v[4] = {a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16};
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (col + r < cols) o[r] = (uint16_t)v[r];
            }
        }
    }
}

template <int FT, int FN, int KS, Src SRC, Dst DST>
int go(const BlockParams& p, hipStream_t s) {
    constexpr bool silu = DST == Dst::kSiluF32;
    const int cols = silu ? p.N / 2 : p.N, per = 16 * (silu ? FN / 2 : FN);
    const int slices = (cols + per - 1) / per;
    const int64_t grid = (int64_t)((p.P + 16 * FT - 1) / (16 * FT)) * slices;
    if (grid >= (int64_t)1 << 31) {
        set_error("fp8 block product: too many tiles");
        return W4A8_ERR_INVALID;
    }
    if (p.K % kBlk != 0) launch_kernel(&block_stream_kernel<FT, FN, KS, SRC, DST, true>, dim3((unsigned)grid), dim3(64 * KS), 0, s, p, slices);
    else launch_kernel(&block_stream_kernel<FT, FN, KS, SRC, DST, false>, dim3((unsigned)grid), dim3(64 * KS), 0, s, p, slices);
    return check_launch("block_stream_kernel");
}

}  // namespace

int launch_block_stream(const BlockArgs& a, hipStream_t s) {
    const BlockParams p = block_params(a);
    if (p.P == 0) return W4A8_OK;
    auto dst = [&](auto src) -> int {
        constexpr Src S = decltype(src)::value;
        switch (a.dst) {
            case Dst::kF16: return go<1, 2, 4, S, Dst::kF16>(p, s);
            case Dst::kBf16: return go<1, 2, 4, S, Dst::kBf16>(p, s);
            case Dst::kSiluF32: return go<1, 2, 4, S, Dst::kSiluF32>(p, s);
            case Dst::kSlotF32: return go<1, 2, 4, S, Dst::kSlotF32>(p, s);
            default: break;
        }
        set_error("fp8 block product: output form not taken by the streaming kernel");
        return W4A8_ERR_INVALID;
    };
    switch (a.src) {
        case Src::kFp8: return dst(std::integral_constant<Src, Src::kFp8>{});
        case Src::kF16: return dst(std::integral_constant<Src, Src::kF16>{});
        case Src::kBf16: return dst(std::integral_constant<Src, Src::kBf16>{});
        default: return dst(std::integral_constant<Src, Src::kF32>{});
    }
}

}  // namespace w4a8
