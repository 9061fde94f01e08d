// int8 products of few rows (gfx950): the weights are streamed once, dense or grouped.
//
// Bound: HBM, every weight once per 16 rows. Weights go from memory to the MFMA operands' registers with no
// detour: of each step of 128 values, lane (q, c) = (lane / 16, lane % 16) holds the 16-byte pieces q and q + 4 of
// row c, for rows and weights alike (a sum of whole numbers may take its k in any order). Weights are the first
// operand: a lane ends up with four adjacent columns of one row.
#include <algorithm>

#include "int8.h"

namespace w4a8 {
namespace {

// The expert and the end of the rows in use of the 16 rows from row0; false: nothing to do.
__device__ __forceinline__ bool block_of(const Int8Params& p, int row0, int c, int& e, int& end) {
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

// KS waves take the steps of K in turn (what they read at one time is contiguous along K), FN column fragments of 16.
constexpr int kRing = 3;          // steps of a wave in flight
template <int FN, int KS, Out8 DST>
__global__ void __launch_bounds__(64 * KS) int8_stream_kernel(Int8Params p, int slices) {
    constexpr bool kSilu = DST == Out8::kSiluF32;
    constexpr int kCols = kSilu ? FN / 2 : FN;                 // column fragments of the output
    __shared__ __attribute__((aligned(16))) v4i part[KS][FN][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, c = lane & 15;
    const int tb = blockIdx.x / slices, sl = blockIdx.x % slices;
    const int row0 = tb * 16;
    int e, end;
    if (!block_of(p, row0, c, e, end)) return;
    const int half = p.N / 2;
    const int cols = kSilu ? half : p.N;
    const int K = p.K;

    const int8_t* wp[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int f = (sl * kCols + j % kCols) * 16, up = kSilu && j >= kCols ? half : 0;
        // (columns past the end read the last one; never stored)
        wp[j] = p.w + ((int64_t)e * p.N + up + min(f + c, cols - 1)) * K;
    }
    int xrow;
    const int slot = int8_slot(p, row0 + c, end, xrow);
    const int8_t* xp = p.x + (int64_t)xrow * p.ldx;
    struct Stage {
        u32x4 w[FN][2], x[2];
    };
    const int G = (K + kStep - 1) / kStep;
    auto load = [&](Stage& s, int step) __attribute__((always_inline)) {
        const int g = step * KS + wave;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // (pieces past the end: the last one, and zeros for the rows')
            const int k = g * kStep + h * 64 + q * 16, at = min(k, K - 16);
#pragma unroll
            for (int j = 0; j < FN; ++j) s.w[j][h] = *reinterpret_cast<const u32x4*>(wp[j] + at);
            s.x[h] = *reinterpret_cast<const u32x4*>(xp + at);
            if (k >= K) s.x[h] = u32x4{0, 0, 0, 0};
        }
    };
    v4i run[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) run[j] = v4i{0, 0, 0, 0};
    auto consume = [&](const Stage& s) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < FN; ++j) run[j] = mfma_i8(s.w[j][h], s.x[h], run[j]);
    };
    const int steps = (G + KS - 1) / KS;
    Stage ring[kRing];
#pragma unroll
    for (int d = 0; d < kRing; ++d) load(ring[d], d);
    for (int s0 = 0; s0 < steps; s0 += kRing) {
#pragma unroll
        for (int d = 0; d < kRing; ++d) {
            consume(ring[d]);
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
        v4i t = part[0][f][lane];
#pragma unroll
        for (int w = 1; w < KS; ++w) t += part[w][f][lane];
        return t;
    };
    const int col = (sl * kCols + wave) * 16 + 4 * q;
    const v4i a = total(wave);
    if (slot < 0 || col >= cols) return;
    const float xs = p.xs[xrow];
    const float* ws = p.ws + (int64_t)e * p.N;
    v4f t;
    if constexpr (kSilu) {
        const v4i b = total(kCols + wave);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = min(col + r, cols - 1);
            t[r] = silu_mul((float)a[r] * (xs * ws[n]), (float)b[r] * (xs * ws[half + n]));
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = min(col + r, cols - 1);
            t[r] = (float)a[r] * (xs * ws[n]);
            if (DST == Out8::k16) t[r] += bias_at(p, n);
        }
    }
    if constexpr (DST == Out8::k16)
        store16(p, row0 + c, col, t);
    else                                                       // (whole layers: multiples of 64 columns)
        *reinterpret_cast<v4f*>(reinterpret_cast<float*>(p.out) + (int64_t)(DST == Out8::kSlotF32 ? slot : row0 + c) * p.ldo + col) = t;
}

template <int FN, int KS, Out8 DST>
int stream_go(const Int8Params& p, hipStream_t s) {
    constexpr bool silu = DST == Out8::kSiluF32;
    const int cols = silu ? p.N / 2 : p.N, per = 16 * (silu ? FN / 2 : FN);
    const int slices = (cols + per - 1) / per;
    const int64_t grid = (int64_t)((p.P + 15) / 16) * slices;
    if (!grid_fits(grid, 64 * KS)) {
        set_error("int8 product: too many tiles");
        return W4A8_ERR_INVALID;
    }
    launch_kernel(&int8_stream_kernel<FN, KS, DST>, dim3((unsigned)grid), dim3(64 * KS), 0, s, p, slices);
    return check_launch("int8_stream_kernel");
}

}  // namespace

int launch_int8_stream(const Int8Args& a, hipStream_t s) {
    const Int8Params p = int8_params(a);
    if (p.P == 0) return W4A8_OK;
    if (a.dst == Out8::kSiluF32) return stream_go<2, 8, Out8::kSiluF32>(p, s);
    if (a.dst == Out8::kSlotF32) return stream_go<2, 4, Out8::kSlotF32>(p, s);
    return stream_go<1, 8, Out8::k16>(p, s);
}

}  // namespace w4a8
