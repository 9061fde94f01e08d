// Block-scaled fp8 operators: matrix-core operands and stores shared by the product kernels.
#pragma once

#include "fp8_block.h"

namespace w4a8 {

using v8bf = __bf16 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v8bf e4m3_to_bf16x8(uint32_t lo, uint32_t hi) {
    using v2bf = __bf16 __attribute__((ext_vector_type(2)));
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, false);
    const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, true);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, false);
    const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, true);
    return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A lane's 32 e4m3 values of one row and group of 128 k (16-byte pieces q and q + 4) as an operand:
// as they are, or (EXACT) as bf16.
//
// The fp8 matrix core cuts products of eight neighbouring k to 2^-13 of their largest; EXACT feeds
// the bf16 one (every e4m3 number is a bf16 number), which adds them as fp32 numbers, at a quarter
// of the rate and for sixteen conversions an operand. It is for sums that are quantised again: an
// error of 1e-4 there moves values across a border between two e4m3 numbers, and the layer's output
// by 1e-3 (one token by up to 6e-3), up to three times what the rounding to bf16 does.
template <bool EXACT>
struct GroupOp {
    v8i b;
};
template <>
struct GroupOp<true> {
    v8bf h[4];
};
template <bool EXACT>
__device__ __forceinline__ GroupOp<EXACT> group_op(const u32x4& lo, const u32x4& hi) {
    GroupOp<EXACT> o;
    if constexpr (EXACT) {
        o.h[0] = e4m3_to_bf16x8(lo[0], lo[1]);
        o.h[1] = e4m3_to_bf16x8(lo[2], lo[3]);
        o.h[2] = e4m3_to_bf16x8(hi[0], hi[1]);
        o.h[3] = e4m3_to_bf16x8(hi[2], hi[3]);
    } else {
        o.b = v8i{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    }
    return o;
}
// Sum over one group: lane (q, c) gets rows 4 q .. 4 q + 3 of the first operand by row c of the second.
template <bool EXACT>
__device__ __forceinline__ v4f group_mfma(const GroupOp<EXACT>& w, const GroupOp<EXACT>& x) {
    const v4f zero{0.f, 0.f, 0.f, 0.f};
    if constexpr (EXACT) {
        v4f t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.h[0], x.h[0], zero, 0, 0, 0);
        t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.h[1], x.h[1], t, 0, 0, 0);
        t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.h[2], x.h[2], t, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.h[3], x.h[3], t, 0, 0, 0);
    } else {
        return mfma_16x16x128(w.b, x.b, zero);
    }
}

// Four adjacent columns of one row, rounded to 16 bits.
__device__ __forceinline__ void store16(const BlockParams& p, int64_t orow, int col, int cols, const v4f& t, bool bf16) {
    uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + orow * p.ldo + col;
    const uint32_t a = pack_out16(t[0], t[1], bf16), b = pack_out16(t[2], t[3], bf16);
    if (p.ldo % 4 == 0 && p.out8) {
        *reinterpret_cast<uint2*>(o) = make_uint2(a, b);
    } else {
        const uint32_t v[4] = {a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16};
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (col + r < cols) o[r] = (uint16_t)v[r];
    }
}
// Eight adjacent columns of one row (an aligned out, ldo a multiple of 8): with four a lane, stores touch
// 32 bytes of a row and the layer's second product of 4096 tokens takes 162 instead of 149 us.
__device__ __forceinline__ void store16x8(const BlockParams& p, int64_t orow, int col, const v4f& a, const v4f& b, bool bf16) {
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + orow * p.ldo + col) =
        make_uint4(pack_out16(a[0], a[1], bf16), pack_out16(a[2], a[3], bf16), pack_out16(b[0], b[1], bf16),
                   pack_out16(b[2], b[3], bf16));
}
template <Dst DST>
__device__ __forceinline__ void store4(const BlockParams& p, int64_t orow, int col, int cols, const v4f& t) {
    if constexpr (DST == Dst::kSlotF32 || DST == Dst::kSiluF32) {
        // (whole layers: multiples of 128 columns)
        *reinterpret_cast<v4f*>(reinterpret_cast<float*>(p.out) + orow * p.ldo + col) = t;
    } else {
        store16(p, orow, col, cols, t, p.out_bf16 != 0);
    }
}

}  // namespace w4a8
