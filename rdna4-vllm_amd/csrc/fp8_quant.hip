// RMS norm with the residual's addition and e4m3 output, and e4m3 rows with a scale per 128 values
// (of 16-bit rows or of silu(gate) * up).
//
// Bound: HBM. A row is read once: W waves hold it in registers (eight values a lane and piece)
// between the sum of squares, the absmaxes and the rounding. A group of 128 values is one piece of
// sixteen neighbouring lanes, so its absmax is four DPP steps. Measured: norm of 8192 x 4096 bf16 with
// residual and 16-bit norm 55.7 us, 5.4 TB/s; silu(gate) * up of 4111 x 12288 fp16 44.6 us, 5.7 TB/s.
#include <algorithm>

#include "fp8_mfma.h"

namespace w4a8 {
namespace {

// Eight 16-bit values of a register vector.
template <bool BF16>
__device__ __forceinline__ void unpack8(const u32x4& v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = v[i];
        if constexpr (BF16) {
            f[2 * i] = __uint_as_float(w << 16);
            f[2 * i + 1] = __uint_as_float(w & 0xFFFF0000u);
        } else {
            f[2 * i] = __half2float(__ushort_as_half((uint16_t)(w & 0xFFFF)));
            f[2 * i + 1] = __half2float(__ushort_as_half((uint16_t)(w >> 16)));
        }
    }
}
template <bool BF16>
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack_out16(f[2 * i], f[2 * i + 1], BF16);
    return v;
}
template <bool BF16>
__device__ __forceinline__ float load16(const void* x, int64_t i) {
    if constexpr (BF16) return __bfloat162float(reinterpret_cast<const __hip_bfloat16*>(x)[i]);
    else return __half2float(reinterpret_cast<const __half*>(x)[i]);
}
template <bool BF16>
__device__ __forceinline__ float round16(float v) {
    if constexpr (BF16) return __bfloat162float(__float2bfloat16(v));
    else return __half2float(__float2half(as_f32(v)));
}
__device__ __forceinline__ float absmax8(const float (&f)[8]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(f[j]));
    return m;
}
__device__ __forceinline__ uint2 quant8(const float (&f)[8], float inv) {
    return make_uint2(pack4_e4m3(as_f32(f[0] * inv), as_f32(f[1] * inv), as_f32(f[2] * inv), as_f32(f[3] * inv)),
                      pack4_e4m3(as_f32(f[4] * inv), as_f32(f[5] * inv), as_f32(f[6] * inv), as_f32(f[7] * inv)));
}

// Combines a value over the W waves of a row (rows of a work-group each have their own slots).
template <int W, typename Op>
__device__ __forceinline__ float row_allreduce(float v, Op op, float* slots, int wave) {
    v = lane_allreduce<6>(v, op);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) slots[wave] = v;
        __syncthreads();
        v = slots[0];
#pragma unroll
        for (int i = 1; i < W; ++i) v = op(v, slots[i]);
    }
    return v;
}

struct NormParams {
    const void* x;
    const void* r;
    const void* w;
    void* z;
    void* y;
    uint8_t* q;
    float* s;
    int64_t ldx, ldr;
    int64_t rows;
    int H, G;
    float eps;
};

// One row by W waves, NV pieces of eight values a lane. The sum z = x + r is rounded to the rows'
// type before the norm: the norm is that of the residual stream that is stored, as a model that
// adds and normalises in two steps computes it. The norm itself stays fp32 up to the e4m3 rounding.
template <int W, int NV, bool BF16, bool RES, bool KEEP, bool WF32, bool PER_ROW>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) rms_norm_quant_kernel(NormParams p) {
    constexpr int kRows = W == 1 ? 4 : 1;      // rows of a work-group
    __shared__ float red[2][W];
    const int wave = W == 1 ? 0 : threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * kRows + (W == 1 ? threadIdx.x >> 6 : 0);
    if (row >= p.rows) return;                 // (W > 1: the whole work-group)
    const int t = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const uint16_t* xr = reinterpret_cast<const uint16_t*>(p.x) + row * p.ldx;
    u32x4 v[NV], rv[RES ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * 64 * W + t) * 8;
        v[i] = u32x4{0, 0, 0, 0};
        if (k < p.H) v[i] = *reinterpret_cast<const u32x4*>(xr + k);
    }
    if constexpr (RES) {
        const uint16_t* rr = reinterpret_cast<const uint16_t*>(p.r) + row * p.ldr;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (i * 64 * W + t) * 8;
            rv[i] = u32x4{0, 0, 0, 0};
            if (k < p.H) rv[i] = *reinterpret_cast<const u32x4*>(rr + k);
        }
    }
    float f[NV][8];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        unpack8<BF16>(v[i], f[i]);
        if constexpr (RES) {
            float b[8];
            unpack8<BF16>(rv[i], b);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[i][j] += b[j];
            const u32x4 zv = pack8<BF16>(f[i]);
            const int k = (i * 64 * W + t) * 8;
            if (k < p.H) *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(p.z) + row * p.H + k) = zv;
            unpack8<BF16>(zv, f[i]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(f[i][j], f[i][j], sum);
    }
    sum = row_allreduce<W>(sum, SumOp{}, red[0], wave);
    const float rstd = 1.0f / sqrtf(sum / (float)p.H + p.eps);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * 64 * W + t) * 8;
        float wv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (k < p.H) {
            if constexpr (WF32) {
                const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.w) + k);
                const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.w) + k + 4);
                wv[0] = a.x; wv[1] = a.y; wv[2] = a.z; wv[3] = a.w;
                wv[4] = b.x; wv[5] = b.y; wv[6] = b.z; wv[7] = b.w;
            } else {
                unpack8<BF16>(*reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.w) + k), wv);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] = f[i][j] * rstd * wv[j];
        if constexpr (KEEP) {
            if (k < p.H)
                *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(p.y) + row * p.H + k) = pack8<BF16>(f[i]);
        }
        float m = absmax8(f[i]);
        if constexpr (PER_ROW) {
            amax = fmaxf(amax, m);
        } else {
            m = lane_allreduce<4>(m, MaxOp{});
            const float s = act_scale_from_absmax(m);
            if (k < p.H) {
                *reinterpret_cast<uint2*>(p.q + row * p.H + k) = quant8(f[i], 1.0f / s);
                if ((t & 15) == 0) p.s[row * p.G + k / kBlk] = s;
            }
        }
    }
    if constexpr (PER_ROW) {
        amax = row_allreduce<W>(amax, MaxOp{}, red[1], wave);
        const float s = act_scale_from_absmax(amax);
        if (t == 0) p.s[row] = s;
        const float inv = 1.0f / s;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (i * 64 * W + t) * 8;
            if (k < p.H) *reinterpret_cast<uint2*>(p.q + row * p.H + k) = quant8(f[i], inv);
        }
    }
}

// Any sizes, strides and alignments: a work-group a row, value by value, z read again where it is
// needed (three reads of the row).
template <bool BF16>
__global__ void __launch_bounds__(256) rms_norm_quant_any_kernel(NormParams p, bool w_f32, bool per_row) {
    __shared__ float red[2][4];
    const int64_t row = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint16_t* z = reinterpret_cast<uint16_t*>(p.z);
    // (z from where it was stored, behind the sum's barrier: it may stand in place of x or r)
    auto value = [&](int k) { return p.r != nullptr ? load16<BF16>(z, row * p.H + k) : load16<BF16>(p.x, row * p.ldx + k); };
    auto put16 = [&](uint16_t* to, float v) { *to = (uint16_t)(pack_out16(v, 0.f, BF16) & 0xFFFF); };
    float sum = 0.f;
    for (int k = threadIdx.x; k < p.H; k += 256) {
        float v = load16<BF16>(p.x, row * p.ldx + k);
        if (p.r != nullptr) {
            v = round16<BF16>(v + load16<BF16>(p.r, row * p.ldr + k));
            put16(z + row * p.H + k, v);
        }
        sum = fmaf(v, v, sum);
    }
    sum = row_allreduce<4>(sum, SumOp{}, red[0], wave);
    const float rstd = 1.0f / sqrtf(sum / (float)p.H + p.eps);
    auto normed = [&](int k) {
        const float w = w_f32 ? reinterpret_cast<const float*>(p.w)[k] : load16<BF16>(p.w, k);
        return value(k) * rstd * w;
    };
    float amax = 0.f;
    if (per_row) {
        for (int k = threadIdx.x; k < p.H; k += 256) amax = fmaxf(amax, fabsf(normed(k)));
        amax = row_allreduce<4>(amax, MaxOp{}, red[1], wave);
        if (threadIdx.x == 0) p.s[row] = act_scale_from_absmax(amax);
    }
    for (int g = wave; g < (p.H + kBlk - 1) / kBlk; g += 4) {      // a wave a group of 128
        const int k0 = g * kBlk + lane, k1 = k0 + 64;
        const float a = k0 < p.H ? normed(k0) : 0.f, b = k1 < p.H ? normed(k1) : 0.f;
        float s = act_scale_from_absmax(amax);
        if (!per_row) {
            s = act_scale_from_absmax(wave_max(fmaxf(fabsf(a), fabsf(b))));
            if (lane == 0) p.s[row * p.G + g] = s;
        }
        const float inv = 1.0f / s;
        if (k0 < p.H) p.q[row * p.H + k0] = (uint8_t)cvt_f32_e4m3(as_f32(a * inv));
        if (k1 < p.H) p.q[row * p.H + k1] = (uint8_t)cvt_f32_e4m3(as_f32(b * inv));
        if (p.y != nullptr) {
            if (k0 < p.H) put16(reinterpret_cast<uint16_t*>(p.y) + row * p.H + k0, a);
            if (k1 < p.H) put16(reinterpret_cast<uint16_t*>(p.y) + row * p.H + k1, b);
        }
    }
}

// e4m3 values as bf16 numbers, eight of them.
__device__ __forceinline__ u32x4 widen8(uint2 v) {
    union {
        v8bf h;
        u32x4 u;
    } o;
    o.h = e4m3_to_bf16x8(v.x, v.y);
    return o.u;
}

// Eight values a lane, sixteen lanes a group of 128, so G * 16 lanes a row.
// WIDE: the e4m3 values as bf16 numbers.
template <bool BF16, bool SILU, bool WIDE>
__global__ void __launch_bounds__(256) act_quant_groups_kernel(const void* __restrict__ x, int64_t rows, int K, int G,
                                                               int64_t ldx, uint8_t* __restrict__ q,
                                                               float* __restrict__ scales) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = i / (G * 16);
    if (row >= rows) return;                                    // whole groups of sixteen lanes
    const int k = (int)(i - row * (G * 16)) * 8;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k < K) {
        const uint16_t* xr = reinterpret_cast<const uint16_t*>(x) + row * ldx + k;
        const u32x4 a = *reinterpret_cast<const u32x4*>(xr);
        if constexpr (SILU) {
            const u32x4 b = *reinterpret_cast<const u32x4*>(xr + K);
            float g[8], u[8];
            unpack8<BF16>(a, g);
            unpack8<BF16>(b, u);
            silu_mul_f32<BF16>(g, u, f);
        } else {
            unpack8<BF16>(a, f);
        }
    }
    const float s = act_scale_from_absmax(lane_allreduce<4>(absmax8(f), MaxOp{}));
    if (k < K) {
        const uint2 v = quant8(f, 1.0f / s);
        if constexpr (WIDE) *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(q) + row * K + k) = widen8(v);
        else *reinterpret_cast<uint2*>(q + row * K + k) = v;
        if ((threadIdx.x & 15) == 0) scales[row * G + k / kBlk] = s;
    }
}

__global__ void __launch_bounds__(256) widen_rows_kernel(const uint2* __restrict__ x, int64_t n8, u32x4* __restrict__ q) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n8) q[i] = widen8(x[i]);
}

// Any sizes and alignments: a wave a group.
template <bool BF16, bool SILU>
__global__ void __launch_bounds__(256) act_quant_groups_any_kernel(const void* __restrict__ x, int64_t rows, int K,
                                                                   int G, int64_t ldx, uint8_t* __restrict__ q,
                                                                   float* __restrict__ scales) {
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t row = i / G;
    if (row >= rows) return;
    const int g = (int)(i - row * G), lane = threadIdx.x & 63;
    float v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = g * kBlk + h * 64 + lane;
        v[h] = 0.f;
        if (k < K) {
            v[h] = load16<BF16>(x, row * ldx + k);
            if constexpr (SILU) {
                const float g[1] = {v[h]}, u[1] = {load16<BF16>(x, row * ldx + K + k)};
                float o[1];
                silu_mul_f32<BF16>(g, u, o);
                v[h] = o[0];
            }
        }
    }
    const float s = act_scale_from_absmax(wave_max(fmaxf(fabsf(v[0]), fabsf(v[1]))));
    const float inv = 1.0f / s;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = g * kBlk + h * 64 + lane;
        if (k < K) q[row * K + k] = (uint8_t)cvt_f32_e4m3(as_f32(v[h] * inv));
    }
    if (lane == 0) scales[row * G + g] = s;
}

// Eight columns a lane; a token's rows are requested together, eight at a time (4096 tokens x 8 rows of 2048:
// 26 us, 5.8 TB/s). A value is scaled back (exactly) before its weight: their scale times the weight can
// leave fp32's range where the product of all three does not.
__global__ void __launch_bounds__(256) block_reduce_kernel(const void* __restrict__ y, const float* __restrict__ ys,
                                                           const int32_t* __restrict__ s2r,
                                                           const float* __restrict__ tw, int N, int top_k,
                                                           void* __restrict__ out) {
    const int64_t t = blockIdx.x;
    const int n = (blockIdx.y * 256 + threadIdx.x) * 8;
    if (n >= N) return;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < top_k; j0 += 8) {
        int32_t r[8];
        u32x4 v[8];
        float w[8], sc[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            r[j] = j0 + j < top_k ? s2r[t * top_k + j0 + j] : -1;
            w[j] = j0 + j < top_k ? tw[t * top_k + j0 + j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = u32x4{0, 0, 0, 0};
            sc[j] = 0.f;
            if (r[j] >= 0) {
                v[j] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(y) + (int64_t)r[j] * N + n);
                sc[j] = ys[(int64_t)r[j] * (N / 32) + n / 32];
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (r[j] < 0) continue;
            float f[8];
            unpack8<false>(v[j], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = fmaf(w[j], f[i] * sc[j], acc[i]);
        }
    }
    *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(out) + t * N + n) = pack8<true>(acc);
}

template <int W, int NV, bool BF16, bool RES, bool KEEP, bool WF32>
void norm_go(const NormParams& p, bool per_row, hipStream_t s) {
    const unsigned grid = (unsigned)(W == 1 ? (p.rows + 3) / 4 : p.rows);
    const unsigned threads = W == 1 ? 256 : 64 * W;
    if (per_row) rms_norm_quant_kernel<W, NV, BF16, RES, KEEP, WF32, true><<<grid, threads, 0, s>>>(p);
    else rms_norm_quant_kernel<W, NV, BF16, RES, KEEP, WF32, false><<<grid, threads, 0, s>>>(p);
}
template <int W, int NV, bool BF16>
void norm_types(const NormParams& p, bool w_f32, bool per_row, hipStream_t s) {
    const bool res = p.r != nullptr, keep = p.y != nullptr;
    auto go = [&](auto r, auto k) {
        if (w_f32) norm_go<W, NV, BF16, decltype(r)::value, decltype(k)::value, true>(p, per_row, s);
        else norm_go<W, NV, BF16, decltype(r)::value, decltype(k)::value, false>(p, per_row, s);
    };
    if (res && keep) go(std::true_type{}, std::true_type{});
    else if (res) go(std::true_type{}, std::false_type{});
    else if (keep) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
}
template <bool BF16>
void norm_sizes(const NormParams& p, bool w_f32, bool per_row, hipStream_t s) {
    if (p.H <= 512) norm_types<1, 1, BF16>(p, w_f32, per_row, s);
    else if (p.H <= 2048) norm_types<4, 1, BF16>(p, w_f32, per_row, s);
    else if (p.H <= 4096) norm_types<4, 2, BF16>(p, w_f32, per_row, s);
    else if (p.H <= 8192) norm_types<4, 4, BF16>(p, w_f32, per_row, s);
    else norm_types<16, 2, BF16>(p, w_f32, per_row, s);
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace

int launch_rms_norm_quant(const NormArgs& a, hipStream_t s) {
    if (a.rows == 0) return W4A8_OK;
    NormParams p{a.x, a.residual, a.weight, a.residual_out, a.norm_out, a.q, a.scales,
                 a.ldx, a.ldr, a.rows, (int)a.H, a.per_row ? 1 : (int)blk_groups(a.H), a.eps};
    const bool whole = a.H % 8 == 0 && a.H <= 16384 && a.ldx % 8 == 0 && (a.residual == nullptr || a.ldr % 8 == 0) &&
                       aligned(a.x, 16) && aligned(a.residual, 16) && aligned(a.weight, 16) &&
                       aligned(a.residual_out, 16) && aligned(a.norm_out, 16) && aligned(a.q, 8);
    if (!grid_fits(whole && a.H <= 512 ? (a.rows + 3) / 4 : a.rows, whole && a.H > 8192 ? 1024 : 256)) {
        set_error("rms_norm_quant: too many rows");
        return W4A8_ERR_INVALID;
    }
    if (whole) {
        if (a.bf16) norm_sizes<true>(p, a.weight_f32, a.per_row, s);
        else norm_sizes<false>(p, a.weight_f32, a.per_row, s);
        return check_launch("rms_norm_quant_kernel");
    }
    if (a.bf16) rms_norm_quant_any_kernel<true><<<(unsigned)a.rows, 256, 0, s>>>(p, a.weight_f32, a.per_row);
    else rms_norm_quant_any_kernel<false><<<(unsigned)a.rows, 256, 0, s>>>(p, a.weight_f32, a.per_row);
    return check_launch("rms_norm_quant_any_kernel");
}

int launch_block_reduce(const void* y, const float* ys, const int32_t* slot_to_row, const float* tw, int64_t T, int64_t N,
                        int64_t top_k, void* out, hipStream_t s) {
    if (T == 0) return W4A8_OK;
    if (!grid_fits(T, 256)) {
        set_error("block_reduce: too many rows");
        return W4A8_ERR_INVALID;
    }
    const dim3 grid((unsigned)T, (unsigned)((N / 8 + 255) / 256));
    block_reduce_kernel<<<grid, 256, 0, s>>>(y, ys, slot_to_row, tw, (int)N, (int)top_k, out);
    return check_launch("block_reduce_kernel");
}

int launch_act_quant_block(const void* x, bool bf16, int64_t rows, int64_t K, int64_t ldx, bool silu, uint8_t* q,
                           float* scales, hipStream_t s) {
    if (rows == 0) return W4A8_OK;
    const int64_t G = blk_groups(K);
    const bool whole = K % 8 == 0 && ldx % 8 == 0 && aligned(x, 16) && aligned(q, 8);
    const int64_t blocks = whole ? (rows * G * 16 + 255) / 256 : (rows * G + 3) / 4;
    if (!grid_fits(blocks, 256)) {
        set_error("act_quant_fp8_block: too many groups");
        return W4A8_ERR_INVALID;
    }
    auto go = [&](auto kernel) { kernel<<<(unsigned)blocks, 256, 0, s>>>(x, rows, (int)K, (int)G, ldx, q, scales); };
    if (whole) {
        if (bf16) silu ? go(act_quant_groups_kernel<true, true, false>) : go(act_quant_groups_kernel<true, false, false>);
        else silu ? go(act_quant_groups_kernel<false, true, false>) : go(act_quant_groups_kernel<false, false, false>);
        return check_launch("act_quant_groups_kernel");
    }
    if (bf16) silu ? go(act_quant_groups_any_kernel<true, true>) : go(act_quant_groups_any_kernel<true, false>);
    else silu ? go(act_quant_groups_any_kernel<false, true>) : go(act_quant_groups_any_kernel<false, false>);
    return check_launch("act_quant_groups_any_kernel");
}

int launch_act_quant_wide(const void* x, bool bf16, int64_t rows, int64_t K, uint16_t* q, float* scales, hipStream_t s) {
    if (rows == 0) return W4A8_OK;
    const int64_t G = blk_groups(K), blocks = (rows * G * 16 + 255) / 256;
    if (K % kBlk != 0 || !aligned(x, 16) || !aligned(q, 16) || !grid_fits(blocks, 256)) {
        set_error("act_quant_fp8_block: sizes not taken by the wide form");
        return W4A8_ERR_INVALID;
    }
    auto go = [&](auto kernel) {
        kernel<<<(unsigned)blocks, 256, 0, s>>>(x, rows, (int)K, (int)G, K, reinterpret_cast<uint8_t*>(q), scales);
    };
    bf16 ? go(act_quant_groups_kernel<true, false, true>) : go(act_quant_groups_kernel<false, false, true>);
    return check_launch("act_quant_groups_kernel");
}

int launch_widen_rows(const void* x, int64_t rows, int64_t K, uint16_t* q, hipStream_t s) {
    if (rows == 0) return W4A8_OK;
    const int64_t n8 = rows * (K / 8), blocks = (n8 + 255) / 256;
    if (K % 8 != 0 || !aligned(x, 8) || !aligned(q, 16) || !grid_fits(blocks, 256)) {
        set_error("widen_rows: sizes not taken");
        return W4A8_ERR_INVALID;
    }
    widen_rows_kernel<<<(unsigned)blocks, 256, 0, s>>>(static_cast<const uint2*>(x), n8, reinterpret_cast<u32x4*>(q));
    return check_launch("widen_rows_kernel");
}

}  // namespace w4a8
