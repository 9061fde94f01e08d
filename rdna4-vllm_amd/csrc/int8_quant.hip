// int8 rows with a scale each (of 16-bit rows, of silu(gate) * up, of the layer's fp32 rows), and the layer's sum
// over a token's slots.
//
// Bound: memory. A row is read once: W waves hold it in registers (eight values a lane and piece) between its
// largest magnitude and its rounding. 32768 rows of 512 fp32 values: 17 us, 4.9 TB/s; the sum of 4096 tokens' eight rows of
// 2048 48 us, 5.9 TB/s.
#include <algorithm>

#include "int8.h"

namespace w4a8 {
namespace {

struct QuantParams {
    const void* x;
    int8_t* q;
    float* s;
    const int32_t* sorted_ids;
    const int32_t* ntp;
    int64_t rows, ldx;
    int K, num_valid;
};

struct UMaxOp {
    __device__ float operator()(float a, float b) const {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    }
};
// The largest of a row's bits over its W waves.
template <int W>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* red) {
    v = __float_as_uint(lane_allreduce<6>(__uint_as_float(v), UMaxOp{}));
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < W; ++i) v = max(v, red[i]);
    }
    return v;
}

template <Rows SRC>
__device__ __forceinline__ float value(const void* x, int64_t i) {
    if constexpr (SRC == Rows::kF32) return reinterpret_cast<const float*>(x)[i];
    const uint16_t v = reinterpret_cast<const uint16_t*>(x)[i];
    if constexpr (SRC == Rows::kBf16) return __uint_as_float((uint32_t)v << 16);
    return __half2float(__ushort_as_half(v));
}

template <Rows SRC>
struct Raw8 {
    u32x4 v[SRC == Rows::kF32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* x, int64_t at) {
        if constexpr (SRC == Rows::kF32) {
            v[0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(x) + at);
            v[1] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(x) + at + 4);
        } else {
            v[0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(x) + at);
        }
    }
    __device__ __forceinline__ void unpack(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (SRC == Rows::kF32) {
                f[i] = __uint_as_float(v[i / 4][i % 4]);
            } else {
                const uint32_t w = v[0][i / 2];
                if constexpr (SRC == Rows::kBf16) f[i] = __uint_as_float((i & 1) ? w & 0xFFFF0000u : w << 16);
                else f[i] = __half2float(__ushort_as_half((uint16_t)((i & 1) ? w >> 16 : w & 0xFFFF)));
            }
        }
    }
};

// One row by W waves (W == 1: four rows a work-group), NV pieces of eight values a lane. K % 8 == 0, rows aligned to
// 16 bytes.
template <Rows SRC, bool SILU, int W, int NV>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) quant_rows_kernel(QuantParams p) {
    __shared__ uint32_t red[W];
    const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
    if (row >= p.rows) return;                 // (W > 1: the whole work-group, here and below)
    if (p.sorted_ids != nullptr) {
        if (row >= p.ntp[0]) return;
        const int s = p.sorted_ids[row];
        if (s < 0 || s >= p.num_valid) return;
    }
    const int t = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t base = row * p.ldx;
    Raw8<SRC> raw[NV], up[SILU ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * 64 * W + t) * 8;
        if (k < p.K) {
            raw[i].load(p.x, base + k);
            if constexpr (SILU) up[i].load(p.x, base + p.K + k);
        }
    }
    float f[NV][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if ((i * 64 * W + t) * 8 < p.K) {
            raw[i].unpack(f[i]);
            if constexpr (SILU) {
                float u[8];
                up[i].unpack(u);
#pragma unroll
                for (int j = 0; j < 8; ++j) f[i][j] = silu_mul(f[i][j], u[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, abs_bits(f[i][j]));
        }
    }
    const RowScale r = row_scale(row_max<W>(top, red));
    if (t == 0) p.s[row] = r.s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * 64 * W + t) * 8;
        if (k < p.K)
            *reinterpret_cast<uint2*>(p.q + row * p.K + k) =
                make_uint2(quant4(f[i][0], f[i][1], f[i][2], f[i][3], r), quant4(f[i][4], f[i][5], f[i][6], f[i][7], r));
    }
}

// Any sizes, strides and alignments: a work-group a row, value by value, the row read twice.
template <Rows SRC, bool SILU>
__global__ void __launch_bounds__(256) quant_any_kernel(QuantParams p) {
    __shared__ uint32_t red[4];
    const int64_t row = blockIdx.x;
    if (p.sorted_ids != nullptr) {
        if (row >= p.ntp[0]) return;
        const int s = p.sorted_ids[row];
        if (s < 0 || s >= p.num_valid) return;
    }
    const int64_t base = row * p.ldx;
    auto at = [&](int k) {
        const float v = value<SRC>(p.x, base + k);
        if constexpr (SILU) return silu_mul(v, value<SRC>(p.x, base + p.K + k));
        else return v;
    };
    uint32_t top = 0;
    for (int k = threadIdx.x; k < p.K; k += 256) top = max(top, abs_bits(at(k)));
    const RowScale r = row_scale(row_max<4>(top, red));
    if (threadIdx.x == 0) p.s[row] = r.s;
    for (int k = threadIdx.x; k < p.K; k += 256) p.q[row * p.K + k] = (int8_t)(quant_bits(at(k), r) & 0xFF);
}

template <Rows SRC, bool SILU>
int quant_go(const QuantParams& p, bool wide, hipStream_t s) {
    auto go = [&](auto kernel, int rows_each, int threads) -> int {
        const int64_t blocks = (p.rows + rows_each - 1) / rows_each;
        if (!grid_fits(blocks, threads)) {
            set_error("act_quant_int8: too many rows");
            return W4A8_ERR_INVALID;
        }
        launch_kernel(kernel, dim3((unsigned)blocks), dim3(threads), 0, s, p);
        return check_launch("act_quant_int8");
    };
    if (!wide || p.K > 32768) return go(&quant_any_kernel<SRC, SILU>, 1, 256);
    if (p.K <= 512) return go(&quant_rows_kernel<SRC, SILU, 1, 1>, 4, 256);
    if (p.K <= 1024) return go(&quant_rows_kernel<SRC, SILU, 1, 2>, 4, 256);
    if (p.K <= 2048) return go(&quant_rows_kernel<SRC, SILU, 4, 1>, 1, 256);
    if (p.K <= 4096) return go(&quant_rows_kernel<SRC, SILU, 4, 2>, 1, 256);
    if (p.K <= 8192) return go(&quant_rows_kernel<SRC, SILU, 8, 2>, 1, 512);
    if (p.K <= 16384) return go(&quant_rows_kernel<SRC, SILU, 16, 2>, 1, 1024);
    return go(&quant_rows_kernel<SRC, SILU, 16, 4>, 1, 1024);
}

// Eight columns a lane; a token's slots in order, their rows requested four at a time.
template <bool BF16>
__global__ void __launch_bounds__(256) int8_reduce_kernel(const float* __restrict__ y, const float* __restrict__ tw,
                                                         const int32_t* __restrict__ ids, const int32_t* __restrict__ emap,
                                                         int emap_len, int E, int N, int top_k, int64_t pieces,
                                                         uint16_t* __restrict__ out) {
    const int64_t piece = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (piece >= pieces) return;
    const int per = N / 8;
    const int64_t t = piece / per;
    const int n = (int)(piece - t * per) * 8;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    constexpr int kAt = 4;                     // slots read together
    for (int j0 = 0; j0 < top_k; j0 += kAt) {
        v4f v[kAt][2];
        float w[kAt];
        int e[kAt];
#pragma unroll
        for (int i = 0; i < kAt; ++i) {
            const int64_t slot = t * top_k + min(j0 + i, top_k - 1);
            e[i] = ids[slot];
            w[i] = tw[slot];
            v[i][0] = *reinterpret_cast<const v4f*>(y + slot * N + n);
            v[i][1] = *reinterpret_cast<const v4f*>(y + slot * N + n + 4);
        }
#pragma unroll
        for (int i = 0; i < kAt; ++i) {
            if (emap != nullptr) e[i] = e[i] >= 0 && e[i] < emap_len ? emap[e[i]] : -1;
            if (j0 + i >= top_k || e[i] < 0 || e[i] >= E) continue;
#pragma unroll
            for (int r = 0; r < 8; ++r) sum[r] = fmaf(w[i], v[i][r / 4][r % 4], sum[r]);
        }
    }
    *reinterpret_cast<uint4*>(out + t * N + n) = make_uint4(pack16<BF16>(sum[0], sum[1]), pack16<BF16>(sum[2], sum[3]),
                                                            pack16<BF16>(sum[4], sum[5]), pack16<BF16>(sum[6], sum[7]));
}

}  // namespace

int launch_act_quant_int8(const void* x, Rows src, int64_t rows, int64_t K, int64_t ldx, bool silu, int8_t* q, float* scales,
                          const int32_t* sorted_ids, const int32_t* ntp, int64_t num_valid, hipStream_t s) {
    if (rows == 0) return W4A8_OK;
    const QuantParams p{x, q, scales, sorted_ids, ntp, rows, ldx, (int)K, (int)num_valid};
    const int size = src == Rows::kF32 ? 4 : 2;
    const bool wide = K % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ldx * size % 16 == 0 || rows == 1) &&
                      reinterpret_cast<uintptr_t>(q) % 8 == 0;
    if (src == Rows::kF32) return quant_go<Rows::kF32, false>(p, wide, s);
    if (src == Rows::kBf16) return silu ? quant_go<Rows::kBf16, true>(p, wide, s) : quant_go<Rows::kBf16, false>(p, wide, s);
    return silu ? quant_go<Rows::kF16, true>(p, wide, s) : quant_go<Rows::kF16, false>(p, wide, s);
}

int launch_int8_reduce(const float* y, const float* tw, const int32_t* ids, const int32_t* emap, int64_t emap_len, int64_t E,
                       int64_t T, int64_t N, int64_t top_k, void* out, bool bf16, hipStream_t s) {
    if (T == 0) return W4A8_OK;
    const int64_t pieces = T * (N / 8), blocks = (pieces + 255) / 256;
    if (!grid_fits(blocks, 256)) {
        set_error("moe_int8_apply: too many tokens");
        return W4A8_ERR_INVALID;
    }
    auto go = [&](auto kernel) {
        launch_kernel(kernel, dim3((unsigned)blocks), dim3(256), 0, s, y, tw, ids, emap, (int)emap_len, (int)E, (int)N, (int)top_k,
                      pieces, static_cast<uint16_t*>(out));
        return check_launch("int8_reduce_kernel");
    };
    return bf16 ? go(&int8_reduce_kernel<true>) : go(&int8_reduce_kernel<false>);
}

}  // namespace w4a8
