// int8 (W8A8) operators: parameters and device helpers shared by their kernels.
//
// Numerics: rows are int8 with one fp32 scale each, weights (N, K) int8 with one fp32 scale per row
// (output channel):
//   out[m, n] = xs[m] ws[n] sum_k x[m, k] w[n, k] + bias[n].
// The sum is whole numbers on the integer matrix cores (exact in 32 bits for K up to 131071, whatever the
// order), the scales and the bias are fp32, and the result is rounded once.
// Quantisation: a = max(absmax, 127 * 2^-100), q = the whole number nearest to 127 v / a (ties to even) as an
// fp32 quotient, xs = a / 127. 127 v is exact for 16-bit v, so that the quotient lies on a border between two
// numbers only where the true one does. A row that holds an infinity or a NaN gets the scale NaN (and zeros):
// what is made of it is NaN.
#pragma once

#include "fp8_block.h"

namespace w4a8 {

using v16i = int __attribute__((ext_vector_type(16)));

constexpr int kStep = 128;                    // values of K that a step takes: one cache line of a row
constexpr int64_t kMaxInt8K = 131071;         // 2^31 / 2^14, less one

// What a product writes.
enum class Out8 : int {
    k16 = 0,        // out[row, n] rounded to fp16 or bf16
    kSiluF32 = 1,   // out[row, n] = silu(gate) * up in fp32, N = [gate | up] halves
    kSlotF32 = 2,   // out[slot, n] in fp32
};

// What the streaming kernels read their rows from.
enum class Src8 : int {
    kI8 = 0,        // int8 rows with their scales
    kF16 = 1,       // fp16, bf16 or fp32 rows, which the kernel quantises into LDS
    kBf16 = 2,
    kF32 = 3,
};
constexpr int kScanSlots = 4096;              // routed slots that a streaming kernel looks through

// Tiles (int8_tiles.hip).
struct Int8Args {
    const int8_t* x;             // (x_rows, K)
    const float* xs;             // (x_rows,)
    int64_t x_rows, K, ldx;
    const int8_t* w;             // (E, N, K)
    const float* ws;             // (E, N)
    const void* bias;            // (N,) or null
    bool bias_f32;               // else the output's type
    int64_t E, N;
    const int32_t* sorted_ids;   // null: one expert, rows in order (dense)
    const int32_t* expert_ids;
    const int32_t* ntp;
    int64_t P;                   // padded rows (dense: rows)
    int64_t top_k, num_valid, block_m;
    bool gather;                 // row r reads x[slot / top_k], else x[r]
    Out8 dst;
    bool bf16;                   // k16: bf16, else fp16
    void* out;
    int64_t ldo;
};

// Streaming kernels (int8_rows.hip).
struct RowsArgs {
    const void* x;               // rows, see Src8
    Src8 src;
    const float* xs;             // int8 rows: their scales
    int64_t rows, K, ldx;        // rows: of x
    const int8_t* w;
    const float* ws;
    const void* bias;
    bool bias_f32;
    int64_t E, N;
    const int32_t* ids;          // (slots,) routed experts; null: one expert, all rows (dense)
    const int32_t* emap;         // global -> local expert, or null
    int64_t emap_len, slots, top_k;
    bool gather;                 // slot s reads x[s / top_k], else x[s]
    Out8 dst;                    // out rows are slots (dense: rows)
    bool bf16;
    void* out;
    int64_t ldo;
};

// What both have on the device.
struct OutParams {
    const int8_t* w;
    const float* ws;
    const void* bias;
    void* out;
    int64_t ldx, ldo;
    int K, N, E, top_k, gather;
    int bf16, bias_f32;
    int out8, out16;             // rows of out are aligned to 8, to 16 bytes
};
struct Int8Params : OutParams {
    const int8_t* x;
    const float* xs;
    const int32_t* sorted_ids;
    const int32_t* expert_ids;
    const int32_t* ntp;
    int P, x_rows, num_valid, block_m;
};
struct RowsParams : OutParams {
    const void* x;
    const float* xs;
    const int32_t* ids;
    const int32_t* emap;
    int rows, slots, emap_len, one_slot;     // one_slot: each slot is a group of its own
};

template <typename A>
inline void out_params(const A& a, OutParams& p) {
    p.w = a.w; p.ws = a.ws; p.bias = a.bias; p.out = a.out; p.ldx = a.ldx; p.ldo = a.ldo;
    p.K = (int)a.K; p.N = (int)a.N; p.E = (int)a.E; p.top_k = (int)a.top_k; p.gather = a.gather ? 1 : 0;
    p.bf16 = a.bf16 ? 1 : 0; p.bias_f32 = a.bias_f32 ? 1 : 0;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.out);
    p.out8 = at % 8 == 0 && a.ldo % 4 == 0 ? 1 : 0;
    p.out16 = at % 16 == 0 && a.ldo % 8 == 0 ? 1 : 0;
}
inline Int8Params int8_params(const Int8Args& a) {
    Int8Params p;
    out_params(a, p);
    p.x = a.x; p.xs = a.xs; p.sorted_ids = a.sorted_ids; p.expert_ids = a.expert_ids; p.ntp = a.ntp;
    p.P = (int)a.P; p.x_rows = (int)a.x_rows; p.num_valid = (int)a.num_valid; p.block_m = (int)a.block_m;
    return p;
}
inline RowsParams rows_params(const RowsArgs& a) {
    RowsParams p;
    out_params(a, p);
    p.x = a.x; p.xs = a.xs; p.ids = a.ids; p.emap = a.emap;
    p.rows = (int)a.rows; p.slots = (int)a.slots; p.emap_len = (int)a.emap_len; p.one_slot = 0;
    return p;
}

// ---- quantisation ----
// A row's largest magnitude as its bits: an unsigned maximum, so that a NaN is the largest of all.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
struct RowScale {
    float s;          // absmax / 127
    float d, inv;     // absmax / 128 and its inverse: 127 v / absmax = (v 127/128) / d
};
__device__ __forceinline__ RowScale row_scale(uint32_t top_bits) {
    constexpr float least = 127.0f * 0x1p-100f;
    const bool real = top_bits < 0x7F800000u;
    const float a = real ? fmaxf(__uint_as_float(top_bits), least) : __builtin_nanf("");
    RowScale r;
    r.s = a / 127.0f;
    r.d = a * 0x1p-7f;
    r.inv = 1.0f / r.d;
    return r;
}
// q + 1.5 * 2^23, whose low byte is q. The quotient is the correctly rounded one: of the product with the
// correctly rounded inverse, corrected by its exact remainder (a NaN scale gives 0).
__device__ __forceinline__ uint32_t quant_bits(float v, const RowScale& r) {
    const float t = v * 0.9921875f;
    const float q0 = t * r.inv;
    const float q = fmaf(fmaf(-q0, r.d, t), r.inv, q0);
    return __float_as_uint(q + 12582912.0f);
}
__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float d, const RowScale& r) {
    const uint32_t lo = __builtin_amdgcn_perm(quant_bits(b, r), quant_bits(a, r), 0x0C0C0400u);
    const uint32_t hi = __builtin_amdgcn_perm(quant_bits(d, r), quant_bits(c, r), 0x04000C0Cu);
    return lo | hi;
}

// silu(g) u in fp32, to about three roundings: rows are quantised by it, where an error moves a value across a
// border between two whole numbers (in the layer each such move costs up to a step). e^-g is the hardware's
// 2^t, t = -g log2(e) with its rounding error put back, and 1 / (1 + e^-g) the hardware's reciprocal corrected
// once. Below -80 e^-g may be no normal number, and u as large as fp32 numbers are: silu(g) = g e^g to 35 digits
// there, as two factors e^(g / 2). Past 128 silu(g) is g, and t is that of 128: g log2(e) may be past fp32's numbers.
__device__ __forceinline__ float silu_mul(float g, float u) {
    constexpr float l2e = 1.44269504088896340736f, l2e_lo = 1.92596299112661746887e-8f;
    const float e = fminf(g, 128.f);
    const float t = -e * l2e;
    const float lo = fmaf(-e, l2e, -t) - e * l2e_lo;
    const float p2 = __builtin_amdgcn_exp2f(t);
    const float d = 1.0f + fmaf(p2 * 0.69314718055994530942f, lo, p2);
    float r = __builtin_amdgcn_rcpf(d);
    r = fmaf(fmaf(-d, r, 1.0f), r, r);
    float h = g * r * u;
    if (g < -80.f) {
        const float m = __builtin_amdgcn_exp2f(g * 0.72134752044448170368f);
        h = (g * m) * (m * u);
    }
    return h;
}

// ---- products ----
__device__ __forceinline__ v4i mfma_i8(const u32x4& a, const u32x4& b, const v4i& c) {
    const v4i x{(int)a[0], (int)a[1], (int)a[2], (int)a[3]}, y{(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(x, y, c, 0, 0, 0);
}

__device__ __forceinline__ float bias_at(const OutParams& p, int n) {
    if (p.bias == nullptr) return 0.f;
    if (p.bias_f32) return reinterpret_cast<const float*>(p.bias)[n];
    const uint16_t v = reinterpret_cast<const uint16_t*>(p.bias)[n];
    return p.bf16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}

// Two values rounded to 16 bits.
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if constexpr (BF16) {
        using v2bf = __bf16 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2bf{(__bf16)a, (__bf16)b});
    } else {
        using v2h = _Float16 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2h{(_Float16)a, (_Float16)b});
    }
}
// Some of N adjacent 16-bit values (words w) from column col on.
template <int N>
__device__ __forceinline__ void store16_some(const OutParams& p, int64_t row, int col, const uint32_t (&w)[N / 2]) {
    uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + row * p.ldo + col;
#pragma unroll
    for (int r = 0; r < N; ++r)
        if (col + r < p.N) o[r] = (uint16_t)(w[r / 2] >> (r % 2 * 16));
}
// Four adjacent columns of one row.
__device__ __forceinline__ void store16(const OutParams& p, int64_t row, int col, const v4f& t) {
    uint32_t w[2];
    if (p.bf16) {
        w[0] = pack16<true>(t[0], t[1]);
        w[1] = pack16<true>(t[2], t[3]);
    } else {
        w[0] = pack16<false>(t[0], t[1]);
        w[1] = pack16<false>(t[2], t[3]);
    }
    if (p.out8 && col + 4 <= p.N)
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + row * p.ldo + col) = make_uint2(w[0], w[1]);
    else
        store16_some<4>(p, row, col, w);
}

// ---- launchers (all enqueue on the stream) ----
enum class Rows : int { kF16 = 0, kBf16 = 1, kF32 = 2 };   // what rows are quantised from
// int8 rows and scales of x (rows, K), or of silu(gate) * up of x = [gate | up] (rows, 2 K). With sorted_ids, padded
// rows r < ntp without a slot in [0, num_valid) are left out.
int launch_act_quant_int8(const void* x, Rows src, int64_t rows, int64_t K, int64_t ldx, bool silu, int8_t* q, float* scales,
                          const int32_t* sorted_ids, const int32_t* ntp, int64_t num_valid, hipStream_t s);
// Weight-streaming product (int8_rows.hip): any sizes, up to kScanSlots slots; rows that are not int8 up to
// int8_rows_quantised_in_kernel().
bool int8_rows_quantised_in_kernel(int64_t K);
int launch_int8_rows(const RowsArgs& a, hipStream_t s);
// The second product (rows by slot, fp32) and the sum over each token's slots in one, rounded to 16 bits: out (T, N).
bool int8_token_supported(int64_t slots, int64_t E, int64_t inter);
int launch_int8_token(const RowsArgs& a, const float* topk_weights, hipStream_t s);
// Tiles (int8_tiles.hip): sizes that 32-bit offsets reach; grouped, blocks of as many rows as a tile has: 64 or 128.
int launch_int8_tiles(const Int8Args& a, hipStream_t s);
// out[t, n] = sum over the slots j in order of tw[t, j] * y[t top_k + j, n], rounded to 16 bits; slots whose (mapped)
// expert is not in [0, E) contribute nothing. N % 8 == 0.
int launch_int8_reduce(const float* y, const float* tw, const int32_t* ids, const int32_t* emap, int64_t emap_len, int64_t E,
                       int64_t T, int64_t N, int64_t top_k, void* out, bool bf16, hipStream_t s);

}  // namespace w4a8
