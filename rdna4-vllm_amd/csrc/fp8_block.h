// Block-scaled fp8 (W8A8) operators: parameters and device helpers shared by their kernels.
//
// Numerics: rows are e4m3 with one fp32 scale per row and 128 values, weights e4m3 with one fp32
// scale per 128 x 128 block (n / 128, k / 128):
//   out[m, n] = sum_g xs[m, g] * ws[n / 128, g] * sum_{k in group g} x[m, k] w[n, k].
// The inner sum is one fp8 MFMA of 128 k with a zero accumulator (fp32), in the layer's first product four
// chained bf16 MFMAs (fp8_mfma.h says why); the outer one is an fp32 FMA chain over g in each wave.
// Quantisation: s = max(absmax / 448, 1e-8), q = e4m3(x * (1 / s)) in fp32, to nearest even; NaN counts for
// no absmax and stays NaN.
#pragma once

#include "grouped_params.h"

namespace w4a8 {

constexpr int kBlk = 128;                     // values a row scale covers, sides of a weight block

inline int64_t blk_groups(int64_t n) { return (n + kBlk - 1) / kBlk; }

// What a product reads its rows from.
enum class Src : int {
    kFp8 = 0,    // e4m3 rows with their scales
    kF16 = 1,    // fp16 / bf16 rows, quantised in registers
    kBf16 = 2,
    kF32 = 3,    // fp32 rows, quantised in registers
    kWide = 4,   // as kFp8, the e4m3 values as the bf16 numbers that they are (tiles of the layer's first product)
};
// What it writes.
enum class Dst : int {
    kF16 = 0,       // out[row, n] rounded to fp16, or to bf16 (the kernels have one form for both)
    kBf16 = 1,
    kSiluF32 = 2,   // out[row, n] = silu(gate) * up in fp32, N = [gate | up] halves
    kSlotF32 = 3,   // out[slot, n] in fp32 (the layer's second product)
    kSiluFp8 = 4,   // silu(gate) * up quantised: e4m3 rows (out) and their scales (out_scales)
    kRowF16 = 5,    // out[row, n] in fp16 with a power of two per row and 32 columns (out_scales), so that
                    // no value overflows and none loses bits to a fixed range
};

struct BlockArgs {
    const void* x;               // rows, see Src
    const float* xs;             // (x_rows, G) scales of e4m3 rows
    int64_t x_rows, K, ldx;      // ldx: elements between rows
    const uint8_t* w;            // (E, N, K)
    const float* ws;             // (E, ceil(N / 128), G)
    int64_t E, N;
    const int32_t* sorted_ids;   // null: one expert, rows in order (dense)
    const int32_t* expert_ids;
    const int32_t* ntp;
    int64_t P;                   // padded rows (dense: rows)
    int64_t top_k, num_valid, block_m;
    bool gather;                 // row r reads x[slot / top_k], else x[r]
    Src src;
    Dst dst;
    void* out;
    float* out_scales;           // kSiluFp8: (P, inter / 128); kRowF16: (P, N / 32)
    int64_t ldo;
    bool all_rows;               // padding rows of out may be written (tiles)
};

// The same on the device, sizes in 32 bits where they fit.
struct BlockParams {
    const void* x;
    const float* xs;
    const uint8_t* w;
    const float* ws;
    const int32_t* sorted_ids;
    const int32_t* expert_ids;
    const int32_t* ntp;
    void* out;
    float* out_scales;
    int64_t ldx, ldo;
    int P, K, N, G, NB, E;
    int x_rows, top_k, num_valid, block_m, gather;
    int out8, out16;             // out is aligned to 8, to 16 bytes
    int out_bf16;                // Dst::kBf16
    int all_rows;
};

inline BlockParams block_params(const BlockArgs& a) {
    BlockParams p;
    p.x = a.x; p.xs = a.xs; p.w = a.w; p.ws = a.ws;
    p.sorted_ids = a.sorted_ids; p.expert_ids = a.expert_ids; p.ntp = a.ntp;
    p.out = a.out; p.out_scales = a.out_scales;
    p.ldx = a.ldx; p.ldo = a.ldo;
    p.P = (int)a.P; p.K = (int)a.K; p.N = (int)a.N; p.G = (int)blk_groups(a.K);
    p.NB = (int)blk_groups(a.N); p.E = (int)a.E;
    p.x_rows = (int)a.x_rows; p.top_k = (int)a.top_k; p.num_valid = (int)a.num_valid;
    p.block_m = (int)a.block_m; p.gather = a.gather ? 1 : 0;
    p.all_rows = a.all_rows ? 1 : 0;
    p.out_bf16 = a.dst == Dst::kBf16 ? 1 : 0;
    p.out8 = reinterpret_cast<uintptr_t>(a.out) % 8 == 0 ? 1 : 0;
    p.out16 = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 ? 1 : 0;
    return p;
}

// Padded row r: its slot (dense: r), or -1 for padding, and the row of x it reads (0 for padding:
// a row that exists, whose results are not stored). end: rows in use.
__device__ __forceinline__ int block_slot(const BlockParams& p, int r, int end, int& xrow) {
    xrow = 0;
    if (r >= end) return -1;
    if (p.sorted_ids == nullptr) {
        xrow = r;
        return r;
    }
    const int s = p.sorted_ids[r];
    if (s < 0 || s >= p.num_valid) return -1;
    const int row = p.gather ? s / p.top_k : r;
    if (row >= p.x_rows) return -1;
    xrow = row;
    return s;
}

// max / min over the four lanes c, c + 16, c + 32, c + 48 that hold a row's values.
__device__ __forceinline__ float rows4_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// SiLU(g) * u in fp32, N of them: 2^(-g log2 e) and the reciprocal from the hardware (each within an ulp),
// so about |g| * 2^-24 relative: far below the e4m3 step (2^-4) that every result is rounded to.
// FAR: u may be as large as fp32 numbers are. The reciprocal of 1 + e^-g is no normal number below -87.3 (the
// hardware gives 0), which a u of 1e30 shows; below -80 SiLU(g) = g e^g to 35 digits, as two factors e^(g / 2) of
// which u takes one. Asked for all N at once: with a choice for each value silu(gate) * up of 4111 x 12288
// bf16 takes 44.3 us for 42.8, and a layer of 4096 tokens 427 for 421. An fp16 u needs none (65504 e^-87 rounds to 0).
template <bool FAR, int N>
__device__ __forceinline__ void silu_mul_f32(const float (&g)[N], const float (&u)[N], float (&h)[N]) {
    float least = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        h[i] = g[i] * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g[i] * -1.44269504088896340736f)) * u[i];
        least = fminf(least, g[i]);
    }
    if constexpr (FAR)
        if (least < -80.f) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float t = __builtin_amdgcn_exp2f(g[i] * 0.72134752044448170368f);
                if (g[i] < -80.f) h[i] = (g[i] * t) * (t * u[i]);
            }
        }
}
__device__ __forceinline__ v4f silu_mul_f32(const v4f& g, const v4f& u) {
    const float a[4] = {g[0], g[1], g[2], g[3]}, b[4] = {u[0], u[1], u[2], u[3]};
    float h[4];
    silu_mul_f32<true>(a, b, h);
    return v4f{h[0], h[1], h[2], h[3]};
}

__device__ __forceinline__ uint32_t pack_out16(float a, float b, bool bf16) {
    if (bf16)
        return (uint32_t)__bfloat16_as_ushort(__float2bfloat16(a)) |
               ((uint32_t)__bfloat16_as_ushort(__float2bfloat16(b)) << 16);
    return (uint32_t)__half_as_ushort(__float2half(as_f32(a))) |
           ((uint32_t)__half_as_ushort(__float2half(as_f32(b))) << 16);
}

// A launch's work-items are counted in 32 bits.
inline bool grid_fits(int64_t blocks, int64_t threads) { return blocks < ((int64_t)1 << 32) / threads; }

// ---- launchers (all enqueue on the stream) ----
struct NormArgs {
    const void* x;
    const void* residual;        // null: none
    const void* weight;
    bool bf16, weight_f32;
    int64_t rows, H, ldx, ldr;
    float eps;
    bool per_row;                // one scale a row, else one per 128 values
    void* residual_out;          // rows, H contiguous; with residual
    void* norm_out;              // or null
    uint8_t* q;
    float* scales;
};
int launch_rms_norm_quant(const NormArgs& a, hipStream_t s);
// e4m3 rows and scales of x (rows, K), or of silu(gate) * up of x = [gate | up] (rows, 2 K).
int launch_act_quant_block(const void* x, bool bf16, int64_t rows, int64_t K, int64_t ldx, bool silu,
                           uint8_t* q, float* scales, hipStream_t s);
// The same rows for Src::kWide, from 16-bit rows (with their scales) or from e4m3 rows; K % 128 == 0,
// rows contiguous and aligned to 16 bytes.
int launch_act_quant_wide(const void* x, bool bf16, int64_t rows, int64_t K, uint16_t* q, float* scales, hipStream_t s);
int launch_widen_rows(const void* x, int64_t rows, int64_t K, uint16_t* q, hipStream_t s);
// Weight-streaming product (fp8_stream.hip): any sizes.
int launch_block_stream(const BlockArgs& a, hipStream_t s);
// Tiles (fp8_tiles.hip): e4m3 rows, sizes that 32-bit offsets reach.
bool block_tiles_supported(const BlockArgs& a);
int launch_block_tiles(const BlockArgs& a, hipStream_t s);
// out[t, n] = sum over the slots j in order of tw[t, j] * y[slot_to_row[t, j], n] in fp32, rounded to
// bf16; y as kRowF16 leaves it, rows < 0 contribute nothing. N % 32 == 0.
int launch_block_reduce(const void* y, const float* ys, const int32_t* slot_to_row, const float* tw, int64_t T, int64_t N,
                        int64_t top_k, void* out, hipStream_t s);

}  // namespace w4a8
