// int8 products of few rows (gfx950): the weights are streamed once, dense or grouped by expert.
//
// Bound: HBM, every weight once per 16 rows. Weights go from memory to the MFMA operands' registers with no
// detour: of each step of 128 values, lane (q, c) = (lane / 16, lane % 16) holds the 16-byte pieces q and q + 4 of
// row c, for rows and weights alike (a sum of whole numbers may take its k in any order). Weights are the first
// operand: a lane ends up with four adjacent columns of one row.
//
// Grouped, a work-group finds its rows itself: it scans the routed ids for the slots of its expert, so that no launch has
// to sort them first.
//
// int8_rows_kernel holds its rows in registers (16 rows by GPW steps a wave, quantised there where they come in 16 or 32
// bits) and walks over column fragments with D of them in flight; KS waves share K and add their sums in LDS.
// int8_stream_kernel takes any K and reads int8 rows again for each column fragment.
#include <algorithm>
#include <type_traits>

#include "int8.h"

namespace w4a8 {
namespace {

// ---- a work-group's rows ----
constexpr int kOneSlot = 2;
struct Routed {
    int e;            // expert
    int n;            // its rows
};
// The expert of slot i (an id of no local expert: -1).
__device__ __forceinline__ int expert_of(const RowsParams& p, int i) {
    int e = p.ids[i];
    if (p.emap != nullptr) e = e >= 0 && e < p.emap_len ? p.emap[e] : -1;
    return e >= 0 && e < p.E ? e : -1;
}
// Group g of rows: dense, all of them; else the slots of one expert, in order, in `list`: of expert g, or (by_slot, for
// fewer slots than experts) of slot g's expert, where slot g is its first; or slot g alone (kOneSlot). WAVES: of the work-group, all of which call
// this.
template <int WAVES>
__device__ __forceinline__ Routed find_rows(const RowsParams& p, int g, uint16_t* list, int* counts) {
    if (p.ids == nullptr) return {0, p.rows};
    const int e = p.by_slot ? __builtin_amdgcn_readfirstlane(expert_of(p, g)) : g;
    if (e < 0) return {0, 0};
    if (p.by_slot == kOneSlot) return {e, 1};
    constexpr int kMost = kScanSlots / (64 * WAVES);             // slots a lane
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per = (p.slots + 64 * WAVES - 1) / (64 * WAVES);   // steps of 64 slots a wave
    const int first = wave * per * 64 + lane;
    uint32_t mine = 0, sooner = 0;                               // bit i: slot first + 64 i
#pragma unroll 4
    for (int i = 0; i < kMost; ++i) {
        if (i >= per) break;
        const int s = first + 64 * i;
        if (s < p.slots && expert_of(p, s) == e) {
            mine |= 1u << i;
            sooner |= s < g ? 1u : 0u;
        }
    }
    int n = 0;
    for (int i = 0; i < per; ++i) n += __popcll(__ballot(mine >> i & 1));
    const bool late = p.by_slot && __ballot(sooner != 0) != 0;
    if (lane == 0) counts[wave] = late ? -1 : n;
    __syncthreads();
    int at = 0;
    n = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (counts[w] < 0) return {e, 0};                        // (all waves)
        if (w < wave) at += counts[w];
        n += counts[w];
    }
    if (n == 0) return {e, 0};
    for (int i = 0; i < per; ++i) {
        const uint64_t m = __ballot(mine >> i & 1);
        if (mine >> i & 1) list[at + __popcll(m & ((1ull << lane) - 1))] = (uint16_t)(first + 64 * i);
        at += __popcll(m);
    }
    __syncthreads();
    return {e, n};
}
// Row r of the group: its slot (dense: r), -1 past the end.
__device__ __forceinline__ int slot_at(const RowsParams& p, const Routed& d, int g, int r, const uint16_t* list) {
    if (r >= d.n) return -1;
    return p.ids == nullptr ? r : p.by_slot == kOneSlot ? g : list[r];
}

// ---- rows' values ----
template <Src8 SRC>
constexpr int kSrcBytes = SRC == Src8::kI8 ? 1 : SRC == Src8::kF32 ? 4 : 2;
template <Src8 SRC>
struct Raw8 {                                                    // eight values of a row
    u32x4 v[SRC == Src8::kF32 ? 2 : 1];
    __device__ __forceinline__ void load(const uint8_t* row, int k) {
#pragma unroll
        for (int b = 0; b < (SRC == Src8::kF32 ? 2 : 1); ++b)
            v[b] = *reinterpret_cast<const u32x4*>(row + (int64_t)k * kSrcBytes<SRC> + 16 * b);
    }
    __device__ __forceinline__ float value(int t) const {
        if constexpr (SRC == Src8::kF32) return __uint_as_float(v[t / 4][t % 4]);
        const uint32_t u = v[0][t / 2];
        if constexpr (SRC == Src8::kBf16) return __uint_as_float((t & 1) ? u & 0xFFFF0000u : u << 16);
        return __half2float(__ushort_as_half((uint16_t)((t & 1) ? u >> 16 : u & 0xFFFF)));
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int t = 0; t < 8; ++t) m = max(m, abs_bits(value(t)));
        return m;
    }
};

struct UMax8 {
    __device__ float operator()(float a, float b) const {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    }
};

// CG groups of KS waves; a group walks over its own `per` column fragments (kSiluF32: fragments of the gate half, each
// with its up fragment), D in flight.
template <int GPW, int KS, int CG, int D, Src8 SRC, Out8 DST>
__global__ void __launch_bounds__(64 * KS * CG, KS * CG <= 4 ? 2 : 1) int8_rows_kernel(RowsParams p, int slices, int per) {
    constexpr bool kSilu = DST == Out8::kSiluF32;
    constexpr int kPair = kSilu ? 2 : 1;                         // fragments of one output fragment
    static_assert(D % kPair == 0, "an output fragment's parts are in flight together");
    constexpr int kUnits = D / kPair;                            // output fragments of one round
    constexpr int kWaves = KS * CG;
    __shared__ __attribute__((aligned(16))) v4i part[KS > 1 ? 2 : 1][KS > 1 ? CG : 1][KS > 1 ? D : 1][KS > 1 ? KS : 1][64];
    __shared__ uint16_t list[kScanSlots];
    __shared__ int counts[kWaves];
    // sixteen quantised rows (16 bytes apart beside their values: sixteen lanes then read different banks) and their scales
    constexpr bool kQuant = SRC != Src8::kI8;
    constexpr int kRowK = GPW * KS * kStep + 16;
    __shared__ __attribute__((aligned(16))) int8_t s_x[kQuant ? 16 * kRowK : 16];
    __shared__ uint32_t s_top[kQuant ? 16 : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = wave % KS, cg = wave / KS;
    const int q = lane >> 4, c = lane & 15;
    const int group = blockIdx.x / slices, sl = blockIdx.x % slices;
    const Routed rt = find_rows<kWaves>(p, group, list, counts);
    if (rt.n == 0) return;
    const int half = p.N / 2;
    const int cols = kSilu ? half : p.N;
    const int K = p.K, G = (K + kStep - 1) / kStep;
    const int frags = (cols + 15) / 16;
    const int f0 = (sl * CG + cg) * per;                         // first output fragment of this group
    const int g0 = ks * GPW;                                     // first step of this wave
    const int8_t* we = p.w + (int64_t)rt.e * p.N * K;
    const float* wse = p.ws + (int64_t)rt.e * p.N;

    // ---- weights: step i is fragment f0 + i / kPair of the gate (i even) or the up half ----
    struct Stage {
        u32x4 w[GPW][2];
    };
    auto load = [&](Stage& s, int i) __attribute__((always_inline)) {
        const int f = min(f0 + min(i / kPair, per - 1), frags - 1);
        const int up = kSilu && (i & 1) ? half : 0;
        // (columns past the end read the last one; never stored)
        const int8_t* wr = we + (int64_t)(up + min(f * 16 + c, cols - 1)) * K;
#pragma unroll
        for (int j = 0; j < GPW; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = min(min(g0 + j, G - 1) * kStep + h * 64 + q * 16, K - 16);
                s.w[j][h] = *reinterpret_cast<const u32x4*>(wr + k);
            }
    };
    Stage ring[D];
    const int mine = min(per, frags - f0);                       // output fragments of this group (may be <= 0)
    const int rounds = (per * kPair + D - 1) / D;                // of the work-group: the barriers agree
    for (int r0 = 0; r0 < rt.n; r0 += 16) {
        // ---- sixteen rows, held ----
        const int slot = slot_at(p, rt, group, r0 + c, list);
        const int row = slot < 0 ? slot_at(p, rt, group, r0, list) : slot;   // (a row that exists; never stored)
        const int xrow = p.gather ? row / p.top_k : row;
        u32x4 x[GPW][2];
        float xs;
        auto first_weights = [&]() __attribute__((always_inline)) {
            if (r0 > 0) return;
#pragma unroll
            for (int d = 0; d < D; ++d) load(ring[d], d);
            __builtin_amdgcn_sched_barrier(0);
        };
        if constexpr (!kQuant) {
            const int8_t* xp = reinterpret_cast<const int8_t*>(p.x) + (int64_t)xrow * p.ldx;
            xs = p.xs[xrow];
#pragma unroll
            for (int j = 0; j < GPW; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    x[j][h] = *reinterpret_cast<const u32x4*>(xp + min(min(g0 + j, G - 1) * kStep + h * 64 + q * 16, K - 16));
            first_weights();
        } else {
            // The work-group quantises its real rows, eight values a thread and turn, into LDS, kHold turns' loads
            // together. The first turns' values stay in registers between the maximum and the rounding; they are loaded
            // before the weights, as loads return in order.
            constexpr int kHold = 4, kThreads = 64 * kWaves;
            const int live = min(16, rt.n - r0), pieces = K / 8, items = live * pieces;
            const bool whole = pieces % 64 == 0;                 // a wave's pieces are of one row
            Raw8<SRC> raw[kHold];
            int rr[kHold], rk[kHold];
            auto read = [&](int first) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    const int item = min(first + i * kThreads, items - 1);
                    rr[i] = item / pieces;
                    rk[i] = (item - rr[i] * pieces) * 8;
                    const int s = slot_at(p, rt, group, r0 + rr[i], list);
                    raw[i].load(reinterpret_cast<const uint8_t*>(p.x) + (int64_t)(p.gather ? s / p.top_k : s) * p.ldx * kSrcBytes<SRC>, rk[i]);
                }
            };
            auto maxima = [&](int first) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    const int item = first + i * kThreads;
                    if (whole) {
                        if (item - lane >= items) break;         // (of the whole wave)
                        const uint32_t m = __float_as_uint(lane_allreduce<6>(__uint_as_float(raw[i].top()), UMax8{}));
                        if (lane == 0) atomicMax(&s_top[rr[i]], m);
                    } else if (item < items) {
                        atomicMax(&s_top[rr[i]], raw[i].top());
                    }
                }
            };
            auto put = [&](int first) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    if (first + i * kThreads >= items) break;
                    const RowScale sc = row_scale(s_top[rr[i]]);
                    *reinterpret_cast<uint2*>(s_x + rr[i] * kRowK + rk[i]) =
                        make_uint2(quant4(raw[i].value(0), raw[i].value(1), raw[i].value(2), raw[i].value(3), sc),
                                   quant4(raw[i].value(4), raw[i].value(5), raw[i].value(6), raw[i].value(7), sc));
                }
            };
            constexpr int kTurn = kHold * kThreads;
            read(tid);
            __builtin_amdgcn_sched_barrier(0);
            first_weights();
            if (r0 > 0) __syncthreads();                         // (the last rows have been read)
            if (tid < 16) s_top[tid] = 0;
            lds_barrier();
            maxima(tid);
            for (int t = tid + kTurn; t - tid < items; t += kTurn) {
                read(t);
                maxima(t);
            }
            lds_barrier();
            if (items > kTurn) read(tid);
            put(tid);
            for (int t = tid + kTurn; t - tid < items; t += kTurn) {
                read(t);
                put(t);
            }
            lds_barrier();
            xs = row_scale(s_top[c]).s;
#pragma unroll
            for (int j = 0; j < GPW; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)                      // (rows that are not real hold anything)
                    x[j][h] = *reinterpret_cast<const u32x4*>(s_x + c * kRowK + (g0 + j) * kStep + h * 64 + q * 16);
        }
        // (what the clamped addresses hold counts in its own place)
#pragma unroll
        for (int j = 0; j < GPW; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if ((g0 + j) * kStep + h * 64 + q * 16 >= K) x[j][h] = u32x4{0, 0, 0, 0};
        __builtin_amdgcn_sched_barrier(0);

        for (int it = 0; it < rounds; ++it) {
            v4i run[D];
#pragma unroll
            for (int d = 0; d < D; ++d) {
                run[d] = v4i{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < GPW; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) run[d] = mfma_i8(ring[d].w[j][h], x[j][h], run[d]);
                __builtin_amdgcn_sched_barrier(0);
                // (behind the last round: the first fragments again, for the next sixteen rows)
                const int next = (it + 1) * D + d;
                load(ring[d], it + 1 < rounds ? next : d);
                __builtin_amdgcn_sched_barrier(0);
            }
            // unit u of the round: an output fragment
            auto put = [&](int u, const v4i& a, const v4i& b) __attribute__((always_inline)) {
                const int of = it * kUnits + u;
                const int col = (f0 + of) * 16 + 4 * q;
                if (of >= mine || slot < 0 || col >= cols) return;
                v4f t;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int n = min(col + r, cols - 1);
                    const float f = xs * wse[n];
                    if constexpr (kSilu) t[r] = silu_mul((float)a[r] * f, (float)b[r] * (xs * wse[half + n]));
                    else if constexpr (DST == Out8::k16) t[r] = fmaf((float)a[r], f, bias_at(p, n));
                    else t[r] = (float)a[r] * f;
                }
                if constexpr (DST == Out8::k16) store16(p, slot, col, t);
                else *reinterpret_cast<v4f*>(reinterpret_cast<float*>(p.out) + (int64_t)slot * p.ldo + col) = t;
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
                        v4i t = buf[d][0][lane];
#pragma unroll
                        for (int w = 1; w < KS; ++w) t += buf[d][w][lane];
                        return t;
                    };
                    const v4i t = total(u * kPair);
                    if constexpr (kSilu) put(u, t, total(u * kPair + 1));
                    else put(u, t, t);
                }
            }
        }
        if (KS > 1) lds_barrier();                               // (an odd number of rounds: the first buffer is read)
    }
}

// Any K, int8 rows: KS waves take the steps of K in turn (what they read at one time is contiguous along K).
constexpr int kRing = 3;          // steps of a wave in flight
template <int FN, int KS, Out8 DST>
__global__ void __launch_bounds__(64 * KS) int8_stream_kernel(RowsParams p, int slices) {
    constexpr bool kSilu = DST == Out8::kSiluF32;
    constexpr int kCols = kSilu ? FN / 2 : FN;                   // column fragments of the output
    __shared__ __attribute__((aligned(16))) v4i part[KS][FN][64];
    __shared__ uint16_t list[kScanSlots];
    __shared__ int counts[KS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, c = lane & 15;
    const int group = blockIdx.x / slices, sl = blockIdx.x % slices;
    const Routed rt = find_rows<KS>(p, group, list, counts);
    if (rt.n == 0) return;
    const int half = p.N / 2;
    const int cols = kSilu ? half : p.N;
    const int K = p.K;
    const int8_t* wp[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int f = (sl * kCols + j % kCols) * 16, up = kSilu && j >= kCols ? half : 0;
        wp[j] = p.w + ((int64_t)rt.e * p.N + up + min(f + c, cols - 1)) * K;
    }
    const float* ws = p.ws + (int64_t)rt.e * p.N;
    const int G = (K + kStep - 1) / kStep, steps = (G + KS - 1) / KS;
    for (int r0 = 0; r0 < rt.n; r0 += 16) {
        const int slot = slot_at(p, rt, group, r0 + c, list);
        const int row = slot < 0 ? slot_at(p, rt, group, r0, list) : slot;
        const int xrow = p.gather ? row / p.top_k : row;
        const int8_t* xp = reinterpret_cast<const int8_t*>(p.x) + (int64_t)xrow * p.ldx;
        struct Stage {
            u32x4 w[FN][2], x[2];
        };
        auto load = [&](Stage& s, int step) __attribute__((always_inline)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // (pieces past the end: the last one, and zeros for the rows')
                const int k = (step * KS + wave) * kStep + h * 64 + q * 16, at = min(k, K - 16);
#pragma unroll
                for (int j = 0; j < FN; ++j) s.w[j][h] = *reinterpret_cast<const u32x4*>(wp[j] + at);
                s.x[h] = *reinterpret_cast<const u32x4*>(xp + at);
                if (k >= K) s.x[h] = u32x4{0, 0, 0, 0};
            }
        };
        v4i run[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) run[j] = v4i{0, 0, 0, 0};
        Stage ring[kRing];
#pragma unroll
        for (int d = 0; d < kRing; ++d) load(ring[d], d);
        for (int s0 = 0; s0 < steps; s0 += kRing) {
#pragma unroll
            for (int d = 0; d < kRing; ++d) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < FN; ++j) run[j] = mfma_i8(ring[d].w[j][h], ring[d].x[h], run[j]);
                __builtin_amdgcn_sched_barrier(0);
                load(ring[d], s0 + d + kRing);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (r0 > 0) __syncthreads();                             // (the last rows' sums have been read)
#pragma unroll
        for (int j = 0; j < FN; ++j) part[wave][j][lane] = run[j];
        __syncthreads();
        // wave j joins column fragment j (four adjacent columns of a row a lane)
        static_assert(kCols <= KS, "a wave a fragment");
        const int col = (sl * kCols + wave) * 16 + 4 * q;
        if (wave >= kCols || slot < 0 || col >= cols) continue;
        auto total = [&](int f) __attribute__((always_inline)) {
            v4i t = part[0][f][lane];
#pragma unroll
            for (int w = 1; w < KS; ++w) t += part[w][f][lane];
            return t;
        };
        const v4i a = total(wave), b = kSilu ? total(kCols + wave) : a;
        const float xs = p.xs[xrow];
        v4f t;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = min(col + r, cols - 1);
            const float f = xs * ws[n];
            if constexpr (kSilu) t[r] = silu_mul((float)a[r] * f, (float)b[r] * (xs * ws[half + n]));
            else if constexpr (DST == Out8::k16) t[r] = fmaf((float)a[r], f, bias_at(p, n));
            else t[r] = (float)a[r] * f;
        }
        if constexpr (DST == Out8::k16) store16(p, slot, col, t);
        else *reinterpret_cast<v4f*>(reinterpret_cast<float*>(p.out) + (int64_t)slot * p.ldo + col) = t;
    }
}

// The layer's second product and its sum over a token's slots, for hardly two slots of one expert: a work-group takes a
// token and FN column fragments, wave w the token's slots w, w + 8, ... in turn. A wave quantises its slot's row of h (fp32)
// alone, multiplies by its expert's weights, and the slots are added in order through LDS. Saves a launch and the slots'
// rows (one token of 256 experts, 2048 x 512: 18.3 -> 16.4 us).
constexpr int kTokenWaves = 8;
constexpr int kTokenK = 4096;
template <int FN>
__global__ void __launch_bounds__(64 * kTokenWaves) int8_token_kernel(RowsParams p, const float* __restrict__ tw, int slices) {
    __shared__ __attribute__((aligned(16))) int8_t s_x[kTokenWaves][kTokenK];
    __shared__ __attribute__((aligned(16))) v4f s_y[kTokenWaves][FN][4];
    __shared__ int s_live[kTokenWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, c = lane & 15;
    const int t = blockIdx.x / slices, f0 = blockIdx.x % slices * FN;
    const int K = p.K, G = (K + kStep - 1) / kStep, cols = p.N;
    v4f sum{0.f, 0.f, 0.f, 0.f};                                 // wave j < FN: of column fragment j, in lanes c == 0
    for (int j0 = 0; j0 < p.top_k; j0 += kTokenWaves) {
        const int slot = t * p.top_k + j0 + wave;
        const int e = j0 + wave < p.top_k ? __builtin_amdgcn_readfirstlane(expert_of(p, slot)) : -1;
        if (e >= 0) {
            // the row's values, eight a lane and piece, before the weights: loads return in order
            const uint8_t* row = reinterpret_cast<const uint8_t*>(p.x) + (int64_t)slot * p.ldx * 4;
            constexpr int kHold = 2;
            Raw8<Src8::kF32> raw[kHold];
#pragma unroll
            for (int i = 0; i < kHold; ++i) raw[i].load(row, min((lane + 64 * i) * 8, K - 8));
            const int8_t* wp[FN];
            float ws[FN][4];
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                wp[j] = p.w + ((int64_t)e * cols + min((f0 + j) * 16 + c, cols - 1)) * K;
#pragma unroll
                for (int r = 0; r < 4; ++r) ws[j][r] = p.ws[(int64_t)e * cols + min((f0 + j) * 16 + 4 * q + r, cols - 1)];
            }
            constexpr int kAhead = 4;                            // steps whose weights are in flight
            u32x4 w[kAhead][FN][2];
            auto load = [&](int i, int g) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        w[i][j][h] = *reinterpret_cast<const u32x4*>(wp[j] + min(min(g, G - 1) * kStep + h * 64 + q * 16, K - 16));
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) load(i, i);
            __builtin_amdgcn_sched_barrier(0);
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kHold; ++i) top = max(top, raw[i].top());
            for (int k = (lane + 64 * kHold) * 8; k < K; k += 512) {
                Raw8<Src8::kF32> more;
                more.load(row, k);
                top = max(top, more.top());
            }
            const RowScale sc = row_scale(__float_as_uint(lane_allreduce<6>(__uint_as_float(top), UMax8{})));
            auto put = [&](const Raw8<Src8::kF32>& v, int k) __attribute__((always_inline)) {
                *reinterpret_cast<uint2*>(&s_x[wave][k]) = make_uint2(quant4(v.value(0), v.value(1), v.value(2), v.value(3), sc),
                                                                      quant4(v.value(4), v.value(5), v.value(6), v.value(7), sc));
            };
#pragma unroll
            for (int i = 0; i < kHold; ++i)
                if ((lane + 64 * i) * 8 < K) put(raw[i], (lane + 64 * i) * 8);
            for (int k = (lane + 64 * kHold) * 8; k < K; k += 512) {
                Raw8<Src8::kF32> more;
                more.load(row, k);
                put(more, k);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
            v4i run[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) run[j] = v4i{0, 0, 0, 0};
            for (int g0 = 0; g0 < G; g0 += kAhead)
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {                // (every lane of the sixteen has the one row)
                        const int k = (g0 + i) * kStep + h * 64 + q * 16;
                        u32x4 x = *reinterpret_cast<const u32x4*>(&s_x[wave][min(k, kTokenK - 16)]);
                        if (k >= K) x = u32x4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < FN; ++j) run[j] = mfma_i8(w[i][j][h], x, run[j]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    load(i, g0 + i + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
            if (c == 0)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    s_y[wave][j][q] = v4f{(float)run[j][0] * (sc.s * ws[j][0]), (float)run[j][1] * (sc.s * ws[j][1]),
                                          (float)run[j][2] * (sc.s * ws[j][2]), (float)run[j][3] * (sc.s * ws[j][3])};
        }
        if (lane == 0) s_live[wave] = e >= 0 ? 1 : 0;
        __syncthreads();
        if (wave < FN && c == 0)
            for (int w = 0; w < kTokenWaves && j0 + w < p.top_k; ++w)
                if (s_live[w]) {
                    const float f = tw[t * p.top_k + j0 + w];
                    const v4f y = s_y[w][wave][q];
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum[r] = fmaf(f, y[r], sum[r]);
                }
        __syncthreads();
    }
    const int col = (f0 + wave) * 16 + 4 * q;
    if (wave < FN && c == 0 && col < cols) store16(p, t, col, sum);
}

int too_many() {
    set_error("int8 product: too many tiles");
    return W4A8_ERR_INVALID;
}
// Groups of rows that work-groups take.
int64_t groups_of(const RowsParams& p) { return p.ids == nullptr ? 1 : std::min(p.slots, p.E); }
template <int FN, int KS, Out8 DST>
int stream_go(const RowsParams& p, hipStream_t s) {
    constexpr bool silu = DST == Out8::kSiluF32;
    const int cols = silu ? p.N / 2 : p.N, per = 16 * (silu ? FN / 2 : FN);
    const int slices = (cols + per - 1) / per;
    const int64_t grid = groups_of(p) * slices;
    if (!grid_fits(grid, 64 * KS)) return too_many();
    launch_kernel(&int8_stream_kernel<FN, KS, DST>, dim3((unsigned)grid), dim3(64 * KS), 0, s, p, slices);
    return check_launch("int8_stream_kernel");
}

// per: output fragments a group of waves walks over. The kernel loads D fragments beforehand whatever `per` is, so few of
// them take a variant with a smaller D.
template <int GPW, int KS, int CG, int D, Src8 SRC, Out8 DST>
int rows_launch(const RowsParams& p, int frags, int64_t per, hipStream_t s) {
    constexpr int pair = DST == Out8::kSiluF32 ? 2 : 1;
    if constexpr (D > pair)
        if (per * pair <= D / 2) return rows_launch<GPW, KS, CG, D / 2, SRC, DST>(p, frags, per, s);
    const int slices = (int)((frags + per * CG - 1) / (per * CG));
    const int64_t grid = groups_of(p) * slices;
    if (!grid_fits(grid, 64 * KS * CG)) return too_many();
    launch_kernel(&int8_rows_kernel<GPW, KS, CG, D, SRC, DST>, dim3((unsigned)grid), dim3(64 * KS * CG), 0, s, p, slices, (int)per);
    return check_launch("int8_rows_kernel");
}

template <int GPW, int KS, int CG, int D, Src8 SRC, Out8 DST>
int rows_go(const RowsParams& p, hipStream_t s) {
    constexpr int unit = D / (DST == Out8::kSiluF32 ? 2 : 1);
    const int frags = ((DST == Out8::kSiluF32 ? p.N / 2 : p.N) + 15) / 16;
    // As many work-groups as run at once (eight waves a CU), those of groups without rows among them, each walking over
    // what that leaves it: some more would run behind all others. us of a layer of 256 experts (2048 x 512, 8 a token), by
    // the first product's fragments a work-group 1 / 2 / 4 / 8 / 16 / 32 (the rule's in brackets): 8 tokens 63 / 53 / (47) /
    // 48 / 62 / 94, 16 tokens 104 / 92 / 82 / (78) / 78 / 107, 64 tokens 229 / 194 / 176 / 170 / (168) / 165.
    const int64_t resident = (int64_t)device_cu_count() * std::max(1, 8 / (KS * CG));
    const int64_t slices = std::max<int64_t>(1, resident / groups_of(p));
    int64_t per = (frags + CG * slices - 1) / (CG * slices);
    if (per > unit) per = (per + unit - 1) / unit * unit;
    return rows_launch<GPW, KS, CG, D, SRC, DST>(p, frags, std::max<int64_t>(1, per), s);
}

// The wave split by the number of steps: a wave holds the rows' values of up to four of them, up to eight waves share K.
template <Src8 SRC, Out8 DST>
int rows_any(const RowsParams& p, hipStream_t s) {
    const int G = (p.K + kStep - 1) / kStep;
    if (G <= 1) return rows_go<1, 1, 4, 4, SRC, DST>(p, s);
    if (G <= 2) return rows_go<2, 1, 4, 4, SRC, DST>(p, s);
    if (G <= 4) return rows_go<4, 1, 4, 2, SRC, DST>(p, s);
    if (G <= 8) return rows_go<2, 4, 1, 4, SRC, DST>(p, s);
    if (G <= 16) return rows_go<4, 4, 1, 2, SRC, DST>(p, s);
    if (G <= 32) return rows_go<4, 8, 1, 2, SRC, DST>(p, s);
    if constexpr (SRC == Src8::kI8) return stream_go<DST == Out8::kSiluF32 ? 2 : 1, 8, DST>(p, s);
    set_error("int8 product: rows too long to be quantised in the kernel");
    return W4A8_ERR_INVALID;
}

}  // namespace

bool int8_rows_quantised_in_kernel(int64_t K) { return K <= 32 * kStep; }

// Hardly two slots of one expert, whose weights would be read twice: no scan for them, either (one token of 256 experts,
// 2048 x 512: 16.4 -> 15.6 us).
bool few_slots(int64_t slots, int64_t E) { return slots * 8 <= E; }
bool int8_token_supported(int64_t slots, int64_t E, int64_t inter) { return few_slots(slots, E) && inter <= kTokenK; }

int launch_int8_token(const RowsArgs& a, const float* topk_weights, hipStream_t s) {
    const RowsParams p = rows_params(a);
    const int frags = (p.N + 15) / 16, tokens = p.slots / p.top_k;
    // one fragment a work-group while those run at once (four a CU), else two
    const bool two = (int64_t)tokens * frags > 4 * (int64_t)device_cu_count();
    const int slices = two ? (frags + 1) / 2 : frags;
    const int64_t grid = (int64_t)tokens * slices;
    if (!grid_fits(grid, 64 * kTokenWaves)) return too_many();
    launch_kernel(two ? &int8_token_kernel<2> : &int8_token_kernel<1>, dim3((unsigned)grid), dim3(64 * kTokenWaves), 0, s, p,
                  topk_weights, slices);
    return check_launch("int8_token_kernel");
}

int launch_int8_rows(const RowsArgs& a, hipStream_t s) {
    RowsParams p = rows_params(a);
    p.by_slot = few_slots(p.slots, p.E) ? kOneSlot : p.slots < p.E ? 1 : 0;
    if (p.rows == 0 || (p.ids != nullptr && p.slots == 0)) return W4A8_OK;
    if (p.ids != nullptr && p.slots > kScanSlots) {
        set_error("int8 product: too many slots for the streaming kernels");
        return W4A8_ERR_INVALID;
    }
    if (a.dst == Out8::kSlotF32) return a.src == Src8::kI8 ? rows_any<Src8::kI8, Out8::kSlotF32>(p, s) : rows_any<Src8::kF32, Out8::kSlotF32>(p, s);
    auto from = [&](auto dst) -> int {
        constexpr Out8 DST = decltype(dst)::value;
        switch (a.src) {
            case Src8::kI8: return rows_any<Src8::kI8, DST>(p, s);
            case Src8::kF16: return rows_any<Src8::kF16, DST>(p, s);
            case Src8::kBf16: return rows_any<Src8::kBf16, DST>(p, s);
            default: break;
        }
        set_error("int8 product: fp32 rows are the layer's second product's");
        return W4A8_ERR_INVALID;
    };
    if (a.dst == Out8::kSiluF32) return from(std::integral_constant<Out8, Out8::kSiluF32>{});
    return from(std::integral_constant<Out8, Out8::k16>{});
}

}  // namespace w4a8
