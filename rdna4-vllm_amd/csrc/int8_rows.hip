// int8 products of few rows (gfx950): the weights are streamed once, dense or grouped by expert.
//
// Bound: HBM, every weight once per 16 rows. Weights go from memory to the MFMA operands' registers with no
// detour: of each step of 128 values, lane (q, c) = (lane / 16, lane % 16) holds the 16-byte pieces q and q + 4 of
// row c, for rows and weights alike (a sum of whole numbers may take its k in any order). Weights are the first
// operand: a lane ends up with four adjacent columns of one row.
//
// Grouped, a work-group counts the routed ids by expert in LDS itself, so that no launch has to sort them first, and takes an
// equal part of what all experts with rows amount to. One or two slots of an expert, two thirds of 256 experts in use (32
// tokens, 8 picks, 2048 x 512): the layer's two products read 510 MB in 100 of its 108 us, 5.1 TB/s (a group a work-group
// column, whatever the number of experts in use: 128 us); reads alone, of the same pieces, reach 6.3.
//
// int8_rows_kernel holds its rows in registers (16 rows by GPW steps a wave, quantised in LDS where they come in 16 or 32
// bits) and walks over column fragments with D of them in flight; KS waves share K and add their sums in LDS. Four fragments
// in flight were slower than two (64 tokens: 103 us for 93 of the first product).
// int8_stream_kernel takes any K and reads int8 rows again for each column fragment.
#include <algorithm>
#include <type_traits>

#include "int8.h"

namespace w4a8 {
namespace {

// ---- groups of up to sixteen rows that share their weights ----
constexpr int kMaxExperts = 1024;
// The expert of slot i (an id of no local expert: -1).
__device__ __forceinline__ int expert_of(const RowsParams& p, int i) {
    int e = p.ids[i];
    if (p.emap != nullptr) e = e >= 0 && e < p.emap_len ? p.emap[e] : -1;
    return e >= 0 && e < p.E ? e : -1;
}
struct Routed {                                                  // in LDS
    uint32_t group[kMaxExperts + kScanSlots / 16];               // expert | its first place in slots << 10 | rows << 23
    uint32_t first[kMaxExperts + 1];                             // an expert's slots, then its first place
    uint32_t sums[16];
    int wide;                                                    // some expert has several groups
    uint16_t slots[kScanSlots];                                  // by expert
};
// The number of groups: dense, sixteen rows each in order; one_slot, a slot each; else the slots counted by expert, their
// experts' groups in order. WAVES: of the work-group, all of which call this.
template <int WAVES>
__device__ __forceinline__ int find_groups(const RowsParams& p, Routed& rt) {
    if (p.ids == nullptr) return (p.rows + 15) / 16;
    if (p.one_slot) return p.slots;
    constexpr int kThreads = 64 * WAVES, kMost = kScanSlots / kThreads, kEach = kMaxExperts / kThreads, kAhead = 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t mine[kMost];                                        // expert << 16 | its slots before this one
#pragma unroll
    for (int j = 0; j < kEach; ++j) rt.first[tid + j * kThreads] = 0;
    if (tid == 0) rt.wide = 0;
    __syncthreads();
#pragma unroll
    for (int i0 = 0; i0 < kMost; i0 += kAhead)
        if (i0 * kThreads < p.slots) {
            int e[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) e[i] = expert_of(p, min(tid + (i0 + i) * kThreads, p.slots - 1));
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                mine[i0 + i] = ~0u;
                if (e[i] >= 0 && tid + (i0 + i) * kThreads < p.slots)
                    mine[i0 + i] = (uint32_t)e[i] << 16 | atomicAdd(&rt.first[e[i]], 1u);
            }
        }
    __syncthreads();
    // slots | groups << 16 of the experts before
    uint32_t n[kEach], all = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        n[j] = rt.first[tid * kEach + j];
        all += n[j] | (n[j] + 15) / 16 << 16;
        if (n[j] > 16) rt.wide = 1;
    }
    uint32_t upto = all;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t o = (uint32_t)__shfl_up((int)upto, d);
        upto += lane >= d ? o : 0u;
    }
    if (lane == 63) rt.sums[wave] = upto;
    __syncthreads();
    uint32_t at = upto - all, total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        at += w < wave ? rt.sums[w] : 0u;
        total += rt.sums[w];
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const uint32_t e = tid * kEach + j;
        rt.first[e] = at & 0xFFFFu;
        for (uint32_t r = 0; r < n[j]; r += 16) {
            rt.group[at >> 16] = e | ((at & 0xFFFFu) + r) << 10 | min(16u, n[j] - r) << 23;
            at += 1u << 16;
        }
        at += n[j];
    }
    if (tid == kThreads - 1) rt.first[kMaxExperts] = at & 0xFFFFu;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMost; ++i)
        if (i * kThreads < p.slots && mine[i] != ~0u)
            rt.slots[rt.first[mine[i] >> 16] + (mine[i] & 0xFFFFu)] = (uint16_t)(tid + i * kThreads);
    __syncthreads();
    if (rt.wide) {
        // Work-groups have counted an expert's slots in orders of their own, but each has to find the same ones in each of
        // its groups: they are put in order.
#pragma unroll
        for (int i = 0; i < kMost; ++i)
            if (i * kThreads < p.slots && mine[i] != ~0u) {
                const uint32_t e = mine[i] >> 16, from = rt.first[e], to = rt.first[e + 1];
                uint32_t rank = 0;
                if (to - from > 16)
                    for (uint32_t j = from; j < to; ++j) rank += rt.slots[j] < tid + i * kThreads ? 1u : 0u;
                else
                    rank = mine[i] & 0xFFFFu;
                mine[i] = from + rank;
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMost; ++i)
            if (i * kThreads < p.slots && mine[i] != ~0u) rt.slots[mine[i]] = (uint16_t)(tid + i * kThreads);
        __syncthreads();
    }
    return __builtin_amdgcn_readfirstlane(total >> 16);
}
struct Group {
    int e;            // expert
    int n;            // rows: 0 to 16
    int at;           // the first one's place
    bool listed;      // places are of Routed's slots, else slots (dense: rows)
};
__device__ __forceinline__ Group group_at(const RowsParams& p, const Routed& rt, int g) {
    if (p.ids == nullptr) return {0, min(16, p.rows - 16 * g), 16 * g, false};
    if (p.one_slot) {
        const int e = __builtin_amdgcn_readfirstlane(expert_of(p, g));
        return {e, e < 0 ? 0 : 1, g, false};
    }
    const uint32_t v = __builtin_amdgcn_readfirstlane(rt.group[g]);
    return {(int)(v & 1023u), (int)(v >> 23), (int)(v >> 10 & 8191u), true};
}
__device__ __forceinline__ int slot_at(const Routed& rt, const Group& g, int i) { return g.listed ? rt.slots[g.at + i] : g.at + i; }
// The units (a group by an output fragment) of a work-group: of one group where that leaves it no more than an eighth over
// an equal part of all, else such a part, those of a group one after another.
struct Walk {
    int left, g, f;
    __device__ __forceinline__ Walk(int groups, int frags) {
        const uint32_t W = gridDim.x, b = blockIdx.x, n = (uint32_t)groups, units = n * (uint32_t)frags;
        const uint32_t s = n > 0 ? W / n : 0;                    // work-groups a group
        const uint32_t per = s > 0 ? ((uint32_t)frags + s - 1) / s : 0;
        if (s > 0 && (uint64_t)per * W * 8 <= (uint64_t)units * 9) {
            g = (int)(b / s);
            f = (int)((b - g * s) * per);
            left = g < groups ? min((int)per, frags - f) : 0;
        } else {
            const uint32_t each = units / W, more = units - each * W, u = b * each + min(b, more);
            left = (int)(each + (b < more ? 1u : 0u));
            g = (int)(u / (uint32_t)frags);
            f = (int)(u - (uint32_t)g * (uint32_t)frags);
        }
    }
    __device__ __forceinline__ int here(int frags) const { return min(left, frags - f); }
    __device__ __forceinline__ void next(int n) { left -= n; ++g; f = 0; }
};

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

// CG groups of KS waves share a work-group's fragments (kSiluF32: fragments of the gate half, each with its up fragment),
// D in flight.
template <int GPW, int KS, int CG, int D, Src8 SRC, Out8 DST>
__global__ void __launch_bounds__(64 * KS * CG, KS * CG <= 4 ? 2 : 1) int8_rows_kernel(RowsParams p) {
    constexpr bool kSilu = DST == Out8::kSiluF32;
    constexpr int kPair = kSilu ? 2 : 1;                         // fragments of one output fragment
    static_assert(D % kPair == 0, "an output fragment's parts are in flight together");
    constexpr int kUnits = D / kPair;                            // output fragments of one round
    constexpr int kWaves = KS * CG;
    __shared__ __attribute__((aligned(16))) v4i part[KS > 1 ? 2 : 1][KS > 1 ? CG : 1][KS > 1 ? D : 1][KS > 1 ? KS : 1][64];
    __shared__ Routed rt;
    // sixteen quantised rows (16 bytes apart beside their values: sixteen lanes then read different banks) and their scales
    constexpr bool kQuant = SRC != Src8::kI8;
    constexpr int kRowK = GPW * KS * kStep + 16;
    __shared__ __attribute__((aligned(16))) int8_t s_x[kQuant ? 16 * kRowK : 16];
    __shared__ uint32_t s_top[kQuant ? 16 : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = wave % KS, cg = wave / KS;
    const int q = lane >> 4, c = lane & 15;
    const int half = p.N / 2;
    const int cols = kSilu ? half : p.N;
    const int K = p.K, G = (K + kStep - 1) / kStep;
    const int frags = (cols + 15) / 16;
    const int g0 = ks * GPW;                                     // first step of this wave

    // ---- what these KS waves take of a group: `per` output fragments from f0 on ----
    struct Part {
        const int8_t* w;
        const float* ws;
        int f0, per;
    };
    auto part_of = [&](int e, int f, int here) __attribute__((always_inline)) {
        const int per = (here + CG - 1) / CG;
        return Part{p.w + (int64_t)e * p.N * K, p.ws + (int64_t)e * p.N, f + cg * per, per};
    };
    // weights: step i is fragment f0 + i / kPair of the gate (i even) or the up half; on: 0 for a load of no use, of one
    // address
    struct Stage {
        u32x4 w[GPW][2];
    };
    auto load = [&](Stage& s, const Part& a, int i, int on) __attribute__((always_inline)) {
        const int f = min(a.f0 + min(i / kPair, a.per - 1), frags - 1);
        const int up = kSilu && (i & 1) ? half : 0;
        // (columns past the end read the last one; never stored)
        const int8_t* wr = a.w + (int64_t)((up + min(f * 16 + c, cols - 1)) & on) * K;
#pragma unroll
        for (int j = 0; j < GPW; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = min(min(g0 + j, G - 1) * kStep + h * 64 + q * 16, K - 16);
                s.w[j][h] = *reinterpret_cast<const u32x4*>(wr + (k & on));
            }
    };
    // Scales of the columns that a wave stores in a round (unit u of it: output fragment f0 + it kUnits + u). Loads return
    // in order: those of the layer are loaded before the round's weights, so that nothing waits for later ones.
    constexpr int kMine = KS == 1 ? kUnits : 1;
    static_assert(KS == 1 || kUnits <= KS, "a wave a unit");
    constexpr bool kEarly = DST != Out8::k16;                    // (whole fragments)
    using v4f1 = float __attribute__((ext_vector_type(4), aligned(4)));
    struct Cols {
        v4f ws[kMine], up[kSilu ? kMine : 1];
    };
    auto load_cols = [&](Cols& t, const Part& a, int it) __attribute__((always_inline)) {
        if constexpr (kEarly)
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int n = min((a.f0 + it * kUnits + (KS == 1 ? i : ks)) * 16, cols - 16) + 4 * q;
                t.ws[i] = *reinterpret_cast<const v4f1*>(a.ws + n);
                if constexpr (kSilu) t.up[i] = *reinterpret_cast<const v4f1*>(a.ws + half + n);
            }
    };

    Stage ring[D];
    Cols now;
    bool again = false, ahead = false;                           // ahead: the first weights of this part are in flight
    Walk walk(find_groups<kWaves>(p, rt), frags);
    for (; walk.left > 0; walk.next(walk.here(frags))) {
        const Group gr = group_at(p, rt, walk.g);
        if (gr.n == 0) {
            ahead = false;
            continue;
        }
        const int here = walk.here(frags);
        const Part cur = part_of(gr.e, walk.f, here);
        const int mine = min(cur.per, walk.f + here - cur.f0);   // real fragments (may be <= 0)
        const int rounds = (cur.per * kPair + D - 1) / D;        // of the work-group: the barriers agree
        Part nxt = cur;                                          // what follows
        bool follows = false;
        if (walk.left > here) {
            const Group gn = group_at(p, rt, walk.g + 1);
            follows = gn.n > 0;
            if (follows) nxt = part_of(gn.e, 0, min(walk.left - here, frags));
        }
        // ---- sixteen rows, held ----
        const int slot = c < gr.n ? slot_at(rt, gr, c) : -1;
        const int row = slot < 0 ? slot_at(rt, gr, 0) : slot;    // (a row that exists; never stored)
        const int xrow = p.gather ? row / p.top_k : row;
        u32x4 x[GPW][2];
        float xs;
        auto first_weights = [&]() __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
            load_cols(now, cur, 0);
#pragma unroll
            for (int d = 0; d < D; ++d) load(ring[d], cur, d, -1);
            __builtin_amdgcn_sched_barrier(0);
        };
        if constexpr (!kQuant) {
            auto read = [&]() __attribute__((always_inline)) {
                const int8_t* xp = reinterpret_cast<const int8_t*>(p.x) + (int64_t)xrow * p.ldx;
                xs = p.xs[xrow];
#pragma unroll
                for (int j = 0; j < GPW; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        x[j][h] = *reinterpret_cast<const u32x4*>(xp + min(min(g0 + j, G - 1) * kStep + h * 64 + q * 16, K - 16));
            };
            read();
            if (!ahead) first_weights();
        } else {
            // The work-group quantises its real rows, eight values a thread and turn, into LDS, kHold turns' loads
            // together. The first turns' values stay in registers between the maximum and the rounding; they are loaded
            // before the weights, as loads return in order.
            constexpr int kHold = 4, kThreads = 64 * kWaves;
            const int pieces = K / 8, items = gr.n * pieces;
            const bool whole = pieces % 64 == 0;                 // a wave's pieces are of one row
            const float each = 1.0f / (float)pieces;
            Raw8<SRC> raw[kHold];
            int rr[kHold], rk[kHold];
            auto read = [&](int first) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < kHold; ++i) {
                    const int item = min(first + i * kThreads, items - 1);
                    rr[i] = (int)(((float)item + 0.5f) * each);  // (item / pieces: both below 2^13)
                    rk[i] = (item - rr[i] * pieces) * 8;
                    const int s = slot_at(rt, gr, rr[i]);
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
            if (again) lds_barrier();                            // (the last group's rows have been read)
            if (tid < 16) s_top[tid] = 0;
            read(tid);
            // (the maxima twice: each side then waits for as many loads as it has behind them)
            if (!ahead) {
                first_weights();
                lds_barrier();
                maxima(tid);
            } else {
                lds_barrier();
                maxima(tid);
            }
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
            const bool end = it + 1 == rounds;                   // behind the last round: the first of what follows
            const Part to{end ? nxt.w : cur.w, end ? nxt.ws : cur.ws, end ? nxt.f0 : cur.f0, end ? nxt.per : cur.per};
            const int first = end ? 0 : (it + 1) * D, on = !end || follows ? -1 : 0;
            v4i run[D];
            Cols next_cols;
            load_cols(next_cols, to, end ? 0 : it + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < D; ++d) {
                run[d] = v4i{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < GPW; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) run[d] = mfma_i8(ring[d].w[j][h], x[j][h], run[d]);
                __builtin_amdgcn_sched_barrier(0);
                load(ring[d], to, first + d, on);
                __builtin_amdgcn_sched_barrier(0);
            }
            // unit u of the round: an output fragment
            auto put = [&](int u, int i, const v4i& a, const v4i& b) __attribute__((always_inline)) {
                const int of = it * kUnits + u;
                const int col = (cur.f0 + of) * 16 + 4 * q;
                if (of >= mine || slot < 0 || col >= cols) return;
                v4f t;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (kSilu) {
                        t[r] = silu_mul((float)a[r] * (xs * now.ws[i][r]), (float)b[r] * (xs * now.up[i][r]));
                    } else if constexpr (DST == Out8::k16) {
                        const int n = min(col + r, cols - 1);
                        t[r] = fmaf((float)a[r], xs * cur.ws[n], bias_at(p, n));
                    } else {
                        t[r] = (float)a[r] * (xs * now.ws[i][r]);
                    }
                }
                if constexpr (DST == Out8::k16) store16(p, slot, col, t);
                else *reinterpret_cast<v4f*>(reinterpret_cast<float*>(p.out) + (int64_t)slot * p.ldo + col) = t;
            };
            if constexpr (KS == 1) {
#pragma unroll
                for (int u = 0; u < kUnits; ++u) put(u, u, run[u * kPair], run[u * kPair + kPair - 1]);
            } else {
                auto& buf = part[it & 1][cg];
#pragma unroll
                for (int d = 0; d < D; ++d) buf[d][ks][lane] = run[d];
                lds_barrier();
                // (the next round writes the other buffer; this one is written again behind its barrier)
                if (ks < kUnits) {
                    auto total = [&](int d) __attribute__((always_inline)) {
                        v4i t = buf[d][0][lane];
#pragma unroll
                        for (int w = 1; w < KS; ++w) t += buf[d][w][lane];
                        return t;
                    };
                    const v4i t = total(ks * kPair);
                    if constexpr (kSilu) put(ks, 0, t, total(ks * kPair + 1));
                    else put(ks, 0, t, t);
                }
            }
            now = next_cols;
        }
        if (KS > 1) lds_barrier();                               // (an odd number of rounds: the first buffer is read)
        again = true;
        ahead = follows;
    }
}

// Any K, int8 rows: KS waves take the steps of K in turn (what they read at one time is contiguous along K).
// Steps of a wave in flight. 8 tokens, 2 picks, half of them among 8 experts of 8192 x 2048: 66 us (two: 61, four: 73); 40
// tokens, 8 picks, 64 experts of 7168 x 2048: 684 us, 4.1 TB/s (632, 737).
constexpr int kRing = 3;
template <int FN, int KS, Out8 DST>
__global__ void __launch_bounds__(64 * KS) int8_stream_kernel(RowsParams p) {
    constexpr bool kSilu = DST == Out8::kSiluF32;
    constexpr int kCols = kSilu ? FN / 2 : FN;                   // column fragments of the output
    __shared__ __attribute__((aligned(16))) v4i part[KS][FN][64];
    __shared__ Routed rt;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane >> 4, c = lane & 15;
    const int half = p.N / 2;
    const int cols = kSilu ? half : p.N;
    const int K = p.K;
    const int G = (K + kStep - 1) / kStep, steps = (G + KS - 1) / KS;
    const int frags = (cols + kCols * 16 - 1) / (kCols * 16);    // of kCols column fragments
    bool again = false;
    Walk walk(find_groups<KS>(p, rt), frags);
    for (; walk.left > 0; --walk.left, walk.f + 1 < frags ? ++walk.f : (++walk.g, walk.f = 0)) {
        const Group gr = group_at(p, rt, walk.g);
        if (gr.n == 0) continue;
        const int8_t* wp[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int f = (walk.f * kCols + j % kCols) * 16, up = kSilu && j >= kCols ? half : 0;
            wp[j] = p.w + ((int64_t)gr.e * p.N + up + min(f + c, cols - 1)) * K;
        }
        const float* ws = p.ws + (int64_t)gr.e * p.N;
        const int slot = c < gr.n ? slot_at(rt, gr, c) : -1;
        const int row = slot < 0 ? slot_at(rt, gr, 0) : slot;
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
        if (again) __syncthreads();                              // (the last sums have been read)
        again = true;
#pragma unroll
        for (int j = 0; j < FN; ++j) part[wave][j][lane] = run[j];
        __syncthreads();
        // wave j joins column fragment j (four adjacent columns of a row a lane)
        static_assert(kCols <= KS, "a wave a fragment");
        const int col = (walk.f * kCols + wave) * 16 + 4 * q;
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
// rows.
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
int64_t groups_of(const RowsParams& p) {
    return p.ids == nullptr ? ((int64_t)p.rows + 15) / 16 : std::min(p.slots, p.E + p.slots / 16);
}
template <int FN, int KS, Out8 DST>
int stream_go(const RowsParams& p, hipStream_t s) {
    constexpr bool silu = DST == Out8::kSiluF32;
    const int cols = silu ? p.N / 2 : p.N, per = 16 * (silu ? FN / 2 : FN);
    // (two work-groups a CU run at once; several rounds of them even out their ends)
    const int64_t units = groups_of(p) * ((cols + per - 1) / per), grid = std::min<int64_t>(units, (int64_t)device_cu_count() * 16);
    if (units >= (int64_t)1 << 31) return too_many();
    launch_kernel(&int8_stream_kernel<FN, KS, DST>, dim3((unsigned)grid), dim3(64 * KS), 0, s, p);
    return check_launch("int8_stream_kernel");
}

// per: output fragments that KS waves walk over. The kernel loads D fragments beforehand whatever `per` is, so few of
// them take a variant with a smaller D.
template <int GPW, int KS, int CG, int D, Src8 SRC, Out8 DST>
int rows_launch(const RowsParams& p, int64_t grid, int64_t per, hipStream_t s) {
    constexpr int pair = DST == Out8::kSiluF32 ? 2 : 1;
    if constexpr (D > pair)
        if (per * pair <= D / 2) return rows_launch<GPW, KS, CG, D / 2, SRC, DST>(p, grid, per, s);
    launch_kernel(&int8_rows_kernel<GPW, KS, CG, D, SRC, DST>, dim3((unsigned)grid), dim3(64 * KS * CG), 0, s, p);
    return check_launch("int8_rows_kernel");
}

template <int GPW, int KS, int CG, int D, Src8 SRC, Out8 DST>
int rows_go(const RowsParams& p, hipStream_t s) {
    const int64_t frags = ((DST == Out8::kSiluF32 ? p.N / 2 : p.N) + 15) / 16, units = groups_of(p) * frags;
    if (units >= (int64_t)1 << 31) return too_many();
    // As many work-groups as run at once (eight waves a CU).
    const int64_t resident = (int64_t)device_cu_count() * std::max(1, 8 / (KS * CG));
    const int64_t grid = std::min(resident, (units + CG - 1) / CG);
    return rows_launch<GPW, KS, CG, D, SRC, DST>(p, grid, (units + grid * CG - 1) / (grid * CG), s);
}

// The wave split by the number of steps: a wave holds the rows' values of up to four of them, up to eight waves share K.
// (Longer K by sixteen waves, or by twice the column fragments: 972 and 719 us for 684, 40 tokens, 8 picks, 64 experts of
// 7168 x 2048.)
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

// Hardly two slots of one expert, whose weights would be read twice: no count, and one launch less. us as ever / with it:
// 256 experts of 2048 x 512, 8 picks, 1 token 18.4 / 14.2, 4 tokens 30.4 / 25.9, 8 tokens 45.3 / 44.3; 64 experts of 4096 x
// 1024, 6 picks, 2 tokens 45.1 / 36.5.
bool few_slots(int64_t slots, int64_t E) { return slots * 4 <= E; }
bool int8_token_supported(int64_t slots, int64_t E, int64_t inter) { return few_slots(slots, E) && inter <= kTokenK; }

int launch_int8_token(const RowsArgs& a, const float* topk_weights, hipStream_t s) {
    const RowsParams p = rows_params(a);
    const int frags = (p.N + 15) / 16, tokens = p.slots / p.top_k;
    // one fragment a work-group while those run at once (four a CU), else two (us with one / two, 2048 x 512: 1 token 14.2 /
    // 17.0, 4 tokens 25.9 / 25.1)
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
    p.one_slot = few_slots(p.slots, p.E) ? 1 : 0;
    if (p.rows == 0 || (p.ids != nullptr && p.slots == 0)) return W4A8_OK;
    if (p.ids != nullptr && p.slots > kScanSlots) {
        set_error("int8 product: too many slots for the streaming kernels");
        return W4A8_ERR_INVALID;
    }
    // (h in int8 is of rows that are too long to be quantised in the kernel)
    if (a.dst == Out8::kSlotF32) return a.src == Src8::kI8 ? stream_go<1, 8, Out8::kSlotF32>(p, s) : rows_any<Src8::kF32, Out8::kSlotF32>(p, s);
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
