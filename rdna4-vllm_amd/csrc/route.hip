// Choice of experts from a router's logits: softmax or sigmoid scores, a bias for balance, groups of experts, top-k,
// renormalised and scaled weights.
//
//   p = softmax(l) or 1 / (1 + e^-l);  c = p + bias
//   group score = the sum of its two largest c (with a bias), or its largest c; the best top_groups groups stay
//   the top_k largest c of those, ties to the lower expert;  w = p [/ sum of the picks' p] * scale
// Experts whose logit or c is -inf or NaN are never picked: a pick that finds none is expert -1 with weight 0.
//
// A choice is that of the true numbers: without a bias both scores grow with the logit, and logits are compared; with
// one, c is formed in fp64 (in fp32 two experts' c may round to one number), compared rounded to fp32 (which keeps the
// order) and, where that is equal, by what was rounded off.
//
// Bound: for many tokens the vector units (busy 0.79 of the time): 16384 tokens of 256 experts, 8 picks in 4 of 8 groups,
// sigmoid with a bias, take 11.5 to 14.0 us with the call (one token a wave: 39), where their logits' bytes take 4; for few
// the launch and the steps' latency, 4 to 6 us.
#include <type_traits>

#include "w4a8_common.h"
#include "w4a8_internal.h"

namespace w4a8 {
namespace {

struct RouteParams {
    const void* logits;
    const float* bias;
    float* tw;
    int32_t* ids;
    int64_t T, ldl;
    int E, top_k, groups, top_groups, size;    // size: experts of a group
    int sigmoid, renorm;
    float scale;
    int nv, vec, bias_vec;                     // sixteen lanes a token: experts a lane; whole pieces of 16 bytes each
};

__device__ __forceinline__ uint32_t order_key(float v) {       // larger for a larger value, 0 for none
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
struct UMax {
    __device__ float operator()(float a, float b) const {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    }
};
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    return __float_as_uint(lane_allreduce<6>(__uint_as_float(v), UMax{}));
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v = fmax(v, __shfl_xor(v, m));
    return v;
}

template <int SRC>                              // 0 fp32, 1 fp16, 2 bf16
__device__ __forceinline__ float logit_at(const void* l, int64_t i) {
    if constexpr (SRC == 0) return reinterpret_cast<const float*>(l)[i];
    const uint16_t v = reinterpret_cast<const uint16_t*>(l)[i];
    if constexpr (SRC == 2) return __uint_as_float((uint32_t)v << 16);
    return __half2float(__ushort_as_half(v));
}

// e^(a - b), a not above b, to about two roundings: what a - b and its product with log2(e) round off is put back.
__device__ __forceinline__ float exp_near(float a, float b) {
    const float x = a - b, y = x - a, off = (a - (x - y)) - (b + y);
    const float t = x * 1.44269504088896340736f;
    const float lo = fmaf(x, 1.44269504088896340736f, -t) + fmaf(off, 1.44269504088896340736f, x * 1.92596299112661746887e-8f);
    const float e = __builtin_amdgcn_exp2f(t);
    return t > -200.f ? fmaf(e * 0.69314718055994530942f, lo, e) : 0.f;
}

// What a wave compares groups by, in LDS: c in fp64, or the logit.
template <int NV, bool BIAS>
struct RouteScratch {
    double c[BIAS ? 64 * NV : 1];
    float l[BIAS ? 1 : 64 * NV];
};

// One token by one wave: lane l holds experts NV l .. NV l + NV - 1.
template <int NV, int SRC, bool BIAS>
__device__ void route_token(const RouteParams& p, int64_t t, int lane, RouteScratch<NV, BIAS>& scratch) {
    const int E = p.E;
    float l[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) l[i] = logit_at<SRC>(p.logits, t * p.ldl + min(lane * NV + i, E - 1));
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        // +inf as the largest finite number, NaN as -inf, -0 as 0
        l[i] = lane * NV + i < E && l[i] > -INFINITY ? fminf(l[i], 3.402823466e38f) + 0.f : -INFINITY;
        m = fmaxf(m, l[i]);
    }
    m = wave_max(m);
    if (m == -INFINITY) m = 0.f;

    // ---- scores ----
    double c[BIAS ? NV : 1], sum = 0.0;
    uint32_t key[NV];
    if constexpr (BIAS) {
        double v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const double x = (double)l[i] - (p.sigmoid ? 0.0 : (double)m);
            v[i] = p.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x);
            sum += v[i];
        }
        if (!p.sigmoid) sum = wave_sum64(sum);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const double b = (double)p.bias[min(lane * NV + i, E - 1)];
            c[i] = (p.sigmoid ? v[i] : v[i] / sum) + b;
            if (l[i] == -INFINITY || !(c[i] > -INFINITY)) c[i] = -INFINITY;
            key[i] = c[i] > -INFINITY ? order_key((float)c[i]) : 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            key[i] = l[i] > -INFINITY ? order_key(l[i]) : 0u;
            sum += (double)exp_near(l[i], m);
        }
        sum = wave_sum64(sum);
    }

    // ---- groups: lane g scores group g, and its rank says whether it stays ----
    if (p.groups > 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (BIAS) scratch.c[lane * NV + i] = c[i];
            else scratch.l[lane * NV + i] = l[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        double score = -INFINITY;
        if (lane < p.groups) {
            double second = -INFINITY;
            for (int i = 0; i < p.size; ++i) {
                double v;
                if constexpr (BIAS) v = scratch.c[lane * p.size + i];
                else v = scratch.l[lane * p.size + i];
                second = fmax(second, fmin(v, score));
                score = fmax(score, v);
            }
            if (BIAS && second > -INFINITY) score += second;
        }
        int rank = 0;
        for (int g = 0; g < p.groups; ++g) {
            const double other = __shfl(score, g);
            rank += other > score || (other == score && g < lane) ? 1 : 0;
        }
        const uint64_t kept = __ballot(lane < p.groups && rank < p.top_groups);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int g = min((lane * NV + i) / p.size, 63);
            if (!(kept >> g & 1)) key[i] = 0u;
        }
    }

    // ---- picks: lane j gets pick j ----
    int mine = -1;
    float mine_l = -INFINITY;
    for (int j = 0; j < p.top_k; ++j) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) best = max(best, key[i]);
        best = wave_umax(best);
        if (best == 0u) break;
        // among equal keys: the largest remainder, then the lowest expert (its lane first)
        double far = -INFINITY;
        if constexpr (BIAS) {
            int holders = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) holders += __popcll(__ballot(key[i] == best));
            if (holders > 1) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (key[i] == best) far = fmax(far, c[i]);
                far = wave_max64(far);
            }
        }
        int at = NV;
        float al = 0.f;
#pragma unroll
        for (int i = NV - 1; i >= 0; --i) {
            bool is = key[i] == best;
            if constexpr (BIAS) is = is && (far == -INFINITY || c[i] == far);
            at = is ? i : at;
            al = is ? l[i] : al;
        }
        const int owner = __builtin_ctzll(__ballot(at < NV));
        const int pick_at = __builtin_amdgcn_readlane(at, owner);
        const float pick_l = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(al), owner));
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane == owner && i == pick_at) key[i] = 0u;
        mine = lane == j ? owner * NV + pick_at : mine;
        mine_l = lane == j ? pick_l : mine_l;
    }

    // ---- weights, in fp64: a renormalised weight is right where p itself is too small for fp32 ----
    double w = 0.0;
    if (mine >= 0) w = p.sigmoid ? 1.0 / (1.0 + exp(-(double)mine_l)) : exp((double)mine_l - (double)m);
    if (p.renorm) {
        const double total = wave_sum64(w);
        w = total > 0.0 ? w / total : 0.0;
    } else if (!p.sigmoid && mine >= 0) {
        w /= sum;
    }
    if (lane < p.top_k) {
        p.tw[t * p.top_k + lane] = (float)(w * (double)p.scale);
        p.ids[t * p.top_k + lane] = mine;
    }
}

template <int NV, int SRC, bool BIAS>
__global__ void __launch_bounds__(256) route_topk_kernel(RouteParams p) {
    __shared__ RouteScratch<NV, BIAS> scratch[4];
    const int wave = threadIdx.x >> 6;
    const int64_t t = (int64_t)blockIdx.x * 4 + wave;
    if (t >= p.T) return;                       // (no work-group barrier below)
    route_token<NV, SRC, BIAS>(p, t, threadIdx.x & 63, scratch[wave]);
}

// ---- four tokens a wave ----
// Sixteen lanes a token, lane s holds experts nv s .. nv s + nv - 1 (at most 256 in all), picks up to 8. An expert's key
// is its score in 24 bits over 255 - expert, so that one unsigned maximum finds score and expert: of 16-bit logits
// without a bias the logit's own bits in their order (exact); else c in fp32, as a part of its range. Picks whose keys lie
// nearer to each other, or to one that was not picked, than all roundings together may be off are put in order by their c
// in fp64 (about one token in 1500, by sigmoids with a bias); where groups, several others or a softmax's sum are in doubt
// (with a bias one token in 400 to 700), the whole wave takes the token again by route_token. Weights are formed in fp64 by
// both: in fp32 a token had other last bits by the one than by the other (65536 tokens, sigmoid, bias: 36.5 us for 35.4).
constexpr int kTop = 8;

__device__ __forceinline__ void order2(uint32_t& a, uint32_t& b) {
    const uint32_t m = max(a, b);
    b = min(a, b);
    a = m;
}
__device__ __forceinline__ void sort8(uint32_t (&v)[8]) {        // descending, odd-even merges
    order2(v[0], v[1]); order2(v[2], v[3]); order2(v[4], v[5]); order2(v[6], v[7]);
    order2(v[0], v[2]); order2(v[1], v[3]); order2(v[4], v[6]); order2(v[5], v[7]);
    order2(v[1], v[2]); order2(v[5], v[6]);
    order2(v[0], v[4]); order2(v[1], v[5]); order2(v[2], v[6]); order2(v[3], v[7]);
    order2(v[2], v[4]); order2(v[3], v[5]);
    order2(v[1], v[2]); order2(v[3], v[4]); order2(v[5], v[6]);
}
__device__ __forceinline__ void merge8(uint32_t (&v)[8]) {       // a bitonic sequence, descending
    order2(v[0], v[4]); order2(v[1], v[5]); order2(v[2], v[6]); order2(v[3], v[7]);
    order2(v[0], v[2]); order2(v[1], v[3]); order2(v[4], v[6]); order2(v[5], v[7]);
    order2(v[0], v[1]); order2(v[2], v[3]); order2(v[4], v[5]); order2(v[6], v[7]);
}
// The 8 largest of two lanes' lists, in both lanes.
template <int S>
__device__ __forceinline__ void join8(uint32_t (&v)[8]) {
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = max(v[i], dpp_step<S>(v[7 - i]));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = o[i];
    merge8(v);
}
__device__ __forceinline__ float row_max(float v) { return lane_allreduce<4>(v, MaxOp{}); }
template <int S>
__device__ __forceinline__ double row_add64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return v + __builtin_bit_cast(double, (uint64_t)dpp_step<S>((uint32_t)(b >> 32)) << 32 | dpp_step<S>((uint32_t)b));
}
__device__ __forceinline__ double row_sum64(double v) { return row_add64<3>(row_add64<2>(row_add64<1>(row_add64<0>(v)))); }
struct AddU {
    __device__ float operator()(float a, float b) const { return __uint_as_float(__float_as_uint(a) + __float_as_uint(b)); }
};
__device__ __forceinline__ uint32_t row_count(uint32_t v) { return __float_as_uint(lane_allreduce<4>(__uint_as_float(v), AddU{})); }
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }
template <int R>
__device__ __forceinline__ int larger_in_row(uint32_t v) {       // lanes of the row of sixteen that hold more than v
    if constexpr (R == 0) return 0;
    else return ((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x120 + R, 0xF, 0xF, true) > v ? 1 : 0) + larger_in_row<R - 1>(v);
}

template <int NV, int SRC, bool BIAS>
__global__ void __launch_bounds__(256) route_rows_kernel(RouteParams p) {
    constexpr bool EXACT = !BIAS && SRC != 0;
    __shared__ RouteScratch<4, BIAS> scratch[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane >> 4, sub = lane & 15;
    const int64_t t0 = ((int64_t)blockIdx.x * 4 + wave) * 4;
    if (t0 >= p.T) return;                      // (no work-group barrier below)
    const int64_t t = min(t0 + row, p.T - 1), at = t * p.ldl;
    const int nv = p.nv, e0 = sub * nv, E = p.E;

    // ---- logits ----
    float l[NV];
    uint32_t bits[NV];                          // EXACT: the logit's own, in their order
    auto one = [&](int i, uint32_t raw) __attribute__((always_inline)) {
        const bool in = i < nv && e0 + i < E;
        if constexpr (SRC == 0) l[i] = __uint_as_float(raw);
        else if constexpr (SRC == 2) l[i] = __uint_as_float(raw << 16);
        else l[i] = __half2float(__ushort_as_half((uint16_t)raw));
        const bool live = in && l[i] > -INFINITY;
        if constexpr (EXACT) {
            const uint32_t b = raw == 0x8000u ? 0u : raw;
            bits[i] = live ? ((b & 0x8000u) ? ~b & 0xFFFFu : b | 0x8000u) : 0u;
        }
        l[i] = live ? fminf(l[i], 3.402823466e38f) : -INFINITY;
    };
    if (p.vec) {                                // a lane's logits are whole pieces of 16 bytes
        constexpr int per = SRC == 0 ? 4 : 8;
        u32x4 v[(NV + per - 1) / per];
#pragma unroll
        for (int i = 0; i < NV; i += per)
            v[i / per] = reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(p.logits) +
                                                        (at + min(e0 + i, E - per)) * (SRC == 0 ? 4 : 2))[0];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t w = v[i / per][SRC == 0 ? i % 4 : i % 8 / 2];
            one(i, SRC == 0 ? w : i % 2 ? w >> 16 : w & 0xFFFFu);
        }
    } else {
        uint32_t v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t a = at + min(e0 + min(i, nv - 1), E - 1);
            if constexpr (SRC == 0) v[i] = reinterpret_cast<const uint32_t*>(p.logits)[a];
            else v[i] = reinterpret_cast<const uint16_t*>(p.logits)[a];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) one(i, v[i]);
    }
    float m = l[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) m = fmaxf(m, l[i]);
    m = row_max(m);
    if (m == -INFINITY) m = 0.f;

    // ---- scores ----
    float c[NV];
    double sum = 1.0;
    if (!p.sigmoid && (BIAS || !p.renorm)) {
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            c[i] = exp_near(l[i], m);
            sum += (double)c[i];
        }
        sum = row_sum64(sum);
    }
    if constexpr (BIAS) {
        const float inv = 1.0f / (float)sum;
        float b[NV];
        if (nv % 4 == 0 && p.bias_vec) {
#pragma unroll
            for (int i = 0; i < NV; i += 4) {
                const v4f v = *reinterpret_cast<const v4f*>(p.bias + min(e0 + i, E - 4));
#pragma unroll
                for (int r = 0; r < 4; ++r) b[i + r] = v[r];
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) b[i] = p.bias[min(e0 + min(i, nv - 1), E - 1)];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const float s = p.sigmoid ? __builtin_amdgcn_rcpf(1.0f + exp_fast(-l[i])) : c[i] * inv;
            // (a NaN is -inf: left as it is, the smaller of it and a group's best were that best, a second time)
            c[i] = fmaxf(l[i] > -INFINITY ? s + b[i] : -INFINITY, -INFINITY);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) c[i] = l[i];
    }

    // With a bias c is off by no more than (slack + |c|) 2^-24. In units of 2^-24: a softmax's e^x and its sum are off by 3
    // each, the inverse and the product by 4 more: below 16 for p up to 1; a sigmoid, whose e^x is off by (2 |x| + 2) e^x, by
    // less than 8; the sum with b by half a step.
    const float slack = !BIAS ? 0.f : p.sigmoid ? 9.f : 17.f;

    // ---- groups: lanes of a group hold its score, and how many lanes hold a larger one ----
    bool sure = true;
    bool kept = true;
    float most = -INFINITY;                     // of the lane's scores
    if (p.groups > 1) {
        float first = -INFINITY, second = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            second = fmaxf(second, fminf(first, c[i]));
            first = fmaxf(first, c[i]);
        }
        most = first;
        auto join = [&](auto step) __attribute__((always_inline)) {
            constexpr int S = decltype(step)::value;
            const float f = __uint_as_float(dpp_step<S>(__float_as_uint(first)));
            const float s = __uint_as_float(dpp_step<S>(__float_as_uint(second)));
            second = fmaxf(fminf(first, f), fmaxf(second, s));
            first = fmaxf(first, f);
        };
        const int lanes = p.size / nv;          // of a group: 1, 2, 4, 8 or 16
        if (lanes > 1) join(std::integral_constant<int, 0>{});
        if (lanes > 2) join(std::integral_constant<int, 1>{});
        if (lanes > 4) join(std::integral_constant<int, 2>{});
        if (lanes > 8) join(std::integral_constant<int, 3>{});
        const bool two = BIAS && second > -INFINITY;
        const float score = first + (two ? second : 0.f);
        uint32_t group_key = order_key(score);
        if constexpr (EXACT) {                  // with the group's number: no two are equal
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) top = max(top, bits[i]);
            if (lanes > 1) top = max(top, dpp_step<0>(top));
            if (lanes > 2) top = max(top, dpp_step<1>(top));
            if (lanes > 4) top = max(top, dpp_step<2>(top));
            if (lanes > 8) top = max(top, dpp_step<3>(top));
            group_key = top << 8 | (uint32_t)(255 - e0 / p.size);
        }
        kept = larger_in_row<15>(group_key) < p.top_groups * lanes;
        // (equal groups at the border are kept together)
        sure = row_count(kept ? 1u : 0u) == (uint32_t)(p.top_groups * lanes);
        if constexpr (BIAS) {
            // two scores and their sum's rounding, and that of what follows
            const float size = fabsf(first) + (two ? fabsf(second) : 0.f);
            const float off = size < INFINITY ? (2.f * slack + 4.f * size) * 0x1p-24f : 0.f;
            const float least = -row_max(kept ? off - score : -INFINITY), out = row_max(kept ? -INFINITY : score + off);
            sure = sure && (out == -INFINITY || least > out);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) most = fmaxf(most, c[i]);
    }

    // ---- keys ----
    uint32_t key[NV], tol = 0;
    if constexpr (EXACT) {
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = kept ? bits[i] << 8 | (uint32_t)(255 - e0 - i) : 0u;
    } else {
        // Scores are taken between the row's largest, hi, and a little below the top_k-th largest of its lanes' largest,
        // which no pick lies below: experts masked by a low number, or far above the others, then leave the others their
        // bits (taken between the row's largest and smallest, tokens with such a mask all went through route_token: 85 us
        // for 24, 65536 tokens of 256 experts). Few lanes, or equal ones: down to the smallest score that is no such mask.
        // The mapping grows with c, so that only what c is off by, and the cut to whole numbers, can hide an order. What c
        // is off by is that of numbers up to three times the range's; of a c far below it is less than its distance.
        if (!kept) most = -INFINITY;
        const float hi = row_max(most);
        float lo = -row_max(larger_in_row<15>(order_key(most)) < max(p.top_k, 2) ? -most : -INFINITY);
        float off = BIAS ? (slack + 3.f * fmaxf(fabsf(lo), fabsf(hi))) * 0x1p-24f : 0.f;
        const bool few = !(lo > -1e30f) || (!BIAS && lo == hi);
        lo -= fmaxf(0.125f * (hi - lo), 16.f * off);
        if (__ballot(few) != 0) {
            float least = INFINITY;
#pragma unroll
            for (int i = 0; i < NV; ++i) least = fminf(least, kept && c[i] > -1e30f ? c[i] : INFINITY);
            least = -row_max(-least);
            if (few) {
                lo = least;
                off = BIAS ? (slack + 3.f * fmaxf(fabsf(lo), fabsf(hi))) * 0x1p-24f : 0.f;
            }
        }
        const float span = hi - lo;
        const bool some = span < 1e30f && span > 1e-30f;
        sure = sure && (some || hi == -INFINITY);
        const float f = some && kept ? 16777000.f / span : 0.f, o = some && kept ? 2.f : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)            // (-inf, and its product with 0, become 0, as what lies below the range)
            key[i] = (uint32_t)__builtin_amdgcn_fmed3f(fmaf(c[i] - lo, f, o), 0.f, 16777215.f) << 8 | (uint32_t)(255 - e0 - i);
        tol = 4u + (uint32_t)fminf(2.f * off * (16777000.f / span), 16777216.f);
    }

    // ---- the eight largest keys of the row, in all its lanes ----
    uint32_t best[kTop];
#pragma unroll
    for (int i = 0; i < kTop; ++i) best[i] = i < NV ? key[i < NV ? i : 0] : 0u;
    if constexpr (NV > 1) sort8(best);
    if constexpr (NV > kTop) {
        uint32_t more[kTop];
#pragma unroll
        for (int i = 0; i < kTop; ++i) more[i] = key[i + kTop < NV ? i + kTop : 0];
        sort8(more);
#pragma unroll
        for (int i = 0; i < kTop; ++i) best[i] = max(best[i], more[kTop - 1 - i]);
        merge8(best);
    }
    join8<0>(best);
    join8<1>(best);
    join8<2>(best);
    join8<3>(best);
    // lane j: pick j (a key below 256 is no expert)
    uint32_t mine = 0, last = 0;
    bool doubt = false;
#pragma unroll
    for (int i = 0; i < kTop; ++i) {
        mine = sub == i && i < p.top_k ? best[i] : mine;
        if (i + 1 == p.top_k) last = best[i];
        // picks in doubt among themselves
        if (!EXACT && i + 1 < kTop && i + 1 < p.top_k)
            doubt = doubt || (best[i + 1] > 255u && (best[i] >> 8) - (best[i + 1] >> 8) <= tol);
    }
    if constexpr (!EXACT) {
        // the last of them with others that were not picked: one of those is taken along
        const uint32_t from = last > 255u ? ((last >> 8) > tol ? (last >> 8) - tol : 1u) << 8 : ~0u;
        uint32_t near = 0, next = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            near += key[i] >= from ? 1u : 0u;
            next = max(next, key[i] < last ? key[i] : 0u);
        }
        near = row_count(near);
        if (near > (uint32_t)p.top_k && last > 255u) {
            doubt = true;
            sure = sure && near == (uint32_t)p.top_k + 1;
        }
        // next to the range's end, or no pick: what lies below it may be one
        const bool low = (last >> 8) <= tol;
        if (__ballot(low) != 0) {
            bool cut = false;
#pragma unroll
            for (int i = 0; i < NV; ++i) cut = cut || (kept && c[i] > -INFINITY && key[i] < 256u);
            cut = row_count(cut ? 1u : 0u) != 0u;
            sure = sure && !(low && cut);
        }
        if (__ballot(doubt) != 0) {
            next = __float_as_uint(lane_allreduce<4>(__uint_as_float(next), UMax{}));
            if (doubt && near > (uint32_t)p.top_k && sub == p.top_k) mine = next;
        }
    }
    mine = mine > 255u ? mine : 0u;

    // ---- weights, in fp64 as route_token's ----
    const int e = 255 - (int)(mine & 255u);
    float x = -INFINITY;
    double w = 0.0;
    if (mine != 0u) {
        x = fminf(logit_at<SRC>(p.logits, at + e), 3.402823466e38f);
        w = exp(p.sigmoid ? -(double)x : (double)x - (double)m);
        if (p.sigmoid) w = 1.0 / (1.0 + w);
    }
    int place = sub;
    if (!EXACT && __ballot(doubt) != 0) {
        // In doubt: sigmoids with a bias, and logits, are compared in fp64 among the row's lanes; a softmax with a bias
        // needs its sum in fp64 too.
        if (BIAS && !p.sigmoid) sure = sure && !doubt;
        double d = -INFINITY;
        if (mine != 0u) d = !BIAS ? (double)x : w + (double)p.bias[e];
        int rank = 0;
        for (int j = 0; j <= kTop; ++j) {
            const double other = __shfl(d, row * 16 + j);
            const int oe = __shfl(e, row * 16 + j);
            rank += other > d || (other == d && oe < e) ? 1 : 0;
        }
        if (doubt) {
            place = mine != 0u ? rank : sub;
            if (place >= p.top_k) {
                mine = 0u;
                w = 0.0;
            }
        }
    }
    if (p.renorm) {
        const double total = row_sum64(w);
        w = total > 0.0 ? w / total : 0.0;
    } else if (!p.sigmoid && mine != 0u) {
        w /= sum;
    }
    if (sure && t0 + row < p.T && place < p.top_k) {
        p.tw[t * p.top_k + place] = (float)(w * (double)p.scale);
        p.ids[t * p.top_k + place] = mine != 0u ? e : -1;
    }
    const uint64_t again = __ballot(!sure);
    if (again == 0) return;
    for (int r = 0; r < 4; ++r)
        if ((again >> (16 * r) & 0xFFFF) != 0 && t0 + r < p.T) route_token<4, SRC, BIAS>(p, t0 + r, lane, scratch[wave]);
}

template <int SRC, bool BIAS>
int route_go(const RouteParams& p, hipStream_t s) {
    // Four tokens a wave: up to 256 experts and 8 picks, groups of whole lanes, a power of two of them.
    const int lanes = p.size / p.nv;
    if (p.E <= 256 && p.top_k <= kTop &&
        (p.groups == 1 || (p.E == 16 * p.nv && p.size % p.nv == 0 && (lanes & (lanes - 1)) == 0 && lanes <= 16))) {
        const dim3 grid((unsigned)((p.T + 15) / 16));
        if (p.nv <= 4) launch_kernel(&route_rows_kernel<4, SRC, BIAS>, grid, dim3(256), 0, s, p);
        else if (p.nv <= 8) launch_kernel(&route_rows_kernel<8, SRC, BIAS>, grid, dim3(256), 0, s, p);
        else launch_kernel(&route_rows_kernel<16, SRC, BIAS>, grid, dim3(256), 0, s, p);
        return check_launch("route_rows_kernel");
    }
    const dim3 grid((unsigned)((p.T + 3) / 4));
    if (p.E <= 64) launch_kernel(&route_topk_kernel<1, SRC, BIAS>, grid, dim3(256), 0, s, p);
    else if (p.E <= 128) launch_kernel(&route_topk_kernel<2, SRC, BIAS>, grid, dim3(256), 0, s, p);
    else if (p.E <= 256) launch_kernel(&route_topk_kernel<4, SRC, BIAS>, grid, dim3(256), 0, s, p);
    else if (p.E <= 512) launch_kernel(&route_topk_kernel<8, SRC, BIAS>, grid, dim3(256), 0, s, p);
    else launch_kernel(&route_topk_kernel<16, SRC, BIAS>, grid, dim3(256), 0, s, p);
    return check_launch("route_topk_kernel");
}

}  // namespace

int launch_route_topk(const RouteArgs& a, hipStream_t s) {
    const int nv = (int)((a.E + 15) / 16), size = a.dtype == W4A8_DTYPE_F32 ? 4 : 2;
    const bool vec = nv * size % 16 == 0 && a.E == 16 * nv && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 &&
                     (a.ldl * size % 16 == 0 || a.T == 1);
    const RouteParams p{a.logits, a.bias, a.tw, a.ids, a.T, a.ldl, (int)a.E, (int)a.top_k, (int)a.groups, (int)a.top_groups,
                        (int)(a.E / a.groups), a.sigmoid ? 1 : 0, a.renorm ? 1 : 0, a.scale, nv, vec ? 1 : 0, a.E % 4 == 0 && reinterpret_cast<uintptr_t>(a.bias) % 16 == 0 ? 1 : 0};
    if (a.dtype == W4A8_DTYPE_F32) return a.bias ? route_go<0, true>(p, s) : route_go<0, false>(p, s);
    if (a.dtype == W4A8_DTYPE_F16) return a.bias ? route_go<1, true>(p, s) : route_go<1, false>(p, s);
    return a.bias ? route_go<2, true>(p, s) : route_go<2, false>(p, s);
}

}  // namespace w4a8
