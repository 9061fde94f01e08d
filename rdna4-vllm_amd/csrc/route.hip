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
// One wave a token: lane l holds experts NV l .. NV l + NV - 1.
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

template <int NV, int SRC, bool BIAS>
__global__ void __launch_bounds__(256) route_topk_kernel(RouteParams p) {
    // what groups are compared by: c in fp64, or the logit
    __shared__ double s_c[BIAS ? 4 : 1][BIAS ? 64 * NV : 1];
    __shared__ float s_l[BIAS ? 1 : 4][BIAS ? 1 : 64 * NV];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = (int64_t)blockIdx.x * 4 + wave;
    if (t >= p.T) return;                       // (no work-group barrier below)
    const int E = p.E;
    float l[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) l[i] = logit_at<SRC>(p.logits, t * p.ldl + min(lane * NV + i, E - 1));
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        // +inf as the largest finite number, NaN as -inf
        l[i] = lane * NV + i < E && l[i] > -INFINITY ? fminf(l[i], 3.402823466e38f) : -INFINITY;
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
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            key[i] = l[i] > -INFINITY ? order_key(l[i]) : 0u;
            s += expf(l[i] - m);
        }
        sum = (double)wave_sum(s);
    }

    // ---- groups: lane g scores group g, and its rank says whether it stays ----
    if (p.groups > 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (BIAS) s_c[wave][lane * NV + i] = c[i];
            else s_l[wave][lane * NV + i] = l[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        double score = -INFINITY;
        if (lane < p.groups) {
            double second = -INFINITY;
            for (int i = 0; i < p.size; ++i) {
                double v;
                if constexpr (BIAS) v = s_c[wave][lane * p.size + i];
                else v = s_l[wave][lane * p.size + i];
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

template <int SRC, bool BIAS>
int route_go(const RouteParams& p, hipStream_t s) {
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
    const RouteParams p{a.logits, a.bias, a.tw, a.ids, a.T, a.ldl, (int)a.E, (int)a.top_k, (int)a.groups, (int)a.top_groups,
                        (int)(a.E / a.groups), a.sigmoid ? 1 : 0, a.renorm ? 1 : 0, a.scale};
    if (a.dtype == W4A8_DTYPE_F32) return a.bias ? route_go<0, true>(p, s) : route_go<0, false>(p, s);
    if (a.dtype == W4A8_DTYPE_F16) return a.bias ? route_go<1, true>(p, s) : route_go<1, false>(p, s);
    return a.bias ? route_go<2, true>(p, s) : route_go<2, false>(p, s);
}

}  // namespace w4a8
