// C ABI entry points of the block-scaled fp8 operators (include/w4a8_moe.h): argument checks,
// workspace carving, the choice of kernel and the whole-layer composition.
#include <algorithm>
#include <string>

#include "fp8_block.h"

namespace w4a8 {
namespace {

#define W4A8_REQUIRE(cond, msg)            \
    do {                                   \
        if (!(cond)) {                     \
            ::w4a8::set_error(msg);        \
            return W4A8_ERR_INVALID;       \
        }                                  \
    } while (0)

hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool is16(int dt) { return dt == W4A8_DTYPE_F16 || dt == W4A8_DTYPE_BF16; }

constexpr int64_t kMaxSide = (int64_t)1 << 24;    // rows of a weight, values of a row
constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 256;
constexpr int64_t kReduceRows = 65535;            // tokens of one slot reduce (its grid's second side)
// Dense rows up to which the weights are streamed: one row block (us, streamed / 64 x 64 tiles with K in two:
// 16 x 4096 x 4096 9.8 / 11.8, 16 x 2048 x 12288 18.7 / 25.9; two row blocks, 32 x 4096 x 4096, 15.2 / 12.0).
constexpr int64_t kStreamRows = 16;

// Sizes and pointers that every product shares.
int check_product(const void* x, int x_dtype, const float* xs, int64_t rows, int64_t K, int64_t ldx, const uint8_t* w,
                  const float* ws, int64_t E, int64_t N) {
    W4A8_REQUIRE(rows >= 0 && rows <= kMaxRows && K > 0 && N > 0 && E > 0, "fp8 block product: invalid sizes");
    W4A8_REQUIRE(K <= kMaxSide && N <= kMaxSide && E <= kMaxSide, "fp8 block product: a size is over 2^24");
    W4A8_REQUIRE(K % 16 == 0, "fp8 block product: K must be a multiple of 16");
    W4A8_REQUIRE(x_dtype == W4A8_DTYPE_E4M3 || is16(x_dtype), "fp8 block product: x must be e4m3, fp16 or bf16");
    if (rows == 0) return W4A8_OK;
    W4A8_REQUIRE(x && w && ws, "fp8 block product: null pointer");
    W4A8_REQUIRE(x_dtype != W4A8_DTYPE_E4M3 || xs, "fp8 block product: e4m3 rows need their scales");
    W4A8_REQUIRE(ldx >= K && ldx * (x_dtype == W4A8_DTYPE_E4M3 ? 1 : 2) % 16 == 0,
                 "fp8 block product: rows of x must start at multiples of 16 bytes");
    W4A8_REQUIRE(aligned16(x) && aligned16(w), "fp8 block product: x and w must be aligned to 16 bytes");
    return W4A8_OK;
}

Src src_of(int x_dtype) {
    return x_dtype == W4A8_DTYPE_E4M3 ? Src::kFp8 : x_dtype == W4A8_DTYPE_BF16 ? Src::kBf16 : Src::kF16;
}
Dst dst_of(int dt) { return dt == W4A8_DTYPE_BF16 ? Dst::kBf16 : Dst::kF16; }

// ---- the gated layer ----
// Few rows an expert: blocks of 16 rows on the streaming kernels (rows quantised in registers, h and
// the slots' rows in fp32). Else tiles: rows quantised beforehand, as bf16 numbers, h by gemm1, blocks of the 64
// rows that a tile's wave takes. The slots' rows are rounded before the sum only where that is lost in the output's
// own rounding: for bf16 output they are fp16 with scales (an eighth of its step: layer error 1.66e-3 -> 1.67e-3), for
// fp16 output fp32 (fp16 there adds as much error as the output's rounding does: 2.1e-4 -> 2.9e-4), which a layer of
// 4096 tokens x 8 (256 experts, 2048 x 512) pays with 466 us for 424.
struct LayerPlan {
    bool tiles;
    int64_t block_m, P, nblk;
};
LayerPlan plan_layer(int64_t T, int64_t H, int64_t inter, int64_t E, int64_t top_k) {
    LayerPlan pl;
    const int64_t lim = (int64_t)1 << 32;
    // us streamed / tiles: 256 experts (2048 x 512), 8 rows each 227 / 252, 12.5 rows 231 / 233; 32 experts, 8 rows
    // 52 / 48, 16 rows 62 / 48; 8 experts, 8 rows 23 / 43, 16 rows 37 / 43
    pl.tiles = T * top_k > 12 * E;
    pl.block_m = pl.tiles ? 64 : 16;
    pl.P = w4a8_moe_align_sorted_len(T * top_k, E, pl.block_m);
    if (pl.tiles && (2 * T * H >= lim || pl.P * inter >= lim || 2 * inter * H >= lim)) {
        pl.tiles = false;
        pl.block_m = 16;
        pl.P = w4a8_moe_align_sorted_len(T * top_k, E, pl.block_m);
    }
    // (every block in use holds a slot: few slots reach a small part of what the experts' padding allows)
    pl.P = std::min(pl.P, T * top_k * pl.block_m);
    pl.nblk = pl.P / pl.block_m;
    return pl;
}
struct LayerScratch {
    int32_t *sti, *eid, *ntp, *s2r;
    void* align_ws;
    size_t align_bytes;
    uint16_t* xq;
    uint8_t* hq;
    float *xs, *hs, *h, *y32, *ys;
    uint16_t* y16;
};
// bf16: of the output
template <typename WS>
void carve_layer(WS& w, const LayerPlan& pl, int64_t T, int64_t H, int64_t inter, int64_t E, int64_t top_k,
                 bool quantise, bool bf16, LayerScratch& m) {
    m = LayerScratch{};
    m.sti = w.template take<int32_t>((size_t)pl.P);
    m.eid = w.template take<int32_t>((size_t)pl.nblk);
    m.ntp = w.template take<int32_t>(1);
    m.align_bytes = align_workspace_bytes(T * top_k, E);
    m.align_ws = w.template take<uint8_t>(m.align_bytes);
    if (!pl.tiles) {
        m.h = w.template take<float>((size_t)(pl.P * inter));
        m.y32 = w.template take<float>((size_t)(T * top_k * H));
        return;
    }
    m.xq = w.template take<uint16_t>((size_t)(T * H));
    m.xs = w.template take<float>(quantise ? (size_t)(T * blk_groups(H)) : 0);
    m.hq = w.template take<uint8_t>((size_t)(pl.P * inter));
    m.hs = w.template take<float>((size_t)(pl.P * blk_groups(inter)));
    if (!bf16) {
        m.y32 = w.template take<float>((size_t)(T * top_k * H));
        return;
    }
    m.s2r = w.template take<int32_t>((size_t)(T * top_k));
    m.y16 = w.template take<uint16_t>((size_t)(pl.P * H));
    m.ys = w.template take<float>((size_t)(pl.P * (H / 32)));
}
struct SizeProbe {
    WorkspaceSize s;
    template <typename T>
    T* take(size_t n) { s.take<T>(n); return nullptr; }
};
// Bytes for either output type (the size that callers ask for does not name it).
size_t layer_bytes(const LayerPlan& pl, int64_t T, int64_t H, int64_t inter, int64_t E, int64_t top_k, bool quantise) {
    size_t most = 0;
    for (const bool bf16 : {false, true}) {
        SizeProbe p;
        LayerScratch m;
        carve_layer(p, pl, T, H, inter, E, top_k, quantise, bf16, m);
        most = std::max(most, p.s.used);
    }
    return most;
}

}  // namespace
}  // namespace w4a8

using namespace w4a8;

extern "C" {

int w4a8_rms_norm_quant_fp8(const void* x, int x_dtype, int64_t rows, int64_t H, int64_t x_stride,
                            const void* residual, int64_t residual_stride, const void* weight, int weight_is_f32,
                            float eps, int scale_per_row, void* residual_out, void* norm_out, uint8_t* q,
                            float* scales, void* stream) {
    clear_error();
    W4A8_REQUIRE(is16(x_dtype), "rms_norm_quant: x must be fp16 or bf16");
    W4A8_REQUIRE(rows >= 0 && rows <= kMaxRows && H > 0 && H <= kMaxSide, "rms_norm_quant: invalid sizes");
    if (rows == 0) return W4A8_OK;
    W4A8_REQUIRE(x && weight && q && scales, "rms_norm_quant: null pointer");
    W4A8_REQUIRE((residual == nullptr) == (residual_out == nullptr),
                 "rms_norm_quant: residual and residual_out go together");
    W4A8_REQUIRE((x_stride >= H || rows == 1) && (residual == nullptr || residual_stride >= H || rows == 1),
                 "rms_norm_quant: rows overlap");
    NormArgs a{x, residual, weight, x_dtype == W4A8_DTYPE_BF16, weight_is_f32 != 0, rows, H, x_stride, residual_stride,
               eps, scale_per_row != 0, residual_out, norm_out, q, scales};
    return launch_rms_norm_quant(a, as_stream(stream));
}

int w4a8_act_quant_fp8_block(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t x_stride, int silu_gate_up,
                             uint8_t* q, float* scales, void* stream) {
    clear_error();
    W4A8_REQUIRE(is16(x_dtype), "act_quant_fp8_block: x must be fp16 or bf16");
    W4A8_REQUIRE(rows >= 0 && rows <= kMaxRows && K > 0 && K <= kMaxSide, "act_quant_fp8_block: invalid sizes");
    if (rows == 0) return W4A8_OK;
    W4A8_REQUIRE(x && q && scales, "act_quant_fp8_block: null pointer");
    W4A8_REQUIRE(x_stride >= (silu_gate_up ? 2 * K : K) || rows == 1, "act_quant_fp8_block: rows overlap");
    return launch_act_quant_block(x, x_dtype == W4A8_DTYPE_BF16, rows, K, x_stride, silu_gate_up != 0, q, scales,
                                  as_stream(stream));
}

size_t w4a8_fp8_block_gemm_workspace_size(int x_dtype, int64_t M, int64_t K) {
    if (x_dtype == W4A8_DTYPE_E4M3 || M <= kStreamRows || K <= 0) return 0;
    WorkspaceSize s;
    s.take<uint8_t>((size_t)(M * K));
    s.take<float>((size_t)(M * blk_groups(K)));
    return s.used;
}

int w4a8_fp8_block_gemm(const void* x, int x_dtype, const float* x_scales, int64_t M, int64_t K, int64_t x_stride,
                        const uint8_t* w, const float* w_scales, int64_t N, void* out, int out_dtype, void* workspace,
                        size_t workspace_bytes, void* stream) {
    clear_error();
    if (int rc = check_product(x, x_dtype, x_scales, M, K, x_stride, w, w_scales, 1, N)) return rc;
    W4A8_REQUIRE(is16(out_dtype), "fp8_block_gemm: out must be fp16 or bf16");
    if (M == 0) return W4A8_OK;
    W4A8_REQUIRE(out, "fp8_block_gemm: null pointer");
    const bool quantise = x_dtype != W4A8_DTYPE_E4M3;
    BlockArgs a{};
    a.x = x; a.xs = x_scales; a.x_rows = M; a.K = K; a.ldx = x_stride;
    a.w = w; a.ws = w_scales; a.E = 1; a.N = N;
    a.P = M; a.top_k = 1; a.num_valid = M; a.block_m = 16; a.gather = false;
    a.src = src_of(x_dtype); a.dst = dst_of(out_dtype); a.out = out; a.ldo = N;
    if (M > kStreamRows && quantise) {
        Workspace w(workspace, workspace_bytes);
        uint8_t* xq = w.take<uint8_t>((size_t)(M * K));
        float* xs = w.take<float>((size_t)(M * blk_groups(K)));
        if (workspace == nullptr || !w.ok()) {
            set_error("fp8_block_gemm: workspace smaller than w4a8_fp8_block_gemm_workspace_size()");
            return W4A8_ERR_WORKSPACE;
        }
        if (int rc = launch_act_quant_block(x, x_dtype == W4A8_DTYPE_BF16, M, K, x_stride, false, xq, xs, as_stream(stream)))
            return rc;
        a.x = xq; a.xs = xs; a.ldx = K; a.src = Src::kFp8;
    }
    if (M > kStreamRows && block_tiles_supported(a)) return launch_block_tiles(a, as_stream(stream));
    return launch_block_stream(a, as_stream(stream));
}

int w4a8_moe_fp8_block_gemm(const void* x, const float* x_scales, int64_t x_rows, int64_t K, int64_t x_stride,
                            const uint8_t* w, const float* w_scales, int64_t E, int64_t N,
                            const int32_t* sorted_token_ids, int64_t P, const int32_t* expert_ids,
                            const int32_t* num_tokens_post_padded, int64_t num_slots, int64_t top_k, int64_t block_m,
                            int gather, void* out, int out_dtype, void* stream) {
    clear_error();
    if (int rc = check_product(x, W4A8_DTYPE_E4M3, x_scales, x_rows, K, x_stride, w, w_scales, E, N)) return rc;
    W4A8_REQUIRE(is16(out_dtype), "moe_fp8_block_gemm: out must be fp16 or bf16");
    W4A8_REQUIRE(P >= 0 && P <= kMaxRows && top_k > 0 && top_k <= kMaxSide && num_slots >= 0 && num_slots <= kMaxRows,
                 "moe_fp8_block_gemm: invalid sizes");
    W4A8_REQUIRE(block_m % 16 == 0 && block_m >= 16 && block_m <= 128,
                 "moe_fp8_block_gemm: block_m must be a multiple of 16 up to 128");
    W4A8_REQUIRE(P % block_m == 0, "moe_fp8_block_gemm: P not divisible by block_m");
    W4A8_REQUIRE(!gather || num_slots <= x_rows * top_k, "moe_fp8_block_gemm: more slots than x has rows for");
    if (P == 0 || x_rows == 0 || num_slots == 0) return W4A8_OK;
    W4A8_REQUIRE(sorted_token_ids && expert_ids && num_tokens_post_padded && out, "moe_fp8_block_gemm: null pointer");
    BlockArgs a{};
    a.x = x; a.xs = x_scales; a.x_rows = x_rows; a.K = K; a.ldx = x_stride;
    a.w = w; a.ws = w_scales; a.E = E; a.N = N;
    a.sorted_ids = sorted_token_ids; a.expert_ids = expert_ids; a.ntp = num_tokens_post_padded;
    a.P = P; a.top_k = top_k; a.num_valid = num_slots; a.block_m = block_m; a.gather = gather != 0;
    a.src = Src::kFp8; a.dst = dst_of(out_dtype); a.out = out; a.ldo = N;
    // Blocks of 16: tiles pass over several experts (256 x 8 rows of 2048 -> 1024: 105 us, streamed 101;
    // 16 rows an expert 137 / 135; 64 rows 110 / 222). Blocks of 64: streaming would find three of four row
    // fragments empty (0.75 rows an expert: 170 us, tiles 58).
    if ((block_m >= 64 || std::min(P, num_slots) > 32 * E) && block_tiles_supported(a)) return launch_block_tiles(a, as_stream(stream));
    return launch_block_stream(a, as_stream(stream));
}

size_t w4a8_moe_fp8_block_workspace_size(int64_t T, int64_t H, int64_t inter, int64_t E, int64_t top_k) {
    if (T <= 0 || H <= 0 || inter <= 0 || E <= 0 || top_k <= 0) return 0;
    return layer_bytes(plan_layer(T, H, inter, E, top_k), T, H, inter, E, top_k, true);
}

int w4a8_moe_fp8_block_apply(const void* x, int x_dtype, const float* x_scales, int64_t T, int64_t H, int64_t inter,
                             int64_t E, int64_t top_k, const uint8_t* w13, const float* w13_scales, const uint8_t* w2,
                             const float* w2_scales, const float* topk_weights, const int32_t* topk_ids,
                             const int32_t* expert_map, int64_t num_global_experts, void* out, int out_dtype,
                             void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    W4A8_REQUIRE(inter > 0 && inter % kBlk == 0 && H > 0 && H % kBlk == 0,
                 "moe_fp8_block_apply: hidden and intermediate sizes must be multiples of 128");
    W4A8_REQUIRE(top_k > 0 && top_k <= 1024, "moe_fp8_block_apply: invalid top_k");
    W4A8_REQUIRE(T >= 0 && T <= kMaxRows / top_k, "moe_fp8_block_apply: invalid sizes");
    if (int rc = check_product(x, x_dtype, x_scales, T, H, H, w13, w13_scales, E, 2 * inter)) return rc;
    W4A8_REQUIRE(is16(out_dtype), "moe_fp8_block_apply: out must be fp16 or bf16");
    const int64_t n_global = num_global_experts > 0 ? num_global_experts : E;
    W4A8_REQUIRE(expert_map != nullptr || n_global == E,
                 "moe_fp8_block_apply: global expert count differs from the local one; pass expert_map");
    W4A8_REQUIRE(E <= 1024 && n_global <= (int64_t)1 << 20, "moe_fp8_block_apply: too many experts");
    if (T == 0) return W4A8_OK;
    W4A8_REQUIRE(w2 && w2_scales && topk_weights && topk_ids && out, "moe_fp8_block_apply: null pointer");
    W4A8_REQUIRE(aligned16(w2) && aligned16(out), "moe_fp8_block_apply: w2 and out must be aligned to 16 bytes");
    const LayerPlan pl = plan_layer(T, H, inter, E, top_k);
    W4A8_REQUIRE(pl.P <= kMaxRows, "moe_fp8_block_apply: too many slots");
    const bool quantise = x_dtype != W4A8_DTYPE_E4M3, bf16 = out_dtype == W4A8_DTYPE_BF16;
    Workspace w(workspace, workspace_bytes);
    LayerScratch m;
    carve_layer(w, pl, T, H, inter, E, top_k, quantise, bf16, m);
    if (workspace == nullptr || !w.ok() || workspace_bytes < layer_bytes(pl, T, H, inter, E, top_k, quantise)) {
        set_error("moe_fp8_block_apply: workspace smaller than w4a8_moe_fp8_block_workspace_size()");
        return W4A8_ERR_WORKSPACE;
    }
    hipStream_t s = as_stream(stream);
    if (int rc = launch_align(topk_ids, T * top_k, E, pl.block_m, expert_map, n_global, m.sti, pl.P, m.eid, m.ntp,
                              m.align_ws, m.align_bytes, s, m.s2r))
        return rc;
    if (pl.tiles)
        if (int rc = quantise ? launch_act_quant_wide(x, x_dtype == W4A8_DTYPE_BF16, T, H, m.xq, m.xs, s)
                              : launch_widen_rows(x, T, H, m.xq, s))
            return rc;
    BlockArgs g1{};
    g1.x = pl.tiles ? m.xq : x;
    g1.xs = pl.tiles && quantise ? m.xs : x_scales;
    g1.x_rows = T; g1.K = H; g1.ldx = H;
    g1.w = w13; g1.ws = w13_scales; g1.E = E; g1.N = 2 * inter;
    g1.sorted_ids = m.sti; g1.expert_ids = m.eid; g1.ntp = m.ntp; g1.P = pl.P;
    g1.top_k = top_k; g1.num_valid = T * top_k; g1.block_m = pl.block_m; g1.gather = true; g1.all_rows = true;
    g1.src = pl.tiles ? Src::kWide : src_of(x_dtype);
    g1.dst = pl.tiles ? Dst::kSiluFp8 : Dst::kSiluF32;
    g1.out = pl.tiles ? (void*)m.hq : (void*)m.h; g1.out_scales = m.hs; g1.ldo = inter;
    BlockArgs g2 = g1;
    g2.x = pl.tiles ? (const void*)m.hq : (const void*)m.h; g2.xs = m.hs; g2.x_rows = pl.P; g2.K = inter; g2.ldx = inter;
    g2.w = w2; g2.ws = w2_scales; g2.N = H; g2.gather = false;
    const bool row16 = pl.tiles && bf16;
    g2.src = pl.tiles ? Src::kFp8 : Src::kF32;
    g2.dst = row16 ? Dst::kRowF16 : Dst::kSlotF32;
    g2.out = row16 ? (void*)m.y16 : (void*)m.y32; g2.out_scales = m.ys; g2.ldo = H; g2.all_rows = row16;
    if (pl.tiles) {
        if (int rc = launch_block_tiles(g1, s)) return rc;
        if (int rc = launch_block_tiles(g2, s)) return rc;
        if (row16) return launch_block_reduce(m.y16, m.ys, m.s2r, topk_weights, T, H, top_k, out, s);
    } else {
        if (int rc = launch_block_stream(g1, s)) return rc;
        if (int rc = launch_block_stream(g2, s)) return rc;
    }
    for (int64_t t = 0; t < T; t += kReduceRows)
        if (int rc = launch_slot_reduce(m.y32 + t * top_k * H, topk_weights + t * top_k, topk_ids + t * top_k, expert_map,
                                        n_global, E, std::min(kReduceRows, T - t), H, top_k,
                                        static_cast<uint16_t*>(out) + t * H, bf16, s))
            return rc;
    return W4A8_OK;
}

}  // extern "C"
