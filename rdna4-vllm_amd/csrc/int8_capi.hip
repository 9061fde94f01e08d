// C ABI entry points of the int8 operators (include/w4a8_int8.h): argument checks, workspace carving, the choice of
// kernel and the whole-layer composition.
#include <algorithm>
#include <string>

#include "../../include/w4a8_int8.h"
#include "int8.h"

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
Src8 src_of(int dt) { return dt == W4A8_DTYPE_INT8 ? Src8::kI8 : dt == W4A8_DTYPE_BF16 ? Src8::kBf16 : Src8::kF16; }
Rows rows_of(int dt) { return dt == W4A8_DTYPE_BF16 ? Rows::kBf16 : Rows::kF16; }

constexpr int64_t kMaxSide = (int64_t)1 << 24;    // rows of a weight
// Dense rows and K up to which the weights are streamed, else tiles. us streamed / tiles, 8 rows: 2048 x 2048 4.4 / 5.1,
// one row: 229376 x 2048 82 / 84, 229376 x 512 29 / 34; but 4096 x 4096 7.3 / 6.8, 12288 x 4096 13.0 / 10.0, 28672 x 8192 63 / 44.
constexpr int64_t kStreamRows = 16, kStreamK = 2048;
constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 256;

// Dense rows that the product's kernel quantises itself; more take a launch of their own. us in the kernel / before tiles,
// 4096 x 4096: 1 row 7.7 / 8.8, 4 rows 8.9 / 9.1; but 12288 x 4096, 1 row 14.3 / 12.1.
bool quantised_in_kernel(int64_t M, int64_t K, int64_t N) {
    return M <= 4 && int8_rows_quantised_in_kernel(K) && (K <= kStreamK || N * K <= (int64_t)1 << 25);
}

// Sizes and pointers that every product shares.
int check_product(const void* x, int x_dtype, const float* xs, int64_t rows, int64_t K, int64_t ldx, const int8_t* w,
                  const float* ws, int64_t E, int64_t N) {
    W4A8_REQUIRE(rows >= 0 && rows <= kMaxRows && K > 0 && N > 0 && E > 0, "int8 product: invalid sizes");
    W4A8_REQUIRE(K <= kMaxInt8K, "int8 product: K is over 131071, where sums may pass 32 bits");
    W4A8_REQUIRE(N <= kMaxSide && E <= kMaxSide, "int8 product: a size is over 2^24");
    W4A8_REQUIRE(K % 16 == 0, "int8 product: K must be a multiple of 16");
    W4A8_REQUIRE(x_dtype == W4A8_DTYPE_INT8 || is16(x_dtype), "int8 product: x must be int8, fp16 or bf16");
    if (rows == 0) return W4A8_OK;
    W4A8_REQUIRE(x && w && ws, "int8 product: null pointer");
    W4A8_REQUIRE(x_dtype != W4A8_DTYPE_INT8 || xs, "int8 product: int8 rows need their scales");
    W4A8_REQUIRE(ldx >= K && ldx * (x_dtype == W4A8_DTYPE_INT8 ? 1 : 2) % 16 == 0,
                 "int8 product: rows of x must start at multiples of 16 bytes");
    W4A8_REQUIRE(aligned16(x) && aligned16(w), "int8 product: x and w must be aligned to 16 bytes");
    return W4A8_OK;
}

// ---- the gated layer ----
// Few rows an expert: the streaming kernels, which find their rows in the routed ids (h and the slots' rows in fp32, by
// slot). Else tiles: rows quantised beforehand, slots aligned to blocks of the rows that a tile has. The slots' rows are
// fp32 in every schedule and summed in the slots' order, so that a token's output has the same bits in any batch (in fp16
// they are half the bytes, but where slots cancel their roundings are all that is left). Tokens are taken in parts of as
// many as either can address.
// Slots an expert from which tiles have 128 rows (us with 64 / 128: 64 experts of 4096 x 1024, 6 picks: 96 slots an expert
// 281 / 278, 192 410 / 373, 384 686 / 639; but 256 experts of 2048 x 512, skewed, 128 slots an expert: 376 / 419).
constexpr int64_t kWideRows = 192;
struct LayerPlan {
    bool tiles;
    int64_t part;                // tokens of a part
    int64_t block_m;             // tiles: rows of a block
    int64_t P, nblk;             // of a part: padded rows and blocks
    bool quant_x, quant_h;       // rows quantised by a launch of their own
};
LayerPlan plan_layer(int64_t T, int64_t H, int64_t inter, int64_t E, int64_t top_k, int x_dtype) {
    LayerPlan pl{};
    const int64_t lim = ((int64_t)1 << 32) - 1, pad = E * 127 + 128;
    // (us streamed / tiles: 256 experts of 2048 x 512, 8 picks, 100 tokens 158 / 178, 176 172 / 183, 256 189 / 187, skewed 176
    // 187 / 163, 256 236 / 175; 32 experts, 4 picks, 64 tokens 38 / 41, 90 53 / 41; 8 experts, 2 picks, 40 tokens 30 / 35, 90
    // 39 / 37.)
    pl.tiles = T * top_k > std::min<int64_t>(5 * E + 128, kScanSlots) && 2 * inter * H <= lim;
    const int64_t most = pl.tiles ? std::min(lim / H, (lim / inter - pad) / top_k) : kScanSlots / top_k;
    pl.part = std::min(T, std::max<int64_t>(1, most));
    const int64_t n = pl.part * top_k;
    pl.block_m = n >= kWideRows * E ? 128 : 64;
    // every block in use holds a slot
    pl.P = pl.tiles ? std::min((n + E * (pl.block_m - 1) + pl.block_m - 1) / pl.block_m * pl.block_m, n * pl.block_m) : n;
    pl.nblk = pl.P / pl.block_m;
    pl.quant_x = x_dtype != W4A8_DTYPE_INT8 && (pl.tiles || !int8_rows_quantised_in_kernel(H));
    pl.quant_h = pl.tiles || !int8_rows_quantised_in_kernel(inter);
    return pl;
}
struct LayerScratch {
    int32_t *sti, *eid, *ntp;
    void* align_ws;
    size_t align_bytes;
    int8_t *xq, *hq;
    float *xs, *hs, *h, *y;
};
template <typename WS>
void carve_layer(WS& w, const LayerPlan& pl, int64_t H, int64_t inter, int64_t E, int64_t top_k, LayerScratch& m) {
    m = LayerScratch{};
    const int64_t n = pl.part * top_k;
    if (pl.tiles) {
        m.sti = w.template take<int32_t>((size_t)pl.P);
        m.eid = w.template take<int32_t>((size_t)pl.nblk);
        m.ntp = w.template take<int32_t>(1);
        m.align_bytes = align_workspace_bytes(n, E);
        m.align_ws = w.template take<uint8_t>(m.align_bytes);
    }
    if (pl.quant_x) {
        m.xq = w.template take<int8_t>((size_t)(pl.part * H));
        m.xs = w.template take<float>((size_t)pl.part);
    }
    m.h = w.template take<float>((size_t)(pl.P * inter));
    if (pl.quant_h) {
        m.hq = w.template take<int8_t>((size_t)(pl.P * inter));
        m.hs = w.template take<float>((size_t)pl.P);
    }
    m.y = w.template take<float>((size_t)(n * H));
}
struct Layer {
    const void* x;
    int x_dtype;
    const float* xs;
    int64_t T, H, inter, E, top_k;
    const int8_t* w13;
    const float* s13;
    const int8_t* w2;
    const float* s2;
    const float* tw;
    const int32_t* ids;
    const int32_t* emap;
    int64_t n_global;
    void* out;
    bool bf16;
};
int run_layer(const Layer& l, const LayerPlan& pl, const LayerScratch& m, hipStream_t s) {
    const int64_t n = l.T * l.top_k;
    const void* x = l.x;
    const float* xs = l.xs;
    if (pl.quant_x) {
        if (int rc = launch_act_quant_int8(x, rows_of(l.x_dtype), l.T, l.H, l.H, false, m.xq, m.xs, nullptr, nullptr, 0, s)) return rc;
        x = m.xq;
        xs = m.xs;
    }
    if (pl.tiles) {
        if (int rc = launch_align(l.ids, n, l.E, pl.block_m, l.emap, l.n_global, m.sti, pl.P, m.eid, m.ntp, m.align_ws,
                                  m.align_bytes, s))
            return rc;
        Int8Args g1{};
        g1.x = static_cast<const int8_t*>(x); g1.xs = xs; g1.x_rows = l.T; g1.K = l.H; g1.ldx = l.H;
        g1.w = l.w13; g1.ws = l.s13; g1.E = l.E; g1.N = 2 * l.inter;
        g1.sorted_ids = m.sti; g1.expert_ids = m.eid; g1.ntp = m.ntp; g1.P = pl.P;
        g1.top_k = l.top_k; g1.num_valid = n; g1.block_m = pl.block_m; g1.gather = true;
        g1.dst = Out8::kSiluF32; g1.out = m.h; g1.ldo = l.inter;
        if (int rc = launch_int8_tiles(g1, s)) return rc;
        if (int rc = launch_act_quant_int8(m.h, Rows::kF32, pl.P, l.inter, l.inter, false, m.hq, m.hs, m.sti, m.ntp, n, s)) return rc;
        Int8Args g2 = g1;
        g2.x = m.hq; g2.xs = m.hs; g2.x_rows = pl.P; g2.K = l.inter; g2.ldx = l.inter;
        g2.w = l.w2; g2.ws = l.s2; g2.N = l.H; g2.gather = false;
        g2.dst = Out8::kSlotF32; g2.out = m.y; g2.ldo = l.H;
        if (int rc = launch_int8_tiles(g2, s)) return rc;
    } else {
        RowsArgs g1{};
        g1.x = x; g1.src = pl.quant_x ? Src8::kI8 : src_of(l.x_dtype); g1.xs = xs; g1.rows = l.T; g1.K = l.H; g1.ldx = l.H;
        g1.w = l.w13; g1.ws = l.s13; g1.E = l.E; g1.N = 2 * l.inter;
        g1.ids = l.ids; g1.emap = l.emap; g1.emap_len = l.n_global; g1.slots = n; g1.top_k = l.top_k;
        g1.gather = true; g1.dst = Out8::kSiluF32; g1.out = m.h; g1.ldo = l.inter;
        if (int rc = launch_int8_rows(g1, s)) return rc;
        RowsArgs g2 = g1;
        g2.x = m.h; g2.src = Src8::kF32; g2.rows = n; g2.K = l.inter; g2.ldx = l.inter;
        if (pl.quant_h) {
            if (int rc = launch_act_quant_int8(m.h, Rows::kF32, n, l.inter, l.inter, false, m.hq, m.hs, nullptr, nullptr, 0, s)) return rc;
            g2.x = m.hq; g2.src = Src8::kI8; g2.xs = m.hs;
        }
        g2.w = l.w2; g2.ws = l.s2; g2.N = l.H; g2.gather = false; g2.ldo = l.H;
        if (int8_token_supported(n, l.E, l.inter)) {
            g2.dst = Out8::k16; g2.out = l.out; g2.bf16 = l.bf16;
            return launch_int8_token(g2, l.tw, s);
        }
        g2.dst = Out8::kSlotF32; g2.out = m.y;
        if (int rc = launch_int8_rows(g2, s)) return rc;
    }
    return launch_int8_reduce(m.y, l.tw, l.ids, l.emap, l.n_global, l.E, l.T, l.H, l.top_k, l.out, l.bf16, s);
}
struct SizeProbe {
    WorkspaceSize s;
    template <typename T>
    T* take(size_t n) { s.take<T>(n); return nullptr; }
};

}  // namespace
}  // namespace w4a8

using namespace w4a8;

extern "C" {

int w4a8_int8_abi_version(void) { return 1; }
const char* w4a8_int8_last_error(void) { return last_error().c_str(); }

int w4a8_act_quant_int8(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t x_stride, int silu_gate_up, int8_t* q,
                        float* scales, void* stream) {
    clear_error();
    W4A8_REQUIRE(is16(x_dtype), "act_quant_int8: x must be fp16 or bf16");
    W4A8_REQUIRE(rows >= 0 && rows <= kMaxRows && K > 0 && K <= kMaxSide, "act_quant_int8: invalid sizes");
    if (rows == 0) return W4A8_OK;
    W4A8_REQUIRE(x && q && scales, "act_quant_int8: null pointer");
    W4A8_REQUIRE(x_stride >= (silu_gate_up ? 2 * K : K) || rows == 1, "act_quant_int8: rows overlap");
    return launch_act_quant_int8(x, rows_of(x_dtype), rows, K, x_stride, silu_gate_up != 0, q, scales, nullptr, nullptr, 0,
                                 as_stream(stream));
}

size_t w4a8_int8_gemm_workspace_size(int x_dtype, int64_t M, int64_t K, int64_t N) {
    if (x_dtype == W4A8_DTYPE_INT8 || M <= 0 || K <= 0 || N <= 0 || quantised_in_kernel(M, K, N)) return 0;
    WorkspaceSize s;
    s.take<int8_t>((size_t)(M * K));
    s.take<float>((size_t)M);
    return s.used;
}

int w4a8_int8_gemm(const void* x, int x_dtype, const float* x_scales, int64_t M, int64_t K, int64_t x_stride, const int8_t* w,
                   const float* w_scales, int64_t N, const void* bias, int bias_is_f32, void* out, int out_dtype,
                   void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    if (int rc = check_product(x, x_dtype, x_scales, M, K, x_stride, w, w_scales, 1, N)) return rc;
    W4A8_REQUIRE(is16(out_dtype), "int8_gemm: out must be fp16 or bf16");
    if (M == 0) return W4A8_OK;
    W4A8_REQUIRE(out, "int8_gemm: null pointer");
    hipStream_t s = as_stream(stream);
    const bool in_kernel = quantised_in_kernel(M, K, N);
    Src8 src = src_of(x_dtype);
    if (src != Src8::kI8 && !in_kernel) {
        Workspace ws(workspace, workspace_bytes);
        int8_t* xq = ws.take<int8_t>((size_t)(M * K));
        float* xs = ws.take<float>((size_t)M);
        if (workspace == nullptr || !ws.ok()) {
            set_error("int8_gemm: workspace smaller than w4a8_int8_gemm_workspace_size()");
            return W4A8_ERR_WORKSPACE;
        }
        if (int rc = launch_act_quant_int8(x, rows_of(x_dtype), M, K, x_stride, false, xq, xs, nullptr, nullptr, 0, s)) return rc;
        x = xq; x_scales = xs; x_stride = K; src = Src8::kI8;
    }
    Int8Args a{};
    a.x = static_cast<const int8_t*>(x); a.xs = x_scales; a.x_rows = M; a.K = K; a.ldx = x_stride;
    a.w = w; a.ws = w_scales; a.E = 1; a.N = N; a.bias = bias; a.bias_f32 = bias_is_f32 != 0;
    a.P = M; a.top_k = 1; a.num_valid = M; a.block_m = 16;
    a.dst = Out8::k16; a.bf16 = out_dtype == W4A8_DTYPE_BF16; a.out = out; a.ldo = N;
    // The tiles address weights and rows in 32 bits: rows past that are taken in parts.
    const int64_t lim = ((int64_t)1 << 32) - 1, part = lim / x_stride / 256 * 256;
    if ((M > kStreamRows || K > kStreamK) && src == Src8::kI8 && N * K <= lim && part > 0) {
        for (int64_t m = 0; m < M; m += part) {
            a.x_rows = a.P = a.num_valid = std::min(part, M - m);
            if (int rc = launch_int8_tiles(a, s)) return rc;
            a.x += part * x_stride;
            a.xs += part;
            a.out = static_cast<uint16_t*>(a.out) + part * N;
        }
        return W4A8_OK;
    }
    RowsArgs r{};
    r.x = x; r.src = src; r.xs = x_scales; r.rows = M; r.K = K; r.ldx = x_stride;
    r.w = w; r.ws = w_scales; r.E = 1; r.N = N; r.bias = bias; r.bias_f32 = a.bias_f32; r.top_k = 1;
    r.dst = Out8::k16; r.bf16 = a.bf16; r.out = out; r.ldo = N;
    return launch_int8_rows(r, s);
}

size_t w4a8_moe_int8_workspace_size(int64_t T, int64_t H, int64_t inter, int64_t E, int64_t top_k) {
    if (T <= 0 || H <= 0 || inter <= 0 || E <= 0 || top_k <= 0) return 0;
    SizeProbe p;
    LayerScratch m;
    carve_layer(p, plan_layer(T, H, inter, E, top_k, W4A8_DTYPE_F16), H, inter, E, top_k, m);
    return p.s.used;
}

int w4a8_moe_int8_apply(const void* x, int x_dtype, const float* x_scales, int64_t T, int64_t H, int64_t inter, int64_t E,
                        int64_t top_k, const int8_t* w13, const float* w13_scales, const int8_t* w2, const float* w2_scales,
                        const float* topk_weights, const int32_t* topk_ids, const int32_t* expert_map,
                        int64_t num_global_experts, void* out, int out_dtype, void* workspace, size_t workspace_bytes,
                        void* stream) {
    clear_error();
    W4A8_REQUIRE(inter > 0 && inter % 64 == 0 && H > 0 && H % 64 == 0 && inter <= kMaxInt8K,
                 "moe_int8_apply: hidden and intermediate sizes must be multiples of 64");
    W4A8_REQUIRE(top_k > 0 && top_k <= 1024, "moe_int8_apply: invalid top_k");
    W4A8_REQUIRE(T >= 0 && T <= kMaxRows / top_k, "moe_int8_apply: invalid sizes");
    if (int rc = check_product(x, x_dtype, x_scales, T, H, H, w13, w13_scales, E, 2 * inter)) return rc;
    W4A8_REQUIRE(is16(out_dtype), "moe_int8_apply: out must be fp16 or bf16");
    const int64_t n_global = num_global_experts > 0 ? num_global_experts : E;
    W4A8_REQUIRE(expert_map != nullptr || n_global == E,
                 "moe_int8_apply: global expert count differs from the local one; pass expert_map");
    W4A8_REQUIRE(E <= 1024 && n_global <= (int64_t)1 << 20, "moe_int8_apply: too many experts");
    if (T == 0) return W4A8_OK;
    W4A8_REQUIRE(w2 && w2_scales && topk_weights && topk_ids && out, "moe_int8_apply: null pointer");
    W4A8_REQUIRE(aligned16(w2) && aligned16(out), "moe_int8_apply: w2 and out must be aligned to 16 bytes");
    const LayerPlan pl = plan_layer(T, H, inter, E, top_k, x_dtype);
    Workspace w(workspace, workspace_bytes);
    LayerScratch m;
    carve_layer(w, pl, H, inter, E, top_k, m);
    if (workspace == nullptr || workspace_bytes < w4a8_moe_int8_workspace_size(T, H, inter, E, top_k)) {
        set_error("moe_int8_apply: workspace smaller than w4a8_moe_int8_workspace_size()");
        return W4A8_ERR_WORKSPACE;
    }
    const int64_t xbytes = x_dtype == W4A8_DTYPE_INT8 ? 1 : 2;
    for (int64_t t = 0; t < T; t += pl.part) {
        const Layer l{static_cast<const char*>(x) + t * H * xbytes, x_dtype, x_scales == nullptr ? nullptr : x_scales + t,
                      std::min(pl.part, T - t), H, inter, E, top_k, w13, w13_scales, w2, w2_scales,
                      topk_weights + t * top_k, topk_ids + t * top_k, expert_map, n_global,
                      static_cast<uint16_t*>(out) + t * H, out_dtype == W4A8_DTYPE_BF16};
        if (int rc = run_layer(l, pl, m, as_stream(stream))) return rc;
    }
    return W4A8_OK;
}

}  // extern "C"
