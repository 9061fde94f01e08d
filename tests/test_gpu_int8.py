"""int8 operators on the GPU against their float64 restatement (oracle/int8.py).

Tolerances are the oracle's: the sums are exact, so that a result is held to a few fp32 roundings and half a step of its
16-bit type, and the layer to what a value of h next to a border can move."""
import numpy as np
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import int8 as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a step, relative


def gen(*parts):
    return torch.Generator().manual_seed(hash(parts) % (1 << 31))


def f64(t):
    return t.double().cpu().numpy()


def hidden(g, rows, K, dtype, scale=1.0):
    """Normal values, some channels eight times as wide, rows of other sizes."""
    x = torch.randn((rows, K), generator=g) * scale
    x *= torch.where(torch.rand((K,), generator=g) < 1 / 16, 8.0, 1.0)
    x *= torch.exp(torch.randn((rows, 1), generator=g))
    return x.to(dtype)


def rows8(g, rows, K):
    return torch.randint(-128, 128, (rows, K), generator=g, dtype=torch.int8), torch.rand((rows, 1), generator=g) * 0.05 + 0.001


def weight(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8), torch.rand(shape[:-1], generator=g) * 2e-3 + 1e-5


def on(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def assert_close(got, ref, tol, dtype):
    got = f64(got)
    t = tol + (np.abs(ref) + tol) * HALF[dtype]
    if dtype == torch.float16:
        t = t + 2.0 ** -25              # half a step of its subnormal numbers
    bad = ~(np.abs(got - ref) <= t)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst by {np.nanmax(np.abs(got - ref) / t):.3g} tolerances"


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 8), (3, 127), (2, 512), (5, 520), (7, 1000), (9, 1024), (3, 2048), (33, 4096),
                                    (2, 8200), (3, 16384), (2, 20000), (2, 32768), (2, 40000), (1030, 64)])
def test_act_quant_is_exact(rows, K, dtype):
    x = hidden(gen(rows, K), rows, K, dtype)
    x[0] = 0                                     # the scale's floor
    if rows > 1 and K > 2:
        x[1] *= 0.1
        x[1, 0], x[1, 1] = 64.0, 32.0            # a border: 63.5
    q, s = W.act_quant_int8(x.to(DEV))
    rq, rs = O.quantise(f64(x))
    assert q.dtype == torch.int8 and tuple(s.shape) == (rows, 1)
    assert np.array_equal(s.cpu().numpy(), rs)
    assert np.array_equal(f64(q), rq)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_act_quant_extremes(dtype):
    top = torch.finfo(dtype).max
    x = torch.zeros((6, 64), dtype=dtype)
    x[0, 3], x[0, 4] = top, -top / 2
    x[1, 5] = torch.finfo(dtype).tiny
    x[2, 1], x[2, 2] = float("inf"), 1.0
    x[3, 1], x[3, 2] = float("nan"), 1.0
    x[4, 0] = -3.0
    q, s = (t.cpu() for t in W.act_quant_int8(x.to(DEV)))
    rq, rs = O.quantise(f64(x))
    assert np.array_equal(f64(q), rq) and np.array_equal(s.numpy(), rs, equal_nan=True)
    assert s[2:4].isnan().all() and q[0, 3] == 127 and q[4, 0] == -127


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,K", [(1, 8), (3, 100), (9, 512), (5, 1001), (64, 1536), (2, 9000)])
def test_silu_quant(rows, K, dtype):
    x = hidden(gen(rows, K, 1), rows, 2 * K, dtype, 2.0)
    q, s = W.act_quant_int8(x.to(DEV), activation="silu")
    v = f64(x)
    h = O.silu_mul(v[:, :K], v[:, K:])
    # exponential (4 roundings), sum, quotient, product
    rel = 8 * O.U32
    a = np.abs(h).max(1, keepdims=True)
    assert np.all(np.abs(f64(s) * 127 - a) <= a * (rel + 2 * O.U32) + 2.0 ** -90)
    t = h * 127.0 / np.maximum(a, O.LEAST)
    off = np.abs(t) * (2 * rel + 4 * O.U32)
    assert np.all(np.abs(f64(q) - t) <= 0.5 + off)


def test_silu_quant_of_far_gates():
    """silu(gate) * up of gates whose e^-gate is no normal number, beside ups near fp32's largest."""
    x = torch.zeros((2, 16), dtype=torch.bfloat16)
    x[:, :8] = torch.tensor([-86.0, -87.5, -88.5, -90.0, -95.0, -100.0, -81.0, -80.0])
    x[0, 8:], x[1, 8:] = 1e30, 3e38
    q, s = W.act_quant_int8(x.to(DEV), activation="silu")
    v = f64(x)
    h = O.silu_mul(v[:, :8], v[:, 8:])
    a = np.abs(h).max(1, keepdims=True)
    assert np.all(np.abs(f64(s) * 127 - a) <= a * 300 * O.U32)          # e^x: a step of the argument is |x| of its value
    assert np.all(np.abs(f64(q) - h * 127 / a) <= 0.5 + 127 * 600 * O.U32)


# ------------------------------------------------------------------ dense
SIZES = [(1, 1, 16), (1, 5, 48), (2, 17, 64), (3, 64, 112), (1, 4096, 4096), (5, 333, 1040), (8, 130, 12288), (16, 48, 128),
         (16, 1000, 2064), (17, 64, 256), (31, 100, 144), (33, 513, 528), (64, 256, 4096), (65, 127, 400), (77, 640, 272),
         (128, 128, 128), (130, 1030, 1008), (200, 96, 64), (256, 512, 1024), (257, 300, 2000), (300, 7, 96),
         (520, 776, 384)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_dense_int8_rows(M, N, K, dtype):
    g = gen(M, N, K)
    (x, xs), (w, ws) = rows8(g, M, K), weight(g, N, K)
    y = W.int8_gemm(*on(x, xs, w, ws), out_dtype=dtype)
    assert y.dtype == dtype and tuple(y.shape) == (M, N)
    assert_close(y, *O.product(f64(x), xs.numpy(), f64(w), ws.numpy()), dtype)


# a size for each dense tile, by the rule's costs on 256 CUs, with ragged sides and K in odd steps and a partial one
REACH = [(64, 4096, 272), (250, 4090, 208), (500, 4100, 144), (1000, 4090, 400), (1500, 4090, 272), (4000, 4100, 208)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", REACH)
def test_dense_tiles(M, N, K, dtype):
    g = gen(M, N, K, 20)
    (x, xs), (w, ws) = rows8(g, M, K), weight(g, N, K)
    y = W.int8_gemm(*on(x, xs, w, ws), out_dtype=dtype)
    # (on the GPU in fp64: the sums of whole numbers below 2^53 are exact in any order)
    X, XS, V, VS = on(x.double(), xs.double(), w.double(), ws.double())
    ref = (X @ V.t()) * XS * VS
    tol = ref.abs() * (4 * O.U32 + HALF[dtype] * (1 + 4 * O.U32)) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert bool(((y.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_dense_16bit_rows_with_bias(M, N, K, dtype):
    g = gen(M, N, K, 2)
    x, (w, ws) = hidden(g, M, K, dtype), weight(g, N, K)
    b = torch.randn((N,), generator=g) * 10
    b = b.to(dtype) if (M + N) % 2 else b
    y = W.int8_gemm(*on(x, None, w, ws), bias=b.to(DEV))
    assert_close(y, *O.product(*O.quantise(f64(x)), f64(w), ws.numpy(), f64(b)), dtype)


def test_dense_largest_sums():
    """Sums next to 2^31: K = 131056 of -128 times -128 is 2147221504."""
    K = 131056
    x, w = torch.full((3, K), -128, dtype=torch.int8), torch.full((5, K), -128, dtype=torch.int8)
    w[1] = 127
    y = W.int8_gemm(*on(x, torch.full((3,), 2.0 ** -20), w, torch.ones(5)), out_dtype=torch.bfloat16)
    assert_close(y, *O.product(f64(x), np.full((3, 1), 2.0 ** -20), f64(w), np.ones(5)), torch.bfloat16)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_dense_strided_and_offset_rows(M):
    g = gen(M, 3)
    w, ws = weight(g, 96, 160)
    big, xs = rows8(g, M, 192)
    ref = W.int8_gemm(*on(big[:, 16:176].contiguous(), xs, w, ws))
    d = big.to(DEV)
    wide = torch.zeros((M, 200), dtype=torch.int8, device=DEV)
    wide[:, 3:163] = d[:, 16:176]
    for view in (d[:, 16:176], wide[:, 3:163]):  # rows at multiples of 16 bytes, and elsewhere (a copy)
        assert torch.equal(W.int8_gemm(view, xs.to(DEV), *on(w, ws)), ref)
    x = hidden(g, M, 192, torch.bfloat16)
    ref = W.int8_gemm(*on(x[:, 8:168].contiguous(), None, w, ws))
    d = x.to(DEV)
    assert torch.equal(W.int8_gemm(d[:, 8:168], None, *on(w, ws)), ref)
    assert torch.equal(W.int8_gemm(d.t().contiguous().t()[:, 8:168], None, *on(w, ws)), ref)


@pytest.mark.parametrize("M", [2, 70])
def test_dense_rows_that_are_not_finite(M):
    g = gen(M, 4)
    x, (w, ws) = hidden(g, M, 256, torch.bfloat16), weight(g, 64, 256)
    clean = W.int8_gemm(*on(x, None, w, ws))
    x[1, 7] = float("inf")
    y = W.int8_gemm(*on(x, None, w, ws))
    assert y[1].isnan().all() and torch.equal(y[0], clean[0]) and torch.equal(y[2:], clean[2:])


def test_dense_no_rows_and_writes_only_its_rows():
    g = gen(5)
    w, ws = weight(g, 48, 64)
    assert W.int8_gemm(torch.empty((0, 64), dtype=torch.int8, device=DEV), torch.empty((0,), device=DEV), *on(w, ws)).shape == (0, 48)
    assert W.act_quant_int8(torch.empty((0, 64), dtype=torch.float16, device=DEV))[0].shape == (0, 64)


# ------------------------------------------------------------------ the layer
def make_layer(g, E, H, I):
    w13, s13 = weight(g, E, 2 * I, H)
    w2, s2 = weight(g, E, H, I)
    return w13, w2, s13 * 0.1, s2


def make_routing(g, T, E, k, skew=0.0):
    logits = torch.randn((T, E), generator=g) - skew * torch.arange(E).log1p()
    top, ids = torch.softmax(logits, 1).topk(k, 1)
    return top / top.sum(1, keepdim=True), ids.to(torch.int32)


def rows16(T, E, k, dtype):
    """Whether the layer rounds its slots' rows to 16 bits: many tokens, bf16 output."""
    return T * k > min(5 * E + 128, 4096) and dtype == torch.bfloat16


LAYERS = [(1, 8, 2, 64, 64), (1, 256, 8, 512, 128), (3, 16, 4, 192, 320), (5, 4, 4, 256, 64), (17, 8, 2, 64, 192), (32, 32, 4, 512, 256),
          (40, 2, 1, 128, 128), (65, 16, 2, 320, 704), (130, 8, 3, 256, 384), (200, 64, 6, 448, 128), (333, 4, 2, 512, 512),
          (700, 8, 8, 128, 192)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,I", LAYERS)
def test_layer(T, E, k, H, I, dtype):
    g = gen(T, E, k, H, I)
    w13, w2, s13, s2 = make_layer(g, E, H, I)
    tw, ids = make_routing(g, T, E, k, 0.5)
    x = hidden(g, T, H, dtype)
    y = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, ids))
    ref, tol = O.layer(*O.quantise(f64(x)), f64(w13), s13.numpy(), f64(w2), s2.numpy(), tw.numpy(), ids.numpy(),
                       rows16=rows16(T, E, k, dtype))
    assert_close(y, ref, tol, dtype)
    q, s = W.act_quant_int8(x.to(DEV))
    assert torch.equal(W.moe_int8_apply(q, *on(w13, w2, s13, s2, tw, ids), x_scales=s, out_dtype=dtype), y)


@pytest.mark.parametrize("T", [4, 90, 400])
def test_layer_expert_map_and_absent_slots(T):
    """Experts of other ranks, ids of no expert, tokens without any slot."""
    E, glob, k, H, I = 8, 24, 4, 256, 128
    g = gen(T, 7)
    w13, w2, s13, s2 = make_layer(g, E, H, I)
    tw, ids = make_routing(g, T, glob, k)
    emap = torch.full((glob,), -1, dtype=torch.int32)
    emap[torch.randperm(glob, generator=g)[:E]] = torch.randperm(E, generator=g).to(torch.int32)
    ids[0] = -1
    ids[1, 1], ids[2, 0] = -1, glob + 5
    x = hidden(g, T, H, torch.bfloat16)
    y = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, ids), expert_map=emap.to(DEV), global_num_experts=glob)
    ref, tol = O.layer(*O.quantise(f64(x)), f64(w13), s13.numpy(), f64(w2), s2.numpy(), tw.numpy(), ids.numpy(), emap.numpy(),
                       rows16=rows16(T, E, k, torch.bfloat16))
    assert_close(y, ref, tol, torch.bfloat16)
    assert not y[0].any()
    none = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, torch.full_like(ids, -1)))
    assert not none.any()


@pytest.mark.parametrize("T", [6, 500])
def test_layer_repeats_and_twice_the_same_expert(T):
    g = gen(T, 8)
    w13, w2, s13, s2 = make_layer(g, 4, 128, 128)
    tw, ids = make_routing(g, T, 4, 2)
    ids[:, 1] = ids[:, 0]                        # both picks the same
    x = hidden(g, T, 128, torch.bfloat16)
    args = on(x, w13, w2, s13, s2, tw, ids)
    y = W.moe_int8_apply(*args)
    ref, tol = O.layer(*O.quantise(f64(x)), f64(w13), s13.numpy(), f64(w2), s2.numpy(), tw.numpy(), ids.numpy(),
                       rows16=rows16(T, 4, 2, torch.bfloat16))
    assert_close(y, ref, tol, torch.bfloat16)
    for _ in range(3):
        assert torch.equal(W.moe_int8_apply(*args), y)


@pytest.mark.parametrize("T", [6, 500])
def test_layer_rows_that_are_not_finite_leave_the_others(T):
    g = gen(T, 9)
    w13, w2, s13, s2 = make_layer(g, 4, 128, 128)
    tw, ids = make_routing(g, T, 4, 2)
    x = hidden(g, T, 128, torch.bfloat16)
    clean = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, ids))
    x[3, 5] = float("nan")
    y = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, ids))
    keep = torch.arange(T) != 3
    assert y[3].isnan().all() and torch.equal(y[keep.to(DEV)], clean[keep.to(DEV)])


@pytest.mark.parametrize("T", [6, 500])
def test_layer_channels_of_other_sizes(T):
    """A channel scale that is infinite, or 2^20 times its neighbours', leaves the columns beside it."""
    g = gen(T, 14)
    w13, w2, s13, s2 = make_layer(g, 4, 128, 128)
    tw, ids = make_routing(g, T, 4, 2)
    x = hidden(g, T, 128, torch.bfloat16)
    s2[:, 40] *= 2.0 ** 20
    args = (O.quantise(f64(x)), f64(w13), s13.numpy(), f64(w2))
    ref, tol = O.layer(*args[0], *args[1:], s2.numpy(), tw.numpy(), ids.numpy(), rows16=rows16(T, 4, 2, torch.bfloat16))
    s2[:, 7] = float("inf")
    y = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, ids))
    keep = [n for n in range(128) if n != 7]
    assert_close(y[:, keep], ref[:, keep], tol[:, keep], torch.bfloat16)
    assert not y[:, 7].isfinite().any()


def test_layer_no_tokens():
    w13, w2, s13, s2 = make_layer(gen(10), 4, 128, 64)
    y = W.moe_int8_apply(*on(torch.empty((0, 128), dtype=torch.bfloat16), w13, w2, s13, s2, torch.empty((0, 2)),
                             torch.empty((0, 2), dtype=torch.int32)))
    assert y.shape == (0, 128)


# ------------------------------------------------------------------ streams, graphs, the run of them together
def test_router_into_layer_into_dense():
    """Router, expert layer and a following projection, as a decoder layer runs them."""
    T, E, k, H, I = 37, 32, 4, 256, 128
    g = gen(11)
    w13, w2, s13, s2 = make_layer(g, E, H, I)
    wr = torch.randn((H, E), generator=g) * 0.1
    bias = torch.randn((E,), generator=g) * 0.1
    wd, sd = weight(g, 96, H)
    x = hidden(g, T, H, torch.bfloat16)
    args = on(x, w13, w2, s13, s2, wr, bias, wd, sd)

    def step(x, w13, w2, s13, s2, wr, bias, wd, sd):
        logits = x.float() @ wr
        tw, ids = W.route_topk(logits, k, scoring="sigmoid", bias=bias, num_groups=8, top_groups=4, scale=2.5)
        y = W.moe_int8_apply(x, w13, w2, s13, s2, tw, ids)
        return logits, tw, ids, y, W.int8_gemm(y, None, wd, sd)

    logits, tw, ids, y, z = step(*args)
    rw, rid = O.route(f64(logits), k, "sigmoid", bias.numpy(), 8, 4, True, 2.5)
    assert np.array_equal(ids.cpu().numpy(), rid) and np.allclose(f64(tw), rw, rtol=1e-6, atol=0)
    ref, tol = O.layer(*O.quantise(f64(x)), f64(w13), s13.numpy(), f64(w2), s2.numpy(), tw.cpu().numpy(), rid)
    assert_close(y, ref, tol, torch.bfloat16)
    assert_close(z, *O.product(*O.quantise(f64(y)), f64(wd), sd.numpy()), torch.bfloat16)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip((logits, tw, ids, y, z), other))


@pytest.mark.parametrize("T", [1, 20, 300])
def test_captured_and_replayed(T):
    """Replays with new inputs, eager work and synchronisation between them, equal the eager calls."""
    E, k, H, I = 16, 2, 256, 128
    g = gen(T, 12)
    w13, w2, s13, s2 = on(*make_layer(g, E, H, I))
    wd, sd = on(*weight(g, 96, H))
    bias = torch.zeros((E,), device=DEV)
    x = torch.zeros((T, H), dtype=torch.bfloat16, device=DEV)
    l = torch.zeros((T, E), device=DEV)

    def step():
        tw, ids = W.route_topk(l, k, scoring="sigmoid", bias=bias)
        y = W.moe_int8_apply(x, w13, w2, s13, s2, tw, ids)
        return tw, ids, y, W.int8_gemm(y, None, wd, sd)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(3):
        x.copy_(hidden(g, T, H, torch.bfloat16))
        l.copy_(torch.randn((T, E), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), n


def test_torch_ops():
    g = gen(13)
    x, (w, ws) = hidden(g, 9, 128, torch.float16).to(DEV), on(*weight(g, 64, 128))
    ops = torch.ops.w4a8_fp8_wmma
    q, s = ops.act_quant_int8(x, None)
    assert torch.equal(ops.int8_gemm(q, s, w, ws, None, torch.float16), W.int8_gemm(x, None, w, ws))
    w13, w2, s13, s2 = on(*make_layer(g, 4, 128, 64))
    l = torch.randn((9, 4), generator=g).to(DEV)
    tw, ids = ops.route_topk(l, 2, "softmax", None, 1, 1, True, 1.0)
    assert torch.equal(ops.moe_int8_apply(x, w13, w2, s13, s2, tw, ids, None, None, torch.float16),
                       W.moe_int8_apply(x, w13, w2, s13, s2, tw, ids))
