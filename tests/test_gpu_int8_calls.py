"""Calls of the int8 operators and the expert choice that their sizes allow beside the ordinary ones: long rows, many and
few experts, more picks, borders of the schedules, offsets past 32 bits, calls at once, scores in doubt."""
import numpy as np
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import int8 as O
from test_gpu_int8 import DEV, assert_close, f64, gen, hidden, make_layer, make_routing, on, rows16, rows8, weight
from test_gpu_route import check as check_route

pytestmark = pytest.mark.gpu


def layer_ok(T, E, k, H, I, dtype=torch.bfloat16, skew=0.0, part=None):
    g = gen(T, E, k, H, I, 40)
    w13, w2, s13, s2 = make_layer(g, E, H, I)
    tw, ids = make_routing(g, T, E, k, skew)
    x = hidden(g, T, H, dtype)
    args = on(x, w13, w2, s13, s2, tw, ids)
    y = W.moe_int8_apply(*args)
    rows = slice(None) if part is None else slice(T - part, T)
    ref, tol = O.layer(*[a[rows] for a in O.quantise(f64(x))], f64(w13), s13.numpy(), f64(w2), s2.numpy(), tw.numpy()[rows],
                       ids.numpy()[rows], rows16=rows16(T, E, k, dtype))
    assert_close(y[rows], ref, tol, dtype)
    assert torch.equal(args[0].cpu(), x)
    return y


# ------------------------------------------------------------------ sizes
@pytest.mark.parametrize("M", [1, 3, 5, 16, 20])
@pytest.mark.parametrize("K", [4096, 4112, 8192, 12304, 20000])
def test_dense_long_rows(M, K):
    g = gen(M, K, 41)
    (x, xs), (w, ws) = rows8(g, M, K), weight(g, 70, K)
    assert_close(W.int8_gemm(*on(x, xs, w, ws)), *O.product(f64(x), xs.numpy(), f64(w), ws.numpy()), torch.bfloat16)
    x = hidden(g, M, K, torch.float16)
    assert_close(W.int8_gemm(*on(x, None, w, ws)), *O.product(*O.quantise(f64(x)), f64(w), ws.numpy()), torch.float16)


@pytest.mark.parametrize("T", [1, 9, 80])
@pytest.mark.parametrize("H,I", [(4160, 64), (64, 4160), (4096, 128), (128, 4096), (1088, 576)])
def test_layer_long_rows(T, H, I):
    """Rows of up to 4096 values are quantised by the product's work-groups, longer ones by a launch of their own."""
    layer_ok(T, 4, 2, H, I)


@pytest.mark.parametrize("T,E,k", [(1, 128, 12), (1, 256, 17), (3, 200, 8), (2, 64, 4), (5, 40, 11), (60, 24, 12), (1, 1, 1), (7, 1, 1), (400, 1, 1)])
def test_layer_picks_and_experts(T, E, k):
    layer_ok(T, E, k, 128, 64)


@pytest.mark.parametrize("T", [1, 5, 40, 600])
def test_layer_many_experts(T):
    """1024 experts; 600 tokens x 8 are more slots than the streaming kernels look through."""
    layer_ok(T, 1024, 8, 64, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("slots", [167, 168, 169, 170, 8 * 192 - 2, 8 * 192])
def test_layer_at_the_schedules_borders(slots, dtype):
    """8 experts: up to 168 slots are streamed, from 1536 on tiles have 128 rows."""
    k = 2 if slots % 2 == 0 else 1
    layer_ok(slots // k, 8, k, 128, 128, dtype)


@pytest.mark.parametrize("T", [130, 700])
def test_layer_skewed(T):
    """Experts without a row, with one, with hundreds."""
    layer_ok(T, 16, 2, 128, 64, skew=4.0)


@pytest.mark.parametrize("T,E,k,kind", [(50, 64, 8, "one"), (50, 64, 8, "two"), (2, 256, 8, "one"), (33, 1024, 8, "one"), (512, 1024, 8, "few"),
                                        (512, 1024, 8, "all"), (16, 1, 8, "one"), (50, 64, 8, "none"), (3, 256, 8, "none"), (50, 64, 8, "odd")])
def test_layer_ids(T, E, k, kind):
    """Every slot at one expert or at few, an expert several times among a token's picks, no slot at all, ids of no expert."""
    H, I = 128, 64
    g = gen(T, E, k, 47)
    w13, w2, s13, s2 = make_layer(g, E, H, I)
    tw = torch.rand((T, k), generator=g)
    pick = {"one": [E - 1], "two": [0, E - 1], "few": [1, 7, 500, 1023], "all": list(range(E)), "none": [-1], "odd": [-5, 3, E, 2 ** 31 - 1]}[kind]
    ids = torch.tensor(pick)[torch.randint(0, len(pick), (T, k), generator=g)].to(torch.int32)
    x = hidden(g, T, H, torch.bfloat16)
    args = on(x, w13, w2, s13, s2, tw, ids)
    y = W.moe_int8_apply(*args)
    live = torch.where((ids >= 0) & (ids < E), ids, -1)
    ref, tol = O.layer(*O.quantise(f64(x)), f64(w13), s13.numpy(), f64(w2), s2.numpy(), tw.numpy(), live.numpy(),
                       rows16=rows16(T, E, k, torch.bfloat16))
    assert_close(y, ref, tol, torch.bfloat16)
    for _ in range(5):
        assert torch.equal(W.moe_int8_apply(*args), y)


def test_layer_many_tokens_of_wide_experts():
    layer_ok(3000, 4, 2, 192, 704, part=40)


# ------------------------------------------------------------------ offsets past 32 bits
def test_layer_experts_past_32_bits():
    """The last of 600 experts lie past 2^32 bytes: the same as a layer of those alone."""
    E, H, I, T, k = 600, 2048, 2048, 5, 2
    g = torch.Generator(device=DEV).manual_seed(3)
    w13 = torch.randint(-128, 128, (E, 2 * I, H), generator=g, dtype=torch.int8, device=DEV)
    w2 = torch.randint(-128, 128, (E, H, I), generator=g, dtype=torch.int8, device=DEV)
    s13 = torch.rand((E, 2 * I), generator=g, device=DEV) * 1e-4
    s2 = torch.rand((E, H), generator=g, device=DEV) * 1e-3
    for T in (1, 40):
        x = torch.randn((T, H), generator=g, device=DEV).bfloat16()
        tw = torch.rand((T, k), generator=g, device=DEV)
        ids = torch.randint(0, 16, (T, k), generator=g, device=DEV, dtype=torch.int32)
        y = W.moe_int8_apply(x, w13, w2, s13, s2, tw, ids + (E - 16))
        small = W.moe_int8_apply(x, *(t[E - 16:].contiguous() for t in (w13, w2, s13, s2)), tw, ids)
        assert torch.equal(y, small)
    # tiles: more slots than are streamed
    T = 1700
    x = torch.randn((T, H), generator=g, device=DEV).bfloat16()
    tw = torch.rand((T, k), generator=g, device=DEV)
    ids = torch.randint(E - 16, E, (T, k), generator=g, device=DEV, dtype=torch.int32)
    y = W.moe_int8_apply(x, w13, w2, s13, s2, tw, ids)
    few = W.moe_int8_apply(x[:64], w13, w2, s13, s2, tw[:64], ids[:64]).float()
    # (64 tokens of 600 experts are streamed: rows in fp32 against fp16, then one rounding each)
    assert bool(((y[:64].float() - few).abs() <= few.abs() * 2.0 ** -7 + few.abs().amax() * 2.0 ** -9).all())


def test_dense_weights_and_outputs_past_32_bits():
    """N K and M N past 2^32: the streaming kernel by its 64-bit addresses, the tiles' stores by theirs."""
    g = torch.Generator(device=DEV).manual_seed(4)
    N, K, M = 70000, 65536, 18                       # 4.6e9 weights: not addressed by the tiles
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8, device=DEV)
    ws = torch.rand((N,), generator=g, device=DEV) * 1e-3
    x = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device=DEV)
    xs = torch.rand((M,), generator=g, device=DEV)
    y = W.int8_gemm(x, xs, w, ws)
    assert torch.equal(y[:, N - 300:], W.int8_gemm(x, xs, w[N - 300:].contiguous(), ws[N - 300:].contiguous()))
    assert torch.equal(y[:, :300], W.int8_gemm(x, xs, w[:300].contiguous(), ws[:300].contiguous()))
    del w, y
    M, N, K = 70000, 65536, 64
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8, device=DEV)
    ws = torch.rand((N,), generator=g, device=DEV) * 1e-3
    x = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device=DEV)
    xs = torch.rand((M,), generator=g, device=DEV)
    y = W.int8_gemm(x, xs, w, ws)
    for rows in (slice(0, 40), slice(M - 40, M)):
        assert torch.equal(y[rows], W.int8_gemm(x[rows].contiguous(), xs[rows], w, ws))


def test_dense_rows_past_32_bits():
    """M K past 2^32: rows in parts."""
    g = torch.Generator(device=DEV).manual_seed(5)
    M, N, K = 270000, 64, 16384
    x = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device=DEV)
    xs = torch.rand((M,), generator=g, device=DEV)
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8, device=DEV)
    ws = torch.rand((N,), generator=g, device=DEV) * 1e-3
    y = W.int8_gemm(x, xs, w, ws)
    for rows in (slice(0, 40), slice(262144 - 300, 262144 + 40), slice(M - 40, M)):
        assert torch.equal(y[rows], W.int8_gemm(x[rows].contiguous(), xs[rows], w, ws))


def test_many_short_rows():
    x = torch.randn((5_000_000, 16), device=DEV, dtype=torch.float16)
    q, s = W.act_quant_int8(x)
    for at in (0, 4_999_000):
        rq, rs = O.quantise(f64(x[at:at + 1000]))
        assert np.array_equal(f64(q[at:at + 1000]), rq) and np.array_equal(s[at:at + 1000].cpu().numpy(), rs)


# ------------------------------------------------------------------ calls at once
def test_calls_on_two_streams():
    """Two layers, products and choices under way at once, each with workspaces of its own."""
    jobs = []
    for n, (T, E, k, H, I) in enumerate([(24, 32, 4, 512, 256), (300, 16, 2, 256, 320)]):
        g = gen(n, 42)
        w13, w2, s13, s2 = on(*make_layer(g, E, H, I))
        x = hidden(g, T, H, torch.bfloat16).to(DEV)
        l = torch.randn((T, E), generator=g).to(DEV)
        b = (torch.randn((E,), generator=g) * 0.1).to(DEV)
        wd, sd = on(*weight(g, 300, H))

        def job(x=x, l=l, b=b, w13=w13, w2=w2, s13=s13, s2=s2, wd=wd, sd=sd, k=k):
            tw, ids = W.route_topk(l, k, scoring="sigmoid", bias=b)
            y = W.moe_int8_apply(x, w13, w2, s13, s2, tw, ids)
            return [tw, ids, y, W.int8_gemm(y, None, wd, sd)]
        jobs.append((job, torch.cuda.Stream()))
    alone = [job() for job, _ in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for n, (job, stream) in enumerate(jobs):
            with torch.cuda.stream(stream):
                got[n].append(job())
    torch.cuda.synchronize()
    for n in range(2):
        for r in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(r, alone[n]))


def test_two_graphs_replayed_in_turn():
    E, k, H, I = 16, 2, 256, 128
    g = gen(43)
    w13, w2, s13, s2 = on(*make_layer(g, E, H, I))
    graphs = []
    for T in (3, 200):
        x = hidden(g, T, H, torch.bfloat16).to(DEV)
        l = torch.randn((T, E), generator=g).to(DEV)

        def step(x=x, l=l):
            tw, ids = W.route_topk(l, k)
            return W.moe_int8_apply(x, w13, w2, s13, s2, tw, ids)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, step, x, l))
    for _ in range(3):
        for graph, out, step, x, l in graphs:
            x.copy_(torch.randn(x.shape, generator=g))
            l.copy_(torch.randn(l.shape, generator=g))
            graph.replay()
        torch.cuda.synchronize()
        for graph, out, step, x, l in graphs:
            assert torch.equal(out, step())


# ------------------------------------------------------------------ arguments of other forms
def test_scales_and_ids_of_other_forms():
    g = gen(44)
    T, E, k, H, I = 12, 8, 2, 128, 64
    w13, w2, s13, s2 = make_layer(g, E, H, I)
    tw, ids = make_routing(g, T, E, k)
    x, xs = rows8(g, T, H)
    ref = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, ids), x_scales=xs.to(DEV))
    y = W.moe_int8_apply(*on(x, w13, w2, s13[..., None], s2[..., None], tw.double().reshape(-1), ids.long()), x_scales=xs[:, 0].to(DEV))
    assert torch.equal(y, ref)
    wide = torch.zeros((T, H + 16), dtype=torch.int8, device=DEV)
    wide[:, :H] = x.to(DEV)
    assert torch.equal(W.moe_int8_apply(wide[:, :H], *on(w13, w2, s13, s2, tw, ids), x_scales=xs.to(DEV)), ref)
    with pytest.raises(RuntimeError, match="aligned"):
        flat = torch.zeros((w2.numel() + 1,), dtype=torch.int8, device=DEV)
        W.moe_int8_apply(*on(x, w13), flat[1:].view(w2.shape), *on(s13, s2, tw, ids), x_scales=xs.to(DEV))


# ------------------------------------------------------------------ the choice
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top", [(256, 1, 1), (256, 8, 4), (64, 1, 1), (24, 1, 1)])
def test_scores_in_doubt(scoring, E, groups, top):
    """Experts whose c differ by a part of fp32's step, next to the last pick and among the picks."""
    g = gen(E, groups, 45)
    T = 64
    l = torch.randn((T, E), generator=g)
    p = torch.softmax(l.double(), 1) if scoring == "softmax" else torch.sigmoid(l.double())
    b = torch.randn((E,), generator=g) * 0.1
    # the bias of expert 2 i + 1 brings its c of token i to that of expert 2 i, to fp32's last bits
    for i in range(E // 2):
        t = i % T
        b[2 * i + 1] = float(p[t, 2 * i] + b[2 * i].double() - p[t, 2 * i + 1])
    for k in (1, 2, 5, 8):
        check_route(l, k, scoring, b, groups, top)
    # logits that are neighbours as fp32 numbers, without a bias
    base = torch.randn((T, E // 2), generator=g)
    pair = torch.stack([base, torch.nextafter(base, torch.full_like(base, 9.0))], 2).reshape(T, E)
    for k in (3, 8):
        check_route(pair, k, scoring, None, groups, top)
    check_route(pair[:, torch.randperm(E, generator=g)], 8, scoring, torch.zeros(E), groups, top)


def test_choice_of_rows_at_odd_places():
    g = gen(46)
    l = torch.randn((9, 300), generator=g).to(DEV)
    b = torch.randn((300,), generator=g).to(DEV)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        wide = l.to(dtype)
        for lo, E in ((1, 256), (3, 64), (16, 256), (7, 250)):
            part, bias = wide[:, lo:lo + E], b[lo:lo + E]
            got = W.route_topk(part, 8, scoring="sigmoid", bias=bias)
            want = W.route_topk(part.clone(), 8, scoring="sigmoid", bias=bias.clone())
            assert all(torch.equal(x, y) for x, y in zip(got, want))
            check_route(part.cpu(), 8, "sigmoid", bias.cpu())


@pytest.mark.parametrize("T", [1, 2, 3, 5, 15, 16, 17, 63, 65])
def test_choice_of_few_tokens_writes_no_more(T):
    l = torch.randn((T, 64), generator=gen(T)).bfloat16()
    check_route(l, 6, "sigmoid", torch.zeros(64), 4, 2)
