"""Block-scaled fp8 operators on the GPU against their float64 restatement (oracle/fp8_block.py).

Tolerances are the oracle's: fp32 sums are held to a bound that counts their roundings, 16-bit
outputs to half a step more, quantised values to what those errors can move."""
import numpy as np
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import fp8_block as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a step, relative


def f64(t):
    return t.float().cpu().numpy().astype(np.float64)


def round16(dtype):
    return lambda v: torch.from_numpy(v.astype(np.float32)).to(dtype).float().numpy().astype(np.float64)


def hidden(g, rows, K, dtype, scale=1.0):
    """Normal values, some channels eight times as wide."""
    x = torch.randn((rows, K), generator=g) * scale
    x *= torch.where(torch.rand((K,), generator=g) < 1 / 16, 8.0, 1.0)
    return x.to(dtype)


def gen(*parts):
    return torch.Generator().manual_seed(hash(parts) % (1 << 31))


def fp8_rows(g, rows, K):
    """e4m3 rows and scales whose groups have sizes of their own."""
    x = torch.randn((rows, K), generator=g).mul(60).clamp(-448, 448).to(FP8)
    s = torch.rand((rows, -(-K // 128)), generator=g) * 0.02 + 0.001
    return x, s


def fp8_weight(g, lead, N, K):
    w = torch.randn((*lead, N, K), generator=g).mul(60).clamp(-448, 448).to(FP8)
    s = torch.rand((*lead, -(-N // 128), -(-K // 128)), generator=g) * 2e-4 + 1e-5
    return w, s


def on(*ts):
    return [t.to(DEV) if t is not None else None for t in ts]


def assert_close(got, ref, tol, dtype=None):
    got = f64(got)
    t = tol + (np.abs(ref) + tol) * HALF[dtype] if dtype is not None else tol
    if dtype == torch.float16:
        t = t + 2.0 ** -25              # half a step of its subnormal numbers
    bad = ~(np.abs(got - ref) <= t)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst by {np.nanmax(np.abs(got - ref) / t):.3g} tolerances"


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 8), (3, 127), (2, 128), (5, 129), (7, 136), (33, 512),
                                    (4, 1000), (2, 4096), (257, 272), (3, 20000)])
def test_act_quant_is_exact(rows, K, dtype):
    x = hidden(gen(rows, K), rows, K, dtype)
    x[0] = 0                                     # the scale's floor
    q, s = W.act_quant_fp8_block(x.to(DEV))
    rq, rs = O.quantise(f64(x))
    assert q.dtype == FP8 and tuple(s.shape) == rs.shape
    assert np.array_equal(s.cpu().numpy(), rs)
    assert np.array_equal(f64(q), rq)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,K", [(1, 8), (3, 100), (2, 128), (9, 512), (5, 1001), (64, 1536)])
def test_silu_quant(rows, K, dtype):
    x = hidden(gen(rows, K, 1), rows, 2 * K, dtype, 2.0)
    q, s = W.act_quant_fp8_block(x.to(DEV), activation="silu")
    v = f64(x)
    g, u = v[:, :K], v[:, K:]
    h = O.silu_mul(g, u)
    dh = np.abs(h) * (2 * np.abs(g) + 8) * O.U32
    rs = O.group_scales(h).astype(np.float64)
    assert np.all(np.abs(s.cpu().numpy() - rs) <= rs * (2 * 90 + 8) * O.U32 * 2)
    each = O.spread(s.cpu().numpy().astype(np.float64), K)
    u = h / each
    du = dh / each + np.abs(u) * 4 * O.U32
    lo, hi = O.round_e4m3(u - du), O.round_e4m3(u + du)
    got = f64(q)
    assert np.all((got >= lo) & (got <= hi))


@pytest.mark.parametrize("silu", [False, True])
def test_quant_of_strided_rows_and_one_row(silu):
    base = hidden(gen(4), 6, 1100, torch.bfloat16).to(DEV)
    for view in (base[:, 8:520], base[::2, 3:515], base[1:2, :512], base.t()[:512].t()):
        a = W.act_quant_fp8_block(view, "silu" if silu else None)
        b = W.act_quant_fp8_block(view.contiguous(), "silu" if silu else None)
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


def test_quant_nan_and_infinity():
    x = torch.ones((3, 256), dtype=torch.float16)
    x[0, 5] = float("nan")
    x[1, 130] = float("inf")
    q, s = W.act_quant_fp8_block(x.to(DEV))
    v, sc = f64(q), s.cpu().numpy()
    assert np.isnan(v[0, 5]) and np.isnan(v[0]).sum() == 1 and np.isfinite(sc[0]).all()
    assert np.isinf(sc[1, 1]) and np.isfinite(sc[1, 0])
    assert np.isnan(v[1, 130]) and not v[1, 131:].any()
    assert np.isfinite(v[2]).all()


# ------------------------------------------------------------------ norm
def check_norm(x, r, w, eps, per_row, keep, got):
    dtype, H = x.dtype, x.shape[1]
    z, y = O.norm(f64(x), None if r is None else f64(r), f64(w), eps, round16(dtype))
    if r is not None:
        # (the fp32 sum before it is rounded to 16 bits is exact unless one number is 2^12 times the
        # other, and then it is off by less than decides between two 16-bit neighbours)
        assert np.array_equal(f64(got.residual), z)
    else:
        assert got.residual is None
    rel = O.norm_rel(H)
    if keep:
        assert_close(got.norm, y, np.abs(y) * rel, dtype)
    else:
        assert got.norm is None
    size = H if per_row else 128
    s = got.scales.cpu().numpy().astype(np.float64)
    rs = O.group_scales(y, size).astype(np.float64)
    assert s.shape == rs.shape and np.all(np.abs(s - rs) <= rs * (rel + 3 * O.U32))
    u = y / np.repeat(s, size, axis=1)[:, :H]
    du = np.abs(u) * (rel + 4 * O.U32)
    q = f64(got.q)
    assert np.all((q >= O.round_e4m3(u - du)) & (q <= O.round_e4m3(u + du)))


@pytest.mark.parametrize("dtype,wf32", [(torch.bfloat16, False), (torch.float16, True)])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 8), (2, 127), (5, 256), (6, 512), (3, 520), (2, 1000),
                                 (3, 2048), (2, 2056), (1, 4096), (2, 4104), (3, 8192), (2, 8200),
                                 (1, 16384), (2, 16392), (3, 2049)])
def test_norm(T, H, dtype, wf32):
    for n, (res, per_row, keep) in enumerate(((True, False, True), (False, True, False), (True, True, False),
                                              (False, False, True))):
        g = gen(T, H, n)
        x, r = hidden(g, T, H, dtype), hidden(g, T, H, dtype) if res else None
        w = (torch.randn((H,), generator=g) * 0.2 + 1).to(torch.float32 if wf32 else dtype)
        got = W.rms_norm_quant_fp8(x.to(DEV), w.to(DEV), 1e-5, residual=None if r is None else r.to(DEV),
                                   group_size=0 if per_row else 128, return_norm=keep)
        check_norm(x, r, w, 1e-5, per_row, keep, got)


def test_norm_strided_zero_rows_and_nan():
    g = gen(9)
    base, rb = hidden(g, 8, 1040, torch.bfloat16), hidden(g, 8, 2000, torch.bfloat16)
    w = torch.ones((1024,), dtype=torch.bfloat16)
    for xs, rs in ((base[:, 8:1032], rb[:, 16:1040]), (base[::2, 1:1025], rb[::2, :1024])):
        got = W.rms_norm_quant_fp8(xs.to(DEV), w.to(DEV), 1e-6, residual=rs.to(DEV))
        d = base.to(DEV), rb.to(DEV)
        dx = d[0][:, 8:1032] if xs.shape[0] == 8 else d[0][::2, 1:1025]
        dr = d[1][:, 16:1040] if xs.shape[0] == 8 else d[1][::2, :1024]
        strided = W.rms_norm_quant_fp8(dx, w.to(DEV), 1e-6, residual=dr)
        check_norm(xs, rs, w, 1e-6, False, False, strided)
        assert torch.equal(got.q.view(torch.uint8), strided.q.view(torch.uint8))
    x = torch.zeros((3, 1024), dtype=torch.float16)
    x[1, 7] = float("nan")
    x[2] = 1
    n = W.rms_norm_quant_fp8(x.to(DEV), torch.ones(1024, dtype=torch.float16, device=DEV))
    v, s = f64(n.q), n.scales.cpu().numpy()
    assert not v[0].any() and np.all(s[:2] == np.float32(1e-8))
    assert np.isnan(v[1]).all() and np.isfinite(v[2]).all()


def test_norm_leaves_its_inputs():
    x, r = hidden(gen(1), 4, 640, torch.float16).to(DEV), hidden(gen(2), 4, 640, torch.float16).to(DEV)
    a, b = x.clone(), r.clone()
    W.rms_norm_quant_fp8(x, torch.ones(640, dtype=torch.float16, device=DEV), residual=r)
    assert torch.equal(x, a) and torch.equal(r, b)


# ------------------------------------------------------------------ dense
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 16, 128), (1, 128, 256), (2, 40, 144), (15, 130, 1040),
                                   (16, 256, 512), (17, 64, 384), (33, 100, 2048), (64, 129, 272),
                                   (65, 384, 640), (100, 250, 1152), (129, 520, 128), (300, 300, 400)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_dense(M, N, K, dtype):
    g = gen(M, N, K)
    x, xs = fp8_rows(g, M, K)
    w, ws = fp8_weight(g, (), N, K)
    out = W.fp8_block_gemm(*on(x, xs, w, ws), out_dtype=dtype)
    ref, err = O.product(f64(x), xs.numpy(), f64(w), ws.numpy())
    assert out.dtype == dtype
    assert_close(out, ref, err, dtype)


@pytest.mark.parametrize("M,N,K", [(1, 48, 128), (3, 200, 400), (16, 128, 1024), (40, 136, 272), (130, 260, 512)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_dense_from_16_bit_rows(M, N, K, dtype):
    g = gen(M, N, K, 3)
    x = hidden(g, M, K, dtype)
    w, ws = fp8_weight(g, (), N, K)
    dx, dw, dws = on(x, w, ws)
    out = W.fp8_block_gemm(dx, None, dw, dws)
    xq, xs = O.quantise(f64(x))
    ref, err = O.product(xq, xs, f64(w), ws.numpy())
    assert out.dtype == dtype
    assert_close(out, ref, err, dtype)
    # the rows that act_quant_fp8_block makes give the same values within the sums' bound
    q, s = W.act_quant_fp8_block(dx)
    assert_close(W.fp8_block_gemm(q, s, dw, dws, out_dtype=dtype), ref, err, dtype)


def test_dense_strided_and_misaligned_rows():
    g = gen(21)
    x, _ = fp8_rows(g, 40, 600)
    w, ws = fp8_weight(g, (), 96, 256)
    xs = torch.rand((20, 2), generator=g) * 0.01
    dx, dw, dws, dxs = on(x, w, ws, xs)
    for view in (dx[:20, :256], dx[:20, 16:272], dx[::2, 3:259], dx[:20, 1:257], dx.t()[:256, :20].t()):
        out = W.fp8_block_gemm(view, dxs, dw, dws)
        ref, err = O.product(f64(view), xs.numpy(), f64(w), ws.numpy())
        assert_close(out, ref, err, torch.bfloat16)


def test_dense_nan_stays_in_its_row_and_column():
    """A NaN of x marks its row, one of w its column; K tails next to NaN bytes add nothing."""
    g = gen(22)
    x, xs = fp8_rows(g, 20, 144)
    w, ws = fp8_weight(g, (), 70, 144)
    x.view(torch.uint8)[3, 140] = 0x7F
    w.view(torch.uint8)[66, 5] = 0xFF
    out = f64(W.fp8_block_gemm(*on(x, xs, w, ws)))
    nan = np.isnan(out)
    want = np.zeros_like(nan)
    want[3] = True
    want[:, 66] = True
    assert np.array_equal(nan, want)


def test_dense_no_rows():
    w, ws = on(*fp8_weight(gen(1), (), 64, 128))
    x = torch.empty((0, 128), dtype=FP8, device=DEV)
    assert W.fp8_block_gemm(x, torch.empty((0, 1), device=DEV), w, ws).shape == (0, 64)
    assert W.rms_norm_quant_fp8(torch.empty((0, 128), dtype=torch.float16, device=DEV),
                                torch.ones(128, dtype=torch.float16, device=DEV)).q.shape == (0, 128)
    assert W.act_quant_fp8_block(torch.empty((0, 128), dtype=torch.float16, device=DEV))[0].shape == (0, 128)


# ------------------------------------------------------------------ grouped
def check_group(out, before, x, xs, w, ws, sti, eid, ntp, top_k, block, dtype, gather=True):
    sti, eid = sti.cpu().numpy(), eid.cpu().numpy()
    xv, wv, before = f64(x), f64(w), f64(before)
    slots = x.shape[0] * top_k
    ref, tol = before.copy(), np.zeros_like(before)
    real = np.zeros(len(sti), bool)
    for b in range(len(sti) // block):
        e = eid[b]
        if b * block >= ntp or not 0 <= e < w.shape[0]:
            continue
        for r in range(b * block, min((b + 1) * block, ntp)):
            if gather and sti[r] >= slots or not gather and sti[r] >= max(slots, len(sti)):
                continue
            real[r] = True
            i = sti[r] // top_k if gather else r
            y, err = O.product(xv[i:i + 1], xs[i:i + 1].numpy(), wv[e], ws[e].numpy())
            ref[r], tol[r] = y[0], err[0]
    assert np.array_equal(f64(out)[~real], before[~real])
    assert_close(out[torch.from_numpy(real).to(out.device)], ref[real], tol[real], dtype)


@pytest.mark.parametrize("T,k,E,N,K,block", [(1, 1, 1, 16, 128, 16), (3, 2, 4, 48, 256, 16), (24, 4, 16, 130, 272, 16),
                                             (50, 2, 3, 128, 384, 64), (97, 3, 8, 200, 128, 64),
                                             (130, 1, 2, 72, 640, 128), (40, 6, 64, 256, 512, 32),
                                             (200, 2, 5, 264, 144, 48)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_group(T, k, E, N, K, block, dtype):
    g = gen(T, k, E, N, K)
    x, xs = fp8_rows(g, T, K)
    w, ws = fp8_weight(g, (E,), N, K)
    ids = torch.rand((T, E), generator=g).argsort(1)[:, :k].to(torch.int32)
    if E > 3:
        ids[ids == 2] = 1                           # an expert without rows, another twice in a token
    sti, eid, ntp = W.moe_align_block_size(ids.to(DEV), block, E)
    before = torch.full((sti.numel(), N), 7.0, dtype=dtype)
    out = before.to(DEV)
    dx, dxs, dw, dws = on(x, xs, w, ws)
    got = W.moe_fp8_block_gemm(dx, dxs, dw, dws, sti, eid, ntp, k, block, out=out)
    assert got.data_ptr() == out.data_ptr()
    check_group(out, before, x, xs, w, ws, sti, eid, int(ntp), k, block, dtype)
    fresh = W.moe_fp8_block_gemm(dx, dxs, dw, dws, sti, eid, ntp, k, block, out_dtype=dtype)
    real = (out != 7.0).any(1)
    assert torch.equal(fresh[real], out[real])


def test_group_rows_by_identity_and_foreign_ids():
    """gather=False reads row r; ids past the slots, experts that are not there and rows past the
    count are left alone."""
    g = gen(31)
    P, N, K, E, block = 96, 80, 256, 3, 16
    x, xs = fp8_rows(g, P, K)
    w, ws = fp8_weight(g, (E,), N, K)
    sti = torch.arange(P, dtype=torch.int32)
    sti[5], sti[17], sti[40] = 1 << 30, -1, P
    eid = torch.tensor([0, 2, 7, -1, 1, 1], dtype=torch.int32)
    before = torch.full((P, N), 3.0, dtype=torch.bfloat16)
    for ntp in (0, 1, 70, 96, 1000):
        out = before.to(DEV)
        W.moe_fp8_block_gemm(*on(x, xs, w, ws, sti, eid, torch.tensor([ntp], dtype=torch.int32)), 1, block,
                             out=out, gather=False)
        s = sti.clone()
        s[17] = 1 << 30
        check_group(out, before, x, xs, w, ws, s, eid, min(ntp, P), 1, block, torch.bfloat16, gather=False)


# ------------------------------------------------------------------ layer
def layer_case(T, k, E, H, I, dtype, seed=0):
    g = gen(T, k, E, H, I, seed)
    x = hidden(g, T, H, dtype)
    w13, s13 = fp8_weight(g, (E,), 2 * I, H)
    w2, s2 = fp8_weight(g, (E,), H, I)
    tw = torch.rand((T, k), generator=g) + 0.1
    ids = torch.rand((T, E), generator=g).argsort(1)[:, :k].to(torch.int32)
    return x, w13, s13, w2, s2, tw, ids


def check_layer(out, x, w13, s13, w2, s2, tw, ids, dtype, q=None):
    xq, xs = O.quantise(f64(x)) if q is None else (f64(q[0]), q[1].cpu().numpy())
    ref, tol = O.layer(xq, xs, f64(w13), s13.numpy(), f64(w2), s2.numpy(), tw.numpy(), ids.numpy(), HALF[dtype])
    assert_close(out, ref, tol, dtype)


@pytest.mark.parametrize("T,k,E,H,I", [(1, 1, 1, 128, 128), (1, 2, 8, 256, 128), (5, 2, 4, 384, 256), (33, 4, 16, 256, 128),
                                       (96, 2, 6, 128, 384), (97, 2, 6, 256, 256), (150, 3, 4, 512, 128),
                                       (400, 2, 3, 256, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer(T, k, E, H, I, dtype):
    x, w13, s13, w2, s2, tw, ids = layer_case(T, k, E, H, I, dtype)
    out = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids))
    assert out.dtype == dtype
    check_layer(out, x, w13, s13, w2, s2, tw, ids, dtype)


@pytest.mark.parametrize("T", [4, 120])
def test_layer_expert_map(T):
    """Global ids mapped to local experts; ids of experts that live elsewhere, and ids that do not
    exist, contribute nothing."""
    x, w13, s13, w2, s2, tw, _ = layer_case(T, 3, 4, 256, 128, torch.bfloat16, 5)
    g = gen(T, 6)
    ids = torch.randint(0, 10, (T, 3), generator=g, dtype=torch.int32)
    ids[1, 0] = 10
    ids[2] = 9                                      # nothing local: a row of zeros
    emap = torch.tensor([-1, 0, -1, 3, 1, -1, -1, 2, -1, -1], dtype=torch.int32)
    local = torch.where(ids < 10, emap[ids.clamp_max(9).long()], torch.tensor(-1)).to(torch.int32)
    out = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids), expert_map=emap.to(DEV), global_num_experts=10)
    check_layer(out, x, w13, s13, w2, s2, tw, local, torch.bfloat16)
    assert not out[2].any()


def test_decoder_half_as_used():
    """Norm with the residual, router, expert layer and a dense layer on the norm's e4m3 rows."""
    g = gen(77)
    T, H, I, E, k = 21, 256, 128, 8, 2
    x, r = hidden(g, T, H, torch.bfloat16), hidden(g, T, H, torch.bfloat16)
    nw = (torch.randn((H,), generator=g) * 0.2 + 1).to(torch.bfloat16)
    _, w13, s13, w2, s2, _, _ = layer_case(T, k, E, H, I, torch.bfloat16)
    wd, sd = fp8_weight(g, (), 192, H)
    rw = torch.randn((H, E), generator=g)
    dx, dr, dnw, dw13, ds13, dw2, ds2, dwd, dsd, drw = on(x, r, nw, w13, s13, w2, s2, wd, sd, rw)
    n = W.rms_norm_quant_fp8(dx, dnw, residual=dr, return_norm=True)
    tw, ids = W.fused_topk(None, n.norm.float() @ drw, k)
    y = W.moe_fp8_block_apply(n.q, dw13, dw2, ds13, ds2, tw, ids, x_scales=n.scales)
    d = W.fp8_block_gemm(n.q, n.scales, dwd, dsd)
    check_norm(x, r, nw, 1e-6, False, True, n)
    check_layer(y, x, w13, s13, w2, s2, tw.cpu(), ids.cpu(), torch.bfloat16, q=(n.q, n.scales))
    ref, err = O.product(f64(n.q), n.scales.cpu().numpy(), f64(wd), sd.numpy())
    assert_close(d, ref, err, torch.bfloat16)


@pytest.mark.parametrize("T", [3, 130])
def test_graph_replays_and_streams(T):
    """The run above in a graph, replayed on new inputs between eager calls, and on another stream."""
    x, w13, s13, w2, s2, tw, ids = layer_case(T, 2, 6, 256, 128, torch.bfloat16, 8)
    dx, dw13, ds13, dw2, ds2, dtw, dids = on(x, w13, s13, w2, s2, tw, ids)
    nw = torch.ones(256, dtype=torch.bfloat16, device=DEV)

    def step():
        n = W.rms_norm_quant_fp8(dx, nw, residual=dx, return_norm=True)
        y = W.moe_fp8_block_apply(n.q, dw13, dw2, ds13, ds2, dtw, dids, x_scales=n.scales)
        h = W.act_quant_fp8_block(y)
        return n.q.view(torch.uint8), y, W.fp8_block_gemm(h[0], h[1], dw13[0], ds13[0])

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(3):
        dx.copy_(hidden(gen(T, turn), T, 256, torch.bfloat16))
        dids.copy_(torch.rand((T, 6), generator=gen(T, turn, 1)).argsort(1)[:, :2].to(torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    for a, b in zip(held, other):
        assert torch.equal(a, b)


def test_torch_ops():
    g = gen(55)
    x, w13, s13, w2, s2, tw, ids = on(*layer_case(6, 2, 4, 256, 128, torch.float16))
    ops = torch.ops.w4a8_fp8_wmma
    nw = torch.ones(256, dtype=torch.float16, device=DEV)
    q, s, z, y = ops.rms_norm_quant_fp8(x, nw, 1e-6, None, 128, True)
    n = W.rms_norm_quant_fp8(x, nw, return_norm=True)
    assert torch.equal(q.view(torch.uint8), n.q.view(torch.uint8)) and z.numel() == 0 and torch.equal(y, n.norm)
    out = ops.moe_fp8_block_apply(q, w13, w2, s13, s2, tw, ids, s, None, torch.float16)
    assert torch.equal(out, W.moe_fp8_block_apply(q, w13, w2, s13, s2, tw, ids, x_scales=s, out_dtype=torch.float16))
    q2, sc2 = ops.act_quant_fp8_block(out, None)
    assert torch.equal(ops.fp8_block_gemm(q2, sc2, w13[0], s13[0], torch.bfloat16),
                       W.fp8_block_gemm(q2, sc2, w13[0], s13[0]))
    sti, eid, ntp = W.moe_align_block_size(ids, 16, 4)
    a = ops.moe_fp8_block_gemm(q, s, w13, s13, sti, eid, ntp, 2, 16, torch.bfloat16)
    b = W.moe_fp8_block_gemm(q, s, w13, s13, sti, eid, ntp, 2, 16)
    real = sti < 12
    assert torch.equal(a[real], b[real])
