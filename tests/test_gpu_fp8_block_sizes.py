"""Block-scaled fp8 operators where their kernels can go wrong by size: every tile, long K, offsets past
32 bits, skewed and empty experts, padding, NaN, alignment, several streams and graphs.

Large products are checked on sampled rows and columns; tolerances are the oracle's."""
import numpy as np
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import fp8_block as O
from test_gpu_fp8_block import (DEV, FP8, assert_close, check_layer, f64, fp8_rows, fp8_weight, gen, hidden, layer_case,
                                on)

pytestmark = pytest.mark.gpu


def sample(n, count, g):
    """Indexes with both ends among them."""
    i = torch.randint(0, n, (count,), generator=g)
    i[0], i[-1] = 0, n - 1
    return i


def dev_fp8(*shape, seed=0):
    """e4m3 values made on the device (all codes but NaN)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    u = torch.randint(0, 0x7F, shape, generator=g, device=DEV, dtype=torch.uint8)
    return (u | torch.randint(0, 2, shape, generator=g, device=DEV, dtype=torch.uint8) << 7).view(FP8)


# ------------------------------------------------------------------ dense
# (M, N, K) for each tile on a card of 256 CUs: rows in registers, 64 x 64 with K in two, 64 x 64,
# 64 x 128, 256 x 128; K with and without a partial group, odd N
@pytest.mark.parametrize("M,N,K", [(7, 24600, 400), (16, 520, 4112), (12, 300, 8208), (17, 1001, 4096), (64, 70, 9232),
                                   (320, 4104, 272), (321, 4099, 384), (1000, 4096, 144), (999, 4101, 640),
                                   (2047, 4096, 128), (2040, 4090, 400), (2048, 4093, 896)])
def test_dense_tiles(M, N, K):
    g = gen(M, N, K)
    x, xs = fp8_rows(g, M, K)
    w, ws = fp8_weight(g, (), N, K)
    for dtype in (torch.bfloat16, torch.float16):
        out = W.fp8_block_gemm(*on(x, xs, w, ws), out_dtype=dtype)
        rows, cols = sample(M, 40, g), sample(N, 300, g).unique()
        wide = ws[cols // 128]                       # a block's scale for each sampled column
        ref, err = np.zeros((40, len(cols))), np.zeros((40, len(cols)))
        for c in range(-(-N // 128)):                # columns of one block share their scales
            at = torch.nonzero(cols // 128 == c).flatten()
            if len(at):
                r, e = O.product(f64(x[rows]), xs[rows].numpy(), f64(w[cols[at]]), wide[at[:1]].numpy())
                ref[:, at.numpy()], err[:, at.numpy()] = r, e
        assert_close(out[rows.to(DEV)][:, cols.to(DEV)], ref, err, dtype)
    assert torch.equal(out, W.fp8_block_gemm(*on(x, xs, w, ws), out_dtype=dtype))


@pytest.mark.parametrize("M", [3, 17])
def test_dense_long_k(M):
    """More groups of 128 than one table of weight scales holds."""
    N, K = 70, 128 * 400 + 48
    g = gen(M, N)
    x, xs = fp8_rows(g, M, K)
    w, ws = fp8_weight(g, (), N, K)
    ref, err = O.product(f64(x), xs.numpy(), f64(w), ws.numpy())
    assert_close(W.fp8_block_gemm(*on(x, xs, w, ws)), ref, err, torch.bfloat16)


def sampled_product(x, xs, w, ws, rows, cols):
    """Rows by columns of one weight block each."""
    ref = [O.product(f64(x[rows]), xs[rows].cpu().numpy(), f64(w[c:c + 1]), ws[c // 128:c // 128 + 1].cpu().numpy())
           for c in cols.tolist()]
    return np.concatenate([r for r, _ in ref], 1), np.concatenate([e for _, e in ref], 1)


def test_dense_offsets_past_32_bits():
    """Rows of more than 4 GiB (streamed), and more than 2^31 outputs (tiles)."""
    for M, N, K in ((1_048_700, 24, 4112), (140_000, 16392, 16)):
        x, xs = dev_fp8(M, K, seed=1), torch.rand((M, -(-K // 128)), device=DEV) * 0.01
        w, ws = dev_fp8(N, K, seed=2), torch.rand((-(-N // 128), -(-K // 128)), device=DEV) * 1e-3
        out = W.fp8_block_gemm(x, xs, w, ws)
        g = gen(M)
        rows, cols = sample(M, 24, g), sample(N, 12, g)
        ref, err = sampled_product(x, xs, w, ws, rows.to(DEV), cols)
        assert_close(out[rows.to(DEV)][:, cols.to(DEV)], ref, err, torch.bfloat16)
        del x, xs, w, out


def test_norm_and_quant_offsets_past_32_bits():
    T, H = 540_000, 4104
    x = torch.empty((T, H), dtype=torch.bfloat16, device=DEV)
    for t in range(0, T, 60_000):
        x[t:t + 60_000] = torch.randn((60_000, H), device=DEV)
    rows = sample(T, 16, gen(T)).to(DEV)
    nw = torch.ones((H,), dtype=torch.bfloat16, device=DEV)
    few = W.rms_norm_quant_fp8(x[rows], nw, residual=x[rows], return_norm=True)
    n = W.rms_norm_quant_fp8(x, nw, residual=x, return_norm=True)
    for a, b in zip(n, few):
        assert torch.equal(a.view(torch.uint8)[rows] if a.dtype == FP8 else a[rows], b.view(torch.uint8) if a.dtype == FP8 else b)
    del n
    q, s = W.act_quant_fp8_block(x)
    fq, fs = W.act_quant_fp8_block(x[rows])
    assert torch.equal(q.view(torch.uint8)[rows], fq.view(torch.uint8)) and torch.equal(s[rows], fs)
    q, s = W.act_quant_fp8_block(x, activation="silu")
    fq, fs = W.act_quant_fp8_block(x[rows], activation="silu")
    assert torch.equal(q.view(torch.uint8)[rows], fq.view(torch.uint8)) and torch.equal(s[rows], fs)


def test_dense_extreme_scales_and_rounding_to_16_bits():
    """Sums past fp16's range become infinities, tiny ones subnormal numbers or zeros; zero rows stay zero."""
    g = gen(3)
    x, xs = fp8_rows(g, 20, 256)
    w, ws = fp8_weight(g, (), 64, 256)
    xs[0], xs[1], xs[2] = 1e6, 1e-9, 0
    out = W.fp8_block_gemm(*on(x, xs, w, ws), out_dtype=torch.float16)
    ref, err = O.product(f64(x), xs.numpy(), f64(w), ws.numpy())
    over = np.abs(ref) > 70000
    assert over[0].any() and np.isinf(f64(out)[over]).all() and not out[2].any()
    inside = ~over & (np.abs(ref) < 65000)
    assert_close(out[torch.from_numpy(inside).to(DEV)], ref[inside], err[inside], torch.float16)


# ------------------------------------------------------------------ grouped
def check_rows(out, before, x, xs, w, ws, sti, eid, ntp, top_k, block, dtype, slots, gather=True):
    """check by expert; before: what rows that are padding hold."""
    sti, eid = sti.cpu(), eid.cpu()
    row = torch.arange(len(sti))
    e = eid[row // block].long()
    real = (row < ntp) & (sti >= 0) & (sti < slots) & (e >= 0) & (e < w.shape[0])
    assert torch.equal(out.cpu()[~real], before[~real])
    for i in torch.unique(e[real]).tolist():
        at = row[real & (e == i)]
        src = sti[at].long() // top_k if gather else at
        ref, err = O.product(f64(x[src]), xs[src].numpy(), f64(w[i]), ws[i].numpy())
        assert_close(out[at.to(DEV)], ref, err, dtype)


# blocks of 16 whose tiles hold several experts, K tails, more rows than a tile, long K, wide blocks
@pytest.mark.parametrize("T,k,E,N,K,block,skew", [(300, 2, 4, 130, 272, 16, True), (257, 4, 5, 256, 400, 16, False),
                                                  (90, 3, 16, 129, 144, 64, True), (500, 2, 3, 384, 128, 128, True),
                                                  (70, 1, 2, 64, 128 * 200 + 16, 64, False), (1, 8, 64, 264, 2048, 64, False),
                                                  (1, 1, 2, 128, 128, 128, False), (400, 6, 8, 40, 1040, 48, True),
                                                  (33, 2, 200, 72, 4112, 32, True)])
def test_group_tiles(T, k, E, N, K, block, skew):
    g = gen(T, k, E, N, K, 1)
    x, xs = fp8_rows(g, T, K)
    w, ws = fp8_weight(g, (E,), N, K)
    p = torch.rand((T, E), generator=g)
    if skew:
        p[:, 1] += 0.7                               # most tokens; and nobody comes to the last expert
        p[:, E - 1] = -1 if k < E else 0
    ids = p.argsort(1, descending=True)[:, :k].to(torch.int32)
    sti, eid, ntp = W.moe_align_block_size(ids.to(DEV), block, E)
    dtype = torch.bfloat16
    before = torch.full((sti.numel(), N), 7.0, dtype=dtype)
    out = before.to(DEV)
    d = on(x, xs, w, ws)
    W.moe_fp8_block_gemm(*d, sti, eid, ntp, k, block, out=out)
    check_rows(out, before, x, xs, w, ws, sti, eid, int(ntp), k, block, dtype, T * k)
    # an output that starts between two 8-byte words, the same rows again
    flat = torch.full((sti.numel() * N + 1,), 7.0, dtype=dtype, device=DEV)
    W.moe_fp8_block_gemm(*d, sti, eid, ntp, k, block, out=flat[1:].view(-1, N))
    assert torch.equal(flat[1:].view(-1, N), out) and flat[0] == 7.0


@pytest.mark.parametrize("T,block", [(4, 16), (300, 16), (40, 64)])
def test_second_product_leaves_padding(T, block):
    """Two grouped products, the second reading the rows of the first in place: with num_slots its
    padding rows stay as they were."""
    g = gen(T, block)
    k, E, N, K = 2, 4, 256, 256
    x, xs = fp8_rows(g, T, K)
    w, ws = fp8_weight(g, (E,), N, K)
    w2, ws2 = fp8_weight(g, (E,), 72, N)
    ids = torch.rand((T, E), generator=g).argsort(1)[:, :k].to(torch.int32)
    sti, eid, ntp = W.moe_align_block_size(ids.to(DEV), block, E)
    P = sti.numel()
    mid = torch.zeros((P, N), dtype=torch.bfloat16, device=DEV)
    W.moe_fp8_block_gemm(*on(x, xs, w, ws), sti, eid, ntp, k, block, out=mid)
    q, s = W.act_quant_fp8_block(mid)
    before = torch.full((P, 72), 5.0, dtype=torch.bfloat16)
    out = before.to(DEV)
    W.moe_fp8_block_gemm(q, s, *on(w2, ws2), sti, eid, ntp, 1, block, out=out, gather=False, num_slots=T * k)
    check_rows(out, before, q.cpu(), s.cpu(), w2, ws2, sti, eid, int(ntp), 1, block, torch.bfloat16, T * k, gather=False)
    with pytest.raises(RuntimeError, match="num_slots"):
        W.moe_fp8_block_gemm(*on(x, xs, w, ws), sti, eid, ntp, k, block, num_slots=T * k + 1)


@pytest.mark.parametrize("T,block", [(3, 16), (60, 64)])
def test_group_weights_past_32_bits(T, block):
    """The last of 256 experts starts at 8.5 GB."""
    E, N, K = 256, 4096, 8192
    w, ws = torch.zeros((E, N, K), dtype=torch.uint8, device=DEV).view(FP8), torch.ones((E, N // 128, K // 128), device=DEV)
    w[E - 1], w[0] = dev_fp8(N, K, seed=3), dev_fp8(N, K, seed=4)
    ws *= 1e-3
    x, xs = fp8_rows(gen(T), T, K)
    ids = torch.full((T, 1), E - 1, dtype=torch.int32)
    ids[0] = 0
    sti, eid, ntp = W.moe_align_block_size(ids.to(DEV), block, E)
    out = W.moe_fp8_block_gemm(*on(x, xs), w, ws, sti, eid, ntp, 1, block)
    cols = sample(N, 12, gen(T, 1))
    sti = sti.cpu()
    for t in range(T):
        r = int(torch.nonzero(sti == t)[0])
        e = int(ids[t])
        ref, err = sampled_product(x, xs, w[e], ws[e], torch.tensor([t]), cols)
        assert_close(out[r:r + 1][:, cols.to(DEV)], ref, err, torch.bfloat16)


# ------------------------------------------------------------------ layer
@pytest.mark.parametrize("T,k,E,H,I", [(40, 2, 8, 256, 256), (49, 2, 8, 256, 256), (300, 3, 5, 384, 128),
                                       (2, 8, 300, 128, 128), (300, 1, 1, 128, 384)])
def test_layer_skew_repeats_and_nobody(T, k, E, H, I):
    """All tokens to one expert, a token that names an expert twice, tokens of no expert."""
    x, w13, s13, w2, s2, tw, ids = layer_case(T, k, E, H, I, torch.bfloat16, 3)
    ids[:, 0] = 0
    ids[T // 2:, k - 1] = ids[T // 2:, 0]
    ids[1] = -1
    out = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids))
    check_layer(out, x, w13, s13, w2, s2, tw, ids, torch.bfloat16)
    assert not out[1].any()
    none = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, torch.full_like(ids, -1)))
    assert not none.any()


@pytest.mark.parametrize("T", [3, 40])
def test_layer_long_rows(T):
    """More groups of 128 than one table of weight scales holds, in both products."""
    x, w13, s13, w2, s2, tw, ids = layer_case(T, 1, 1, 128 * 200, 128, torch.bfloat16, 4)
    check_layer(W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids)), x, w13, s13, w2, s2, tw, ids, torch.bfloat16)
    x, w13, s13, w2, s2, tw, ids = layer_case(T, 1, 1, 128, 128 * 200, torch.bfloat16, 4)
    check_layer(W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids)), x, w13, s13, w2, s2, tw, ids, torch.bfloat16)


@pytest.mark.parametrize("T", [4, 130])
def test_layer_nan_stays_in_its_token(T):
    x, w13, s13, w2, s2, tw, ids = layer_case(T, 2, 4, 256, 128, torch.bfloat16, 9)
    clean = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids))
    x[2, 100] = float("nan")
    x[0, 5] = float("nan")
    out = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids))
    rest = [t for t in range(T) if t not in (0, 2)]
    assert out[0].isnan().all() and out[2].isnan().all() and torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("T", [5, 200])
def test_layer_strided_inputs(T):
    x, w13, s13, w2, s2, tw, ids = layer_case(T, 2, 4, 256, 128, torch.float16, 6)
    want = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids))
    wide = torch.zeros((T, 300), dtype=torch.float16, device=DEV)
    wide[:, 3:259] = x.to(DEV)
    tws, idl = torch.zeros((T, 4), device=DEV), torch.zeros((T, 4), dtype=torch.int64, device=DEV)
    tws[:, ::2], idl[:, ::2] = tw.to(DEV), ids.to(DEV).long()
    got = W.moe_fp8_block_apply(wide[:, 3:259], *on(w13, w2, s13, s2), tws[:, ::2], idl[:, ::2])
    assert torch.equal(got, want)


# ------------------------------------------------------------------ streams and graphs
def test_two_graphs_and_two_streams_at_once():
    """Two captured layers replayed at the same time on two streams, beside eager calls of both."""
    cases = [layer_case(T, 2, 6, 256, 128, torch.bfloat16, T) for T in (5, 150)]
    args = [on(x, w13, w2, s13, s2, tw, ids) for x, w13, s13, w2, s2, tw, ids in cases]

    def run(a):
        y = W.moe_fp8_block_apply(*a)
        return y, W.fp8_block_gemm(y, None, a[1][0], a[3][0])

    want = [run(a) for a in args]
    graphs, held = [], []
    for a in args:
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(run(a))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        torch.cuda.synchronize()
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        eager = [run(a) for a in args]
        torch.cuda.synchronize()
        for h, e, w in zip(held, eager, want):
            for i in range(2):
                assert torch.equal(h[i], w[i]) and torch.equal(e[i], w[i])
                h[i].zero_()
