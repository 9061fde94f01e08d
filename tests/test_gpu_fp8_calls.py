"""Block-scaled fp8 operators called in ways that the interface allows and that are not a model's usual ones:
outputs in place of inputs, more than eight slots a token, ids of nothing, no rows, fp16 layers with NaN."""
import numpy as np
import pytest
import torch

import fp8_layer_check as C
import test_gpu_fp8_block_sizes as S
import w4a8_fp8_wmma as W
from oracle import fp8_block as O
from test_gpu_fp8_block import check_layer, check_norm, f64, fp8_rows, fp8_weight, gen, hidden, layer_case, on
from test_gpu_fp8_layer_error import args_of, rows_of
from w4a8_fp8_wmma._lib import check, lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn


@pytest.mark.parametrize("H", [256, 1024, 4096, 8192, 16384, 1001, 16392])
@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_in_place(H, per_row, dtype):
    """residual_out in place of the residual or of x, norm_out in place of x: the same bits as apart."""
    g = gen(H, 5)
    T = 9
    x, r = hidden(g, T, H, dtype).to(DEV), hidden(g, T, H, dtype).to(DEV)
    w = (torch.randn((H,), generator=g) * 0.2 + 1).to(DEV)
    size = 0 if per_row else 128
    for res in (False, True):
        want = W.rms_norm_quant_fp8(x, w, 1e-6, residual=r if res else None, group_size=size, return_norm=True)
        places = [(None, True)] if not res else [("r", True), ("r", False), ("x", False)]
        for place, norm in places:
            a, b = x.clone(), r.clone()
            q, s = torch.empty_like(want.q), torch.empty_like(want.scales)
            z = {None: None, "r": b, "x": a}[place]
            check(lib.w4a8_rms_norm_quant_fp8(
                a.data_ptr(), 1 if dtype == torch.bfloat16 else 0, T, H, H, b.data_ptr() if res else None, H, w.data_ptr(),
                1, 1e-6, 1 if per_row else 0, z.data_ptr() if res else None, a.data_ptr() if norm else None, q.data_ptr(),
                s.data_ptr(), torch.cuda.current_stream().cuda_stream), "rms_norm_quant_fp8")
            assert torch.equal(q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(s, want.scales)
            assert z is None or torch.equal(z, want.residual)
            assert not norm or torch.equal(a, want.norm)


@pytest.mark.parametrize("H", [512, 4104, 777])
def test_norm_bf16_rows_with_fp32_weight(H):
    g = gen(H, 6)
    x, r = hidden(g, 3, H, torch.bfloat16), hidden(g, 3, H, torch.bfloat16)
    w = torch.randn((H,), generator=g) * 0.2 + 1
    check_norm(x, r, w, 1e-6, False, True, W.rms_norm_quant_fp8(*on(x, w), 1e-6, residual=r.to(DEV), return_norm=True))


@pytest.mark.parametrize("T", [10, 60])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_of_more_than_eight_slots(T, dtype):
    case = C.exact_case(T, 11, 12, 256, 128)
    tiles = T * 11 > 12 * 12
    out = W.moe_fp8_block_apply(rows_of(case, dtype, False)[0], *args_of(case))
    half = C.ROW_HALF if tiles and dtype == torch.bfloat16 else 0.0
    assert C.complaints(out.double().cpu().numpy(), dtype, O.known_layer(*case, half)) == []


@pytest.mark.parametrize("T,k,E,H,I", [(49, 2, 8, 256, 256), (300, 3, 5, 384, 128), (2, 8, 300, 128, 128)])
def test_fp16_layer_skew_repeats_and_nobody(T, k, E, H, I):
    x, w13, s13, w2, s2, tw, ids = layer_case(T, k, E, H, I, torch.float16, 3)
    ids[:, 0] = 0
    ids[T // 2:, k - 1] = ids[T // 2:, 0]
    ids[1] = -1
    out = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids))
    check_layer(out, x, w13, s13, w2, s2, tw, ids, torch.float16)
    assert not out[1].any()
    assert not W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, torch.full_like(ids, -1))).any()


@pytest.mark.parametrize("T", [4, 130])
def test_fp16_layer_nan_stays_in_its_token(T):
    x, w13, s13, w2, s2, tw, ids = layer_case(T, 2, 4, 256, 128, torch.float16, 9)
    clean = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids))
    x[2, 100] = x[0, 5] = float("nan")
    out = W.moe_fp8_block_apply(*on(x, w13, w2, s13, s2, tw, ids))
    rest = [t for t in range(T) if t not in (0, 2)]
    assert out[0].isnan().all() and out[2].isnan().all() and torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("block", [64, 128, 80])
def test_tiles_rows_by_identity_and_foreign_ids(block):
    """gather=False in tiles: ids past the slots, experts that are not there, rows past the count and rows that x does
    not have are left alone."""
    g = gen(32, block)
    N, K, E, dtype = 200, 272, 3, torch.bfloat16
    P = 6 * block
    x, xs = fp8_rows(g, P - 40, K)
    w, ws = fp8_weight(g, (E,), N, K)
    sti = torch.arange(P, dtype=torch.int32)
    sti[5], sti[17], sti[100] = 1 << 30, -1, P
    eid = torch.tensor([0, 2, 7, -1, 1, 1], dtype=torch.int32)
    before = torch.full((P, N), 3.0, dtype=dtype)
    for ntp in (0, 1, 70, P - 40, P, 1 << 20):
        out = before.to(DEV)
        W.moe_fp8_block_gemm(*on(x, xs, w, ws, sti, eid, torch.tensor([ntp], dtype=torch.int32)), 1, block, out=out,
                             gather=False)
        S.check_rows(out, before, x, xs, w, ws, sti, eid, min(ntp, P - 40), 1, block, dtype, P, gather=False)


@pytest.mark.parametrize("block", [16, 64])
def test_group_of_fewer_slots(block):
    """num_slots below tokens * top_k: the slots past it are padding."""
    g = gen(33, block)
    T, k, E, N, K = 90, 2, 4, 130, 256
    x, xs = fp8_rows(g, T, K)
    w, ws = fp8_weight(g, (E,), N, K)
    ids = torch.rand((T, E), generator=g).argsort(1)[:, :k].to(torch.int32)
    sti, eid, ntp = W.moe_align_block_size(ids.to(DEV), block, E)
    before = torch.full((sti.numel(), N), 7.0, dtype=torch.float16)
    for slots in (0, 1, 77):
        out = before.to(DEV)
        W.moe_fp8_block_gemm(*on(x, xs, w, ws), sti, eid, ntp, k, block, out=out, num_slots=slots)
        S.check_rows(out, before, x, xs, w, ws, sti, eid, int(ntp), k, block, torch.float16, slots)


@pytest.mark.parametrize("M", [5, 40])
def test_dense_16_bit_rows_with_nan_and_infinity(M):
    """A NaN or an infinity marks its row; the others' bits stay."""
    g = gen(34, M)
    x = hidden(g, M, 400, torch.bfloat16)
    w, ws = fp8_weight(g, (), 72, 400)
    clean = W.fp8_block_gemm(x.to(DEV), None, *on(w, ws))
    x[1, 399], x[3, 0] = float("nan"), float("-inf")
    out = W.fp8_block_gemm(x.to(DEV), None, *on(w, ws))
    rest = [m for m in range(M) if m not in (1, 3)]
    assert out[1].isnan().all() and out[3].isnan().all() and torch.equal(out[rest], clean[rest])


def test_strided_scales():
    """Scales of columns in memory, of every second row, and of one row for all."""
    g = gen(35)
    x, xs = on(*fp8_rows(g, 20, 384))
    w, ws = on(*fp8_weight(g, (), 70, 384))
    want = W.fp8_block_gemm(x, xs, w, ws)
    assert torch.equal(W.fp8_block_gemm(x, xs.t().contiguous().t(), w, ws), want)
    assert torch.equal(W.fp8_block_gemm(x, xs.repeat_interleave(2, 0)[::2], w, ws), want)
    one = xs[:1].expand(20, 3)
    assert torch.equal(W.fp8_block_gemm(x, one, w, ws), W.fp8_block_gemm(x, one.contiguous(), w, ws))
    rows = x[:1].expand(20, 384)
    assert torch.equal(W.fp8_block_gemm(rows, xs, w, ws), W.fp8_block_gemm(rows.contiguous(), xs, w, ws))


def test_no_tokens():
    x, w13, s13, w2, s2, tw, ids = layer_case(4, 2, 4, 256, 128, torch.bfloat16)
    out = W.moe_fp8_block_apply(*on(x[:0], w13, w2, s13, s2, tw[:0], ids[:0]))
    assert out.shape == (0, 256) and out.dtype == torch.bfloat16
    e = torch.empty((0,), dtype=torch.int32, device=DEV)
    q, s = on(*fp8_rows(gen(1), 4, 256))
    got = W.moe_fp8_block_gemm(q, s, *on(w13, s13), e, e, torch.zeros(1, dtype=torch.int32, device=DEV), 2, 64)
    assert got.shape == (0, 256)


def test_two_graphs_of_fp16_layers_at_once():
    """Two captured layers in fp16 (slots' rows in fp32), replayed at the same time beside eager calls."""
    args = [on(x, w13, w2, s13, s2, tw, ids) for x, w13, s13, w2, s2, tw, ids in
            (layer_case(T, 2, 6, 256, 128, torch.float16, T) for T in (5, 150))]
    want = [W.moe_fp8_block_apply(*a) for a in args]
    graphs, held = [], []
    for a in args:
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(W.moe_fp8_block_apply(*a))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        torch.cuda.synchronize()
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        eager = [W.moe_fp8_block_apply(*a) for a in args]
        torch.cuda.synchronize()
        for h, e, w in zip(held, eager, want):
            assert torch.equal(h, w) and torch.equal(e, w)
            h.zero_()
