"""The gated fp8 layer's accuracy on the GPU, held to what its design says (fp8_layer_check.py): rows that are
streamed and rows in tiles, from 16-bit rows and from e4m3 rows with their scales, in both output types."""
import numpy as np
import pytest
import torch

import fp8_layer_check as C
import w4a8_fp8_wmma as W
from oracle import fp8_block as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn


def dev8(v):
    return torch.from_numpy(np.asarray(v, np.float32)).to(DEV).to(FP8)


def dev(v):
    return torch.from_numpy(np.ascontiguousarray(v)).to(DEV)


def args_of(case):
    x, xs, w13, s13, w2, s2, tw, ids = case
    return dev8(w13), dev8(w2), dev(s13), dev(s2), dev(tw), dev(ids)


def rows_of(case, dtype, e4m3):
    return (dev8(case[0]), dev(case[1])) if e4m3 else (C.rows16(case[0], case[1], dtype).to(DEV), None)


def check(case, dtype, e4m3, tiles):
    for e in range(len(case[2])):
        assert O.sums_are_exact(case[0][:8], case[1][:8], case[2][e], case[3][e])
    x, xs = rows_of(case, dtype, e4m3)
    out = W.moe_fp8_block_apply(x, *args_of(case), x_scales=xs, out_dtype=dtype)
    half = C.ROW_HALF if tiles and dtype == torch.bfloat16 else 0.0
    assert C.complaints(out.double().cpu().numpy(), dtype, O.known_layer(*case, half)) == []


# up to 12 slots an expert are streamed; K groups: 2 and 1, 5 and 3, 40 and 1
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,k,E,H,I", [(24, 2, 8, 256, 128), (21, 4, 8, 640, 384), (20, 2, 4, 5120, 128)])
def test_streamed(T, k, E, H, I, dtype, e4m3):
    assert T * k <= 12 * E
    check(C.exact_case(T, k, E, H, I), dtype, e4m3, False)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("T,k,E,H,I", [(96, 2, 4, 256, 256), (61, 4, 8, 640, 384), (70, 2, 4, 5120, 128)])
def test_tiles_bf16(T, k, E, H, I, e4m3):
    assert T * k > 12 * E
    check(C.exact_case(T, k, E, H, I), torch.bfloat16, e4m3, True)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("T,k,E,H,I", [(96, 2, 4, 256, 256), (61, 4, 8, 640, 384), (70, 2, 4, 5120, 128)])
def test_tiles_fp16(T, k, E, H, I, e4m3):
    """Slots' rows in fp32: in fp16 they would add as much error as the output's own rounding."""
    assert T * k > 12 * E
    check(C.exact_case(T, k, E, H, I), torch.float16, e4m3, True)


@pytest.mark.parametrize("T", [3, 80])
def test_expert_map_fp16(T):
    """Slots of experts that live elsewhere have no rows: what their place in the workspace holds does not count."""
    case = C.exact_case(T, 3, 12, 256, 128)
    x, xs, w13, s13, w2, s2, tw, ids = case
    emap = np.full(12, -1, np.int32)
    emap[[1, 4, 5, 9]] = [2, 0, 3, 1]
    local = emap[ids]
    small = (x, xs, w13[:4], s13[:4], w2[:4], s2[:4], tw, local)
    if T * 3 > 48:
        torch.full((1 << 24,), float("nan"), device=DEV)            # (freed: the workspace's memory)
    out = W.moe_fp8_block_apply(rows_of(case, torch.float16, False)[0], *args_of(small)[:4], dev(tw), dev(ids),
                                expert_map=dev(emap))
    assert C.complaints(out.double().cpu().numpy(), torch.float16, O.known_layer(*small)) == []


def test_decoder_half_in_tiles():
    """Norm with the residual, router and expert layer from the norm's e4m3 rows, more than 12 slots an expert:
    against the oracle, element by element."""
    from test_gpu_fp8_block import check_layer, check_norm, gen, hidden, layer_case, on
    g = gen(78)
    T, H, I, E, k = 90, 256, 128, 8, 2
    x, r = hidden(g, T, H, torch.bfloat16), hidden(g, T, H, torch.bfloat16)
    nw = (torch.randn((H,), generator=g) * 0.2 + 1).to(torch.bfloat16)
    _, w13, s13, w2, s2, _, _ = layer_case(T, k, E, H, I, torch.bfloat16)
    rw = torch.randn((H, E), generator=g)
    dx, dr, dnw, dw13, ds13, dw2, ds2, drw = on(x, r, nw, w13, s13, w2, s2, rw)
    n = W.rms_norm_quant_fp8(dx, dnw, residual=dr, return_norm=True)
    tw, ids = W.fused_topk(None, n.norm.float() @ drw, k)
    y = W.moe_fp8_block_apply(n.q, dw13, dw2, ds13, ds2, tw, ids, x_scales=n.scales)
    check_norm(x, r, nw, 1e-6, False, True, n)
    check_layer(y, x, w13, s13, w2, s2, tw.cpu(), ids.cpu(), torch.bfloat16, q=(n.q, n.scales))


def far_case(T, power, weight):
    """Column 5 of the second product is some 2^17 times as large as the others, column 9 is zero."""
    x, xs, w13, s13, w2, s2, tw, ids = C.exact_case(T, 1, 4, 256, 128)
    w2 = np.sign(w2) * 2.0 ** -9
    w2[:, 5], w2[:, 9] = 448 * np.sign(w2[:, 5]), 0
    s2 = np.exp2(np.full(s2.shape, power)).astype(np.float32)
    tw = np.exp2(np.full(tw.shape, weight)).astype(np.float32)
    return x, xs, w13, s13, w2, s2, tw, ids


def check_far(T, power, weight):
    case = far_case(T, power, weight)
    out = W.moe_fp8_block_apply(rows_of(case, torch.bfloat16, False)[0], *args_of(case)).double().cpu().numpy()
    ref, tol, _, clear = O.known_layer(*case, C.ROW_HALF)
    # (bf16's subnormal numbers lie 2^-126 / 2^7 = 2^-133 apart: a rounding among them is off by up to 2^-134)
    tol = tol + (np.abs(ref) + tol) * C.HALF[torch.bfloat16] + 2.0 ** -134
    over, inside = (np.abs(ref) > 4e38) & clear[:, None], (np.abs(ref) < 3e38) & clear[:, None]
    assert np.array_equal(out[over], np.sign(ref[over]) * np.inf)
    assert (np.abs(out - ref)[inside] <= tol[inside]).all()
    return over


@pytest.mark.parametrize("T", [20, 96])
def test_an_infinite_column_leaves_the_others(T):
    """A sum past fp32's range is infinite; the columns beside it, finite in bf16, stay as they are."""
    assert check_far(T, 118, 0)[:, 5].any()
    check_far(T, 0, 0)


@pytest.mark.parametrize("T", [20, 96])
def test_weights_far_from_one(T):
    """Sums of 2^124 in one column, a router's weight of 2^20: zeros stay zeros, small columns finite."""
    assert check_far(T, 110, 20)[:, 5].all()
    check_far(T, -110, -20)
