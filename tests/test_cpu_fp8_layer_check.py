"""The layer's check (fp8_layer_check.py) against layers computed here: a right one passes, and each of the
mistakes and roundings that the layer's design rules out is found."""
import numpy as np
import pytest
import torch

import fp8_layer_check as C
from oracle import fp8_block as O

CASE = (48, 2, 4, 256, 256)


def cut_product(x, w):
    """(M, K), (N, K) of one group -> sums as the fp8 matrix core takes them: of eight neighbouring products
    each is cut, towards zero, to a multiple of 2^(E - 13)."""
    top = lambda v: np.where(v != 0, np.frexp(np.maximum(np.abs(v), 2.0 ** -6))[1] - 1.0, -99.0)   # noqa: E731
    ex, ew, out = top(x), top(w), 0.0
    for k in range(0, x.shape[1], 8):
        p = x[:, None, k:k + 8] * w[None, :, k:k + 8]
        unit = np.exp2((ex[:, None, k:k + 8] + ew[None, :, k:k + 8]).max(-1, keepdims=True) - 13)
        out = out + (np.trunc(p / unit) * unit).sum(-1)
    return out


def scaled_product(x, xs, w, ws, cut):
    each, out = np.repeat(ws.astype(np.float64), 128, axis=0), 0.0
    for g in range(x.shape[1] // 128):
        k = slice(128 * g, 128 * g + 128)
        t = cut_product(x[:, k], w[:, k]) if cut else x[:, k] @ w[:, k].T
        out = out + t * xs[:, g:g + 1].astype(np.float64) * each[None, :, g]
    return out


def layer(case, dtype, rows=None, wrong=None):
    """rows: what the slots' rows are rounded to; wrong: a mistake."""
    x, xs, w13, s13, w2, s2, tw, ids = case
    rng = np.random.default_rng(1)
    out = np.zeros(x.shape)
    for e in range(len(w13)):
        t, j = np.nonzero(ids == e)
        gu = scaled_product(x[t], xs[t], w13[e], s13[e], wrong == "first product cut")
        inter = gu.shape[1] // 2
        h = O.silu_mul(gu[:, :inter], gu[:, inter:])
        if wrong == "noise":
            h = h * (1 + 0.01 * rng.standard_normal(h.shape))
        if wrong == "h in bf16":
            h = C.round16(h, torch.bfloat16)
        q, s = O.quantise(h)
        if wrong == "h not quantised":
            q = h / O.spread(s.astype(np.float64), inter)
        if wrong == "a group dropped":
            q[:, :128] = 0
        if wrong == "scales swapped":
            s = s[:, ::-1]
        y = scaled_product(q, s, w2[e], s2[e], True)
        if rows is not None:
            power = np.exp2(14 - np.floor(np.log2(np.abs(y).reshape(len(t), -1, 32).max(-1)))).repeat(32, axis=1)
            y = C.round16(y * power, rows) / power
        np.add.at(out, t, y * tw[t, j].astype(np.float64)[:, None])
    if wrong == "one per cent":
        out *= 1.01
    if wrong == "one token off":
        out[5] *= 1.004
    return C.round16(out, dtype)


@pytest.fixture(scope="module")
def case():
    c = C.exact_case(*CASE)
    assert all(O.sums_are_exact(c[0], c[1], c[2][e], c[3][e]) for e in range(len(c[2])))
    return c


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_quantise_to_what_they_were_made_of(case, dtype):
    q, s = O.quantise(C.rows16(case[0], case[1], dtype).double().numpy())
    assert np.array_equal(q, case[0]) and np.array_equal(s, case[1])


@pytest.mark.parametrize("dtype,rows,half", [(torch.bfloat16, None, 0.0), (torch.float16, None, 0.0),
                                             (torch.bfloat16, torch.float16, C.ROW_HALF)])
def test_right_layers_pass(case, dtype, rows, half):
    assert C.complaints(layer(case, dtype, rows), dtype, O.known_layer(*case, half)) == []


@pytest.mark.parametrize("wrong", ["first product cut", "noise", "h in bf16", "h not quantised", "a group dropped",
                                   "scales swapped", "one per cent", "one token off"])
@pytest.mark.parametrize("dtype,rows,half", [(torch.bfloat16, torch.float16, C.ROW_HALF), (torch.float16, None, 0.0)])
def test_mistakes_are_found(case, dtype, rows, half, wrong):
    assert C.complaints(layer(case, dtype, rows, wrong), dtype, O.known_layer(*case, half)) != []


@pytest.mark.parametrize("dtype,half", [(torch.bfloat16, C.ROW_HALF), (torch.bfloat16, 0.0), (torch.float16, 0.0)])
def test_rows_in_the_outputs_own_type_are_found(case, dtype, half):
    """Slots' rows in bf16 before a bf16 sum, or in fp16 before an fp16 one."""
    assert "whole" in C.complaints(layer(case, dtype, dtype), dtype, O.known_layer(*case, half))
