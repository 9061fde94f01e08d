"""silu(gate) * up far from zero: gates whose exponential leaves fp32's range beside large up values."""
import numpy as np
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import fp8_block as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [256, 250])                # eight values a lane; value by value
def test_far_gates(K):
    """bf16 gates of -60 to -123, a row each, and up of 2^90 to 2^127 (silu(-88) * 2^127 is -90)."""
    R = 64
    g = np.repeat(-60.0 - np.arange(R)[:, None], K, axis=1)
    rng = np.random.default_rng(5)
    u = rng.choice([-1, 1], (R, K)) * np.exp2(rng.integers(90, 128, (R, 1))) * (1 + rng.integers(0, 128, (R, K)) / 128)
    x = torch.from_numpy(np.concatenate([g, u], 1)).to(torch.bfloat16)
    q, s = W.act_quant_fp8_block(x.to("cuda"), activation="silu")
    v = x.double().numpy()
    g, u = v[:, :K], v[:, K:]
    h = O.silu_mul(g, u)
    # the exponential's argument, its result, the reciprocal and the products: |g| steps and a few more; then as
    # any group's scale and values
    rel = (2 * 124 + 8) * O.U32
    want, got = O.group_scales(h).astype(np.float64), s.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - want) <= want * (rel + 3 * O.U32))
    w = h / O.spread(got, K)
    d = np.abs(w) * (rel + 4 * O.U32)
    q = q.double().cpu().numpy()
    assert np.all((q >= O.round_e4m3(w - d)) & (q <= O.round_e4m3(w + d)))


def test_ends():
    """A gate of -infinity or NaN marks its value only; a large negative one next to ordinary up is zero."""
    x = torch.ones((1, 256), dtype=torch.bfloat16)
    x[0, 3], x[0, 4], x[0, 5], x[0, 6] = float("-inf"), float("nan"), -1e30, 1e30
    x[0, 128 + 6] = 1e-30
    q, s = W.act_quant_fp8_block(x.to("cuda"), activation="silu")
    v = q.double().cpu().numpy()[0] * float(s)
    assert np.isnan(v[3]) and np.isnan(v[4]) and v[5] == 0 and abs(v[6] - 1) <= 2.0 ** -4
    rest = np.delete(v, [3, 4, 5, 6])
    assert (np.abs(rest - 1 / (1 + np.exp(-1.0))) <= 0.7311 * 2.0 ** -4 * 1.0001).all()
