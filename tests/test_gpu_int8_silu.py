"""silu(gate) * up of gates next to fp32's largest number: silu(gate) is the gate there, and the row is finite."""
import numpy as np
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import int8 as O
from test_gpu_int8 import DEV, f64, on

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [8, 7, 1024])
def test_quant_of_large_gates(K):
    gates = torch.tensor([1e38, 2.3e38, 2.37e38, 2.5e38, 3e38, 3.38e38, 130.0, 100.0])
    x = torch.zeros((5, 2 * K), dtype=torch.bfloat16)
    x[:, :K] = gates.repeat(-(-K // 8))[:K]
    for row, up in enumerate((0.5, -1.0, 1e-3, 1e-30, 1e-38)):
        x[row, K:] = up
    q, s = W.act_quant_int8(x.to(DEV), activation="silu")
    v = f64(x)
    h = O.silu_mul(v[:, :K], v[:, K:])
    a = np.abs(h).max(1, keepdims=True)
    # the product's rounding and the scale's; of a value its own and the quotient's
    assert np.all(np.abs(f64(s) * 127 - a) <= a * 3 * O.U32)
    assert np.all(np.abs(f64(q) - h * 127 / a) <= 0.5 + 127 * 8 * O.U32)


@pytest.mark.parametrize("T", [2, 40, 400])
def test_layer_of_large_gates(T):
    """Gates of 2.6e38 and more beside ups of 1e-30: the same h as gates of 2^-40 of that beside ups of 2^40 as much."""
    E, k, H, I = 2, 1, 64, 64
    g = torch.Generator().manual_seed(T)
    w13 = torch.randint(1, 128, (E, 2 * I, H), generator=g, dtype=torch.int8)
    w2 = torch.randint(-128, 128, (E, H, I), generator=g, dtype=torch.int8)
    x, xs = torch.full((T, H), 127, dtype=torch.int8), torch.ones((T, 1))
    ids = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    tw, s2 = torch.ones((T, k)), torch.full((E, H), 1e-12)
    total = w13.double().sum(2) * 127
    gate = 2.6e38 + 0.7e38 * torch.rand((E, I), generator=g).double()
    s13 = torch.cat([gate / total[:, :I], torch.full((E, I), 1e-30).double() / total[:, I:]], 1).float()
    half = s13.clone()
    half[:, :I] *= 2.0 ** -40
    half[:, I:] *= 2.0 ** 40
    y = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, ids), x_scales=xs.to(DEV))
    z = W.moe_int8_apply(*on(x, w13, w2, half, s2, tw, ids), x_scales=xs.to(DEV))
    assert y.isfinite().all() and torch.equal(y, z)
