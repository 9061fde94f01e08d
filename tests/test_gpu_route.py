"""The expert choice on the GPU against a float64 restatement (oracle/int8.py ``route``): ids equal, weights to fp32's
rounding. A renormalised weight in fp32: the pick's p is off by up to 5 half steps (exponential 3, sum, quotient), the sum of
eight by as much and 3 more of its tree, the quotient and the scale by one each: 15. Not renormalised: a softmax's
denominator is a sum of up to 256 fp32 exponentials, each off by |x| + 3 half steps of itself (|x| e^-|x| sums up to less
than ln 256 = 5.6 of the whole) and 8 of the tree: with p and two more, 24."""
import numpy as np
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import int8 as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(*parts):
    return torch.Generator().manual_seed(hash(parts) % (1 << 31))


def check(l, k, scoring="softmax", bias=None, groups=1, top=1, renorm=True, scale=1.0):
    w, ids = W.route_topk(l.to(DEV), k, scoring=scoring, bias=None if bias is None else bias.to(DEV), num_groups=groups,
                          top_groups=top, renormalize=renorm, scale=scale)
    rw, rid = O.route(l.double().numpy(), k, scoring, None if bias is None else bias.numpy(), groups, top, renorm, scale)
    assert np.array_equal(ids.cpu().numpy(), rid)
    got = w.double().cpu().numpy()
    assert np.all(np.abs(got - rw) <= np.abs(rw) * (24 if not renorm else 15) * O.U32 + 2.0 ** -148)
    return w, ids


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("T,E,k,groups,top", [(1, 1, 1, 1, 1), (1, 2, 2, 2, 2), (5, 8, 3, 1, 1), (3, 60, 4, 4, 2), (7, 64, 8, 8, 4),
                                              (9, 65, 6, 5, 2), (4, 100, 10, 1, 1), (66, 128, 8, 16, 3), (13, 160, 6, 8, 3),
                                              (33, 256, 8, 8, 4), (2, 256, 64, 4, 3), (3, 384, 8, 64, 5), (5, 512, 16, 1, 1),
                                              (2, 1000, 8, 50, 7), (3, 1024, 8, 16, 4), (2, 1024, 64, 64, 64)])
def test_choice(T, E, k, groups, top, with_bias, scoring, dtype):
    g = gen(T, E, k, groups)
    l = (torch.randn((T, E), generator=g) * 2 - 1).to(dtype)     # (16-bit logits: many are equal)
    b = torch.randn((E,), generator=g) * 0.1 if with_bias else None
    check(l, k, scoring, b, groups, top)
    check(l, k, scoring, b, groups, top, renorm=False, scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [None, 0.25])
@pytest.mark.parametrize("groups,top", [(1, 1), (4, 2)])
def test_ties_go_to_the_lower_expert(scoring, bias, groups, top):
    b = None if bias is None else torch.full((16,), bias)
    _, ids = check(torch.zeros((3, 16)), 5, scoring, b, groups, top)
    assert ids[0].tolist() == [0, 1, 2, 3, 4]
    l = torch.zeros((1, 16))
    l[0, 9] = l[0, 13] = 1.0
    _, ids = check(l, 3, scoring, b, groups, top)
    assert ids[0].tolist() == ([9, 13, 8] if groups == 4 else [9, 13, 0])


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_that_fp32_cannot_tell_apart(scoring):
    """c differs by less than fp32 holds: sigmoids next to one, and biases of 2^20 beside scores that differ by 2^-20."""
    l = torch.tensor([[18.0, 19.0, 20.0, 17.0, 21.0, 16.0, 15.0, 22.0]])
    _, ids = check(l, 4, scoring, torch.zeros(8))
    assert ids[0].tolist() == [7, 4, 2, 1]
    check(l, 4, scoring, torch.full((8,), 0.125), 2, 1)
    l = torch.linspace(-0.3, 0.3, 64)[torch.randperm(64, generator=gen(3))][None]
    check(l, 8, scoring, torch.full((64,), 2.0 ** 20))
    check(l, 8, scoring, torch.full((64,), -2.0 ** 20), 8, 3)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups,top", [(1, 1), (8, 3)])
def test_masked_experts(with_bias, scoring, groups, top):
    """-inf and NaN are never picked, rows that leave too few or none give -1 and 0, the lowest value is a value."""
    g = gen(5)
    l = torch.randn((12, 64), generator=g)
    b = torch.randn((64,), generator=g) * 0.1 if with_bias else None
    l[0] = -torch.inf
    l[1, 3:] = -torch.inf
    l[2, torch.rand(64, generator=g) < 0.9] = -torch.inf
    l[3] = torch.nan
    l[4, ::2] = torch.nan
    l[5, 1:] = torch.finfo(torch.float32).min
    l[6, 7] = torch.inf
    l[7, 7] = l[7, 9] = torch.inf
    l[8] = torch.finfo(torch.float32).min
    l[9] = torch.finfo(torch.float32).max
    l[10] = -200.0 + l[10]
    w, ids = check(l, 8, scoring, b, groups, top)
    assert ids[0].tolist() == [-1] * 8 and not w[0].any() and ids[3].tolist() == [-1] * 8
    assert w.isfinite().all()
    check(l, 8, scoring, b, groups, top, renorm=False)
    if with_bias:
        b[5:9] = torch.tensor([-torch.inf, torch.nan, torch.inf, torch.inf])
        w, ids = check(l, 8, scoring, b, groups, top)
        assert not ((ids == 5) | (ids == 6)).any()


def test_strided_rows_and_no_rows():
    g = gen(6)
    l = torch.randn((10, 96), generator=g).to(DEV)
    part = l[::2, 16:80]
    for a, b in zip(W.route_topk(part, 6), W.route_topk(part.contiguous(), 6)):
        assert torch.equal(a, b)
    for a, b in zip(W.route_topk(l.t().contiguous().t(), 6), W.route_topk(l, 6)):
        assert torch.equal(a, b)
    w, ids = W.route_topk(l[:0], 4)
    assert w.shape == ids.shape == (0, 4)


def test_agrees_with_the_plain_router():
    l = torch.randn((77, 256), generator=gen(7)).to(DEV)
    for renorm in (True, False):
        w, ids = W.route_topk(l, 8, renormalize=renorm)
        pw, pids = W.fused_topk(None, l, 8, renorm)
        assert torch.equal(ids, pids) and torch.allclose(w, pw, rtol=2e-6, atol=0)


def test_many_tokens():
    g = gen(8)
    l = torch.randn((5000, 64), generator=g).bfloat16()
    check(l, 6, "sigmoid", torch.randn((64,), generator=g) * 0.1, 8, 4)
