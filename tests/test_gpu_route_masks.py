"""The expert choice with masks beside ordinary scores, and its weights, against the float64 restatement (oracle/int8.py ``route``)."""
import numpy as np
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import int8 as O
from test_gpu_route import DEV, check, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top", [(64, 8, 3), (64, 4, 2), (128, 16, 5), (256, 8, 4), (160, 5, 2), (512, 8, 3)])
def test_bias_that_is_nan_leaves_its_groups_score(E, groups, top, scoring, dtype):
    """A masked expert behind live ones of its lane counts for neither of its group's two best."""
    g = gen(E, groups, 63)
    l = torch.randn((200, E), generator=g).to(dtype)
    for masks in (1, 2, E // groups - 2):
        b = torch.randn((E,), generator=g) * 0.1
        # in half of the groups, whose best and second best then are live experts beside the masked ones
        for first in range(0, E, 2 * E // groups):
            b[first + 1 + torch.randperm(E // groups - 1, generator=g)[:masks]] = torch.nan
        w, ids = check(l, min(8, top), scoring, b, groups, top)
        assert not b[ids.cpu().long().clamp_min(0)].isnan().any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,k,groups,top,wide", [(256, 8, 8, 4, 1.0), (60, 4, 1, 1, 6.0), (16, 2, 1, 1, 20.0), (300, 9, 1, 1, 3.0), (256, 8, 1, 1, 60.0)])
def test_weights_are_rounded_once(E, k, groups, top, wide, with_bias, scoring, dtype):
    """Weights are formed in fp64 and rounded to fp32. Without renormalisation a softmax's denominator is a sum in fp64 of
    fp32 exponentials, each off by 3 half steps (the hardware's 2^t by two, the correction of t by one)."""
    g = gen(E, k, groups, 64)
    l = (torch.randn((300, E), generator=g) * wide).to(dtype)
    b = torch.randn((E,), generator=g) * 0.1 if with_bias else None
    for renorm in (True, False):
        w, ids = W.route_topk(l.to(DEV), k, scoring=scoring, bias=None if b is None else b.to(DEV), num_groups=groups,
                              top_groups=top, renormalize=renorm, scale=1.75)
        rw, rid = O.route(l.double().numpy(), k, scoring, None if b is None else b.numpy(), groups, top, renorm, 1.75)
        assert np.array_equal(ids.cpu().numpy(), rid)
        halves = 1 if renorm or scoring == "sigmoid" else 4
        # (2^-150: half of fp32's least number)
        assert np.all(np.abs(w.double().cpu().numpy() - rw) <= np.abs(rw) * halves * O.U32 * (1 + 2.0 ** -20) + 2.0 ** -150)
