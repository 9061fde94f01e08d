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


LOW = {torch.float32: (torch.finfo(torch.float32).min, -1e30, -1e9, -1e4), torch.bfloat16: (torch.finfo(torch.bfloat16).min, -1e9)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top,k", [(256, 1, 1, 8), (256, 8, 4, 8), (128, 16, 2, 8), (64, 4, 1, 6), (64, 1, 1, 1), (60, 1, 1, 2), (24, 1, 1, 8), (8, 1, 1, 4)])
def test_low_numbers_as_masks_and_far_logits(E, groups, top, k, scoring, dtype):
    """Rows of which a part, nearly all or all experts are masked by a low finite number, in the logits or in the bias; one
    logit far above the others; groups of equal logits."""
    g = gen(E, groups, k, 65)
    for low in LOW[dtype]:
        l = torch.randn((120, E), generator=g)
        l[:30] = torch.where(torch.rand((30, E), generator=g) < 0.5, low, l[:30])
        l[30:50] = torch.where(torch.rand((20, E), generator=g) < 0.97, low, l[30:50])
        l[50:54] = low
        l[54:58, 1:] = low
        l[58:70, E // 2] = -low if low > -1e30 else 1e30
        l[70:80, E // 3] = low
        l[80:90] = l[80:90].round()
        l[90] = l[91, 0]
        l[91:95, : E // 2] = -torch.inf
        l[95:100] *= 1e-6
        l[100:105] *= 1e4
        for bias in (None, torch.randn((E,), generator=g) * 0.1):
            check(l.to(dtype), k, scoring, bias, groups, top)
        b = torch.randn((E,), generator=g) * 0.1
        b[torch.rand((E,), generator=g) < 0.3] = low
        check(l.to(dtype), k, scoring, b, groups, top)
        b[E // 2] = 1e4
        check(l.to(dtype), k, scoring, b, groups, top)


def best_us(calls, n=20, rounds=7):
    """The shortest of some rounds' mean times, of calls in turn."""
    times = [[] for _ in calls]
    for r in range(rounds + 1):
        for at, call in enumerate(calls):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(n):
                call()
            b.record()
            torch.cuda.synchronize()
            if r > 0:
                times[at].append(a.elapsed_time(b) / n * 1e3)
    return [min(t) for t in times]


@pytest.mark.parametrize("with_bias", [False, True])
def test_low_masks_take_no_longer(with_bias):
    """Tokens whose experts are masked by a low finite number do not all fall back to one token a wave (which takes four
    times as long)."""
    g = torch.Generator(device=DEV).manual_seed(66)
    l = torch.randn((1 << 18, 256), generator=g, device=DEV)
    b = torch.randn((256,), generator=g, device=DEV) * 0.1 if with_bias else None
    for low in (torch.finfo(torch.float32).min, -1e9):
        if with_bias:
            m, mb = l, torch.where(torch.rand((256,), generator=g, device=DEV) < 0.3, low, b)
        else:
            m, mb = torch.where(torch.rand(l.shape, generator=g, device=DEV) < 0.3, low, l), None
        plain, masked = best_us([lambda: W.route_topk(l, 8, scoring="sigmoid", bias=b), lambda: W.route_topk(m, 8, scoring="sigmoid", bias=mb)])
        assert masked < 2 * plain, (plain, masked)
