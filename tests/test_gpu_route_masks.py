"""Masks of the expert choice beside ordinary scores, against the float64 restatement (oracle/int8.py ``route``)."""
import pytest
import torch

from test_gpu_route import check, gen

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
