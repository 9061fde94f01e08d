"""64-bit expert ids and maps of the int8 layer: numbers past 32 bits name no expert, whatever their low words are."""
import pytest
import torch

import w4a8_fp8_wmma as W
from test_gpu_int8 import DEV, gen, hidden, make_layer, make_routing, on

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [2, 30, 200])
def test_ids_past_32_bits(T):
    E, k, H, I = 8, 4, 128, 64
    g = gen(T, 67)
    w13, w2, s13, s2 = make_layer(g, E, H, I)
    tw, ids = make_routing(g, T, E, k)
    x = hidden(g, T, H, torch.bfloat16)
    least = torch.iinfo(torch.int64).min
    far = torch.tensor([least, 1 << 32, (1 << 32) + 3, -(1 << 32) + 1, torch.iinfo(torch.int64).max, 1 << 31])
    ids = ids.long()
    out = torch.rand((T, k), generator=g) < 0.4
    none, wide = ids.clone(), ids.clone()
    none[out] = -1
    wide[out] = far[torch.randint(0, len(far), (int(out.sum()),), generator=g)]
    args = on(x, w13, w2, s13, s2, tw)
    ref = W.moe_int8_apply(*args, none.to(torch.int32).to(DEV))
    assert torch.equal(W.moe_int8_apply(*args, wide.to(DEV)), ref)
    assert not torch.equal(W.moe_int8_apply(*args, ids.to(DEV)), ref)
    # the same by a map from 2 E global experts
    local = torch.arange(2 * E) % E
    away, lost = local.clone(), local.clone()
    away[::3] = -1
    lost[::3] = far[torch.arange(len(lost[::3])) % len(far)]
    ids = torch.randint(0, 2 * E, (T, k), generator=g)
    ref = W.moe_int8_apply(*args, ids.to(DEV), expert_map=away.to(torch.int32).to(DEV))
    assert torch.equal(W.moe_int8_apply(*args, ids.to(DEV), expert_map=lost.to(DEV)), ref)
