"""The int8 layer's sum over a token's slots holds their rows in fp32 in every schedule: held to the oracle's fp32 roundings
where many tokens go through tiles and where slots cancel, and the same bits whatever the batch a token is in."""
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import int8 as O
from test_gpu_int8 import assert_close, f64, gen, hidden, make_layer, make_routing, on

pytestmark = pytest.mark.gpu

# (T, E, k, H, I): more slots than are streamed, blocks of 64 and of 128 rows
TILES = [(150, 4, 2, 192, 128), (300, 16, 4, 128, 192), (900, 4, 2, 128, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,I", TILES)
def test_many_tokens(T, E, k, H, I, dtype):
    g = gen(T, E, k, H, I, 60)
    w13, w2, s13, s2 = make_layer(g, E, H, I)
    tw, ids = make_routing(g, T, E, k)
    x = hidden(g, T, H, dtype)
    y = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, ids))
    assert_close(y, *O.layer(*O.quantise(f64(x)), f64(w13), s13.numpy(), f64(w2), s2.numpy(), tw.numpy(), ids.numpy()), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [3, 40, 300, 800])
def test_slots_that_cancel(T, dtype):
    """A token's second slot takes away its first one's row but for a part in 2^10: experts in pairs of the same weights,
    whose scales differ by 1.3. What is left is held to the roundings of the two rows."""
    E, k, H, I = 4, 2, 128, 64
    g = gen(T, 61)
    w13, w2, s13, s2 = make_layer(g, E, H, I)
    w13[2:], w2[2:], s13[2:], s2[2:] = w13[:2], w2[:2], s13[:2], s2[:2] * 1.3
    first = torch.randint(0, 2, (T, 1), generator=g, dtype=torch.int32)
    ids = torch.cat([first, first + 2], 1)
    a = torch.rand((T, 1), generator=g) + 0.5
    tw = torch.cat([a, a * (-(1 - 2.0 ** -10) / 1.3)], 1)
    x = hidden(g, T, H, dtype)
    y = W.moe_int8_apply(*on(x, w13, w2, s13, s2, tw, ids))
    assert_close(y, *O.layer(*O.quantise(f64(x)), f64(w13), s13.numpy(), f64(w2), s2.numpy(), tw.numpy(), ids.numpy()), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,I", TILES + [(400, 64, 4, 256, 128)])
def test_the_same_bits_in_any_batch(T, E, k, H, I, dtype):
    """Tiles of many tokens, streamed experts of some, a slot at a time of few."""
    g = gen(T, E, k, H, I, 62)
    w13, w2, s13, s2 = on(*make_layer(g, E, H, I))
    tw, ids = on(*make_routing(g, T, E, k))
    x = hidden(g, T, H, dtype).to(ids.device)
    y = W.moe_int8_apply(x, w13, w2, s13, s2, tw, ids)
    for n in (1, 4, 30):
        for at in (0, T // 2, T - n):
            part = slice(at, at + n)
            assert torch.equal(W.moe_int8_apply(x[part], w13, w2, s13, s2, tw[part], ids[part]), y[part]), (n, at)
