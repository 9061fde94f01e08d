"""Calls of the int8 layer that are taken in several parts of tokens, the last of them ragged: the same bits as calls on
tokens from all over the batch."""
import pytest
import torch

import w4a8_fp8_wmma as W

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layer_in_parts(T, E, k, H, I, part, int8):
    """part: tokens of a part, by the sizes' limits."""
    assert part < T < 2 * part
    g = torch.Generator(device=DEV).manual_seed(T + E + k)
    w13 = torch.randint(-128, 128, (E, 2 * I, H), generator=g, dtype=torch.int8, device=DEV)
    w2 = torch.randint(-128, 128, (E, H, I), generator=g, dtype=torch.int8, device=DEV)
    s13 = torch.rand((E, 2 * I), generator=g, device=DEV) * 1e-4
    s2 = torch.rand((E, H), generator=g, device=DEV) * 1e-3
    tw = torch.rand((T, k), generator=g, device=DEV)
    ids = torch.randint(-1, E, (T, k), generator=g, dtype=torch.int32, device=DEV)
    if int8:
        x, xs = torch.randint(-128, 128, (T, H), generator=g, dtype=torch.int8, device=DEV), torch.rand((T, 1), generator=g, device=DEV)
    else:
        x, xs = torch.randn((T, H), generator=g, device=DEV).bfloat16(), None
    for dtype in (torch.bfloat16, torch.float16):
        y = W.moe_int8_apply(x, w13, w2, s13, s2, tw, ids, x_scales=xs, out_dtype=dtype)
        assert y.isfinite().all()
        for at in (0, 1000, part - 20, part, T - 40):
            rows = slice(at, at + 40)
            few = W.moe_int8_apply(x[rows], w13, w2, s13, s2, tw[rows], ids[rows], x_scales=None if xs is None else xs[rows], out_dtype=dtype)
            assert few.any() and torch.equal(y[rows], few), at
        del y


def test_tiles_by_their_rows():
    """Rows of x up to 2^32 bytes a part."""
    H, part = 131008, ((1 << 32) - 1) // 131008
    layer_in_parts(part + 60, 2, 1, H, 64, part, True)


@pytest.mark.parametrize("int8", [False, True])
def test_tiles_by_their_hidden_rows(int8):
    """Rows of h, padded to blocks, up to 2^32 bytes a part."""
    I, E, k = 131008, 3, 2
    part = (((1 << 32) - 1) // I - (E * 127 + 128)) // k
    layer_in_parts(part + 333, E, k, 64, I, part, int8)


def test_streamed():
    """An expert of more than 2^32 bytes is streamed whatever the number of tokens, 4096 slots a part."""
    H = I = 46400
    assert 2 * H * I >= 1 << 32
    layer_in_parts(2048 + 70, 2, 2, H, I, 2048, False)
