"""Checks of the gated fp8 layer that see its accuracy: inputs whose first product has exact sums, and what a
right output of them may be off by, element by element, as a whole and token by token."""
import numpy as np
import torch

from oracle import fp8_block as O

FP8 = torch.float8_e4m3fn
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a step, relative
ROW_HALF = 2.0 ** -11                                             # slots' rows in fp16 (many tokens, bf16 output)


def round16(v, dtype):
    return torch.from_numpy(np.asarray(v, np.float32)).to(dtype).double().numpy()


def whole_e4m3(rng, shape, width):
    return O.round_e4m3(np.rint(rng.standard_normal(shape) * width))


def exact_case(T, k, E, H, I, seed=0):
    """(e4m3 values and scales of rows, w13, s13, w2, s2, tw, ids): small whole numbers, among them in every
    group of 128 (up to 1024 values) two pairs, eight apart, of large ones whose products cancel. The fp8 matrix
    core cuts the products beside such a number to multiples of 8, which a sum of few hundred shows."""
    rng = np.random.default_rng([T, k, E, H, I, seed])
    x, w = whole_e4m3(rng, (T, H), 8), whole_e4m3(rng, (E, 2 * I, H), 8)
    x[:, ::128] = 448 * rng.choice([-1, 1], (T, H // 128))                 # a group's scale is its largest / 448
    for g in range(0, min(H, 1024), 128):
        for p in (g + 3, g + 69):
            x[:, p] = x[:, p + 8] = 448 * rng.choice([-1, 1], T)
            w[..., p] = 256 * rng.choice([-1, 1], (E, 2 * I))
            w[..., p + 8] = -w[..., p]
    xs = np.exp2(rng.integers(0, 2, (T, H // 128))).astype(np.float32)
    size = int(np.rint(np.log2(323 * 2.25 * np.sqrt(H) / 2)))               # gate and up of standard deviation 2
    s13 = np.exp2(rng.integers(0, 2, (E, 2 * I // 128, H // 128)) - size).astype(np.float32)
    w2 = O.round_e4m3(rng.standard_normal((E, H, I)) * 60)
    s2 = (rng.random((E, H // 128, I // 128)) * 2e-3 + 1e-4).astype(np.float32)
    tw = (rng.random((T, k)) + 0.1).astype(np.float32)
    ids = rng.random((T, E)).argsort(1)[:, :k].astype(np.int32)
    return x, xs, w, s13, w2, s2, tw, ids


def rows16(x, xs, dtype):
    """16-bit rows that quantise to x and xs."""
    return torch.from_numpy(x * O.spread(xs.astype(np.float64), x.shape[1])).to(dtype)


def complaints(out, dtype, known):
    """What is wrong with a layer's output (float64 values of dtype), as a list of words.

    Element by element: the fp32 bounds and half a step. As a whole and token by token, in the root of the
    summed squares: the output's own rounding error and what `known_layer` gives for the steps before. Both
    are sums over hundreds of values evenly spread in a step, whose relative deviation is below
    sqrt(0.8 / values): 3 % of a token of 256 values in the root, so 1.4 leaves eight deviations (the two
    roundings that are compared are alike in the main), and 1.1 as many over 20 tokens."""
    ref, tol, var, clear = known
    assert clear.mean() > 0.5, "inputs leave too few tokens known"
    ref, tol, var, err = ref[clear], tol[clear], var[clear], np.asarray(out)[clear] - ref[clear]
    bad = []
    limit = tol + (np.abs(ref) + tol) * HALF[dtype] + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    if not (np.abs(err) <= limit).all():
        bad.append("element")
    own = (round16(ref, dtype) - ref) ** 2 + var
    if not (err ** 2).sum() <= 1.1 ** 2 * own.sum():
        bad.append("whole")
    if not ((err ** 2).sum(1) <= 1.4 ** 2 * own.sum(1)).all():
        bad.append("token")
    return bad
