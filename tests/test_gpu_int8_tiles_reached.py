"""int8 tiles: sizes that reach every one of them, with whole and partial steps of K and with several tiles a work-group,
checked by the names of the kernels that ran, and their results."""
import json
import os
import re
import subprocess
import sys

import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import int8 as O
from test_gpu_int8 import HALF

pytestmark = pytest.mark.gpu
DEV = "cuda"
CUS = 256
STEP = 128

# tile (waves by rows, by columns, row and column fragments a wave, steps in LDS, parts of K): (M, N, K)
DENSE = {"1, 1, 1, 1, 4, 4": [(33, 1001, 4096), (17, 513, 2064), (1000, 200, 640), (40, 190, 144)],
         "2, 1, 1, 1, 4, 2": [(64, 4100, 272), (65, 4090, 384), (64, 8190, 4096)],
         "2, 2, 1, 1, 4, 1": [(65, 4100, 208), (77, 6000, 640), (64, 65600, 400), (64, 65600, 256)],
         "4, 2, 1, 1, 4, 1": [(100, 12300, 144), (128, 12288, 256), (192, 8190, 1152)],
         "2, 4, 2, 1, 4, 1": [(250, 12300, 208), (333, 6000, 128), (400, 8192, 896), (4000, 4100, 208), (4096, 4100, 384)],
         "4, 2, 2, 2, 3, 1": [(500, 12300, 272), (700, 8190, 384), (4096, 6000, 128), (3000, 8190, 400)],
         "2, 4, 4, 2, 2, 1": [(1030, 8190, 208), (1030, 12300, 128), (4096, 12288, 256), (2000, 4100, 4112), (4096, 4096, 1024)]}
# tiles with more of them than work-groups run at once
SEVERAL = {"2, 2, 1, 1, 4, 1": (64, 65600), "2, 4, 2, 1, 4, 1": (4000, 4100), "4, 2, 2, 2, 3, 1": (4096, 6000), "2, 4, 4, 2, 2, 1": (4096, 12288)}
# (first, second tile of a layer): (T, k, E, H, I)
LAYER = {("1, 4, 2, 2, 2, 1", "2, 4, 1, 2, 2, 1"): [(600, 4, 40, 256, 384), (600, 4, 40, 320, 192), (600, 4, 40, 192, 256)],
         ("2, 4, 2, 2, 3, 1", "2, 4, 2, 2, 3, 1"): [(600, 4, 8, 256, 384), (600, 4, 8, 320, 192), (600, 4, 8, 192, 256)]}


def zeros8(*shape):
    return torch.zeros(shape, dtype=torch.int8, device=DEV)


def ones(*shape):
    return torch.ones(shape, device=DEV)


def trace(path):
    """Runs every case once under torch's profiler and writes [[case, kernel, work-groups], ...]."""
    calls = []
    for shapes in DENSE.values():
        for M, N, K in shapes:
            a = zeros8(M, K), ones(M, 1), zeros8(N, K), ones(N)
            calls.append(((M, N, K), lambda a=a: W.int8_gemm(*a)))
    for shapes in LAYER.values():
        for T, k, E, H, I in shapes:
            ids = torch.arange(T * k, dtype=torch.int32, device=DEV).remainder(E).view(T, k)
            for dtype in (torch.bfloat16, torch.float16):
                a = torch.zeros((T, H), dtype=dtype, device=DEV), zeros8(E, 2 * I, H), zeros8(E, H, I), ones(E, 2 * I), ones(E, H), ones(T, k), ids
                calls.append(((T, k, E, H, I, str(dtype)), lambda a=a: W.moe_int8_apply(*a)))
    got = []
    for case, call in calls:
        call()
        torch.cuda.synchronize()
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
            call()
            torch.cuda.synchronize()
        p.export_chrome_trace(path)
        with open(path) as f:
            events = json.load(f)["traceEvents"]
        got += [[case, e["name"], e["args"]["grid"][0]] for e in events if e.get("cat") == "kernel" and "int8_tiles_kernel" in e["name"]]
        print(case, flush=True)
    with open(path, "w") as f:
        json.dump(got, f)


@pytest.fixture(scope="module")
def tiles(tmp_path_factory):
    """case -> [(tile, whether its last step is a partial one, work-groups)], from a process of its own: the profiler's
    hooks stay out of this one."""
    path = str(tmp_path_factory.mktemp("trace") / "kernels.json")
    here = os.path.dirname(os.path.abspath(__file__))
    paths = [here, os.path.dirname(here), os.path.join(os.path.dirname(here), "rdna4-vllm_amd")]
    code = f"import sys; sys.path[:0] = {paths!r}; import test_gpu_int8_tiles_reached as t; t.trace({path!r})"
    run = subprocess.run([sys.executable, "-u", "-c", code], capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stdout[-500:] + run.stderr[-2000:]
    found = {}
    with open(path) as f:
        for case, name, grid in json.load(f):
            m = re.search(r"int8_tiles_kernel<.*?Tile<([\d, ]+), \d+, (?:true|false)>, \(w4a8::Out8\)\d+, (true|false), ", name)
            found.setdefault(tuple(case), []).append((m.group(1), m.group(2) == "true", grid))
    return found


def test_every_dense_tile_is_reached(tiles):
    assert torch.cuda.get_device_properties(0).multi_processor_count == CUS
    for tile, shapes in DENSE.items():
        for shape in shapes:
            assert [t[:2] for t in tiles[shape]] == [(tile, shape[2] % STEP != 0)], shape
        assert {K % STEP != 0 for _, _, K in shapes} == {False, True}
    for tile, (M, N) in SEVERAL.items():
        wt, wn, ft, fn = (int(v) for v in tile.split(", ")[:4])
        count = -(-M // (wt * ft * 32)) * -(-N // (wn * fn * 32))
        assert all(tiles[s][0][2] < count for s in DENSE[tile] if s[:2] == (M, N)), tile


def test_every_tile_of_a_layer_is_reached(tiles):
    for (first, second), shapes in LAYER.items():
        for shape in shapes:
            for dtype in (torch.bfloat16, torch.float16):
                got = [t[:2] for t in tiles[(*shape, str(dtype))]]
                assert got == [(first, shape[3] % STEP != 0), (second, shape[4] % STEP != 0)], shape
        assert {s[3] % STEP for s in shapes} == {s[4] % STEP for s in shapes} == {0, 64}


def weights(g, *shape):
    return (torch.randint(-128, 128, shape, generator=g, dtype=torch.int8, device=DEV),
            torch.rand(shape[:-1], generator=g, device=DEV) * 2e-3 + 1e-5)


def rows(g, M, K):
    return torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device=DEV), torch.rand((M, 1), generator=g, device=DEV) * 0.05 + 0.001


@pytest.mark.parametrize("M,N,K", [s for shapes in DENSE.values() for s in shapes])
def test_dense(M, N, K):
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    (x, xs), (w, ws) = rows(g, M, K), weights(g, N, K)
    bias = torch.randn((N,), generator=g, device=DEV) * 10
    # (fp64 sums of whole numbers below 2^53 are exact in any order)
    part = (x.double() @ w.double().t()) * xs.double() * ws.double()
    for dtype in (torch.bfloat16, torch.float16):
        for b in (None, bias):
            ref = part if b is None else part + b.double()
            # the sum, the scales' product and their product; the sum with the bias, or its rounding; the output's
            off = part.abs() * 3 * O.U32 + ref.abs() * O.U32
            tol = off * (1 + 8 * O.U32) + (ref.abs() + off) * HALF[dtype] + (2.0 ** -25 if dtype == torch.float16 else 0)
            y = W.int8_gemm(x, xs, w, ws, bias=b, out_dtype=dtype)
            assert bool(((y.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("T,k,E,H,I", [s for shapes in LAYER.values() for s in shapes])
def test_layer(T, k, E, H, I):
    """Against calls of few tokens, whose experts are streamed: the same bits."""
    g = torch.Generator(device=DEV).manual_seed(T + E + H + I)
    (w13, s13), (w2, s2) = weights(g, E, 2 * I, H), weights(g, E, H, I)
    ids = torch.randint(0, E, (T, k), generator=g, device=DEV, dtype=torch.int32)
    tw = torch.rand((T, k), generator=g, device=DEV)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn((T, H), generator=g, device=DEV).to(dtype)
        y = W.moe_int8_apply(x, w13, w2, s13 * 0.1, s2, tw, ids)
        few = [W.moe_int8_apply(x[t:t + 30], w13, w2, s13 * 0.1, s2, tw[t:t + 30], ids[t:t + 30]) for t in range(0, T, 30)]
        assert torch.equal(y, torch.cat(few))
