"""Block-scaled fp8 tiles: sizes that reach every one of them (checked by the names of the kernels that ran), and
work-groups that take two column tiles one after the other (checked by the size of the grid)."""
import json
import os
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

import fp8_layer_check as C
import test_gpu_fp8_block_sizes as S
import w4a8_fp8_wmma as W
from oracle import fp8_block as O
from test_gpu_fp8_layer_error import args_of, dev, rows_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
CUS = 256

# tile (waves by rows, by columns, row and column fragments a wave, parts of K): (M, N, K), K with and without a
# partial group, groups that the parts of K do not divide, odd N
DENSE = {"2, 2, 2, 1, 4": [(17, 1001, 4096), (33, 4101, 2320), (40, 190, 128 * 70 + 32)],
         "2, 2, 2, 1, 2": [(48, 1003, 1040), (20, 72, 2048), (64, 8192, 16)],
         "1, 4, 4, 1, 2": [(64, 12300, 400), (100, 6001, 4112), (17, 16001, 144), (64, 12288, 384)],
         "1, 4, 4, 1, 1": [(320, 4104, 272), (321, 4099, 384)],
         "1, 4, 4, 2, 1": [(1000, 4096, 144), (700, 5003, 656), (699, 5000, 1024)],
         "4, 2, 4, 4, 1": [(2047, 4096, 128), (2040, 4085, 144), (1793, 4096, 1152)]}
# grouped, two column tiles a work-group: (T, k, E, N, K, block); an odd number of them, a K tail, rows of 4096 bytes
TWO = [(600, 4, 64, 2944, 400, 16), (600, 4, 64, 2944, 400, 64), (600, 4, 64, 2936, 4096, 64), (600, 4, 64, 2944, 4096, 16),
       (300, 8, 128, 1920, 384, 64)]
# the same for a layer's products, an odd number of tiles in both: (T, k, E, H, I)
TWO_LAYER = (700, 4, 200, 1152, 640)
BASE = 7                                                # different experts of the layer case


def column_tiles_of(grid, rows_padded, columns, bt, bn):
    """How many column tiles a work-group of a grouped launch takes, from its grid: XCDs take runs of four row tiles."""
    row_tiles, tiles = -(-rows_padded // bt), -(-columns // bn)
    run = min(4, row_tiles)
    groups = -(-(-(-row_tiles // run)) // 8) * 8 * run
    found = [c for c in (1, 2) if grid == groups * -(-tiles // c)]
    return found[0] if len(found) == 1 else None


def zeros8(*shape):
    return torch.zeros(shape, dtype=torch.uint8, device=DEV).view(FP8)


def ones(*shape):
    return torch.ones(shape, device=DEV)


def trace(path):
    """Runs every case once under torch's profiler and writes [[case, kernel, grid], ...]."""
    calls = []
    for shapes in DENSE.values():
        for M, N, K in shapes:
            a = zeros8(M, K), ones(M, -(-K // 128)), zeros8(N, K), ones(-(-N // 128), -(-K // 128))
            calls.append(((M, N, K), lambda a=a: W.fp8_block_gemm(*a)))
    for case in TWO:
        T, k, E, N, K, block = case
        ids = torch.arange(T * k, dtype=torch.int32, device=DEV).remainder(E).view(T, k)
        a = (zeros8(T, K), ones(T, -(-K // 128)), zeros8(E, N, K), ones(E, -(-N // 128), -(-K // 128)),
             *W.moe_align_block_size(ids, block, E), k, block)
        calls.append(((*case, a[4].numel()), lambda a=a: W.moe_fp8_block_gemm(*a)))
    T, k, E, H, I = TWO_LAYER
    ids = torch.arange(T * k, dtype=torch.int32, device=DEV).remainder(E).view(T, k)
    for dtype in (torch.bfloat16, torch.float16):
        a = (torch.zeros((T, H), dtype=dtype, device=DEV), zeros8(E, 2 * I, H), zeros8(E, H, I),
             ones(E, 2 * I // 128, H // 128), ones(E, H // 128, I // 128), ones(T, k), ids)
        calls.append(((*TWO_LAYER, str(dtype)), lambda a=a: W.moe_fp8_block_apply(*a)))
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
        got += [[case, e["name"], e["args"]["grid"]] for e in events if e.get("cat") == "kernel" and "_kernel" in e["name"]]
        print(case, flush=True)
    with open(path, "w") as f:
        json.dump(got, f)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """What ran, from a process of its own: the profiler's hooks stay out of this one."""
    path = str(tmp_path_factory.mktemp("trace") / "kernels.json")
    here = os.path.dirname(os.path.abspath(__file__))
    paths = [here, os.path.dirname(here), os.path.join(os.path.dirname(here), "rdna4-vllm_amd")]
    code = f"import sys; sys.path[:0] = {paths!r}; import test_gpu_fp8_tiles_reached as t; t.trace({path!r})"
    run = subprocess.run([sys.executable, "-u", "-c", code], capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stdout[-500:] + run.stderr[-2000:]
    with open(path) as f:
        return [(tuple(case), name, grid) for case, name, grid in json.load(f)]


def tiles_of(kernels, case):
    """[(tile, Dst, grid)] of a case's tile kernels."""
    found = []
    for c, name, grid in kernels:
        m = re.search(r"block_tiles_kernel<.*?TileCfg<([\d, ]+), \d+>, \(w4a8::Dst\)(\d+)", name)
        if c == case and m:
            found.append((m.group(1), int(m.group(2)), grid[0]))
    return found


def test_every_dense_tile_is_reached(kernels):
    assert torch.cuda.get_device_properties(0).multi_processor_count == CUS
    for tile, shapes in DENSE.items():
        for shape in shapes:
            assert [t for t, _, _ in tiles_of(kernels, shape)] == [tile], shape


def test_two_column_tiles_are_reached(kernels):
    for case in TWO:
        P, = {c[-1] for c, _, _ in kernels if c[:-1] == case}
        (tile, _, grid), = tiles_of(kernels, (*case, P))
        assert tile == "1, 4, 4, 2, 1" and column_tiles_of(grid, P, case[3], 64, 128) == 2, case
    T, k, E, H, I = TWO_LAYER
    P = min(T * k * 64, (T * k + E * 63 + 63) // 64 * 64)
    for dtype, second in ((torch.bfloat16, 5), (torch.float16, 3)):
        (a, d1, g1), (b, d2, g2) = tiles_of(kernels, (*TWO_LAYER, str(dtype)))
        assert (a, d1, b, d2) == ("1, 8, 4, 2, 1", 4, "1, 4, 4, 2, 1", second)
        assert column_tiles_of(g1, P, I, 64, 128) == 2 and column_tiles_of(g2, P, H, 64, 128) == 2


@pytest.mark.parametrize("M,N,K", [s for shapes in DENSE.values() for s in shapes])
def test_dense(M, N, K):
    S.test_dense_tiles(M, N, K)


@pytest.mark.parametrize("T,k,E,N,K,block", TWO)
def test_group(T, k, E, N, K, block):
    """All rows and columns against float64 products made on the device; padding left as it was."""
    g = torch.Generator(device=DEV).manual_seed(T + N + K + block)
    x, w = (torch.randn(s, generator=g, device=DEV).mul_(60).clamp_(-448, 448).to(FP8) for s in ((T, K), (E, N, K)))
    xs = torch.rand((T, -(-K // 128)), generator=g, device=DEV) * 0.02 + 0.001
    ws = torch.rand((E, -(-N // 128), -(-K // 128)), generator=g, device=DEV) * 2e-4 + 1e-5
    p = torch.rand((T, E), generator=g, device=DEV)
    p[:, 1] += 0.7                                       # one expert with most tokens, one with none
    p[:, E - 1] = -1
    ids = p.argsort(1, descending=True)[:, :k].to(torch.int32)
    sti, eid, ntp = W.moe_align_block_size(ids, block, E)
    for dtype in (torch.bfloat16, torch.float16):
        out = torch.full((sti.numel(), N), 7.0, dtype=dtype, device=DEV)
        W.moe_fp8_block_gemm(x, xs, w, ws, sti, eid, ntp, k, block, out=out)
        row = torch.arange(sti.numel(), device=DEV)
        real = (row < ntp) & (sti < T * k)
        assert (out[~real] == 7.0).all() and int(real.sum()) == T * k
        a = x.double() * xs.double().repeat_interleave(128, 1)[:, :K]
        expert = eid[row // block]
        for e in torch.unique(expert[real]).tolist():
            at = row[real & (expert == e)]
            b = w[e].double() * ws[e].double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
            r = a[sti[at].long() // k]
            ref, got = r @ b.t(), out[at].double()
            # the matrix core's cuts: 2^E is at most the largest product of an eight, so seven of them lose at most
            # 7 * 2^-13 of the eight's magnitudes, and their variance is at most 7 / 3 * 2^-26 of its squares
            mag, var = r.abs() @ b.abs().t(), (r * r) @ (b * b).t() * (7 / 3 * 2.0 ** -26)
            tol = mag * (7 * 2.0 ** -13 + (256 + K // 128 + 19) * O.U32)
            err = got - ref
            assert (err.abs() <= tol + (ref.abs() + tol) * C.HALF[dtype] + 2.0 ** -25).all(), e
            own = (ref.to(dtype).double() - ref) ** 2 + var
            # (a sum of n evenly spread errors squared deviates by sqrt(0.8 / n): eight deviations for a row, and
            # for a column tile, which with few rows has some hundred values)
            for s in range(0, N, 128):
                c = slice(s, min(s + 128, N))
                assert (err[:, c] ** 2).sum() <= 1.7 ** 2 * own[:, c].sum(), (e, s)
            assert ((err ** 2).sum(1) <= 1.2 ** 2 * own.sum(1)).all(), e


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer(dtype, e4m3):
    """Experts repeat after seven; tokens sampled, from all over the batch."""
    T, k, E, H, I = TWO_LAYER
    case = C.exact_case(T, k, BASE, H, I)
    ids = np.random.default_rng(3).random((T, E)).argsort(1)[:, :k].astype(np.int32)
    x, xs = rows_of(case, dtype, e4m3)
    w13, w2, s13, s2, tw, _ = args_of(case)
    of = torch.arange(E, device=DEV) % BASE
    spread8 = lambda w: w.view(torch.uint8)[of].view(FP8)                    # noqa: E731
    out = W.moe_fp8_block_apply(x, spread8(w13), spread8(w2), s13[of], s2[of], tw, dev(ids), x_scales=xs, out_dtype=dtype)
    at = np.unique(np.linspace(0, T - 1, 60).astype(int))
    few = (case[0][at], case[1][at], *case[2:6], case[6][at], ids[at] % BASE)
    assert all(O.sums_are_exact(few[0][:4], few[1][:4], few[2][e], few[3][e]) for e in range(BASE))
    half = C.ROW_HALF if dtype == torch.bfloat16 else 0.0
    assert C.complaints(out[torch.from_numpy(at).to(DEV)].double().cpu().numpy(), dtype, O.known_layer(*few, half)) == []
