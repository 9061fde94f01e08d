"""int8 operators and the expert choice without a GPU: what they refuse, workspace sizes, fake implementations for
traced programs, the second library's exports and its matrix-core waits, and the oracle against plain arithmetic."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import test_cpu_mfma_waits as waits
import w4a8_fp8_wmma as W
from oracle import int8 as O
from w4a8_fp8_wmma import _lib, _lib8

L = _lib8.lib
F16, BF16, E4M3, INT8, F32 = 0, 1, 2, 3, 4
INVALID, WORKSPACE = 1, 3
P16 = 4096                                              # an address that is aligned and never read
HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "w4a8_int8.h")


def err():
    return L.w4a8_int8_last_error().decode()


# ------------------------------------------------------------------ the library
def test_library_exports_exactly_the_header():
    syms = sorted(set(re.findall(r"W4A8_API\s+[\w\s\*]+?\b(w4a8_\w+)\s*\(", open(HEADER).read())))
    out = subprocess.run(["nm", "-D", "--defined-only", str(_lib8.LIB_PATH)], capture_output=True, text=True,
                         check=True).stdout
    assert sorted(l.split()[-1] for l in out.splitlines() if " T " in l and "w4a8_" in l) == syms
    assert sorted(_lib8.SIGNATURES) == syms
    assert L.w4a8_int8_abi_version() == 1


@pytest.mark.skipif(not os.path.exists(waits.OBJDUMP), reason="needs the ROCm toolchain's llvm-objdump")
def test_every_mfma_result_is_waited_for(tmp_path, monkeypatch):
    monkeypatch.setitem(waits.PASSES, "v_mfma_i32_16x16x64_i8", 4)
    monkeypatch.setitem(waits.PASSES, "v_mfma_i32_32x32x32_i8", 8)
    mfmas, found = 0, []
    for n, obj in enumerate(waits.code_objects(_lib8.LIB_PATH)):
        path = tmp_path / f"{n}.o"
        path.write_bytes(obj)
        text = subprocess.run([waits.OBJDUMP, "-d", str(path)], capture_output=True, text=True, check=True).stdout
        for name, code in waits.parse(text.splitlines()):
            mfmas += sum(op.startswith("v_mfma") for _, op, _ in code)
            found += [(name, *f) for f in waits.too_early(code)]
    assert mfmas > 10 and not found, found[:8]


# ------------------------------------------------------------------ the C entries
def gemm(**k):
    a = dict(x=P16, xd=INT8, xs=P16, M=4, K=128, ldx=128, w=P16, ws=P16, N=64, bias=None, bf=0, out=P16, od=BF16, work=None,
             nb=0)
    a.update(k)
    return L.w4a8_int8_gemm(*a.values(), None)


@pytest.mark.parametrize("bad,says", [
    (dict(K=0, ldx=0), "sizes"), (dict(N=0), "sizes"), (dict(M=-1), "sizes"), (dict(K=120, ldx=128), "multiple of 16"),
    (dict(K=131072, ldx=131072), "131071"), (dict(xd=E4M3), "int8"), (dict(xd=F32), "int8"), (dict(x=None), "null"),
    (dict(w=None), "null"), (dict(ws=None), "null"), (dict(xs=None), "scales"), (dict(out=None), "null"),
    (dict(ldx=112), "16 bytes"), (dict(ldx=136), "16 bytes"), (dict(x=P16 + 8), "aligned"), (dict(w=P16 + 8), "aligned"),
    (dict(od=INT8), "out"), (dict(M=1 << 31), "sizes"), (dict(N=1 << 25), "2^24")])
def test_dense_refusals(bad, says):
    assert gemm(**bad) == INVALID and says in err()


def test_dense_workspace():
    size = L.w4a8_int8_gemm_workspace_size
    assert size(INT8, 0, 4096, 64) == 0 and size(BF16, 0, 128, 64) == 0
    assert size(BF16, 1, 4096, 4096) == 0 and size(BF16, 1, 4096, 65536) >= 4096 + 4
    need = size(BF16, 4097, 400, 64)
    assert need >= 4097 * 400 + 4097 * 4
    assert gemm(xd=BF16, xs=None, M=4097, K=400, ldx=400) == WORKSPACE and "workspace" in err()
    assert gemm(xd=BF16, xs=None, M=4097, K=400, ldx=400, work=P16, nb=need - 1) == WORKSPACE
    assert gemm(M=0, x=None, w=None) == 0


def apply(**k):
    a = dict(x=P16, xd=BF16, xs=None, T=4, H=256, I=128, E=8, k=2, w13=P16, s13=P16, w2=P16, s2=P16, tw=P16, ids=P16,
             emap=None, ng=0, out=P16, od=BF16, work=P16, nb=1 << 30)
    a.update(k)
    return L.w4a8_moe_int8_apply(*a.values(), None)


@pytest.mark.parametrize("bad,says", [
    (dict(H=200), "multiples of 64"), (dict(I=96), "multiples of 64"), (dict(H=0), "multiples of 64"),
    (dict(k=0), "top_k"), (dict(k=1025), "top_k"), (dict(T=-1), "sizes"), (dict(xd=E4M3), "int8"),
    (dict(xd=INT8), "scales"), (dict(w13=None), "null"), (dict(w2=None), "null"), (dict(s2=None), "null"),
    (dict(tw=None), "null"), (dict(ids=None), "null"), (dict(out=None), "null"), (dict(od=INT8), "out"),
    (dict(ng=16), "expert_map"), (dict(E=1025), "experts"), (dict(w2=P16 + 8), "aligned"), (dict(out=P16 + 8), "aligned"),
    (dict(T=1 << 30), "sizes"), (dict(H=131072), "131071")])
def test_layer_refusals(bad, says):
    assert apply(**bad) == INVALID and says in err()


def test_layer_workspace():
    need = L.w4a8_moe_int8_workspace_size(4, 256, 128, 8, 2)
    assert need > 0 and L.w4a8_moe_int8_workspace_size(0, 256, 128, 8, 2) == 0
    assert apply(nb=need - 1) == WORKSPACE and "workspace" in err()
    assert apply(work=None) == WORKSPACE
    assert apply(T=0, x=None) == 0


def test_quant_refusals():
    def q(x=P16, xd=BF16, R=4, K=64, ld=64, silu=0, out=P16, s=P16):
        return L.w4a8_act_quant_int8(x, xd, R, K, ld, silu, out, s, None)
    for bad in (dict(xd=INT8), dict(K=0), dict(R=-1), dict(x=None), dict(out=None), dict(s=None), dict(ld=63),
                dict(silu=1, ld=127), dict(K=(1 << 24) + 1, ld=1 << 25)):
        assert q(**bad) == INVALID
    assert q(R=0, x=None) == 0


def route(**k):
    a = dict(l=P16, dt=F32, T=4, E=64, ld=64, k=4, sc=0, bias=None, g=1, tg=1, rn=1, scale=1.0, tw=P16, ids=P16)
    a.update(k)
    return _lib.lib.w4a8_route_topk(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(dt=INT8), dict(dt=E4M3), dict(T=-1), dict(E=0), dict(E=1025, ld=1025), dict(k=0), dict(k=65), dict(k=5, E=4, ld=4),
    dict(sc=2), dict(g=0), dict(g=7), dict(g=65, E=65, ld=65), dict(tg=0), dict(g=4, tg=5), dict(g=8, tg=1, k=9),
    dict(l=None), dict(tw=None), dict(ids=None), dict(ld=63), dict(T=1 << 25)])
def test_route_refusals(bad):
    assert route(**bad) == INVALID and "route_topk" in _lib.lib.w4a8_last_error().decode()
    assert route(T=0, l=None) == 0


# ------------------------------------------------------------------ Python
def i8(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def f32(*shape):
    return torch.ones(shape)


@pytest.mark.parametrize("call,says", [
    (lambda: W.int8_gemm(i8(2, 64), None, i8(8, 64), f32(8)), "scales"),
    (lambda: W.int8_gemm(f32(2, 64).half(), f32(2), i8(8, 64), f32(8)), "int8 rows only"),
    (lambda: W.int8_gemm(f32(2, 64), None, i8(8, 64), f32(8)), "int8, fp16 or bf16"),
    (lambda: W.int8_gemm(i8(2, 64), f32(3), i8(8, 64), f32(8)), "x_scales"),
    (lambda: W.int8_gemm(i8(2, 64), f32(2).double(), i8(8, 64), f32(8)), "x_scales"),
    (lambda: W.int8_gemm(i8(2, 64), f32(2), i8(8, 80), f32(8)), "w must be"),
    (lambda: W.int8_gemm(i8(2, 64), f32(2), i8(8, 64).half(), f32(8)), "w must be"),
    (lambda: W.int8_gemm(i8(2, 64), f32(2), i8(8, 64), f32(8, 2)), "w scales"),
    (lambda: W.int8_gemm(i8(2, 64), f32(2), i8(64, 8).t(), f32(8)), "contiguous"),
    (lambda: W.int8_gemm(i8(2, 64), f32(2), i8(8, 64), f32(8), bias=f32(9)), "bias"),
    (lambda: W.int8_gemm(i8(2, 64), f32(2), i8(8, 64), f32(8), bias=f32(8).half()), "bias"),
    (lambda: W.int8_gemm(i8(2, 64), f32(2), i8(8, 64), f32(8), out_dtype=torch.float32), "out_dtype"),
    (lambda: W.int8_gemm(i8(2, 64), f32(2), i8(8, 64), f32(8)), "CUDA"),
    (lambda: W.act_quant_int8(i8(2, 64)), "fp16/bf16"), (lambda: W.act_quant_int8(f32(2, 64).half(), "gelu"), "activation"),
    (lambda: W.act_quant_int8(f32(2, 63).half(), "silu"), "2 K"), (lambda: W.act_quant_int8(f32(2, 0).half()), "columns"),
    (lambda: W.moe_int8_apply(i8(2, 64), i8(4, 128, 64), i8(4, 64, 64), f32(4, 128), f32(4, 64), f32(2, 2), i8(2, 2)), "scales"),
    (lambda: W.moe_int8_apply(f32(2, 96).half(), i8(4, 128, 96), i8(4, 96, 64), f32(4, 128), f32(4, 96), f32(2, 2), i8(2, 2)),
     "multiples of 64"),
    (lambda: W.moe_int8_apply(f32(2, 64).half(), i8(4, 128, 64), i8(4, 64, 64), f32(4, 128), f32(4, 64), f32(2, 2), i8(3, 2)),
     "topk_ids"),
    (lambda: W.moe_int8_apply(f32(2, 64).half(), i8(4, 128, 64), i8(4, 64, 64), f32(4, 128), f32(4, 64), f32(2, 3), i8(2, 2)),
     "topk_weights"),
    (lambda: W.moe_int8_apply(f32(2, 64).half(), i8(4, 128, 64), i8(4, 64, 64), f32(4, 64), f32(4, 64), f32(2, 2), i8(2, 2)),
     "w13 scales"),
    (lambda: W.moe_int8_apply(f32(2, 64).half(), i8(4, 128, 64), i8(4, 64, 64), f32(4, 128), f32(4, 64), f32(2, 2), i8(2, 2),
                              global_num_experts=8), "expert_map"),
    (lambda: W.route_topk(i8(2, 8), 2), "router_logits"), (lambda: W.route_topk(f32(2, 8), 2, scoring="relu"), "scoring"),
    (lambda: W.route_topk(f32(2, 8), 2, bias=f32(7)), "bias"), (lambda: W.route_topk(f32(2, 8), 2, bias=f32(8).half()), "bias"),
    (lambda: W.route_topk(f32(2, 8), 2), "CUDA")])
def test_python_refusals(call, says):
    with pytest.raises(RuntimeError, match=says):
        call()


def test_fake_implementations():
    ops = torch.ops.w4a8_fp8_wmma
    with torch._subclasses.FakeTensorMode():
        x = torch.empty((5, 128), dtype=torch.bfloat16, device="cuda")
        q, s = ops.act_quant_int8(x, None)
        assert q.shape == (5, 128) and q.dtype == torch.int8 and s.shape == (5, 1) and s.dtype == torch.float32
        q, s = ops.act_quant_int8(x, "silu")
        assert q.shape == (5, 64)
        w, ws = torch.empty((96, 128), dtype=torch.int8, device="cuda"), torch.empty((96,), device="cuda")
        y = ops.int8_gemm(x, None, w, ws, None, torch.float16)
        assert y.shape == (5, 96) and y.dtype == torch.float16
        w13, w2 = (torch.empty((4, 2 * 64, 128), dtype=torch.int8, device="cuda"),
                   torch.empty((4, 128, 64), dtype=torch.int8, device="cuda"))
        l = torch.empty((5, 4), device="cuda")
        tw, ids = ops.route_topk(l, 2, "sigmoid", None, 1, 1, True, 1.0)
        assert tw.shape == ids.shape == (5, 2) and ids.dtype == torch.int32 and tw.dtype == torch.float32
        y = ops.moe_int8_apply(x, w13, w2, torch.empty((4, 128), device="cuda"), torch.empty((4, 128), device="cuda"), tw, ids,
                               None, None, torch.bfloat16)
        assert y.shape == (5, 128) and y.dtype == torch.bfloat16


# ------------------------------------------------------------------ the oracle
def test_oracle_quantises_as_fp32_arithmetic_does():
    g = torch.Generator().manual_seed(1)
    for dt in (torch.bfloat16, torch.float16):
        x = torch.randn((64, 200), generator=g).to(dt)
        x[0] = 0
        x[1, :2] = torch.tensor([1.5, 0.75], dtype=dt)           # 63.5: a border
        x[1, 2:] *= 0.1
        q, s = O.quantise(x.double().numpy())
        top = x.float().abs().amax(1, keepdim=True).clamp_min(O.LEAST)
        assert np.array_equal(q, torch.round(x.float() * 127 / top).numpy())
        assert np.array_equal(s, (top / torch.full_like(top, 127.0)).numpy())
        assert q[1, 1] == 64 and not q[0].any()
    q, s = O.quantise(np.array([[1.0, np.inf], [np.nan, 1.0], [2.0, -1.0]]))
    assert np.isnan(s[:2]).all() and not q[:2].any() and list(q[2]) == [127, -64]


def test_oracle_silu_far():
    g = np.array([-1000.0, -800.0, -90.0, 0.0, 5.0])
    with np.errstate(all="ignore"):
        assert np.allclose(O.silu_mul(g[2:], np.ones(3)), g[2:] / (1 + np.exp(-g[2:])))
    assert O.silu_mul(np.array([-800.0]), np.array([1e300]))[0] == pytest.approx(-800 * np.exp(-400.0) * (np.exp(-400.0) * 1e300))


def test_oracle_routes_by_hand():
    l = np.array([[0.0, 2.0, 2.0, -1.0, 1.0, 0.5]])
    w, ids = O.route(l, 2, "softmax", None, 1, 1, True, 1.0)
    assert list(ids[0]) == [1, 2] and np.allclose(w, 0.5)
    w, ids = O.route(l, 2, "sigmoid", np.array([0, 0, 0, 9.0, 0, 0]), 3, 1, True, 2.0)
    assert list(ids[0]) == [3, 2]                                # the group of 2 and 3
    p = 1 / (1 + np.exp(-l[0]))
    assert np.allclose(w[0], 2 * p[[3, 2]] / p[[3, 2]].sum())
    w, ids = O.route(np.full((1, 4), -np.inf), 2, "softmax", None, 2, 1, True, 1.0)
    assert list(ids[0]) == [-1, -1] and not w.any()


def test_layer_oracle_counts_borders():
    """A value of h on a border may fall on either side: the tolerance holds a step of it, and no more elsewhere."""
    rng = np.random.default_rng(0)
    q = rng.integers(-127, 128, (6, 64))
    w13, w2 = rng.integers(-127, 128, (128, 64)), rng.integers(-127, 128, (64, 64))
    s13, s2 = np.full(128, 1e-4, np.float32), np.full(64, 0.01, np.float32)
    y, tol = O.expert(q, np.full((6, 1), 0.02, np.float32), w13, s13, w2, s2)
    # (a border is near for about one value in 10^3: most rows have roundings only)
    assert np.median(tol.max(1)) < 1e-4 * np.abs(y).max()
    # gate 0 has silu(0) = 0; all h equal but one at half of the largest, times 127: 63.5
    w13 = np.zeros((128, 64), np.int64)
    w13[:64, 0] = 100
    w13[64:, 0] = 100
    w13[64, 0] = 50
    y, tol = O.expert(q, np.full((6, 1), 0.02, np.float32), w13, s13, w2, s2)
    rows = q[:, 0] != 0
    gu, _ = O.product(q, np.full((6, 1), 0.02, np.float32), w13, s13)
    hs = O.quantise(O.silu_mul(gu[:, :64], gu[:, 64:]))[1]
    step = np.abs(w2[:, 0]) * 0.01 * hs
    assert (tol[rows] >= step[rows] * 0.999).all() and (tol[rows] < step[rows] + 1e-4 * np.abs(y).max()).all()
