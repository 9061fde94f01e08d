"""Block-scaled fp8 operators without a GPU: what they refuse, workspace sizes, fake implementations
for traced programs, and the oracle's roundings against torch's."""
import numpy as np
import pytest
import torch

import w4a8_fp8_wmma as W
from oracle import fp8_block as O
from w4a8_fp8_wmma import _lib

L = _lib.lib
F16, BF16, E4M3 = 0, 1, 2
FP8 = torch.float8_e4m3fn
INVALID, WORKSPACE = 1, 3


def err():
    return L.w4a8_last_error().decode()


# ------------------------------------------------------------------ the oracle's roundings
def test_oracle_rounds_to_e4m3_as_torch_does():
    codes = torch.arange(256, dtype=torch.uint8).view(FP8).double()
    real = codes[~codes.isnan()].numpy()
    assert np.array_equal(O.round_e4m3(real), real)
    edges = np.unique(real)
    mid = (edges[1:] + edges[:-1]) / 2                  # ties
    near = np.concatenate([mid, np.nextafter(mid.astype(np.float32), np.float32(np.inf)).astype(np.float64),
                           np.nextafter(mid.astype(np.float32), np.float32(-np.inf)).astype(np.float64)])
    want = torch.from_numpy(near.astype(np.float32)).to(FP8).double().numpy()
    assert np.array_equal(O.round_e4m3(near.astype(np.float32)), want)
    assert O.round_e4m3(1e9) == 448 and O.round_e4m3(-np.inf) == -448 and np.isnan(O.round_e4m3(np.nan))


@pytest.mark.parametrize("K", [1, 127, 128, 129, 400])
def test_oracle_quantises_as_fp32_arithmetic_does(K):
    x = torch.randn((5, K), generator=torch.Generator().manual_seed(K)).bfloat16().float()
    x[0] = 0
    q, s = O.quantise(x.double().numpy())
    for g in range(-(-K // 128)):
        part = x[:, 128 * g:128 * (g + 1)]
        # (a tensor as divisor: a number would be multiplied by its reciprocal)
        ts = (part.abs().amax(1) / torch.tensor(448.0)).clamp_min(1e-8)
        tq = (part * (1.0 / ts)[:, None]).to(FP8).double().numpy()
        assert np.array_equal(s[:, g], ts.numpy())
        assert np.array_equal(q[:, 128 * g:128 * (g + 1)], tq)


# ------------------------------------------------------------------ the C entries
P16 = 4096                                              # an address that is aligned and never read


def gemm(**k):
    a = dict(x=P16, xd=E4M3, xs=P16, M=4, K=128, ldx=128, w=P16, ws=P16, N=64, out=P16, od=BF16, work=None, nb=0)
    a.update(k)
    return L.w4a8_fp8_block_gemm(*a.values(), None)


@pytest.mark.parametrize("bad,says", [
    (dict(K=0, ldx=0), "sizes"), (dict(N=0), "sizes"), (dict(M=-1), "sizes"), (dict(K=120, ldx=128), "multiple of 16"),
    (dict(K=1 << 25, ldx=1 << 25), "2^24"), (dict(xd=3), "e4m3"), (dict(x=None), "null"), (dict(w=None), "null"),
    (dict(ws=None), "null"), (dict(xs=None), "scales"), (dict(out=None), "null"), (dict(ldx=120), "16 bytes"),
    (dict(ldx=136), "16 bytes"), (dict(x=P16 + 8), "aligned"), (dict(w=P16 + 8), "aligned"), (dict(od=E4M3), "out"),
    (dict(M=(1 << 31)), "sizes")])
def test_dense_refusals(bad, says):
    assert gemm(**bad) == INVALID and says in err()


def test_dense_workspace():
    size = L.w4a8_fp8_block_gemm_workspace_size
    assert size(E4M3, 1000, 4096) == 0 and size(BF16, 16, 4096) == 0 and size(BF16, 0, 128) == 0
    need = size(BF16, 17, 400)
    assert need >= 17 * 400 + 17 * 4 * 4
    assert gemm(xd=BF16, xs=None, M=17, K=400, ldx=400) == WORKSPACE and "workspace" in err()
    assert gemm(xd=BF16, xs=None, M=17, K=400, ldx=400, work=P16, nb=need - 1) == WORKSPACE
    assert gemm(M=0, x=None, w=None) == 0


def grouped(**k):
    a = dict(x=P16, xs=P16, rows=8, K=128, ldx=128, w=P16, ws=P16, E=4, N=64, sti=P16, P=64, eid=P16, ntp=P16,
             slots=16, top_k=2, block=16, gather=1, out=P16, od=BF16)
    a.update(k)
    return L.w4a8_moe_fp8_block_gemm(*a.values(), None)


@pytest.mark.parametrize("bad,says", [
    (dict(block=8), "block_m"), (dict(block=144), "block_m"), (dict(P=40), "divisible"), (dict(P=-16), "sizes"),
    (dict(top_k=0), "sizes"), (dict(slots=-1), "sizes"), (dict(slots=17), "more slots"), (dict(sti=None), "null"),
    (dict(eid=None), "null"), (dict(ntp=None), "null"), (dict(out=None), "null"), (dict(E=0), "sizes"),
    (dict(xs=None), "scales"), (dict(K=136, ldx=144), "multiple of 16"), (dict(od=7), "out")])
def test_grouped_refusals(bad, says):
    assert grouped(**bad) == INVALID and says in err()


def layer(**k):
    a = dict(x=P16, xd=BF16, xs=None, T=4, H=256, I=128, E=4, top_k=2, w13=P16, s13=P16, w2=P16, s2=P16, tw=P16,
             ids=P16, emap=None, ng=0, out=P16, od=BF16, work=P16, nb=1 << 40)
    a.update(k)
    return L.w4a8_moe_fp8_block_apply(*a.values(), None)


@pytest.mark.parametrize("bad,says", [
    (dict(H=192), "128"), (dict(I=64), "128"), (dict(top_k=0), "top_k"), (dict(top_k=1025), "top_k"), (dict(T=-1), "sizes"),
    (dict(T=1 << 31), "sizes"), (dict(xd=E4M3), "scales"), (dict(ng=8), "expert_map"), (dict(E=2000), "too many experts"),
    (dict(w2=None), "null"), (dict(tw=None), "null"), (dict(ids=None), "null"), (dict(out=None), "null"),
    (dict(w2=P16 + 8), "aligned"), (dict(out=P16 + 2), "aligned"), (dict(od=E4M3), "out"), (dict(w13=None), "null")])
def test_layer_refusals(bad, says):
    assert layer(**bad) == INVALID and says in err()


def test_layer_workspace():
    size = L.w4a8_moe_fp8_block_workspace_size
    assert size(0, 256, 128, 4, 2) == 0
    few, many = size(4, 256, 128, 4, 2), size(400, 256, 128, 4, 2)
    assert few >= 8 * 256 * 4 and many >= 400 * 256 + 800 * 256 * 2
    for T, need in ((4, few), (400, many)):
        assert layer(T=T, nb=need - 1) == WORKSPACE and "workspace" in err()
        assert layer(T=T, work=None) == WORKSPACE
    assert layer(T=0) == 0


def norm(**k):
    a = dict(x=P16, xd=BF16, rows=2, H=256, ldx=256, r=None, ldr=0, w=P16, wf=0, eps=1e-6, per_row=0, ro=None, no=None,
             q=P16, s=P16)
    a.update(k)
    return L.w4a8_rms_norm_quant_fp8(*a.values(), None)


@pytest.mark.parametrize("bad,says", [
    (dict(xd=E4M3), "fp16 or bf16"), (dict(rows=-1), "sizes"), (dict(H=0), "sizes"), (dict(x=None), "null"),
    (dict(w=None), "null"), (dict(q=None), "null"), (dict(s=None), "null"), (dict(r=P16, ldr=256), "go together"),
    (dict(ro=P16), "go together"), (dict(rows=1 << 24, H=7, ldx=7), "too many rows"),
    (dict(rows=1 << 30), "too many rows"), (dict(ldx=255), "overlap"), (dict(r=P16, ro=P16, ldr=100), "overlap")])
def test_norm_refusals(bad, says):
    assert norm(**bad) == INVALID and says in err()


@pytest.mark.parametrize("bad,says", [
    (dict(xd=E4M3), "fp16 or bf16"), (dict(rows=-1), "sizes"), (dict(K=0), "sizes"), (dict(x=None), "null"),
    (dict(q=None), "null"), (dict(s=None), "null"), (dict(ldx=255), "overlap"), (dict(silu=1, ldx=300), "overlap"),
    (dict(rows=1 << 30), "too many groups"), (dict(rows=1 << 26, K=7, ldx=7), "too many groups")])
def test_quant_refusals(bad, says):
    a = dict(x=P16, xd=BF16, rows=2, K=256, ldx=256, silu=0, q=P16, s=P16)
    a.update(bad)
    assert L.w4a8_act_quant_fp8_block(*a.values(), None) == INVALID and says in err()


# ------------------------------------------------------------------ the Python entries
def f8(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(FP8)


def f32(*shape):
    return torch.ones(shape)


def b16(*shape):
    return torch.ones(shape, dtype=torch.bfloat16)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("call,says", [
    (lambda: W.rms_norm_quant_fp8(f32(2, 8), f32(8)), "fp16/bf16"),
    (lambda: W.rms_norm_quant_fp8(b16(8), b16(8)), "fp16/bf16"),
    (lambda: W.rms_norm_quant_fp8(b16(2, 0), b16(0)), "no columns"),
    (lambda: W.rms_norm_quant_fp8(b16(2, 8), b16(9)), "weight"),
    (lambda: W.rms_norm_quant_fp8(b16(2, 8), b16(8).half()), "weight"),
    (lambda: W.rms_norm_quant_fp8(b16(2, 8), b16(8), residual=b16(3, 8)), "residual"),
    (lambda: W.rms_norm_quant_fp8(b16(2, 8), b16(8), group_size=64), "group_size"),
    (lambda: W.rms_norm_quant_fp8(b16(2, 8), b16(8)), "CUDA"),
    (lambda: W.act_quant_fp8_block(f32(2, 8)), "fp16/bf16"),
    (lambda: W.act_quant_fp8_block(b16(2, 8), activation="gelu"), "activation"),
    (lambda: W.act_quant_fp8_block(b16(2, 9), activation="silu"), "gate"),
    (lambda: W.act_quant_fp8_block(b16(2, 0)), "no columns"),
    (lambda: W.act_quant_fp8_block(b16(2, 8)), "CUDA"),
    (lambda: W.fp8_block_gemm(f8(2, 128), None, f8(8, 128), f32(1, 1)), "scales"),
    (lambda: W.fp8_block_gemm(f8(2, 128), f32(2, 2), f8(8, 128), f32(1, 1)), "x_scales"),
    (lambda: W.fp8_block_gemm(b16(2, 128), f32(2, 1), f8(8, 128), f32(1, 1)), "e4m3 rows only"),
    (lambda: W.fp8_block_gemm(f32(2, 128), None, f8(8, 128), f32(1, 1)), "x must be"),
    (lambda: W.fp8_block_gemm(b16(2, 128), None, f8(8, 144), f32(1, 2)), "w must be"),
    (lambda: W.fp8_block_gemm(b16(2, 128), None, f8(8, 128), f32(1, 2)), "w scales"),
    (lambda: W.fp8_block_gemm(b16(2, 128), None, f8(128, 8).t(), f32(1, 1)), "contiguous"),
    (lambda: W.fp8_block_gemm(b16(2, 128), None, f8(8, 128), f32(1, 1), out_dtype=torch.float32), "out_dtype"),
    (lambda: W.fp8_block_gemm(b16(2, 128), None, f8(8, 128), f32(1, 1)), "CUDA")])
def test_python_refusals(call, says):
    with pytest.raises(RuntimeError, match=says):
        call()


@pytest.mark.parametrize("bad,says", [
    (dict(x=b16(4, 128), x_scales=None), "float8_e4m3fn"), (dict(w=f8(8, 128)), "w must be"),
    (dict(sorted_token_ids=torch.zeros(32, dtype=torch.int64)), "int32"), (dict(block_m=24), "block_m"),
    (dict(block_m=0), "block_m"), (dict(top_k=0), "top_k"), (dict(expert_ids=i32(3)), "expert_ids"),
    (dict(num_tokens_post_padded=i32(2)), "expert_ids"), (dict(out=b16(31, 8)), "out must be"),
    (dict(out=b16(32, 16)[:, :8]), "out must be"), (dict(out_dtype=torch.float32), "out_dtype"),
    (dict(), "CUDA")])
def test_python_grouped_refusals(bad, says):
    a = dict(x=f8(4, 128), x_scales=f32(4, 1), w=f8(2, 8, 128), w_scales=f32(2, 1, 1), sorted_token_ids=i32(32),
             expert_ids=i32(2), num_tokens_post_padded=i32(1), top_k=2, block_m=16)
    a.update(bad)
    with pytest.raises(RuntimeError, match=says):
        W.moe_fp8_block_gemm(**a)


@pytest.mark.parametrize("bad,says", [
    (dict(x=b16(4, 200), w13=f8(2, 256, 200), w2=f8(2, 200, 128)), "multiples of 128"), (dict(w13=f8(2, 255, 256)), "w13"),
    (dict(w2=f8(2, 256, 256)), "w2"), (dict(w13_scales=f32(2, 2, 1)), "w13 scales"), (dict(topk_ids=i32(3, 2)), "topk_ids"),
    (dict(topk_ids=i32(4, 0)), "topk_ids"), (dict(topk_weights=f32(4, 3)), "topk_weights"),
    (dict(global_num_experts=4), "expert_map"), (dict(expert_map=i32(2, 2)), "1-d"),
    (dict(expert_map=i32(6), global_num_experts=4), "expert count"), (dict(out_dtype=torch.float32), "out_dtype"),
    (dict(), "CUDA")])
def test_python_layer_refusals(bad, says):
    a = dict(x=b16(4, 256), w13=f8(2, 256, 256), w2=f8(2, 256, 128), w13_scales=f32(2, 2, 2), w2_scales=f32(2, 2, 1),
             topk_weights=f32(4, 2), topk_ids=i32(4, 2))
    a.update(bad)
    with pytest.raises(RuntimeError, match=says):
        W.moe_fp8_block_apply(**a)


def test_fake_implementations():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.w4a8_fp8_wmma
    with FakeTensorMode():
        cuda = dict(device="cuda")
        x = torch.empty((5, 384), dtype=torch.bfloat16, **cuda)
        nw = torch.empty((384,), dtype=torch.bfloat16, **cuda)
        q, s, z, y = ops.rms_norm_quant_fp8(x, nw, 1e-6, x, 128, False)
        assert q.shape == (5, 384) and q.dtype == FP8 and s.shape == (5, 3) and z.shape == (5, 384) and y.shape == (0,)
        assert ops.rms_norm_quant_fp8(x, nw, 1e-6, None, 0, True)[1].shape == (5, 1)
        q2, s2 = ops.act_quant_fp8_block(x, "silu")
        assert q2.shape == (5, 192) and s2.shape == (5, 2)
        w, ws = torch.empty((70, 384), dtype=FP8, **cuda), torch.empty((1, 3), **cuda)
        out = ops.fp8_block_gemm(q, s, w, ws, torch.float16)
        assert out.shape == (5, 70) and out.dtype == torch.float16 and out.device.type == "cuda"
        ids = torch.empty((64,), dtype=torch.int32, **cuda)
        got = ops.moe_fp8_block_gemm(q, s, w[None], ws[None], ids, ids[:4], ids[:1], 1, 16, torch.bfloat16)
        assert got.shape == (64, 70)
        got = ops.moe_fp8_block_apply(q, w[None], w[None], ws[None], ws[None], x[:, :2].float(), ids[:10].view(5, 2), s,
                                      None, torch.bfloat16)
        assert got.shape == (5, 384) and got.dtype == torch.bfloat16
