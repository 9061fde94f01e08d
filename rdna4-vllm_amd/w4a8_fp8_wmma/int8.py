"""int8 (W8A8) layers on gfx950: activation quantisation, dense products and the gated expert layer, for
checkpoints whose weights are int8 with one fp32 scale per output channel. (No reference counterpart: the
reference serves int4 and E2M1 weights.)

Activations are ``torch.int8`` rows with one fp32 scale each, as ``act_quant_int8`` makes them, or 16-bit rows
that a call quantises; weights are (N, K) or (E, N, K) ``torch.int8`` with fp32 scales (N,) or (E, N) (a last
dimension of one is taken too).

A decoder layer's expert half, as a serving program runs it::

    tw, ids = route_topk(router_logits, top_k, scoring="sigmoid", bias=balance, num_groups=8, top_groups=4)
    y = moe_int8_apply(x, w13, w2, s13, s2, tw, ids)

Plain functions over the C ABI, and the same as torch ops (``torch.ops.w4a8_fp8_wmma.*``) with fake
implementations for traced programs. Every call enqueues on torch's current stream of its tensors' device and
never synchronises. Inference only: no gradients.
"""
from __future__ import annotations

import torch

from . import _ops
from ._lib8 import check, lib
from ._ops import _fail, _ptr, _workspace
from .fp8_block import _mfma_rows, _on, _out_dtype, _rows2d, _same_device, _stream, _stride

INT8 = torch.int8
MAX_K = 131071                  # sums of larger K may pass 32 bits
_DT = {torch.float16: 0, torch.bfloat16: 1, INT8: 3}


def act_quant_int8(x: torch.Tensor, activation: str | None = None):
    """int8 rows with one fp32 scale each: (q (R, K), scales (R, 1)).

    x (R, K) fp16 / bf16, or with ``activation="silu"`` x = [gate | up] (R, 2 K), whose silu(gate) * up is
    formed in fp32. q is the whole number nearest to 127 v / a, ties to even, a = max(absmax, 127 * 2^-100) of the
    row, and the scale a / 127. A row that holds an infinity or a NaN gets the scale NaN. Rows may be strided."""
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2:
        _fail(f"x must be fp16/bf16 (R, K), got {x.dtype} {tuple(x.shape)}")
    if activation not in (None, "silu"):
        _fail(f"activation must be None or 'silu', got {activation!r}")
    R, K = x.shape
    if activation is not None:
        if K % 2 != 0:
            _fail(f"x must be [gate | up] (R, 2 K), got {tuple(x.shape)}")
        K //= 2
    if K == 0:
        _fail("x has no columns")
    dev = x.device
    _same_device(dev)
    x = _mfma_rows(x, "x") if K % 8 == 0 else _rows2d(x, "x")
    q = torch.empty((R, K), dtype=INT8, device=dev)
    s = torch.empty((R, 1), dtype=torch.float32, device=dev)
    with _on(dev):
        check(lib.w4a8_act_quant_int8(_ptr(x), _DT[x.dtype], R, K, _stride(x), 0 if activation is None else 1,
                                      _ptr(q), _ptr(s), _stream(x)), "act_quant_int8")
    return q, s


def _check_scale(s, shape, name):
    """fp32 scales of ``shape``, with or without a last dimension of one; contiguous."""
    if s.dtype != torch.float32 or s.shape != shape and s.shape != (*shape, 1):
        _fail(f"{name} must be fp32 {tuple(shape)}; got {s.dtype} {tuple(s.shape)}")
    return s if s.is_contiguous() else s.contiguous()


def _check_rows(x, x_scales):
    """int8 rows with scales, or 16-bit rows without."""
    if x.dim() != 2:
        _fail(f"x must be 2D, got {tuple(x.shape)}")
    if x.dtype == INT8:
        if x_scales is None:
            _fail("x in int8 needs its scales")
        return _check_scale(x_scales, (x.shape[0],), "x_scales")
    if x.dtype not in (torch.float16, torch.bfloat16):
        _fail(f"x must be int8, fp16 or bf16, got {x.dtype}")
    if x_scales is not None:
        _fail("x_scales go with int8 rows only")
    return None


def _check_weight(w, s, shape, name):
    """int8 weights and their channel scales; contiguous (weights are never copied)."""
    if w.dtype != INT8 or w.shape != shape:
        _fail(f"{name} must be int8 {tuple(shape)}; got {w.dtype} {tuple(w.shape)}")
    if not w.is_contiguous():
        _fail(f"{name} must be contiguous")
    if w.data_ptr() % 16 != 0:
        _fail(f"{name} must be aligned to 16 bytes")
    return _check_scale(s, shape[:-1], f"{name} scales")


def int8_gemm(x: torch.Tensor, x_scales: torch.Tensor | None, w: torch.Tensor, w_scales: torch.Tensor,
              bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Dense layer x (M, K) times w (N, K) transposed, with scales of rows and channels, -> (M, N).

    x is int8 with x_scales (M,) or (M, 1), or fp16 / bf16 with ``x_scales=None``: rows that the call quantises as
    ``act_quant_int8`` does. The sum is exact; scales and bias (N,) (fp32 or out_dtype) are applied in fp32 (the product
    of a row's and a channel's scale is formed first, and has to be a number of its range).
    out_dtype: fp16 or bf16 (default: x's, bf16 for int8 x). K must be a multiple of 16, up to 131071."""
    xs = _check_rows(x, x_scales)
    M, K = x.shape
    if w.dim() != 2:
        _fail(f"w must be (N, K), got {tuple(w.shape)}")
    N = w.shape[0]
    ws = _check_weight(w, w_scales, (N, K), "w")
    dt = _out_dtype(out_dtype if out_dtype is not None else (torch.bfloat16 if x.dtype == INT8 else x.dtype))
    if bias is not None:
        if bias.shape != (N,) or bias.dtype not in (torch.float32, dt):
            _fail(f"bias must be ({N},) in fp32 or out_dtype, got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    dev = x.device
    _same_device(dev, xs, w, ws, bias)
    x = _mfma_rows(x, "x")
    out = torch.empty((M, N), dtype=dt, device=dev)
    nbytes = 0 if xs is not None else lib.w4a8_int8_gemm_workspace_size(_DT[x.dtype], M, K, N)
    work = _workspace(nbytes, dev) if nbytes else None
    with _on(dev):
        check(lib.w4a8_int8_gemm(
            _ptr(x), _DT[x.dtype], _ptr(xs), M, K, _stride(x), _ptr(w), _ptr(ws), N, _ptr(bias),
            1 if bias is not None and bias.dtype == torch.float32 else 0, _ptr(out), _DT[dt], _ptr(work), nbytes,
            _stream(x)), "int8_gemm")
    return out


def _ids32(ids):
    """Expert ids in 32 bits. Numbers past those name no expert, whatever their low words are."""
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, (1 << 31) - 1)
    return ids.to(torch.int32).contiguous()


def moe_int8_apply(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, w13_scales: torch.Tensor,
                   w2_scales: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor,
                   x_scales: torch.Tensor | None = None, expert_map: torch.Tensor | None = None,
                   global_num_experts: int | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Whole SiLU-gated expert layer in one call: x (T, H) -> (T, H).

    x is fp16 / bf16 (quantised here) or int8 with x_scales; w13 (E, 2 inter, H) = [gate | up] and w2 (E, H, inter)
    int8 with scales (E, 2 inter) and (E, H); H and inter multiples of 64. Between the products h = silu(gate) * up
    stays fp32 until each slot's row is quantised. topk_ids (T, top_k) hold global expert ids; with expert_map
    (global_num_experts entries, -1 = not local) they are mapped to the E local experts. Ids that name no local
    expert (-1 among them) contribute nothing. The slots' rows are summed in fp32, in the slots' order: a token's
    output has the same bits in any batch. out_dtype: x's, bf16 for int8 x."""
    xs = _check_rows(x, x_scales)
    T, H = x.shape
    if w13.dim() != 3 or w2.dim() != 3 or w13.shape[1] % 2 != 0:
        _fail("w13 must be (E, 2*inter, H) and w2 (E, H, inter)")
    E, inter = w13.shape[0], w13.shape[1] // 2
    if H % 64 != 0 or inter % 64 != 0:
        _fail(f"hidden and intermediate sizes must be multiples of 64, got {H} and {inter}")
    s13 = _check_weight(w13, w13_scales, (E, 2 * inter, H), "w13")
    s2 = _check_weight(w2, w2_scales, (E, H, inter), "w2")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != T or topk_ids.shape[1] == 0:
        _fail(f"topk_ids must be (T, top_k) with T={T}, got {tuple(topk_ids.shape)}")
    top_k = topk_ids.shape[1]
    if topk_weights.numel() != T * top_k:
        _fail(f"topk_weights must have T*top_k={T * top_k} entries")
    dev = x.device
    emap = None
    if expert_map is not None:
        if expert_map.dim() != 1:
            _fail("expert_map must be 1-d (global_num_experts,)")
        emap = _ids32(expert_map.to(device=dev))
    n_global = E if emap is None else emap.numel()
    if global_num_experts is not None and int(global_num_experts) != n_global:
        _fail(f"global_num_experts={global_num_experts} differs from the expert count {n_global}"
              + ("; pass expert_map" if emap is None else " of expert_map"))
    dt = _out_dtype(out_dtype if out_dtype is not None else (torch.bfloat16 if x.dtype == INT8 else x.dtype))
    _same_device(dev, xs, w13, w2, s13, s2, topk_weights, topk_ids)
    x = _mfma_rows(x, "x")
    if not x.is_contiguous():
        x = x.contiguous()
    tw = topk_weights.to(torch.float32).contiguous()
    ids = _ids32(topk_ids)
    out = torch.empty((T, H), dtype=dt, device=dev)
    nbytes = lib.w4a8_moe_int8_workspace_size(T, H, inter, E, top_k)
    work = _workspace(nbytes, dev)
    with _on(dev):
        check(lib.w4a8_moe_int8_apply(
            _ptr(x), _DT[x.dtype], _ptr(xs), T, H, inter, E, top_k, _ptr(w13), _ptr(s13), _ptr(w2), _ptr(s2),
            _ptr(tw), _ptr(ids), _ptr(emap), n_global, _ptr(out), _DT[dt], _ptr(work), nbytes, _stream(x)),
            "moe_int8_apply")
    return out


# --------------------------------------------------------------------------- #
# torch ops (for traced programs)
# --------------------------------------------------------------------------- #
_SCHEMAS = (
    "act_quant_int8(Tensor x, str? activation) -> (Tensor, Tensor)",
    "int8_gemm(Tensor x, Tensor? x_scales, Tensor w, Tensor w_scales, Tensor? bias, ScalarType out_dtype) -> Tensor",
    "moe_int8_apply(Tensor x, Tensor w13, Tensor w2, Tensor w13_scales, Tensor w2_scales, Tensor topk_weights, "
    "Tensor topk_ids, Tensor? x_scales, Tensor? expert_map, ScalarType out_dtype) -> Tensor",
)
for _schema in _SCHEMAS:
    _ops._library.define(_schema, tags=_ops._TAGS)


def _act_quant_fake(x, activation):
    R, K = x.shape
    K = K // 2 if activation == "silu" else K
    return x.new_empty((R, K), dtype=INT8), x.new_empty((R, 1), dtype=torch.float32)


def _gemm_fake(x, x_scales, w, w_scales, bias, out_dtype):
    return x.new_empty((x.shape[0], w.shape[0]), dtype=out_dtype)


def _apply_op(x, w13, w2, w13_scales, w2_scales, topk_weights, topk_ids, x_scales, expert_map, out_dtype):
    return moe_int8_apply(x, w13, w2, w13_scales, w2_scales, topk_weights, topk_ids, x_scales, expert_map,
                          out_dtype=out_dtype)


def _apply_fake(x, w13, w2, w13_scales, w2_scales, topk_weights, topk_ids, x_scales, expert_map, out_dtype):
    return x.new_empty(x.shape, dtype=out_dtype)


for _name, _impl, _fake in (("act_quant_int8", act_quant_int8, _act_quant_fake),
                            ("int8_gemm", int8_gemm, _gemm_fake),
                            ("moe_int8_apply", _apply_op, _apply_fake)):
    _ops._library.impl(_name, _impl, "CUDA")
    torch.library.register_fake(f"{_ops.NS}::{_name}", _fake)
