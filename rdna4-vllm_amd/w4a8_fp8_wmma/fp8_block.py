"""Block-scaled fp8 (W8A8) layers on gfx950: norm, activation quantisation, dense and grouped
products and the gated expert layer, for checkpoints whose weights are e4m3 with one fp32 scale per
128 x 128 block. (No reference counterpart: the reference serves int4 and E2M1 weights.)

Activations are ``torch.float8_e4m3fn`` rows with one fp32 scale per row and 128 values, as
``rms_norm_quant_fp8`` and ``act_quant_fp8_block`` make them; weights are (N, K) or (E, N, K)
``torch.float8_e4m3fn`` with fp32 scales (..., ceil(N / 128), ceil(K / 128)).

A decoder layer's expert half, as a serving program runs it::

    n = rms_norm_quant_fp8(x, norm_w, eps, residual=r, return_norm=True)
    tw, ids = fused_topk(None, n.norm @ router_w, top_k)
    y = moe_fp8_block_apply(n.q, w13, w2, s13, s2, tw, ids, x_scales=n.scales, out_dtype=x.dtype)

Plain functions over the C ABI, and the same as torch ops (``torch.ops.w4a8_fp8_wmma.*``) with fake
implementations for traced programs. Every call enqueues on torch's current stream of its tensors'
device and never synchronises. Inference only: no gradients.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _ops
from ._lib import check, lib
from ._ops import _fail, _ptr, _workspace

BLOCK = 128
FP8 = torch.float8_e4m3fn
_DT = {torch.float16: 0, torch.bfloat16: 1, FP8: 2}


class NormQuant(NamedTuple):
    q: torch.Tensor                       # (T, H) e4m3
    scales: torch.Tensor                  # (T, ceil(H / 128)) or (T, 1) fp32
    residual: Optional[torch.Tensor]      # x + residual, where one was given
    norm: Optional[torch.Tensor]          # the norm in x's dtype, where it was asked for


# (torch.cuda.current_device / current_stream without their Python layers, which cost more than the
# launch does; the tensors of a call have initialised torch.cuda)
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


class _on:
    """Makes a tensor's device the current one (a call on another device than the current one
    launches on the tensors' device)."""
    __slots__ = ("to", "back")

    def __init__(self, device):
        self.to = device.index
        self.back = None

    def __enter__(self):
        now = _current_device()
        if self.to != now:
            self.back = now
            torch.cuda.set_device(self.to)

    def __exit__(self, *exc):
        if self.back is not None:
            torch.cuda.set_device(self.back)


def _stream(t):
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _groups(n: int) -> int:
    return -(-n // BLOCK)


def _rows2d(x, name):
    """x with contiguous rows (row strides and padding between rows are kept)."""
    if x.dim() != 2:
        _fail(f"{name} must be 2D, got {tuple(x.shape)}")
    if x.is_contiguous():
        return x
    if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        return x.contiguous()
    return x


def _stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _mfma_rows(x, name):
    """Rows that start at multiples of 16 bytes (a copy where they do not)."""
    x = _rows2d(x, name)
    if x.data_ptr() % 16 != 0 or _stride(x) * x.element_size() % 16 != 0:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _same_device(device, *tensors):
    for t in tensors:
        if t is not None and t.device != device:
            _fail(f"all tensors must be CUDA tensors on x's device {device}, got {t.device}")
    if device.type != "cuda":
        _fail("all tensors must be CUDA tensors")


def _check_scaled(q, s, rows, K, name):
    if s.dtype != torch.float32 or s.shape != (rows, _groups(K)):
        _fail(f"{name} must be fp32 (rows, ceil(K/128))=({rows},{_groups(K)}); got {s.dtype} {tuple(s.shape)}")
    return s if s.is_contiguous() else s.contiguous()


def _check_weight(w, s, lead, N, K, name):
    """e4m3 weights (*lead, N, K) and their block scales; contiguous (weights are never copied)."""
    if w.dtype != FP8 or w.shape != (*lead, N, K):
        _fail(f"{name} must be float8_e4m3fn {(*lead, N, K)}; got {w.dtype} {tuple(w.shape)}")
    if s.dtype != torch.float32 or s.shape != (*lead, _groups(N), _groups(K)):
        _fail(f"{name} scales must be fp32 {(*lead, _groups(N), _groups(K))}; got {s.dtype} {tuple(s.shape)}")
    if not (w.is_contiguous() and s.is_contiguous()):
        _fail(f"{name} and its scales must be contiguous")
    if w.data_ptr() % 16 != 0:
        _fail(f"{name} must be aligned to 16 bytes")


def _out_dtype(dtype):
    if dtype not in (torch.float16, torch.bfloat16):
        _fail(f"out_dtype must be fp16 or bf16, got {dtype}")
    return dtype


def rms_norm_quant_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                       residual: torch.Tensor | None = None, group_size: int = BLOCK,
                       return_norm: bool = False) -> NormQuant:
    """RMS norm with the residual's addition and e4m3 output, in one pass over the rows.

    x (T, H) fp16 / bf16; z = x + residual rounded to x's dtype (returned as ``residual``; x and
    residual are left as they are), y = z / sqrt(mean(z^2) + eps) * weight in fp32, quantised with
    one scale per 128 values (``group_size=128``) or one a row (``group_size=0``). ``return_norm``
    also returns y in x's dtype (what a router or an unquantised layer reads). weight (H,) in x's
    dtype or fp32. Rows may be strided."""
    if x.dtype not in (torch.float16, torch.bfloat16) or x.dim() != 2:
        _fail(f"x must be fp16/bf16 (T, H), got {x.dtype} {tuple(x.shape)}")
    T, H = x.shape
    if H == 0:
        _fail("x has no columns")
    if group_size not in (0, BLOCK):
        _fail(f"group_size must be 128 or 0 (one scale a row), got {group_size}")
    if weight.shape != (H,) or weight.dtype not in (x.dtype, torch.float32):
        _fail(f"weight must be ({H},) in x's dtype or fp32, got {weight.dtype} {tuple(weight.shape)}")
    if residual is not None:
        if residual.dtype != x.dtype or residual.shape != x.shape:
            _fail(f"residual must be {x.dtype} {tuple(x.shape)}, got {residual.dtype} {tuple(residual.shape)}")
        residual = _rows2d(residual, "residual")
    dev = x.device
    _same_device(dev, weight, residual)
    if H % 8 == 0:
        # (the same kernel, so the same bits, whatever the rows' strides)
        x = _mfma_rows(x, "x")
        residual = None if residual is None else _mfma_rows(residual, "residual")
    else:
        x = _rows2d(x, "x")
    w = weight.contiguous()
    if w.data_ptr() % 16 != 0:
        w = w.clone()
    q = torch.empty((T, H), dtype=FP8, device=dev)
    s = torch.empty((T, 1 if group_size == 0 else _groups(H)), dtype=torch.float32, device=dev)
    z = None if residual is None else torch.empty((T, H), dtype=x.dtype, device=dev)
    y = torch.empty((T, H), dtype=x.dtype, device=dev) if return_norm else None
    with _on(dev):
        check(lib.w4a8_rms_norm_quant_fp8(
            _ptr(x), _DT[x.dtype], T, H, _stride(x), None if residual is None else _ptr(residual),
            0 if residual is None else _stride(residual), _ptr(w),
            1 if w.dtype == torch.float32 else 0, float(eps), 1 if group_size == 0 else 0, _ptr(z),
            _ptr(y), _ptr(q), _ptr(s), _stream(x)), "rms_norm_quant_fp8")
    return NormQuant(q, s, z, y)


def act_quant_fp8_block(x: torch.Tensor, activation: str | None = None):
    """e4m3 rows with one fp32 scale per row and 128 values: (q (R, K), scales (R, ceil(K / 128))).

    x (R, K) fp16 / bf16, or with ``activation="silu"`` x = [gate | up] (R, 2 K), whose
    silu(gate) * up is formed and quantised in fp32. Rows may be strided."""
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
    q = torch.empty((R, K), dtype=FP8, device=dev)
    s = torch.empty((R, _groups(K)), dtype=torch.float32, device=dev)
    with _on(dev):
        check(lib.w4a8_act_quant_fp8_block(_ptr(x), _DT[x.dtype], R, K, _stride(x),
                                           0 if activation is None else 1, _ptr(q), _ptr(s),
                                           _stream(x)), "act_quant_fp8_block")
    return q, s


def _check_rows(x, x_scales, name="x"):
    """e4m3 rows with scales, or 16-bit rows without."""
    if x.dim() != 2:
        _fail(f"{name} must be 2D, got {tuple(x.shape)}")
    if x.dtype == FP8:
        if x_scales is None:
            _fail(f"{name} in e4m3 needs its scales")
        return _check_scaled(x, x_scales, x.shape[0], x.shape[1], f"{name}_scales")
    if x.dtype not in (torch.float16, torch.bfloat16):
        _fail(f"{name} must be float8_e4m3fn, fp16 or bf16, got {x.dtype}")
    if x_scales is not None:
        _fail(f"{name}_scales go with e4m3 rows only")
    return None


def fp8_block_gemm(x: torch.Tensor, x_scales: torch.Tensor | None, w: torch.Tensor,
                   w_scales: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Dense layer x (M, K) times w (N, K) transposed with block scales -> (M, N).

    x is e4m3 with x_scales (M, ceil(K / 128)), or fp16 / bf16 with ``x_scales=None``: rows that the
    call quantises as ``act_quant_fp8_block`` does. Each group of 128 k is summed by the matrix
    cores, scaled by the row's and the block's scale and added in fp32. out_dtype: fp16 or bf16
    (default: x's, bf16 for e4m3 x). K must be a multiple of 16."""
    xs = _check_rows(x, x_scales)
    M, K = x.shape
    if w.dim() != 2:
        _fail(f"w must be (N, K), got {tuple(w.shape)}")
    N = w.shape[0]
    _check_weight(w, w_scales, (), N, K, "w")
    dt = _out_dtype(out_dtype if out_dtype is not None else (torch.bfloat16 if x.dtype == FP8 else x.dtype))
    dev = x.device
    _same_device(dev, xs, w, w_scales)
    x = _mfma_rows(x, "x")
    out = torch.empty((M, N), dtype=dt, device=dev)
    nbytes = 0 if xs is not None else lib.w4a8_fp8_block_gemm_workspace_size(_DT[x.dtype], M, K)
    ws = _workspace(nbytes, dev) if nbytes else None
    with _on(dev):
        check(lib.w4a8_fp8_block_gemm(
            _ptr(x), _DT[x.dtype], _ptr(xs), M, K, _stride(x), _ptr(w), _ptr(w_scales), N,
            _ptr(out), _DT[dt], _ptr(ws), nbytes, _stream(x)), "fp8_block_gemm")
    return out


def moe_fp8_block_gemm(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor,
                       w_scales: torch.Tensor, sorted_token_ids: torch.Tensor,
                       expert_ids: torch.Tensor, num_tokens_post_padded: torch.Tensor, top_k: int,
                       block_m: int, out: torch.Tensor | None = None,
                       out_dtype: torch.dtype | None = None, gather: bool = True,
                       num_slots: int | None = None) -> torch.Tensor:
    """Products grouped by expert, in the padded sorted layout of ``moe_align_block_size``.

    Row r < num_tokens_post_padded with slot s = sorted_token_ids[r] takes x[s // top_k] (or, with
    ``gather=False``, x[r]: the rows of an earlier grouped product) times the weights of expert
    expert_ids[r // block_m] -> (P, N) in out_dtype (bf16 by default) or in ``out``. Rows whose slot
    is not in [0, num_slots) are padding and not written (without ``out``, and from the torch op, they
    hold anything); num_slots is the number of routed slots, tokens * top_k (default: x.shape[0] *
    top_k, which with ``gather=False`` counts padding rows of x as slots too: pass it there to leave
    them as they are). w (E, N, K) e4m3; block_m a multiple of 16 up to 128."""
    xs = _check_rows(x, x_scales)
    if xs is None:
        _fail("x must be float8_e4m3fn")
    if w.dim() != 3:
        _fail(f"w must be (E, N, K), got {tuple(w.shape)}")
    E, N, _ = w.shape
    rows, K = x.shape
    _check_weight(w, w_scales, (E,), N, K, "w")
    for t, name in ((sorted_token_ids, "sorted_token_ids"), (expert_ids, "expert_ids"),
                    (num_tokens_post_padded, "num_tokens_post_padded")):
        if t.dtype != torch.int32 or not t.is_contiguous():
            _fail(f"{name} must be contiguous int32")
    P = sorted_token_ids.numel()
    if block_m <= 0 or block_m > 128 or block_m % 16 != 0:
        _fail(f"block_m must be a multiple of 16 up to 128, got {block_m}")
    if top_k <= 0:
        _fail("top_k must be positive")
    if P % block_m != 0 or expert_ids.numel() != P // block_m or num_tokens_post_padded.numel() != 1:
        _fail(f"expert_ids must have P/block_m={P}/{block_m} entries and num_tokens_post_padded one")
    dev = x.device
    if out is None:
        out = torch.empty((P, N), dtype=_out_dtype(out_dtype if out_dtype is not None else torch.bfloat16),
                          device=dev)
    else:
        if tuple(out.shape) != (P, N) or not out.is_contiguous() or (out_dtype is not None and out.dtype != out_dtype):
            _fail(f"out must be contiguous (P, N)=({P},{N}), got {out.dtype} {tuple(out.shape)}")
        _out_dtype(out.dtype)
    _same_device(dev, xs, w, w_scales, sorted_token_ids, expert_ids, num_tokens_post_padded, out)
    x = _mfma_rows(x, "x")
    if num_slots is None:
        num_slots = rows * top_k if gather else max(rows * top_k, P)
    elif num_slots < 0 or gather and num_slots > rows * top_k:
        _fail(f"num_slots must be in 0 .. {rows * top_k}, got {num_slots}")
    with _on(dev):
        check(lib.w4a8_moe_fp8_block_gemm(
            _ptr(x), _ptr(xs), rows, K, _stride(x), _ptr(w), _ptr(w_scales), E, N,
            _ptr(sorted_token_ids), P, _ptr(expert_ids), _ptr(num_tokens_post_padded), int(num_slots),
            int(top_k), int(block_m), 1 if gather else 0, _ptr(out), _DT[out.dtype], _stream(x)),
            "moe_fp8_block_gemm")
    return out


def moe_fp8_block_apply(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor,
                        w13_scales: torch.Tensor, w2_scales: torch.Tensor,
                        topk_weights: torch.Tensor, topk_ids: torch.Tensor,
                        x_scales: torch.Tensor | None = None,
                        expert_map: torch.Tensor | None = None,
                        global_num_experts: int | None = None,
                        out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Whole SiLU-gated expert layer in one call: x (T, H) -> (T, H).

    x is fp16 / bf16 (quantised here) or e4m3 with x_scales; w13 (E, 2 inter, H) = [gate | up] and
    w2 (E, H, inter) e4m3 with block scales; H and inter multiples of 128. Between the products
    h = silu(gate) * up stays fp32 until it is quantised. topk_ids (T, top_k) hold global expert
    ids; with expert_map (global_num_experts entries, -1 = not local) they are mapped to the E local
    experts and the others contribute nothing. out_dtype: x's, bf16 for e4m3 x."""
    xs = _check_rows(x, x_scales)
    T, H = x.shape
    if w13.dim() != 3 or w2.dim() != 3 or w13.shape[1] % 2 != 0:
        _fail("w13 must be (E, 2*inter, H) and w2 (E, H, inter)")
    E, inter = w13.shape[0], w13.shape[1] // 2
    if H % BLOCK != 0 or inter % BLOCK != 0:
        _fail(f"hidden and intermediate sizes must be multiples of 128, got {H} and {inter}")
    _check_weight(w13, w13_scales, (E,), 2 * inter, H, "w13")
    _check_weight(w2, w2_scales, (E,), H, inter, "w2")
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
        emap = expert_map.to(device=dev, dtype=torch.int32).contiguous()
    n_global = E if emap is None else emap.numel()
    if global_num_experts is not None and int(global_num_experts) != n_global:
        _fail(f"global_num_experts={global_num_experts} differs from the expert count {n_global}"
              + ("; pass expert_map" if emap is None else " of expert_map"))
    dt = _out_dtype(out_dtype if out_dtype is not None else (torch.bfloat16 if x.dtype == FP8 else x.dtype))
    _same_device(dev, xs, w13, w2, w13_scales, w2_scales, topk_weights, topk_ids)
    x = _mfma_rows(x, "x")
    if not x.is_contiguous():
        x = x.contiguous()
    tw = topk_weights.to(torch.float32).contiguous()
    ids = topk_ids.to(torch.int32).contiguous()
    out = torch.empty((T, H), dtype=dt, device=dev)
    nbytes = lib.w4a8_moe_fp8_block_workspace_size(T, H, inter, E, top_k)
    ws = _workspace(nbytes, dev)
    with _on(dev):
        check(lib.w4a8_moe_fp8_block_apply(
            _ptr(x), _DT[x.dtype], _ptr(xs), T, H, inter, E, top_k, _ptr(w13), _ptr(w13_scales),
            _ptr(w2), _ptr(w2_scales), _ptr(tw), _ptr(ids), _ptr(emap), n_global, _ptr(out),
            _DT[dt], ws.data_ptr(), ws.numel(), _stream(x)), "moe_fp8_block_apply")
    return out


# --------------------------------------------------------------------------- #
# torch ops (for traced programs)
# --------------------------------------------------------------------------- #
_SCHEMAS = {
    "rms_norm_quant_fp8": "rms_norm_quant_fp8(Tensor x, Tensor weight, float eps, Tensor? residual, "
                          "int group_size, bool return_norm) -> (Tensor, Tensor, Tensor, Tensor)",
    "act_quant_fp8_block": "act_quant_fp8_block(Tensor x, str? activation) -> (Tensor, Tensor)",
    "fp8_block_gemm": "fp8_block_gemm(Tensor x, Tensor? x_scales, Tensor w, Tensor w_scales, "
                      "ScalarType out_dtype) -> Tensor",
    "moe_fp8_block_gemm": "moe_fp8_block_gemm(Tensor x, Tensor x_scales, Tensor w, Tensor w_scales, "
                          "Tensor sorted_token_ids, Tensor expert_ids, "
                          "Tensor num_tokens_post_padded, int top_k, int block_m, "
                          "ScalarType out_dtype, bool gather=True, int? num_slots=None) -> Tensor",
    "moe_fp8_block_apply": "moe_fp8_block_apply(Tensor x, Tensor w13, Tensor w2, Tensor w13_scales, "
                           "Tensor w2_scales, Tensor topk_weights, Tensor topk_ids, "
                           "Tensor? x_scales, Tensor? expert_map, ScalarType out_dtype) -> Tensor",
}
for _schema in _SCHEMAS.values():
    _ops._library.define(_schema, tags=_ops._TAGS)


def _rms_norm_op(x, weight, eps, residual, group_size, return_norm):
    """Absent outputs are empty tensors."""
    n = rms_norm_quant_fp8(x, weight, eps, residual, group_size, return_norm)
    none = x.new_empty((0,))
    return (n.q, n.scales, none if n.residual is None else n.residual,
            x.new_empty((0,)) if n.norm is None else n.norm)


def _rms_norm_fake(x, weight, eps, residual, group_size, return_norm):
    T, H = x.shape
    return (x.new_empty((T, H), dtype=FP8),
            x.new_empty((T, 1 if group_size == 0 else (H + BLOCK - 1) // BLOCK), dtype=torch.float32),
            x.new_empty((0,) if residual is None else (T, H)),
            x.new_empty((T, H) if return_norm else (0,)))


def _act_quant_fake(x, activation):
    R, K = x.shape
    K = K // 2 if activation == "silu" else K
    return (x.new_empty((R, K), dtype=FP8),
            x.new_empty((R, (K + BLOCK - 1) // BLOCK), dtype=torch.float32))


def _gemm_fake(x, x_scales, w, w_scales, out_dtype):
    return x.new_empty((x.shape[0], w.shape[0]), dtype=out_dtype)


def _moe_gemm_op(x, x_scales, w, w_scales, sorted_token_ids, expert_ids, num_tokens_post_padded,
                 top_k, block_m, out_dtype, gather=True, num_slots=None):
    return moe_fp8_block_gemm(x, x_scales, w, w_scales, sorted_token_ids, expert_ids,
                              num_tokens_post_padded, top_k, block_m, out_dtype=out_dtype,
                              gather=gather, num_slots=num_slots)


def _moe_gemm_fake(x, x_scales, w, w_scales, sorted_token_ids, expert_ids, num_tokens_post_padded,
                   top_k, block_m, out_dtype, gather=True, num_slots=None):
    return x.new_empty((sorted_token_ids.shape[0], w.shape[1]), dtype=out_dtype)


def _apply_op(x, w13, w2, w13_scales, w2_scales, topk_weights, topk_ids, x_scales, expert_map, out_dtype):
    return moe_fp8_block_apply(x, w13, w2, w13_scales, w2_scales, topk_weights, topk_ids, x_scales,
                               expert_map, out_dtype=out_dtype)


def _apply_fake(x, w13, w2, w13_scales, w2_scales, topk_weights, topk_ids, x_scales, expert_map, out_dtype):
    return x.new_empty(x.shape, dtype=out_dtype)


for _name, _impl, _fake in (("rms_norm_quant_fp8", _rms_norm_op, _rms_norm_fake),
                            ("act_quant_fp8_block", act_quant_fp8_block, _act_quant_fake),
                            ("fp8_block_gemm", fp8_block_gemm, _gemm_fake),
                            ("moe_fp8_block_gemm", _moe_gemm_op, _moe_gemm_fake),
                            ("moe_fp8_block_apply", _apply_op, _apply_fake)):
    _ops._library.impl(_name, _impl, "CUDA")
    torch.library.register_fake(f"{_ops.NS}::{_name}", _fake)
