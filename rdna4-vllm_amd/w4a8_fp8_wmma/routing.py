"""Choice of experts from a router's logits on gfx950, beyond the plain softmax top-k of ``fused_topk``. (No
reference counterpart.)

A plain function over the C ABI, and the same as a torch op (``torch.ops.w4a8_fp8_wmma.route_topk``) with a fake
implementation for traced programs. Enqueues on torch's current stream of the logits' device and never synchronises.
Inference only: no gradients.
"""
from __future__ import annotations

import torch

from . import _ops
from ._lib import check, lib
from ._ops import _fail, _ptr
from .fp8_block import _on, _rows2d, _same_device, _stream, _stride

_DT = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 4}
_SCORING = {"softmax": 0, "sigmoid": 1}


def route_topk(router_logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: torch.Tensor | None = None,
               num_groups: int = 1, top_groups: int = 1, renormalize: bool = True, scale: float = 1.0):
    """(topk_weights fp32 (T, top_k), topk_ids int32 (T, top_k)) of router_logits (T, E) fp32 / bf16 / fp16.

    p = softmax(logits) or sigmoid(logits), c = p + bias (bias (E,) fp32). The E experts are num_groups equal runs;
    a group's score is the sum of its two largest c with a bias, its largest c without, and the top_groups best groups
    stay. Picks are the top_k largest c of those, in descending order, ties to the lower expert (and group), as the
    true numbers compare; their weights p, divided by their sum with ``renormalize``, times scale.

    A logit of -inf or NaN masks its expert, as a bias of -inf or NaN does: it is never picked, and picks that find no
    expert are -1 with weight 0 (expert layers leave them out). +inf counts as the largest finite number. E up to
    1024, top_k and num_groups up to 64; rows may be strided."""
    if router_logits.dim() != 2 or router_logits.dtype not in _DT:
        _fail(f"router_logits must be (T, E) in fp32, bf16 or fp16, got {router_logits.dtype} {tuple(router_logits.shape)}")
    if scoring not in _SCORING:
        _fail(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    T, E = router_logits.shape
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (E,):
            _fail(f"bias must be fp32 ({E},), got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    dev = router_logits.device
    _same_device(dev, bias)
    l = _rows2d(router_logits, "router_logits")
    w = torch.empty((T, top_k), dtype=torch.float32, device=dev)
    ids = torch.empty((T, top_k), dtype=torch.int32, device=dev)
    with _on(dev):
        check(lib.w4a8_route_topk(_ptr(l), _DT[l.dtype], T, E, _stride(l), top_k, _SCORING[scoring], _ptr(bias),
                                  num_groups, top_groups, 1 if renormalize else 0, scale, _ptr(w), _ptr(ids),
                                  _stream(l)), "route_topk")
    return w, ids


_ops._library.define("route_topk(Tensor router_logits, int top_k, str scoring, Tensor? bias, int num_groups, "
                     "int top_groups, bool renormalize, float scale) -> (Tensor, Tensor)", tags=_ops._TAGS)
_ops._library.impl("route_topk", route_topk, "CUDA")


def _route_fake(router_logits, top_k, scoring, bias, num_groups, top_groups, renormalize, scale):
    T = router_logits.shape[0]
    return (router_logits.new_empty((T, top_k), dtype=torch.float32),
            router_logits.new_empty((T, top_k), dtype=torch.int32))


torch.library.register_fake(f"{_ops.NS}::route_topk", _route_fake)
