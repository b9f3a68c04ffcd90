"""Behind the router projection: each token's experts and their weights from its logits (``route``), on this
build's own sm_100a kernel (``muse_route``). The reference computes the router's FP32 logits and stops
(submission.py:1027-1076); a step that uses them runs::

    logits = project(x, state, "router")                     # FP32 [M, 256]
    weights, experts = route(logits, top_k, scoring="sigmoid", bias=balance, groups=8, top_groups=4)
"""

from __future__ import annotations

import torch

from . import _lib
from .attention import _call, _check_cuda, _vector

_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
_SCORINGS = ("softmax", "sigmoid")


def route(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
          top_groups: int = 1, renormalize: bool = True, scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(weights FP32 [M, top_k], experts int32 [M, top_k]) of logits [M, E] (FP32, BF16 or FP16, E <= 1024),
    in descending order of choice, ties to the lowest index.

    Scores are the softmax over the experts or the sigmoid of each. The choice goes by the logits, or with a
    ``bias`` (FP32 [E], for balance) by score + bias; the bias never enters a weight. With ``groups`` > 1 the
    experts are that many equal runs, a group worth its best choice (with a bias: the sum of its best two),
    and only the best ``top_groups`` take part. ``renormalize`` divides the chosen scores by their sum; all are
    multiplied by ``scale``. An expert masked by -inf (or NaN) comes after every other and weighs 0."""
    kind = _TYPES.get(logits.dtype)
    if logits.dim() != 2 or kind is None or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError(f"logits: expected [tokens, experts] in float32, bfloat16 or float16 with contiguous rows, got "
                         f"{tuple(logits.shape)} {logits.dtype} with strides {logits.stride()}")
    if scoring not in _SCORINGS:
        raise ValueError(f"unknown scoring {scoring!r}")
    dev = logits.get_device()
    m, experts = logits.shape
    balance = 0 if bias is None else _vector("bias", bias, dev, torch.float32, experts)
    if top_k < 1:
        raise ValueError(f"top_k must be positive (got {top_k})")
    _check_cuda(logits, dev)
    device = logits.device
    weights = torch.empty((m, top_k), dtype=torch.float32, device=device)
    ids = torch.empty((m, top_k), dtype=torch.int32, device=device)
    _call(dev, _lib.route, _lib.PACK_ROUTE(logits.data_ptr(), balance, weights.data_ptr(), ids.data_ptr(), logits.stride(0), m, experts, top_k,
                                           groups, top_groups, scoring == "sigmoid", renormalize, kind, scale))
    return weights, ids
