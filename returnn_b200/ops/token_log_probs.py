"""
Log probabilities of given tokens, with the entropy of their distributions and the best alternatives, in one pass over the logits; with gradient
(``csrc/token_log_probs.cu``). What scoring, rescoring and sequence training with a language model read off its output layer.

With ``p = softmax(x)`` per row: ``log_probs = log p[target]``, ``entropy = -sum p log p``, ``top_labels`` the ``num_top`` largest logits (the lowest
label first among equal ones, NaN counts as the largest, numbers below 2^-126 in size as 0) and ``top_log_probs`` their ``log p``. Sums are taken in 32 bits.

A target outside ``0 .. V - 1`` (a padded position) has log probability 0 without a gradient. A label of logit -inf has probability 0. A row in which no label
has a probability has entropy 0, log probabilities -inf and no gradient.
"""

from __future__ import annotations
from typing import NamedTuple, Optional
import ctypes
import math
import torch
from . import _lib, nodes

__all__ = ["TokenLogProbs", "token_log_probs", "token_log_probs_reference", "MAX_TOP"]

_vp, _i32, _i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
MAX_TOP = 32


class TokenLogProbs(NamedTuple):
    """
    what :func:`token_log_probs` returns; None: not asked for. On the GPU the tensors may share one allocation: one that is kept keeps the memory of all (copy it to keep it alone).
    """

    log_probs: torch.Tensor  # [rows] fp32
    entropy: Optional[torch.Tensor] = None  # [rows] fp32
    top_log_probs: Optional[torch.Tensor] = None  # [rows, num_top] fp32
    top_labels: Optional[torch.Tensor] = None  # [rows, num_top] int32


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(logits: torch.Tensor) -> torch.Tensor:
    return logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()


class _TokenLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, entropy, num_top):
        with torch.cuda.device_of(logits):
            x, targets = _rows(logits), targets.contiguous()
            rows, v = x.shape
            dev = x.device
            lp = torch.empty(rows, dtype=torch.float32, device=dev)
            ent = torch.empty(rows, dtype=torch.float32, device=dev) if entropy else None
            top = torch.empty(rows, num_top, dtype=torch.float32, device=dev) if num_top else None
            labels = torch.empty(rows, num_top, dtype=torch.int32, device=dev) if num_top else None
            norm = torch.empty(rows, 2, dtype=torch.float32, device=dev) if ctx.needs_input_grad[0] else None
            fn = _lib.bind("rb200_token_log_probs_fwd", [_vp, _i64, _vp, _i32, _i64, _i32, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp])
            _lib.check(fn(x.data_ptr(), x.stride(0), targets.data_ptr(), 1 if targets.dtype == torch.int64 else 0, rows, v, num_top,
                          1 if x.dtype == torch.bfloat16 else 0, lp.data_ptr(), _p(norm), _p(ent), _p(top), _p(labels), _lib.stream_ptr()), "token_log_probs")
            _lib.count_launch()
        ctx.save_for_backward(x, targets, norm, ent, labels)
        ctx.num_top = num_top
        ctx.set_materialize_grads(False)
        if labels is not None:
            ctx.mark_non_differentiable(labels)
        return lp, ent, top, labels

    @staticmethod
    def backward(ctx, d_lp, d_ent, d_top, _labels):
        x, targets, norm, ent, labels = ctx.saved_tensors
        rows, v = x.shape
        with torch.cuda.device_of(x):
            dx = torch.empty(rows, v, dtype=x.dtype, device=x.device)
            fn = _lib.bind("rb200_token_log_probs_bwd", [_vp, _i64, _vp, _i32, _vp, _vp, _vp, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _vp, _i64, _i32, _i32, _i32, _vp])
            _lib.check(fn(x.data_ptr(), x.stride(0), targets.data_ptr(), 1 if targets.dtype == torch.int64 else 0, norm.data_ptr(), _p(ent), _p(labels),
                          _p(d_lp), d_lp.stride(0) if d_lp is not None else 0, _p(d_ent), d_ent.stride(0) if d_ent is not None else 0,
                          _p(d_top), *(d_top.stride() if d_top is not None else (0, 0)), dx.data_ptr(), rows, v, ctx.num_top,
                          1 if x.dtype == torch.bfloat16 else 0, _lib.stream_ptr()), "token_log_probs_bwd")
            _lib.count_launch()
        return nodes.first_order("token_log_probs", (dx, None, None, None), (d_lp, d_ent, d_top, x))


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor, *, entropy: bool = False, num_top: int = 0) -> TokenLogProbs:
    """
    See the module docstring; differentiable in ``logits`` (through all three results), once.

    :param logits: [rows, V] bf16 or fp32, unit stride over V (rows may lie further apart: the first V columns of a padded product)
    :param targets: [rows] int32 or int64
    :param entropy: also the entropy of each row
    :param num_top: also that many best labels, at most 32 and at most V
    """
    what = "token_log_probs"
    mod = nodes.of(logits)
    if mod is not None:
        res = mod.token_log_probs(logits, targets, entropy, num_top)
        if res is not None:
            return TokenLogProbs(*res)
    if logits.dim() != 2 or targets.shape != logits.shape[:1]:
        raise ValueError("%s: logits %s must be [rows, V], targets %s [rows]" % (what, tuple(logits.shape), tuple(targets.shape)))
    if targets.dtype not in (torch.int32, torch.int64) or targets.device != logits.device:
        raise TypeError("%s: targets must be int32 or int64 on %s, got %s on %s" % (what, logits.device, targets.dtype, targets.device))
    if logits.shape[1] < 1 or not 0 <= num_top <= min(MAX_TOP, logits.shape[1]):
        raise ValueError("%s: num_top %r of %i labels (at most %i)" % (what, num_top, logits.shape[1], MAX_TOP))
    if not (logits.is_cuda and _lib.use_native(logits)):
        return token_log_probs_reference(logits, targets, entropy=entropy, num_top=num_top)
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("%s: bf16 and fp32 on the GPU, got %s" % (what, logits.dtype))
    return TokenLogProbs(*_TokenLogProbsFn.apply(logits, targets, bool(entropy), int(num_top)))


def token_log_probs_reference(logits, targets, *, entropy=False, num_top=0):
    """plain torch in fp32, or in 64 bits where the logits are (differentiable)"""
    x = logits.to(torch.promote_types(logits.dtype, torch.float32))
    none = (x == -math.inf).all(dim=-1)
    lp = torch.log_softmax(torch.where(none[:, None], 0.0, x), dim=-1)
    lp = torch.where(none[:, None], -math.inf, lp)  # (constants: no gradient)
    given = (targets >= 0) & (targets < x.shape[1])
    out = lp.gather(-1, targets.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    out = torch.where(given, out, torch.zeros_like(out))
    res = TokenLogProbs(out)
    if entropy:
        finite = torch.where(lp == -math.inf, 0.0, lp)
        res = res._replace(entropy=-(lp.exp() * finite).sum(dim=-1))
    if num_top:
        order = torch.where(x.isnan(), math.nan, x).detach()
        if x.dtype == torch.float32:
            order = torch.where(order.abs() < torch.finfo(torch.float32).tiny, 0.0, order)
        labels = torch.sort(order, dim=-1, descending=True, stable=True)[1][:, :num_top]
        res = res._replace(top_log_probs=lp.gather(-1, labels), top_labels=labels.to(torch.int32))
    return res
