"""
Rotary positions of queries and keys, with an RMS norm per head before them, in one pass over both (``csrc/norm_rope.cu``); with gradient, and in
a form for serving that writes keys and values to their slots of a paged cache (:mod:`returnn_b200.ops.paged`).

Per (token, head) row ``x`` of ``D`` features: ``y = x / sqrt(mean(x^2) + eps) * scale`` (without scales: ``y = x``), then the first ``2 F`` features are
``F`` pairs, and pair ``i`` is turned by ``position * frequencies[i]`` and multiplied by ``amplitude``. The pairs are ``(2i, 2i + 1)`` with
``interleaved=True`` (the layout of ``rf.RotaryPosSelfAttention``, returnn/frontend/attention.py:535) and ``(i, i + F)`` otherwise.

Sums, angles and rotations are taken in 32 bits (the angle's reduction in 64), with one rounding to the type of the input at the end.
"""

from __future__ import annotations
from typing import Any, Dict, Optional, Tuple
import ctypes
import math
import torch
from . import _lib, nodes

__all__ = ["rope_frequencies", "norm_rope", "norm_rope_to_cache", "norm_rope_reference"]

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
MAX_HEAD_DIM = 256


def rope_frequencies(rotary_dim: int, *, base: float = 10_000.0, scaling: Optional[Dict[str, Any]] = None, device=None) -> Tuple[torch.Tensor, float]:
    """
    :param rotary_dim: features of a head that are rotated (even)
    :param base: frequency ``i`` is ``base ** (-2 i / rotary_dim)``
    :param scaling: for contexts longer than the model was trained on, a dict with ``"type"`` and

        * ``"linear"``: ``factor``; all frequencies are divided by it (positions are squeezed)
        * ``"base"``: ``factor``; the base grows so that the lowest frequency is divided by the factor and the highest stays
        * ``"by_parts"``: ``factor``, ``original_length``, ``low`` = 1.0, ``high`` = 32.0: a frequency that makes more than ``high`` turns over the original
          length stays, one of fewer than ``low`` turns is divided by the factor, those in between are mixed linearly in the number of
          turns; ``amplitude`` (default ``0.1 ln(factor) + 1``) is returned with them
    :return: frequencies [rotary_dim / 2] fp32, amplitude
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rope_frequencies: rotary dim %r must be even" % (rotary_dim,))
    scaling = dict(scaling or {})
    kind = scaling.pop("type", None)
    amplitude = 1.0
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / max(rotary_dim, 1)
    if kind is None:
        freq = base ** -exponent
    else:
        if kind not in ("linear", "base", "by_parts"):
            raise ValueError("rope_frequencies: unknown scaling type %r" % (kind,))
        factor = float(scaling.pop("factor"))
        if not factor > 0:
            raise ValueError("rope_frequencies: scaling factor %r" % (factor,))
        if kind == "linear":
            freq = base ** -exponent / factor
        elif kind == "base":
            if rotary_dim > 2:
                base = base * factor ** (rotary_dim / (rotary_dim - 2))
            freq = base ** -exponent
        else:
            length, low, high = float(scaling.pop("original_length")), float(scaling.pop("low", 1.0)), float(scaling.pop("high", 32.0))
            if not (length > 0 and high > low):
                raise ValueError("rope_frequencies: by_parts wants original_length > 0 and high > low")
            freq = base ** -exponent
            keep = ((freq * length / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
            freq = freq * keep + freq / factor * (1.0 - keep)
            amplitude = float(scaling.pop("amplitude", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0))
    if scaling:
        raise ValueError("rope_frequencies: unexpected scaling options %r" % (sorted(scaling),))
    return freq.to(torch.float32).to(device), amplitude


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _rows(x: torch.Tensor) -> torch.Tensor:
    """[..., H, D] -> [N, H, D] with unit stride over D; a view where the strides allow it"""
    x = x.reshape(math.prod(x.shape[:-2]), *x.shape[-2:]) if x.dim() != 3 else x
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def _strides(*tensors):
    return [s for t in tensors for s in t.stride()[:-1]]


def _check(q, k, positions, frequencies, q_scale, k_scale, what: str):
    if q.dim() < 3 or k.dim() != q.dim() or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError("%s: q %s and k %s must be [..., heads, dim] over the same tokens" % (what, tuple(q.shape), tuple(k.shape)))
    if q.dtype != k.dtype or q.device != k.device:
        raise TypeError("%s: q is %s on %s, k %s on %s" % (what, q.dtype, q.device, k.dtype, k.device))
    d = q.shape[-1]
    if frequencies is not None:
        if positions is None or positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("%s: positions must be int32 or int64" % what)
        if positions.dim() > q.dim() - 2 or tuple(positions.shape) != tuple(q.shape[q.dim() - 2 - positions.dim(): -2]):
            raise ValueError("%s: positions %s do not fit the tokens %s" % (what, tuple(positions.shape), tuple(q.shape[:-2])))
        if frequencies.dim() != 1 or frequencies.dtype != torch.float32 or 2 * frequencies.shape[0] > d:
            raise ValueError("%s: frequencies must be fp32 [<= %i], got %s %s" % (what, d // 2, frequencies.dtype, tuple(frequencies.shape)))
        if positions.device != q.device or frequencies.device != q.device:
            raise ValueError("%s: positions on %s and frequencies on %s, q on %s" % (what, positions.device, frequencies.device, q.device))
        if (torch.is_grad_enabled() and frequencies.requires_grad) or nodes.has_tangent(frequencies):
            raise RuntimeError("%s: there is no gradient of the frequencies: detach them" % what)
    if (q_scale is None) != (k_scale is None):
        raise ValueError("%s: scales for both q and k, or for neither" % what)
    if q_scale is not None:
        for s in (q_scale, k_scale):
            if s.shape != (d,) or s.dtype != q_scale.dtype or s.device != q.device:
                raise ValueError("%s: scales must be [%i] of one type on %s, got %s %s on %s" % (what, d, q.device, tuple(s.shape), s.dtype, s.device))


def _native_ok(q: torch.Tensor, q_scale: Optional[torch.Tensor], what: str) -> bool:
    if not (q.is_cuda and _lib.use_native(q)):
        return False
    if q.dtype not in (torch.bfloat16, torch.float32) or (q_scale is not None and q_scale.dtype not in (torch.bfloat16, torch.float32)):
        raise TypeError("%s: bf16 and fp32 on the GPU, got %s%s" % (what, q.dtype, "" if q_scale is None else " with scales of %s" % q_scale.dtype))
    if q.shape[-1] > MAX_HEAD_DIM:
        raise ValueError("%s: head dim %i, at most %i" % (what, q.shape[-1], MAX_HEAD_DIM))
    return True


class _Positions:
    """pointers of positions and frequencies as the kernels take them; positions of the trailing token axes repeat over the others"""

    def __init__(self, positions, frequencies):
        self.positions = positions.contiguous() if frequencies is not None else None
        self.frequencies = frequencies.contiguous() if frequencies is not None else None
        self.rot = 0 if frequencies is None else 2 * frequencies.shape[0]
        self.count = 1 if positions is None else positions.numel()
        self.is64 = 1 if positions is not None and positions.dtype == torch.int64 else 0


_FWD = [_vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _f32, _f32, _vp]
_CACHE = [_vp, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _i32, _i32, _i32, _i64, _i32, _i32, _i32, _i32, _f32, _f32, _vp]
_BWD = [_vp, _vp, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _f32, _f32, _vp]


class _NormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, q_scale, k_scale, eps, interleaved, amplitude):
        with torch.cuda.device_of(q):
            q3, k3 = _rows(q), _rows(k)
            n, hq, d = q3.shape
            hk = k3.shape[1]
            pos = _Positions(positions, frequencies)
            wq = q_scale.contiguous() if q_scale is not None else None
            wk = k_scale.contiguous() if k_scale is not None else None
            out_q = torch.empty(n, hq, d, dtype=q.dtype, device=q.device)
            out_k = torch.empty(n, hk, d, dtype=q.dtype, device=q.device)
            fn = _lib.bind("rb200_norm_rope_fwd", _FWD)
            st = (_i64 * 4)(*_strides(q3, k3))
            _lib.check(fn(_ptr(q3), _ptr(k3), _ptr(pos.positions), pos.count, _ptr(pos.frequencies), _ptr(wq), _ptr(wk), _ptr(out_q), _ptr(out_k), st, n, hq, hk, d,
                          pos.rot, 1 if q.dtype == torch.bfloat16 else 0, pos.is64, 1 if wq is not None and wq.dtype == torch.bfloat16 else 0,
                          1 if interleaved else 0, eps, amplitude, _lib.stream_ptr()), "norm_rope")
            _lib.count_launch()
        # without a norm the gradient is a rotation back: the inputs are not kept
        ctx.save_for_backward(*((q3, k3) if wq is not None else (None, None)), pos.positions, pos.frequencies, wq, wk)
        ctx.opts = (pos.count, pos.rot, pos.is64, float(eps), bool(interleaved), float(amplitude))
        ctx.shapes = (q.shape, k.shape)
        return out_q.view(q.shape), out_k.view(k.shape)

    @staticmethod
    def backward(ctx, dq, dk):
        q3, k3, positions, frequencies, wq, wk = ctx.saved_tensors
        count, rot, is64, eps, interleaved, amplitude = ctx.opts
        with torch.cuda.device_of(dq):
            dq3, dk3 = _rows(dq), _rows(dk)
            n, hq, d = dq3.shape
            hk = dk3.shape[1]
            gq = torch.empty(n, hq, d, dtype=dq.dtype, device=dq.device)
            gk = torch.empty(n, hk, d, dtype=dq.dtype, device=dq.device)
            part = dwq = dwk = None
            if wq is not None:
                rows = _lib.get_lib(required=True).rb200_norm_rope_parts()
                part = torch.empty(rows, 2 * d, dtype=torch.float32, device=dq.device)
                dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
            st = (_i64 * 8)(*_strides(dq3, dk3), *(_strides(q3, k3) if wq is not None else [0] * 4))
            fn = _lib.bind("rb200_norm_rope_bwd", _BWD)
            _lib.check(fn(_ptr(dq3), _ptr(dk3), _ptr(q3), _ptr(k3), _ptr(positions), count, _ptr(frequencies), _ptr(wq), _ptr(wk), _ptr(gq), _ptr(gk), _ptr(part),
                          _ptr(dwq), _ptr(dwk), st, n, hq, hk, d, rot, 1 if dq.dtype == torch.bfloat16 else 0, is64,
                          1 if wq is not None and wq.dtype == torch.bfloat16 else 0, 1 if interleaved else 0, eps, amplitude, _lib.stream_ptr()),
                       "norm_rope_bwd")
            _lib.count_launch(2 if wq is not None else 1)
        return nodes.first_order("norm_rope", (gq.view(ctx.shapes[0]), gk.view(ctx.shapes[1]), None, None, dwq, dwk, None, None, None), (dq, dk, q3, k3, wq, wk))


def norm_rope(q: torch.Tensor, k: torch.Tensor, positions: Optional[torch.Tensor], frequencies: Optional[torch.Tensor], *,
              q_scale: Optional[torch.Tensor] = None, k_scale: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = True,
              amplitude: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    Norm per head and rotation of queries and keys (see the module docstring); differentiable in ``q``, ``k`` and the scales, once. Frequencies that require a gradient are
    refused.

    :param q: [..., heads, D] bf16 or fp32; any strides with unit stride over D (slices of a fused projection are read in place)
    :param k: [..., key heads, D] over the same tokens
    :param positions: int32 / int64 of the shape of the token axes, or of the last of them (then the same for all others)
    :param frequencies: fp32 [F], ``2 F <= D`` features are rotated (:func:`rope_frequencies`); None: no rotation
    :param q_scale: [D] scale of the norm of the queries; None (both): no norm
    :param k_scale: [D] scale of the norm of the keys
    :return: rotated q and k, contiguous
    """
    mod = nodes.of(q)
    if mod is not None:
        res = mod.norm_rope(q, k, positions, frequencies, q_scale, k_scale, eps, interleaved, amplitude)
        if res is not None:
            return res
    _check(q, k, positions, frequencies, q_scale, k_scale, "norm_rope")
    if _native_ok(q, q_scale, "norm_rope"):
        return _NormRopeFn.apply(q, k, positions, frequencies, q_scale, k_scale, float(eps), bool(interleaved), float(amplitude))
    return norm_rope_reference(q, k, positions, frequencies, q_scale=q_scale, k_scale=k_scale, eps=eps, interleaved=interleaved, amplitude=amplitude)


def norm_rope_to_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: Optional[torch.Tensor], frequencies: Optional[torch.Tensor],
                       k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *, q_scale: Optional[torch.Tensor] = None,
                       k_scale: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = True, amplitude: float = 1.0) -> torch.Tensor:
    """
    The same for serving, without gradient: normed and rotated keys and the values as they are go to the slots of their tokens.

    :param q: [N, heads, D]
    :param k: [N, key heads, D]
    :param v: [N, key heads, D]
    :param positions: [N] int32 / int64
    :param k_cache: [pages, key heads, page size, D] of the type of ``q``, any strides with unit stride over D; written in place
    :param v_cache: the same for the values
    :param slots: [N] int32, page * page size + place in the page (:func:`returnn_b200.ops.paged.append_tokens`). A token whose slot is negative or past
        the end is not stored. Two tokens of one call must not share a slot.
    :return: rotated q [N, heads, D]
    """
    what = "norm_rope_to_cache"
    mod = nodes.of(q)
    if mod is not None:
        res = mod.norm_rope_to_cache(q, k, v, k_cache, v_cache, slots, positions, frequencies, q_scale, k_scale, eps, interleaved, amplitude)
        if res is not None:
            return res
    _check(q, k, positions, frequencies, q_scale, k_scale, what)
    if q.dim() != 3 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError("%s: q %s, k %s, v %s %s must be [N, heads, D] of one type" % (what, tuple(q.shape), tuple(k.shape), tuple(v.shape), v.dtype))
    for c in (k_cache, v_cache):
        if c.dim() != 4 or c.shape[1] != k.shape[1] or c.shape[3] != k.shape[2] or c.shape != k_cache.shape or c.dtype != q.dtype or c.device != q.device:
            raise ValueError("%s: caches must be [pages, %i, page size, %i] %s on %s, got %s %s on %s" % (
                what, k.shape[1], k.shape[2], q.dtype, q.device, tuple(c.shape), c.dtype, c.device))
        if c.stride(3) != 1 and c.shape[3] > 1:
            raise ValueError("%s: caches need unit stride over the features" % what)
    if slots.shape != q.shape[:1] or slots.dtype != torch.int32 or slots.device != q.device:
        raise ValueError("%s: slots must be int32 [%i] on %s" % (what, q.shape[0], q.device))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, q_scale, k_scale, k_cache, v_cache)):
        raise RuntimeError("%s has no gradient: call it under torch.no_grad()" % what)
    if nodes.has_tangent(q, k, v, q_scale, k_scale, k_cache, v_cache):
        raise RuntimeError("%s has no derivative" % what)
    pages, page = k_cache.shape[0], k_cache.shape[2]
    if not _native_ok(q, q_scale, what):
        q, k = norm_rope_reference(q, k, positions, frequencies, q_scale=q_scale, k_scale=k_scale, eps=eps, interleaved=interleaved, amplitude=amplitude)
        keep = (slots >= 0) & (slots < pages * page)
        at = slots[keep].long()
        k_cache[at // page, :, at % page] = k[keep]
        v_cache[at // page, :, at % page] = v[keep]
        return q
    if page == 0:
        raise ValueError("%s: pages of no tokens" % what)
    with torch.cuda.device_of(q):
        q3, k3, v3 = _rows(q), _rows(k), _rows(v)
        n, hq, d = q3.shape
        hk = k3.shape[1]
        pos = _Positions(positions, frequencies)
        wq = q_scale.contiguous() if q_scale is not None else None
        wk = k_scale.contiguous() if k_scale is not None else None
        slots = slots.contiguous()
        out_q = torch.empty(n, hq, d, dtype=q.dtype, device=q.device)
        st = (_i64 * 12)(*_strides(q3, k3, v3, k_cache, v_cache))
        fn = _lib.bind("rb200_norm_rope_cache", _CACHE)
        _lib.check(fn(_ptr(q3), _ptr(k3), _ptr(v3), _ptr(pos.positions), pos.count, _ptr(pos.frequencies), _ptr(wq), _ptr(wk), _ptr(out_q), _ptr(k_cache),
                      _ptr(v_cache), _ptr(slots), st, n, hq, hk, d, pos.rot, page, pages * page, 1 if q.dtype == torch.bfloat16 else 0, pos.is64,
                      1 if wq is not None and wq.dtype == torch.bfloat16 else 0, 1 if interleaved else 0, float(eps), float(amplitude), _lib.stream_ptr()),
                   "norm_rope_to_cache")
        _lib.count_launch()
        nodes.written(k_cache, v_cache)
    return out_q


def norm_rope_reference(q, k, positions, frequencies, *, q_scale=None, k_scale=None, eps=1e-6, interleaved=True, amplitude=1.0):
    """plain torch in fp32 (differentiable)"""

    def one(x, scale):
        y = x.float()
        if scale is not None:
            y = y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + eps) * scale.float()
        if frequencies is None or not frequencies.numel():
            return y.to(x.dtype).clone(memory_format=torch.contiguous_format)
        f = frequencies.shape[0]
        rot, rest = y[..., : 2 * f], y[..., 2 * f:]
        a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :f], rot[..., f:])
        a, b = (a * cos - b * sin) * amplitude, (a * sin + b * cos) * amplitude
        rot = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
        return torch.cat([rot, rest], dim=-1).to(x.dtype).contiguous()

    cos = sin = None
    if frequencies is not None:
        angle = positions.double()[..., None, None] * frequencies.double()  # (a far position needs more than the 24 bits of a float)
        cos, sin = angle.cos().float(), angle.sin().float()
    return one(q, q_scale), one(k, k_scale)
