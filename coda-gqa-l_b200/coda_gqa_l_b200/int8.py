"""Rows in 8 bits: RMS norm with the residual's addition, quantisation, and the product of 8-bit rows.

The projections of a decoder layer with 8-bit weights and activations (no counterpart upstream, whose projections are
``nn.Linear`` modules): the hidden state is normed and quantised one row (token) at a time, a weight is quantised once,
one row (output channel) at a time, and the product runs in integers on the tensor cores::

    q, h = add_rms_norm(x, norm.weight, residual=r, int8=True)      # h = x + r, q = its norm in 8 bits
    w = quantize_int8(linear.weight)                                # once
    y = int8_linear(q, w, linear.bias)                              # ~ linear(norm(x + r))

``CoDAGQALandmarkPerf2.use_int8_projections`` and ``CoDAStack(norms=...)`` put them to use.  Everything here is for
inference (activations that need a gradient are refused), runs on the current stream of the tensors' device and may be
captured into a CUDA graph.  Tensors are float32 or bfloat16, as everywhere in this package; scales are float32.

A call is one native function (torch_ext/torch_binding.cpp: checks, allocation, launch; the C ABI below it is
``coda_b200_add_rms_norm`` and its neighbours in include/coda_b200.h), because the rows of a decode step take the GPU less
time than the host takes to ask for them.  Under a dispatch mode (fake tensors, tracers) and under ``torch.jit.trace`` the
calls go through the operators of the same names in ``torch.ops.coda_b200``.
"""
from __future__ import annotations

from typing import Dict, NamedTuple, Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as forward_ad

__all__ = ["Int8Rows", "add_rms_norm", "int8_linear", "int8_status", "quantize_int8"]

_STATUS: Dict[int, torch.Tensor] = {}      # per device: code of a bounded wait that expired in int8_linear
_modes = torch._C._len_torch_dispatch_stack
_tracing = torch._C._get_tracing_state
_native = None


class _Ops:
    """The native module's functions, through the dispatcher, with its refusals of derivatives."""

    def __init__(self, ns):
        self._ns = ns

    @staticmethod
    def _inference(what, *activations, weights=(), parameter=False):
        for t in (*activations, *weights):
            if t is not None and forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} is for inference: it has no derivative (a tensor carries a tangent)")
        for t in activations:
            if t is not None and t.requires_grad and torch.is_grad_enabled() and not (parameter and isinstance(t, torch.nn.Parameter)):
                raise RuntimeError(f"{what} is for inference: it has no gradient (use torch.no_grad())")

    def quantize_int8(self, x):
        self._inference("quantize_int8", x, parameter=True)
        return self._ns.quantize_int8(x)

    def dequantize_int8(self, values, scale, dtype):
        self._inference("dequantize", values, scale)
        return self._ns.dequantize_int8(values, scale, dtype)

    def add_rms_norm(self, x, weight, residual, eps, int8):
        self._inference("add_rms_norm", x, residual, weights=(weight,))
        if not eps > 0.0:
            raise ValueError("add_rms_norm: eps must be positive")
        out = (self._ns.add_rms_norm_int8 if int8 else self._ns.add_rms_norm)(x, weight, residual, eps)
        return out if residual is not None else (*out[:-1], x)

    def int8_linear(self, x, x_scale, w, w_scale, bias, residual, dtype, status, w_ready):
        self._inference("int8_linear", x, x_scale, residual, weights=(w, w_scale, bias))
        return self._ns.int8_linear(x, x_scale, w, w_scale, bias, residual, dtype, status, w_ready)


def _calls():
    global _native
    if _modes() or _tracing() is not None:
        from . import torch_ops
        return _Ops(torch_ops.load())
    if _native is None:
        from . import torch_ops
        _native = torch_ops.native()
    return _native


class Int8Rows(NamedTuple):
    """Rows in 8 bits: ``values`` int8 (..., K) and ``scale`` float32 (...), standing for ``values * scale[..., None]``.

    The functions here make rows that start every ``(K + 15) // 16 * 16`` bytes, with nothing in between; other layouts are
    accepted and copied into that one by every call that needs it."""
    values: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values the rows stand for, each rounded once to ``dtype`` (float32 or bfloat16)."""
        return _calls().dequantize_int8(self.values, self.scale, dtype)


def quantize_int8(x: torch.Tensor) -> Int8Rows:
    """Rows of ``x`` (..., K) in 8 bits: a row's scale is its largest magnitude over 127 (rounded to float32), its values
    are the integers nearest to 127 times an element over that magnitude, ties to even.  A row whose largest magnitude is
    under 2^-100 becomes zeros with scale 0; a row that holds a NaN or an infinity gets scale NaN, and NaN is what any
    product with it is.  For activations (a row is a token) and, once, for a ``nn.Linear`` weight (a row is an output
    channel)."""
    return Int8Rows(*_calls().quantize_int8(x))


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 int8: bool = False) -> Tuple[Union[torch.Tensor, Int8Rows], torch.Tensor]:
    """``(norm(s), s)`` of ``s = x + residual`` over the last dimension, in one pass:
    ``norm(s) = s * rsqrt(mean(s^2) + eps) * weight``, of the sum before it is rounded to the type of ``x``.

    ``int8=True``: the normed rows in 8 bits (:func:`quantize_int8` of the unrounded norm) instead of the type of ``x``.
    Without ``residual`` the second result is ``x`` itself.  ``x`` (..., D), ``residual`` the same shape, ``weight``
    (D,), all of one type.  Squares are summed in float32: rows with magnitudes over 1e19 are out of range."""
    if int8:
        values, scale, total = _calls().add_rms_norm(x, weight, residual, eps, True)
        return Int8Rows(values, scale), total
    return _calls().add_rms_norm(x, weight, residual, eps, False)


def _status_word(t: torch.Tensor) -> Optional[torch.Tensor]:
    if _modes():                                           # (fake tensors do not mix with this one)
        return None
    word = _STATUS.get(t.get_device())
    if word is None and t.is_cuda:
        if torch.cuda.is_current_stream_capturing():       # (its zero would be written by the replays, not now)
            return None
        word = _STATUS[t.get_device()] = torch.zeros(1, dtype=torch.int32, device=t.device)
    return word


def int8_status(device: Union[torch.device, str, int, None] = None) -> int:
    """0, or the code of a bounded device-side wait that expired in an :func:`int8_linear` on ``device`` (default: the
    current one) -- what it returned since then is not valid.  Synchronises.  A call captured into a CUDA graph reports
    here if one outside a capture went before it."""
    device = torch.device("cuda" if device is None else device)
    idx = device.index if device.index is not None else torch.cuda.current_device()
    return int(_STATUS[idx].item()) if idx in _STATUS else 0


def int8_linear(x: Int8Rows, weight: Int8Rows, bias: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ weight.T (+ bias) (+ residual)`` of 8-bit rows, (..., K) by (N, K) to (..., N) in ``dtype``.

    The products are summed exactly in 32-bit integers (hence ``K`` up to 131071), scaled by the token's and the
    channel's scale, bias and residual are added in float32 and the result is rounded once.  ``bias`` (N,) and
    ``residual`` (..., N) are of ``dtype``."""
    return int8_gemm(x, weight, bias, residual, dtype, _status_word(x[0]))


def int8_gemm(x: Int8Rows, weight: Int8Rows, bias: Optional[torch.Tensor], residual: Optional[torch.Tensor], dtype: torch.dtype,
              status: Optional[torch.Tensor], w_ready: bool = False) -> torch.Tensor:
    """:func:`int8_linear` for a caller with a status word of its own.  ``w_ready``: the weight's values were complete
    before this call, or before an earlier product on this stream began, so they may be requested while the kernels ahead
    of this one still run."""
    return _calls().int8_linear(x[0], x[1], weight[0], weight[1], bias, residual, dtype, status, w_ready)
