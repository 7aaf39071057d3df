"""Rotary position embedding of attention heads, alone or behind a per-head RMS norm.

``rotary`` turns the heads of one tensor; ``qk_norm_rotary`` norms the queries and keys of a
layer per head and turns them, in one launch (csrc/rotary.cu).  Both take any strides over
batch, head and token (so views of a packed q|k|v projection are used as they lie), explicit
positions (a decode step passes the cache positions of its tokens), the interleaved or the
half layout, and tables narrower than the head: lanes beyond the table are only normed.
Both are differentiable.  ``rotary_tables`` builds the tables, with the frequencies scaled
for contexts longer than the one trained on if wanted.

The reference has the interleaved rotation of whole heads only, without a norm
(src/llmlab/model/attention.py:10-58).
"""

from __future__ import annotations

import math
from ctypes import Structure, c_float, c_int, c_long, c_void_p
from dataclasses import dataclass
from functools import lru_cache
from struct import Struct

import torch
from torch.autograd.function import once_differentiable

from . import lib as _lib

LAYOUTS = ("interleaved", "half")
SCALINGS = ("linear", "ntk", "parts")
MAX_HEAD_DIM = 256
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class RotaryTensor(Structure):
    """Mirror of ``SflRotaryTensor`` in csrc/sfl.h."""

    _fields_ = [("x", c_void_p), ("y", c_void_p), ("dy", c_void_p), ("weight", c_void_p),
                ("x_b", c_long), ("x_h", c_long), ("x_t", c_long),
                ("y_b", c_long), ("y_h", c_long), ("y_t", c_long),
                ("dy_b", c_long), ("dy_h", c_long), ("dy_t", c_long), ("heads", c_int)]


class RotaryTable(Structure):
    """Mirror of ``SflRotaryTable`` in csrc/sfl.h."""

    _fields_ = [("cos", c_void_p), ("sin", c_void_p), ("positions", c_void_p),
                ("pos_b", c_long), ("pos_t", c_long), ("rows", c_int), ("rotated", c_int)]


# Calls pass the two records as packed bytes (the layouts above): filling ctypes structures field
# by field costs several microseconds, which a decode step pays per layer.
_TENSOR = Struct("4P9li4x")
_TABLE = Struct("3P2l2i")

_P = c_void_p
_lib.register_signature("sfl_rotary", [_P, c_int, _P, c_int, c_int, c_int, c_float, c_int, c_int,
                                       c_int, _P])
_lib.register_signature("sfl_rotary_bwd_partial_bytes", [c_int, c_int, c_int, c_int, c_int])
_lib.register_signature("sfl_rotary_bwd", [_P, c_int, _P, c_int, c_int, c_int, c_float, c_int, c_int,
                                           _P, c_long, _P, _P, _P])


# ------------------------------------------------------------------------ tables --
@dataclass(frozen=True)
class RotaryScaling:
    """Frequencies for contexts ``factor`` times longer than the ``trained`` positions.

    * ``"linear"``: every frequency divided by ``factor`` (positions interpolated);
    * ``"ntk"``: the base raised by ``factor ** (R / (R - 2))``, which keeps the fastest
      frequency and divides the slowest by ``factor``;
    * ``"parts"``: frequencies that turn at most ``slow_turns`` times within the trained
      positions are divided by ``factor``, those that turn at least ``fast_turns`` times are
      kept, and the ones in between are interpolated linearly in the number of turns.
    """

    kind: str
    factor: float
    trained: int = 0
    slow_turns: float = 1.0
    fast_turns: float = 4.0

    def __post_init__(self):
        if self.kind not in SCALINGS:
            raise ValueError("kind must be one of " + ", ".join(SCALINGS))
        if not math.isfinite(self.factor) or self.factor < 1:
            raise ValueError("factor must be finite and at least 1")
        if self.kind == "parts":
            if type(self.trained) is not int or self.trained <= 0:
                raise ValueError("'parts' needs the number of positions trained on")
            if not 0 < self.slow_turns < self.fast_turns:
                raise ValueError("require 0 < slow_turns < fast_turns")


def rotary_frequencies(rotated: int, theta: float = 10000.0,
                       scaling: RotaryScaling | None = None) -> torch.Tensor:
    """Angle per position of each rotated pair: float64 ``[rotated / 2]`` on the CPU."""
    if type(rotated) is not int or rotated <= 0 or rotated % 2:
        raise ValueError("rotated must be positive and even because pairs of lanes turn together")
    if not math.isfinite(theta) or theta <= 0:
        raise ValueError("theta must be finite and positive")
    if scaling is not None and scaling.kind == "ntk":
        if rotated == 2:
            raise ValueError("'ntk' needs more than one frequency")
        theta = theta * scaling.factor ** (rotated / (rotated - 2))
    freq = theta ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)
    if scaling is None or scaling.kind == "ntk":
        return freq
    if scaling.kind == "linear":
        return freq / scaling.factor
    turns = scaling.trained * freq / (2 * math.pi)
    keep = (turns - scaling.slow_turns) / (scaling.fast_turns - scaling.slow_turns)
    keep = keep.clamp(0.0, 1.0)
    return freq * keep + freq / scaling.factor * (1.0 - keep)


def rotary_tables(rotated: int, positions: int, theta: float = 10000.0,
                  scaling: RotaryScaling | None = None, device=None):
    """``(cos, sin)``, fp32 ``[positions, rotated / 2]``.  The angles are computed in float64:
    at position 100,000 an fp32 angle is off by up to 0.004 radians."""
    if type(positions) is not int or positions <= 0:
        raise ValueError("positions must be a positive integer")
    freq = rotary_frequencies(rotated, theta, scaling).to(device)
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return angles.cos().float(), angles.sin().float()


# -------------------------------------------------------------------- validation --
def _check_heads(x: torch.Tensor, name: str) -> None:
    if not isinstance(x, torch.Tensor) or x.ndim != 4:
        raise ValueError(f"{name} must be [batch, heads, tokens, head_dim]")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name} must be bf16, fp16 or fp32")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    _, heads, _, dim = x.shape
    if heads < 1 or not 1 <= dim <= MAX_HEAD_DIM:
        raise ValueError(f"{name} needs at least one head and a head dimension of 1 to "
                         f"{MAX_HEAD_DIM}")
    if dim > 1 and x.stride(3) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")


def _check_table(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions) -> None:
    device = x.device
    for t, name in ((cos, "cos"), (sin, "sin")):
        if (t.dtype != torch.float32 or t.ndim != 2 or t.device != device
                or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp32 [positions, rotated / 2] tensor on "
                             "the device of the heads")
    rows, half = cos.shape
    if sin.shape != cos.shape or rows < 1:
        raise ValueError("cos and sin must have the same shape with at least one position")
    if rows >= 2**31:
        raise ValueError("tables of 2**31 positions or more are not supported")
    B, _, T, D = x.shape
    if 2 * half > D:
        raise ValueError("the tables rotate more lanes than a head has")
    if positions is None:
        if T > rows:
            raise ValueError("more tokens than positions in the tables")
        return
    if positions.dtype != torch.int64 or positions.device != device:
        raise ValueError("positions must be int64 on the device of the heads")
    if positions.shape != (B, T) and positions.shape != (T,):
        raise ValueError("positions must be [tokens] or [batch, tokens]")


def _check_out(out: torch.Tensor, x: torch.Tensor, name: str) -> None:
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{name} must have the shape, type and device of its input")
    if out.shape[3] > 1 and out.stride(3) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError(f"{name} must not be an expanded tensor")


# ----------------------------------------------------------------------- launches --
def _new(x: torch.Tensor) -> torch.Tensor:
    """A result laid out token-major ([B, T, H, D] in memory), as a projection leaves heads."""
    B, H, T, D = x.shape
    return torch.empty_strided((B, H, T, D), (T * H * D, D, H * D, 1), dtype=x.dtype,
                               device=x.device)


def _record(x, y, dy, weight) -> bytes:
    x_b, x_h, x_t, _ = x.stride()
    y_b, y_h, y_t, _ = y.stride()
    dy_b, dy_h, dy_t, _ = (0, 0, 0, 0) if dy is None else dy.stride()
    return _TENSOR.pack(x.data_ptr(), y.data_ptr(), 0 if dy is None else dy.data_ptr(),
                        0 if weight is None else weight.data_ptr(), x_b, x_h, x_t, y_b, y_h, y_t,
                        dy_b, dy_h, dy_t, x.shape[1])


def _table(cos, sin, positions) -> bytes:
    rows, half = cos.shape
    at, pos_b, pos_t = 0, 0, 0
    if positions is not None:
        at, pos_t = positions.data_ptr(), positions.stride(-1)
        pos_b = positions.stride(0) if positions.ndim == 2 else 0
    return _TABLE.pack(cos.data_ptr(), sin.data_ptr(), at, pos_b, pos_t, rows, 2 * half)


def _launch(xs, ys, weights, cos, sin, positions, eps, layout, inverse=False) -> None:
    x = xs[0]
    B, _, T, D = x.shape
    if B == 0 or T == 0:
        return
    records = b"".join([_record(x, y, None, weight) for x, y, weight in zip(xs, ys, weights)])
    with _lib.on_device(x.device):
        code = _lib.lib().sfl_rotary(records, len(xs), _table(cos, sin, positions), B, T, D, eps,
                                     layout == "half", inverse, _DTYPES[x.dtype],
                                     _lib.stream_ptr())
    if code:
        _lib.check(code, "sfl_rotary")


@lru_cache(maxsize=64)
def _partial_bytes(device_index: int, dim: int) -> int:
    """Scratch of the backward grid on a device (current when this is called)."""
    size = _lib.lib().sfl_rotary_bwd_partial_bytes(1, 1, 1, 1, dim)
    if size <= 0:
        raise RuntimeError("sfl_rotary_bwd_partial_bytes refused the head dimension")
    return size


def _rows(grad: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    """A gradient in the type of its tensor whose head rows are contiguous."""
    if grad.dtype != like.dtype:
        grad = grad.to(like.dtype)
    return grad if grad.shape[3] == 1 or grad.stride(3) == 1 else grad.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin, positions, layout):
        y = _new(x)
        _launch([x], [y], [None], cos, sin, positions, 0.0, layout)
        ctx.save_for_backward(cos, sin, positions)
        ctx.layout = layout
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        cos, sin, positions = ctx.saved_tensors
        dy = _rows(dy, dy)
        dx = _new(dy)
        _launch([dy], [dx], [None], cos, sin, positions, 0.0, ctx.layout, inverse=True)
        return dx, None, None, None, None


class _QKNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, layout):
        ys = (_new(q), _new(k))
        _launch([q, k], ys, [q_weight, k_weight], cos, sin, positions, eps, layout)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps, ctx.layout = eps, layout
        return ys

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        dq, dk, dqw, dkw = qk_norm_rotary_grad(q, k, q_weight, k_weight, cos, sin, positions,
                                               dq_out, dk_out, eps=ctx.eps, layout=ctx.layout)
        return dq, dk, dqw, dkw, None, None, None, None, None


def qk_norm_rotary_grad(q, k, q_weight, k_weight, cos, sin, positions, dq_out, dk_out, *,
                        eps: float, layout: str, out=None):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of ``qk_norm_rotary`` for the gradients of its
    results; ``out`` names the tensors that receive dq and dk, which may be the incoming gradients
    themselves (a warp reads a head before it writes it).  The weight gradients are summed in a
    fixed order."""
    xs, gs = (q, k), (_rows(dq_out, q), _rows(dk_out, k))
    dxs = out if out is not None else (_new(q), _new(k))
    B, _, T, D = q.shape
    if B == 0 or T == 0:
        return (*dxs, torch.zeros_like(q_weight), torch.zeros_like(k_weight))
    device = q.device
    dqw, dkw = torch.empty(2, D, dtype=torch.float32, device=device).unbind(0)
    records = b"".join([_record(x, dx, dy, weight) for x, dx, dy, weight
                        in zip(xs, dxs, gs, (q_weight, k_weight))])
    with _lib.on_device(device):
        size = _partial_bytes(device.index, D)
        partial = torch.empty(size, dtype=torch.uint8, device=device)
        code = _lib.lib().sfl_rotary_bwd(records, 2, _table(cos, sin, positions), B, T, D, eps,
                                         layout == "half", _DTYPES[q.dtype], partial.data_ptr(),
                                         size, dqw.data_ptr(), dkw.data_ptr(), _lib.stream_ptr())
    if code:
        _lib.check(code, "sfl_rotary_bwd")
    return (*dxs, dqw, dkw)


def qk_norm_rotary_into(q, k, q_weight, k_weight, cos, sin, positions=None, *, eps: float,
                        layout: str = "interleaved", out) -> None:
    """``qk_norm_rotary`` into ``out`` without argument checks or autograd: the building block of
    models/fused.py, next to ``qk_norm_rotary_grad``."""
    _launch([q, k], out, [q_weight, k_weight], cos, sin, positions, eps, layout)


def _no_grad_out(out, *inputs) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in inputs):
        raise ValueError("out= is for inference: its result carries no gradient")


# -------------------------------------------------------------------------- public --
def rotary(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
           positions: torch.Tensor | None = None, *, layout: str = "interleaved",
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns the first ``2 * cos.shape[1]`` lanes of every head of ``x [B, H, T, D]``.

    ``positions`` (int64 ``[T]`` or ``[B, T]``) are rows of the tables; without them token ``t``
    is at position ``t``.  A position outside the tables makes the rotated lanes of its token
    NaN.  ``layout`` pairs lanes (2i, 2i+1) or (i, i + R/2).  The result is rounded once from
    fp32 to the type of ``x``; ``out`` (inference only) receives it; it may be ``x`` and must not overlap it in any other way.
    """
    if layout not in LAYOUTS:
        raise ValueError("layout must be one of " + ", ".join(LAYOUTS))
    _check_heads(x, "x")
    _check_table(x, cos, sin, positions)
    if out is not None:
        _no_grad_out(out, x)
        _check_out(out, x, "out")
        _launch([x], [out], [None], cos, sin, positions, 0.0, layout)
        return out
    if torch.is_grad_enabled() and x.requires_grad:
        return _Rotary.apply(x, cos, sin, positions, layout)
    out = _new(x)
    _launch([x], [out], [None], cos, sin, positions, 0.0, layout)
    return out


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
                   k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                   positions: torch.Tensor | None = None, *, eps: float = 1e-5,
                   layout: str = "interleaved", out=None):
    """``(q', k')``: every head of ``q [B, Hq, T, D]`` and ``k [B, Hk, T, D]`` divided by the root
    of its mean square plus ``eps``, multiplied by its fp32 weight ``[D]`` and turned as by
    ``rotary``.  Statistics and rotation are fp32; each result is rounded once.  ``out``
    (inference only) is a pair of tensors that receive the results, for example the rows of a
    KV cache that the new keys belong to; they may be ``q`` and ``k`` themselves
    and must not overlap either in any other way.
    """
    if layout not in LAYOUTS:
        raise ValueError("layout must be one of " + ", ".join(LAYOUTS))
    _check_heads(q, "q")
    _check_heads(k, "k")
    if k.dtype != q.dtype or k.device != q.device:
        raise TypeError("q and k must have the same type and device")
    if (k.shape[0], *k.shape[2:]) != (q.shape[0], *q.shape[2:]):
        raise ValueError("q and k must agree in batch, tokens and head dimension")
    for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if (t.dtype != torch.float32 or t.shape != (q.shape[3],) or not t.is_contiguous()
                or t.device != q.device):
            raise ValueError(f"{name} must be a contiguous fp32 [head_dim] tensor on the device of "
                             "the heads")
    if not math.isfinite(eps) or eps < 0:
        raise ValueError("eps must be finite and nonnegative")
    _check_table(q, cos, sin, positions)
    inputs = (q, k, q_weight, k_weight)
    if out is not None:
        _no_grad_out(out, *inputs)
        _check_out(out[0], q, "out[0]")
        _check_out(out[1], k, "out[1]")
        _launch([q, k], out, [q_weight, k_weight], cos, sin, positions, eps, layout)
        return tuple(out)
    if torch.is_grad_enabled() and any(t.requires_grad for t in inputs):
        return _QKNormRotary.apply(*inputs, cos, sin, positions, eps, layout)
    ys = (_new(q), _new(k))
    _launch([q, k], ys, [q_weight, k_weight], cos, sin, positions, eps, layout)
    return ys
