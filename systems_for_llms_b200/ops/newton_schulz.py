"""Orthogonalised updates by Newton-Schulz products (csrc/newton_schulz.cu).

``newton_schulz(update)`` takes a matrix or a stack of matrices and returns, for each, the
matrix with the same singular vectors whose singular values went through ``steps`` applications
of an odd quintic: with the default coefficients values between 0.003 and 1 of the norm end
between 0.7 and 1.2.  It is what ``optim.FusedMuon`` does to its momentum.  The reference has
no counterpart (it trains with AdamW, src/llmlab/train.py:169).
"""

from __future__ import annotations

import math
from ctypes import POINTER, Structure, byref, c_float, c_int, c_long, c_void_p
from functools import lru_cache

import torch

from . import lib as _lib
from .gemm import captured_status_word

QUINTIC = (3.4445, -4.7750, 2.0315)
MAX_STEPS = 64
MAX_STACK = 65535
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class NewtonSchulz(Structure):
    """Mirror of ``SflNewtonSchulz`` in csrc/sfl.h."""

    _fields_ = [("update", c_void_p), ("stride0", c_long), ("stride1", c_long), ("row", c_long),
                ("inner", c_int), ("batch", c_int), ("m", c_int), ("n", c_int), ("steps", c_int),
                ("dtype", c_int), ("a", c_float), ("b", c_float), ("c", c_float), ("eps", c_float),
                ("out", c_void_p), ("work", c_void_p), ("work_bytes", c_long),
                ("status", c_void_p)]


_P = c_void_p
_lib.register_signature("sfl_newton_schulz_bytes", [c_int, c_int, c_int])
_lib.register_signature("sfl_newton_schulz_kernels", [c_int, c_int, c_int])
_lib.register_signature("sfl_newton_schulz", [POINTER(NewtonSchulz), _P])

_lib.register_signature("sfl_muon_momentum", [_P, _P, _P, c_int, c_long, c_long, c_float, c_int, _P,
                                              _P, _P])
_lib.register_signature("sfl_muon_apply", [_P, _P, _P, c_int, c_long, c_long, c_float, c_float, _P,
                                           _P])


def muon_momentum(grad: torch.Tensor, buffer: torch.Tensor, update: torch.Tensor, *,
                  momentum: float, nesterov: bool, coef: torch.Tensor | None = None,
                  ok_flag: torch.Tensor | None = None) -> None:
    """Momentum of the rows (layers) of two equally strided fp32 views ``[rows, len]`` and the
    packed ``update`` that is to be orthogonalised."""
    rows, length = grad.shape
    if buffer.shape != grad.shape or buffer.stride() != grad.stride() or grad.stride(1) != 1:
        raise ValueError("grad and buffer must be equally strided rows")
    if update.numel() != grad.numel() or not update.is_contiguous():
        raise ValueError("update must be contiguous with the elements of grad")
    with _lib.on_device(grad.device):
        code = _lib.lib().sfl_muon_momentum(grad.data_ptr(), buffer.data_ptr(), update.data_ptr(),
                                            rows, length, grad.stride(0), float(momentum),
                                            int(nesterov), _lib.ptr(coef), _lib.ptr(ok_flag),
                                            _lib.stream_ptr())
    _lib.check(code, "sfl_muon_momentum")


def muon_apply(param: torch.Tensor, shadow: torch.Tensor | None, update: torch.Tensor, *,
               decay: float, rate: float, ok_flag: torch.Tensor | None = None) -> None:
    """``param <- decay * param - rate * update`` on the rows of a view ``[rows, len]``, and the
    equally strided bf16 copy."""
    rows, length = param.shape
    if shadow is not None and (shadow.shape != param.shape or shadow.stride() != param.stride()):
        raise ValueError("shadow must have the rows of param")
    if update.numel() != param.numel() or not update.is_contiguous() or param.stride(1) != 1:
        raise ValueError("update must be contiguous with the elements of param")
    with _lib.on_device(param.device):
        code = _lib.lib().sfl_muon_apply(param.data_ptr(), _lib.ptr(shadow), update.data_ptr(), rows,
                                         length, param.stride(0), float(decay), float(rate),
                                         _lib.ptr(ok_flag), _lib.stream_ptr())
    _lib.check(code, "sfl_muon_apply")


def largest_singular_value(coefficients=QUINTIC, steps: int = 5) -> float:
    """Largest value that singular values starting in [0, 1] reach within ``steps`` applications
    of ``a s + b s^3 + c s^5``; infinite when they run away."""
    a, b, c = coefficients
    low, high, worst = 0.0, 1.0, 1.0
    for _ in range(steps):
        points = [low, high]
        # interior extrema: a + 3 b s^2 + 5 c s^4 = 0
        if c == 0:
            squares = [-a / (3 * b)] if b else []
        else:
            inside = 9 * b * b - 20 * a * c
            squares = ([(-3 * b + sign * math.sqrt(inside)) / (10 * c) for sign in (1, -1)]
                       if inside >= 0 else [])
        points += [s for s in (math.sqrt(q) for q in squares if q > 0) if low < s < high]
        images = [s * (a + s * s * (b + c * s * s)) for s in points]
        # the sign of a singular value does not matter to the next step
        high = max(abs(v) for v in images)
        low = 0.0
        worst = max(worst, high)
        if not high < 1e6:
            return math.inf
    return worst


_largest_singular_value = lru_cache(maxsize=64)(largest_singular_value)


def _strided(update: torch.Tensor) -> torch.Tensor:
    """``update`` with rows the kernels can read (last dimension contiguous) and at most two
    leading dimensions; copies only what does not lie that way."""
    if update.ndim > 4:
        update = update.reshape(-1, *update.shape[-2:])
    if update.shape[-1] > 1 and update.stride(-1) != 1:
        update = update.contiguous()
    return update


def _overlap(out: torch.Tensor, update: torch.Tensor) -> bool:
    """Whether contiguous ``out`` lies within the bytes that ``update`` spans without being it."""
    begin, size = update.data_ptr(), update.element_size()
    end = begin + size * (1 + sum((n - 1) * s for n, s in zip(update.shape, update.stride())))
    at = out.data_ptr()
    if at >= end or at + 2 * out.numel() <= begin:
        return False
    return not (at == begin and update.dtype == out.dtype and update.is_contiguous())


def newton_schulz(update: torch.Tensor, *, steps: int = 5, coefficients=QUINTIC,
                  eps: float = 1e-7, out: torch.Tensor | None = None) -> torch.Tensor:
    """Orthogonalises every matrix of ``update [..., m, n]`` (bf16, fp16 or fp32).

    Each matrix is divided by its Frobenius norm plus ``eps`` and taken through ``steps`` times
    ``X <- a X + (b G + c G G) X`` with ``G`` the Gram matrix of its shorter side and
    ``coefficients = (a, b, c)``.  Up to two leading dimensions may have any strides (the same
    parameter of all layers inside a flat buffer is one call).  The result is bf16, contiguous,
    computed with fp16 operands whose rounding does not compound (off by about 0.002 of its norm,
    rounding to bf16 included; the normalised matrix is held to 2^-37 absolutely, which only shows
    where ``eps`` dwarfs the norm and the result is far below 1).  A matrix of zeros gives zeros
    (NaN, as 0 / 0 is, where ``eps`` is 0); one that holds an infinity or NaN
    gives NaN without touching its neighbours.  ``out`` receives the result; it may be a contiguous
    bf16 ``update`` itself and is otherwise refused when it lies within the bytes the update spans.
    Coefficients under which singular values starting below 1 exceed 2 are refused: the operands are
    scaled for bounded ones.  The operator is not differentiable.
    """
    if not isinstance(update, torch.Tensor) or not update.is_cuda:
        raise ValueError("update must be a CUDA tensor")
    if update.dtype not in _DTYPES:
        raise TypeError("update must be bf16, fp16 or fp32")
    if update.ndim < 2:
        raise ValueError("update must be a matrix or a stack of matrices")
    if update.requires_grad and torch.is_grad_enabled():
        raise ValueError("newton_schulz is not differentiable: detach the update or call it under "
                         "torch.no_grad()")
    if type(steps) is not int or not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"steps must be an integer in [1, {MAX_STEPS}]")
    if not math.isfinite(eps) or eps < 0:
        raise ValueError("eps must be finite and nonnegative")
    a, b, c = (float(v) for v in coefficients)
    if not all(math.isfinite(v) for v in (a, b, c)):
        raise ValueError("coefficients must be finite")
    # Bounded by 2 on [0, 1], |a| is at most 10 and |b s^2 + c s^4| at most 14 (twice Chebyshev's
    # polynomial of degree five is the extreme), which fp16 holds times 2^12.
    if _largest_singular_value((a, b, c), steps) > 2.0 * (1 + 1e-12):      # a rounding above is 2
        raise ValueError("these coefficients let singular values exceed 2")
    m, n = update.shape[-2:]
    if max(m, n) >= 2**31:
        raise ValueError("matrices of 2**31 rows or columns are not supported")
    if out is None:
        out = torch.empty(update.shape, dtype=torch.bfloat16, device=update.device)
    elif (out.shape != update.shape or out.dtype != torch.bfloat16 or not out.is_contiguous()
          or out.device != update.device):
        raise ValueError("out must be a contiguous bf16 tensor of the update's shape on its device")
    elif out.numel() and _overlap(out, update):
        raise ValueError("out must be update itself (contiguous bf16) or lie apart from it")
    if update.numel() == 0:
        return out
    x = _strided(update)
    lead = x.shape[:-2]
    batch = math.prod(lead)
    if batch > MAX_STACK:
        raise ValueError(f"a stack holds at most {MAX_STACK} matrices")
    handle = _lib.lib()
    size = handle.sfl_newton_schulz_bytes(batch, m, n)
    if size <= 0:
        raise ValueError("matrices too large")
    work = torch.empty(size, dtype=torch.uint8, device=x.device)
    args = NewtonSchulz(update=x.data_ptr(), row=x.stride(-2), inner=1, batch=batch, m=m, n=n,
                        steps=steps, dtype=_DTYPES[x.dtype], a=a, b=b, c=c, eps=eps,
                        out=out.data_ptr(), work=work.data_ptr(), work_bytes=size,
                        status=captured_status_word(x.device).data_ptr())
    if len(lead) == 1:
        args.stride0 = x.stride(0)
    elif len(lead) == 2:
        args.stride0, args.stride1, args.inner = x.stride(0), x.stride(1), lead[1]
    with _lib.on_device(x.device):
        code = handle.sfl_newton_schulz(byref(args), _lib.stream_ptr())
    _lib.check(code, "sfl_newton_schulz")
    _lib.count_kernels(handle.sfl_newton_schulz_kernels(m, n, steps))
    return out


def newton_schulz_portable(update: torch.Tensor, *, steps: int = 5, coefficients=QUINTIC,
                           eps: float = 1e-7) -> torch.Tensor:
    """The same in fp32 PyTorch operators, for devices without the kernels; fp32 result."""
    a, b, c = coefficients
    x = update.float()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.mT if tall else x
