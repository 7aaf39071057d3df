"""Softmax cross entropy of a vocabulary projection that keeps no logits.

``linear_cross_entropy(hidden, weight, targets)`` is
``cross_entropy(hidden @ weight.T, targets)`` and its gradients, computed by csrc/linear_ce.cu
in pieces of the vocabulary: forward keeps one log-sum-exp per row, backward computes the
logits of a piece again and consumes them at once.  Memory beyond inputs and results is
``2 * rows * piece`` bytes for the piece in hand (``piece_size``) and 16 bytes per row and 256
entries of the vocabulary for the statistics.

The head of models/fused.py that keeps bf16 logits does fewer operations (6 N D V against
8 N D V) and rounds them; this one is for vocabularies whose logits are too large to keep, and
never rounds a logit.  The reference materialises logits and softmax
(src/llmlab/training/loss.py:4-22).
"""

from __future__ import annotations

from ctypes import Structure, c_int, c_int64, c_long, c_void_p
from struct import Struct

import torch
from torch.autograd.function import once_differentiable

from . import lib as _lib
from .gemm import captured_status_word

REDUCTIONS = ("mean", "sum", "none")
PIECE_STEP = 256                 # a piece is whole 256-column tiles
PIECE_BYTES = 192 << 20          # of dl in flight
MIN_PIECE = 2048
_DTYPES = (torch.bfloat16, torch.float16)
_OUT_16, _OUT_F32, _OUT_F32_ADD, _OUT_NONE = range(4)


class LinearCe(Structure):
    """Mirror of ``SflLinearCe`` in csrc/sfl.h."""

    _fields_ = [("hidden", c_void_p), ("ld_hidden", c_long), ("weight", c_void_p),
                ("ld_weight", c_long), ("targets", c_void_p), ("ignore_index", c_int64),
                ("rows", c_int), ("dim", c_int), ("vocab", c_int), ("fp16", c_int),
                ("lse2", c_void_p), ("status", c_void_p)]


class LinearCeGrad(Structure):
    """Mirror of ``SflLinearCeGrad`` in csrc/sfl.h."""

    _fields_ = [("grad", c_void_p), ("totals", c_void_p), ("dlogits", c_void_p),
                ("dh_sum", c_void_p), ("dh_sum_bytes", c_long), ("dh", c_void_p), ("ld_dh", c_long), ("dw", c_void_p),
                ("ld_dw", c_long), ("dw_kind", c_int), ("piece", c_int)]


# Calls pass the two records as packed bytes (the layouts above), as ops/rotary.py does.
_CALL = Struct("PlPlPq4i2P")
_GRAD = Struct("4PlPlPl2i")

_P = c_void_p
_lib.register_signature("sfl_linear_ce_part_bytes", [c_int, c_int])
_lib.register_signature("sfl_linear_ce_fwd", [_P, _P, c_long, _P, c_int, _P, _P, _P])
_lib.register_signature("sfl_linear_ce_dh_sum_bytes", [c_int, c_int, c_int, c_int, c_int])
_lib.register_signature("sfl_linear_ce_bwd", [_P, _P, _P])


def piece_size(rows: int, vocab: int) -> int:
    """Entries of the vocabulary per piece: as many as keep dl at ``PIECE_BYTES``, at least
    ``MIN_PIECE`` (smaller pieces leave the products too few tiles for the SMs), at most all.

    Forward and backward of 4096 x 1024 x 10000 take 0.25 ms in one piece, 0.35 ms with 9472
    entries in the first and 0.36 ms in pieces of 4096; 8192 x 2048 x 131072 takes 13.7 to 13.9 ms in pieces of
    12288, 14.3 to 14.5 of 2048, 14.2 to 14.6 in one (2.1 GB of dl)."""
    fit = PIECE_BYTES // (2 * rows) // PIECE_STEP * PIECE_STEP
    return min(max(fit, MIN_PIECE), -(-vocab // PIECE_STEP) * PIECE_STEP)


def _check(hidden, weight, targets) -> None:
    if not isinstance(hidden, torch.Tensor) or not hidden.is_cuda:
        raise ValueError("hidden must be a CUDA tensor")
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise TypeError("hidden and weight must both be bf16 or both be fp16")
    if hidden.ndim < 1 or weight.ndim != 2 or weight.shape[1] != hidden.shape[-1]:
        raise ValueError("expected hidden [..., dim] and weight [vocab, dim]")
    if weight.device != hidden.device or targets.device != hidden.device:
        raise ValueError("hidden, weight and targets must be on the same device")
    dim = hidden.shape[-1]
    if dim == 0 or dim % 8:
        raise ValueError("dim must be a positive multiple of 8")
    if weight.shape[0] == 0:
        raise ValueError("the vocabulary is empty")
    if targets.dtype != torch.int64 or targets.shape != hidden.shape[:-1]:
        raise ValueError("targets must be int64 with the shape of hidden without its last dimension")
    if max(targets.numel(), weight.shape[0]) >= 2**31:
        raise ValueError("2**31 rows or vocabulary entries are not supported")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as a matrix whose rows TMA can address (16-byte aligned, contiguous), copying only
    what does not lie that way already."""
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    pitch, step = t.stride()
    if step != 1 or pitch % 8 or pitch < t.shape[1] or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _call(hidden, weight, targets, ignore_index, lse2: int) -> bytes:
    rows, dim = hidden.shape
    return _CALL.pack(hidden.data_ptr(), hidden.stride(0), weight.data_ptr(), weight.stride(0),
                      targets.data_ptr(), ignore_index, rows, dim, weight.shape[0],
                      hidden.dtype == torch.float16, lse2,
                      captured_status_word(hidden.device).data_ptr())


def _forward(hidden, weight, targets, ignore_index: int, mean: bool | None, row_loss):
    """``(kept, loss)``: ``kept`` is lse2 of the rows and behind them the two totals.  Without a
    tensor for them the rows' losses stay in scratch."""
    rows = hidden.shape[0]
    dev = hidden.device
    handle = _lib.lib()
    size = handle.sfl_linear_ce_part_bytes(rows, weight.shape[0])
    scratch = torch.empty(size + 4 * rows, dtype=torch.uint8, device=dev)
    part = scratch.data_ptr()
    kept = torch.empty(rows + 2, dtype=torch.float32, device=dev)
    lse2 = kept.data_ptr()
    loss = None if mean is None else torch.empty((), dtype=torch.float32, device=dev)
    args = _call(hidden, weight, targets, ignore_index, lse2)
    with _lib.on_device(dev):
        code = handle.sfl_linear_ce_fwd(args, part, size,
                                        part + size if row_loss is None else row_loss.data_ptr(),
                                        bool(mean), None if loss is None else lse2 + 4 * rows,
                                        _lib.ptr(loss), _lib.stream_ptr())
    _lib.check(code, "sfl_linear_ce_fwd")
    _lib.count_kernels(2 if loss is None else 3)
    return kept, loss


def _backward(hidden, weight, targets, ignore_index: int, lse2: int, grad, totals: int | None, dw,
              accumulate: bool, piece: int | None, need_dh: bool) -> torch.Tensor | None:
    rows, dim = hidden.shape
    vocab = weight.shape[0]
    dev = hidden.device
    if dw is None and not need_dh:
        raise ValueError("nothing to compute")
    if dw is None:
        kind = _OUT_NONE
    elif dw.dtype == torch.float32:
        kind = _OUT_F32_ADD if accumulate else _OUT_F32
    elif dw.dtype == hidden.dtype and not accumulate:
        kind = _OUT_16
    else:
        raise ValueError("dw must be fp32, or of the operands' type when it is overwritten")
    if piece is None:
        piece = piece_size(rows, vocab)
    dh = torch.empty(rows, dim, dtype=hidden.dtype, device=dev) if need_dh else None
    args = _call(hidden, weight, targets, ignore_index, lse2)
    handle = _lib.lib()
    with _lib.on_device(dev):
        size = (handle.sfl_linear_ce_dh_sum_bytes(rows, dim, vocab, piece, dw is not None)
                if need_dh else 0)
        dl_bytes = -(-2 * rows * piece // 256) * 256
        scratch = torch.empty(dl_bytes + size, dtype=torch.uint8, device=dev)
        dlogits = scratch.data_ptr()
        grads = _GRAD.pack(0 if grad is None else grad.data_ptr(), totals or 0, dlogits,
                           dlogits + dl_bytes if size > 0 else 0, size,
                           0 if dh is None else dh.data_ptr(), dim,
                           0 if dw is None else dw.data_ptr(), 0 if dw is None else dw.stride(0),
                           kind, piece)
        code = handle.sfl_linear_ce_bwd(args, grads, _lib.stream_ptr())
    _lib.check(code, "sfl_linear_ce_bwd")
    _lib.count_kernels(2 * -(-vocab // piece) + (size > 0))
    return dh


def linear_ce_forward(hidden, weight, targets, ignore_index: int, mean: bool | None):
    """Kernels of the forward pass over prepared matrices: ``(row_loss, lse2, totals, loss)``.
    ``mean`` None leaves out the reduction (totals and loss are None)."""
    rows = hidden.shape[0]
    row_loss = torch.empty(rows, dtype=torch.float32, device=hidden.device)
    kept, loss = _forward(hidden, weight, targets, ignore_index, mean, row_loss)
    return row_loss, kept[:rows], None if mean is None else kept[rows:], loss


def linear_ce_backward(hidden, weight, targets, ignore_index: int, lse2, grad, totals, dw,
                       accumulate: bool = False, piece: int | None = None,
                       need_dh: bool = True) -> torch.Tensor | None:
    """Kernels of the backward pass: writes (or, for fp32 ``dw``, adds to) the weight gradient and
    returns dh.  ``grad`` is a device scalar; with ``totals`` both are divided by the count.  Without
    ``dw``, or without ``need_dh``, that product is not computed."""
    return _backward(hidden, weight, targets, ignore_index, lse2.data_ptr(), grad, _lib.ptr(totals),
                     dw, accumulate, piece, need_dh)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, mean):
        h, w = _rows(hidden), _rows(weight)
        t = _flat(targets)
        kept, loss = _forward(h, w, t, ignore_index, mean, None)
        ctx.save_for_backward(h, w, t, kept)
        ctx.ignore_index, ctx.mean, ctx.shape = ignore_index, mean, hidden.shape
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        h, w, t, kept = ctx.saved_tensors
        lse2 = kept.data_ptr()
        need_dh, need_dw = ctx.needs_input_grad[:2]      # a frozen head, or frozen hidden states
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if need_dw else None
        dh = _backward(h, w, t, ctx.ignore_index, lse2, grad.float(),
                       lse2 + 4 * h.shape[0] if ctx.mean else None, dw, False, None, need_dh)
        if need_dh and dh.shape != ctx.shape:
            dh = dh.view(ctx.shape)
        return dh, dw, None, None, None


def _flat(targets: torch.Tensor) -> torch.Tensor:
    return targets if targets.ndim == 1 and targets.is_contiguous() else targets.reshape(-1).contiguous()


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``hidden [..., dim] @ weight [vocab, dim].T`` with ``targets [...]``.

    ``hidden`` and ``weight`` are both bf16 or both fp16, ``dim`` a multiple of 8, ``targets``
    int64.  Rows whose target is ``ignore_index`` add nothing to the loss or the gradients (their
    hidden states must still be finite: a product with them runs); any other target outside the
    vocabulary makes the result NaN.  ``"mean"`` divides by the rows that count (NaN when none
    does, with zero gradients), ``"sum"`` does not; both return an fp32 scalar that is
    differentiable in ``hidden`` and ``weight``, with gradients in their type; only those that are
    asked for are computed (backward of 8192 x 2048 x 131072: 10.2 ms, with a frozen head 7.0).  ``"none"`` returns
    the fp32 loss of each row for scoring and is refused where a gradient would be needed.
    """
    if reduction not in REDUCTIONS:
        raise ValueError("reduction must be one of " + ", ".join(REDUCTIONS))
    if type(ignore_index) is not int or not -2**63 <= ignore_index < 2**63:
        raise ValueError("ignore_index must be an integer")
    _check(hidden, weight, targets)
    needs_grad = torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)
    if reduction == "none" and needs_grad:
        raise ValueError("reduction='none' is for scoring and carries no gradient: detach hidden "
                         "and weight, or call it under torch.no_grad()")
    if targets.numel() == 0:
        if reduction == "none":
            return torch.zeros(targets.shape, dtype=torch.float32, device=hidden.device)
        # the sum of nothing keeps its place in the graph; the mean of nothing is NaN
        nothing = hidden.float().sum() + weight[:0].float().sum()
        return nothing + float("nan") if reduction == "mean" else nothing
    if needs_grad:
        return _LinearCrossEntropy.apply(hidden, weight, targets, ignore_index, reduction == "mean")
    h, w = _rows(hidden), _rows(weight)
    t = _flat(targets)
    if reduction == "none":
        row_loss = torch.empty(targets.shape, dtype=torch.float32, device=hidden.device)
        _forward(h, w, t, ignore_index, None, row_loss)
        return row_loss
    return _forward(h, w, t, ignore_index, reduction == "mean", None)[1]
