"""Refusals and sizes of the projection cross entropy (CPU)."""

import ctypes

import pytest
import torch

from systems_for_llms_b200.ops.linear_loss import (LinearCe, LinearCeGrad, MIN_PIECE, PIECE_BYTES,
                                                   PIECE_STEP, _rows, linear_cross_entropy,
                                                   piece_size)


def test_cpu_tensors_and_bad_options_are_refused():
    h, w, t = torch.zeros(4, 8).bfloat16(), torch.zeros(6, 8).bfloat16(), torch.zeros(4).long()
    with pytest.raises(ValueError, match="CUDA"):
        linear_cross_entropy(h, w, t)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(h, w, t, reduction="batchmean")
    for bad in (1.0, None, True, 2 ** 63):
        with pytest.raises(ValueError, match="ignore_index"):
            linear_cross_entropy(h, w, t, ignore_index=bad)


@pytest.mark.parametrize("rows", [1, 173, 4096, 100_000, 10_000_000])
@pytest.mark.parametrize("vocab", [1, 255, 256, 257, 10000, 131072])
def test_piece_sizes(rows, vocab):
    piece = piece_size(rows, vocab)
    assert piece % PIECE_STEP == 0 and piece >= PIECE_STEP
    assert piece - PIECE_STEP < vocab                      # no tile beyond the vocabulary
    assert 2 * rows * piece <= max(PIECE_BYTES, 2 * rows * MIN_PIECE)
    if piece < vocab:
        assert piece >= MIN_PIECE


def test_rows_are_copied_only_when_they_have_to_be():
    x = torch.arange(64.0).view(4, 16).bfloat16()
    assert _rows(x).data_ptr() == x.data_ptr()
    pitched = torch.zeros(4, 24).bfloat16()[:, :16]
    assert _rows(pitched).data_ptr() == pitched.data_ptr()
    for odd in (torch.zeros(4, 17).bfloat16()[:, :16], x.t().contiguous().t(),
                torch.zeros(65).bfloat16()[1:].view(4, 16), x[:1].expand(4, 16)):
        got = _rows(odd)
        assert got.is_contiguous() and got.data_ptr() % 16 == 0 and torch.equal(got, odd)


def test_entry_points_refuse_before_launching():
    from systems_for_llms_b200.ops import build as builder
    from systems_for_llms_b200.ops import lib
    try:
        builder.build()
        handle = lib.lib()
    except Exception as error:
        pytest.skip(f"kernel library unavailable: {error}")
    assert handle.sfl_linear_ce_part_bytes(0, 5) == -1
    assert handle.sfl_linear_ce_part_bytes(3, 257) == 3 * (4 * 8 + 4)
    assert handle.sfl_linear_ce_part_bytes(2 ** 20, 2 ** 17) > 2 ** 32        # beyond 32 bits
    good = dict(hidden=256, ld_hidden=64, weight=512, ld_weight=64, targets=256, rows=4, dim=64,
                vocab=100, lse2=256)
    fwd = lambda part=10 ** 6, totals=256, **kw: handle.sfl_linear_ce_fwd(
        ctypes.byref(LinearCe(**{**good, **kw})), 256, part, 256, 1, totals, 256, None)
    for kw in (dict(rows=0), dict(dim=60), dict(vocab=0), dict(hidden=8), dict(ld_weight=65),
               dict(ld_hidden=56), dict(targets=None), dict(lse2=None), dict(part=16),
               dict(totals=None)):
        assert fwd(**kw) == -2, kw
    spec = dict(dlogits=256, dh=256, ld_dh=64, dw=256, ld_dw=64, dw_kind=0, piece=256)
    bwd = lambda kw: handle.sfl_linear_ce_bwd(
        ctypes.byref(LinearCe(**good)), ctypes.byref(LinearCeGrad(**{**spec, **kw})), None)
    for kw in (dict(piece=0), dict(piece=300), dict(dw_kind=3), dict(dw=None), dict(ld_dh=60),
               dict(dlogits=8)):
        assert bwd(kw) == -2, kw
    small = dict(good, vocab=300)                                   # two pieces, no place for their sum
    assert handle.sfl_linear_ce_bwd(ctypes.byref(LinearCe(**small)),
                                    ctypes.byref(LinearCeGrad(**spec)), None) == -2


def test_a_gradient_left_out_is_said_twice():
    from systems_for_llms_b200.ops import build as builder
    from systems_for_llms_b200.ops import lib
    try:
        builder.build()
        handle = lib.lib()
    except Exception as error:
        pytest.skip(f"kernel library unavailable: {error}")
    args = LinearCe(hidden=256, ld_hidden=64, weight=512, ld_weight=64, targets=256, rows=4, dim=64,
                    vocab=100, lse2=256)
    spec = dict(dlogits=256, dh=256, ld_dh=64, dw=256, ld_dw=64, dw_kind=0, piece=256)
    for kw in (dict(dw_kind=3), dict(dw=None, dw_kind=1), dict(dh=None, dw=None, dw_kind=3),
               dict(dw_kind=4, dw=None)):
        grads = LinearCeGrad(**{**spec, **kw})
        assert handle.sfl_linear_ce_bwd(ctypes.byref(args), ctypes.byref(grads), None) == -2, kw


def test_records_match_the_compiled_library():
    from systems_for_llms_b200.ops import build as builder
    from systems_for_llms_b200.ops import lib
    from systems_for_llms_b200.ops.newton_schulz import NewtonSchulz
    from systems_for_llms_b200.ops.rotary import RotaryTable, RotaryTensor
    try:
        builder.build()
        call = lib.lib()._handle.sfl_operator_struct_sizes
    except Exception as error:
        pytest.skip(f"kernel library unavailable: {error}")
    call.argtypes, call.restype = [ctypes.POINTER(ctypes.c_int), ctypes.c_int], ctypes.c_int
    sizes = (ctypes.c_int * 8)()
    mirrors = [RotaryTensor, RotaryTable, LinearCe, LinearCeGrad, NewtonSchulz]
    assert call(sizes, 8) == len(mirrors)
    assert [ctypes.sizeof(m) for m in mirrors] == list(sizes)[:len(mirrors)]
