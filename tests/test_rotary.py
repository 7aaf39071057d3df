"""Rotary tables and the refusals of the rotary operators (CPU)."""

import math

import pytest
import torch

from systems_for_llms_b200.ops.rotary import (RotaryScaling, _check_heads, _check_out, _check_table,
                                              qk_norm_rotary, rotary, rotary_frequencies,
                                              rotary_tables)


def test_tables_without_scaling_match_the_model_module():
    from systems_for_llms_b200.models.attention import RotaryPositionalEmbedding
    cos, sin = rotary_tables(64, 1024, 10000.0)
    module = RotaryPositionalEmbedding(10000.0, 64, 1024)
    # the module's fp32 angles are off by up to position * 2^-23 (frequency and product)
    bound = torch.arange(1024)[:, None] * 2.0 ** -22 + 2.0 ** -23
    assert ((cos - module.cos).abs() <= bound).all() and ((sin - module.sin).abs() <= bound).all()
    assert cos.dtype == torch.float32 and cos.shape == (1024, 32)


@pytest.mark.parametrize("position", [0, 1, 4095, 131071])
def test_far_positions_are_exact(position):
    cos, sin = rotary_tables(8, 131072, 500.0)
    for i in range(4):
        angle = position * 500.0 ** (-2 * i / 8)
        assert abs(cos[position, i].item() - math.cos(angle)) < 2.0 ** -24 + 1e-9
        assert abs(sin[position, i].item() - math.sin(angle)) < 2.0 ** -24 + 1e-9


def test_scalings():
    base = rotary_frequencies(64)
    assert torch.equal(rotary_frequencies(64, scaling=RotaryScaling("linear", 4.0)), base / 4)
    ntk = rotary_frequencies(64, scaling=RotaryScaling("ntk", 4.0))
    assert ntk[0] == 1.0 and ntk[-1].item() == pytest.approx(base[-1].item() / 4, rel=1e-12)
    parts = rotary_frequencies(64, scaling=RotaryScaling("parts", 8.0, trained=4096))
    turns = 4096 * base / (2 * math.pi)
    assert torch.equal(parts[turns >= 4], base[turns >= 4])
    assert torch.allclose(parts[turns <= 1], base[turns <= 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 4)
    assert between.any() and ((parts < base) & (parts > base / 8))[between].all()
    assert (parts.diff() < 0).all()
    same = rotary_frequencies(64, scaling=RotaryScaling("parts", 1.0, trained=4096))
    assert torch.allclose(same, base, rtol=1e-15)


@pytest.mark.parametrize("arguments", [
    dict(kind="yarn", factor=2.0), dict(kind="linear", factor=0.5), dict(kind="ntk", factor=math.inf),
    dict(kind="parts", factor=2.0), dict(kind="parts", factor=2.0, trained=16, slow_turns=4.0),
])
def test_bad_scalings_are_refused(arguments):
    with pytest.raises(ValueError):
        RotaryScaling(**arguments)


@pytest.mark.parametrize("arguments", [(0, 4), (7, 4), (-2, 4), (8, 0), (8, 2.0), (8, 4, -1.0),
                                       (8, 4, math.nan), (2, 4, 10.0, RotaryScaling("ntk", 2.0))])
def test_bad_tables_are_refused(arguments):
    with pytest.raises(ValueError):
        rotary_tables(*arguments)


def test_bad_calls_are_refused():
    x = torch.zeros(2, 3, 4, 8)
    cos, sin = rotary_tables(8, 16)
    w = torch.ones(8)
    with pytest.raises(ValueError, match="CUDA"):
        rotary(x, cos, sin)
    with pytest.raises(ValueError, match="layout"):
        rotary(x, cos, sin, layout="quarter")
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rotary(x, x, w, w, cos, sin)
    with pytest.raises(ValueError, match="head_dim"):
        _check_heads(x[0], "x")
    with pytest.raises(TypeError):
        _check_heads(x.double(), "x")
    for t in (cos[:, :0], cos.double(), cos.t(), cos[None]):
        with pytest.raises(ValueError):
            _check_table(x, t, sin, None)
    with pytest.raises(ValueError, match="more lanes"):
        _check_table(x, *rotary_tables(10, 16), None)
    with pytest.raises(ValueError, match="more tokens"):
        _check_table(x, cos[:3], sin[:3], None)
    for positions in (torch.arange(4, dtype=torch.int32), torch.arange(5), torch.zeros(3, 4).long()):
        with pytest.raises(ValueError, match="positions"):
            _check_table(x, cos, sin, positions)
    _check_table(x, cos, sin, torch.arange(4))
    _check_table(x, cos, sin, torch.zeros(2, 4).long())
    for out in (x[:1], x.half(), x.new_zeros(1, 3, 4, 8).expand(2, 3, 4, 8),
                x.new_zeros(2, 3, 8, 4).transpose(2, 3)):
        with pytest.raises(ValueError):
            _check_out(out, x, "out")


def test_entry_points_refuse_before_launching():
    import ctypes

    from systems_for_llms_b200.ops import build as builder
    from systems_for_llms_b200.ops import lib
    from systems_for_llms_b200.ops.rotary import RotaryTable, RotaryTensor
    try:
        builder.build()
        handle = lib.lib()
    except Exception as error:
        pytest.skip(f"kernel library unavailable: {error}")
    slots = (RotaryTensor * 2)()
    table = RotaryTable(cos=256, sin=512, rows=8, rotated=64)
    call = lambda count=1, dim=64, dtype=0: handle.sfl_rotary(
        slots, count, ctypes.byref(table), 1, 1, dim, 0.0, 0, 0, dtype, None)
    assert call() == -2                       # no tensors
    slots[0].x, slots[0].y, slots[0].heads = 256, 512, 1
    assert call(count=3) == -2 and call(dim=512) == -2 and call(dtype=3) == -2
    table.rotated = 63
    assert call() == -2
    table.rotated, table.rows = 64, 0
    assert call() == -2
    table.rows = 8
    assert call(dim=32) == -2                 # rotates more lanes than there are
    slots[1].x, slots[1].y, slots[1].heads, slots[1].weight = 256, 512, 1, 256
    assert call(count=2) == -2                # one side with a norm, one without
    bwd = lambda: handle.sfl_rotary_bwd(slots, 1, ctypes.byref(table), 1, 1, 64, 0.0, 0, 0, 256, 0,
                                        256, 256, None)
    assert bwd() == -2                        # nothing to differentiate without a norm


def test_packed_records_have_the_layout_of_the_structures():
    import ctypes

    from systems_for_llms_b200.ops import rotary as R
    assert R._TENSOR.size == ctypes.sizeof(R.RotaryTensor)
    assert R._TABLE.size == ctypes.sizeof(R.RotaryTable)
    x, y, dy = (torch.zeros(2, 3, 4, 8)[:, :, :, :n] for n in (8, 7, 6))
    w = torch.ones(8)
    record = R.RotaryTensor.from_buffer_copy(R._record(x, y, dy, w))
    assert (record.x, record.y, record.dy, record.weight) == (x.data_ptr(), y.data_ptr(),
                                                              dy.data_ptr(), w.data_ptr())
    assert (record.x_b, record.x_h, record.x_t) == x.stride()[:3] and record.heads == 3
    assert (record.y_b, record.y_h, record.y_t) == y.stride()[:3]
    assert (record.dy_b, record.dy_h, record.dy_t) == dy.stride()[:3]
    cos, sin = rotary_tables(8, 16)
    positions = torch.zeros(2, 6).long()[:, ::2]
    table = R.RotaryTable.from_buffer_copy(R._table(cos, sin, positions))
    assert (table.cos, table.sin, table.positions) == (cos.data_ptr(), sin.data_ptr(),
                                                       positions.data_ptr())
    assert (table.pos_b, table.pos_t, table.rows, table.rotated) == (6, 2, 16, 8)
    shared = R.RotaryTable.from_buffer_copy(R._table(cos, sin, positions[0]))
    assert (shared.pos_b, shared.pos_t) == (0, 2)
    assert R.RotaryTable.from_buffer_copy(R._table(cos, sin, None)).positions is None
