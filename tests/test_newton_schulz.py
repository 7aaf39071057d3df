"""Host side of the Newton-Schulz operator (CPU)."""

import ctypes
import math

import pytest
import torch

from systems_for_llms_b200.ops.newton_schulz import (NewtonSchulz, QUINTIC, _strided,
                                                     largest_singular_value, newton_schulz)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        newton_schulz(torch.zeros(4, 4))


def test_largest_singular_value_bounds_a_dense_scan():
    values = torch.linspace(0, 1, 20001, dtype=torch.float64)
    for coefficients in (QUINTIC, (1.875, -1.25, 0.375), (1.5, -0.5, 0.0), (2.0, -1.5, 0.5)):
        a, b, c = coefficients
        s, worst = values, 1.0
        for steps in range(1, 7):
            s = s * (a + s ** 2 * (b + c * s ** 2))
            worst = max(worst, s.abs().max().item())
            bound = largest_singular_value(coefficients, steps)
            assert worst <= bound + 1e-12
            assert bound < 1.3
    assert largest_singular_value((3.0, 0.0, 0.0), 5) > 2
    assert largest_singular_value((10.0, 5.0, 5.0), 64) == math.inf


def test_strided_views_are_not_copied():
    x = torch.zeros(3, 4, 10, 12)
    for view in (x, x[0], x[0, 0], x[:, 1:3, 2:8, 1:9], x[:1].expand(3, 4, 10, 12)):
        assert _strided(view).data_ptr() == view.data_ptr()
    assert _strided(x.mT).is_contiguous()
    assert _strided(torch.zeros(2, 3, 4, 5, 6)).shape == (24, 5, 6)


def test_entry_point_refuses_before_launching():
    from systems_for_llms_b200.ops import build as builder
    from systems_for_llms_b200.ops import lib
    try:
        builder.build()
        handle = lib.lib()
    except Exception as error:
        pytest.skip(f"kernel library unavailable: {error}")
    size = handle.sfl_newton_schulz_bytes(2, 10, 12)
    # two hi and a lo of pitch 16, two Gram matrices of pitch 16, norms
    assert size == 3 * 768 + 2 * 768 + 1024
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (70000, 1, 1)):
        assert handle.sfl_newton_schulz_bytes(*bad) == -1
    assert handle.sfl_newton_schulz_bytes(96, 4096, 16384) > 2 ** 32      # beyond 32 bits
    good = dict(update=256, stride0=120, row=12, inner=1, batch=2, m=10, n=12, steps=5, dtype=2,
                a=3.4, b=-4.7, c=2.0, eps=1e-7, out=256, work=256, work_bytes=size)
    for kw in (dict(batch=0), dict(batch=70000), dict(m=0), dict(n=0), dict(inner=0), dict(steps=0),
               dict(steps=65), dict(dtype=3), dict(update=None), dict(out=None), dict(work=None),
               dict(work=264), dict(work_bytes=size - 1)):
        args = NewtonSchulz(**{**good, **kw})
        assert handle.sfl_newton_schulz(ctypes.byref(args), None) == -2, kw
