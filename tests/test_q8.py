"""Refusals of the 8-bit operators: by the wrappers on host tensors and by the C
entry points on arguments that are checked before any device call."""

from __future__ import annotations

import pytest
import torch

from stateful_llm_compiler_hip import _native, backends

P = 0x1000  # 4 KiB-aligned, never dereferenced on these paths
F32, F16, BF16, I32 = 0, 1, 2, 3


def test_wrappers_refuse_host_tensors():
    x, w = torch.zeros(2, 8), torch.ones(8)
    codes, scales = torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)
    for call in (
        lambda: backends.hip_quantize_q8(x),
        lambda: backends.hip_rms_norm_q8(x, w, epsilon=1e-6),
        lambda: backends.hip_add_rms_norm_q8(x, x, w, epsilon=1e-6),
        lambda: backends.hip_swiglu_q8(x, x),
        lambda: backends.hip_linear_q8(codes, scales, codes, scales),
    ):
        with pytest.raises(ValueError, match="on the GPU"):
            call()


def quantize(x=P, codes=P, scales=P, dtype=BF16, rows=2, hidden=8, rs=8):
    return _native.library().slc_hip_quantize_q8(x, codes, scales, dtype, rows, hidden, rs, None)


def norm(x=P, residual=P, w=P, summed=P, codes=P, scales=P, dtype=BF16, rows=2, hidden=8, eps=1e-6):
    return _native.library().slc_hip_rms_norm_q8(x, residual, w, summed, codes, scales, dtype, rows, hidden,
                                                 hidden, hidden, eps, None)


def swiglu(gate=P, up=P, codes=P, scales=P, dtype=BF16, rows=2, hidden=8):
    return _native.library().slc_hip_swiglu_q8(gate, up, codes, scales, dtype, rows, hidden, hidden, hidden, None)


def linear(x=P, sx=P, w=P, sw=P, bias=None, y=P, dtype=BF16, rows=2, n=16, k=64, x_rs=64, y_rs=16):
    return _native.library().slc_hip_linear_q8(x, sx, w, sw, bias, y, dtype, rows, n, k, x_rs, y_rs, None)


@pytest.mark.parametrize("call", [quantize, norm, swiglu])
def test_row_entry_points_refuse(call):
    for bad in ({"dtype": I32}, {"dtype": 99}, {"rows": -1}, {"rows": 2**31}, {"hidden": 0}, {"hidden": -8},
                {"hidden": 131072}, {"codes": None}, {"scales": None}, {"scales": P + 2}):
        assert call(**bad) == -1, bad
    assert call(rows=0) == 0  # nothing to do, nothing launched
    assert call(rows=0, codes=None) == 0


def test_row_entry_points_refuse_their_own_operands():
    assert quantize(x=None) == -1 and quantize(x=P + 1) == -1 and quantize(x=P + 2, dtype=F32) == -1
    assert norm(x=None) == -1 and norm(w=None) == -1 and norm(w=P + 1) == -1
    assert norm(residual=None) == -1 and norm(summed=None) == -1  # one without the other
    assert all(norm(eps=eps) == -1 for eps in (-1e-6, float("nan"), float("inf")))
    assert norm(residual=P + 1) == -1 and norm(summed=P + 1) == -1
    assert swiglu(gate=None) == -1 and swiglu(up=None) == -1 and swiglu(up=P + 1) == -1
    assert b"slc_hip_swiglu_q8" in _native.library().slc_hip_last_error()


def test_linear_entry_point_refuses():
    for bad in ({"dtype": I32}, {"rows": -1}, {"rows": 2**31}, {"n": 0}, {"n": 2**31}, {"k": 0}, {"k": 131072},
                {"x": None}, {"sx": None}, {"w": None}, {"sw": None}, {"y": None}, {"sx": P + 2}, {"sw": P + 1},
                {"y": P + 1}, {"bias": P + 1}, {"y": P + 2, "dtype": F32}, {"x_rs": -64}, {"y_rs": 15}, {"y_rs": -16}):
        assert linear(**bad) == -1, bad
    assert linear(rows=0) == 0
