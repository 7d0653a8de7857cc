"""8-bit linears: rows as int8 codes with an fp32 scale each, and their product.

A row ``y`` has ``scale = max|y| / 127`` and ``codes`` = the whole numbers nearest
to ``127 y / max|y|`` (ties to even), decided as 64-bit arithmetic does;
``code * scale`` is the value that a code stands for.  A row of zeros has scale 0; a
row with a NaN or an infinity (or whose scale fp32 cannot hold) has scale NaN, so
that whatever is computed from it is NaN too.

A layer's linears run on them as ``hip_add_rms_norm_q8`` -> ``hip_linear_q8``
(Q/K/V, or gate and up in one weight), ``hip_quantize_q8`` of the attention output
-> ``hip_linear_q8`` (O), ``hip_swiglu_q8`` -> ``hip_linear_q8`` (down).
``hip_quantize_q8`` of a weight ``[N, K]`` gives its codes and the scales of its
output channels.  The reference has no 8-bit path.

The operators stand beside ``hip_rms_norm``, ``hip_swiglu`` and ``hip_linear`` and
name their tensors alike, but compute other values than codes of those operators'
results: nothing is rounded to a 16-bit type before the codes are.  So the norm has no
``round_before_weight`` (the order of Qwen2's own norm, which rounds twice; a layer that
needs it runs ``hip_rms_norm`` and ``hip_quantize_q8``), its weight has the input's
dtype, and SwiGLU's silu is not rounded by itself.
"""

from __future__ import annotations

import torch

from .. import _native

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_MOST_EPSILON = torch.finfo(torch.float32).max

MAX_FEATURES = 131071  # SLC_Q8_MAX_K: sums of so many products of codes fit 32 bits


_CONTIGUOUS = torch.contiguous_format


# A tensor's device index, shape and strides are read once per call: each read takes
# the host 0.05 to 0.2 us of a call's 7.


def _check_rows(what: str, first: torch.Tensor, second: torch.Tensor | None = None) -> tuple[int, torch.Size]:
    """Device index and shape of float tensors on one GPU, of one shape and dtype,
    with a last axis to code."""

    index, shape = first.get_device(), first.shape
    if index < 0 or (second is not None and second.get_device() != index):
        raise ValueError(f"{what}: all tensors must be on the GPU, and on one")
    if second is not None and (second.shape != shape or second.dtype != first.dtype):
        raise ValueError(f"{what}: tensors need one shape and dtype")
    if first.dtype not in _FLOATS:
        raise ValueError(f"{what}: unsupported dtype {first.dtype}")
    if not shape or not 1 <= shape[-1] <= MAX_FEATURES:
        raise ValueError(f"{what}: the last axis must hold 1 to {MAX_FEATURES} values")
    return index, shape


def _rows(tensor: torch.Tensor, hidden: int) -> tuple[torch.Tensor, int]:
    """``tensor``, or a copy of it where its rows are no view of evenly strided
    ones, and their stride."""

    if tensor.is_contiguous():
        return tensor, hidden
    strides = tensor.stride()
    if strides[-1] == 1 or hidden == 1:
        if len(strides) == 2:
            return tensor, strides[0]
        try:
            return tensor, tensor.view(-1, hidden).stride(0)
        except RuntimeError:
            pass
    return tensor.contiguous(), hidden


def _codes_and_scales(tensor: torch.Tensor, shape: torch.Size) -> tuple[torch.Tensor, torch.Tensor]:
    return (torch.empty_like(tensor, dtype=torch.int8, memory_format=_CONTIGUOUS),
            tensor.new_empty(shape[:-1], dtype=torch.float32))


def _call(name: str, index: int, *arguments) -> None:
    """The entry point on GPU ``index``'s current stream, with that GPU current."""

    function = getattr(_native.library(), name)
    if index == torch._C._cuda_getDevice():
        status = function(*arguments, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = function(*arguments, torch._C._cuda_getCurrentRawStream(index))
    if status != 0:
        _native.check(status, name)


def hip_quantize_q8(tensor: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of ``tensor`` [..., K] along its last axis."""

    index, shape = _check_rows("HIP quantize q8", tensor)
    codes, scales = _codes_and_scales(tensor, shape)
    count = tensor.numel()
    if count:
        hidden = shape[-1]
        rows, stride = _rows(tensor, hidden)
        _call("slc_hip_quantize_q8", index, rows.data_ptr(), codes.data_ptr(), scales.data_ptr(),
              _native.dtype_tag(tensor.dtype), count // hidden, hidden, stride)
    return codes, scales


def _norm(what, tensor, residual, weight, epsilon):
    index, shape = _check_rows(what, tensor, residual)
    hidden = shape[-1]
    if weight.get_device() != index or weight.dtype != tensor.dtype:
        raise ValueError(f"{what}: the weight needs the input's dtype and device")
    if weight.shape != (hidden,):
        raise ValueError(f"{what}: weight must be [{hidden}], got {tuple(weight.shape)}")
    epsilon = float(epsilon)
    if not 0.0 <= epsilon <= _MOST_EPSILON:
        raise ValueError(f"{what}: epsilon must be finite and not negative, got {epsilon}")
    codes, scales = _codes_and_scales(tensor, shape)
    summed = None if residual is None else torch.empty_like(tensor, memory_format=_CONTIGUOUS)
    count = tensor.numel()
    if count:
        rows, stride = _rows(tensor, hidden)
        other, other_stride = (None, 0) if residual is None else _rows(residual, hidden)
        weight = weight.contiguous()
        _call("slc_hip_rms_norm_q8", index, rows.data_ptr(), None if other is None else other.data_ptr(),
              weight.data_ptr(), None if summed is None else summed.data_ptr(), codes.data_ptr(), scales.data_ptr(),
              _native.dtype_tag(tensor.dtype), count // hidden, hidden, stride, other_stride, epsilon)
    return summed, codes, scales


def hip_rms_norm_q8(
    tensor: torch.Tensor, weight: torch.Tensor, *, epsilon: float
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of ``tensor * rsqrt(mean(tensor^2) + epsilon) * weight``
    over the last axis; nothing is rounded before the codes are."""

    return _norm("HIP RMSNorm q8", tensor, None, weight, epsilon)[1:]


def hip_add_rms_norm_q8(
    tensor: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *, epsilon: float
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(summed, codes, scales)``: ``hip_add(tensor, residual)``, bit for bit (of two
    NaNs either may be the sum's), and ``hip_rms_norm_q8`` of it, in one pass."""

    return _norm("HIP add RMSNorm q8", tensor, residual, weight, epsilon)


def hip_swiglu_q8(gate: torch.Tensor, up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of ``silu(gate) * up``; nothing is rounded before the
    codes are.  ``gate`` and ``up`` may be the halves of a fused projection."""

    index, shape = _check_rows("HIP swiglu q8", gate, up)
    codes, scales = _codes_and_scales(gate, shape)
    count = gate.numel()
    if count:
        hidden = shape[-1]
        a, a_stride = _rows(gate, hidden)
        b, b_stride = _rows(up, hidden)
        _call("slc_hip_swiglu_q8", index, a.data_ptr(), b.data_ptr(), codes.data_ptr(), scales.data_ptr(),
              _native.dtype_tag(gate.dtype), count // hidden, hidden, a_stride, b_stride)
    return codes, scales


def hip_linear_q8(
    codes: torch.Tensor,
    scales: torch.Tensor,
    weight: torch.Tensor,
    weight_scales: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    output_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """``codes`` [..., K] times ``weight`` [N, K]^T, each output times its token's
    and its channel's scale (+ ``bias`` [N], of the output's dtype).

    ``codes`` and ``weight`` are int8 (-128 included), ``scales`` [...] and
    ``weight_scales`` [N] fp32.  The sum over K is exact; float(sum) * scale *
    weight scale + bias runs in fp32 in this order (the last product and the bias in
    one fma) and is rounded once to ``output_dtype``.
    """

    what = "HIP linear q8"
    index = codes.get_device()
    if index < 0 or scales.get_device() != index or weight.get_device() != index or (
        weight_scales.get_device() != index or (bias is not None and bias.get_device() != index)
    ):
        raise ValueError(f"{what}: all tensors must be on the GPU, and on one")
    if codes.dtype != torch.int8 or weight.dtype != torch.int8:
        raise ValueError(f"{what}: codes and weight must be int8")
    if scales.dtype != torch.float32 or weight_scales.dtype != torch.float32:
        raise ValueError(f"{what}: scales must be fp32")
    if output_dtype not in _FLOATS:
        raise ValueError(f"{what}: unsupported output dtype {output_dtype}")
    shape, weight_shape = codes.shape, weight.shape
    if not shape or len(weight_shape) != 2:
        raise ValueError(f"{what}: codes need at least one axis and the weight two")
    features, width = weight_shape
    if shape[-1] != width:
        raise ValueError(f"{what}: input K does not match weight K")
    if not 1 <= width <= MAX_FEATURES or features < 1:
        raise ValueError(f"{what}: K must be 1 to {MAX_FEATURES} and N at least 1")
    tokens = shape[:-1]
    if scales.shape != tokens or weight_scales.shape != (features,):
        raise ValueError(f"{what}: one scale per token and one per output channel are needed")
    if bias is not None and (bias.shape != (features,) or bias.dtype != output_dtype):
        raise ValueError(f"{what}: bias must be [{features}] of the output's dtype")
    if not (codes.is_contiguous() and scales.is_contiguous() and weight.is_contiguous()
            and weight_scales.is_contiguous()) or (bias is not None and not bias.is_contiguous()):
        raise ValueError(f"{what}: tensors must be contiguous")
    output = codes.new_empty((*tokens, features), dtype=output_dtype)
    count = codes.numel()
    if count:
        _call("slc_hip_linear_q8", index, codes.data_ptr(), scales.data_ptr(), weight.data_ptr(),
              weight_scales.data_ptr(), None if bias is None else bias.data_ptr(), output.data_ptr(),
              _native.dtype_tag(output_dtype), count // width, features, width, width, features)
    return output
