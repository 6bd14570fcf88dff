"""Residual addition and root-mean-square norm: the step in front of the expert layer.

No counterpart in the reference, which starts at the layer's hidden states.  One kernel adds
the layer input to the residual stream, stores the new residual and writes the normalised rows
either in BF16 (what :func:`b200moe.b300_moe_forward` and :func:`b200moe.b300_moe_layer` take)
or as E4M3 codes with one FP32 scale per row, the format of :func:`b200moe.quantize_rows_fp8`.
"""

from __future__ import annotations

import math

import torch

from . import _lib

MAX_NORM_HIDDEN = 32768
_FLOATS = (torch.bfloat16, torch.float32)


def _check_buffer(name: str, t: object, shape, dtype: torch.dtype, device: torch.device) -> None:
    """A caller's output tensor."""

    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor or None")
    if t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous() \
            or t.requires_grad:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on "
                         f"{device} that does not require grad")


def _check(hidden_states, residual, weight, eps, step: int) -> None:
    for name, t in (("hidden_states", hidden_states), ("weight", weight)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    if residual is not None and not isinstance(residual, torch.Tensor):
        raise TypeError("residual must be a torch.Tensor or None")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)):
        raise TypeError("eps must be a number")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError("eps must be finite and not negative")
    if hidden_states.ndim < 1:
        raise ValueError("hidden_states must have shape [..., hidden_size]")
    hidden = hidden_states.shape[-1]
    if weight.shape != (hidden,):
        raise ValueError("weight must have shape [hidden_size]")
    if residual is not None and residual.shape != hidden_states.shape:
        raise ValueError("residual and hidden_states must have the same shape")
    if hidden_states.dtype is not torch.bfloat16:
        raise TypeError("hidden_states must have dtype torch.bfloat16")
    if weight.dtype not in _FLOATS or (residual is not None and residual.dtype not in _FLOATS):
        raise TypeError("residual and weight must have dtype torch.bfloat16 or torch.float32")
    tensors = (hidden_states, weight) if residual is None else (hidden_states, weight, residual)
    device = hidden_states.device
    if any(t.device != device for t in tensors):
        raise ValueError("all inputs must be on the same device")
    if any(not t.is_contiguous() for t in tensors):
        raise ValueError("all inputs must be contiguous")
    if any(t.requires_grad for t in tensors):
        raise ValueError("the native norm does not support autograd")
    if hidden < 1 or hidden % step or hidden > MAX_NORM_HIDDEN:
        raise ValueError(f"hidden_size must be a multiple of {step} and at most {MAX_NORM_HIDDEN}")
    if hidden_states.numel() // hidden > 0x7FFFFFFF:
        raise ValueError("the native norm supports at most 2**31 - 1 rows")
    if device.type != "cuda":
        raise ValueError("the native norm requires CUDA tensors")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    a0, b0 = a.data_ptr(), b.data_ptr()
    return a0 < b0 + b.numel() * b.element_size() and b0 < a0 + a.numel() * a.element_size()


def _check_aliases(hidden_states, residual, weight, outputs) -> None:
    """An output may be the hidden states or the residual themselves (in-place use); any other
    overlap would let one row's stores reach another row's loads."""

    for i, out in enumerate(outputs):
        for other in outputs[i + 1:]:
            if _overlap(out, other):
                raise ValueError("the output tensors must not overlap")
        if _overlap(out, weight):
            raise ValueError("the output tensors must not overlap the weight")
        for t in (hidden_states,) if residual is None else (hidden_states, residual):
            if _overlap(out, t) and not (out.data_ptr() == t.data_ptr() and out.shape == t.shape
                                         and out.dtype == t.dtype):
                raise ValueError("an output may only overlap an input by being that tensor")


def _launch(hidden_states, residual, weight, eps, out, codes, scale, residual_out) -> None:
    rows = hidden_states.numel() // hidden_states.shape[-1]
    if rows == 0:
        return
    device = hidden_states.device
    index = device.index
    args = (
        hidden_states.data_ptr(),
        None if residual is None else residual.data_ptr(),
        residual is not None and residual.dtype is torch.float32,
        weight.data_ptr(), weight.dtype is torch.float32, rows, hidden_states.shape[-1], eps,
        None if out is None else out.data_ptr(), None if codes is None else codes.data_ptr(),
        None if scale is None else scale.data_ptr(),
        None if residual is None else residual_out.data_ptr(),
        torch._C._cuda_getCurrentRawStream(index),
    )
    fn = _lib.load().b200moe_add_rms_norm
    if torch.cuda.current_device() == index:
        code = fn(*args)
    else:
        with torch.cuda.device(device):
            code = fn(*args)
    if code:
        _lib.check(code, "b200moe_add_rms_norm")


def _residual_buffer(hidden_states, residual, residual_out):
    if residual is None:
        if residual_out is not None:
            raise ValueError("residual_out needs a residual")
        return None
    if residual_out is None:
        return torch.empty_like(residual)
    _check_buffer("residual_out", residual_out, residual.shape, residual.dtype, residual.device)
    return residual_out


def add_rms_norm(
    hidden_states: torch.Tensor,
    residual: torch.Tensor | None,
    weight: torch.Tensor,
    *,
    eps: float = 1e-6,
    out: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(normed, new_residual)`` of ``s = hidden_states + residual``:
    ``normed = s / sqrt(mean(s**2) + eps) * weight`` in BF16, ``new_residual = s`` in the
    residual's dtype.

    ``hidden_states`` [..., H] BF16, ``residual`` of the same shape in BF16 or FP32, ``weight``
    [H] in BF16 or FP32; contiguous, on one CUDA device, H a multiple of 8 and at most 32768.
    The sum is normalised in FP32, before the rounding that stores it.  Without a residual
    (``None``, the first norm of a model) ``hidden_states`` itself is normalised and returned
    as the new residual.

    ``out`` and ``residual_out`` name where the results go instead of fresh tensors.  Each may
    be an input of its own dtype (``residual_out=residual`` updates the stream in place); no
    other overlap is allowed.
    """

    _check(hidden_states, residual, weight, eps, 8)
    if out is None:
        out = torch.empty_like(hidden_states)
    else:
        _check_buffer("out", out, hidden_states.shape, torch.bfloat16, hidden_states.device)
    residual_out = _residual_buffer(hidden_states, residual, residual_out)
    _check_aliases(hidden_states, residual, weight,
                   (out,) if residual is None else (out, residual_out))
    _launch(hidden_states, residual, weight, eps, out, None, None, residual_out)
    return out, hidden_states if residual is None else residual_out


def add_rms_norm_fp8(
    hidden_states: torch.Tensor,
    residual: torch.Tensor | None,
    weight: torch.Tensor,
    *,
    eps: float = 1e-6,
    out: torch.Tensor | None = None,
    scale_out: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(codes, scale, new_residual)``: :func:`add_rms_norm` with the normalised rows as E4M3.

    ``codes`` uint8 [..., H] and ``scale`` FP32 [...] follow :func:`quantize_rows_fp8`:
    ``scale = max|row| / 448`` (1 for a row of zeros), ``code = E4M3(value / scale)`` rounded to
    nearest even, taken from the FP32 values, not from their BF16 rounding.  H must be a
    multiple of 16.
    """

    _check(hidden_states, residual, weight, eps, 16)
    if out is None:
        out = torch.empty(hidden_states.shape, dtype=torch.uint8, device=hidden_states.device)
    else:
        _check_buffer("out", out, hidden_states.shape, torch.uint8, hidden_states.device)
    if scale_out is None:
        scale_out = torch.empty(hidden_states.shape[:-1], dtype=torch.float32,
                                device=hidden_states.device)
    else:
        _check_buffer("scale_out", scale_out, hidden_states.shape[:-1], torch.float32,
                      hidden_states.device)
    residual_out = _residual_buffer(hidden_states, residual, residual_out)
    _check_aliases(hidden_states, residual, weight,
                   (out, scale_out) if residual is None else (out, scale_out, residual_out))
    _launch(hidden_states, residual, weight, eps, None, out, scale_out, residual_out)
    return out, scale_out, hidden_states if residual is None else residual_out
