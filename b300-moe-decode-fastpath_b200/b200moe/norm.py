"""Residual addition and root-mean-square norm: the step in front of the expert layer.

No counterpart in the reference, which starts at the layer's hidden states.  One kernel adds
the layer input to the residual stream, stores the new residual and writes the normalised rows
either in BF16 (what every layer of this package takes) or, for products of the caller's own, as
E4M3 codes with one FP32 scale per row, the format of :func:`b200moe.quantize_rows_fp8`.
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
    if t.shape != shape or t.dtype is not dtype or t.device != device or not t.is_contiguous() \
            or t.requires_grad:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on "
                         f"{device} that does not require grad")


def _check(x, residual, weight, eps, step: int) -> int:
    """Checks of the inputs; the number of rows.  Written out flat: a decode step calls this once
    per layer, and its host time is of the order of the kernel's."""

    if not isinstance(x, torch.Tensor):
        raise TypeError("hidden_states must be a torch.Tensor")
    if not isinstance(weight, torch.Tensor):
        raise TypeError("weight must be a torch.Tensor")
    if residual is not None and not isinstance(residual, torch.Tensor):
        raise TypeError("residual must be a torch.Tensor or None")
    if type(eps) is not float and (isinstance(eps, bool) or not isinstance(eps, (int, float))):
        raise TypeError("eps must be a number")
    if not 0.0 <= eps < math.inf:
        raise ValueError("eps must be finite and not negative")
    shape = x.shape
    if len(shape) < 1:
        raise ValueError("hidden_states must have shape [..., hidden_size]")
    hidden = shape[-1]
    if weight.shape != (hidden,):
        raise ValueError("weight must have shape [hidden_size]")
    if residual is not None and residual.shape != shape:
        raise ValueError("residual and hidden_states must have the same shape")
    if x.dtype is not torch.bfloat16:
        raise TypeError("hidden_states must have dtype torch.bfloat16")
    if weight.dtype not in _FLOATS or (residual is not None and residual.dtype not in _FLOATS):
        raise TypeError("residual and weight must have dtype torch.bfloat16 or torch.float32")
    device = x.device
    if weight.device != device or (residual is not None and residual.device != device):
        raise ValueError("all inputs must be on the same device")
    if not x.is_contiguous() or not weight.is_contiguous() or \
            (residual is not None and not residual.is_contiguous()):
        raise ValueError("all inputs must be contiguous")
    if x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad):
        raise ValueError("the native norm does not support autograd")
    if hidden < 1 or hidden % step or hidden > MAX_NORM_HIDDEN:
        raise ValueError(f"hidden_size must be a multiple of {step} and at most {MAX_NORM_HIDDEN}")
    rows = x.numel() // hidden
    if rows > 0x7FFFFFFF:
        raise ValueError("the native norm supports at most 2**31 - 1 rows")
    if device.type != "cuda":
        raise ValueError("the native norm requires CUDA tensors")
    return rows


def _launch(x, residual, weight, eps, rows: int, out, scale, residual_out) -> None:
    """Checks what the results may overlap, and enqueues the kernel.  An output may be the hidden
    states or the residual themselves (in-place use, same dtype); any other overlap would let one
    row's stores reach another row's loads."""

    if rows == 0:
        return
    hidden = x.shape[-1]
    count = rows * hidden
    x_at, w_at, out_at = x.data_ptr(), weight.data_ptr(), out.data_ptr()
    w_f32 = weight.dtype is torch.float32
    out_size = 2 if scale is None else 1
    x_end, out_end = x_at + 2 * count, out_at + out_size * count
    w_end = w_at + (4 if w_f32 else 2) * hidden
    r_at = kept_at = scale_at = None
    r_f32 = False
    r_size, r_end, kept_end = 0, 0, 0
    if residual is not None:
        r_f32 = residual.dtype is torch.float32
        r_size = 4 if r_f32 else 2
        r_at, kept_at = residual.data_ptr(), residual_out.data_ptr()
        r_end, kept_end = r_at + r_size * count, kept_at + r_size * count
    elif scale is None and out_at == x_at:
        raise ValueError("without a residual, out must not be hidden_states: they are returned as "
                         "the new residual")
    # (start, end, element size; 0: never the same as an input) of every result
    written = [(out_at, out_end, out_size)]
    if residual is not None:
        if out_at < kept_end and kept_at < out_end:
            raise ValueError("the output tensors must not overlap")
        written.append((kept_at, kept_end, r_size))
    if scale is not None:
        scale_at = scale.data_ptr()
        scale_end = scale_at + 4 * rows
        if (scale_at < out_end and out_at < scale_end) or \
                (residual is not None and scale_at < kept_end and kept_at < scale_end):
            raise ValueError("the output tensors must not overlap")
        written.append((scale_at, scale_end, 0))
    for start, end, size in written:
        if start < w_end and w_at < end:
            raise ValueError("the output tensors must not overlap the weight")
        if (start < x_end and x_at < end and (start != x_at or size != 2)) or \
                (start < r_end and residual is not None and r_at < end
                 and (start != r_at or size != r_size)):
            raise ValueError("an output may only overlap an input by being that tensor")
    index = x.device.index
    args = (x_at, r_at, r_f32, w_at, w_f32, rows, hidden, eps, out_at if scale is None else None,
            None if scale is None else out_at, scale_at, kept_at,
            torch._C._cuda_getCurrentRawStream(index))
    fn = _lib.load().b200moe_add_rms_norm
    if torch._C._cuda_getDevice() == index:
        code = fn(*args)
    else:
        with torch.cuda.device(index):
            code = fn(*args)
    if code:
        _lib.check(code, "b200moe_add_rms_norm")


def _residual_buffer(residual, residual_out):
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
    The sum is normalised in FP32, before the rounding that stores it; a row's result depends on
    that row alone.  Squares and products with the weight are FP32 too: a row whose mean square
    or products leave its range (elements beyond about 1e18) has no finite or meaningful result,
    as in any FP32 norm.  Without a residual
    (``None``, the first norm of a model) ``hidden_states`` itself is normalised and returned
    as the new residual.

    ``out`` and ``residual_out`` name where the results go instead of fresh tensors.  Each may
    be an input of its own dtype (``residual_out=residual`` updates the stream in place); no
    other overlap is allowed, nor is ``out=hidden_states`` without a residual, since those are
    then the new residual.
    """

    rows = _check(hidden_states, residual, weight, eps, 8)
    if out is None:
        out = torch.empty_like(hidden_states)
    else:
        _check_buffer("out", out, hidden_states.shape, torch.bfloat16, hidden_states.device)
    residual_out = _residual_buffer(residual, residual_out)
    _launch(hidden_states, residual, weight, eps, rows, out, None, residual_out)
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
    multiple of 16.  The rows are for products of the caller's own that take E4M3 operands: the
    layers of this package take BF16 rows, those of :func:`add_rms_norm`.
    """

    rows = _check(hidden_states, residual, weight, eps, 16)
    device = hidden_states.device
    if out is None:
        out = torch.empty(hidden_states.shape, dtype=torch.uint8, device=device)
    else:
        _check_buffer("out", out, hidden_states.shape, torch.uint8, device)
    if scale_out is None:
        scale_out = torch.empty(hidden_states.shape[:-1], dtype=torch.float32, device=device)
    else:
        _check_buffer("scale_out", scale_out, hidden_states.shape[:-1], torch.float32, device)
    residual_out = _residual_buffer(residual, residual_out)
    _launch(hidden_states, residual, weight, eps, rows, out, scale_out, residual_out)
    return out, scale_out, hidden_states if residual is None else residual_out
