"""Sampling of one token per row of logits: the step behind the model's head.

No counterpart in the reference.  Like :func:`b200moe.topk_routing` it selects from logits and
normalises what it selected; here over a whole vocabulary, with temperature, top-k, top-p and
min-p, and a draw from random numbers that the caller supplies.
"""

from __future__ import annotations

import torch

from . import _lib

MAX_SAMPLE_ROWS = 1 << 20
MAX_SAMPLE_VOCAB = 1 << 18


def _setting(name: str, value, rows: int, device, low: float, high: float):
    """``(device pointer or None, value)`` of one FP32 setting."""

    if isinstance(value, torch.Tensor):
        if value.dtype is not torch.float32:
            raise TypeError(f"{name} must be a number or a float32 tensor")
        if value.shape != (rows,) or not value.is_contiguous() or value.device != device:
            raise ValueError(f"{name} must be a contiguous [{rows}] tensor on the logits' device")
        return value.data_ptr(), 0.0
    if isinstance(value, bool) or not isinstance(value, (int, float)):
        raise TypeError(f"{name} must be a number or a float32 tensor")
    if not low <= value <= high:  # NaN fails too
        raise ValueError(f"{name} must be between {low} and {high}, got {value}")
    return None, value


def sample_tokens(
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    *,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
    return_logprobs: bool = False,
    out: torch.Tensor | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Ids [T] int64 of one token per row of ``logits`` [T,V] (BF16 or FP32), drawn with
    ``uniforms`` [T] FP32 in [0, 1).

    With ``w = exp((logit - max) / temperature)`` and tokens ordered by descending logit (equal
    ones by ascending id): ``min_p`` drops tokens with ``w < min_p``, ``top_k`` keeps the first k
    of the order, ``top_p`` of those the shortest run of the order that holds at least ``top_p``
    of their weight.  The result is the first token, in id order, at which the running sum of
    the kept weights exceeds ``uniform * sum``.  Weights are summed exactly, so a row's
    token depends on that row alone.

    Each setting is a number for all rows or a [T] tensor on the logits' device (FP32;
    ``top_k`` int32).  Off: ``top_k=0``, ``top_p=1``, ``min_p=0``.  ``temperature=0`` takes the
    largest logit.  Tensor values are not checked: a temperature that is not above 0 takes the
    largest logit and an infinite one weighs all finite logits alike (beside an infinite logit
    they weigh nothing), ``top_k <= 0`` is off, ``top_p >= 1`` or NaN is off and ``top_p <= 0`` keeps
    one token, ``min_p`` not above 0 is off and above 1 counts as 1; a uniform of 1 or more draws
    the last kept token.  Numbers are held in FP32.

    NaN logits count as ``-inf`` and tokens at ``-inf`` are never drawn; a row of nothing else
    gives -1.  ``return_logprobs=True`` also returns, in FP32, the logarithm of the probability
    with which the token was drawn (0 for the largest logit at ``temperature=0``, ``-inf`` with
    -1).  Rows may be further apart than V (a padded vocabulary: ``logits[:, :V]``); V is at most
    262144.  ``out`` names where the ids go; it must not overlap an input.
    """

    if not isinstance(logits, torch.Tensor) or not isinstance(uniforms, torch.Tensor):
        raise TypeError("logits and uniforms must be torch.Tensors")
    if not isinstance(return_logprobs, bool):
        raise TypeError("return_logprobs must be a bool")
    if logits.ndim != 2:
        raise ValueError(f"logits must have shape [num_rows, vocab], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if rows < 1 or vocab < 1:
        raise ValueError("logits must contain at least one row and token")
    if rows > MAX_SAMPLE_ROWS or vocab > MAX_SAMPLE_VOCAB:
        raise ValueError(f"the native sampler supports at most {MAX_SAMPLE_ROWS} rows and "
                         f"{MAX_SAMPLE_VOCAB} tokens")
    is_f32 = logits.dtype is torch.float32
    if not is_f32 and logits.dtype is not torch.bfloat16:
        raise TypeError("the native sampler supports float32 and bfloat16 logits")
    device = logits.device
    stride = logits.stride(0) if rows > 1 else vocab
    if (vocab > 1 and logits.stride(1) != 1) or stride < vocab:
        raise ValueError("each row of logits must be contiguous and rows may not overlap")
    if uniforms.dtype is not torch.float32:
        raise TypeError("uniforms must have dtype torch.float32")
    if uniforms.shape != (rows,) or not uniforms.is_contiguous() or uniforms.device != device:
        raise ValueError(f"uniforms must be a contiguous [{rows}] tensor on the logits' device")
    if logits.requires_grad or uniforms.requires_grad:
        raise ValueError("the native sampler does not support autograd")
    heat, heat_v = _setting("temperature", temperature, rows, device, 0.0, 3e38)
    p, p_v = _setting("top_p", top_p, rows, device, 0.0, 1.0)
    low, low_v = _setting("min_p", min_p, rows, device, 0.0, 1.0)
    if isinstance(top_k, torch.Tensor):
        if top_k.dtype is not torch.int32:
            raise TypeError("top_k must be an integer or an int32 tensor")
        if top_k.shape != (rows,) or not top_k.is_contiguous() or top_k.device != device:
            raise ValueError(f"top_k must be a contiguous [{rows}] tensor on the logits' device")
        k, k_v = top_k.data_ptr(), 0
    else:
        if isinstance(top_k, bool) or not isinstance(top_k, int):
            raise TypeError("top_k must be an integer or an int32 tensor")
        if top_k < 0:
            raise ValueError(f"top_k must not be negative, got {top_k}")
        k, k_v = None, min(top_k, MAX_SAMPLE_VOCAB)
    if out is not None:
        if not isinstance(out, torch.Tensor):
            raise TypeError("out must be a torch.Tensor or None")
        if out.shape != (rows,) or out.dtype is not torch.int64 or out.device != device or \
                not out.is_contiguous():
            raise ValueError(f"out must be a contiguous int64 [{rows}] tensor on the logits' device")
        # a row's id is stored while other rows are still being read
        start, end = out.data_ptr(), out.data_ptr() + 8 * rows
        if any(at is not None and start < at + size and at < end for at, size in
               ((logits.data_ptr(), ((rows - 1) * stride + vocab) * logits.element_size()),
                (uniforms.data_ptr(), 4 * rows), (heat, 4 * rows), (k, 4 * rows), (p, 4 * rows),
                (low, 4 * rows))):
            raise ValueError("out must not overlap an input")
    if device.type != "cuda":
        raise ValueError("the native sampler requires CUDA tensors")
    ids = out if out is not None else torch.empty(rows, dtype=torch.int64, device=device)
    logprobs = torch.empty(rows, device=device) if return_logprobs else None
    args = (logits.data_ptr(), is_f32, stride, rows, vocab, uniforms.data_ptr(), heat, heat_v, k,
            k_v, p, p_v, low, low_v, ids.data_ptr(),
            None if logprobs is None else logprobs.data_ptr(),
            torch._C._cuda_getCurrentRawStream(device.index))
    fn = _lib.load().b200moe_sample
    if torch._C._cuda_getDevice() == device.index:
        code = fn(*args)
    else:
        with torch.cuda.device(device):
            code = fn(*args)
    if code:
        _lib.check(code, "b200moe_sample")
    return (ids, logprobs) if return_logprobs else ids
