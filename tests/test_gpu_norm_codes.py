"""The residual norm's E4M3 rows beside the row quantiser, and its rows of tiny values.

Tolerances of ordinary rows as in test_gpu_norm.py.  Rows of tiny values: s is a multiple of 2^-133
(BF16 subnormals), its product with a weight of about 1 is rounded to a multiple of 2^-149, that is
by 2^-17 of it at most; with eps = 1e-6 the result is a thousand times larger and normal.  The
scale, y / 448, may be subnormal itself: at least 2^-132, so that its rounding is 2^-18 of it at
most.  2^-15 covers both and the ordinary 2^-18.
"""

from __future__ import annotations

import pytest
import torch

from b200moe import add_rms_norm_fp8, quantize_rows_fp8
from test_gpu_norm import _formula, _near

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -15


def _tiny_rows(device, weight):
    x = torch.zeros(9, 256, dtype=torch.bfloat16)
    x[0, 17] = 1e-40                                      # one subnormal among zeros
    x[1, :8] = torch.tensor([1, -2, 3, 5, -7, 100, 127, 0]).bfloat16() * 2.0 ** -133
    g = torch.Generator().manual_seed(2)
    for row, size in ((2, 1e-39), (3, 1e-38), (4, 1e-37), (5, 1e-36), (6, 1e-33)):
        x[row] = (torch.randn(256, generator=g) * size).bfloat16()
    x[7] = torch.randn(256, generator=g).bfloat16()       # an ordinary row between them
    w = (1 + 0.2 * torch.randn(256, generator=g)).abs().clamp(min=0.5).to(weight)
    return x.to(device), w.to(device)


@pytest.mark.parametrize("weight", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
def test_e4m3_rows_of_tiny_values(cuda_device, weight, residual) -> None:
    x, w = _tiny_rows(cuda_device, weight)
    r = None if residual is None else torch.zeros_like(x, dtype=residual)
    codes, scale, _ = add_rms_norm_fp8(x, r, w)
    _, y = _formula(x, r, w, 1e-6)
    want = y.abs().amax(-1) / 448.0
    assert bool((codes[8] == 0).all()) and float(scale[8]) == 1.0
    want[8] = 1.0
    _near(scale, want, TINY)
    values = codes.view(torch.float8_e4m3fn).float()
    assert bool(values.isfinite().all()) and bool((values[x == 0] == 0).all())
    _near(values, y / want[:, None], 2.0 ** -4 + 3 * TINY, 2.0 ** -10)


def test_tiny_rows_follow_the_row_quantiser(cuda_device) -> None:
    """eps = 2^-20 is all that is left of mean(s^2) + eps, so that y = 2^10 s, which BF16 holds."""

    x, _ = _tiny_rows(cuda_device, torch.bfloat16)
    x[7] = 0
    w = torch.ones(256, dtype=torch.bfloat16, device=cuda_device)
    codes, scale, _ = add_rms_norm_fp8(x, None, w, eps=2.0 ** -20)
    q, qs = quantize_rows_fp8((x * 1024).contiguous())
    assert torch.equal(codes, q) and torch.equal(scale, qs)


def test_codes_at_every_rounding_border_follow_the_row_quantiser(cuda_device) -> None:
    """|s| = 1 throughout and eps = 0 make y = +-w; w runs through all BF16 mantissas below each
    largest one, so that the quotients fall on and beside the borders between codes."""

    ladder = (torch.arange(128, 256).float()[None] * 2.0 ** torch.arange(-16, -6).float()[:, None])
    ladder = ladder.flatten().bfloat16().to(cuda_device)                  # ten octaves, 1280 values
    x = torch.ones(1, 1280, dtype=torch.bfloat16, device=cuda_device)
    x[0, ::3] = -1
    for top in range(128, 256):
        w = ladder.clone()
        w[ladder > top * 2.0 ** -7] = top * 2.0 ** -7
        codes, scale, _ = add_rms_norm_fp8(x, None, w, eps=0.0)
        q, qs = quantize_rows_fp8((x * w).contiguous())
        assert torch.equal(scale, qs) and torch.equal(codes, q), top
