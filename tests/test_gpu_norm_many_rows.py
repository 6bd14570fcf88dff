"""The residual norm's form for many rows.

Tolerances as in test_gpu_norm.py.
"""

from __future__ import annotations

import pytest
import torch

from b200moe import add_rms_norm, add_rms_norm_fp8
from test_gpu_norm import FP32, TYPES, _check_residual, _formula, _inputs, _near

pytestmark = pytest.mark.gpu

# more rows than two a SM: 256 threads and one, two or four vectors of a row each
MANY = [(297, 2048), (601, 2880), (400, 4096), (333, 5120), (300, 7168), (310, 8208), (299, 16384),
        (298, 16400), (297, 32768)]


@pytest.mark.parametrize("rows, hidden", MANY)
@pytest.mark.parametrize("residual, weight", TYPES)
def test_many_rows(cuda_device, rows, hidden, residual, weight) -> None:
    x, r, w = _inputs(cuda_device, rows, hidden, residual, weight)
    s, y = _formula(x, r, w, 1e-6)
    out, kept = add_rms_norm(x, r, w)
    _near(out, y, 2.0 ** -8 + FP32)
    codes, scale, kept8 = add_rms_norm_fp8(x, r, w)
    want = y.abs().amax(-1) / 448.0
    _near(scale, want, FP32)
    _near(codes.view(torch.float8_e4m3fn).float(), y / want[:, None], 2.0 ** -4 + 3 * FP32, 2.0 ** -10)
    if r is not None:
        _check_residual(kept, s, r)
        assert torch.equal(kept8, kept)
