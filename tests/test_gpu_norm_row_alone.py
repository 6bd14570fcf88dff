"""A row's norm depends on that row alone: the same row in calls of any number of rows."""

from __future__ import annotations

import pytest
import torch

from b200moe import add_rms_norm, add_rms_norm_fp8
from test_gpu_norm import TYPES, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [16, 208, 2048, 2880, 7168, 16384, 20000])
@pytest.mark.parametrize("residual, weight", TYPES)
def test_rows_alone_and_among_others(cuda_device, hidden, residual, weight) -> None:
    x, r, w = _inputs(cuda_device, 900, hidden, residual, weight)
    want, kept = add_rms_norm(x, r, w)
    codes, scale, _ = add_rms_norm_fp8(x, r, w)
    for s in (slice(0, 1), slice(7, 12), slice(100, 396), slice(500, 797)):
        part = None if r is None else r[s].clone()
        got, kept_part = add_rms_norm(x[s].clone(), part, w)
        assert torch.equal(got, want[s]) and torch.equal(kept_part, kept[s])
        c, f, _ = add_rms_norm_fp8(x[s].clone(), part, w)
        assert torch.equal(c, codes[s]) and torch.equal(f, scale[s])
