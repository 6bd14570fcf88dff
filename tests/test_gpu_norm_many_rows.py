"""The residual norm's form for many rows, and launches that follow one another.

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


@pytest.mark.parametrize("hidden", [1024, 4096, 7168])
def test_a_chain_of_norms_over_the_same_rows(cuda_device, hidden) -> None:
    """Each launch may begin before the one in front has ended and reads what that one stores: the
    rows, the residual and, in the third norm of a turn, the weight."""

    x, r, w = _inputs(cuda_device, 1500, hidden, torch.float32, torch.bfloat16)

    def turn(x, r, wait):
        _, r = add_rms_norm(x, r, w, out=x, residual_out=r)
        wait()
        one, _ = add_rms_norm(x[:400], None, w)
        wait()
        row = one[7]                                  # a weight that the kernel in front stored
        y, r = add_rms_norm(x, r, row, residual_out=r)
        wait()
        codes, scale, r = add_rms_norm_fp8(y, r, w, residual_out=r)
        wait()
        return y, r, codes, scale

    def run(wait):
        a, b, seen = x.clone(), r.clone(), []
        for _ in range(6):
            a, b, codes, scale = turn(a, b, wait)
            seen += [codes, scale]
        torch.cuda.synchronize()
        return [a, b, *seen]

    want = run(torch.cuda.synchronize)
    for _ in range(5):
        assert all(torch.equal(g, t) for g, t in zip(run(lambda: None), want))
