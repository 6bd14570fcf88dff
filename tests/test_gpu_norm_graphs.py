"""Norms of many rows in captured graphs, behind nodes of every kind: their launches may overlap the
kernel in front, and with none, or several, or a copy in front they have to wait all the same."""

from __future__ import annotations

import pytest
import torch

from b200moe import add_rms_norm, add_rms_norm_fp8
from test_gpu_norm import _inputs

pytestmark = pytest.mark.gpu


def _steps(x, r, w, x2, side):
    """A copy, a norm, a fork to another stream with a norm on either, a join, a norm of both."""

    main = torch.cuda.current_stream()
    a = torch.empty_like(x)
    a.copy_(x)                                            # a copy in front
    y, kept = add_rms_norm(a, r, w)                       # another norm in front
    z, kept = add_rms_norm(y, kept, w, residual_out=kept)
    side.wait_stream(main)
    with torch.cuda.stream(side):
        one, _ = add_rms_norm(z, None, w)                 # first of its stream
    two, kept2 = add_rms_norm(x2, kept, w)                # beside it
    main.wait_stream(side)
    total, last = add_rms_norm(one, kept2, w)             # two in front
    b = torch.zeros_like(x)                               # a fill in front
    codes, scale, end = add_rms_norm_fp8(total + two + b, last, w)
    return two, total, codes, scale, end


@pytest.mark.parametrize("rows, hidden", [(500, 4096), (3000, 256), (300, 7168), (20, 4096)])
def test_norms_in_a_graph(cuda_device, rows, hidden) -> None:
    x, r, w = _inputs(cuda_device, rows, hidden, torch.float32, torch.bfloat16)
    x2 = _inputs(cuda_device, rows, hidden, None, torch.bfloat16, seed=9)[0]
    side = torch.cuda.Stream()
    _steps(x, r, w, x2, side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _steps(x, r, w, x2, side)
    for seed in (20, 21, 22):
        nx, nr, _ = _inputs(cuda_device, rows, hidden, torch.float32, torch.bfloat16, seed=seed)
        want = _steps(nx, nr, w, x2, side)
        x.copy_(nx)
        r.copy_(nr)
        graph.replay()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
