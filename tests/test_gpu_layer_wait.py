"""The one-kernel layer's bounded waits.  A counter of the grid barrier that starts at -1 stays one
below what the blocks wait for: all of them give up after a second, the call reports it, and the
workspace is as good as new."""

from __future__ import annotations

import pytest
import torch

from b200moe import (B300MoEWorkspace, b300_moe_forward, b300_moe_layer, b300_moe_layer_fp8,
                     quantize_expert_weights_fp8, topk_routing)
from b200moe import _lib
from test_gpu_layer_few import _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("barrier", [0, 1])
@pytest.mark.parametrize("fp8", [False, True])
def test_a_wait_that_runs_out_is_reported_and_leaves_the_workspace_usable(cuda_device, barrier,
                                                                          fp8) -> None:
    x, r, gate_up, down = _inputs(cuda_device, 4, 512, 256, 16)
    ws = B300MoEWorkspace(4, device=cuda_device)
    options = dict(num_experts=16, top_k=4, workspace=ws)
    weights = (quantize_expert_weights_fp8(gate_up, down),) if fp8 else (gate_up, down)
    layer = b300_moe_layer_fp8 if fp8 else b300_moe_layer
    want = layer(x, r, *weights, **options)
    torch.cuda.synchronize()
    counters = ws.scratch[192:204].view(torch.int32)
    counters[barrier] = -1
    with pytest.raises(RuntimeError, match="bounded device-side wait gave up"):
        layer(x, r, *weights, check_status=True, **options)
    assert ws.status() == _lib.STATUS_PIPE_TIMEOUT and counters.tolist() == [0, 0, 0]

    assert torch.equal(layer(x, r, *weights, check_status=True, **options), want)
    ids, shares = topk_routing(x.float() @ r.float().T, 4)
    alone = b300_moe_forward(x, ids, shares.bfloat16(), gate_up, down, num_experts=16, top_k=4)
    assert torch.equal(b300_moe_forward(x, ids, shares.bfloat16(), gate_up, down, **options), alone)
    assert torch.equal(layer(x, r, *weights, **options), want)
    assert ws.status() == 0 and counters.tolist() == [0, 0, 0] and ws.allocation_count == 1
