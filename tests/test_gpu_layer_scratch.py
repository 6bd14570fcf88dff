"""The one-kernel layer and the staged forward take turns on one workspace, whose bytes they share:
every result is what it is on a workspace of its own."""

from __future__ import annotations

import pytest
import torch

from b200moe import (B300MoEWorkspace, b300_moe_forward, b300_moe_forward_fp8,
                     b300_moe_forward_nvfp4, b300_moe_layer, b300_moe_layer_fp8,
                     quantize_expert_weights_fp8, quantize_expert_weights_nvfp4, topk_routing)
from test_gpu_layer_few import _inputs

pytestmark = pytest.mark.gpu


# the last shape asks for more than the forward does
@pytest.mark.parametrize("tokens, hidden, inter, experts, top_k",
                         [(1, 256, 512, 8, 2), (8, 512, 256, 16, 4), (5, 128, 1024, 32, 8),
                          (8, 64, 64, 256, 8)])
def test_layer_and_forward_take_turns(cuda_device, tokens, hidden, inter, experts, top_k) -> None:
    x, r, gate_up, down = _inputs(cuda_device, tokens, hidden, inter, experts)
    fp8 = quantize_expert_weights_fp8(gate_up, down)
    fp4 = quantize_expert_weights_nvfp4(gate_up, down)
    ids, shares = topk_routing(x.float() @ r.float().T, top_k)
    shares = shares.bfloat16()
    sizes = dict(num_experts=experts, top_k=top_k)
    calls = [lambda ws: b300_moe_layer(x, r, gate_up, down, workspace=ws, **sizes),
             lambda ws: b300_moe_forward(x, ids, shares, gate_up, down, workspace=ws, **sizes),
             lambda ws: b300_moe_layer_fp8(x, r, fp8, workspace=ws, **sizes),
             lambda ws: b300_moe_forward_fp8(x, ids, shares, fp8, workspace=ws, **sizes),
             lambda ws: b300_moe_forward_nvfp4(x, ids, shares, fp4, workspace=ws, **sizes)]
    want = [call(B300MoEWorkspace(tokens, device=cuda_device)) for call in calls]
    torch.cuda.synchronize()
    shared = B300MoEWorkspace(tokens, device=cuda_device)
    side = torch.cuda.Stream()
    order = torch.randint(len(calls), (60,), generator=torch.Generator().manual_seed(4)).tolist()
    got = []
    for i, which in enumerate([0, 1, 0, 3, 2, 1, 2, 4, 0, 4, 2, 3] + order):
        with torch.cuda.stream(side if i % 7 == 6 else torch.cuda.current_stream()):
            got.append((which, calls[which](shared)))
    torch.cuda.synchronize()
    for which, out in got:
        assert torch.equal(out, want[which]), which
    assert shared.status() == 0 and shared.allocation_count == 1
