"""The one-kernel layer with E4M3 expert weights and an FP32 router, in both of its stage shapes.

Bounds as in test_gpu_layer_few.py.
"""

from __future__ import annotations

import pytest
import torch

from b200moe import b300_moe_layer_fp8, quantize_expert_weights_fp8
from test_gpu_layer_few import SHAPES, _check, _formula, _inputs, _route

pytestmark = pytest.mark.gpu

# stages of 32 rows up to 32 output rows a block, of 16 rows above
WIDE = [(8, 4736, 144, 8, 4), (5, 4752, 208, 16, 8), (8, 8192, 80, 8, 2), (3, 2368, 272, 4, 2),
        (4, 2384, 48, 32, 8), (2, 144, 16, 4, 1)]


@pytest.mark.parametrize("tokens, hidden, inter, experts, top_k",
                         [s for s in SHAPES if s[1] % 16 == 0 and s[2] % 16 == 0] + WIDE)
def test_fp8_weights_with_an_fp32_router(cuda_device, tokens, hidden, inter, experts, top_k) -> None:
    x, r, gate_up, down = _inputs(cuda_device, tokens, hidden, inter, experts, torch.float32)
    fw = quantize_expert_weights_fp8(gate_up, down)
    out, ids, weights = b300_moe_layer_fp8(x, r, fw, num_experts=experts, top_k=top_k,
                                           return_routing=True, check_status=True)
    want_ids, want_weights = _route(x, r, top_k)
    assert torch.equal(ids, want_ids)
    assert float((weights.double() - want_weights).abs().max()) <= 2.0 ** -21

    def matrix(q, scale):
        return lambda e: q[e].view(torch.float8_e4m3fn).double() * scale[e].double()[:, None]

    _check(out, *_formula(x, matrix(fw.gate_up_q, fw.gate_up_scale),
                          matrix(fw.down_q, fw.down_scale), ids, want_weights, fp8=True))
