"""Without a residual the hidden states are the new residual: the result must not replace them."""

from __future__ import annotations

import pytest
import torch

from b200moe import add_rms_norm, add_rms_norm_fp8

pytestmark = pytest.mark.gpu


def test_hidden_states_that_are_the_new_residual_are_not_overwritten(cuda_device) -> None:
    x = torch.randn(5, 64, device=cuda_device).bfloat16()
    held = x.clone()
    w = torch.full((64,), 2.0, device=cuda_device)
    for out in (x, x.view(64, 5).view(5, 64)):
        with pytest.raises(ValueError, match="must not be hidden_states"):
            add_rms_norm(x, None, w, out=out)
    with pytest.raises(ValueError, match="overlap"):
        add_rms_norm_fp8(x, None, w, out=x.view(torch.uint8).view(-1)[:320].view(5, 64))
    assert torch.equal(x, held)
    out, kept = add_rms_norm(x, None, w, out=torch.empty_like(x))
    assert kept is x and torch.equal(x, held) and not torch.equal(out, x)
    r = torch.zeros_like(x)
    out, kept = add_rms_norm(x, r, w, out=x)     # with a residual the result may be in place
    assert out is x and torch.equal(kept, held)
