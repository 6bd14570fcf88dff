"""Sampling with an infinite temperature in a tensor: every weight of a finite logit is one."""

from __future__ import annotations

import pytest
import torch

from b200moe import sample_tokens

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("top_k", [0, 7, 900, 3000, 4999])
@pytest.mark.parametrize("vocab", [5000, 70001])
def test_all_tokens_alike_at_an_infinite_temperature(cuda_device, vocab, top_k) -> None:
    """Logits further apart than FP32's largest number.  Kept are the first top_k of the order, and
    as all weights are one, the token is number floor(u * kept) of them in id order."""

    rows = 6
    logits = torch.full((rows, vocab), 3e38, device=cuda_device)
    logits[:, 1::2] = -3e38
    logits[:, 5] = -INF
    u = (torch.arange(rows, device=cuda_device) + 0.5).float() / rows
    heat = torch.full((rows,), INF, device=cuda_device)
    ids, logprobs = sample_tokens(logits, u, temperature=heat, top_k=top_k, return_logprobs=True)
    order = torch.cat([torch.arange(0, vocab, 2), torch.arange(1, vocab, 2)])
    order = order[order != 5]
    kept = (order[:top_k] if top_k else order).sort().values
    want = kept[(u.double().cpu() * len(kept)).floor().long()]
    assert torch.equal(ids.cpu(), want)
    share = -torch.tensor(float(len(kept)), dtype=torch.float64).log()
    assert float((logprobs.double().cpu() - share).abs().max()) <= 2.0 ** -24 * 12 + 2.0 ** -27


@pytest.mark.parametrize("top_k, top_p", [(0, 1.0), (1, 1.0), (1500, 1.0), (1500, 0.5), (0, 0.5)])
def test_an_infinite_logit_at_an_infinite_temperature(cuda_device, top_k, top_p) -> None:
    logits = torch.randn(3, 5000, device=cuda_device,
                         generator=torch.Generator(cuda_device).manual_seed(8))
    logits[0, 4321] = INF
    logits[1, [17, 4000]] = INF
    u = torch.tensor([0.9, 0.75, 0.5], device=cuda_device)
    heat = torch.tensor([INF, INF, 1.0], device=cuda_device)
    ids, logprobs = sample_tokens(logits, u, temperature=heat, top_k=top_k, top_p=top_p,
                                  return_logprobs=True)
    # one of two infinite logits holds half the weight, which top_p = 0.5 is satisfied with
    second = 17 if top_k == 1 or top_p == 0.5 else 4000
    assert ids[:2].tolist() == [4321, second]
    assert float(logprobs[0]) == 0.0
    alone = sample_tokens(logits[2:], u[2:].contiguous(), top_k=top_k, top_p=top_p)
    assert int(ids[2]) == int(alone)
