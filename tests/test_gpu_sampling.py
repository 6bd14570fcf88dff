"""The sampler on the GPU against the definition in 64 bits; tokens have to be equal.

Tolerance of the log-probabilities: its FP32 rounding (2^-24 relative) and the rounding of the
weights to multiples of 2^-45, at most 2^18 tokens * 2^-46 against a sum of at least 1 (2^-28);
2^-27 covers that and the 64-bit logarithm.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from b200moe import sample_tokens

pytestmark = pytest.mark.gpu


def _oracle(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, log-probability) of one row."""

    x = logits.double().cpu().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    best = x.max()
    if best == -np.inf:
        return -1, -math.inf
    if not temperature > 0:
        return int(x.argmax()), 0.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    w = np.exp(np.where(x[order] == best, 0.0, x[order] - best) / temperature)
    keep = w >= min(min_p, 1.0)
    order, w = order[keep], w[keep]
    if top_p < 1:
        count = int(np.searchsorted(np.cumsum(w), max(top_p, 0.0) * w.sum())) + 1
        order, w = order[:count], w[:count]
    place = np.argsort(order)
    order, w = order[place], w[place]
    upto = np.cumsum(w)
    at = int(np.searchsorted(upto, min(max(u, 0.0), 1.0) * upto[-1], side="right"))
    at = min(at, int(np.nonzero(w)[0][-1]))
    return int(order[at]), float(np.log(w[at] / upto[-1]))


def _check(logits, u, ids, logprobs=None, **settings):
    """Every row against the oracle; settings are numbers (held in FP32, as documented) or [T]
    tensors."""

    rows = logits.shape[0]
    each = {k: (v.tolist() if isinstance(v, torch.Tensor)
                else [v if isinstance(v, int) else float(np.float32(v))] * rows)
            for k, v in settings.items()}
    for r in range(rows):
        want, logp = _oracle(logits[r], float(u[r]), **{k: v[r] for k, v in each.items()})
        assert int(ids[r]) == want, (r, int(ids[r]), want, {k: v[r] for k, v in each.items()})
        if logprobs is not None:
            got = float(logprobs[r])
            assert got == logp or abs(got - logp) <= 2.0 ** -24 * abs(logp) + 2.0 ** -27, (r, got, logp)


def _run(logits, u, **settings):
    ids, logprobs = sample_tokens(logits, u, return_logprobs=True, **settings)
    assert ids.dtype is torch.int64 and logprobs.dtype is torch.float32
    _check(logits, u, ids, logprobs, **settings)
    return ids, logprobs


def _logits(device, rows, vocab, dtype=torch.float32, spread=2.5, seed=21):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device=device) * spread
    return x.to(dtype), torch.rand(rows, generator=g, device=device)


VOCABS = [1, 2, 31, 200, 513, 4097, 32003, 129280, 262144]
SETTINGS = [
    {},
    {"temperature": 0.0},
    {"temperature": 0.7, "top_k": 5},
    {"top_k": 50, "top_p": 0.9},
    {"temperature": 1.3, "top_p": 0.95},
    {"temperature": 0.8, "min_p": 0.05},
    {"temperature": 2.0, "top_k": 1000, "top_p": 0.8, "min_p": 0.01},
    {"top_p": 0.3},
    {"temperature": 50.0, "top_p": 0.5},
    {"temperature": 0.01, "top_k": 300},
]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_settings(cuda_device, vocab, settings) -> None:
    logits, u = _logits(cuda_device, 3, vocab)
    _run(logits, u, **settings)


@pytest.mark.parametrize("rows, vocab", [(1, 32000), (17, 32003), (64, 5000), (200, 129)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.3, 2.5, 8.0])
def test_settings_of_each_row(cuda_device, rows, vocab, dtype, spread) -> None:
    logits, u = _logits(cuda_device, rows, vocab, dtype, spread)
    g = torch.Generator().manual_seed(rows)
    pick = lambda values: torch.tensor(values)[torch.randint(len(values), (rows,), generator=g)]  # noqa: E731
    _run(logits, u,
         temperature=pick([0.0, 0.5, 0.9, 1.0, 1.7]).to(cuda_device),
         top_k=pick([0, 0, 1, 7, 40, 100000]).int().to(cuda_device),
         top_p=pick([1.0, 1.0, 0.99, 0.7, 0.1, 0.0]).to(cuda_device),
         min_p=pick([0.0, 0.0, 0.001, 0.2, 1.0]).to(cuda_device))


def test_padded_and_unaligned_rows(cuda_device) -> None:
    for dtype in (torch.float32, torch.bfloat16):
        held, u = _logits(cuda_device, 5, 5003, dtype)
        for view in (held[:, :4999], held[:, 1:], held[:, 3:4000], held[1:4, 7:]):
            _run(view, u[: view.shape[0]].contiguous(), top_p=0.9, top_k=200)
        held[:, 4999:] = float("inf")  # what lies behind the vocabulary is not read
        _run(held[:, :4999], u)


@pytest.mark.parametrize("vocab", [64, 3001, 40000])
def test_equal_logits(cuda_device, vocab) -> None:
    """Few different values: thresholds fall inside runs of equal logits."""

    logits, u = _logits(cuda_device, 24, vocab, spread=1.5)
    logits = logits.round()
    row = torch.arange(24, device=cuda_device)
    _run(logits, u, top_k=(1 + row * vocab // 30).int())
    _run(logits, u, top_p=(0.02 + 0.04 * row).float())
    _run(logits, u, top_k=(1 + row * vocab // 30).int(), top_p=(0.02 + 0.04 * row).float(),
         temperature=0.5)
    flat = torch.full_like(logits, -3.25)  # all equal: k of them, the first ones
    _run(flat, u, top_k=7)
    _run(flat, u, top_p=0.5)
    ids = _run(flat, u)[0]
    # w * V * u is exact: the token is floor(u V)
    assert torch.equal(ids, (u.double() * vocab).floor().long())


def test_masks(cuda_device) -> None:
    logits, u = _logits(cuda_device, 12, 9001)
    inf, low = float("inf"), torch.finfo(torch.float32).min
    logits[0] = -inf                       # nothing left
    logits[1] = float("nan")               # nothing left either
    logits[2] = -inf
    logits[2, 8000] = -50.0                # one token left
    logits[3, ::2] = float("nan")
    logits[4, 100:] = -inf                 # fewer than top-k left
    logits[5] = low                        # all at the type's lowest value: all alike
    logits[6, 10:] = low
    logits[7, [5, 900]] = inf              # two tokens share all weight
    logits[8] = -inf
    logits[8, 4:9] = low
    logits[9] = 0.0
    logits[9, ::3] = -0.0                  # equal to 0
    logits[10, 1:] = -inf
    logits[11, 8999] = 1e38
    for settings in ({}, {"top_k": 200}, {"top_p": 0.9}, {"top_k": 300, "top_p": 0.5, "min_p": 0.1},
                     {"temperature": 0.0}, {"temperature": 1e-30, "top_p": 0.9},
                     {"temperature": 1e30, "top_k": 4000, "top_p": 0.7}):
        ids, logprobs = _run(logits, u, **settings)
        assert ids[:2].tolist() == [-1, -1] and logprobs[:2].tolist() == [-inf, -inf]
        assert int(ids[2]) == 8000 and int(ids[7]) in (5, 900) and int(ids[10]) == 0


def test_random_numbers_at_the_ends(cuda_device) -> None:
    logits, _ = _logits(cuda_device, 1, 700)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 2.0 ** -30, 1.0, 2.0, -1.0], device=cuda_device)
    rows = logits.expand(6, 700).contiguous()
    for settings in ({}, {"top_k": 20}, {"top_p": 0.5}):
        _run(rows, u, **settings)
    ids = sample_tokens(rows, torch.full_like(u, float("nan")), top_k=20)
    assert torch.equal(ids, sample_tokens(rows, torch.zeros_like(u), top_k=20))


def test_settings_outside_their_range_in_tensors(cuda_device) -> None:
    logits, u = _logits(cuda_device, 4, 3000)
    nan = float("nan")

    def held(*values):
        return torch.tensor(values, device=cuda_device)

    plain = sample_tokens(logits, u)
    greedy = sample_tokens(logits, u, temperature=0.0)
    assert torch.equal(greedy, logits.argmax(-1))
    assert torch.equal(sample_tokens(logits, u, temperature=held(-1.0, nan, 0.0, -0.0)), greedy)
    assert torch.equal(sample_tokens(logits, u, top_k=held(-5, 0, 3000, 2 ** 31 - 1).int()), plain)
    assert torch.equal(sample_tokens(logits, u, top_p=held(nan, 1.0, 7.0, float("inf"))), plain)
    assert torch.equal(sample_tokens(logits, u, top_p=held(-1.0, 0.0, -0.0, -float("inf"))), greedy)
    assert torch.equal(sample_tokens(logits, u, min_p=held(nan, 0.0, -3.0, -0.0)), plain)
    assert torch.equal(sample_tokens(logits, u, min_p=held(1.0, 2.0, 1e30, float("inf"))), greedy)


def test_a_rows_token_depends_on_that_row_alone(cuda_device) -> None:
    """Batches of other sizes cut rows into other pieces; tokens stay."""

    logits, u = _logits(cuda_device, 150, 40000, spread=0.4)
    for settings in ({}, {"top_p": 0.8}, {"top_k": 5000, "top_p": 0.9}):
        ids, logprobs = sample_tokens(logits, u, return_logprobs=True, **settings)
        for rows in (1, 5, 40):
            some, logp = sample_tokens(logits[:rows], u[:rows].contiguous(), return_logprobs=True,
                                       **settings)
            assert torch.equal(some, ids[:rows]) and torch.equal(logp, logprobs[:rows])


def test_frequencies_follow_the_probabilities(cuda_device) -> None:
    """With u at the midpoints of 10000 equal steps every token is drawn as often as its share
    says, to within one draw (its share of the steps, rounded up or down at either end)."""

    logits, _ = _logits(cuda_device, 1, 50, spread=1.0)
    n = 10000
    u = ((torch.arange(n, device=cuda_device) + 0.5) / n).float()
    ids = sample_tokens(logits.expand(n, 50).contiguous(), u, temperature=0.9)
    share = torch.softmax(logits[0].double() / float(np.float32(0.9)), -1) * n
    counts = torch.bincount(ids, minlength=50).double()
    assert float((counts - share).abs().max()) <= 1.0 + 1e-3


def test_out_streams_and_graphs(cuda_device) -> None:
    logits, u = _logits(cuda_device, 9, 32000)
    want = sample_tokens(logits, u, top_p=0.9)
    out = torch.empty(9, dtype=torch.int64, device=cuda_device)
    assert sample_tokens(logits, u, top_p=0.9, out=out) is out and torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample_tokens(logits, u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    heat = torch.ones(9, device=cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, logp = sample_tokens(logits, u, temperature=heat, top_k=40, return_logprobs=True)
    other, u2 = _logits(cuda_device, 9, 32000, seed=4)
    logits.copy_(other)
    u.copy_(u2)
    heat.fill_(0.6)
    graph.replay()
    _check(other, u2, ids, logp, temperature=heat, top_k=40)
    with pytest.raises(ValueError, match="uniforms must be"):
        sample_tokens(logits, u.cpu())
