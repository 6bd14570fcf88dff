"""The operators around the layer where offsets pass 32 bits, and where several threads call them at
once: results are those of small calls, of the same rows alone."""

from __future__ import annotations

import threading

import pytest
import torch

from b200moe import (B300MoEWorkspace, Fp8ExpertWeights, add_rms_norm, add_rms_norm_fp8,
                     b300_moe_layer, b300_moe_layer_fp8, sample_tokens)
from test_gpu_layer_few import _inputs
from test_gpu_norm import FP32, _check_residual, _formula, _near

pytestmark = pytest.mark.gpu


def _generator(device, seed=3):
    return torch.Generator(device=device).manual_seed(seed)


def test_norm_of_more_than_two_to_the_31_elements(cuda_device) -> None:
    """Rows at either end bit for bit as in a call of 300 rows; ten rows between, which in a call of
    their own are summed in another order, against the formula (tolerances of test_gpu_norm.py)."""

    rows, hidden = 270001, 8192
    x = torch.empty(rows, hidden, device=cuda_device, dtype=torch.bfloat16)
    x.normal_(generator=_generator(cuda_device))
    r = torch.empty_like(x).normal_(generator=_generator(cuda_device, 4))
    w = torch.rand(hidden, device=cuda_device, generator=_generator(cuda_device, 5))
    ends, between = [slice(0, 300), slice(rows - 300, rows)], slice(262140, 262150)
    want = [add_rms_norm(x[s].clone(), r[s].clone(), w) for s in ends]
    want8 = [add_rms_norm_fp8(x[s].clone(), r[s].clone(), w) for s in ends]
    total, y = _formula(x[between], r[between], w, 1e-6)
    codes, scale, kept = add_rms_norm_fp8(x, r, w)
    for s, (c, f, k) in zip(ends, want8):
        assert torch.equal(codes[s], c) and torch.equal(scale[s], f) and torch.equal(kept[s], k)
    exact = y.abs().amax(-1) / 448.0
    _near(scale[between], exact, FP32)
    _near(codes[between].view(torch.float8_e4m3fn).float(), y / exact[:, None],
          2.0 ** -4 + 3 * FP32, 2.0 ** -10)
    del codes, kept
    held = r[between].clone()
    add_rms_norm(x, r, w, out=x, residual_out=r)
    for s, (out, k) in zip(ends, want):
        assert torch.equal(x[s], out) and torch.equal(r[s], k)
    _near(x[between], y, 2.0 ** -8 + FP32)
    _check_residual(r[between], total, held)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sampling_from_more_than_two_to_the_31_logits(cuda_device, dtype) -> None:
    rows, vocab, pitch = 33001, 65000, 65537          # rows with odd addresses
    logits = torch.empty(rows, pitch, device=cuda_device, dtype=dtype)
    logits.normal_(0, 2, generator=_generator(cuda_device))
    u = torch.rand(rows, device=cuda_device, generator=_generator(cuda_device, 4))
    ids, logp = sample_tokens(logits[:, :vocab], u, top_k=300, top_p=0.9, return_logprobs=True)
    for s in (slice(0, 40), slice(32760, 32790), slice(rows - 40, rows)):
        some, p = sample_tokens(logits[s, :vocab].clone(), u[s].clone(), top_k=300, top_p=0.9,
                                return_logprobs=True)
        assert torch.equal(ids[s], some) and torch.equal(logp[s], p)


@pytest.mark.parametrize("fp8", [False, True])
def test_experts_behind_four_gigabytes(cuda_device, fp8) -> None:
    """The last experts of a bank of 10.5 GB (BF16; E4M3 5.2 GB), and the same experts in a bank of
    their own."""

    hidden, inter, experts, last, tokens = 4096, 4096, 104, 8, 5
    g = _generator(cuda_device)
    if fp8:  # codes of finite values: no NaN pattern
        def bank(*shape):
            return torch.randint(0, 120, shape, device=cuda_device, dtype=torch.uint8, generator=g)
    else:
        def bank(*shape):
            return torch.empty(*shape, device=cuda_device, dtype=torch.bfloat16).normal_(0, 0.02, generator=g)
    gate_up, down = bank(experts, 2 * inter, hidden), bank(experts, hidden, inter)
    assert gate_up.numel() * gate_up.element_size() > 3 * 2 ** 30
    x = torch.empty(tokens, hidden, device=cuda_device, dtype=torch.bfloat16).normal_(generator=g)
    router = torch.empty(experts, hidden, device=cuda_device).normal_(0, 0.02, generator=g)
    x[:, 0] = 4.0                                       # in favour of the last experts
    router[:, 0] = -20.0
    router[-last:, 0] = 20.0
    options = dict(top_k=4, return_routing=True, check_status=True)
    if fp8:
        scales = [torch.rand(experts, n, device=cuda_device, generator=g) * 1e-4 for n in (2 * inter, hidden)]
        out, ids, shares = b300_moe_layer_fp8(
            x, router, Fp8ExpertWeights(gate_up, scales[0], down, scales[1]), num_experts=experts, **options)
        own = Fp8ExpertWeights(*(t[-last:].clone() for t in (gate_up, scales[0], down, scales[1])))
        alone = b300_moe_layer_fp8(x, router[-last:].clone(), own, num_experts=last, **options)
    else:
        out, ids, shares = b300_moe_layer(x, router, gate_up, down, num_experts=experts, **options)
        alone = b300_moe_layer(x, router[-last:].clone(), gate_up[-last:].clone(),
                               down[-last:].clone(), num_experts=last, **options)
    assert int(ids.min()) >= experts - last and bool(out.isfinite().all()) and bool((out != 0).any())
    assert torch.equal(ids - (experts - last), alone[1]) and torch.equal(shares, alone[2])
    assert torch.equal(out, alone[0])


def test_threads_that_call_at_once(cuda_device) -> None:
    """Four threads on streams of their own; two of them share a workspace, which orders them."""

    x, r, gate_up, down = _inputs(cuda_device, 4, 512, 256, 16)
    w = torch.rand(512, device=cuda_device, generator=_generator(cuda_device))
    logits = torch.randn(4, 9000, device=cuda_device, generator=_generator(cuda_device, 2))
    u = torch.rand(4, device=cuda_device, generator=_generator(cuda_device, 3))
    spaces = [B300MoEWorkspace(4, device=cuda_device) for _ in range(3)]

    def step(space):
        y, kept = add_rms_norm(x, x, w)
        out = b300_moe_layer(y, r, gate_up, down, num_experts=16, top_k=4, workspace=space)
        return y, kept, out, sample_tokens(logits, u, top_p=0.9)

    want = step(spaces[0])
    torch.cuda.synchronize()
    failures: list = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got = step(spaces[min(i, 2)])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want)):
                        failures.append((i, "differs"))
        except Exception as error:  # noqa: BLE001
            failures.append((i, repr(error)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures and all(space.status() == 0 for space in spaces)
