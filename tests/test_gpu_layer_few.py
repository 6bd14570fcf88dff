"""The one-kernel layer on the GPU against the formula in 64 bits.

Tolerances.  One matrix instruction adds 16 products and the accumulator; whether it rounds or
cuts each of the 17 aligned terms, it is off by at most 17 * 2^-23 of the sum of their
magnitudes.  A warp chains at most ceil(units / 16) * 4 (BF16) or * 8 (E4M3) of them (a unit is
64 or 128 elements) and 16 partial sums follow: `chain` below, times the sum of the products'
magnitudes, bounds a dot product.  silu changes by at most 1.1 times its argument.  Activations
are held as two BF16 numbers (2^-16), with E4M3 weights as FP16 numbers scaled so that the
largest of a row is at least 2^13 (2^-12, and 2^-25 / 2^13 of the largest for those that become
subnormal; the token rows, eight bits, only have the latter); the few FP32 operations on them
add 2^-20.  The result is rounded to BF16 (2^-8).  The bound is propagated element by element.
"""

from __future__ import annotations

import math

import pytest
import torch

from b200moe import (B300MoEWorkspace, b300_moe_forward, b300_moe_layer, b300_moe_layer_fp8,
                     quantize_expert_weights_fp8, topk_routing)

pytestmark = pytest.mark.gpu


def _chain(length: int, fp8: bool, columns: int = 1) -> float:
    units = columns * math.ceil(length / (128 if fp8 else 64))
    return (math.ceil(units / 16) * (8 if fp8 else 4) * 17 + 32) * 2.0 ** -23


def _inputs(device, tokens, hidden, inter, experts, router=torch.bfloat16, seed=11):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, std):
        return torch.empty(*shape, device=device, dtype=torch.bfloat16).normal_(0, std, generator=g)

    x = normal(tokens, hidden, std=1.0)
    r = torch.empty(experts, hidden, device=device).normal_(0, hidden ** -0.5, generator=g).to(router)
    return x, r, normal(experts, 2 * inter, hidden, std=hidden ** -0.5), \
        normal(experts, hidden, inter, std=inter ** -0.5)


def _route(x, router, top_k):
    logits = (x.double()[:, None] * router.double()[None]).sum(-1)
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    return order.indices[:, :top_k], torch.softmax(order.values[:, :top_k], -1)


def _formula(x, gate_up, down, ids, weights, fp8=False):
    """(output, bound on the kernel's error) in 64 bits; gate_up(e) and down(e) give matrices."""

    x = x.double()
    out, bound = torch.zeros_like(x), torch.zeros_like(x)
    used = int(ids.unique().numel())
    for e in ids.unique().tolist():
        gu, dn = gate_up(e), down(e)
        inter = gu.shape[0] // 2
        eh, ei = _chain(gu.shape[1], fp8), _chain(inter, fp8, used)
        for t, k in (ids == e).nonzero().tolist():
            both, size = gu @ x[t], gu.abs() @ x[t].abs()
            if fp8:
                size = size + gu.abs().sum(-1) * x[t].abs().max() * 2.0 ** -38 / eh
            gate, up = both[:inter], both[inter:]
            silu, p = gate * torch.sigmoid(gate), float(weights[t, k])
            act = p * silu * up
            off = p * eh * (1.1 * size[:inter] * (up.abs() + eh * size[inter:])
                            + silu.abs() * size[inter:]) + act.abs() * (2.0 ** -16 + 2.0 ** -20)
            if fp8:
                off = off + act.abs() * 2.0 ** -12 + act.abs().max() * 2.0 ** -38
            out[t] += dn @ act
            # high and low part are multiplied one after the other: two chains
            bound[t] += dn.abs() @ (off + 2 * ei * (act.abs() + off))
    return out, bound + 2.0 ** -8 * (out.abs() + bound)


def _check(got, want, bound):
    over = (got.double() - want).abs() - bound
    assert bool((over <= 0).all()), float(over.max())


# tokens, hidden, inter, experts, top_k
SHAPES = [(1, 8, 8, 1, 1), (8, 64, 96, 16, 8), (3, 72, 200, 4, 2), (5, 256, 512, 8, 2),
          (2, 2880, 2880, 8, 8), (8, 8192, 64, 256, 8), (1, 4096, 1024, 4, 4), (7, 264, 1040, 16, 4),
          (4, 16, 65536, 2, 1), (6, 2048, 768, 128, 8), (1, 7168, 2048, 16, 8), (8, 1024, 72, 3, 1)]


@pytest.mark.parametrize("tokens, hidden, inter, experts, top_k", SHAPES)
@pytest.mark.parametrize("router", [torch.bfloat16, torch.float32])
def test_bf16_weights(cuda_device, tokens, hidden, inter, experts, top_k, router) -> None:
    x, r, gate_up, down = _inputs(cuda_device, tokens, hidden, inter, experts, router)
    out, ids, weights = b300_moe_layer(x, r, gate_up, down, num_experts=experts, top_k=top_k,
                                       return_routing=True, check_status=True)
    want_ids, want_weights = _route(x, r, top_k)
    assert ids.dtype is torch.int64 and torch.equal(ids, want_ids)
    assert weights.dtype is torch.float32
    assert float((weights.double() - want_weights).abs().max()) <= 2.0 ** -21
    _check(out, *_formula(x, lambda e: gate_up[e].double(), lambda e: down[e].double(), ids,
                          want_weights))
    alone = b300_moe_layer(x, r, gate_up, down, num_experts=experts, top_k=top_k)
    assert torch.equal(alone, out)


@pytest.mark.parametrize("tokens, hidden, inter, experts, top_k",
                         [s for s in SHAPES if s[1] % 16 == 0 and s[2] % 16 == 0])
def test_fp8_weights(cuda_device, tokens, hidden, inter, experts, top_k) -> None:
    x, r, gate_up, down = _inputs(cuda_device, tokens, hidden, inter, experts)
    fw = quantize_expert_weights_fp8(gate_up, down)
    out, ids, _ = b300_moe_layer_fp8(x, r, fw, num_experts=experts, top_k=top_k,
                                     return_routing=True, check_status=True)
    want_ids, want_weights = _route(x, r, top_k)
    assert torch.equal(ids, want_ids)

    def matrix(q, scale):
        return lambda e: q[e].view(torch.float8_e4m3fn).double() * scale[e].double()[:, None]

    _check(out, *_formula(x, matrix(fw.gate_up_q, fw.gate_up_scale),
                          matrix(fw.down_q, fw.down_scale), ids, want_weights, fp8=True))


def test_every_token_count_agrees_with_the_regular_path(cuda_device) -> None:
    """Same routing into b300_moe_forward: both round the same FP32-accurate sum to BF16, and the
    regular path's routing weights are BF16 too (2^-8), which bounds each expert's share."""

    x, r, gate_up, down = _inputs(cuda_device, 8, 512, 256, 32)
    for tokens in range(1, 9):
        xt = x[:tokens].contiguous()
        out, ids, weights = b300_moe_layer(xt, r, gate_up, down, num_experts=32, top_k=4,
                                           return_routing=True)
        rounded = weights.bfloat16()
        other = b300_moe_forward(xt, ids, rounded, gate_up, down, num_experts=32, top_k=4)
        matrices = (lambda e: gate_up[e].double(), lambda e: down[e].double(), ids)
        want, bound = _formula(xt, *matrices, weights.double())
        _check(out, want, bound)
        want, bound = _formula(xt, *matrices, rounded.double())
        # chains of the other path are of the same length at most; its tiles are 64 wide too
        _check(other, want, 2 * bound)
        few = b300_moe_layer(x, r, gate_up, down, num_experts=32, top_k=4)[:tokens]
        want8, bound8 = _formula(xt, *matrices, weights.double())
        _check(few, want8, 2 * bound8)


def test_neighbouring_logits_are_told_apart(cuda_device) -> None:
    """Two experts whose router rows differ in the last bit of one FP32 element: their logits
    differ by less than FP32 sums resolve, and the larger one has to win wherever it stands."""

    hidden = 4096
    x, r, gate_up, down = _inputs(cuda_device, 4, hidden, 64, 6, torch.float32)
    for low, high in ((1, 4), (4, 1)):
        r[high] = r[low] + 3 * x[0].float() / hidden  # token 0's favourites
        r[low] = r[high]
        at = int(x[0].float().abs().argmax())
        up = r[low, at].nextafter(torch.tensor(math.inf * float(x[0, at].sign()), device=cuda_device))
        r[high, at] = up
        want, _ = _route(x, r, 1)
        assert int(want[0]) == high
        _, ids, _ = b300_moe_layer(x, r, gate_up, down, num_experts=6, top_k=1, return_routing=True)
        assert torch.equal(ids, want)


def test_equal_logits_go_to_the_lower_ids(cuda_device) -> None:
    x, r, gate_up, down = _inputs(cuda_device, 3, 128, 64, 40)
    r[:] = r[7]
    out, ids, weights = b300_moe_layer(x, r, gate_up, down, num_experts=40, top_k=4,
                                       return_routing=True)
    assert torch.equal(ids.cpu(), torch.arange(4).repeat(3, 1))
    assert torch.equal(weights, torch.full_like(weights, 0.25))
    x0 = torch.zeros_like(x)  # all logits 0, activations 0
    out, ids, _ = b300_moe_layer(x0, r, gate_up, down, num_experts=40, top_k=4, return_routing=True)
    assert torch.equal(ids.cpu(), torch.arange(4).repeat(3, 1)) and bool((out == 0).all())
    again, same = topk_routing((x0.float() @ r.float().T), 4)[0], ids
    assert torch.equal(again, same)


@pytest.mark.parametrize("fp8", [False, True])
def test_non_finite_values_stay_with_their_token(cuda_device, fp8) -> None:
    x, r, gate_up, down = _inputs(cuda_device, 8, 256, 320, 16)

    def run(x, gate_up, down):
        if fp8:
            return b300_moe_layer_fp8(x, r, gate_up, num_experts=16, top_k=2, return_routing=True)
        return b300_moe_layer(x, r, gate_up, down, num_experts=16, top_k=2, return_routing=True)

    weights = quantize_expert_weights_fp8(gate_up, down) if fp8 else gate_up
    clean, ids, _ = run(x, weights, down)
    bad = x.clone()
    bad[3, 100] = float("nan")
    bad[5] = float("inf")
    out, bad_ids, _ = run(bad, weights, down)
    rest = [t for t in range(8) if t not in (3, 5)]
    # tokens 3 and 5 may pull other experts into the call, which changes the order of the sums
    want, bound = _formula(
        x, (lambda e: weights.gate_up_q[e].view(torch.float8_e4m3fn).double()
            * weights.gate_up_scale[e].double()[:, None]) if fp8 else (lambda e: gate_up[e].double()),
        (lambda e: weights.down_q[e].view(torch.float8_e4m3fn).double()
         * weights.down_scale[e].double()[:, None]) if fp8 else (lambda e: down[e].double()),
        ids, _route(x, r, 2)[1], fp8)
    _check(out[rest], want[rest], 2 * bound[rest])
    assert bool(out[3].isnan().all()) and bool(out[5].isnan().all())
    assert torch.equal(bad_ids[rest], ids[rest])
    assert torch.equal(bad_ids[3].cpu(), torch.tensor([0, 1]))  # NaN logits: all equal, lower ids

    # an expert whose weights are not numbers reaches the tokens routed to it and no other
    e = int(ids[0, 0])
    hit = (ids == e).any(-1)
    assert bool(hit.any()) and not bool(hit.all())
    if fp8:
        import dataclasses
        scale = weights.down_scale.clone()
        scale[e] = float("nan")
        out, _, _ = run(x, dataclasses.replace(weights, down_scale=scale), down)
    else:
        broken, broken_down = gate_up.clone(), down.clone()
        broken[e, 0], broken_down[e] = float("inf"), float("nan")
        out, _, _ = run(x, broken, broken_down)
    assert torch.equal(out[~hit], clean[~hit])
    assert bool(out[hit].isnan().all())


def test_repeated_calls_are_bitwise_equal_and_share_the_workspace(cuda_device) -> None:
    x, r, gate_up, down = _inputs(cuda_device, 8, 512, 256, 16)
    ws = B300MoEWorkspace(8, device=cuda_device)
    options = dict(num_experts=16, top_k=2, workspace=ws)
    first = b300_moe_layer(x, r, gate_up, down, **options)
    ids, weights = topk_routing(x.float() @ r.float().T, 2)
    forward = b300_moe_forward(x, ids, weights.bfloat16(), gate_up, down, **options)
    for i in range(20):
        tokens = 1 + i % 8
        few = b300_moe_layer(x[:tokens].contiguous(), r, gate_up, down, **options)
        assert few.shape == (tokens, 512)
        assert torch.equal(b300_moe_layer(x, r, gate_up, down, **options), first)
        assert torch.equal(b300_moe_forward(x, ids, weights.bfloat16(), gate_up, down, **options),
                           forward)
    assert ws.allocation_count == 1 and ws.status() == 0
    # the counters between the status word and the end of its 256 bytes are back at zero
    assert int(ws.scratch[192:256].view(torch.int32).abs().sum()) == 0


def test_out_and_in_place(cuda_device) -> None:
    x, r, gate_up, down = _inputs(cuda_device, 4, 256, 128, 8)
    ws = B300MoEWorkspace(4, device=cuda_device)
    options = dict(num_experts=8, top_k=2, workspace=ws)
    want = b300_moe_layer(x, r, gate_up, down, **options)
    out = torch.empty_like(x)
    assert b300_moe_layer(x, r, gate_up, down, out=out, **options) is out and torch.equal(out, want)
    b300_moe_layer(x, r, gate_up, down, out=x, **options)
    assert torch.equal(x, want)
    with pytest.raises(ValueError, match="on the inputs' device"):
        b300_moe_layer(x, r, gate_up, down, out=torch.empty(4, 256, dtype=torch.bfloat16).pin_memory(),
                       **options)
    with pytest.raises(ValueError, match="same device"):
        b300_moe_layer(x, r.cpu(), gate_up, down, **options)


def test_streams_and_graphs(cuda_device) -> None:
    x, r, gate_up, down = _inputs(cuda_device, 3, 512, 256, 16)
    y = _inputs(cuda_device, 3, 512, 256, 16, seed=12)[0]
    ws = B300MoEWorkspace(3, device=cuda_device)
    options = dict(num_experts=16, top_k=4, workspace=ws)
    want_x = b300_moe_layer(x, r, gate_up, down, **options)
    want_y = b300_moe_layer(y, r, gate_up, down, **options)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the workspace orders the two streams
        got = [b300_moe_layer(y, r, gate_up, down, **options) for _ in range(3)]
    got.append(b300_moe_layer(x, r, gate_up, down, **options))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want_y) for g in got[:3]) and torch.equal(got[3], want_x)

    held = x.clone()
    graphs, outs = [], []
    for _ in range(2):  # two graphs over one workspace, replayed one after the other
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(b300_moe_layer(held, r, gate_up, down, **options))
        graphs.append(graph)
    for source, want in ((x, want_x), (y, want_y), (x, want_x)):
        held.copy_(source)
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="capture"):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b300_moe_layer(held, r, gate_up, down, num_experts=16, top_k=4)
    assert torch.equal(b300_moe_layer(x, r, gate_up, down, **options), want_x)


def test_a_workspace_reserved_on_a_busy_stream_is_used_on_another(cuda_device) -> None:
    """The clearing of the workspace's status area is queued behind other work; the first call, on
    another stream, waits for it."""

    x, r, gate_up, down = _inputs(cuda_device, 2, 256, 128, 8)
    want = b300_moe_layer(x, r, gate_up, down, num_experts=8, top_k=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    junk = torch.full((1 << 20,), 255, dtype=torch.uint8, device=cuda_device)
    del junk  # so that the workspace may get memory that is not zero
    ws = B300MoEWorkspace(2, device=cuda_device)
    torch.cuda._sleep(20_000_000)  # about 10 ms
    ws.reserve(num_tokens=2, num_experts=8, top_k=2, hidden_size=256, intermediate_size=128,
               device=cuda_device, dtype=torch.bfloat16, backend="b200_bf16", quant_mode="bf16")
    with torch.cuda.stream(side):
        got = b300_moe_layer(x, r, gate_up, down, num_experts=8, top_k=2, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and ws.status() == 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tokens, hidden, inter, experts, top_k",
                         [(8, 4736, 144, 8, 4), (5, 4752, 208, 16, 8), (8, 8192, 80, 8, 2),
                          (3, 2368, 272, 4, 2), (4, 2384, 48, 32, 8), (2, 144, 16, 4, 1)])
def test_output_rows_of_a_block(cuda_device, tokens, hidden, inter, experts, top_k, fp8) -> None:
    """Both sides of 16, 32 and 48 output rows a block, and expert widths that end inside a run of
    64 activations."""
    x, r, gate_up, down = _inputs(cuda_device, tokens, hidden, inter, experts)
    want_ids, want_weights = _route(x, r, top_k)
    if fp8:
        fw = quantize_expert_weights_fp8(gate_up, down)
        out, ids, _ = b300_moe_layer_fp8(x, r, fw, num_experts=experts, top_k=top_k,
                                         return_routing=True, check_status=True)

        def matrix(q, scale):
            return lambda e: q[e].view(torch.float8_e4m3fn).double() * scale[e].double()[:, None]

        gate_up_of, down_of = (matrix(fw.gate_up_q, fw.gate_up_scale),
                               matrix(fw.down_q, fw.down_scale))
    else:
        out, ids, _ = b300_moe_layer(x, r, gate_up, down, num_experts=experts, top_k=top_k,
                                     return_routing=True, check_status=True)
        gate_up_of, down_of = (lambda e: gate_up[e].double()), (lambda e: down[e].double())
    assert torch.equal(ids, want_ids)
    _check(out, *_formula(x, gate_up_of, down_of, ids, want_weights, fp8=fp8))
