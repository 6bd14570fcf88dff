"""The operators of a decode step in a row, as a model with expert layers runs them: residual
norm, router and experts, residual norm, head, sampling -- eagerly and as one captured graph,
against the same chain in 64 bits.

Tolerances are those of the single operators: the head's logits are compared within the BF16
roundings of the norms, the layers and the head (2^-8 each, relative to the row's norm: the chain
has no larger factor than 1), the token against the definition on the logits that the sampler was
given.  Which experts a token gets is no continuous function of its row, so the chain in 64 bits
takes the experts that the layer took, and those are compared with the top-k of the very rows that
the layer was given.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from b200moe import (B300MoEWorkspace, add_rms_norm, add_rms_norm_fp8, b300_moe_forward,
                     b300_moe_layer, b300_moe_layer_fp8, dequantize_rows_fp8,
                     quantize_expert_weights_fp8, sample_tokens, topk_routing)

pytestmark = pytest.mark.gpu

H, I, E, K, V = 512, 256, 16, 4, 5003


def _model(device, layers=3, seed=31):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, std):
        return torch.empty(*shape, device=device, dtype=torch.bfloat16).normal_(0, std, generator=g)

    return {
        "norms": [1 + normal(H, std=0.1) for _ in range(layers + 1)],
        "routers": [normal(E, H, std=H ** -0.5) for _ in range(layers)],
        "gate_up": [normal(E, 2 * I, H, std=H ** -0.5) for _ in range(layers)],
        "down": [normal(E, H, I, std=I ** -0.5) for _ in range(layers)],
        "head": normal(V, H, std=3 * H ** -0.5),
        "generator": g,
    }


def _step(m, x, u, workspace, fp8=None, trace=None):
    """(tokens, logits): x [T,H] in, an FP32 residual stream inside.  ``trace`` collects the rows
    and the experts of every layer."""

    residual = x.float()
    normed, _ = add_rms_norm(x, None, m["norms"][0])
    for layer, router in enumerate(m["routers"]):
        options = dict(num_experts=E, top_k=K, workspace=workspace,
                       return_routing=trace is not None)
        if fp8 is None:
            out = b300_moe_layer(normed, router, m["gate_up"][layer], m["down"][layer], **options)
        else:
            out = b300_moe_layer_fp8(normed, router, fp8[layer], **options)
        if trace is not None:
            out, ids, _ = out
            trace.append((normed, ids))
        normed, residual = add_rms_norm(out, residual, m["norms"][layer + 1])
    logits = normed @ m["head"].T
    return sample_tokens(logits, u, temperature=0.8, top_k=200, top_p=0.9), logits


def _top(rows, router):
    logits = (rows.double()[:, None] * router.double()[None]).sum(-1)
    return torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :K]


def _chain(m, x, chosen, fp8=None):
    """The logits in 64 bits, with the experts that were chosen."""

    def norm(s, w):
        return s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()

    residual = x.double()
    normed = norm(residual, m["norms"][0])
    for layer, router in enumerate(m["routers"]):
        ids = chosen[layer]
        p = torch.softmax((normed @ router.double().T).gather(1, ids), -1)
        out = torch.zeros_like(residual)
        for t in range(x.shape[0]):
            for k in range(K):
                e = int(ids[t, k])
                if fp8 is None:
                    gu, dn = m["gate_up"][layer][e].double(), m["down"][layer][e].double()
                else:
                    f = fp8[layer]
                    gu = f.gate_up_q[e].view(torch.float8_e4m3fn).double() * f.gate_up_scale[e].double()[:, None]
                    dn = f.down_q[e].view(torch.float8_e4m3fn).double() * f.down_scale[e].double()[:, None]
                gate, up = (gu @ normed[t]).chunk(2)
                out[t] += p[t, k] * (dn @ (gate * torch.sigmoid(gate) * up))
        residual = residual + out
        normed = norm(residual, m["norms"][layer + 1])
    return normed @ m["head"].double().T


def _token(logits, u):
    x = logits.double().cpu().numpy()
    order = np.argsort(-x, kind="stable")[:200]
    w = np.exp((x[order] - x.max()) / float(np.float32(0.8)))
    count = int(np.searchsorted(np.cumsum(w), float(np.float32(0.9)) * w.sum())) + 1
    order, w = order[:count], w[:count]
    place = np.argsort(order)
    order, upto = order[place], np.cumsum(w[place])
    return int(order[min(int(np.searchsorted(upto, u * upto[-1], side="right")), count - 1)])


@pytest.mark.parametrize("tokens", [1, 5, 8])
@pytest.mark.parametrize("quantised", [False, True])
def test_decode_step(cuda_device, tokens, quantised) -> None:
    m = _model(cuda_device)
    fp8 = [quantize_expert_weights_fp8(a, b) for a, b in zip(m["gate_up"], m["down"])] \
        if quantised else None
    workspace = B300MoEWorkspace(8, device=cuda_device)
    g = m["generator"]

    def inputs():
        return (torch.empty(tokens, H, device=cuda_device, dtype=torch.bfloat16).normal_(generator=g),
                torch.rand(tokens, device=cuda_device, generator=g))

    x, u = inputs()
    trace: list = []
    ids, logits = _step(m, x, u, workspace, fp8, trace)
    for (rows, chosen), router in zip(trace, m["routers"]):
        assert torch.equal(chosen, _top(rows, router))
    want = _chain(m, x, [chosen for _, chosen in trace], fp8)
    # 3 layers: 4 norms, 3 layer outputs and the head's own rounding
    off = (logits.double() - want).norm(dim=-1) / want.norm(dim=-1)
    assert float(off.max()) <= 8 * 2.0 ** -8
    assert ids.tolist() == [_token(r, float(v)) for r, v in zip(logits, u)]

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_logits = _step(m, x, u, workspace, fp8)
    for _ in range(4):
        x2, u2 = inputs()
        want_ids, want_logits = _step(m, x2, u2, workspace, fp8)
        x.copy_(x2)
        u.copy_(u2)
        graph.replay()
        assert torch.equal(got, want_ids) and torch.equal(got_logits, want_logits)
    assert workspace.status() == 0 and workspace.allocation_count == 1


def test_two_steps_at_once_on_two_streams(cuda_device) -> None:
    """Each stream with a workspace of its own: the cooperative launches may wait for one another,
    results stay what they are alone."""

    m = _model(cuda_device)
    spaces = [B300MoEWorkspace(8, device=cuda_device) for _ in range(2)]
    g = m["generator"]
    xs = [torch.empty(4, H, device=cuda_device, dtype=torch.bfloat16).normal_(generator=g) for _ in range(2)]
    u = torch.rand(4, device=cuda_device, generator=g)
    want = [_step(m, x, u, spaces[0]) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_step(m, xs[i], u, spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])
        assert spaces[i].status() == 0


def test_the_regular_path_takes_what_the_few_token_path_gives(cuda_device) -> None:
    """Nine tokens: the norm's rows go to topk_routing and b300_moe_forward, on a workspace that
    the one-kernel layer uses for eight of them; both agree within the BF16 routing weights."""

    m = _model(cuda_device, layers=1)
    g = m["generator"]
    workspace = B300MoEWorkspace(9, device=cuda_device)
    x = torch.empty(9, H, device=cuda_device, dtype=torch.bfloat16).normal_(generator=g)
    normed, _ = add_rms_norm(x, None, m["norms"][0])
    options = dict(num_experts=E, top_k=K, workspace=workspace)
    few, ids8, _ = b300_moe_layer(normed[:8], m["routers"][0], m["gate_up"][0], m["down"][0],
                                  return_routing=True, **options)
    ids, weights = topk_routing(normed.float() @ m["routers"][0].float().T, K)
    out = b300_moe_forward(normed, ids, weights.bfloat16(), m["gate_up"][0], m["down"][0], **options)
    assert torch.equal(ids[:8], ids8)
    off = (few.double() - out[:8].double()).norm(dim=-1) / out[:8].double().norm(dim=-1)
    assert float(off.max()) <= 3 * 2.0 ** -8  # two results and the weights, each rounded once
    codes, scale, _ = add_rms_norm_fp8(x, None, m["norms"][0])
    back = dequantize_rows_fp8(codes, scale)
    off = (back.double() - normed.double()).norm(dim=-1) / normed.double().norm(dim=-1)
    assert float(off.max()) <= 2.0 ** -4 + 2 * 2.0 ** -8
