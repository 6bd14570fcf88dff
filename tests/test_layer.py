"""Refusals of the one-kernel layer's entry points; they answer before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch

from b200moe import B300MoEWorkspace, Fp8ExpertWeights, b300_moe_layer, b300_moe_layer_fp8


def _inputs(tokens=2, hidden=32, inter=48, experts=8):
    bf16 = torch.bfloat16
    return [torch.zeros(tokens, hidden, dtype=bf16), torch.zeros(experts, hidden, dtype=bf16),
            torch.zeros(experts, 2 * inter, hidden, dtype=bf16),
            torch.zeros(experts, hidden, inter, dtype=bf16)]


def _fp8(hidden=32, inter=48, experts=8):
    return Fp8ExpertWeights(torch.zeros(experts, 2 * inter, hidden, dtype=torch.uint8),
                            torch.ones(experts, 2 * inter),
                            torch.zeros(experts, hidden, inter, dtype=torch.uint8),
                            torch.ones(experts, hidden))


def _call(args, **options):
    options = {"num_experts": 8, "top_k": 2, **options}
    return b300_moe_layer(*args, **options)


def _replace(i, make):
    def change(args):
        args[i] = make(args[i])
    return change


@pytest.mark.parametrize(
    "change, error, match",
    [
        (_replace(0, lambda t: None), TypeError, "hidden_states must be a torch.Tensor"),
        (_replace(1, lambda t: 0), TypeError, "router_weight must be a torch.Tensor"),
        (_replace(0, lambda t: t[0]), ValueError, "num_tokens, hidden_size"),
        (_replace(0, lambda t: t[:0]), ValueError, "num_tokens, hidden_size"),
        (_replace(0, lambda t: t.repeat(5, 1)), ValueError, "at most 8 tokens"),
        (_replace(1, lambda t: t[:7]), ValueError, "router_weight must have shape"),
        (_replace(1, lambda t: t.t().contiguous()), ValueError, "router_weight must have shape"),
        (_replace(2, lambda t: t[:7]), ValueError, r"\[E, 2I, H\]"),
        (_replace(2, lambda t: t[:, :95]), ValueError, r"\[E, 2I, H\]"),
        (_replace(3, lambda t: t[:, :, :40]), ValueError, r"\[E, H, I\]"),
        (_replace(0, lambda t: t.float()), TypeError, "hidden_states must have dtype"),
        (_replace(1, lambda t: t.half()), TypeError, "router_weight must have dtype"),
        (_replace(2, lambda t: t.float()), TypeError, "must have dtype torch.bfloat16"),
        (_replace(0, lambda t: t.t().contiguous().t()), ValueError, "contiguous"),
        (_replace(1, lambda t: t.requires_grad_()), ValueError, "autograd"),
    ],
)
def test_bad_inputs_are_refused(change, error, match) -> None:
    args = _inputs()
    change(args)
    with pytest.raises(error, match=match):
        _call(args)


def test_bad_options_are_refused() -> None:
    for options, error, match in (
        ({"top_k": 3}, ValueError, "top_k must be one of"),
        ({"top_k": True}, TypeError, "top_k"),
        ({"num_experts": 4, "top_k": 8}, ValueError, "must not exceed"),
        ({"num_experts": 257}, ValueError, "at most 256"),
        ({"num_experts": 7}, ValueError, "router_weight must have shape"),
        ({"return_routing": 1}, TypeError, "return_routing"),
        ({"check_status": None}, TypeError, "check_status"),
        ({"out": 3}, TypeError, "out must be"),
        ({"out": torch.zeros(2, 32)}, ValueError, "out must be"),
        ({"workspace": 1}, TypeError, "workspace must be"),
    ):
        with pytest.raises(error, match=match):
            _call(_inputs(), **options)
    with pytest.raises(ValueError, match="divisible by 8"):
        _call(_inputs(hidden=36))
    with pytest.raises(ValueError, match="divisible by 8"):
        _call(_inputs(inter=44))
    with pytest.raises(ValueError, match="hidden_size up to 8192"):
        _call(_inputs(hidden=8200, inter=8))
    with pytest.raises(ValueError, match="intermediate_size up to 65536"):
        _call(_inputs(hidden=8, inter=65544, experts=2), num_experts=2)


def test_cpu_tensors_are_refused_and_leave_the_workspace_alone() -> None:
    workspace = B300MoEWorkspace(2)
    with pytest.raises(ValueError, match="requires CUDA"):
        _call(_inputs(), workspace=workspace)
    assert workspace.allocation_count == 0


def test_fp8_inputs_are_checked() -> None:
    x, router = _inputs()[:2]
    options = {"num_experts": 8, "top_k": 2}
    with pytest.raises(TypeError, match="Fp8ExpertWeights"):
        b300_moe_layer_fp8(x, router, None, **options)
    good = _fp8()
    for bad, error, match in (
        (Fp8ExpertWeights(good.gate_up_q.float(), good.gate_up_scale, good.down_q, good.down_scale),
         TypeError, "uint8"),
        (Fp8ExpertWeights(good.gate_up_q, good.gate_up_scale[:, :48], good.down_q, good.down_scale),
         ValueError, "scales"),
        (Fp8ExpertWeights(good.gate_up_q, good.gate_up_scale.half(), good.down_q, good.down_scale),
         TypeError, "scales"),
        (Fp8ExpertWeights(good.gate_up_q, good.gate_up_scale, good.down_q,
                          good.down_scale.t().contiguous().t()), ValueError, "contiguous"),
    ):
        with pytest.raises(error, match=match):
            b300_moe_layer_fp8(x, router, bad, **options)
    with pytest.raises(ValueError, match="divisible by 16"):
        b300_moe_layer_fp8(_inputs(hidden=40)[0], _inputs(hidden=40)[1], _fp8(hidden=40), **options)
    with pytest.raises(ValueError, match="requires CUDA"):
        b300_moe_layer_fp8(x, router, good, **options)


def test_c_entry_checks_its_arguments() -> None:
    from b200moe import _lib

    fn = _lib.load().b200moe_layer

    def call(router=4096, **fields):
        a = _lib.B200MoeArgs()
        values = dict(hidden_states=4096, gate_up_weight=4096, down_weight=4096, num_tokens=2,
                      top_k=2, num_experts=8, hidden_size=64, intermediate_size=64, rows_cap=4,
                      output=4096, scratch=4096, scratch_bytes=1 << 30)
        values.update(fields)
        for name, value in values.items():
            setattr(a, name, value)
        return fn(ctypes.byref(a), router, 0, None, None, None)

    assert fn(None, 4096, 0, None, None, None) == -1
    assert call(router=None) == call(hidden_states=None) == call(gate_up_weight=None) == -1
    assert call(output=None) == -1
    assert call(flags=_lib.FLAG_NVFP4_WEIGHTS) == call(flags=_lib.FLAG_LOCAL_EXPERTS) == -7
    assert call(num_tokens=9, rows_cap=18) == call(hidden_size=8200) == -8
    assert call(intermediate_size=65544) == -8
    assert call(top_k=3) == call(num_tokens=0) == call(num_experts=257) == call(rows_cap=3) == -2
    assert call(hidden_size=60) == -3
