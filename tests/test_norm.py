"""Refusals of the residual norm's entry points; they answer before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch

from b200moe import add_rms_norm, add_rms_norm_fp8


def _inputs(rows=3, hidden=32, residual=torch.bfloat16, weight=torch.bfloat16):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(rows, hidden, generator=g).bfloat16()
    r = None if residual is None else torch.randn(rows, hidden, generator=g).to(residual)
    return [x, r, torch.ones(hidden, dtype=weight)]


@pytest.mark.parametrize("fn", [add_rms_norm, add_rms_norm_fp8])
@pytest.mark.parametrize(
    "change, error, match",
    [
        (lambda a: a.__setitem__(0, None), TypeError, "hidden_states must be a torch.Tensor"),
        (lambda a: a.__setitem__(1, 1.0), TypeError, "residual must be"),
        (lambda a: a.__setitem__(2, [1.0]), TypeError, "weight must be"),
        (lambda a: a.__setitem__(0, torch.zeros((), dtype=torch.bfloat16)), ValueError, "hidden_size"),
        (lambda a: a.__setitem__(2, a[2][:16].clone()), ValueError, "weight must have shape"),
        (lambda a: a.__setitem__(1, a[1][:2].clone()), ValueError, "same shape"),
        (lambda a: a.__setitem__(0, a[0].float()), TypeError, "bfloat16"),
        (lambda a: a.__setitem__(1, a[1].half()), TypeError, "bfloat16 or torch.float32"),
        (lambda a: a.__setitem__(2, a[2].double()), TypeError, "bfloat16 or torch.float32"),
        (lambda a: a.__setitem__(0, a[0].t().contiguous().t()), ValueError, "contiguous"),
        (lambda a: a.__setitem__(1, a[1].requires_grad_()), ValueError, "autograd"),
    ],
)
def test_bad_inputs_are_refused(fn, change, error, match) -> None:
    args = _inputs()
    change(args)
    with pytest.raises(error, match=match):
        fn(*args)


@pytest.mark.parametrize("eps, error", [(None, TypeError), (True, TypeError), (-1e-6, ValueError),
                                        (float("nan"), ValueError), (float("inf"), ValueError)])
def test_bad_eps_is_refused(eps, error) -> None:
    with pytest.raises(error, match="eps"):
        add_rms_norm(*_inputs(), eps=eps)


def test_hidden_sizes_outside_the_range_are_refused() -> None:
    for fn, hidden in ((add_rms_norm, 36), (add_rms_norm_fp8, 24), (add_rms_norm, 32776),
                       (add_rms_norm_fp8, 32784), (add_rms_norm, 0)):
        with pytest.raises(ValueError, match="hidden_size must be a multiple"):
            fn(*_inputs(hidden=hidden))


def test_cpu_tensors_are_refused() -> None:
    with pytest.raises(ValueError, match="requires CUDA"):
        add_rms_norm(*_inputs())
    with pytest.raises(ValueError, match="requires CUDA"):
        add_rms_norm_fp8(*_inputs(residual=None))


def test_c_entry_checks_its_arguments() -> None:
    from b200moe import _lib

    fn = _lib.load().b200moe_add_rms_norm
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)

    def call(hidden=p, residual=p, weight=p, rows=1, size=64, eps=1e-6, out=p, codes=None,
             scale=None, residual_out=p):
        return fn(hidden, residual, 0, weight, 0, rows, size, eps, out, codes, scale,
                  residual_out, None)

    assert call(hidden=None) == call(weight=None) == call(out=None) == -1
    assert call(codes=p, scale=p) == call(out=None, codes=p) == -1   # both results; no scale
    assert call(residual=None) == call(residual_out=None) == -1
    assert call(rows=0) == call(size=0) == call(size=32776) == call(eps=-1.0) == -2
    assert call(eps=float("nan")) == -2
    assert call(size=60) == call(out=None, codes=p, scale=p, size=72) == -3
    assert call(hidden=odd) == call(residual=odd) == call(weight=odd) == call(out=odd) == -3
    assert call(residual_out=odd) == -3
