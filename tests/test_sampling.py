"""Refusals of the sampler's entry points; they answer before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch

from b200moe import sample_tokens


def _call(logits=None, uniforms=None, **options):
    logits = torch.zeros(3, 10) if logits is None else logits
    uniforms = torch.zeros(3) if uniforms is None else uniforms
    return sample_tokens(logits, uniforms, **options)


@pytest.mark.parametrize(
    "options, error, match",
    [
        ({"logits": [0.0]}, TypeError, "torch.Tensors"),
        ({"uniforms": 0.5}, TypeError, "torch.Tensors"),
        ({"logits": torch.zeros(10)}, ValueError, "num_rows, vocab"),
        ({"logits": torch.zeros(0, 10)}, ValueError, "at least one"),
        ({"logits": torch.zeros(3, 0)}, ValueError, "at least one"),
        ({"logits": torch.zeros(1, 262145)}, ValueError, "at most"),
        ({"logits": torch.zeros(1048577, 1)}, ValueError, "at most"),
        ({"logits": torch.zeros(3, 10, dtype=torch.float16)}, TypeError, "float32 and bfloat16"),
        ({"logits": torch.zeros(3, 20)[:, ::2]}, ValueError, "contiguous"),
        ({"logits": torch.zeros(10).expand(3, 10)}, ValueError, "contiguous"),
        ({"uniforms": torch.zeros(3).double()}, TypeError, "uniforms"),
        ({"uniforms": torch.zeros(4)}, ValueError, "uniforms"),
        ({"uniforms": torch.zeros(6)[::2]}, ValueError, "uniforms"),
        ({"logits": torch.zeros(3, 10, requires_grad=True)}, ValueError, "autograd"),
        ({"temperature": -0.1}, ValueError, "temperature"),
        ({"temperature": float("nan")}, ValueError, "temperature"),
        ({"temperature": float("inf")}, ValueError, "temperature"),
        ({"temperature": True}, TypeError, "temperature"),
        ({"temperature": torch.ones(3).double()}, TypeError, "temperature"),
        ({"temperature": torch.ones(2)}, ValueError, "temperature"),
        ({"top_p": 1.5}, ValueError, "top_p"),
        ({"top_p": "1"}, TypeError, "top_p"),
        ({"min_p": -0.5}, ValueError, "min_p"),
        ({"min_p": torch.ones(3, 1)}, ValueError, "min_p"),
        ({"top_k": -1}, ValueError, "top_k"),
        ({"top_k": 2.0}, TypeError, "top_k"),
        ({"top_k": torch.ones(3, dtype=torch.int64)}, TypeError, "top_k"),
        ({"top_k": torch.ones(2, dtype=torch.int32)}, ValueError, "top_k"),
        ({"return_logprobs": 1}, TypeError, "return_logprobs"),
        ({"out": torch.zeros(3)}, ValueError, "out must be"),
        ({"out": 1}, TypeError, "out must be"),
        ({}, ValueError, "requires CUDA"),
    ],
)
def test_bad_arguments_are_refused(options, error, match) -> None:
    with pytest.raises(error, match=match):
        _call(**options)


def test_c_entry_checks_its_arguments() -> None:
    from b200moe import _lib

    fn = _lib.load().b200moe_sample
    p = ctypes.c_void_p(4096)

    def call(logits=p, f32=1, stride=16, rows=2, vocab=16, uniforms=p, ids=p):
        return fn(logits, f32, stride, rows, vocab, uniforms, None, 1.0, None, 0, None, 1.0, None,
                  0.0, ids, None, None)

    assert call(logits=None) == call(uniforms=None) == call(ids=None) == -1
    assert call(rows=0) == call(vocab=0) == call(stride=15) == -2
    assert call(rows=1048577) == call(vocab=262145, stride=262145) == -8
    assert call(logits=ctypes.c_void_p(4098)) == call(logits=ctypes.c_void_p(4097), f32=0) == -3


@pytest.mark.parametrize("shared", ["logits", "uniforms", "temperature", "top_k", "top_p", "min_p"])
def test_out_may_not_overlap_an_input(shared) -> None:
    rows, vocab = 4, 16
    held = torch.zeros(rows * vocab)
    ids = held.view(torch.int64)[:rows]
    inputs = {"logits": torch.zeros(rows, vocab), "uniforms": torch.zeros(rows)}
    part = held.view(rows, vocab) if shared == "logits" else held[2 * rows - 1:3 * rows - 1]
    inputs[shared] = part.view(torch.int32) if shared == "top_k" else part
    with pytest.raises(ValueError, match="must not overlap an input"):
        sample_tokens(inputs.pop("logits"), inputs.pop("uniforms"), out=ids, **inputs)


def test_out_next_to_the_inputs_is_taken() -> None:
    held = torch.zeros(4 + 8 + 4 + 64)
    with pytest.raises(ValueError, match="requires CUDA"):  # all other checks have passed
        sample_tokens(held[16:].view(4, 16), held[:4], temperature=held[12:16],
                      out=held[4:12].view(torch.int64))
