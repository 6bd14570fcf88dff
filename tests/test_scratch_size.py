"""Bytes of scratch: the one-kernel layer works in the bytes of the staged forward and asks for none
of its own, wherever the forward's are enough (sizes of the forward alone, in bytes)."""

from __future__ import annotations

import pytest

from b200moe import _lib

FORWARD = [((1, 2, 8, 4096, 14336), 406784), ((64, 2, 8, 4096, 14336), 25954560),
           ((64, 8, 128, 2048, 768), 37495808), ((1, 8, 128, 2048, 768), 587008),
           ((8, 8, 32, 2880, 2880), 6821632), ((64, 4, 32, 2880, 2880), 27283712),
           ((8, 8, 256, 7168, 2048), 16320768), ((1, 1, 2, 16, 65536), 329472),
           ((512, 1, 4, 64, 96), 1301504), ((3, 2, 4, 72, 200), 21504)]


@pytest.mark.parametrize("shape, size", FORWARD)
def test_scratch_of_the_forward_is_enough_for_the_layer(shape, size) -> None:
    assert _lib.scratch_bytes(*shape) == size


def test_the_layers_scratch_fits_the_smallest_shapes() -> None:
    """[T, E] FP64 logits, 64 maxima and [T K, I to whole 64] words behind the schedule."""

    for tokens, top_k, experts, hidden, inter in ((1, 1, 1, 8, 8), (1, 8, 256, 8, 8), (8, 8, 256, 8, 8)):
        need = 256 + 64 * experts + 256 + min(tokens * top_k, 64) * (-(-inter // 64) * 64) * 4
        assert _lib.scratch_bytes(tokens, top_k, experts, hidden, inter) >= need
