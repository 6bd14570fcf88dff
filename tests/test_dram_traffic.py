"""The recorded DRAM traffic of the GEMMs belongs to the kernel sources as they are, so that the
benchmark reports it."""

from __future__ import annotations

import pytest

import bench


@pytest.mark.parametrize("key", ["gate_up_mixtral_T1_bf16", "gate_up_mixtral_T1_fp8",
                                 "gate_up_mixtral_T1_nvfp4"])
def test_recorded_traffic_is_of_these_sources(key) -> None:
    traffic, source = bench.measured_traffic(key)
    assert traffic is not None and traffic > 0, source
