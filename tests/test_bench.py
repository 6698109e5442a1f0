"""The benchmark's legs that run the reference's own code, where the reference is not installed."""

from __future__ import annotations

import sys

import pytest

import bench


@pytest.mark.parametrize("leg", [bench.run_decoder_layer, bench.run_engine])
def test_a_leg_without_the_reference_says_so(leg, monkeypatch) -> None:
    for name in [n for n in sys.modules if n.split(".")[0] == "mxwave"]:
        monkeypatch.delitem(sys.modules, name)
    monkeypatch.setitem(sys.modules, "mxwave", None)  # an import of it fails
    assert "not installed" in leg(None, None)["unavailable"]
