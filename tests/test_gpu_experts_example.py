"""The example of a routed layer runs its whole way, with the router's choice, affine experts
and a single token in two launches."""

from __future__ import annotations

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def test_the_example_runs():
    path = os.path.join(os.path.dirname(__file__), "..", "examples", "experts_forward.py")
    spec = importlib.util.spec_from_file_location("experts_forward", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    e = mod.main(["--experts", "6", "--hidden", "128", "--inter", "64", "--tokens", "50", "--top-k", "3"])
    assert {"mxfp4 solved", "affine nearest", "int8 nearest", "single token"} <= set(e)
    assert all(v == v for v in e.values())
