"""CPU: the bench's line does not need the compiled reference."""
import argparse

import pytest

import bench
from oracle import bind


@pytest.mark.parametrize("built,off,want", [(True, False, True), (True, True, False), (False, False, False),
                                            (False, True, False)])
def test_cpu_baseline_only_where_the_reference_was_built(monkeypatch, built, off, want):
    monkeypatch.setattr(bind, "reference_available", lambda: built)
    assert bench.times_cpu_baseline(argparse.Namespace(no_cpu_baseline=off)) is want
