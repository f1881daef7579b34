"""The cases of perf/more_operators.py, and some more of their ranges, against its definitions in 64 bits: the sizes at
which the operators for long contexts are timed take forms that small sizes do not."""
import importlib.util
import pathlib
import random

import numpy as np
import pytest

from _paged import U24
from _util import host
from jieyu_b200 import _capi

pytestmark = pytest.mark.gpu

_spec = importlib.util.spec_from_file_location(
    "more_operators", pathlib.Path(__file__).resolve().parent.parent / "perf" / "more_operators.py")
ops = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(ops)

CASES = ops.listed() + [dict(ops.draw(random.Random(seed)), name="drawn %d" % seed) for seed in range(12)]


def _run(case, own):
    ops.own = own
    try:
        return {name: host(x).copy() for name, x in ops.run(ops.prepare(case, 5)).items()}
    finally:
        ops.own = False


def _size(x):
    return np.sqrt(np.mean(np.square(x, dtype=np.float64)))


@pytest.mark.parametrize("case", CASES, ids=[c["name"] for c in CASES])
def test_case(cuda, case):
    lib = _capi.load()
    lib.jyc_paged_error(1)
    got = _run(case, True)
    assert lib.jyc_paged_error(1) == 0
    want = {name: x if isinstance(x, np.ndarray) else host(x) for name, x in ops.exact(case, 5).items()}
    assert sorted(got) == sorted(want)
    op = case["op"]
    if op in ("append", "evict"):  # stored bits, as the values they stand for, rounded once
        for name in want:
            assert np.array_equal(got[name], want[name].astype(got[name].dtype)), name
    elif op == "rope":
        # a product of at most the largest value of a head, and a sum of at most sqrt(2) times that, one rounding each;
        # (1 + 2^-20) for cosines and sines that are themselves rounded
        shape = (case["rows"], case["heads"], case["hd"])
        x = host(ops.prepare(case, 5)["x"]).reshape(shape)
        most = np.abs(x).max(-1, keepdims=True).astype(np.float64)
        err = np.abs(got["y"].reshape(shape) - want["y"].reshape(shape))
        assert np.all(err <= U24 * (1 + 2.0 ** 0.5) * (1 + 2.0 ** -20) * most)
    elif op == "product":
        # the sum, the scales' product and their product are rounded, then the sum with the bias
        bias = host(ops.prepare(case, 5)["bias"]).astype(np.float64) if case["bias"] else 0.0
        err = np.abs(got["y"] - want["y"])
        assert np.all(err <= U24 * (1 + 2.0 ** -20) * (3 * np.abs(want["y"] - bias) + np.abs(want["y"])))
    else:
        # in the root mean square no further off than four times what elementary fp32 operations are, and 2^-21 of the
        # result's own size (weights as two halves; a weight's own sum over a few heads)
        plain = _run(case, False)
        for name in want:
            off, size = _size(got[name] - want[name]), _size(want[name])
            near = _size(plain[name] - want[name])
            print(case["name"], name, "off", off / max(size, 1e-300), "plain", near / max(size, 1e-300))
            assert off <= 4 * near + 2.0 ** -21 * size, name
