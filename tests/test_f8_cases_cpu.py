"""CPU tier: the timed cases of perf/more_operators.py, listed and drawn, pass the operators' argument checks and
give results of the shapes and types that the plain forms give (fake tensors: nothing is computed)."""
import os
import random
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf"))
import more_operators as cases  # noqa: E402


class _Generator:
    """In the place of a GPU's generator, which fake tensors do not need."""

    def __init__(self, device=None):
        pass

    def manual_seed(self, seed):
        return None


def _drawn(n):
    rng = random.Random(7)
    return [cases.draw(rng) for _ in range(n)]


def _layout(out):
    out = out if isinstance(out, (tuple, list)) else (out,)
    return [(tuple(t.shape), t.dtype) for t in out]


def test_norms_alone_that_keep_statistics_are_drawn():
    assert any(c["op"] == "norm" and c["parts"].split() == ["keep"] for c in _drawn(200))


@pytest.mark.parametrize("which", ["listed", "drawn"])
def test_cases_pass_the_checks(which, monkeypatch):
    monkeypatch.setattr(torch, "Generator", _Generator)
    with FakeTensorMode():
        for i, case in enumerate(cases.listed() if which == "listed" else _drawn(200)):
            state = cases.prepare(case, i)
            got, want = [], []
            for own, out in ((True, got), (False, want)):
                monkeypatch.setattr(cases, "own", own)
                out += _layout(cases.run(state))
            assert got == want, case
