"""The timing cases' own calls run on whatever stream is current, and can be captured."""

from __future__ import annotations

import importlib.util

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.fixture()
def cases(cuda_device):
    spec = importlib.util.spec_from_file_location("operator_cases", REPO / "perf" / "operators.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.own = True
    return module


@pytest.mark.parametrize("name", ["grouped_one_token", "int8_one_token", "linear8_decode_batch", "backward_short_odd"])
def test_a_case_runs_on_the_current_stream(cases, name):
    case = next(c for c in cases.listed() if c["name"] == name)
    state = cases.prepare(case, 3)

    def outputs():
        out = cases.run(state)
        return out if isinstance(out, tuple) else (out,)

    want = [o.clone() for o in outputs()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)   # still running when the calls are made
        for o in outputs():
            o.fill_(7)
        got = [o.clone() for o in outputs()]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = outputs()
    for o in out:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
