"""perf/more_operators.py: its passes by the framework's operators are in order with torch's own work on their inputs
and outputs, without a synchronisation in between, and other passes leave their results as they were."""
import importlib.util
import os

import pytest
import torch

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture()
def cases():
    spec = importlib.util.spec_from_file_location("more_operator_cases", os.path.join(ROOT, "perf", "more_operators.py"))
    M = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(M)
    before = torch.cuda.current_stream()
    M.own = True
    yield M
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)


def outputs(r):
    return r if isinstance(r, tuple) else (r,)


@pytest.mark.parametrize("name", ["rope far", "append batch", "attend token", "attend drafts", "attend pieces", "layer batch"])
def test_inputs_come_before_and_readers_after(cases, name):
    case = {c["name"]: c for c in cases.listed()}[name]
    s = cases.prepare(dict(case), 3)
    torch.cuda.synchronize()
    want = [t.clone() for t in outputs(cases.run(s))]
    torch.cuda.synchronize()
    for seed in (4, 3):  # other inputs, then the first again, in memory that the states before gave back
        torch.cuda._sleep(40_000_000)  # the inputs are made some 20 ms after the calls
        s = cases.prepare(dict(case), seed)
        r = outputs(cases.run(s))
        got = [t.clone() for t in r]
        for t in r:
            t.zero_()
    for g, w in zip(got, want):
        assert torch.equal(g.view(torch.uint8), w.view(torch.uint8))
