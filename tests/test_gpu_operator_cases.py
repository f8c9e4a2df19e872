"""perf/operators.py: its passes by the framework's operators are in order with torch's own work on
their inputs and outputs, without a synchronisation in between."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture()
def cases():
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    M = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(M)
    before = torch.cuda.current_stream()
    M.own = True
    yield M
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)


def outputs(r):
    return r if isinstance(r, tuple) else (r,)


@pytest.mark.parametrize("name", ["quantize ragged slice", "gemm token up", "norm per image"])
def test_inputs_come_before_and_readers_after(cases, name):
    case = {c["name"]: c for c in cases.listed()}[name]
    s = cases.prepare(dict(case), 3)
    torch.cuda.synchronize()
    r = cases.run(s)
    torch.cuda.synchronize()
    want = [t.float().cpu().numpy() for t in outputs(r)]
    for seed in (4, 3):  # other inputs, then the first again, in memory that the states before gave back
        torch.cuda._sleep(40_000_000)  # the inputs are made some 20 ms after the calls
        s = cases.prepare(dict(case), seed)
        r = cases.run(s)
        got = [t.float().clone() for t in outputs(r)]
        for t in outputs(r):
            t.zero_()
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g.cpu().numpy(), w)
