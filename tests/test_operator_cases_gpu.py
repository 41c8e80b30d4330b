"""The kernels' calls of perf/operators.py among a program's other work: they
take what the current stream has written, and what follows on it finds their
results."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def cases():
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    before = torch.cuda.current_stream()
    m.own = True
    yield m
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)
    if m.CONTEXT:
        m.CONTEXT[0].close()


def leaves(x):
    return list(x.values()) if isinstance(x, dict) else [x]


@pytest.mark.parametrize("name", ["append_32rows", "attend_32rows_prefix_2048", "adjust_32rows"])
@pytest.mark.parametrize("other", [False, True])
def test_calls_are_ordered_with_the_current_stream(cases, name, other):
    case = next(c for c in cases.listed() if c["name"] == name)
    busy = torch.randn(4096, 4096, device="cuda")
    if other:
        torch.cuda.synchronize()
        torch.cuda.set_stream(torch.cuda.Stream())
    s = cases.prepare(case, 5)
    want = [t.clone() for t in leaves(cases.run(s))]
    torch.cuda.synchronize()
    for _ in range(20):
        torch.mm(busy, busy)
    written = leaves(s["result"])
    for t in written if case["op"] != "append" else written[:1]:  # a cache keeps what it holds
        t.fill_(3)
    got = [t.clone() for t in leaves(cases.run(s))]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
