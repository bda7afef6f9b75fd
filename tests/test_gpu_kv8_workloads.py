"""The measured workloads of the 8-bit KV cache call the framework on the stream that is current at each call."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def workloads():
    spec = importlib.util.spec_from_file_location("kv8_workloads", os.path.join(ROOT, "perf", "operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.own = True
    return module


@pytest.mark.parametrize("name", ["write_step", "read_prompt", "decode_b7_odd", "shared_b8"])
def test_runs_on_the_current_stream(workloads, name):
    """A pass on the default stream first, then passes captured on two other streams (after one that makes the
    stream's context): their replays give the first pass's results, which an empty graph could not."""
    import torch
    case = next(c for c in workloads.listed() if c["name"] == name)
    state = workloads.prepare(case, 1)
    as_list = lambda r: list(r) if isinstance(r, tuple) else [r]  # noqa: E731
    want = [x.clone() for x in as_list(workloads.run(state))]
    torch.cuda.synchronize()
    for _ in range(2):
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            workloads.run(state)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            got = as_list(workloads.run(state))
        for x in got:
            x.zero_()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        graph.reset()
