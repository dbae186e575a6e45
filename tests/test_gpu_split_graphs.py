"""GPU: operand splits that ops.as_split keeps for a plain weight, used in captured graphs."""
import pytest
import torch

from gpu_util import report

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops():
    from matris_b200 import ops
    ops.linear(torch.randn(512, 128, device="cuda"), torch.randn(128, 128, device="cuda"))  # a process's first launch is no part of a graph
    ops._split_cache.clear()
    yield ops
    ops._split_cache.clear()


def product(x, w):
    return x.double() @ w.double().t()


def capture(ops, x, w):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.linear(x, w)
    return g, y


def test_splits_built_in_a_capture_are_not_handed_to_others(ops):
    """Their values exist when the graph has run, and whenever it runs."""
    x, w = torch.randn(512, 128, device="cuda"), torch.randn(128, 128, device="cuda")
    g, y = capture(ops, x, w)
    report("eager before the first replay", ops.linear(x, w), product(x, w), 1e-4, scaled=True)
    g2, y2 = capture(ops, x, w)
    g2.replay()
    report("second graph before the first", y2, product(x, w), 1e-4, scaled=True)
    g.replay()
    report("first graph", y, product(x, w), 1e-4, scaled=True)


@pytest.mark.parametrize("warm", [False, True])
def test_a_graph_keeps_the_splits_that_it_reads(ops, warm):
    """300 other weights make room between capture and replay, and their memory is written."""
    x, w = torch.randn(512, 128, device="cuda"), torch.randn(128, 128, device="cuda")
    if warm:
        ops.linear(x, w)
    g, y = capture(ops, x, w)
    for _ in range(2):
        y.fill_(float("nan"))
        others = [torch.randn(128, 128, device="cuda") for _ in range(300)]
        for o in others:
            ops.as_split(o)
        g.replay()
        report(f"replay, warm={warm}", y, product(x, w), 1e-4, scaled=True)
