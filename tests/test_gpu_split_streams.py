"""GPU: operand splits that ops.as_split keeps for a plain weight, used on several streams."""
import pytest
import torch

from gpu_util import report

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops():
    from matris_b200 import ops
    ops._split_cache.clear()
    yield ops
    ops._split_cache.clear()


def product(x, w):
    return x.double() @ w.double().t()


def test_a_stream_waits_for_the_splits_that_another_one_builds(ops):
    """The splits are built behind other work of the first stream; the second one looks them up at once."""
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    for i in range(4):
        x, w = torch.randn(512, 128, device="cuda"), torch.randn(128, 128, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(first):
            torch.cuda._sleep(20_000_000)  # some 10 ms
            kept = ops.as_split(w)
        with torch.cuda.stream(second):
            assert ops.as_split(w) is kept
            y = ops.linear(x, w)
        torch.cuda.synchronize()
        report(f"second stream {i}", y, product(x, w), 1e-4, scaled=True)


def test_splits_that_make_room_stay_until_other_streams_have_read_them(ops):
    """An entry goes while a launch of another stream that reads it is still to come; the memory is wanted again at once."""
    other = torch.cuda.Stream()
    x, w = torch.randn(512, 128, device="cuda"), torch.randn(128, 128, device="cuda")

    def write(n):
        return [torch.full((128, 128), float("nan"), device="cuda", dtype=t) for t in (torch.float32, torch.bfloat16) for _ in range(n)]

    write(1)  # kernels are loaded at their first launch, which waits for the device
    ops.linear(x, w.clone())
    ops.as_split(w)
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        torch.cuda._sleep(20_000_000)
        y = ops.linear(x, w)
    ops._split_cache.clear()
    over = write(200)
    torch.cuda.synchronize()
    report("read late", y, product(x, w), 1e-4, scaled=True)
    assert len(over) == 400
