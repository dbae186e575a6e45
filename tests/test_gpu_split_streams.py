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


def test_threads_on_their_own_streams_share_plain_weights(ops):
    """Four threads, each on a stream of its own, 300 weights between them: more than are kept, so that entries go while others read."""
    import threading
    weights = [torch.randn(128, 128, device="cuda") for _ in range(300)]
    x = torch.randn(256, 128, device="cuda")
    want = [product(x, w) for w in weights]
    torch.cuda.synchronize()
    errors, worst = [], [0.0] * 4

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in range(600):
                    j = (k * (2 * i + 1) + 75 * i) % 300
                    y = ops.linear(x, weights[j])
                    worst[i] = max(worst[i], float((y.double() - want[j]).abs().max()))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[:3]
    # 128 terms of size 1, operands of two bfloat16 parts: 2^-17 of each term
    assert max(worst) <= 2.0 ** -17 * 128 * 4, worst
