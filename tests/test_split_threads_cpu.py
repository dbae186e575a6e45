"""CPU: ops.as_split called by several threads, and what keeps the splits of a call alive."""
import sys
import threading
import weakref
from types import SimpleNamespace

import pytest
import torch

from matris_b200 import ops


@pytest.fixture
def many_switches():
    """Threads take turns every microsecond, and the cache is empty before and after."""
    interval = sys.getswitchinterval()
    ops._split_cache.clear()
    sys.setswitchinterval(1e-6)
    yield
    sys.setswitchinterval(interval)
    ops._split_cache.clear()


def in_threads(n, work):
    errors = []

    def run(i):
        try:
            work(i)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[:3]


def test_a_hit_returns_the_splits_that_are_kept(many_switches):
    """A weight that is there is never missing for another thread, so nobody builds it again."""
    weights = [torch.full((2, 4), float(i)) for i in range(8)]
    first = [ops.as_split(w) for w in weights]
    other = []

    def work(i):
        for k in range(5_000):
            j = (k + 3 * i) % 8
            if ops.as_split(weights[j]) is not first[j]:
                other.append(j)

    in_threads(4, work)
    assert not other, f"{len(other)} of 20000 look-ups"
    assert {id(e[1]) for e in ops._split_cache.values()} == {id(s) for s in first}


def test_threads_that_build_one_weight_at_once_leave_one(many_switches):
    for i in range(20):
        w, got, start = torch.full((2, 4), float(i)), [None] * 4, threading.Barrier(4)

        def work(k):
            start.wait(10)
            got[k] = ops.as_split(w)

        in_threads(4, work)
        assert all(torch.equal(s.w, w) for s in got)
        kept = ops.as_split(w)
        assert any(kept is s for s in got) and ops.as_split(w) is kept


def test_a_full_cache_makes_room_in_several_threads(many_switches):
    """More weights than are kept, from four threads: each gets its own weight's splits, and nothing is raised."""
    weights = [torch.full((2, 4), float(i)) for i in range(600)]

    def work(i):
        for k in range(2_000):
            j = (k * (2 * i + 1) + 150 * i) % 600
            assert float(ops.as_split(weights[j]).w[0, 0]) == j

    in_threads(4, work)
    assert len(ops._split_cache) <= 257


def packed(**kw):
    return SimpleNamespace(b1=None, b2=None, nc=torch.ones(128), ng=torch.ones(128), **kw)


def w(rows, cols):
    return torch.randn(rows, cols)


X = torch.randn(4, 128)
CALLS = {
    "gemm": lambda: ops.gemm(4, [ops.B([ops.S(X)], w(128, 128), out=torch.empty(4, 128)) for _ in range(3)]),
    "linear": lambda: ops.linear(X, w(256, 128)),
    "gated_mlp_fwd": lambda: ops.gated_mlp_fwd(packed(w1=w(256, 128), w2=w(256, 128)), 4, [ops.S(X)]),
    "ffn_fwd": lambda: ops.ffn_fwd(packed(w1=w(128, 128), w2=w(128, 128)), X),
    "mlp_bwd": lambda: ops.mlp_bwd(X, w(128, 128), w(128, 128), torch.randn(4, 128), gated=False, ext=torch.randn(4, 128), w3t=w(128, 128)),
}


@pytest.mark.parametrize("name", CALLS)
def test_a_call_holds_its_splits_until_the_launch(name, monkeypatch):
    """Whatever other threads do to the cache: the splits whose addresses a launch gets are alive when it is made."""
    made, seen = [], []

    def build(weight):
        ops._split_cache.clear()  # another thread has made room
        split = ops.SplitWeight(weight)
        made.append([weakref.ref(t) for t in (split.hi, split.lo, split.hi16, split.lo16)])
        return split

    monkeypatch.setattr(ops, "as_split", lambda weight: weight if isinstance(weight, ops.SplitWeight) else build(weight))
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "call", lambda *a: seen.append([r() is not None for refs in made for r in refs]))
    CALLS[name]()
    assert len(seen) == 1 and seen[0] and all(seen[0]), seen
