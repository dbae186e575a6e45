"""GPU: router with padded rows and barred experts on 16-bit logits."""
import math

import pytest
import torch

from test_gpu_routed import check_route, logits_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("n,n_exp,k", [(1, 8, 2), (40, 8, 2), (77, 7, 3), (900, 64, 6), (600, 30, 4), (50, 300, 9)])
def test_masks(n, n_exp, k, renorm, dtype):
    """Rows that are padding, rows without an expert, with one, and with fewer than top_k; what padding holds does not matter."""
    l = logits_of(n, n_exp, dtype, 5, barred=0.6)
    valid = torch.rand(n, generator=torch.Generator().manual_seed(6)).cuda() > 0.2
    if n > 8:
        l[5] = -math.inf
        l[6], l[6, n_exp - 1] = -math.inf, 0.25
        valid[:7] = torch.tensor([False, False, False, True, True, True, True])
    r = check_route(l, k, valid=valid, renorm=renorm)
    assert (r.ids[~valid] == -1).all() and not r.weights[~valid].any() and (r.slot_of[~valid] == -1).all()
    if n > 8:
        from matris_b200 import ops
        dirty = l.clone()
        dirty[0], dirty[1], dirty[2] = math.nan, math.inf, torch.finfo(dtype).min
        q = ops.route_fwd(dirty, k, valid=valid, renorm=renorm)
        assert all(torch.equal(a, b) for a, b in zip(q[:-1], r[:-1]))
        dw, dl = torch.randn(n, k, device="cuda"), torch.ones((), device="cuda")
        assert torch.equal(ops.route_bwd(dirty, q, dw, dl), ops.route_bwd(l, r, dw, dl))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lowest_values_of_the_type_are_available(dtype):
    """A mask of the type's lowest value, not minus infinity: such experts come last, with weight zero beside others, and share a row that has
    nothing else."""
    from matris_b200 import ops
    low = torch.finfo(dtype).min
    l = torch.full((3, 12), low, dtype=dtype, device="cuda")
    l[0, 4], l[0, 9] = 1.0, 2.0
    l[1, 3] = -math.inf
    r = ops.route_fwd(l, 3)
    assert r.ids.tolist() == [[9, 4, 0], [0, 1, 2], [0, 1, 2]] and float(r.weights[0, 2]) == 0.0
    assert torch.allclose(r.weights[1:], torch.full((2, 3), 1 / 3, device="cuda"), atol=2.0 ** -22)
    assert int(r.totals[-1]) == 3
