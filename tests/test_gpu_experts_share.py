"""GPU: a share of a grouping's experts - offsets that begin above zero and end below the last slot."""
import math

import pytest
import torch

from test_gpu_routed import grouped

pytestmark = pytest.mark.gpu
N, EXPERTS, K = 300, 8, 2


def dirty(*shape):
    """The allocator hands this memory out next: what a kernel leaves out shows."""
    t = torch.full(shape, math.nan, device="cuda")
    torch.cuda.synchronize()
    del t


def setup(n_in=128, n_out=256):
    offsets, row_of, slot_of = grouped(N, EXPERTS, K, 7)
    x, w = torch.randn(N, n_in, device="cuda"), torch.randn(EXPERTS, n_out, n_in, device="cuda")
    return offsets, row_of, slot_of, x, w


SHARES = [(0, 8), (0, 3), (3, 6), (5, 8), (4, 5)]


@pytest.mark.parametrize("a,z", SHARES)
def test_products_of_a_share_of_the_experts(a, z):
    """Its slots as in the whole, zeros elsewhere; a given output keeps the rest."""
    from matris_b200 import ops
    offsets, row_of, _, x, w = setup()
    y = ops.experts_linear(x, w, offsets, idx=row_of)
    part = offsets[a:z + 1].contiguous()
    from_, to = int(part[0]), int(part[-1])
    dirty(N * K, 256)
    got = ops.experts_linear(x, w[a:z], part, idx=row_of)
    assert torch.equal(got[from_:to], y[from_:to])
    assert not got[:from_].any() and not got[to:].any()
    out = torch.full((N * K, 256), math.nan, device="cuda")
    ops.experts_linear(x, w[a:z], part, idx=row_of, out=out)
    assert torch.equal(out[from_:to], y[from_:to]) and out[:from_].isnan().all() and out[to:].isnan().all()
    dy = torch.randn(N * K, 256, device="cuda")
    dw, db = ops.experts_grad_w(dy, x, offsets, idx=row_of)
    dy[:from_], dy[to:] = math.nan, math.nan
    part_dw, part_db = ops.experts_grad_w(dy, x, part, idx=row_of)
    for e in range(a, z):
        size = dy[int(offsets[e]):int(offsets[e + 1])].double().abs()
        rows = x.double()[row_of[int(offsets[e]):int(offsets[e + 1])].long()].abs()
        # the same sums, cut at other rows: at most a rounding a row on either side
        off = 2 * size.shape[0] * 2.0 ** -24
        assert ((part_dw[e - a].double() - dw[e].double()).abs() <= off * (size.t() @ rows)).all()
        assert ((part_db[e - a].double() - db[e].double()).abs() <= off * size.sum(0)).all()


@pytest.mark.parametrize("a,z", SHARES)
def test_combination_of_a_share_of_the_experts(a, z):
    """Choices of other experts count as none: nothing comes of them forward, and their slots and weights have zero gradients, the same
    on every call."""
    from matris_b200 import ops
    offsets, row_of, slot_of, x, w = setup()
    weights, dout = torch.rand(N, K, device="cuda"), torch.randn(N, 256, device="cuda")
    part = offsets[a:z + 1].contiguous()
    from_, to = int(part[0]), int(part[-1])
    y = ops.experts_linear(x, w, offsets, idx=row_of)
    whole_dy, whole_dw = ops.experts_combine_bwd(dout, y, slot_of, weights, offsets)
    dirty(N * K, 256)
    mine = ops.experts_linear(x, w[a:z], part, idx=row_of)
    held = (slot_of >= from_) & (slot_of < to)
    out = ops.experts_combine_fwd(mine, slot_of, weights)
    assert torch.equal(out, ops.experts_combine_fwd(y, torch.where(held, slot_of, -1), weights))
    mine[:from_], mine[to:] = math.nan, math.nan  # not read by the gradient
    for _ in range(5):
        dirty(N * K, 256)
        dy, dw = ops.experts_combine_bwd(dout, mine, slot_of, weights, part)
        assert torch.equal(dy[from_:to], whole_dy[from_:to]) and not dy[:from_].any() and not dy[to:].any()
        assert torch.equal(dw, torch.where(held, whole_dw, 0.0))


def test_shares_add_up_to_the_whole():
    from matris_b200 import ops
    offsets, row_of, slot_of, x, w = setup()
    weights = torch.rand(N, K, device="cuda")
    whole = ops.experts_combine_fwd(ops.experts_linear(x, w, offsets, idx=row_of), slot_of, weights)
    total = torch.zeros_like(whole)
    for a, z in [(0, 3), (3, 6), (6, 8)]:
        dirty(N * K, 256)
        total += ops.experts_combine_fwd(ops.experts_linear(x, w[a:z], offsets[a:z + 1].contiguous(), idx=row_of), slot_of, weights)
    # two terms a row, in the same order or the other one, each rounded as before: one more rounding of the sum
    assert ((total - whole).abs() <= 4 * 2.0 ** -24 * (total.abs() + whole.abs()) + 2.0 ** -22 * whole.abs().max()).all()


def test_gradient_of_slots_that_no_choice_has_without_offsets():
    from matris_b200 import ops
    offsets, _, slot_of = grouped(50, 4, 2, 3)
    slot_of = slot_of.clone()
    slot_of[7], slot_of[20, 1] = -1, -1
    y, dout = torch.randn(130, 128, device="cuda"), torch.randn(50, 128, device="cuda")
    dirty(130, 128)
    dy, _ = ops.experts_combine_bwd(dout, y, slot_of)
    named = torch.zeros(130, dtype=torch.bool, device="cuda")
    named[slot_of[slot_of >= 0].long()] = True
    assert not dy[~named].any() and (dy[named] != 0).any(1).all()
