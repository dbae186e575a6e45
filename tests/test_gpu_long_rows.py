"""Norm, router, experts and combination on tensors of more than 2^31 elements: the rows behind that number against the same rows alone
or against the definition."""
import pytest
import torch

from test_gpu_group_norm import U, check, close, inputs, plain, stats_of
from test_gpu_routed import logits_of, plain_experts, product_bound

pytestmark = pytest.mark.gpu


def test_group_norm():
    from matris_b200 import ops
    rows, tail = 8_500_000, 100_000  # rows of 256: row 8,388,608 starts at element 2^31
    small, w, b, dy_small, tail_ptr = inputs([0, 99_000, tail], 256, torch.bfloat16, 5)
    x = torch.ones(rows, 256, dtype=torch.bfloat16, device="cuda")
    x[-tail:] = small
    dy = torch.zeros_like(x)
    dy[-tail:] = dy_small
    ends = [0, rows - tail, rows - 1000, rows]
    seg_ptr = torch.tensor(ends, dtype=torch.int32, device="cuda")
    y, stats = ops.group_norm_fwd(x, w, b, 8, seg_ptr=seg_ptr, act=1)
    dx, dw, db = ops.group_norm_bwd(dy, x, w, b, stats, 8, seg_ptr=seg_ptr, act=1)
    _, _, dx_small, dw_small, db_small = check(small, w, b, dy_small, tail_ptr, 8, 1, [0, 99_000, tail])
    x64, w64, b64 = small.double(), w.double(), b.double()
    mean, rstd = stats_of(x64, [0, 99_000, tail], 8)
    xh = (x64 - mean) * rstd
    z = (xh * w64).abs() + b64.abs()
    off = 1.1 * 64 * U * ((x64.abs() * rstd + xh.abs()) * w64.abs() + z) + 8 * U * z  # as the bound of `check`
    close(y[-tail:], plain(x64, w64, b64, [0, 99_000, tail], 8, 1), off, torch.bfloat16)
    # rows that are all the same: xh = 0
    const = torch.nn.functional.silu(b64)
    assert ((y[:1000].double() - const).abs() <= (2.0 ** -8 + 16 * U) * const.abs()).all()
    assert not dx[:1000].any()
    # both are within half a step of bfloat16 (2^-8) and 2^-8 in all of the definition: 64 u (4e-6) of products of dy, xh and w below 300
    assert ((dx[-tail:].double() - dx_small.double()).abs() <= 2.0 ** -7 * (dx_small.double().abs() + 1)).all()
    # the rows ahead add zeros
    for got, want, size in ((db, db_small, dy_small.double().abs()), (dw, dw_small, dy_small.double().abs() * xh.abs())):
        assert ((got.double() - want.double()).abs() <= 2 * 256 * U * (1.1 * size * (1 + z + x64.abs() * rstd)).sum(0)).all()


def test_router():
    from matris_b200 import ops
    n, tail, k = 2_200_000, 500, 3  # rows of 1024: row 2,097,152 starts at element 2^31
    last = logits_of(tail, 1024, torch.bfloat16, 6)
    logits = torch.zeros(n, 1024, dtype=torch.bfloat16, device="cuda")
    logits[:, ::7] = -1
    logits[-tail:] = last
    r, alone = ops.route_fwd(logits, k), ops.route_fwd(last, k)
    assert torch.equal(r.ids[-tail:], alone.ids) and torch.equal(r.weights[-tail:], alone.weights)
    assert torch.equal(r.ids[:-tail], torch.arange(1, k + 1, dtype=torch.int32, device="cuda").expand(n - tail, k))
    order = torch.argsort(r.ids.reshape(-1), stable=True)
    assert torch.equal(r.row_of.long(), order // k)
    assert torch.equal(r.slot_of.view(-1)[order].long(), torch.arange(n * k, device="cuda"))
    dw = torch.randn(n, k, generator=torch.Generator().manual_seed(7)).cuda()
    assert torch.equal(ops.route_bwd(logits, r, dw)[-tail:], ops.route_bwd(last, alone, dw[-tail:].contiguous()))


def test_experts_and_combination():
    from matris_b200 import ops
    g = torch.Generator().manual_seed(8)
    slots, tail, n_in, n_out = 4_300_000, 300, 128, 512  # rows of 512: row 4,194,304 starts at element 2^31
    ends = [0, 1_000_000, 4_250_000, slots]
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    x, w = torch.randn(1000, n_in, generator=g).cuda(), torch.randn(3, n_out, n_in, generator=g).cuda()
    idx = (torch.arange(slots, device="cuda", dtype=torch.int32) * 7) % 1000
    laid = ops.ExpertWeights(w)
    y = ops.experts_linear(x, laid, offsets, idx=idx)
    rows, alone = x.double()[idx[-tail:].long()], torch.tensor([0, 0, 0, tail])
    want, size = plain_experts(rows, w.double(), None, alone, 0)
    assert ((y[-tail:].double() - want).abs() <= product_bound(n_in) * size).all()
    dx = ops.experts_linear(y, laid, offsets, transposed=True)
    want, size = plain_experts(y[-tail:].double(), w.double().transpose(1, 2), None, alone, 0)
    assert ((dx[-tail:].double() - want).abs() <= product_bound(n_out) * size).all()
    dw, db = ops.experts_grad_w(y, x, offsets, idx=idx)
    dy, rows = y[ends[2]:].double(), x.double()[idx[ends[2]:].long()]
    assert ((dw[2].double() - dy.t() @ rows).abs() <= product_bound(4096) * (dy.abs().t() @ rows.abs())).all()
    assert ((db[2].double() - dy.sum(0)).abs() <= product_bound(4096) * dy.abs().sum(0)).all()
    slot_of = (slots - 1 - torch.randperm(2000, generator=g, dtype=torch.int32)).view(1000, 2).cuda()
    share, dout = torch.rand(1000, 2, generator=g).cuda(), torch.randn(1000, n_out, generator=g).cuda()
    picked = y[slot_of.long()].double()
    out = ops.experts_combine_fwd(y, slot_of, share)
    assert ((out.double() - (share.double().unsqueeze(2) * picked).sum(1)).abs() <= 4 * U * (share.double().unsqueeze(2) * picked).abs().sum(1)).all()
    d, dshare = ops.experts_combine_bwd(dout, y, slot_of, share)
    prod = picked * dout.double().unsqueeze(1)
    assert ((dshare.double() - prod.sum(2)).abs() <= (n_out / 32 + 12) * U * prod.abs().sum(2)).all()
    want = share.double().unsqueeze(2) * dout.double().unsqueeze(1)
    assert ((d[slot_of.long()].double() - want).abs() <= U * want.abs()).all()
