"""Router, experts' dense layers and combination on the GPU against the definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of float32


# ------------------------------------------------------------------ router
def plain_route(logits, k, valid, renorm):
    """The definition, on the CPU: whole numbers exactly, the rest in 64 bits with gradients."""
    n, n_exp = logits.shape
    l = logits.detach().double().cpu().requires_grad_()
    ok = torch.isfinite(l).any(1) if valid is None else torch.isfinite(l).any(1) & valid.cpu()
    p = torch.zeros_like(l)
    p[ok] = torch.softmax(l[ok], 1)
    order = sorted
    ids = torch.full((n, k), -1)
    for t, row in enumerate(l.tolist()):
        if ok[t]:
            best = order((i for i in range(n_exp) if row[i] > -math.inf), key=lambda i: (-row[i], i))[:k]
            ids[t, :len(best)] = torch.tensor(best)
    held = ids >= 0
    w = torch.where(held, p.gather(1, ids.clamp(min=0)), 0.0)
    if renorm:
        w = w / torch.where(ok, w.sum(1), 1.0).unsqueeze(1)
    counts = torch.bincount(ids[held], minlength=n_exp)
    rows = int(ok.sum())
    loss = n_exp / (k * rows * rows) * (counts.double() * p.sum(0)).sum() if rows else l.sum() * 0
    pairs = sorted((int(ids[t, j]), t, j) for t in range(n) for j in range(k) if held[t, j])
    row_of, slot_of = torch.full((n * k,), -1), torch.full((n, k), -1)
    for s, (_, t, j) in enumerate(pairs):
        row_of[s], slot_of[t, j] = t, s
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
    return l, dict(ids=ids, weights=w, counts=counts, loss=loss, offsets=offsets, row_of=row_of, slot_of=slot_of, rows=rows)


def check_route(logits, k, valid=None, renorm=True, seed=0):
    """ops against the definition.  Bounds, u = 2^-24: exp is good to 2 steps and its argument l - m, rounded once, to u |l - m|; a sum of
    up to 1024 positive terms is a tree of at most 32 + 5 roundings; so p is off by at most (48 + |l - m|) u p, the weights by twice
    that.  The loss averages such p.  A logit's gradient is p (g - sum p g): the error of p times what it multiplies, plus the sum's."""
    from matris_b200 import ops
    r = ops.route_fwd(logits, k, valid=valid, renorm=renorm)
    l, want = plain_route(logits, k, valid, renorm)
    for name in ("ids", "counts", "offsets", "row_of", "slot_of"):
        assert torch.equal(getattr(r, name).cpu().long(), want[name].long()), name
    assert int(r.totals[-1]) == want["rows"]
    g = torch.Generator().manual_seed(seed)
    n = max(1, logits.shape[0])
    dw, dl = torch.randn(logits.shape[0], k, generator=g) / n, torch.rand((), generator=g) + 0.5
    (want["weights"] * dw.double()).sum().add(want["loss"] * dl.double()).backward()
    got = ops.route_bwd(logits, r, dw.cuda(), dl.cuda()).cpu().double()
    with torch.no_grad():
        finite = torch.where(torch.isfinite(l), l, 0.0)
        rel = 96 * U * (1 + (finite.amax(1) - finite.amin(1)).unsqueeze(1) / 32) if l.numel() else torch.zeros(0, 1)
        assert ((r.weights.cpu().double() - want["weights"]).abs() <= 2 * rel * want["weights"]).all()
        assert abs(float(r.loss) - float(want["loss"])) <= 2 * float(rel.max() if rel.numel() else 0) * abs(float(want["loss"])) + U * abs(float(want["loss"]))
        rows = max(1, want["rows"])
        share = float(dl) * logits.shape[1] / (k * rows * rows) * want["counts"].double()
        p = torch.softmax(finite.masked_fill(~torch.isfinite(l), -math.inf), 1).nan_to_num(0.0)
        held = want["ids"] >= 0
        at = want["ids"].clamp(min=0)
        sel = torch.zeros_like(l).scatter_add(1, at, held * (want["weights"] if renorm else p.gather(1, at)))
        mass = (held * want["weights"] * dw.double().abs()).sum(1, keepdim=True) if renorm else (p.gather(1, at) * held * dw.double().abs()).sum(1, keepdim=True)
        dws = torch.zeros_like(l).scatter_add(1, at, held * dw.double().abs())
        bound = 4 * rel * (p * (share + (p * share).sum(1, keepdim=True) + (0 if renorm else mass)) + sel * (dws + mass))
        half = torch.finfo(logits.dtype).eps / 2
        small = 2.0 ** -25 if logits.dtype == torch.float16 else 2.0 ** -140
        off = (got - l.grad).abs()
        assert (off <= bound + half * (l.grad.abs() + bound) + small).all(), (off - bound).max()
    return r


def logits_of(n, n_exp, dtype, seed, barred=0.0):
    g = torch.Generator().manual_seed(seed)
    l = 1.5 * torch.randn(n, n_exp, generator=g) + 0.5 * torch.randn(1, n_exp, generator=g)
    if barred:
        l[torch.rand(n, n_exp, generator=g) < barred] = -math.inf
    return l.to(dtype).cuda()


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,n_exp,k", [(1, 8, 2), (0, 8, 2), (1, 1, 1), (3, 4, 4), (33, 7, 3), (100, 16, 5), (257, 32, 2), (700, 64, 6), (1500, 60, 8), (65, 128, 32),
                                       (400, 256, 8), (50, 1000, 17), (3000, 5, 1)])
def test_router_against_the_definition(n, n_exp, k, dtype, renorm):
    check_route(logits_of(n, n_exp, dtype, n + n_exp), k, renorm=renorm)


@pytest.mark.parametrize("n,n_exp,k", [(40, 8, 2), (900, 64, 6), (600, 30, 4)])
@pytest.mark.parametrize("renorm", [True, False])
def test_router_with_masks(n, n_exp, k, renorm):
    """Padded rows (with whatever they hold), barred experts, rows without any, rows with fewer than top_k."""
    l = logits_of(n, n_exp, torch.float32, 3, barred=0.6)
    l[5] = -math.inf
    l[6] = -math.inf
    l[6, 3] = 0.25
    valid = torch.rand(n, generator=torch.Generator().manual_seed(4)).cuda() > 0.2
    valid[:5] = False
    clean = l.clone()
    l[0] = math.nan
    l[1] = math.inf
    l[2] = -math.inf
    clean[:3] = -math.inf
    r = check_route(clean, k, valid=valid, renorm=renorm)
    from matris_b200 import ops
    q = ops.route_fwd(l, k, valid=valid, renorm=renorm)
    assert all(torch.equal(a, b) for a, b in zip(q[:-1], r[:-1]))
    dw, dl = torch.randn(n, k, device="cuda"), torch.ones((), device="cuda")
    assert torch.equal(ops.route_bwd(l, q, dw, dl), ops.route_bwd(clean, r, dw, dl))


def test_router_ties_and_zeros():
    """Equal logits go to the lowest index, 0 and -0 are equal, and even loads have loss 1."""
    from matris_b200 import ops
    l = torch.zeros(64, 8, device="cuda")
    l[1::2] = -0.0
    l[3, 5:] = 1.0
    r = check_route(l, 3)
    assert r.ids[0].tolist() == [0, 1, 2] and r.ids[3].tolist() == [5, 6, 7]
    l = torch.where(torch.eye(8, device="cuda").repeat(8, 1) > 0, 40.0, 0.0)
    assert abs(float(ops.route_fwd(l, 1).loss) - 1) <= 64 * U


def test_router_nan_and_infinity():
    from matris_b200 import ops
    l = torch.zeros(3, 8, device="cuda")
    l[1, 4], l[2, 2] = math.nan, math.inf
    r = ops.route_fwd(l, 2)
    assert r.ids.tolist() == [[0, 1], [4, 0], [2, 0]]
    assert torch.isfinite(r.weights[0]).all() and r.weights[1].isnan().all() and r.weights[2].isnan().any() and r.loss.isnan()
    assert int(r.totals[-1]) == 3 and int(r.counts.sum()) == 6


def test_router_strides_and_missing_gradients():
    from matris_b200 import ops
    wide = torch.randn(300, 130, device="cuda")
    for shift in (0, 1, 4):
        l = wide[:, shift:shift + 24]
        r = check_route(l, 4)
        d = l.contiguous()
        dw, dl = torch.randn(300, 4, device="cuda"), torch.rand((), device="cuda")
        both = ops.route_bwd(d, r, dw, dl)
        assert torch.equal(both, ops.route_bwd(l, r, dw, dl))
        assert not ops.route_bwd(l, r).any()
        apart = ops.route_bwd(l, r, dw).double() + ops.route_bwd(l, r, None, dl).double()
        assert (both.double() - apart).abs().max() <= 16 * U * apart.abs().max()


def test_router_long_input_against_torch():
    """Whole numbers of a long input (many blocks) by torch's stable sort."""
    from matris_b200 import ops
    n, n_exp, k = 200_003, 24, 3
    l = logits_of(n, n_exp, torch.float32, 9)
    r = ops.route_fwd(l, k)
    ids = l.sort(dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.ids.long(), ids)
    assert torch.equal(r.counts.long(), torch.bincount(ids.reshape(-1), minlength=n_exp))
    order = torch.argsort(ids.reshape(-1), stable=True)
    assert torch.equal(r.row_of.long(), order // k)
    assert torch.equal(r.slot_of.view(-1)[order].long(), torch.arange(n * k, device="cuda"))
    p = torch.softmax(l.double(), 1).sum(0)
    want = n_exp / (k * n * n) * (r.counts.double() * p).sum()
    assert abs(float(r.loss) - float(want)) <= 200 * U * float(want)
    assert all(torch.equal(a, b) for a, b in zip(r[:-1], ops.route_fwd(l, k)[:-1]))


# ------------------------------------------------------------------ experts
def grouped(n, n_exp, k, seed, empty=()):
    """Random choices as a Route's grouping: offsets, row_of, slot_of."""
    g = torch.Generator().manual_seed(seed)
    score = torch.randn(n, n_exp, generator=g)
    if empty:
        score[:, list(empty)] = -math.inf
    ids = score.topk(k, 1).indices
    order = torch.argsort(ids.reshape(-1), stable=True)
    slot_of = torch.empty(n * k, dtype=torch.int32)
    slot_of[order] = torch.arange(n * k, dtype=torch.int32)
    offsets = torch.zeros(n_exp + 1, dtype=torch.int32)
    offsets[1:] = torch.bincount(ids.reshape(-1), minlength=n_exp).cumsum(0)
    return offsets.cuda(), (order // k).int().cuda(), slot_of.view(n, k).cuda()


def silu64(v):
    return v * torch.sigmoid(v)


def plain_experts(x, w, b, offsets, act):
    """Rows already gathered; |values| of the products too."""
    ends = offsets.tolist()
    y, size = (torch.zeros(x.shape[0], w.shape[1], dtype=torch.double, device="cuda") for _ in range(2))
    for e, (a, z) in enumerate(zip(ends[:-1], ends[1:])):
        y[a:z] = x[a:z] @ w[e].t() + (0 if b is None else b[e])
        size[a:z] = x[a:z].abs() @ w[e].abs().t() + (0 if b is None else b[e].abs())
    return y, size


def product_bound(k):
    """A product of k terms in 64-bit-free arithmetic: operands carry at least 22 bits (a relative error of 2^-22 each, whichever core
    runs), sums of k terms in float32 at most (k / 8 + 16) roundings in a row."""
    return (2 * 2.0 ** -22 + (k / 8 + 16) * U)


SHAPES = [(1, 8, 2, 128, 128), (32, 8, 2, 128, 128), (5, 3, 1, 256, 384), (300, 7, 3, 128, 256), (1000, 4, 2, 384, 128), (129, 2, 2, 1024, 128),
          (257, 16, 4, 512, 512), (4000, 5, 1, 128, 128), (64, 64, 1, 128, 1024)]


@pytest.mark.parametrize("n,n_exp,k,n_in,n_out", SHAPES)
def test_experts_linear_against_the_definition(n, n_exp, k, n_in, n_out):
    from matris_b200 import ops
    g = torch.Generator().manual_seed(n + n_in)
    offsets, row_of, _ = grouped(n, n_exp, k, 1, empty=(1,) if n_exp > k + 1 else ())
    x, w = torch.randn(n, n_in, generator=g).cuda(), (torch.randn(n_exp, n_out, n_in, generator=g) / math.sqrt(n_in)).cuda()
    b, z = torch.randn(n_exp, n_out, generator=g).cuda(), torch.randn(n * k, n_out, generator=g).cuda()
    for kw in (dict(), dict(bias=b), dict(bias=b, out_act=1), dict(in_act=1), dict(gate=z)):
        y = ops.experts_linear(x, w, offsets, idx=row_of, **kw)
        rows = x.double()[row_of.long()]
        in_off = 0.0
        if kw.get("in_act"):
            rows, in_off = silu64(rows), 16 * U * (1 + rows.abs().max())  # SiLU's own error, relative
        want, size = plain_experts(rows, w.double(), kw.get("bias", None) if kw.get("bias") is None else b.double(), offsets, 0)
        bound = (product_bound(n_in) + in_off) * size
        if kw.get("out_act"):
            bound = 1.1 * bound + 16 * U * (1 + want.abs()) * want.abs()
            want = silu64(want)
        if kw.get("gate") is not None:
            s = torch.sigmoid(z.double())
            d = s * (1 + z.double() * (1 - s))
            bound = bound * d.abs() + 16 * U * (1 + z.double().abs()) * want.abs() * (d.abs() + 0.5)
            want = want * d
        off = (y.double() - want).abs()
        assert (off <= bound + U * want.abs()).all(), (sorted(kw), (off / bound).max())
    # the data gradient: the same on the transposed weights, rows in place
    dy = torch.randn(n * k, n_out, generator=g).cuda()
    dx = ops.experts_linear(dy, ops.ExpertWeights(w), offsets, transposed=True)
    want, size = plain_experts(dy.double(), w.double().transpose(1, 2), None, offsets, 0)
    assert ((dx.double() - want).abs() <= product_bound(n_out) * size).all()


@pytest.mark.parametrize("n,n_exp,k,n_in,n_out", SHAPES)
def test_experts_weight_gradient_against_the_definition(n, n_exp, k, n_in, n_out):
    """Sums over an expert's slots: the operands' 2^-22 each, and trees or runs of at most 4096 rows in float32 (each 8 to a
    matrix instruction) before the partial sums are joined."""
    from matris_b200 import ops
    g = torch.Generator().manual_seed(n + n_in)
    empty = (1,) if n_exp > k + 1 else ()
    offsets, row_of, _ = grouped(n, n_exp, k, 1, empty=empty)
    x, dy = torch.randn(n, n_in, generator=g).cuda(), torch.randn(n * k, n_out, generator=g).cuda()
    for in_act in (0, 1):
        dw, db = ops.experts_grad_w(dy, x, offsets, idx=row_of, in_act=in_act)
        rows = x.double()[row_of.long()]
        in_off = 0.0
        if in_act:
            rows, in_off = silu64(rows), 16 * U * (1 + rows.abs().max())
        ends = offsets.tolist()
        for e, (a, z) in enumerate(zip(ends[:-1], ends[1:])):
            want, size = dy[a:z].double().t() @ rows[a:z], dy[a:z].double().abs().t() @ rows[a:z].abs()
            assert ((dw[e].double() - want).abs() <= (product_bound(min(z - a, 4096)) + in_off) * size).all()
            assert ((db[e].double() - dy[a:z].double().sum(0)).abs() <= product_bound(min(z - a, 4096)) * dy[a:z].double().abs().sum(0)).all()
    for e in empty:
        assert not dw[e].any() and not db[e].any()
    assert torch.equal(ops.experts_grad_w(dy, x, offsets, idx=row_of, in_act=1, want_bias=False)[0], dw)


def test_experts_slots_behind_the_last_and_given_outputs():
    from matris_b200 import ops
    offsets, row_of, _ = grouped(50, 4, 2, 2)
    x, w = torch.randn(50, 128, device="cuda"), torch.randn(4, 256, 128, device="cuda")
    more = torch.cat([row_of, torch.full((300,), -1, dtype=torch.int32, device="cuda")])
    y = ops.experts_linear(x, w, offsets, idx=row_of)
    z = ops.experts_linear(x, w, offsets, idx=more)
    assert torch.equal(z[:100], y) and not z[100:].any()
    wide = torch.full((400, 264), math.nan, device="cuda")
    out = wide[:, 4:260]
    assert ops.experts_linear(x, w, offsets, idx=more, out=out) is out
    assert torch.equal(out[:100], y) and wide[100:].isnan().all() and wide[:, :4].isnan().all() and wide[:, 260:].isnan().all()
    dy = torch.randn(400, 256, device="cuda")
    dy[100:] = math.nan
    dw, db = ops.experts_grad_w(dy, x, offsets, idx=more)
    dw2, db2 = ops.experts_grad_w(dy[:100].contiguous(), x, offsets, idx=row_of)
    assert torch.equal(dw, dw2) and torch.equal(db, db2)


def test_experts_without_any_slot():
    from matris_b200 import ops
    offsets = torch.zeros(5, dtype=torch.int32, device="cuda")
    w = torch.randn(4, 128, 128, device="cuda")
    none = torch.empty(0, 128, device="cuda")
    assert ops.experts_linear(none, w, offsets).shape == (0, 128)
    x = torch.full((6, 128), math.nan, device="cuda")
    idx = torch.full((12,), -1, dtype=torch.int32, device="cuda")
    assert not ops.experts_linear(x, w, offsets, idx=idx).any()
    for args in ((none, none, offsets), (torch.full((12, 128), math.nan, device="cuda"), x, offsets, idx)):
        dw, db = ops.experts_grad_w(*args)
        assert not dw.any() and not db.any()


def test_offsets_and_indices_outside_their_ranges_are_cut():
    """They are on the device and cannot be refused: nothing outside the tensors is read or written."""
    from matris_b200 import ops
    x, w = torch.randn(20, 128, device="cuda"), torch.randn(3, 128, 128, device="cuda")
    idx = torch.randint(-30, 60, (200,), dtype=torch.int32, device="cuda")
    bad = torch.tensor([-5, 100, 90, 1000], dtype=torch.int32, device="cuda")
    good = torch.tensor([0, 100, 100, 200], dtype=torch.int32, device="cuda")
    y = ops.experts_linear(x, w, bad, idx=idx)
    cut = idx.clamp(0, 19)
    want = ops.experts_linear(x, w, good, idx=cut)
    # expert 1 has no slots in either; expert 2 starts at 90 in the first, where expert 0 has written too
    assert torch.equal(y[:90], want[:90]) and torch.equal(y[100:], want[100:])
    slot_of = torch.randint(-9, 300, (20, 3), dtype=torch.int32, device="cuda")
    out = ops.experts_combine_fwd(y, slot_of)
    keep = (slot_of >= 0) & (slot_of < 200)
    want = torch.where(keep.unsqueeze(2), y[slot_of.clamp(0, 199).long()].double(), 0.0).sum(1)
    assert ((out.double() - want).abs() <= 4 * U * torch.where(keep.unsqueeze(2), y[slot_of.clamp(0, 199).long()].double().abs(), 0.0).sum(1)).all()


@pytest.mark.parametrize("n,n_exp,k,width", [(1, 8, 2, 128), (0, 4, 2, 128), (33, 7, 3, 4), (1000, 16, 4, 132), (5000, 8, 1, 128), (70, 40, 32, 512), (129, 9, 5, 1024)])
def test_combine_against_the_definition(n, n_exp, k, width):
    """Sums of k products (k + 1 roundings) and of `width` products (a lane's run of width / 32 of them, then 5 joins)."""
    from matris_b200 import ops
    g = torch.Generator().manual_seed(n + width)
    offsets, _, slot_of = grouped(n, n_exp, k, 3) if n else (torch.zeros(n_exp + 1, dtype=torch.int32, device="cuda"), None, torch.empty(0, k, dtype=torch.int32, device="cuda"))
    y, dout, w = torch.randn(n * k + 5, width, generator=g).cuda(), torch.randn(n, width, generator=g).cuda(), torch.rand(n, k, generator=g).cuda()
    slot_of = slot_of.clone()
    if n > 3:
        slot_of[2] = -1
        slot_of[3, 0] = -1
    at, held = slot_of.clamp(min=0).long(), (slot_of >= 0).unsqueeze(2)
    picked = torch.where(held, y.double()[at], 0.0)
    for weights in (w, None):
        ww = (torch.ones_like(w) if weights is None else w).double().unsqueeze(2)
        out = ops.experts_combine_fwd(y, slot_of, weights)
        assert ((out.double() - (ww * picked).sum(1)).abs() <= (k + 2) * U * (ww * picked).abs().sum(1)).all()
        dy, dw = ops.experts_combine_bwd(dout, y, slot_of, weights, offsets)
        prod = picked * dout.double().unsqueeze(1)
        assert ((dw.double() - prod.sum(2)).abs() <= (width / 32 + 12) * U * prod.abs().sum(2)).all()
        want = (ww * dout.double().unsqueeze(1)).expand(n, k, width)
        rows = slot_of[slot_of >= 0].long()
        assert ((dy[rows].double() - want[slot_of >= 0]).abs() <= U * want[slot_of >= 0].abs()).all()
        assert not dy[n * k:].any()


# ------------------------------------------------------------------ together
def routed_block(ops, x, seg_ptr, p, valid, k):
    """norm -> router -> two dense layers an expert -> weighted sum, and the gradients of a scalar of it."""
    h, stats = ops.group_norm_fwd(x, p["gw"], p["gb"], 8, seg_ptr=seg_ptr, act=1)
    logits = h @ p["wr"].t()
    r = ops.route_fwd(logits, k, valid=valid)
    w1, w2 = ops.ExpertWeights(p["w1"]), ops.ExpertWeights(p["w2"])
    z = ops.experts_linear(h, w1, r.offsets, bias=p["b1"], idx=r.row_of)
    y = ops.experts_linear(z, w2, r.offsets, in_act=1)
    out = ops.experts_combine_fwd(y, r.slot_of, r.weights)
    dy, dweights = ops.experts_combine_bwd(p["dout"], y, r.slot_of, r.weights, r.offsets)
    dz = ops.experts_linear(dy, w2, r.offsets, gate=z, transposed=True)
    dw2, _ = ops.experts_grad_w(dy, z, r.offsets, in_act=1, want_bias=False)
    dw1, db1 = ops.experts_grad_w(dz, h, r.offsets, idx=r.row_of)
    dlogits = ops.route_bwd(logits, r, dweights, p["dloss"])
    dh = ops.experts_combine_fwd(ops.experts_linear(dz, w1, r.offsets, transposed=True), r.slot_of) + dlogits @ p["wr"]
    dx, dgw, dgb = ops.group_norm_bwd(dh, x, p["gw"], p["gb"], stats, 8, seg_ptr=seg_ptr, act=1)
    return dict(out=out, loss=r.loss, dx=dx, dgw=dgw, dgb=dgb, dw1=dw1, db1=db1, dw2=dw2, dwr=dlogits.t() @ h), r


def block_inputs(n_seg, rows, n_exp, seed):
    g = torch.Generator().manual_seed(seed)
    def r(*shape, scale=1.0):
        return (scale * torch.randn(shape, generator=g)).cuda()
    p = dict(gw=1 + r(128, scale=0.1), gb=r(128, scale=0.1), wr=r(n_exp, 128, scale=0.3), w1=r(n_exp, 256, 128, scale=0.09), b1=r(n_exp, 256, scale=0.1),
             w2=r(n_exp, 128, 256, scale=0.06), dout=r(rows, 128), dloss=torch.tensor(3.0, device="cuda"))
    cuts = sorted(torch.randint(0, rows - 6, (n_seg - 1,), generator=g).tolist())
    seg_ptr = torch.tensor([0, *cuts, rows - 6], dtype=torch.int32, device="cuda")
    valid = torch.ones(rows, dtype=torch.bool, device="cuda")
    valid[rows - 6:] = False
    p["dout"][rows - 6:] = 0
    return r(rows, 128), seg_ptr, p, valid


@pytest.mark.parametrize("n_seg,rows,n_exp,k", [(3, 60, 4, 2), (40, 1500, 8, 2)])
def test_a_routed_block_against_autograd(n_seg, rows, n_exp, k):
    """All operators in a run, a padded batch, against automatic differentiation of the definitions in 64 bits with the same choices.
    Outputs are some thousand-term sums of products good to 2^-22: 1e-5 of the tensor's largest value leaves a factor of ten."""
    from matris_b200 import ops
    x, seg_ptr, p, valid = block_inputs(n_seg, rows, n_exp, rows)
    got, r = routed_block(ops, x, seg_ptr, p, valid, k)
    q = {name: t.double() for name, t in p.items()}
    x64 = x.double().requires_grad_()
    leaves = {name: q[name].requires_grad_() for name in ("gw", "gb", "wr", "w1", "b1", "w2")}
    ends = seg_ptr.tolist()
    h = []
    for a, z in zip(ends[:-1], ends[1:]):
        v = x64[a:z].reshape(z - a, 8, 16)
        if z > a:
            v = (v - v.mean((0, 2), keepdim=True)) / torch.sqrt(v.var((0, 2), correction=0, keepdim=True) + 1e-5)
        h.append(silu64(v.reshape(z - a, 128) * leaves["gw"] + leaves["gb"]))
    h = torch.cat(h)
    m = h.shape[0]
    probs = torch.softmax(h @ leaves["wr"].t(), 1)
    ids = r.ids[:m].long()
    w = probs.gather(1, ids)
    w = w / w.sum(1, keepdim=True)
    out = torch.zeros(m, 128, dtype=torch.double, device="cuda")
    for j in range(k):
        e = ids[:, j]
        z = torch.einsum("tk,tnk->tn", h, leaves["w1"][e]) + leaves["b1"][e]
        out = out + w[:, j:j + 1] * torch.einsum("tn,tmn->tm", silu64(z), leaves["w2"][e])
    loss = n_exp / (k * m * m) * (r.counts.double() * probs.sum(0)).sum()
    ((out * q["dout"][:m]).sum() + 3 * loss).backward()
    want = dict(out=out.detach(), loss=loss.detach(), dx=x64.grad, dgw=leaves["gw"].grad, dgb=leaves["gb"].grad, dw1=leaves["w1"].grad,
                db1=leaves["b1"].grad, dw2=leaves["w2"].grad, dwr=leaves["wr"].grad)
    for name, t in want.items():
        u = got[name].double()
        if name == "out":
            assert not u[m:].any()
            u = u[:m]
        assert (u - t).abs().max() <= 1e-5 * t.abs().max(), (name, ((u - t).abs().max() / t.abs().max()).item())


def test_a_routed_block_repeats_in_streams_and_graphs():
    """Same bits on every call, on another stream, and from two captured graphs in turn, with new contents in the captured inputs."""
    from matris_b200 import ops
    sets = [block_inputs(5, 700, 8, s) for s in (1, 2)]
    want = [routed_block(ops, *s, 2)[0] for s in sets]
    for s, w in zip(sets, want):
        got = routed_block(ops, *s, 2)[0]
        assert all(torch.equal(got[name], w[name]) for name in w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = routed_block(ops, *sets[0], 2)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[name], want[0][name]) for name in got)
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = routed_block(ops, *s, 2)[0]
        graphs.append((g, out))
    for _ in range(2):
        for (g, out), w in zip(graphs, want):
            for t in out.values():
                t.fill_(math.nan)
            g.replay()
            assert all(torch.equal(out[name], w[name]) for name in w)
    for a, b in zip(sets[0][:2], sets[1][:2]):
        a.copy_(b)
    for name in sets[0][2]:
        sets[0][2][name].copy_(sets[1][2][name])
    graphs[0][0].replay()
    assert all(torch.equal(graphs[0][1][name], want[1][name]) for name in want[1])
