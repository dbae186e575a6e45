"""Routed dense layers and segment norms: the cases they are measured on.

Four operators of ``matris_b200.ops``: a group norm over the rows of every structure (with SiLU, forward and
backward), the router of a mixture of experts (top-k, balance loss, per-expert counts, grouping of the rows, and its
gradient), the experts' dense products (gathered rows, data and weight gradients) and the weighted sum of their
outputs.  ``own`` selects the library's kernels; otherwise ``run`` is the same mathematics in elementary torch
operations.
"""
import math
import random

import torch

own = False

ACT_SILU = 1
EPS = 1e-5


def listed():
    return [
        # one small crystal in a relaxation or MD loop: latency
        dict(name="norm one crystal", op="norm", train=False, dtype="float32", rows=32, segments=1, spread=1.0, channels=128, groups=8, act=True),
        # a batch of 256 random crystals of 8-64 atoms, a training step on atom features
        dict(name="norm crystals train", op="norm", train=True, dtype="float32", rows=9216, segments=256, spread=8.0, channels=128, groups=8, act=True),
        # bond features of a batch of 512 forty-atom cells, a training step: the largest
        dict(name="norm bonds train", op="norm", train=True, dtype="float32", rows=573894, segments=512, spread=1.5, channels=128, groups=8, act=True),
        # both halves of a gated layer's features of one large cell, kept in 16 bits
        dict(name="norm cell bf16", op="norm", train=False, dtype="bfloat16", rows=409601, segments=1, spread=1.0, channels=256, groups=32, act=True),
        # one row through a small router
        dict(name="route one row", op="route", train=False, dtype="float32", rows=1, experts=8, top_k=2, renorm=True, padded=0, barred=0.0),
        # atoms of a 16,000-atom cell over many experts, with padded rows and experts that some rows may not take
        dict(name="route atoms train", op="route", train=True, dtype="bfloat16", rows=16000, experts=64, top_k=6, renorm=False, padded=500, barred=0.1),
        # bonds of a batch
        dict(name="route bonds train", op="route", train=True, dtype="float32", rows=573894, experts=32, top_k=2, renorm=True, padded=0, barred=0.0),
        # one small crystal through eight experts
        dict(name="experts one crystal", op="experts", train=False, rows=32, experts=8, top_k=2, width_in=128, width_out=128, act=True),
        # atoms of a 16,000-atom cell, the first layer of a gated pair (256 wide), a training step
        dict(name="experts atoms train", op="experts", train=True, rows=16000, experts=16, top_k=2, width_in=128, width_out=256, act=False),
        # bonds of a batch, a training step
        dict(name="experts bonds train", op="experts", train=True, rows=286947, experts=32, top_k=2, width_in=256, width_out=128, act=False),
        # a 4,096-atom cell in MD
        dict(name="combine atoms", op="combine", train=False, rows=4096, experts=16, top_k=4, width=128),
        # bonds of a batch, a training step
        dict(name="combine bonds train", op="combine", train=True, rows=286947, experts=32, top_k=2, width=128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "route", "route", "experts", "experts", "combine"])
    train = rng.random() < 0.6
    if op == "norm":
        channels = rng.choice([32, 64, 96, 128, 160, 256, 320, 512])
        groups = rng.choice([g for g in (1, 2, 4, 8, 16, 32) if channels % g == 0])
        rows = _log_int(rng, 16, 70_000_000 // channels)
        segments = min(rows, _log_int(rng, 1, 2048))
        return dict(op=op, train=train, dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]), rows=rows, segments=segments,
                    spread=rng.choice([1.0, 2.0, 8.0, 30.0]), channels=channels, groups=groups, act=rng.random() < 0.75)
    if op == "route":
        experts = rng.choice([4, 7, 8, 16, 24, 32, 60, 64, 128, 256])
        rows = _log_int(rng, 1, min(573894, 18_000_000 // experts))
        top_k = rng.randint(1, min(8, experts))
        return dict(op=op, train=train, dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]), rows=rows, experts=experts, top_k=top_k,
                    renorm=rng.random() < 0.5, padded=rng.choice([0, 0, rows // 9]), barred=rng.choice([0.0, 0.0, 0.1, 0.4]))
    experts = rng.choice([2, 4, 7, 8, 16, 32, 48, 64])
    top_k = rng.randint(1, min(4, experts))
    if op == "experts":
        width_in, width_out = rng.choice([128, 128, 256, 384, 512]), rng.choice([128, 128, 256, 384, 512])
        most = int(573894 * 128 * 256 / (width_in * width_out * top_k))
        return dict(op=op, train=train, rows=_log_int(rng, 1, most), experts=experts, top_k=top_k, width_in=width_in, width_out=width_out,
                    act=not train and rng.random() < 0.5)
    width = rng.choice([128, 128, 256, 512])
    return dict(op=op, train=train, rows=_log_int(rng, 1, 573894 * 128 // (width * top_k)), experts=experts, top_k=top_k, width=width)


# ------------------------------------------------------------------ inputs
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _row_ranges(case, seed):
    """Offsets of the structures' rows: sizes spread over a factor, their sum as the case says."""
    r = random.Random(seed)
    sizes = [r.uniform(1.0, case["spread"]) for _ in range(case["segments"])]
    scale, at, offsets = case["rows"] / sum(sizes), 0.0, [0]
    for s in sizes:
        at += s * scale
        offsets.append(min(case["rows"], round(at)))
    offsets[-1] = case["rows"]
    return torch.tensor(offsets, dtype=torch.int32)


def _assignment(case, gen):
    """Experts of every row, as skewed as a router's, and the grouping of the rows by expert (in row order within an expert)."""
    n, k, n_exp = case["rows"], case["top_k"], case["experts"]
    score = _normal(gen, n, n_exp) + 0.7 * _normal(gen, 1, n_exp)
    ids = score.topk(k, dim=1).indices
    order = torch.argsort(ids.reshape(-1), stable=True)
    slot_of = torch.empty(n * k, dtype=torch.int32, device="cuda")
    slot_of[order] = torch.arange(n * k, dtype=torch.int32, device="cuda")
    counts = (ids.reshape(-1, 1) == torch.arange(n_exp, device="cuda")).sum(0) if n * k * n_exp < 1 << 27 else torch.bincount(ids.reshape(-1), minlength=n_exp)
    offsets = torch.zeros(n_exp + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    row_of = (order // k).to(torch.int32)
    return dict(offsets=offsets, row_of=row_of, slot_of=slot_of.view(n, k), most=int(counts.max()))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(case=case)
    op = case["op"]
    if op == "norm":
        dtype, rows, ch = getattr(torch, case["dtype"]), case["rows"], case["channels"]
        # features after a few layers: channels with offsets and scales of their own
        x = _normal(gen, rows, ch) * (0.5 + torch.rand(ch, generator=gen, device="cuda")) + _normal(gen, ch)
        state.update(x=x.to(dtype), seg_ptr=_row_ranges(case, seed).cuda(), weight=1 + 0.2 * _normal(gen, ch), bias=0.2 * _normal(gen, ch))
        if case["train"]:
            state["dy"] = _normal(gen, rows, ch).to(dtype)
    elif op == "route":
        dtype, n, n_exp = getattr(torch, case["dtype"]), case["rows"], case["experts"]
        logits = 1.5 * _normal(gen, n, n_exp) + 0.5 * _normal(gen, 1, n_exp)
        if case["barred"]:
            logits[torch.rand(n, n_exp, generator=gen, device="cuda") < case["barred"]] = -math.inf
        state["logits"] = logits.to(dtype)
        state["valid"] = None
        if case["padded"]:
            keep = torch.ones(n, dtype=torch.bool, device="cuda")
            keep[torch.randperm(n, generator=gen, device="cuda")[: case["padded"]]] = False
            state["valid"] = keep
        if case["train"]:
            # gradients of a mean over the rows, and the usual size of the balance loss's coefficient
            state["dweights"] = _normal(gen, n, case["top_k"]) / n
            state["dloss"] = torch.full((), 0.1, device="cuda") * (1 + torch.rand((), generator=gen, device="cuda"))
    elif op == "experts":
        n, k, width_in, width_out = case["rows"], case["top_k"], case["width_in"], case["width_out"]
        state.update(_assignment(case, gen))
        state["x"] = _normal(gen, n, width_in)
        state["weight"] = _normal(gen, case["experts"], width_out, width_in) / math.sqrt(width_in)
        state["bias"] = 0.1 * _normal(gen, case["experts"], width_out)
        if case["train"]:
            state["dy"] = _normal(gen, n * k, width_out)
        elif own:  # weights that do not change are laid out once; a training step lays them out itself
            from matris_b200 import ops
            state["laid_out"] = ops.ExpertWeights(state["weight"])
    else:
        n, k = case["rows"], case["top_k"]
        state.update(_assignment(case, gen))
        state["y"] = _normal(gen, n * k, case["width"])
        state["weights"] = torch.softmax(_normal(gen, n, k), dim=1)
        if case["train"]:
            state["dout"] = _normal(gen, n, case["width"])
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        from matris_b200 import ops
        return {"norm": _own_norm, "route": _own_route, "experts": _own_experts, "combine": _own_combine}[case["op"]](ops, case, state)
    return {"norm": _norm, "route": _route, "experts": _experts, "combine": _combine}[case["op"]](case, state)


def _own_norm(ops, case, s):
    act = ACT_SILU if case["act"] else 0
    y, stats = ops.group_norm_fwd(s["x"], s["weight"], s["bias"], case["groups"], seg_ptr=s["seg_ptr"], eps=EPS, act=act)
    if not case["train"]:
        return dict(y=y)
    dx, dweight, dbias = ops.group_norm_bwd(s["dy"], s["x"], s["weight"], s["bias"], stats, case["groups"], seg_ptr=s["seg_ptr"], act=act)
    return dict(y=y, dx=dx, dweight=dweight, dbias=dbias)


def _own_route(ops, case, s):
    r = ops.route_fwd(s["logits"], case["top_k"], valid=s["valid"], renorm=case["renorm"])
    out = dict(ids=r.ids, weights=r.weights, counts=r.counts, loss=r.loss, offsets=r.offsets, row_of=r.row_of, slot_of=r.slot_of)
    if case["train"]:
        out["dlogits"] = ops.route_bwd(s["logits"], r, s["dweights"], s["dloss"])
    return out


def _own_experts(ops, case, s):
    if not case["train"]:
        return dict(y=ops.experts_linear(s["x"], s["laid_out"], s["offsets"], bias=s["bias"], idx=s["row_of"], out_act=ACT_SILU if case["act"] else 0))
    w = ops.ExpertWeights(s["weight"])
    y = ops.experts_linear(s["x"], w, s["offsets"], bias=s["bias"], idx=s["row_of"])
    dx = ops.experts_linear(s["dy"], w, s["offsets"], transposed=True)
    dweight, dbias = ops.experts_grad_w(s["dy"], s["x"], s["offsets"], idx=s["row_of"])
    return dict(y=y, dx=dx, dweight=dweight, dbias=dbias)


def _own_combine(ops, case, s):
    out = ops.experts_combine_fwd(s["y"], s["slot_of"], s["weights"])
    if not case["train"]:
        return dict(out=out)
    dy, dweights = ops.experts_combine_bwd(s["dout"], s["y"], s["slot_of"], s["weights"], s["offsets"])
    return dict(out=out, dy=dy, dweights=dweights)


# ------------------------------------------------------------------ plain forms
def _segment_sums(v, seg_ptr):
    """[rows, G] -> [segments, G], summed in 64 bits."""
    total = torch.zeros(v.shape[1], v.shape[0] + 1, dtype=torch.float64, device=v.device)
    torch.cumsum(v.double().t().contiguous(), 1, out=total[:, 1:])
    total = total.t()
    at = seg_ptr.long()
    return total[at[1:]] - total[at[:-1]]


def _norm(case, s):
    x, seg_ptr, groups = s["x"], s["seg_ptr"].long(), case["groups"]
    rows, ch = x.shape
    x = x.float().view(rows, groups, ch // groups)
    w, b = s["weight"].view(groups, -1), s["bias"].view(groups, -1)
    size = (seg_ptr[1:] - seg_ptr[:-1]).double().clamp(min=1).unsqueeze(1) * (ch // groups)
    seg = torch.repeat_interleave(torch.arange(case["segments"], device=x.device), seg_ptr[1:] - seg_ptr[:-1], output_size=rows)
    mean = (_segment_sums(x.sum(2), seg_ptr) / size).float()
    x = x - mean[seg].unsqueeze(2)
    rstd = torch.rsqrt((_segment_sums((x * x).sum(2), seg_ptr) / size).float() + EPS)
    xh = x * rstd[seg].unsqueeze(2)
    z = xh * w + b
    sig = torch.sigmoid(z)
    y = (z * sig if case["act"] else z).view(rows, ch).to(s["x"].dtype)
    if not case["train"]:
        return dict(y=y)
    dz = s["dy"].float().view(rows, groups, -1)
    if case["act"]:
        dz = dz * sig * (1 + z * (1 - sig))
    dbias = dz.view(rows, ch).double().sum(0).float()
    dweight = (dz * xh).view(rows, ch).double().sum(0).float()
    g = dz * w
    m1 = (_segment_sums(g.sum(2), seg_ptr) / size).float()
    m2 = (_segment_sums((g * xh).sum(2), seg_ptr) / size).float()
    dx = (g - m1[seg].unsqueeze(2) - xh * m2[seg].unsqueeze(2)) * rstd[seg].unsqueeze(2)
    return dict(y=y, dx=dx.view(rows, ch).to(s["x"].dtype), dweight=dweight, dbias=dbias)


def _route(case, s):
    n, n_exp, k = case["rows"], case["experts"], case["top_k"]
    l = s["logits"].float()
    routed = l.amax(1) > -math.inf
    if s["valid"] is not None:
        routed = routed & s["valid"]
    top = l.sort(dim=1, descending=True, stable=True)
    ids = top.indices[:, :k]
    held = routed.unsqueeze(1) & (top.values[:, :k] > -math.inf)
    p = torch.exp(l - torch.where(routed, top.values[:, 0], 0.0).unsqueeze(1)).masked_fill(~routed.unsqueeze(1), 0.0)
    p = p / p.sum(1, keepdim=True).clamp(min=1e-30)
    ids = ids.masked_fill(~held, -1)
    weights = p.gather(1, ids.clamp(min=0).long()) * held
    if case["renorm"]:
        weights = weights / weights.sum(1, keepdim=True).clamp(min=1e-30)
    flat = ids.reshape(-1).masked_fill(~held.reshape(-1), n_exp)
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=n_exp + 1)[:n_exp]
    offsets = torch.zeros(n_exp + 1, dtype=torch.int32, device=l.device)
    offsets[1:] = counts.cumsum(0)
    place = torch.arange(n * k, device=l.device)
    slot_of = torch.empty_like(place)
    slot_of[order] = place
    slot_of = slot_of.masked_fill(~held.reshape(-1), -1).view(n, k).int()
    row_of = (order // k).masked_fill(place >= offsets[-1], -1).int()
    rows = routed.sum().double().clamp(min=1)
    share = counts.double() * (n_exp / k) / (rows * rows)  # d loss / d p
    loss = (share * p.double().sum(0)).sum().float()
    out = dict(ids=ids.int(), weights=weights, counts=counts.int(), loss=loss, offsets=offsets, row_of=row_of, slot_of=slot_of)
    if not case["train"]:
        return out
    g = (s["dloss"] * share).float().expand(n, n_exp)
    dw = s["dweights"] * held
    at = ids.clamp(min=0).long()
    if not case["renorm"]:
        g = g.scatter_add(1, at, dw)
    dl = p * (g - (p * g).sum(1, keepdim=True))
    if case["renorm"]:
        dl = dl.scatter_add(1, at, weights * (dw - (weights * dw).sum(1, keepdim=True)))
    out["dlogits"] = dl.to(s["logits"].dtype)
    return out


def _experts(case, s):
    n_exp, width_in = case["experts"], case["width_in"]
    slots, most = case["rows"] * case["top_k"], s["most"]
    offsets = s["offsets"].long()
    place = torch.arange(slots, device="cuda")
    expert = torch.bucketize(place, offsets[1:], right=True)
    at = expert * most + place - offsets[expert]  # the slot's row in a layout with room for `most` rows an expert
    x = torch.zeros(n_exp * most, width_in, device="cuda")
    x[at] = s["x"][s["row_of"].long()]
    x = x.view(n_exp, most, width_in)
    y = torch.bmm(x, s["weight"].transpose(1, 2)) + s["bias"].unsqueeze(1)
    y = y.view(n_exp * most, -1)[at]
    if case["act"]:
        y = y * torch.sigmoid(y)
    if not case["train"]:
        return dict(y=y)
    dy = torch.zeros(n_exp * most, case["width_out"], device="cuda")
    dy[at] = s["dy"]
    dy = dy.view(n_exp, most, -1)
    dx = torch.bmm(dy, s["weight"]).view(n_exp * most, -1)[at]
    return dict(y=y, dx=dx, dweight=torch.bmm(dy.transpose(1, 2), x), dbias=dy.double().sum(1).float())


def _combine(case, s):
    n, k = case["rows"], case["top_k"]
    at = s["slot_of"].long()
    y = s["y"][at]
    out = (s["weights"].unsqueeze(2) * y).sum(1)
    if not case["train"]:
        return dict(out=out)
    dy = torch.empty_like(s["y"])
    dy[at.reshape(-1)] = (s["weights"].unsqueeze(2) * s["dout"].unsqueeze(1)).view(n * k, -1)
    return dict(out=out, dy=dy, dweights=(s["dout"].unsqueeze(1) * y).sum(2))


# ------------------------------------------------------------------ bytes and operations
def work(case):
    n, op, train = case["rows"], case["op"], case["train"]
    if op == "norm":
        values, size = n * case["channels"], 4 if case["dtype"] == "float32" else 2
        # read x, write y; the backward pass: read dy, write dx
        return dict(bytes=values * size * (4 if train else 2) + 8 * case["channels"] * (2 if train else 1) + 4 * case["segments"],
                    flops=values * (30 if train else 12))
    if op == "route":
        size, k, n_exp = (4 if case["dtype"] == "float32" else 2), case["top_k"], case["experts"]
        return dict(bytes=n * n_exp * size * (2 if train else 1) + n * k * (20 if train else 16) + 8 * n_exp + (n if case["padded"] else 0),
                    flops=n * n_exp * (14 if train else 8))
    slots = n * case["top_k"]
    if op == "experts":
        a, b, e = case["width_in"], case["width_out"], case["experts"]
        weights = 4 * e * (a + 1) * b
        if not train:
            return dict(bytes=4 * (n * a + slots * b + slots) + weights, flops=2 * slots * a * b)
        return dict(bytes=4 * (n * a + 2 * slots * b + slots * a + slots) + 2 * weights, flops=6 * slots * a * b)
    w = case["width"]
    return dict(bytes=4 * (slots * w * (2 if train else 1) + n * w * (2 if train else 1) + slots * (3 if train else 2)),
                flops=slots * w * (5 if train else 2))


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    return {"norm": _exact_norm, "route": _exact_route, "experts": _exact_experts, "combine": _exact_combine}[case["op"]](case, s)


def _exact_norm(case, s):
    groups, ch, ends = case["groups"], case["channels"], s["seg_ptr"].tolist()
    out = {name: torch.zeros_like(s["x"]) for name in (("y", "dx") if case["train"] else ("y",))}
    dweight, dbias = torch.zeros_like(s["weight"]), torch.zeros_like(s["bias"])
    for a, b in zip(ends[:-1], ends[1:]):
        if a == b:
            continue
        block = s["x"][a:b].reshape(b - a, groups, ch // groups)
        var, mean = torch.var_mean(block, dim=(0, 2), correction=0, keepdim=True)
        scale = 1 / torch.sqrt(var + EPS)
        xh = (block - mean) * scale
        z = (xh.reshape(b - a, ch) * s["weight"] + s["bias"])
        e = 1 / (1 + torch.exp(-z))
        out["y"][a:b] = z * e if case["act"] else z
        if case["train"]:
            dz = s["dy"][a:b]
            if case["act"]:
                dz = dz * (e + z * e * (1 - e))
            dbias += dz.sum(0)
            dweight += (dz * xh.reshape(b - a, ch)).sum(0)
            g = (dz * s["weight"]).reshape(b - a, groups, -1)
            dx = scale * (g - g.mean(dim=(0, 2), keepdim=True) - xh * (g * xh).mean(dim=(0, 2), keepdim=True))
            out["dx"][a:b] = dx.reshape(b - a, ch)
    if case["train"]:
        out.update(dweight=dweight, dbias=dbias)
    return out


def _exact_route(case, s):
    l, k, n_exp = s["logits"], case["top_k"], case["experts"]
    usable = torch.isfinite(l).any(1)
    if s["valid"] is not None:
        usable &= s["valid"]
    p = torch.zeros_like(l)
    p[usable] = torch.softmax(l[usable], dim=1)
    # the k largest, one after another, the lowest index among equals
    left = l.masked_fill(~usable.unsqueeze(1), -math.inf)
    lanes = torch.arange(n_exp, device=l.device)
    chosen, taken = [], torch.zeros_like(l, dtype=torch.bool)
    for _ in range(k):
        best = left.amax(1, keepdim=True)
        at = torch.where((left == best) & (best > -math.inf) & ~taken, lanes, n_exp).amin(1)
        chosen.append(at)
        hit = lanes == at.unsqueeze(1)
        taken |= hit
        left = left.masked_fill(hit, -math.inf)
    ids = torch.stack(chosen, 1)
    held = ids < n_exp
    weights = torch.where(held, p.gather(1, ids.clamp(max=n_exp - 1)), 0.0)
    total = weights.sum(1, keepdim=True)
    if case["renorm"]:
        weights = torch.where(held, weights / total.clamp(min=1e-300), 0.0)
    rows = max(1, int(usable.sum()))
    share = taken.sum(0).double() / (k * rows)
    loss = n_exp * (share * (p.sum(0) / rows)).sum()
    out = dict(ids=None, weights=weights, counts=None, loss=loss, offsets=None, row_of=None, slot_of=None)
    if case["train"]:
        # by the product rule, through the softmax's Jacobian p_i (delta_ij - p_j)
        dw = torch.where(held, s["dweights"], 0.0)
        if case["renorm"]:
            dw = torch.where(held, (dw - (dw * weights).sum(1, keepdim=True)) / total.clamp(min=1e-300), 0.0)
        dp = s["dloss"] * n_exp * share / rows * usable.unsqueeze(1)
        dp = torch.cat([dp, torch.zeros_like(dp[:, :1])], 1).scatter_add(1, ids, dw)[:, :n_exp]
        out["dlogits"] = p * dp - p * (p * dp).sum(1, keepdim=True)
    return out


def _exact_experts(case, s):
    ends = s["offsets"].tolist()
    x = s["x"][s["row_of"].long()]
    y = torch.empty(x.shape[0], case["width_out"], dtype=torch.float64, device=x.device)
    dx, dweight, dbias = torch.empty_like(x), torch.zeros_like(s["weight"]), torch.zeros_like(s["bias"])
    for e, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
        y[a:b] = torch.addmm(s["bias"][e], x[a:b], s["weight"][e].t())
        if case["train"]:
            dx[a:b] = s["dy"][a:b] @ s["weight"][e]
            dweight[e] = s["dy"][a:b].t() @ x[a:b]
            dbias[e] = s["dy"][a:b].sum(0)
    if case["act"]:
        y = y / (1 + torch.exp(-y))
    return dict(y=y, dx=dx, dweight=dweight, dbias=dbias) if case["train"] else dict(y=y)


def _exact_combine(case, s):
    out = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda")
    dy, dweights = torch.zeros_like(s["y"]), torch.zeros_like(s["weights"])
    for j in range(case["top_k"]):
        at, w = s["slot_of"][:, j].long(), s["weights"][:, j: j + 1]
        out += w * s["y"][at]
        if case["train"]:
            dy[at] = w * s["dout"]
            dweights[:, j] = torch.einsum("tc,tc->t", s["dout"], s["y"][at])
    return dict(out=out, dy=dy, dweights=dweights) if case["train"] else dict(out=out)
