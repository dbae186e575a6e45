"""Group norm with SiLU on the GPU against the definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of float32


def plain(x, w, b, ends, groups, act, eps=1e-5):
    """The definition, segment by segment, in the type of x; rows of no segment are zero."""
    out = []
    at = 0
    for a, z in zip(ends[:-1], ends[1:]):
        out.append(torch.zeros_like(x[at:a]))
        if z > a:
            v = x[a:z].reshape(z - a, groups, -1)
            mean = v.mean((0, 2), keepdim=True)
            v = (v - mean) / torch.sqrt(((v - mean) ** 2).mean((0, 2), keepdim=True) + eps)
            v = v.reshape(z - a, -1) * w + b
            out.append(v * torch.sigmoid(v) if act else v)
        at = max(a, z)
    out.append(torch.zeros_like(x[at:]))
    return torch.cat(out)


def stats_of(x, ends, groups):
    """mean and 1 / deviation of every row's groups, spread over the row's channels (0 and 0 outside the segments)."""
    mean, rstd = torch.zeros_like(x), torch.zeros_like(x)
    for a, z in zip(ends[:-1], ends[1:]):
        if z > a:
            v = x[a:z].reshape(z - a, groups, -1)
            m = v.mean((0, 2), keepdim=True)
            r = torch.rsqrt(((v - m) ** 2).mean((0, 2), keepdim=True) + 1e-5)
            mean[a:z], rstd[a:z] = m.expand_as(v).reshape(z - a, -1), r.expand_as(v).reshape(z - a, -1)
    return mean, rstd


def close(got, want, bound, dtype):
    """|got - want| <= bound (the float32 arithmetic's) + half a step of the output's type."""
    half = torch.finfo(dtype).eps / 2
    tiny = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}[dtype]  # half a step of float16's subnormals
    off = (got.double() - want).abs()
    worst = (off - (bound + half * (want.abs() + bound) + tiny)).max() if off.numel() else torch.tensor(-1.0)
    assert worst <= 0, f"off by up to {off.max():.3g}, {worst:.3g} over the bound"


def inputs(ends, channels, dtype, seed, offset=1.0, rows=None):
    g = torch.Generator().manual_seed(seed)
    rows = ends[-1] if rows is None else rows
    x = torch.randn(rows, channels, generator=g) * (0.5 + torch.rand(channels, generator=g)) + offset * torch.randn(channels, generator=g)
    w, b = 1 + 0.2 * torch.randn(channels, generator=g), 0.2 * torch.randn(channels, generator=g)
    dy = torch.randn(rows, channels, generator=g)
    return x.to(dtype).cuda(), w.cuda(), b.cuda(), dy.to(dtype).cuda(), torch.tensor(ends, dtype=torch.int32, device="cuda")


def check(x, w, b, dy, seg_ptr, groups, act, ends):
    """Forward and backward of ops against the definition.

    Bounds, u = 2^-24.  mean and 1 / deviation come from a tree of joins with at most 48 roundings in a row at these sizes (8 rows of
    a thread, up to 16 such batches, lanes, warps or chunks), each at most u of the running value, and the deviations' squares
    from as many: xh is off by at most 50 u |x| rstd + 50 u |xh|.  z = xh w + b adds 2 u, SiLU (slope at most 1.1) a few more of
    |z|: 64 u in all.  The gradient multiplies dy by SiLU' (off by 8 u plus its slope, at most 0.5, times z's error), w and rstd, and
    subtracts two means of n terms: their sums are trees of at most 64 roundings of sums of magnitudes."""
    from matris_b200 import ops
    y, stats = ops.group_norm_fwd(x, w, b, groups, seg_ptr=seg_ptr, act=act)
    dx, dw, db = ops.group_norm_bwd(dy, x, w, b, stats, groups, seg_ptr=seg_ptr, act=act)
    x64, w64, b64 = (t.double().requires_grad_() for t in (x, w, b))
    want = plain(x64, w64, b64, ends, groups, act) + 0 * (x64.sum() + w64.sum() + b64.sum())  # with no rows, too, it depends on them
    want.backward(dy.double())
    with torch.no_grad():
        mean, rstd = stats_of(x64, ends, groups)
        xh = (x64 - mean) * rstd
        z = (xh * w64).abs() + b64.abs()
        off_z = 64 * U * ((x64.abs() * rstd + xh.abs()) * w64.abs() + z)
        close(y, want.detach(), (1.1 * off_z + 8 * U * z) if act else off_z, x.dtype)
        inside = torch.zeros(x.shape[0], 1, device="cuda", dtype=torch.double)
        inside[ends[0]:ends[-1]] = 1
        g = dy.double().abs() * inside * (1.1 if act else 1.0)
        off_g = (0.5 * off_z if act else 0) * dy.double().abs() * inside + 16 * U * g  # of dz
        # magnitudes of what the two means sum, spread back over rows and channels
        def spread(v):
            out = torch.zeros_like(v)
            for a, e in zip(ends[:-1], ends[1:]):
                if e > a:
                    u = v[a:e].reshape(e - a, groups, -1)
                    out[a:e] = u.mean((0, 2), keepdim=True).expand_as(u).reshape(e - a, -1)
            return out
        off_xh = 64 * U * (x64.abs() * rstd + xh.abs())
        gw, ow = g * w64.abs(), off_g * w64.abs()
        m1, m2 = spread(ow + 64 * U * gw), spread(ow * xh.abs() + gw * off_xh + 64 * U * gw * xh.abs())
        top = spread(gw * xh.abs())
        off_dx = rstd * (ow + m1 + xh.abs() * m2 + off_xh * top + 8 * U * (gw + spread(gw) + xh.abs() * top)) + 64 * U * x64.grad.abs()
        close(dx, x64.grad, off_dx, x.dtype)
        close(db, b64.grad, (off_g + 64 * U * g).sum(0), torch.float32)
        close(dw, w64.grad, (off_g * xh.abs() + g * off_xh + 64 * U * g * xh.abs()).sum(0), torch.float32)
    return y, stats, dx, dw, db


CASES = [  # offsets, channels, groups
    ([0, 1], 128, 8), ([0, 32], 128, 8), ([0, 0, 5, 5, 6, 40, 41], 128, 8), ([0, 17, 64], 32, 32), ([0, 33], 128, 1), ([0, 33], 96, 4),
    ([0, 7, 30], 7, 7), ([0, 7, 30], 7, 1), ([0, 3, 31], 130, 10), ([0, 13], 1, 1), ([0, 9, 30], 1024, 4), ([0, 9, 30], 1022, 2),
    ([0, 9, 30], 160, 5), ([0, 20, 5000, 5000, 5003, 9800], 128, 8), ([0, 9001], 128, 16), ([0, 4096, 8193], 64, 2), ([0, 6000], 320, 32),
    ([0, 5001, 5001, 12000], 36, 6), ([0, 4999, 5030], 30, 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ends,channels,groups", CASES)
def test_against_the_definition(ends, channels, groups, dtype):
    act = (len(ends) + channels) % 2 if channels != 128 else 1
    x, w, b, dy, seg_ptr = inputs(ends, channels, dtype, 3)
    check(x, w, b, dy, seg_ptr, groups, act, ends)
    check(x, w, b, dy, seg_ptr, groups, 1 - act, ends)


@pytest.mark.parametrize("offset", [1e2, 1e4])
@pytest.mark.parametrize("ends", [[0, 40, 90], [0, 7000]])
def test_offsets_of_many_deviations(ends, offset):
    """Variances are taken from deviations: a large common offset costs the rounding of the inputs and no more."""
    x, w, b, dy, seg_ptr = inputs(ends, 128, torch.float32, 4, offset=0.0)
    check(x + offset, w, b, dy, seg_ptr, 8, 1, ends)


def test_constant_rows_and_no_affine():
    from matris_b200 import ops
    x = torch.full((50, 128), 3.0, device="cuda")
    seg_ptr = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    y, stats = ops.group_norm_fwd(x, None, None, 4, seg_ptr=seg_ptr)
    assert torch.equal(y, torch.zeros_like(y))
    dx, dw, db = ops.group_norm_bwd(torch.ones_like(x), x, None, None, stats, 4, seg_ptr=seg_ptr, want_affine=False)
    assert torch.equal(dx, torch.zeros_like(dx)) and dw is None and db is None


@pytest.mark.parametrize("ends", [[3, 10, 30], [2, 6000, 6400], [5, 5], [0, 0]])
def test_rows_of_no_segment(ends):
    """Zero in a returned tensor, left as they are in a given one."""
    from matris_b200 import ops
    rows = ends[-1] + 9
    x, w, b, dy, seg_ptr = inputs(ends, 128, torch.float32, 5, rows=rows)
    y, stats, dx, dw, db = check(x, w, b, dy, seg_ptr, 8, 1, ends)
    for t in (y, dx):
        assert not t[:ends[0]].any() and not t[ends[-1]:].any()
    for call, want in ((lambda o: ops.group_norm_fwd(x, w, b, 8, seg_ptr=seg_ptr, act=1, out=o)[0], y),
                       (lambda o: ops.group_norm_bwd(dy, x, w, b, stats, 8, seg_ptr=seg_ptr, act=1, out=o)[0], dx)):
        out = torch.full_like(x, float("nan"))
        assert call(out) is out
        assert torch.equal(out[ends[0]:ends[-1]], want[ends[0]:ends[-1]])
        assert out[:ends[0]].isnan().all() and out[ends[-1]:].isnan().all()


@pytest.mark.parametrize("ends,channels", [([0, 12, 50], 128), ([0, 5200], 128), ([0, 12, 50], 30)])
def test_strides_alignment_and_in_place(ends, channels):
    from matris_b200 import ops
    x, w, b, dy, seg_ptr = inputs(ends, channels, torch.float32, 6)
    y, stats, dx, dw, db = check(x, w, b, dy, seg_ptr, 2, 1, ends)
    for shift in (0, 1, 4):  # columns of a wider tensor: aligned to 16 bytes or not
        wide = torch.zeros(x.shape[0], channels + 12, device="cuda")
        wide[:, shift:shift + channels] = x
        xs = wide[:, shift:shift + channels]
        check(xs, w, b, dy, seg_ptr, 2, 1, ends)
    here = x.clone()
    ops.group_norm_fwd(here, w, b, 2, seg_ptr=seg_ptr, act=1, out=here)
    assert torch.equal(here, y)
    here = dy.clone()
    ops.group_norm_bwd(here, x, w, b, stats, 2, seg_ptr=seg_ptr, act=1, out=here)
    assert torch.equal(here, dx)


@pytest.mark.parametrize("shape", [(1, 128), (3, 5, 7, 64), (2, 90, 100, 32), (4, 0, 32), (0, 5, 32)])
def test_dense_batches(shape):
    """[batch, .., channels] without offsets: the same bits as with them."""
    from matris_b200 import ops
    g = torch.Generator().manual_seed(7)
    x, dy = torch.randn(shape, generator=g).cuda(), torch.randn(shape, generator=g).cuda()
    channels, per = shape[-1], int(torch.tensor(shape[1:-1]).prod()) if len(shape) > 2 else 1
    ends = [per * i for i in range(shape[0] + 1)]
    seg_ptr = torch.tensor(ends, dtype=torch.int32, device="cuda")
    w, b = torch.randn(channels, generator=g).cuda(), torch.randn(channels, generator=g).cuda()
    y, stats = ops.group_norm_fwd(x, w, b, 4, act=1)
    dx, dw, db = ops.group_norm_bwd(dy, x, w, b, stats, 4, act=1)
    y2, s2, dx2, dw2, db2 = check(x.view(ends[-1], channels), w, b, dy.view(ends[-1], channels), seg_ptr, 4, 1, ends)
    assert y.shape == x.shape and dx.shape == x.shape
    assert torch.equal(y.view_as(y2), y2) and torch.equal(dx.view_as(dx2), dx2) and torch.equal(dw, dw2) and torch.equal(db, db2)


def test_gradient_against_differences():
    """<dx, v> against (L(x + h v) - L(x - h v)) / 2 h of the definition in 64 bits, L = <y, dy>: the quotient is off by h^2 times a
    third derivative of order one times the number of values it sums, and the kernel by the bounds of ``check``."""
    from matris_b200 import ops
    ends = [0, 9, 31]
    x, w, b, dy, seg_ptr = inputs(ends, 128, torch.float32, 8)
    _, stats = ops.group_norm_fwd(x, w, b, 8, seg_ptr=seg_ptr, act=1)
    dx, dw, db = ops.group_norm_bwd(dy, x, w, b, stats, 8, seg_ptr=seg_ptr, act=1)
    h = 1e-4
    for which, grad in ((0, dx), (1, dw), (2, db)):
        at = [x.double(), w.double(), b.double()]
        v = torch.randn(at[which].shape, generator=torch.Generator().manual_seed(9)).double().cuda()
        value = []
        for s in (1, -1):
            moved = list(at)
            moved[which] = at[which] + s * h * v
            value.append((plain(*moved, ends, 8, 1) * dy.double()).sum())
        want, got = (value[0] - value[1]) / (2 * h), (grad.double() * v).sum()
        size = (grad.double().abs() * v.abs()).sum()
        assert (got - want).abs() <= 1e-5 * size, (got, want, size)


def test_repeats_streams_and_graphs():
    """The same bits on every call, on another stream, and from two captured graphs whose replays alternate."""
    from matris_b200 import ops
    ends = [0, 30, 5200, 5230, 11000]
    args = [inputs(ends, 128, torch.float32, s) for s in (10, 11)]

    def step(x, w, b, dy, seg_ptr):
        y, stats = ops.group_norm_fwd(x, w, b, 8, seg_ptr=seg_ptr, act=1)
        return y, *ops.group_norm_bwd(dy, x, w, b, stats, 8, seg_ptr=seg_ptr, act=1)

    want = [step(*a) for a in args]
    for a, w in zip(args, want):
        assert all(torch.equal(p, q) for p, q in zip(step(*a), w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*args[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(other, want[0]))
    graphs = []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*a)
        graphs.append((g, out))
    for _ in range(2):
        for (g, out), w in zip(graphs, want):
            for t in out:
                t.fill_(float("nan"))
            g.replay()
            assert all(torch.equal(p, q) for p, q in zip(out, w))


def test_offsets_outside_the_rows_are_cut():
    """Offsets are on the device and cannot be refused: they are cut to the rows that are there, and nothing else is touched."""
    from matris_b200 import ops
    x, w, b, dy, _ = inputs([0, 50], 128, torch.float32, 12)
    seg_ptr = torch.tensor([-7, 20, 90], dtype=torch.int32, device="cuda")
    y, _ = ops.group_norm_fwd(x, w, b, 8, seg_ptr=seg_ptr, act=1)
    want, _ = ops.group_norm_fwd(x, w, b, 8, seg_ptr=torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda"), act=1)
    assert torch.equal(y, want)
