"""GPU: infinite, undefined and largest finite values in the experts' products."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LARGE = [3.4028234663852886e38, -3.4028234663852886e38, 3.4024e38, 3.4020e38]  # two of them within half a step of 11 bits of 2^128


def alike(got, want, bound):
    """Infinities and NaN where the definition has them, finite values within the bound."""
    got = got.double()
    finite = torch.isfinite(want)
    assert torch.equal(got.isnan(), want.isnan())
    rest = ~finite & ~want.isnan()
    assert torch.equal(got[rest], want[rest])
    assert ((got - want).abs()[finite] <= bound[finite]).all()


def products(n_in, n_out, seed):
    """Three experts, 300 rows; weights of every kind: 24 bits, 11 bits (no second part), zeros."""
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(300, n_in, generator=g), torch.randn(3, n_out, n_in, generator=g) / math.sqrt(n_in)
    w[:, 1::4] = (w[:, 1::4] * 64).round() / 64 + 1 / 64
    w[:, 2::4, ::7] = 0
    offsets = torch.tensor([0, 130, 131, 300], dtype=torch.int32)
    return x.cuda(), w.cuda(), offsets.cuda(), [(0, 0, 130), (1, 130, 131), (2, 131, 300)]


def definition(x, w, spans):
    """Terms in 64 bits, added in 64 bits; a sum with an infinite term is that of its infinite terms."""
    out = torch.empty(x.shape[0], w.shape[1], dtype=torch.double, device="cuda")
    size = torch.empty_like(out)
    for e, a, z in spans:
        for r in range(a, z, 64):
            terms = x[r:min(r + 64, z)].double().unsqueeze(1) * w[e].double().unsqueeze(0)
            out[r:min(r + 64, z)] = terms.sum(2)
            size[r:min(r + 64, z)] = terms.abs().sum(2)
    return out, size


def bound_of(size, k):
    return (2 * 2.0 ** -22 + (k / 8 + 16) * U) * size


@pytest.mark.parametrize("n_in,n_out", [(128, 128), (128, 256), (512, 128)])
def test_infinite_rows(n_in, n_out):
    from matris_b200 import ops
    x, w, offsets, spans = products(n_in, n_out, 1)
    x[3, 5], x[64, 127], x[130, 0], x[200, 77] = math.inf, -math.inf, math.inf, -math.inf
    x[7, 1:3] = math.inf                                    # two of them: NaN where the weights' signs differ
    x[8, n_in - 1], x[250, 9] = math.nan, -math.nan
    want, size = definition(x, w, spans)
    assert want.isinf().any() and want.isnan().any()
    y = ops.experts_linear(x, w, offsets)
    alike(y, want, bound_of(size, n_in))
    y = ops.experts_linear(x, ops.ExpertWeights(w.transpose(1, 2).contiguous()), offsets, transposed=True)
    alike(y, want, bound_of(size, n_in))


@pytest.mark.parametrize("n_in,n_out", [(128, 128), (384, 256)])
def test_infinite_weights(n_in, n_out):
    from matris_b200 import ops
    x, w, offsets, spans = products(n_in, n_out, 2)
    x[::5, 3] = (x[::5, 3] * 64).round() / 64 + 1 / 64       # rows without a second part, and zeros
    x[::7, 3] = 0
    w[0, 5, 3], w[2, 100, n_in - 1], w[1, 0, 0], w[2, 9, 3] = math.inf, -math.inf, -math.inf, math.nan
    want, size = definition(x, w, spans)
    assert want.isinf().any() and want.isnan().any()
    alike(ops.experts_linear(x, w, offsets), want, bound_of(size, n_in))
    alike(ops.experts_linear(x, w.transpose(1, 2).contiguous(), offsets, transposed=True), want, bound_of(size, n_in))


def test_largest_finite_values():
    """Products that stay finite: rows and weights next to 2^128 keep 20 bits (both parts are cut)."""
    from matris_b200 import ops
    x, w, offsets, spans = products(128, 128, 3)
    for i, v in enumerate(LARGE):
        x[40 + i] = 0
        x[40 + i, 30 + i] = v
    w *= 2.0 ** -20
    want, size = definition(x, w, spans)
    assert torch.isfinite(want).all()
    alike(ops.experts_linear(x, w, offsets), want, bound_of(size, 128) + 2.0 ** -20 * size)
    x, w, offsets, spans = products(128, 128, 4)
    w[:, 10] = 0
    w[0, 10, 0], w[1, 10, 1], w[2, 10, 2], w[2, 10, 3] = LARGE
    x *= 2.0 ** -20
    want, size = definition(x, w, spans)
    assert torch.isfinite(want).all()
    alike(ops.experts_linear(x, w, offsets), want, bound_of(size, 128) + 2.0 ** -20 * size)


def test_weight_gradient_of_infinite_rows():
    from matris_b200 import ops
    x, _, offsets, spans = products(128, 128, 5)
    dy = torch.randn(300, 256, device="cuda")
    x[3, 5], dy[140, 200] = math.inf, -math.inf
    dy[131:200, 7], x[260, 100] = 0, math.inf
    x[10, 64], dy[299, 0] = math.nan, math.nan
    dy[50:53], x[50:53] = 0, 0
    dy[50:53, 33], x[50:53, 33] = 2.0 ** -30, LARGE[0]
    dw, db = ops.experts_grad_w(dy, x, offsets)
    for e, a, z in spans:
        want = torch.empty(256, 128, dtype=torch.double, device="cuda")
        size = torch.empty_like(want)
        for n in range(0, 256, 64):
            terms = dy[a:z, n:n + 64].double().t().unsqueeze(2) * x[a:z].double().unsqueeze(0)
            want[n:n + 64], size[n:n + 64] = terms.sum(1), terms.abs().sum(1)
        alike(dw[e], want, bound_of(size, z - a) + 2.0 ** -20 * size)
        alike(db[e], dy[a:z].double().sum(0), bound_of(dy[a:z].double().abs().sum(0), z - a))


def test_an_infinite_row_times_an_infinite_weight_is_undefined():
    """The one product that the two parts of an operand cannot say; and its neighbours are not touched."""
    from matris_b200 import ops
    x, w, offsets, _ = products(128, 128, 6)
    plain = ops.experts_linear(x, w, offsets)
    x[5, 3], w[0, 7, 3] = math.inf, math.inf
    y = ops.experts_linear(x, w, offsets)
    assert y[5, 7].isnan()
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[5], keep[:130, 7] = False, False
    assert torch.equal(y[keep], plain[keep])
