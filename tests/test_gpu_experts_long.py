"""GPU: experts with hundreds of thousands of slots - sums whose error must not grow with their length."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def bound(rows, shares):
    """Relative to the sum of the terms' sizes: operands good to 2^-22 each; a run of 4,096 rows in float32, each 8 to an addition (with
    eight of a tree); the runs of a share in a row, and the shares."""
    return 2 * 2.0 ** -22 + (4096 / 8 + 16) * U + (rows / 4096 + shares) * U


@pytest.mark.parametrize("sizes,n_in,n_out", [([400_000], 1024, 1024), ([300_001, 70, 99_990], 1024, 1024), ([5, 900_000, 4097], 128, 256),
                                              ([700_000, 0, 1, 500_000], 256, 128)])
def test_weight_gradients_of_long_experts(sizes, n_in, n_out):
    """Values that are rounded the same way every time: what each addition loses has one sign for long stretches."""
    from matris_b200 import ops
    n = sum(sizes)
    offsets = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(n)
    row, col = torch.rand(n_out, device="cuda", generator=g) + 0.1, torch.rand(n_in, device="cuda", generator=g) + 0.1
    dy, x = row.expand(n, n_out).contiguous(), col.expand(n, n_in).contiguous()
    dw, db = ops.experts_grad_w(dy, x, offsets)
    for e, rows in enumerate(sizes):
        want = rows * row.double().unsqueeze(1) * col.double().unsqueeze(0)
        off = ((dw[e].double() - want).abs() - bound(rows, 148) * want).max()
        print(f"expert {e} of {rows}: dw off by {((dw[e].double() - want).abs() / want.clamp(min=1e-30)).max():.2e}, "
              f"bias by {((db[e].double() - rows * row.double()).abs() / (rows * row.double()).clamp(min=1e-30)).max():.2e}, bound {bound(rows, 148):.2e}")
        assert off <= 0
        assert ((db[e].double() - rows * row.double()).abs() <= bound(rows, 148) * rows * row.double()).all()


def test_wide_experts_against_the_definition():
    """1024 -> 1024, three directions, runs that are folded and runs that are not."""
    from matris_b200 import ops
    sizes = [9000, 3, 0, 20_000]
    n = sum(sizes)
    offsets = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = torch.randn(n, 1024, device="cuda", generator=g), torch.randn(n, 1024, device="cuda", generator=g)
    w = torch.randn(4, 1024, 1024, device="cuda", generator=g) / 32
    y, dx = ops.experts_linear(x, w, offsets), ops.experts_linear(dy, w, offsets, transposed=True)
    dw, db = ops.experts_grad_w(dy, x, offsets)
    ends = offsets.tolist()
    per_row = 2 * 2.0 ** -22 + (1024 / 8 + 16) * U
    for e, (a, z) in enumerate(zip(ends[:-1], ends[1:])):
        for got, rows, m in ((y, x, w[e].t()), (dx, dy, w[e])):
            want, size = rows[a:z].double() @ m.double(), rows[a:z].double().abs() @ m.double().abs()
            assert ((got[a:z].double() - want).abs() <= per_row * size).all()
        want, size = dy[a:z].double().t() @ x[a:z].double(), dy[a:z].double().abs().t() @ x[a:z].double().abs()
        assert ((dw[e].double() - want).abs() <= bound(z - a, 2) * size).all()
        assert ((db[e].double() - dy[a:z].double().sum(0)).abs() <= bound(z - a, 2) * dy[a:z].double().abs().sum(0)).all()
    again = ops.experts_grad_w(dy, x, offsets)
    assert torch.equal(dw, again[0]) and torch.equal(db, again[1])
