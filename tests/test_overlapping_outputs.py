"""CPU: outputs that share memory with what the kernels still read are refused; the same rows, or columns beside them, are not."""
import pytest
import torch

from matris_b200 import ops

I = torch.int32
WIDE = torch.zeros(40, 384)
OFFSETS = torch.tensor([0, 20], dtype=I)


def refused(call, what):
    with pytest.raises(ValueError, match=what):
        call()


@pytest.fixture
def weights():
    """Laid-out weights without a launch."""
    w = ops.ExpertWeights.__new__(ops.ExpertWeights)
    w.shape, w.parts, w.ptrs = (1, 128, 128), torch.zeros(4, 128 * 128), (0, 0, 0, 0)
    return w


def test_experts_linear(weights):
    x, gate = torch.zeros(20, 128), torch.zeros(20, 128)
    refused(lambda: ops.experts_linear(x, weights, OFFSETS, out=x), "out overlaps x")
    refused(lambda: ops.experts_linear(x, weights, OFFSETS, gate=gate, out=gate), "out overlaps gate")
    rows = torch.zeros(30, 128)
    refused(lambda: ops.experts_linear(rows[:20], weights, OFFSETS, out=rows[10:]), "out overlaps x")
    refused(lambda: ops.experts_linear(WIDE[:20, :128], weights, OFFSETS, out=WIDE[:20, 64:192]), "out overlaps x")
    refused(lambda: ops.experts_linear(WIDE[:20, 64:192], weights, OFFSETS, out=WIDE[5:25, :128]), "out overlaps x")
    # beside it, behind it: as far as the check of the device
    for x_, out in ((WIDE[:20, :128], WIDE[:20, 128:256]), (WIDE[:20, 256:], WIDE[:20, :128]), (WIDE[:20, 128:256], WIDE[3:23, 256:]),
                    (WIDE[3:23, 128:256], WIDE[:20, :128]), (rows[:15].repeat(2, 1)[:20], rows[:20]), (WIDE[:20, :128], WIDE[20:, :128])):
        refused(lambda: ops.experts_linear(x_, weights, OFFSETS, out=out), "on the CPU")


def test_group_norm():
    ptr = torch.tensor([0, 20], dtype=I)
    x = torch.zeros(30, 64)
    refused(lambda: ops.group_norm_fwd(x[:20], None, None, 8, seg_ptr=ptr, out=x[:20]), "on the CPU")
    refused(lambda: ops._norm_out(x[:20], 20, 64, x[1:21], ptr), "out overlaps x")
    refused(lambda: ops._norm_out(WIDE[:20, :64], 20, 64, WIDE[:20, 32:96], ptr), "out overlaps x")
    refused(lambda: ops._norm_out(x[:20], 20, 64, WIDE[:20, 32:96], ptr, WIDE[:20, :64]), "out overlaps dy")
    flat = torch.zeros(3, 10, 64)
    refused(lambda: ops._norm_out(flat[:2], 20, 64, flat[1:], None), "out overlaps x")
    for like, out, seg_ptr, dy in ((x[:20], x[:20], ptr, None), (x[:20], WIDE[:20, :64], ptr, WIDE[:20, :64]), (WIDE[:20, :64], WIDE[:20, 64:128], ptr, None),
                                   (flat[:2], flat[:2], None, flat[:2])):
        assert ops._norm_out(like, 20, 64, out, seg_ptr, dy)[0] is out


@pytest.mark.parametrize("a,b,shared", [
    (WIDE[:, :128], WIDE[3:4, 128:256], False), (WIDE[3:4, 128:256], WIDE[:, :128], False), (WIDE[:, :128], WIDE[3:4, 100:228], True),
    (WIDE[3:4, 100:228], WIDE[:, :128], True), (WIDE[3:4, 100:228], WIDE[3:4, 200:328], True), (WIDE[3:4, :128], WIDE[3:4, 128:256], False),
    (WIDE[::2, :128], WIDE[1::2, :128], False), (WIDE[::2, :128], WIDE[1:, :128], True), (WIDE[:0, :128], WIDE[:, :128], False),
    (WIDE, WIDE, True), (WIDE[:10], WIDE[10:], False), (WIDE[:11], WIDE[10:], True)])
def test_memory_in_common(a, b, shared):
    assert ops._share(a, b) is shared and ops._share(b, a) is shared
