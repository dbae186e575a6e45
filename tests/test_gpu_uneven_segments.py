"""GPU: group norm of batches that one structure dominates."""
import pytest
import torch

import test_gpu_group_norm as norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ends,channels,groups", [
    ([0, 100, 220, 15220, 15330, 15440, 15600, 15800, 16000], 128, 8),   # 15,000 rows of one segment in a block a slab
    ([0, 100, 220, 15220, 15330, 15440, 15600, 15800, 16000], 128, 1),
    ([0, 15000, 15001, 15001, 15300, 15400, 15500, 15600, 16000], 30, 3),
    ([0, *range(10, 310, 10), 40_000, *range(40_010, 40_300, 10)], 64, 4),  # by chunks among short ones
])
def test_one_long_segment(ends, channels, groups, dtype, monkeypatch):
    """The bounds of ``check`` count 48 roundings in a row, with up to 16 batches of 8 rows a thread; here a thread of 32 in a column has up to
    60 (469 rows), one of 8 (whole rows of 128 channels) up to 235 in float32: 48 - 16 + 235 roundings at the most, six times as many."""
    monkeypatch.setattr(norm, "U", 6 * norm.U)
    x, w, b, dy, seg_ptr = norm.inputs(ends, channels, dtype, 11)
    norm.check(x, w, b, dy, seg_ptr, groups, 1, ends)
