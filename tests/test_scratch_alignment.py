"""CPU: scratch memory that the norm's and the router's kernels could not read in whole words is refused, not launched on."""
import ctypes as C

import pytest

from matris_b200 import _lib, build

NORM = dict(n_rows=100_000, n_seg=4, channels=64, groups=8, eps=1.0, ld_x=64, ld_y=64, ld_dy=64, ld_dx=64)
ROUTE = dict(n_rows=100_000, n_experts=32, top_k=2, ld_logits=32, ld_dlogits=32)


@pytest.mark.parametrize("struct,name,fields", [(_lib.MbGroupNorm, "mb_group_norm_fwd", NORM), (_lib.MbGroupNorm, "mb_group_norm_bwd", NORM),
                                                (_lib.MbRoute, "mb_route_fwd", ROUTE)])
@pytest.mark.parametrize("off", [4, 8])
def test_scratch_off_a_16_byte_boundary_is_refused(struct, name, fields, off):
    build.build()
    d = struct(**fields)
    for field, kind in struct._fields_:
        if kind is C.c_void_p:
            setattr(d, field, 1 << 12)
    d.scratch = (1 << 12) + off
    assert getattr(_lib.load(), name)(C.byref(d), None) == _lib.MB_ERR_INVALID
