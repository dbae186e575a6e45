"""CPU: what the norm's, the router's and the experts' entry points refuse, before anything is launched."""
import ctypes as C

import pytest
import torch

from matris_b200 import _lib, build, ops


@pytest.fixture(scope="module", autouse=True)
def library():
    build.build()
    return _lib.load()


def x(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


I = torch.int32
PTR = torch.tensor([0, 4], dtype=I)


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: ops.group_norm_fwd(x(4, 8, dtype=torch.float64), None, None, 2, seg_ptr=PTR)),
    (TypeError, lambda: ops.group_norm_fwd([1.0], None, None, 2, seg_ptr=PTR)),
    (TypeError, lambda: ops.group_norm_fwd(x(4, 8), None, None, 2, seg_ptr=PTR.long())),
    (TypeError, lambda: ops.group_norm_fwd(x(4, 8), x(8, dtype=torch.bfloat16), None, 2, seg_ptr=PTR)),
    (ValueError, lambda: ops.group_norm_fwd(x(4, 8), x(7), None, 2, seg_ptr=PTR)),
    (ValueError, lambda: ops.group_norm_fwd(x(4, 8), None, None, 3, seg_ptr=PTR)),
    (ValueError, lambda: ops.group_norm_fwd(x(4, 8), None, None, 0, seg_ptr=PTR)),
    (ValueError, lambda: ops.group_norm_fwd(x(4, 8), None, None, 2, seg_ptr=PTR, act=2)),
    (ValueError, lambda: ops.group_norm_fwd(x(4, 8), None, None, 2, seg_ptr=PTR, eps=0.0)),
    (ValueError, lambda: ops.group_norm_fwd(x(4, 8), None, None, 2, seg_ptr=PTR, eps=float("nan"))),
    (ValueError, lambda: ops.group_norm_fwd(x(4, 8), None, None, 2, seg_ptr=PTR[:0])),
    (ValueError, lambda: ops.group_norm_fwd(x(8), None, None, 2)),
    (ValueError, lambda: ops.group_norm_fwd(x(8, 4).t(), None, None, 2, seg_ptr=PTR)),
    (ValueError, lambda: ops.group_norm_fwd(x(1, 8).expand(4, 8), None, None, 2, seg_ptr=PTR)),
    (ValueError, lambda: ops.group_norm_fwd(x(2, 8, 4).transpose(1, 2), None, None, 2)),
    (ValueError, lambda: ops.group_norm_fwd(x(4, 8), None, None, 2, seg_ptr=PTR, out=x(4, 9))),
    (NotImplementedError, lambda: ops.group_norm_fwd(x(4, 1032), None, None, 2, seg_ptr=PTR)),
    (ValueError, lambda: ops.group_norm_fwd(x(4, 8), None, None, 2, seg_ptr=PTR)),  # not on a GPU
    (ValueError, lambda: ops.group_norm_bwd(x(4, 8), x(4, 8), None, None, x(1, 3, 2), 2, seg_ptr=PTR)),
    (TypeError, lambda: ops.group_norm_bwd(x(4, 8, dtype=torch.float16), x(4, 8), None, None, x(1, 2, 2), 2, seg_ptr=PTR)),
    (TypeError, lambda: ops.route_fwd(x(4, 8, dtype=torch.int64), 2)),
    (ValueError, lambda: ops.route_fwd(x(4), 2)),
    (ValueError, lambda: ops.route_fwd(x(4, 8), 0)),
    (ValueError, lambda: ops.route_fwd(x(4, 8), 9)),
    (ValueError, lambda: ops.route_fwd(x(4, 64), 33)),
    (NotImplementedError, lambda: ops.route_fwd(x(4, 1025), 2)),
    (TypeError, lambda: ops.route_fwd(x(4, 8), 2, valid=x(4))),
    (ValueError, lambda: ops.route_fwd(x(4, 8), 2, valid=torch.ones(5, dtype=torch.bool))),
    (ValueError, lambda: ops.route_fwd(x(8, 4).t(), 2)),
    (ValueError, lambda: ops.route_fwd(x(4, 8), 2)),  # not on a GPU
    (NotImplementedError, lambda: ops.ExpertWeights(x(2, 100, 128))),
    (NotImplementedError, lambda: ops.ExpertWeights(x(2, 128, 1152))),
    (NotImplementedError, lambda: ops.ExpertWeights(x(0, 128, 128))),
    (ValueError, lambda: ops.ExpertWeights(x(128, 128))),
    (TypeError, lambda: ops.ExpertWeights(x(2, 128, 128, dtype=torch.bfloat16))),
    (NotImplementedError, lambda: ops.experts_grad_w(x(4, 100), x(4, 128), PTR)),
    (ValueError, lambda: ops.experts_grad_w(x(5, 128), x(4, 128), PTR)),
    (ValueError, lambda: ops.experts_grad_w(x(4, 128), x(4, 132)[:, 1:129], PTR)),
    (ValueError, lambda: ops.experts_grad_w(x(4, 128), x(4, 128), PTR, in_act=2)),
    (TypeError, lambda: ops.experts_grad_w(x(4, 128), x(4, 128), PTR, idx=torch.zeros(4, dtype=torch.int64))),
    (ValueError, lambda: ops.experts_grad_w(x(4, 128), x(0, 128), PTR, idx=torch.zeros(4, dtype=I))),
    (NotImplementedError, lambda: ops.experts_combine_fwd(x(4, 6), torch.zeros(2, 2, dtype=I))),
    (NotImplementedError, lambda: ops.experts_combine_fwd(x(4, 8), torch.zeros(2, 0, dtype=I))),
    (NotImplementedError, lambda: ops.experts_combine_fwd(x(4, 8), torch.zeros(2, 33, dtype=I))),
    (ValueError, lambda: ops.experts_combine_fwd(x(4, 8), torch.zeros(2, 2, dtype=I), x(2, 3))),
    (TypeError, lambda: ops.experts_combine_fwd(x(4, 8), torch.zeros(2, 2))),
    (ValueError, lambda: ops.experts_combine_bwd(x(2, 9), x(4, 8), torch.zeros(2, 2, dtype=I))),
    (ValueError, lambda: ops.experts_combine_bwd(x(2, 8), x(4, 8), torch.zeros(2, 2, dtype=I), None, PTR[:0])),
])
def test_refused(error, call):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("struct,name,fields", [
    (_lib.MbGroupNorm, "mb_group_norm_fwd", dict(n_rows=4, n_seg=1, channels=2048, groups=1, eps=1.0)),
    (_lib.MbGroupNorm, "mb_group_norm_fwd", dict(n_rows=4, n_seg=1, channels=8, groups=3, eps=1.0)),
    (_lib.MbGroupNorm, "mb_group_norm_fwd", dict(n_rows=4, n_seg=1, channels=8, groups=2, eps=1.0)),  # null pointers
    (_lib.MbGroupNorm, "mb_group_norm_fwd", dict(n_rows=4, n_seg=3, channels=8, groups=2, eps=1.0)),  # 4 rows in 3 equal segments
    (_lib.MbGroupNorm, "mb_group_norm_bwd", dict(n_rows=-1, n_seg=1, channels=8, groups=2, eps=1.0)),
    (_lib.MbRoute, "mb_route_fwd", dict(n_rows=4, n_experts=8, top_k=9)),
    (_lib.MbRoute, "mb_route_fwd", dict(n_rows=4, n_experts=8, top_k=2, dtype=3)),
    (_lib.MbRoute, "mb_route_bwd", dict(n_rows=4, n_experts=8, top_k=2)),
    (_lib.MbExperts, "mb_experts_linear", dict(n_slots=4, n_rows=4, n_experts=2, n_in=100, n_out=128)),
    (_lib.MbExperts, "mb_experts_linear", dict(n_slots=4, n_rows=4, n_experts=2, n_in=128, n_out=128)),
    (_lib.MbExperts, "mb_experts_grad_w", dict(n_slots=4, n_rows=4, n_experts=0, n_in=128, n_out=128)),
    (_lib.MbCombine, "mb_experts_combine_fwd", dict(n_rows=4, n_slots=4, top_k=2, width=6)),
    (_lib.MbCombine, "mb_experts_combine_bwd", dict(n_rows=4, n_slots=4, top_k=2, width=8)),
])
def test_the_library_refuses(struct, name, fields, library):
    d = struct(**fields)
    assert getattr(library, name)(C.byref(d), None) == _lib.MB_ERR_INVALID
    assert getattr(library, name)(None, None) == _lib.MB_ERR_INVALID


@pytest.mark.parametrize("struct,name,fields", [
    (_lib.MbRoute, "mb_route_fwd", dict(n_rows=1 << 60, n_experts=32, top_k=16, ld_logits=32)),  # 2^64 choices are 0 in 64 bits
    (_lib.MbRoute, "mb_route_bwd", dict(n_rows=1 << 60, n_experts=32, top_k=16, ld_logits=32, ld_dlogits=32)),
    (_lib.MbCombine, "mb_experts_combine_fwd", dict(n_rows=1 << 60, n_slots=4, top_k=16, width=8, ld_y=8, ld_out=8)),
    (_lib.MbCombine, "mb_experts_combine_bwd", dict(n_rows=4, n_slots=4, top_k=2, width=8, n_experts=-1, ld_y=8, ld_dout=8, ld_dy=8)),
])
def test_the_library_refuses_sizes(struct, name, fields, library):
    """All pointers given (and not looked at): the sizes alone are refused."""
    d = struct(**fields)
    for field, kind in struct._fields_:
        if kind is C.c_void_p:
            setattr(d, field, 1 << 12)
    assert getattr(library, name)(C.byref(d), None) == _lib.MB_ERR_INVALID


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import subprocess
    from conftest import ROOT
    names = {"mb_group_norm": _lib.MbGroupNorm, "mb_route": _lib.MbRoute, "mb_experts": _lib.MbExperts, "mb_combine": _lib.MbCombine}
    lines = [f'printf("{n} %zu", sizeof({n}));' + "".join(f'printf(" %zu", offsetof({n}, {f[0]}));' for f in s._fields_) + 'printf("\\n");'
             for n, s in names.items()]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "matris_b200.h"\nint main(void) {' + "".join(lines) + "return 0; }")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "t")])
    for line in subprocess.check_output([str(tmp_path / "t")], text=True).splitlines():
        n, *got = line.split()
        assert [int(v) for v in got] == [C.sizeof(names[n])] + [getattr(names[n], f[0]).offset for f in names[n]._fields_], n


def test_combination_wants_tensors():
    with pytest.raises(TypeError):
        ops.experts_combine_fwd([1.0], torch.zeros(1, 1, dtype=I))
