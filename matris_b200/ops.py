"""Thin Python wrappers over the C-ABI kernels (device pointers in, nothing computed here).

Tensors are float32 / int32, contiguous, on the current CUDA device.  Every
wrapper launches on torch's current stream.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import NamedTuple

import torch

from . import _lib
from ._lib import OUT_ADD, OUT_ATOMIC, OUT_STORE, call, ptr  # noqa: F401

D = 128


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    """Raw handle of torch's current stream on the current device (the stream every entry point launches on)."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


def new(rows, cols, like, zero=False):
    f = torch.zeros if zero else torch.empty
    return f((int(rows), int(cols)), dtype=torch.float32, device=like.device)


# ------------------------------------------------------------------ GEMM descriptors
class SplitWeight:
    """A weight matrix [n_out, K] with its tensor-core operand splits, all in the layout of ``w``:
    ``hi16`` = bf16(w), ``lo16`` = bf16(w - hi16) for the 3xBF16 core (the default);
    ``hi`` = tf32-rounded values, ``lo`` = w - hi (float32) for the 3xTF32 cores.
    ``w`` itself feeds the exact-fp32 SIMT core."""

    __slots__ = ("w", "hi", "lo", "hi16", "lo16", "shape", "ptrs", "ldw")

    def __init__(self, w: torch.Tensor):
        w = w.detach().contiguous()
        bits = w.view(torch.int32)
        hi = ((bits + 0x1000) & ~0x1FFF).view(torch.float32)  # round to nearest (ties away) at 10 mantissa bits
        self.w, self.hi, self.lo, self.shape = w, hi.contiguous(), (w - hi).contiguous(), w.shape
        self.hi16 = w.to(torch.bfloat16).contiguous()          # round to nearest even
        self.lo16 = (w - self.hi16.float()).to(torch.bfloat16).contiguous()
        # device addresses and row stride, looked up once: the descriptor packing runs for every launch
        self.ptrs = (w.data_ptr(), self.hi.data_ptr(), self.lo.data_ptr(), self.hi16.data_ptr(), self.lo16.data_ptr())
        self.ldw = w.stride(0)
        assert w.dim() == 2 and w.stride(1) == 1

    def t(self) -> "SplitWeight":
        return SplitWeight(self.w.t())


_split_cache: dict = {}


def as_split(W) -> SplitWeight:
    if isinstance(W, SplitWeight):
        return W
    # an entry keeps W, so that its address is not handed out again; views of one storage differ in shape or strides
    key = (W.data_ptr(), tuple(W.shape), W.stride(), W._version)
    entry = _split_cache.get(key)
    if entry is None:
        if len(_split_cache) > 256:
            _split_cache.clear()
        entry = _split_cache[key] = (W.detach(), SplitWeight(W))
    return entry[1]


def S(t, idx=None, col=0, act=0):
    """One 128-wide K segment: rows of ``t`` (optionally gathered by ``idx``), columns col..col+127."""
    return (t, idx, col, act)


def B(srcs, W, w_row=0, bias=None, bias_off=0, gate=None, gate_col=0, out_act=0, res=None, res_col=0, res_w=None,
      out=None, out_idx=None, out_col=0, mode=OUT_STORE, scale=1.0):
    """One 128-column output block (see mb_colblock)."""
    return dict(srcs=srcs, W=W, w_row=w_row, bias=bias, bias_off=bias_off, gate=gate, gate_col=gate_col,
                out_act=out_act, res=res, res_col=res_col, res_w=res_w, out=out, out_idx=out_idx, out_col=out_col,
                mode=mode, scale=scale)


# Byte layout of mb_colblock / mb_gemm_desc (little endian, every member naturally aligned; checked against the
# ctypes mirror at import).  The descriptor is packed with one struct call per column block: filling the ctypes
# mirror field by field costs more host time than a small launch takes on the device.
_BLK_FMT = struct.Struct("<ii" + "QQqii" * 4 + "QQQQQqQ" + "Qqii" + "QQqii" + "QQqif")
_HDR_FMT = struct.Struct("<qii")
_BLK_OFF, _BLK_SIZE, _DESC_SIZE = _lib.MbGemmDesc.blk.offset, C.sizeof(_lib.MbColBlock), C.sizeof(_lib.MbGemmDesc)
assert _BLK_FMT.size == _BLK_SIZE and _HDR_FMT.size == _BLK_OFF and _DESC_SIZE == _BLK_OFF + 4 * _BLK_SIZE
_NO_SRC = (0, 0, 0, 0, 0)


_PAD = ((), _NO_SRC, _NO_SRC * 2, _NO_SRC * 3, _NO_SRC * 4)  # by number of missing sources


def gemm(n_rows: int, blocks: list[dict]) -> None:
    if n_rows == 0:
        return
    buf = bytearray(_DESC_SIZE)
    _HDR_FMT.pack_into(buf, 0, n_rows, len(blocks), 0)
    off = _BLK_OFF
    last_srcs = flat = None
    for b in blocks:
        srcs = b["srcs"]
        n_src = len(srcs)
        if srcs is not last_srcs:  # column blocks that share one list of sources share its packed form
            flat = []
            for t, idx, col, act in srcs:
                assert t.dtype == torch.float32 and t.stride(-1) == 1
                flat += (t.data_ptr(), 0 if idx is None else idx.data_ptr(), t.stride(0), col, act)
            flat += _PAD[4 - n_src]
            last_srcs = srcs
        sw = b["W"]
        if type(sw) is not SplitWeight:
            sw = as_split(sw)
        ldw = sw.ldw
        assert sw.shape[1] >= D * n_src
        w_off = 4 * ldw * b["w_row"]
        w_off16 = w_off // 2
        pw, ph, pl, ph16, pl16 = sw.ptrs
        bias, gate, res, res_w, out, out_idx = b["bias"], b["gate"], b["res"], b["res_w"], b["out"], b["out_idx"]
        _BLK_FMT.pack_into(
            buf, off, n_src, b["out_act"], *flat,
            pw + w_off, ph + w_off, pl + w_off, ph16 + w_off16, pl16 + w_off16, ldw,
            0 if bias is None else bias.data_ptr() + 4 * b["bias_off"],
            0 if gate is None else gate.data_ptr(), 0 if gate is None else gate.stride(0),
            0 if gate is None else b["gate_col"], 0,
            0 if res is None else res.data_ptr(), 0 if res is None or res_w is None else res_w.data_ptr(),
            0 if res is None else res.stride(0), 0 if res is None else b["res_col"], b["mode"],
            out.data_ptr(), 0 if out_idx is None else out_idx.data_ptr(), out.stride(0), b["out_col"],
            b["scale"])
        off += _BLK_SIZE
    if _lib.profile is not None:
        _lib.profile_meta = dict(flops=sum(2.0 * n_rows * D * D * len(b["srcs"]) for b in blocks), rows=int(n_rows),
                                 k=D * len(blocks[0]["srcs"]), n=D * len(blocks),
                                 bytes=4.0 * n_rows * D * (len(blocks[0]["srcs"]) + len(blocks) +
                                                           sum(b.get("gate") is not None for b in blocks) +
                                                           sum(b.get("res") is not None for b in blocks)))
    call("mb_gemm", C.byref(_lib.MbGemmDesc.from_buffer(buf)), _stream())


_GATED_FMT = struct.Struct("<qii" + "QQqii" * 4 + "QQQQQqQ" + "QQQQQqQ" + "QQ" + "Qq" * 3 + "QQq" + "Qq" + "ii" + "QQq" * 3)
_NO_ADDS = (0,) * 11
assert _GATED_FMT.size == C.sizeof(_lib.MbGatedMlp)


def gated_mlp_fwd(p, n_rows, srcs, want_h=True, res=None, res_w=None, save=True, adds=()):
    """GatedMLP forward as one fused kernel (mb_gated_mlp_fwd).  ``p`` holds the packed weights (w1 [256,K], b1,
    w2 [256,128], b2, nc, ng).  Returns (z1, z2, h, out2); z1 / z2 only when ``save`` (the backward pass reads
    them), h only when ``want_h``, out2 = h + res_w * res only when ``res`` is given.  ``adds``: up to three (table
    [*,256], idx) pairs whose gathered rows are added to layer 1 (``srcs`` may then be empty)."""
    ref = srcs[0][0] if srcs else adds[0][0]
    n_rows = int(n_rows)
    # the composed path of the non-default GEMM modes uses z1 / z2 as scratch
    save = save or _gemm_mode != 0
    z1 = new(n_rows, 2 * D, ref) if save else None
    z2 = new(n_rows, 2 * D, ref) if save else None
    h = new(n_rows, D, ref) if want_h else None
    out2 = new(n_rows, D, ref) if res is not None else None
    if n_rows == 0:
        return z1, z2, h, out2
    flat = []
    for t, idx, col, act in srcs:
        assert t.dtype == torch.float32 and t.stride(-1) == 1
        flat += (t.data_ptr(), 0 if idx is None else idx.data_ptr(), t.stride(0), int(col), int(act))
    for _ in range(4 - len(srcs)):
        flat += _NO_SRC
    w1, w2 = as_split(p.w1), as_split(p.w2)
    assert w1.shape[0] == 2 * D and (not srcs or w1.shape[1] == D * len(srcs)) and tuple(w2.shape) == (2 * D, D)
    extra = []
    for t, idx in adds:
        assert t.dtype == torch.float32 and t.stride(-1) == 1
        extra += (t.data_ptr(), 0 if idx is None else idx.data_ptr(), t.stride(0))
    extra += (0, 0, 0) * (3 - len(adds))

    def pl(t):
        return (0, 0) if t is None else (t.data_ptr(), t.stride(0))

    buf = _GATED_FMT.pack(
        n_rows, len(srcs), 0, *flat,
        *w1.ptrs, w1.ldw,
        0 if p.b1 is None else p.b1.data_ptr(),
        *w2.ptrs, w2.ldw,
        0 if p.b2 is None else p.b2.data_ptr(),
        p.nc.data_ptr(), p.ng.data_ptr(), *pl(z1), *pl(z2), *pl(h),
        0 if res is None else res.data_ptr(), 0 if res is None or res_w is None else res_w.data_ptr(),
        0 if res is None else res.stride(0), *pl(out2), len(adds), 0, *extra)
    if _lib.profile is not None:
        cols = len(srcs) + (4 if z1 is not None else 0) + (h is not None) + 2 * (out2 is not None)
        _lib.profile_meta = dict(flops=2.0 * n_rows * 2 * D * D * (len(srcs) + 1), rows=n_rows, k=D * len(srcs),
                                 n=2 * D, fused=True, bytes=4.0 * n_rows * D * cols)
    call("mb_gated_mlp_fwd", C.byref(_lib.MbGatedMlp.from_buffer_copy(buf)), _stream())
    return z1, z2, h, out2


def ffn_fwd(p, x, want_y=True, res=None, res_w=None, save=True):
    """Two-layer perceptron  y = W2 SiLU(W1 x + b1) + b2  as one launch of the fused kernel in its plain form
    (mb_gated_mlp_fwd with kind = MB_MLP_PLAIN).  ``p`` holds w1 [128, K], b1, w2 [128, 128], b2.  Returns
    (z1, y, out2): z1 = W1 x + b1 only when ``save`` (the backward pass reads it), y only when ``want_y``,
    out2 = y + res_w * res only when ``res`` is given."""
    n_rows = int(x.shape[0])
    w1, w2 = as_split(p.w1), as_split(p.w2)
    k = w1.shape[1]
    assert w1.shape[0] == D and k % D == 0 and x.shape[1] == k and tuple(w2.shape) == (D, D)
    assert x.dtype == torch.float32 and x.stride(-1) == 1
    save = save or _gemm_mode != 0  # the composed path of the non-default GEMM modes uses z1 as scratch
    z1 = new(n_rows, D, x) if save else None
    y = new(n_rows, D, x) if want_y else None
    out2 = new(n_rows, D, x) if res is not None else None
    if n_rows == 0:
        return z1, y, out2
    n_src = k // D
    flat = []
    for s in range(n_src):
        flat += (x.data_ptr(), 0, x.stride(0), D * s, 0)
    for _ in range(4 - n_src):
        flat += _NO_SRC

    def pl(t):
        return (0, 0) if t is None else (t.data_ptr(), t.stride(0))

    buf = _GATED_FMT.pack(
        n_rows, n_src, 1, *flat,
        *w1.ptrs, w1.ldw, 0 if p.b1 is None else p.b1.data_ptr(),
        *w2.ptrs, w2.ldw, 0 if p.b2 is None else p.b2.data_ptr(),
        0, 0, *pl(z1), 0, 0, *pl(y),
        0 if res is None else res.data_ptr(), 0 if res is None or res_w is None else res_w.data_ptr(),
        0 if res is None else res.stride(0), *pl(out2), *_NO_ADDS)
    if _lib.profile is not None:
        cols = n_src + (z1 is not None) + (y is not None) + 2 * (out2 is not None)
        _lib.profile_meta = dict(flops=2.0 * n_rows * D * D * (n_src + 1), rows=n_rows, k=k, n=D, fused=True,
                                 bytes=4.0 * n_rows * D * cols)
    call("mb_gated_mlp_fwd", C.byref(_lib.MbGatedMlp.from_buffer_copy(buf)), _stream())
    return z1, y, out2


def mlp_bwd(dy, w2t, w1t, z1, gated, want_dz1=True, res=None, res_w=None, idx=None, scale=1.0, ext=None, w3t=None):
    """Data gradient of a gated (dy = dz2 [rows,256]) or plain (dy [*,128], optionally gathered) two-layer MLP as one
    launch (mb_mlp_bwd_data): returns (dz1, dx) with dx = dz1 W1 (+ ext W3) (+ res_w * res) for one input segment."""
    n_rows, width = z1.shape
    want_dz1 = want_dz1 or _gemm_mode != 0  # the composed path of the other GEMM modes uses it
    dz1 = new(n_rows, width, z1) if want_dz1 else None
    dx = new(n_rows, D, z1)
    m = _lib.MbMlpBwd()
    m.n_rows, m.kind, m.scale = n_rows, 0 if gated else 1, scale
    m.dy = _lib.MbSrc(dy.data_ptr(), 0 if idx is None else idx.data_ptr(), dy.stride(0), 0, 0)
    m.W2t, m.W1t = (_lib.MbWeight(*s.ptrs, s.ldw) for s in (as_split(w2t), as_split(w1t)))
    if ext is not None:
        m.n_ext = ext.shape[1] // D
        for j in range(m.n_ext):
            m.ext[j] = _lib.MbSrc(ext.data_ptr(), 0, ext.stride(0), D * j, 0)
        w3 = as_split(w3t)
        m.W3t = _lib.MbWeight(*w3.ptrs, w3.ldw)
    m.z1, m.ld_z1, m.dx, m.ld_dx = z1.data_ptr(), z1.stride(0), dx.data_ptr(), dx.stride(0)
    if dz1 is not None:
        m.dz1, m.ld_dz1 = dz1.data_ptr(), dz1.stride(0)
    if res is not None:
        m.res, m.res_w, m.ld_res = res.data_ptr(), ptr(res_w), res.stride(0)
    call("mb_mlp_bwd_data", C.byref(m), _stream())
    return dz1, dx


def linear(x, W, bias=None, out_act=0, in_act=0, gate=None, res=None, res_w=None, scale=1.0, idx=None, out=None):
    """y[R,128*nb] = epilogue(x[R,128*ns] @ W^T): plain dense layer built on gemm()."""
    n_rows = x.shape[0] if idx is None else idx.shape[0]
    W = as_split(W)
    n_out, k = W.shape
    assert n_out % D == 0 and k % D == 0
    if out is None:
        out = new(n_rows, n_out, x)
    srcs = [S(x, idx, D * s, in_act) for s in range(k // D)]
    gemm(n_rows, [B(srcs, W, w_row=D * j, bias=bias, bias_off=D * j, gate=gate, gate_col=D * j, out_act=out_act,
                    res=res, res_col=D * j, res_w=res_w, out=out, out_col=D * j, scale=scale)
                  for j in range(n_out // D)])
    return out


# ------------------------------------------------------------------ row-wise kernels
def gate_fwd(z, wc, wg, want_h=True, res=None, res_w=None):
    n = z.shape[0]
    h = new(n, D, z) if want_h else None
    out2 = new(n, D, z) if res is not None else None
    call("mb_gate_fwd", n, ptr(z), ptr(wc), ptr(wg), ptr(h), ptr(res), ptr(res_w), ptr(out2), _stream())
    return h, out2


def gate_bwd(z, wc, wg, dh):
    dz = torch.empty_like(z)
    call("mb_gate_bwd", z.shape[0], ptr(z), ptr(wc), ptr(wg), ptr(dh), ptr(dz), _stream())
    return dz


def seg_attn_fwd(n_nodes, tgt_ptr, src_ptr, src_perm, emap, logits, h):
    agg_t, agg_s, stats = new(n_nodes, D, h), new(n_nodes, D, h), new(n_nodes, 4 * D, h)
    call("mb_seg_attn_fwd", n_nodes, ptr(tgt_ptr), ptr(src_ptr), ptr(src_perm), ptr(emap), ptr(logits), ptr(h),
         ptr(agg_t), ptr(agg_s), ptr(stats), _stream())
    return agg_t, agg_s, stats


def seg_attn_bwd(tgt, src, emap, logits, h, agg_t, agg_s, stats, dagg_t, dagg_s, dh_in, dh_map, dh_scale, gate=None):
    """``gate`` = (z2, w_core, w_gate): the row gradient goes straight through the gated MLP's tail adjoint and the
    first result is dz2 [rows,256] instead of dh [rows,128]."""
    n = h.shape[0]
    dlogits = new(n, 2 * D, h)
    if gate is None:
        first, gz, gc, gg = new(n, D, h), None, None, None
    else:
        gz, gc, gg = gate
        first = new(n, 2 * D, h)
    call("mb_seg_attn_bwd", n, ptr(tgt), ptr(src), 1, ptr(emap), ptr(logits), ptr(h), ptr(agg_t), ptr(agg_s),
         ptr(stats), ptr(dagg_t), ptr(dagg_s), ptr(dh_in), ptr(dh_map), float(dh_scale),
         ptr(first) if gate is None else None, ptr(dlogits), ptr(gz), ptr(gc), ptr(gg),
         None if gate is None else ptr(first), _stream())
    return first, dlogits


def seg_smooth_sum_fwd(n_nodes, tgt_ptr, emap, src, env, h):
    agg = new(n_nodes, D, h)
    call("mb_seg_smooth_sum_fwd", n_nodes, ptr(tgt_ptr), ptr(emap), ptr(src), 1, ptr(env), ptr(h), ptr(agg), _stream())
    return agg


def seg_smooth_sum_bwd_rows(tgt, src, emap, env, dagg, dh, accumulate=True, gate=None):
    """``gate`` = (z2, w_core, w_gate): returns dz2 [rows,256], the finished row gradient passed through the gated
    MLP's tail adjoint (dh is then read, if ``accumulate``, but not written); otherwise updates dh in place."""
    gz, gc, gg = gate if gate is not None else (None, None, None)
    dz = new(dh.shape[0], 2 * D, dh) if gate is not None else None
    call("mb_seg_smooth_sum_bwd_rows", dh.shape[0], ptr(tgt), ptr(src), 1, ptr(emap), ptr(env), ptr(dagg), ptr(dh),
         int(accumulate), ptr(gz), ptr(gc), ptr(gg), ptr(dz), _stream())
    return dz


def seg_smooth_sum_bwd_env(n_nodes, tgt_ptr, src_ptr, src_perm, tgt, src, u2d, rev, env, h, dagg, drow=None):
    denv = new(n_nodes, D, h)
    call("mb_seg_smooth_sum_bwd_env", n_nodes, ptr(tgt_ptr), ptr(src_ptr), ptr(src_perm), ptr(tgt), ptr(src), 1,
         ptr(u2d), ptr(rev), ptr(env), ptr(h), ptr(dagg), ptr(drow), ptr(denv), _stream())
    return denv


def mul_rows_gather(x, s, idx=None):
    """y[r] = x[r] * s[idx[r]] channel-wise."""
    y = torch.empty_like(x)
    call("mb_mul_rows_gather", x.shape[0], ptr(x), ptr(s), ptr(idx), ptr(y), _stream())
    return y


def seg_sum(n_nodes, tgt_ptr, src_ptr, src_perm, x, ctr=None, ctr_out=None):
    """[n_nodes,512]: sums of the rows of x [*,256] by target node | by source node; ``ctr_out`` [*,256] accumulates them
    by centre atom."""
    out = new(n_nodes, 4 * D, x)
    call("mb_seg_sum", n_nodes, x.shape[0], ptr(tgt_ptr), ptr(src_ptr), ptr(src_perm), ptr(ctr), ptr(x), ptr(out), ptr(ctr_out),
         _stream())
    return out


def pair_sum(n_bonds, u2d, rev, a, b=None):
    """[n_bonds,256]: sum of the two directed rows of every bond, with ``b`` [n_bonds,512]: of both tensors."""
    out = new(n_bonds, 2 * D if b is None else 4 * D, a)
    call("mb_pair_sum", n_bonds, ptr(u2d), ptr(rev), ptr(a), ptr(b), ptr(out), _stream())
    return out


def pair_mean_res(n_bonds, u2d, rev, y, res=None, res_w=None):
    out = new(n_bonds, D, y)
    call("mb_pair_mean_res", n_bonds, ptr(u2d), ptr(rev), ptr(y), ptr(res), ptr(res_w), ptr(out), _stream())
    return out


def scale_rows(x, a, y=None, accumulate=False):
    if y is None:
        y = torch.empty_like(x)
    call("mb_scale_rows", x.shape[0], ptr(x), ptr(a), ptr(y), int(accumulate), _stream())
    return y


def small_linear_fwd(x, w):
    y = new(x.shape[0], D, x)
    call("mb_small_linear_fwd", x.shape[0], x.shape[1], ptr(x), ptr(w), ptr(y), _stream())
    return y


def small_linear_bwd(dy, w, dx=None, accumulate=False):
    k = w.shape[1]
    if dx is None:
        dx = new(dy.shape[0], k, dy)
    call("mb_small_linear_bwd", dy.shape[0], k, ptr(dy), ptr(w), ptr(dx), int(accumulate), _stream())
    return dx


def layernorm_fwd(x, w, b):
    y = torch.empty_like(x)
    call("mb_layernorm_fwd", x.shape[0], ptr(x), ptr(w), ptr(b), ptr(y), _stream())
    return y


def layernorm_bwd(x, w, dy):
    dx = torch.empty_like(x)
    call("mb_layernorm_bwd", x.shape[0], ptr(x), ptr(w), ptr(dy), ptr(dx), _stream())
    return dx


def rmsnorm_fwd(x, w):
    y = torch.empty_like(x)
    call("mb_rmsnorm_fwd", x.shape[0], ptr(x), ptr(w), ptr(y), _stream())
    return y


def rmsnorm_bwd(x, w, dy):
    dx = torch.empty_like(x)
    call("mb_rmsnorm_bwd", x.shape[0], ptr(x), ptr(w), ptr(dy), ptr(dx), _stream())
    return dx


def embedding(idx, offset, table):
    y = new(idx.shape[0], D, table)
    call("mb_embedding", idx.shape[0], ptr(idx), int(offset), ptr(table), ptr(y), _stream())
    return y


def head_dot_fwd(z, w, b, take_abs=False):
    out = torch.empty(z.shape[0], dtype=torch.float32, device=z.device)
    call("mb_head_dot_fwd", z.shape[0], z.shape[1], ptr(z), ptr(w), ptr(b), int(take_abs), ptr(out), _stream())
    return out


def head_dot_bwd(z, w, seed=None, seed_map=None):
    dz = torch.empty_like(z)
    call("mb_head_dot_bwd", z.shape[0], z.shape[1], ptr(z), ptr(w), ptr(seed), ptr(seed_map), ptr(dz), _stream())
    return dz


def silu_bwd(dy, z):
    dz = torch.empty_like(z)
    call("mb_silu_bwd", z.shape[0], ptr(dy), ptr(z), ptr(dz), _stream())
    return dz


def segment_sum_scalar(n_seg, seg_ptr, x):
    out = torch.empty(n_seg, dtype=torch.float32, device=x.device)
    call("mb_segment_sum_scalar", n_seg, ptr(seg_ptr), ptr(x), ptr(out), _stream())
    return out


# ------------------------------------------------------------------ group norm and mixture of experts
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _take(t, name, dtype, shape=None, dense=True):
    """Check one argument: element type, shape (None: any size), layout.  The device is checked last (``_here``)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor is wanted, got {type(t).__name__}")
    if t.dtype not in (dtype if isinstance(dtype, (tuple, dict)) else (dtype,)):
        raise TypeError(f"{name}: element type {t.dtype}")
    if shape is not None and (t.dim() != len(shape) or any(w is not None and w != h for w, h in zip(shape, t.shape))):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, {tuple('any' if w is None else w for w in shape)} is wanted")
    if dense and not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous tensor is wanted, got strides {t.stride()}")
    return t


def _row_stride(t, name):
    """Row stride of a [rows, width] tensor whose rows are contiguous and do not overlap."""
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the values of a row have to be neighbours, got strides {t.stride()}")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name}: rows overlap, got strides {t.stride()}")
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _aligned_rows(t, name):
    """``_row_stride`` of rows that are read in 16-byte pieces."""
    ld = _row_stride(t, name)
    if t.data_ptr() % 16 or (t.shape[0] > 1 and ld * t.element_size() % 16):
        raise ValueError(f"{name}: rows have to start on 16-byte boundaries")
    return ld


def _here(**tensors):
    """The launches go to the current device: every tensor has to be there."""
    for name, t in tensors.items():
        if t is not None and (t.device.type != "cuda" or t.device.index != torch.cuda.current_device()):
            raise ValueError(f"{name} is on {t.device}: it has to be on the current CUDA device")


def _norm_rows(x, weight, bias, seg_ptr, n_groups, act, eps):
    """[rows, channels] view, row stride and number of segments of a group norm's input."""
    _take(x, "x", _DTYPES, dense=False)
    if seg_ptr is None:
        if x.dim() < 2:
            raise ValueError("x: [batch, .., channels] is wanted without seg_ptr")
        if not x.is_contiguous():
            raise ValueError(f"x: a contiguous tensor is wanted without seg_ptr, got strides {x.stride()}")
        n_seg, x = x.shape[0], x.view(math.prod(x.shape[:-1]), x.shape[-1])
    else:
        _take(x, "x", _DTYPES, (None, None), dense=False)
        n_seg = _take(seg_ptr, "seg_ptr", torch.int32, (None,)).shape[0] - 1
        if n_seg < 0:
            raise ValueError("seg_ptr: [segments + 1] offsets are wanted, got none")
    channels = x.shape[1]
    if not 1 <= channels <= 1024:
        raise NotImplementedError(f"group norm takes 1 to 1024 channels, got {channels}")
    if n_groups < 1 or channels % n_groups:
        raise ValueError(f"{channels} channels do not divide into {n_groups} groups")
    if act not in (0, 1):
        raise ValueError(f"act={act!r}: 0 (none) or 1 (SiLU)")
    if not eps > 0:
        raise ValueError(f"eps={eps!r} has to be positive")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _take(t, name, torch.float32, (channels,))
    _row_stride(x, "x")
    if x.shape[0] >= 1 << 31:
        raise NotImplementedError("group norm takes fewer than 2**31 rows")
    return x, n_seg


def _norm_desc(x, weight, bias, n_groups, n_seg, seg_ptr, eps, act, stats):
    d = _lib.MbGroupNorm()
    d.n_rows, d.n_seg, d.channels, d.groups = x.shape[0], n_seg, x.shape[1], n_groups
    d.dtype, d.act, d.eps = _DTYPES[x.dtype], act, eps
    d.weight, d.bias, d.seg_ptr, d.x, d.ld_x, d.stats = ptr(weight), ptr(bias), ptr(seg_ptr), ptr(x), _row_stride(x, "x"), ptr(stats)
    return d


def _norm_out(x, x_given, out, name):
    """The output rows (same shape and type as the input) and whether rows of no segment are to be cleared."""
    if out is None:
        return torch.empty(x_given.shape, dtype=x.dtype, device=x.device), True
    _take(out, name, x.dtype, tuple(x_given.shape), dense=x_given.dim() != 2)
    return out, False


def group_norm_fwd(x, weight, bias, n_groups, seg_ptr=None, eps=1e-5, act=0, out=None):
    """Group norm with an optional SiLU (``act=1``), features last: every segment of rows and group of neighbouring channels
    has its own mean and variance (float32 arithmetic; x float32, bfloat16 or float16; weight and bias float32 [channels] or None).

    ``x`` [rows, channels] with ``seg_ptr`` (int32 [segments + 1] row offsets on the device, as a batch's ``atom_ptr``), or
    [batch, .., channels] without.  Returns (y, stats): stats [segments, groups, 2] (mean, 1 / deviation) is what
    ``group_norm_bwd`` reads.  Rows of no segment are zero in a returned tensor and left alone in a given ``out``, which may be x."""
    rows, n_seg = _norm_rows(x, weight, bias, seg_ptr, n_groups, act, eps)
    y, zero = _norm_out(rows, x, out, "out")
    _here(x=x, weight=weight, bias=bias, seg_ptr=seg_ptr, out=out)
    if zero and n_seg == 0:
        y.zero_()
    stats = new(n_seg * n_groups, 2, x, zero=not rows.shape[0]).view(n_seg, n_groups, 2)
    d = _norm_desc(rows, weight, bias, n_groups, n_seg, seg_ptr, eps, act, stats)
    yr = y if seg_ptr is not None else y.view(rows.shape)
    d.y, d.ld_y, d.zero_rest = ptr(yr), _row_stride(yr, "out"), int(zero)
    scratch = torch.empty(_lib.load().mb_group_norm_scratch(d.n_rows, n_seg, d.channels), dtype=torch.uint8, device=x.device)
    d.scratch = ptr(scratch)
    call("mb_group_norm_fwd", C.byref(d), _stream())
    return y, stats


def group_norm_bwd(dy, x, weight, bias, stats, n_groups, seg_ptr=None, act=0, out=None, want_affine=True):
    """Gradients (dx, dweight, dbias) of ``group_norm_fwd`` from its inputs and ``stats``; dweight and dbias are None unless
    ``want_affine``.  dx is written to ``out`` where given (it may be dy or x)."""
    rows, n_seg = _norm_rows(x, weight, bias, seg_ptr, n_groups, act, 1.0)
    _take(dy, "dy", x.dtype, tuple(x.shape), dense=seg_ptr is None)
    _take(stats, "stats", torch.float32, (n_seg, n_groups, 2))
    dx, zero = _norm_out(rows, x, out, "out")
    _here(x=x, dy=dy, weight=weight, bias=bias, stats=stats, seg_ptr=seg_ptr, out=out)
    if zero and n_seg == 0:
        dx.zero_()
    d = _norm_desc(rows, weight, bias, n_groups, n_seg, seg_ptr, 1.0, act, stats)
    dyr, dxr = (dy, dx) if seg_ptr is not None else (dy.view(rows.shape), dx.view(rows.shape))
    d.dy, d.ld_dy, d.dx, d.ld_dx, d.zero_rest = ptr(dyr), _row_stride(dyr, "dy"), ptr(dxr), _row_stride(dxr, "out"), int(zero)
    dweight = dbias = None
    if want_affine:
        dweight, dbias = torch.empty(2, d.channels, dtype=torch.float32, device=x.device).unbind(0)
        d.dweight, d.dbias = ptr(dweight), ptr(dbias)
    scratch = torch.empty(_lib.load().mb_group_norm_scratch(d.n_rows, n_seg, d.channels), dtype=torch.uint8, device=x.device)
    d.scratch = ptr(scratch)
    call("mb_group_norm_bwd", C.byref(d), _stream())
    return dx, dweight, dbias


class Route(NamedTuple):
    """What ``route_fwd`` returns: choices and weights of every row [rows, top_k], the balance loss (scalar), the rows that took
    every expert, and the grouping of the (row, choice) pairs by expert (``offsets``, ``row_of``, ``slot_of``)."""

    ids: torch.Tensor
    weights: torch.Tensor
    loss: torch.Tensor
    totals: torch.Tensor  # [experts + 1]: rows of every expert, rows routed
    offsets: torch.Tensor
    row_of: torch.Tensor
    slot_of: torch.Tensor
    renorm: bool

    @property
    def counts(self):
        return self.totals[:-1]


def _route_desc(logits, top_k, renorm):
    _take(logits, "logits", _DTYPES, (None, None), dense=False)
    n, n_experts = logits.shape
    if not 1 <= n_experts <= 1024:
        raise NotImplementedError(f"the router takes 1 to 1024 experts, got {n_experts}")
    if not 1 <= top_k <= min(32, n_experts):
        raise ValueError(f"top_k={top_k}: 1 to {min(32, n_experts)} of {n_experts} experts")
    if n * top_k >= 1 << 31:
        raise NotImplementedError("the router takes fewer than 2**31 choices")
    d = _lib.MbRoute()
    d.n_rows, d.n_experts, d.top_k, d.dtype, d.renorm = n, n_experts, top_k, _DTYPES[logits.dtype], int(renorm)
    d.logits, d.ld_logits = ptr(logits), _row_stride(logits, "logits")
    return d


def route_fwd(logits, top_k, valid=None, renorm=True) -> Route:
    """Router of a mixture of experts.  p = softmax over a row's available experts (logit > -inf); the ``top_k`` largest are
    taken, equal ones by the lowest index; weights p, or p over their sum with ``renorm``.  ``valid`` [rows] bool: False rows are
    padding.  Padding and rows without an available expert have ids -1, weights 0 and no slot, and count nowhere.

    loss = experts / (top_k T^2) sum_e counts_e sum_rows p_e with T the rows routed: 1 where both are even.  Slots 0, 1, ..
    hold the pairs in order of expert, then of row: expert e has slots offsets[e] .. offsets[e+1] - 1, slot s is of row row_of[s]
    (-1 behind the last), choice j of row t has slot slot_of[t, j]."""
    d = _route_desc(logits, top_k, renorm)
    n, n_experts = logits.shape
    if valid is not None:
        _take(valid, "valid", torch.bool, (n,))
    _here(logits=logits, valid=valid)
    dev = logits.device
    ints = torch.empty(2 * n_experts + 2, dtype=torch.int32, device=dev)
    ids, slot_of, row_of = torch.empty(3, n * top_k, dtype=torch.int32, device=dev).unbind(0)
    weights, loss = torch.empty(n, top_k, dtype=torch.float32, device=dev), torch.empty((), dtype=torch.float32, device=dev)
    totals, offsets = ints[:n_experts + 1], ints[n_experts + 1:]
    scratch = torch.empty(_lib.load().mb_route_scratch(n, n_experts), dtype=torch.uint8, device=dev)
    d.valid, d.ids, d.weights, d.counts, d.loss = ptr(valid), ptr(ids), ptr(weights), ptr(totals), ptr(loss)
    d.offsets, d.row_of, d.slot_of, d.scratch = ptr(offsets), ptr(row_of), ptr(slot_of), ptr(scratch)
    call("mb_route_fwd", C.byref(d), _stream())
    return Route(ids.view(n, top_k), weights, loss, totals, offsets, row_of, slot_of.view(n, top_k), bool(renorm))


def route_bwd(logits, route: Route, dweights=None, dloss=None):
    """Gradient of the logits from those of the weights [rows, top_k] and of the balance loss (a scalar tensor); None: zero."""
    n, top_k = route.ids.shape
    d = _route_desc(logits, top_k, route.renorm)
    _take(route.ids, "route.ids", torch.int32, (logits.shape[0], top_k))
    _take(route.weights, "route.weights", torch.float32, (n, top_k))
    _take(route.totals, "route.totals", torch.int32, (logits.shape[1] + 1,))
    if dweights is not None:
        _take(dweights, "dweights", torch.float32, (n, top_k))
    if dloss is not None and _take(dloss, "dloss", torch.float32).numel() != 1:
        raise ValueError(f"dloss: a scalar is wanted, got shape {tuple(dloss.shape)}")
    _here(logits=logits, ids=route.ids, weights=route.weights, totals=route.totals, dweights=dweights, dloss=dloss)
    dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    d.ids, d.weights, d.counts, d.dweights, d.dloss = ptr(route.ids), ptr(route.weights), ptr(route.totals), ptr(dweights), ptr(dloss)
    d.dlogits, d.ld_dlogits = ptr(dlogits), logits.shape[1]
    call("mb_route_bwd", C.byref(d), _stream())
    return dlogits


class ExpertWeights:
    """Weights [experts, n_out, n_in] of the experts' dense layers, laid out once for ``experts_linear`` in both directions:
    two tf32 parts each, w = hi + lo to 2^-23, 16 bytes a weight.  It copies: a later change of ``w`` does not reach it."""

    __slots__ = ("shape", "parts")

    def __init__(self, w: torch.Tensor):
        w = _take(w.detach(), "weights", torch.float32, (None, None, None), dense=False).contiguous()
        if not 1 <= w.shape[0] <= 1024:
            raise NotImplementedError(f"1 to 1024 experts, got {w.shape[0]}")
        _expert_widths(w.shape[2], w.shape[1])
        _here(weights=w)
        self.shape, self.parts = tuple(w.shape), new(4, w.numel(), w)
        call("mb_experts_split", *self.shape, ptr(w), ptr(self.parts), _stream())


def _expert_widths(n_in, n_out):
    for n in (n_in, n_out):
        if n % D or not D <= n <= 1024:
            raise NotImplementedError(f"the experts' kernels take widths 128, 256 .. 1024, got {n_in} -> {n_out}")


def _experts_desc(x, offsets, idx, n_in, n_out, in_act):
    _take(x, "x", torch.float32, (None, n_in), dense=False)
    _take(offsets, "offsets", torch.int32, (None,))
    d = _lib.MbExperts()
    d.n_rows = d.n_slots = x.shape[0]
    if idx is not None:
        d.n_slots = _take(idx, "idx", torch.int32, (None,)).shape[0]
        if d.n_slots and not d.n_rows:
            raise ValueError("idx: there are no rows to take")
    if d.n_slots >= 1 << 31:
        raise NotImplementedError("fewer than 2**31 slots")
    if in_act not in (0, 1):
        raise ValueError(f"in_act={in_act!r}: 0 (none) or 1 (SiLU)")
    d.n_experts, d.n_in, d.n_out, d.in_act = offsets.shape[0] - 1, n_in, n_out, in_act
    d.offsets, d.idx, d.x, d.ld_x = ptr(offsets), ptr(idx), ptr(x), _aligned_rows(x, "x")
    return d


def experts_linear(x, weights, offsets, bias=None, idx=None, in_act=0, out_act=0, gate=None, transposed=False, out=None):
    """Dense layers of a mixture of experts on rows grouped by expert: for the slots s of expert e
    y[s] = act(f(x[idx[s]]) W_e^T + bias_e), times SiLU'(gate[s]) where ``gate`` [slots, n_out] is given (idx None: row s itself).

    ``weights``: ExpertWeights, or a [experts, n_out, n_in] tensor that is laid out in the call; ``transposed``: W_e in the place
    of its transpose, the data gradient.  ``in_act`` / ``out_act`` 1: SiLU.  ``offsets``, ``idx``: ``Route.offsets``, ``Route.row_of``.
    Slots behind the last are zero in a returned tensor and left alone in a given ``out``."""
    if not isinstance(weights, ExpertWeights):
        weights = ExpertWeights(weights)
    n_experts, n_out, n_in = weights.shape
    w_hi = ptr(weights.parts) + (8 * weights.parts.shape[1] if transposed else 0)
    if transposed:
        n_out, n_in = n_in, n_out
    d = _experts_desc(x, offsets, idx, n_in, n_out, in_act)
    if d.n_experts != n_experts:
        raise ValueError(f"offsets: [{n_experts + 1}] is wanted, got {tuple(offsets.shape)}")
    if out_act not in (0, 1):
        raise ValueError(f"out_act={out_act!r}: 0 (none) or 1 (SiLU)")
    if bias is not None:
        _take(bias, "bias", torch.float32, (n_experts, n_out))
    if gate is not None:
        _take(gate, "gate", torch.float32, (d.n_slots, n_out), dense=False)
        d.gate, d.ld_gate = ptr(gate), _aligned_rows(gate, "gate")
    if out is not None:
        _take(out, "out", torch.float32, (d.n_slots, n_out), dense=False)
    _here(x=x, weights=weights.parts, offsets=offsets, bias=bias, idx=idx, gate=gate, out=out)
    y = new(d.n_slots, n_out, x) if out is None else out
    d.w_hi, d.w_lo = w_hi, w_hi + 4 * weights.parts.shape[1]
    d.bias, d.out_act, d.zero_rest = ptr(bias), out_act, int(out is None)
    d.y, d.ld_y = ptr(y), _aligned_rows(y, "out")
    call("mb_experts_linear", C.byref(d), _stream())
    return y


def experts_grad_w(dy, x, offsets, idx=None, in_act=0, want_bias=True):
    """Weight gradients of ``experts_linear``: (dW [experts, n_out, n_in], dbias [experts, n_out] or None) with
    dW_e = sum over the slots of e of dy[s]^T f(x[idx[s]]), summed in a fixed order.  An expert without slots has zeros."""
    _take(dy, "dy", torch.float32, (None, None), dense=False)
    if x.dim() != 2:
        raise ValueError(f"x: [rows, n_in] is wanted, got shape {tuple(x.shape)}")
    _expert_widths(x.shape[1], dy.shape[1])
    d = _experts_desc(x, offsets, idx, x.shape[1], dy.shape[1], in_act)
    if dy.shape[0] != d.n_slots:
        raise ValueError(f"dy: {d.n_slots} slots are wanted, got {dy.shape[0]}")
    if not 1 <= d.n_experts <= 1024:
        raise NotImplementedError(f"1 to 1024 experts, got {d.n_experts}")
    d.dy, d.ld_dy = ptr(dy), _aligned_rows(dy, "dy")
    _here(dy=dy, x=x, offsets=offsets, idx=idx)
    dw = torch.empty(d.n_experts, d.n_out, d.n_in, dtype=torch.float32, device=x.device)
    dbias = torch.empty(d.n_experts, d.n_out, dtype=torch.float32, device=x.device) if want_bias else None
    scratch = torch.empty(_lib.load().mb_experts_grad_scratch(d.n_slots, d.n_experts, d.n_in, d.n_out), dtype=torch.uint8, device=x.device)
    d.dw, d.dbias, d.scratch = ptr(dw), ptr(dbias), ptr(scratch)
    call("mb_experts_grad_w", C.byref(d), _stream())
    return dw, dbias


def _combine_desc(y, slot_of, weights):
    _take(y, "y", torch.float32, (None, None), dense=False)
    n, k = _take(slot_of, "slot_of", torch.int32, (None, None)).shape
    if y.shape[1] % 4 or not y.shape[1]:
        raise NotImplementedError(f"widths that are multiples of 4, got {y.shape[1]}")
    if k < 1 or n * k >= 1 << 31 or y.shape[0] >= 1 << 31:
        raise NotImplementedError(f"1 choice a row or more, fewer than 2**31 in all, got {n} x {k}")
    if weights is not None:
        _take(weights, "weights", torch.float32, (n, k))
    d = _lib.MbCombine()
    d.n_rows, d.n_slots, d.top_k, d.width = n, y.shape[0], k, y.shape[1]
    d.slot_of, d.weights, d.y, d.ld_y = ptr(slot_of), ptr(weights), ptr(y), _aligned_rows(y, "y")
    return d


def experts_combine_fwd(y, slot_of, weights=None):
    """The experts' outputs back to their rows: out[t] = sum_j weights[t, j] y[slot_of[t, j]] over the choices with a slot
    (weights None: 1, the sum that the gradient of the gathered rows takes)."""
    d = _combine_desc(y, slot_of, weights)
    _here(y=y, slot_of=slot_of, weights=weights)
    out = new(d.n_rows, d.width, y)
    d.out, d.ld_out = ptr(out), d.width
    call("mb_experts_combine_fwd", C.byref(d), _stream())
    return out


def experts_combine_bwd(dout, y, slot_of, weights=None, offsets=None):
    """Gradients (dy, dweights) of ``experts_combine_fwd``: dy [slots, width], dweights [rows, top_k] (0 for a choice without a
    slot).  Slots that no choice has are zero from ``offsets[-1]`` on; without ``offsets`` every slot has to have its choice."""
    d = _combine_desc(y, slot_of, weights)
    _take(dout, "dout", torch.float32, (d.n_rows, d.width), dense=False)
    if offsets is not None:
        d.n_experts, d.offsets = _take(offsets, "offsets", torch.int32, (None,)).shape[0] - 1, ptr(offsets)
        if d.n_experts < 0:
            raise ValueError("offsets: [experts + 1] is wanted, got none")
    d.dout, d.ld_dout = ptr(dout), _aligned_rows(dout, "dout")
    _here(dout=dout, y=y, slot_of=slot_of, weights=weights, offsets=offsets)
    dy, dweights = new(d.n_slots, d.width, y), new(d.n_rows, d.top_k, y)
    d.dy, d.ld_dy, d.dweights = ptr(dy), d.width, ptr(dweights)
    call("mb_experts_combine_bwd", C.byref(d), _stream())
    return dy, dweights


# ------------------------------------------------------------------ geometry and bases
def edge_geometry_fwd(cart, lattice, atom_struct, center, neighbor, image):
    ne = center.shape[0]
    vec, unit = new(ne, 3, cart), new(ne, 3, cart)
    length = torch.empty(ne, dtype=torch.float32, device=cart.device)
    call("mb_edge_geometry_fwd", ne, ptr(cart), ptr(lattice), ptr(atom_struct), ptr(center), ptr(neighbor),
         ptr(image), ptr(vec), ptr(length), ptr(unit), _stream())
    return vec, length, unit


def edge_geometry_bwd(n_atoms, n_struct, edge_ptr, atom_ptr, rev, vec, length, unit, dlen, dunit):
    ne = rev.shape[0]
    g = new(ne, 3, vec)
    dcart, virial_atom, dstrain = new(n_atoms, 3, vec), new(n_atoms, 9, vec), new(n_struct, 9, vec)
    call("mb_edge_geometry_bwd", n_atoms, n_struct, ne, ptr(edge_ptr), ptr(atom_ptr), ptr(rev), ptr(vec), ptr(length),
         ptr(unit), ptr(dlen), ptr(dunit), ptr(g), ptr(dcart), ptr(virial_atom), ptr(dstrain), _stream())
    return dcart, dstrain.view(n_struct, 3, 3), g


def bessel_fwd(u2d, length, fa, ca, fb, cb, p):
    nb = u2d.shape[0]
    ra, rb = new(nb, 7, length), new(nb, 7, length)
    call("mb_bessel_fwd", nb, ptr(u2d), ptr(length), ptr(fa), float(ca), ptr(fb), float(cb), int(p), ptr(ra), ptr(rb),
         _stream())
    return ra, rb


def bessel_bwd(u2d, length, fa, ca, fb, cb, p, dra, drb):
    dlen = torch.zeros_like(length)
    call("mb_bessel_bwd", u2d.shape[0], ptr(u2d), ptr(length), ptr(fa), float(ca), ptr(fb), float(cb), int(p),
         ptr(dra), ptr(drb), ptr(dlen), _stream())
    return dlen


def gaussian_fwd(u2d, length, oa, ca, ob, cb):
    nb = u2d.shape[0]
    ra, rb = new(nb, 7, length), new(nb, 7, length)
    call("mb_gaussian_fwd", nb, ptr(u2d), ptr(length), ptr(oa), float(ca), ptr(ob), float(cb), ptr(ra), ptr(rb), _stream())
    return ra, rb


def gaussian_bwd(u2d, length, oa, ca, ob, cb, dra, drb):
    dlen = torch.zeros_like(length)
    call("mb_gaussian_bwd", u2d.shape[0], ptr(u2d), ptr(length), ptr(oa), float(ca), ptr(ob), float(cb), ptr(dra),
         ptr(drb), ptr(dlen), _stream())
    return dlen


def fourier_basis_fwd(line_graph, unit, freq):
    nt = line_graph.shape[0]
    basis = new(nt, 7, unit)
    call("mb_fourier_basis_fwd", nt, ptr(line_graph), ptr(unit), ptr(freq), ptr(basis), _stream())
    return basis


def fourier_basis_bwd(line_graph, unit, freq, dbasis):
    dunit = torch.zeros_like(unit)
    call("mb_fourier_basis_bwd", line_graph.shape[0], ptr(line_graph), ptr(unit), ptr(freq), ptr(dbasis), ptr(dunit),
         _stream())
    return dunit


def angle_basis_fwd(line_graph, unit, factor, cutoff):
    nt = line_graph.shape[0]
    basis = new(nt, 16, unit)
    call("mb_angle_basis_fwd", nt, ptr(line_graph), ptr(unit), float(factor), float(cutoff), ptr(basis), _stream())
    return basis


def angle_basis_bwd(line_graph, unit, factor, cutoff, dbasis):
    dunit = torch.zeros_like(unit)
    call("mb_angle_basis_bwd", line_graph.shape[0], ptr(line_graph), ptr(unit), float(factor), float(cutoff),
         ptr(dbasis), ptr(dunit), _stream())
    return dunit


# ------------------------------------------------------------------ GEMM core selection / status
_gemm_mode = 0


def set_gemm_mode(mode: str) -> None:
    """'tcgen05' (default): persistent tensor-core kernels (GEMM and fused gated MLP), 3-term BF16 operand split;
    'tcgen05_tf32': the persistent GEMM with a 3-term TF32 split; 'tcgen05_tile': a one-tile-per-CTA tensor-core
    kernel (3-term TF32); 'simt': exact fp32 FMA cross-check.  Outside the default mode a gated MLP is composed from
    two GEMM launches and the gate kernel.  A test knob."""
    global _gemm_mode
    _gemm_mode = {"tcgen05": 0, "simt": 1, "tcgen05_tile": 2, "tcgen05_tf32": 3}[mode]
    _lib.check(_lib.load().mb_set_gemm_mode(_gemm_mode), "mb_set_gemm_mode")


def gemm_status_async(pinned_int32: torch.Tensor) -> None:
    """Enqueue a copy of the tensor-core kernels' status word into a pinned int32 tensor (no synchronisation)."""
    assert pinned_int32.dtype == torch.int32 and pinned_int32.is_pinned()
    call("mb_gemm_status_async", pinned_int32.data_ptr(), _stream())


def gemm_status_clear() -> None:
    """Zero the status word in stream order."""
    call("mb_gemm_status_clear", _stream())


def selftest_wait_expiry() -> None:
    """Launch the one-CTA self-test whose bounded wait runs out (sets bit 0 of the status word)."""
    call("mb_selftest_wait_expiry", _stream())


def mma_rate(kind: str = "tf32", iters: int = 20000):
    """Timed tcgen05.mma issue rate with resident operands: (TFLOP/s, elapsed ms)."""
    ms, sms = C.c_float(0), C.c_int(0)
    k = {"tf32": 0, "bf16": 1}[kind]
    _lib.check(_lib.load().mb_bench_mma_rate(k, int(iters), C.byref(ms), C.byref(sms), _stream()), "mb_bench_mma_rate")
    flops = 2.0 * 128 * 128 * (8 if k == 0 else 16) * 4 * iters * sms.value
    return flops / (ms.value * 1e-3) / 1e12, ms.value


def gemm_status() -> int:
    """Synchronise and return (then clear) the tensor-core kernel's status word; 0 = no wait expired."""
    st = C.c_int(0)
    _lib.check(_lib.load().mb_gemm_status(C.byref(st), _stream()), "mb_gemm_status")
    return st.value
