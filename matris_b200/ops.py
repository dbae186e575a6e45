"""Thin Python wrappers over the C-ABI kernels (device pointers in, nothing computed here).

Tensors are float32 / int32, contiguous, on the current CUDA device.  Every
wrapper launches on torch's current stream.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
import threading
from collections import OrderedDict
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


class _Kept(NamedTuple):
    weight: torch.Tensor   # so that its address is not handed out again
    split: SplitWeight
    built: object          # event behind the splits' kernels (None on the CPU)
    streams: set           # raw handles of the streams that are ordered behind it

    def reach(self, stream: int) -> None:
        """Before the first use on another stream than the one that built the splits: it waits for them, and their memory is not
        handed out again before it has read them."""
        here = torch.cuda.current_stream()
        here.wait_event(self.built)
        for t in (self.split.w, self.split.hi, self.split.lo, self.split.hi16, self.split.lo16):
            t.record_stream(here)
        self.streams.add(stream)


_split_cache: OrderedDict = OrderedDict()  # used longest ago first
_split_graphs: dict = {}  # entries that captured graphs read: these stay
_split_lock = threading.Lock()
_SPLITS_KEPT = 257


def as_split(W) -> SplitWeight:
    """The operand splits of a weight, kept for the next call with it on any stream.  The caller holds what it gets until its launch
    is made: another thread may make room in the meantime, and addresses alone keep nothing alive.

    In a capture, splits that were there before stay for good, since the graph may be replayed at any time; others become part of the
    graph and are nobody else's, for they hold values only when it has run."""
    if isinstance(W, SplitWeight):
        return W
    # views of one storage differ in shape or strides
    key = (W.data_ptr(), tuple(W.shape), W.stride(), W._version)
    stream = _stream() if W.is_cuda else 0
    capturing = stream != 0 and torch.cuda.is_current_stream_capturing()
    with _split_lock:
        entry = _split_cache.get(key)
        if entry is not None:
            _split_cache.move_to_end(key)
            if capturing:
                _split_graphs[key] = entry
            elif stream not in entry.streams:
                entry.reach(stream)
            return entry.split
    split = SplitWeight(W)
    if capturing:
        return split
    entry = _Kept(W.detach(), split, torch.cuda.current_stream().record_event() if W.is_cuda else None, {stream})
    with _split_lock:
        _split_cache.setdefault(key, entry)  # of threads that built it at once, the first one's stays
        while len(_split_cache) > _SPLITS_KEPT:
            _split_cache.popitem(last=False)
    return split


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
    held = []  # splits looked up here, until the launch is made
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
            held.append(sw)
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
    w2, w1 = as_split(w2t), as_split(w1t)
    m.W2t, m.W1t = (_lib.MbWeight(*s.ptrs, s.ldw) for s in (w2, w1))
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
# These calls serve single structures and single rows too, where the host's share counts: shapes are compared as tuples, outputs
# that live together share an allocation, descriptors are packed with one struct call (layouts checked against ctypes below).
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_F32, _I32 = torch.float32, torch.int32
_NORM_FMT = struct.Struct("<q6ifi" + "QQqQQQqQ" + "QqQq" + "QQQ")
_ROUTE_FMT = struct.Struct("<q4i" + "QqQQQQQ" + "QQQ" + "QQ" + "QqQ")
_EXPERTS_FMT = struct.Struct("<qq6i" + "QQ" + "Qq" + "QQQ" + "Qq" * 3 + "QQQ")
_COMBINE_FMT = struct.Struct("<qq4i" + "QQQ" + "Qq" * 4 + "Q")
assert [f.size for f in (_NORM_FMT, _ROUTE_FMT, _EXPERTS_FMT, _COMBINE_FMT)] == [
    C.sizeof(t) for t in (_lib.MbGroupNorm, _lib.MbRoute, _lib.MbExperts, _lib.MbCombine)]
_cuda_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _take(t, name, dtype, shape):
    """Check a contiguous argument of a given element type and shape.  The device is checked last (``_here``)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor is wanted, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: element type {t.dtype}, {dtype} is wanted")
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, {shape} is wanted")
    if not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous tensor is wanted, got strides {t.stride()}")
    return t


def _take_vector(t, name):
    """Check a contiguous int32 vector; its length."""
    if not isinstance(t, torch.Tensor) or t.dtype != _I32:
        raise TypeError(f"{name}: an int32 tensor is wanted, got {getattr(t, 'dtype', type(t).__name__)}")
    if t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous vector is wanted, got shape {tuple(t.shape)}, strides {t.stride()}")
    return t.shape[0]


def _take_rows(t, name, dtype, n=None, width=None, aligned=False):
    """Check a [rows, width] argument whose rows are contiguous and do not overlap (``aligned``: and start on 16-byte
    boundaries, for kernels that read them in such pieces); its row stride."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor is wanted, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: element type {t.dtype}, {dtype} is wanted")
    shape = t.shape
    if len(shape) != 2 or (n is not None and shape[0] != n) or (width is not None and shape[1] != width):
        raise ValueError(f"{name}: shape {tuple(shape)}, ({'rows' if n is None else n}, {'width' if width is None else width}) is wanted")
    rows, cols = shape
    ld, step = t.stride()
    if cols > 1 and step != 1:
        raise ValueError(f"{name}: the values of a row have to be neighbours, got strides {t.stride()}")
    if rows <= 1:
        ld = cols
    elif ld < cols:
        raise ValueError(f"{name}: rows overlap, got strides {t.stride()}")
    if aligned and (t.data_ptr() % 16 or (rows > 1 and ld * t.element_size() % 16)):
        raise ValueError(f"{name}: rows have to start on 16-byte boundaries")
    return ld


def _here(*tensors):
    """The launches go to the current device: every tensor has to be there.  Returns its number."""
    if not all([t is None or t.is_cuda for t in tensors]):
        raise ValueError(f"tensors on the CPU ({[str(t.device) for t in tensors if t is not None]}): they have to be on the current CUDA device")
    device = _cuda_device()
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ValueError(f"a tensor on {t.device}: it has to be on the current CUDA device, cuda:{device}")
    return device


def _share(a, b):
    """Whether two [rows, width] tensors with neighbouring values have memory in common."""
    if not a.numel() or not b.numel():
        return False
    size, ends = a.element_size(), []
    for t in (a, b):
        first, (rows, width) = t.data_ptr(), t.shape
        ends.append((first, first + ((rows - 1) * t.stride(0) + width) * size))
    if ends[0][1] <= ends[1][0] or ends[1][1] <= ends[0][0]:
        return False
    lds = {t.stride(0) for t in (a, b) if t.shape[0] > 1}
    if b.element_size() != size or len(lds) != 1 or (ends[1][0] - ends[0][0]) % size:
        return True
    ld = lds.pop()
    at = (ends[1][0] - ends[0][0]) // size % ld  # columns of one wider tensor: b begins `at` columns behind a
    return at < a.shape[1] or at + b.shape[1] > ld


def _apart(out, name, t, may_be=False):
    """``out`` and an input that the kernels read while they write: no memory in common (``may_be``: or the very same rows)."""
    if t is None or (may_be and out.data_ptr() == t.data_ptr() and out.stride() == t.stride()):
        return
    if _share(out, t):
        raise ValueError(f"out overlaps {name}")


def _launch(name, struct_type, data, device):
    d = struct_type.from_buffer_copy(data)
    call(name, C.byref(d), _stream() if _raw_stream is None else _raw_stream(device))


def _scratch(size, like):
    return torch.empty(size, dtype=torch.uint8, device=like.device) if size else None


def _norm_rows(x, weight, bias, seg_ptr, n_groups, act, eps):
    """Rows (a [rows, channels] view), channels, row stride and number of segments of a group norm's input."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES:
        raise TypeError(f"x: a float32, bfloat16 or float16 tensor is wanted, got {getattr(x, 'dtype', type(x).__name__)}")
    if seg_ptr is None:
        if x.dim() < 2:
            raise ValueError("x: [batch, .., channels] is wanted without seg_ptr")
        if not x.is_contiguous():
            raise ValueError(f"x: a contiguous tensor is wanted without seg_ptr, got strides {x.stride()}")
        n_seg, x = x.shape[0], x.view(math.prod(x.shape[:-1]), x.shape[-1])
    else:
        n_seg = _take_vector(seg_ptr, "seg_ptr") - 1
        if n_seg < 0:
            raise ValueError("seg_ptr: [segments + 1] offsets are wanted, got none")
    ld = _take_rows(x, "x", x.dtype)
    rows, channels = x.shape
    if not 1 <= channels <= 1024:
        raise NotImplementedError(f"group norm takes 1 to 1024 channels, got {channels}")
    if n_groups < 1 or channels % n_groups:
        raise ValueError(f"{channels} channels do not divide into {n_groups} groups")
    if act != 0 and act != 1:
        raise ValueError(f"act={act!r}: 0 (none) or 1 (SiLU)")
    if not eps > 0:
        raise ValueError(f"eps={eps!r} has to be positive")
    if weight is not None:
        _take(weight, "weight", _F32, (channels,))
    if bias is not None:
        _take(bias, "bias", _F32, (channels,))
    if rows >= 1 << 31:
        raise NotImplementedError("group norm takes fewer than 2**31 rows")
    return x, rows, channels, ld, n_seg


def _norm_out(like, rows, channels, out, seg_ptr, dy=None):
    """The output, its row stride, and whether rows of no segment are to be cleared."""
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device), channels, 1
    if seg_ptr is None:
        _take(out, "out", like.dtype, like.shape)
        ld = channels
    else:
        ld = _take_rows(out, "out", like.dtype, rows, channels)
    flat = (rows, channels)
    for name, t in (("x", like), ("dy", dy)):
        if t is not None:
            _apart(out if seg_ptr is not None else out.view(flat), name, t if seg_ptr is not None else t.view(flat), may_be=True)
    return out, ld, 0


def group_norm_fwd(x, weight, bias, n_groups, seg_ptr=None, eps=1e-5, act=0, out=None):
    """Group norm with an optional SiLU (``act=1``), features last: every segment of rows and group of neighbouring channels
    has its own mean and variance (float32 arithmetic; x float32, bfloat16 or float16; weight and bias float32 [channels] or None).

    ``x`` [rows, channels] with ``seg_ptr`` (int32 [segments + 1] row offsets on the device, as ``BatchedGraph.atom_ptr``), or
    [batch, .., channels] without.  Returns (y, stats): stats [segments, groups, 2] (mean, 1 / deviation) is what
    ``group_norm_bwd`` reads.  Rows of no segment are zero in a returned tensor and left alone in a given ``out``, which may be x and does
    not overlap it otherwise."""
    xr, rows, channels, ld, n_seg = _norm_rows(x, weight, bias, seg_ptr, n_groups, act, eps)
    device = _here(x, weight, bias, seg_ptr, out)
    y, ld_y, zero = _norm_out(x, rows, channels, out, seg_ptr)
    stats = torch.empty((n_seg, n_groups, 2), dtype=_F32, device=x.device)
    if not rows:
        stats.zero_()
    if zero and not n_seg:
        y.zero_()
    scratch = _scratch(_lib.load().mb_group_norm_scratch(rows, n_seg, channels, 0), x)
    _launch("mb_group_norm_fwd", _lib.MbGroupNorm, _NORM_FMT.pack(
        rows, n_seg, channels, n_groups, _DTYPES[x.dtype], act, zero, eps, 0, ptr(seg_ptr) or 0, xr.data_ptr(), ld, ptr(weight) or 0,
        ptr(bias) or 0, y.data_ptr(), ld_y, stats.data_ptr(), 0, 0, 0, 0, 0, 0, ptr(scratch) or 0), device)
    return y, stats


def group_norm_bwd(dy, x, weight, bias, stats, n_groups, seg_ptr=None, act=0, out=None, want_affine=True):
    """Gradients (dx, dweight, dbias) of ``group_norm_fwd`` from its inputs and ``stats``; dweight and dbias are None unless
    ``want_affine``.  dx is written to ``out`` where given (it may be dy or x)."""
    xr, rows, channels, ld, n_seg = _norm_rows(x, weight, bias, seg_ptr, n_groups, act, 1.0)
    if seg_ptr is None:
        _take(dy, "dy", x.dtype, x.shape)
        ld_dy = channels
    else:
        ld_dy = _take_rows(dy, "dy", x.dtype, rows, channels)
    _take(stats, "stats", _F32, (n_seg, n_groups, 2))
    device = _here(x, dy, weight, bias, stats, seg_ptr, out)
    dx, ld_dx, zero = _norm_out(x, rows, channels, out, seg_ptr, dy)
    if zero and not n_seg:
        dx.zero_()
    dweight = dbias = None
    if want_affine:
        dweight, dbias = torch.empty((2, channels), dtype=_F32, device=x.device).unbind(0)
    scratch = _scratch(_lib.load().mb_group_norm_scratch(rows, n_seg, channels, 1), x)
    _launch("mb_group_norm_bwd", _lib.MbGroupNorm, _NORM_FMT.pack(
        rows, n_seg, channels, n_groups, _DTYPES[x.dtype], act, zero, 1.0, 0, ptr(seg_ptr) or 0, xr.data_ptr(), ld, ptr(weight) or 0,
        ptr(bias) or 0, 0, 0, stats.data_ptr(), dy.data_ptr(), ld_dy, dx.data_ptr(), ld_dx, ptr(dweight) or 0, ptr(dbias) or 0,
        ptr(scratch) or 0), device)
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


def _route_args(logits, top_k):
    """Row stride, rows and experts of the router's logits."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES:
        raise TypeError(f"logits: a float32, bfloat16 or float16 tensor is wanted, got {getattr(logits, 'dtype', type(logits).__name__)}")
    ld = _take_rows(logits, "logits", logits.dtype)
    n, n_experts = logits.shape
    if not 1 <= n_experts <= 1024:
        raise NotImplementedError(f"the router takes 1 to 1024 experts, got {n_experts}")
    if not 1 <= top_k <= min(32, n_experts):
        raise ValueError(f"top_k={top_k}: 1 to {min(32, n_experts)} of {n_experts} experts")
    if n * top_k >= 1 << 31:
        raise NotImplementedError("the router takes fewer than 2**31 choices")
    return ld, n, n_experts


def route_fwd(logits, top_k, valid=None, renorm=True) -> Route:
    """Router of a mixture of experts.  p = softmax over a row's available experts (logit > -inf); the ``top_k`` largest are
    taken, equal ones by the lowest index; weights p, or p over their sum with ``renorm``.  ``valid`` [rows] bool: False rows are
    padding.  Padding and rows without an available expert have ids -1, weights 0 and no slot, and count nowhere.

    loss = experts / (top_k T^2) sum_e counts_e sum_rows p_e with T the rows routed: 1 where both are even.  Slots 0, 1, ..
    hold the pairs in order of expert, then of row: expert e has slots offsets[e] .. offsets[e+1] - 1, slot s is of row row_of[s]
    (-1 behind the last), choice j of row t has slot slot_of[t, j]."""
    ld, n, n_experts = _route_args(logits, top_k)
    if valid is not None:
        _take(valid, "valid", torch.bool, (n,))
    device = _here(logits, valid)
    renorm, pairs = bool(renorm), n * top_k
    dev, shape = logits.device, (n, top_k)
    block = torch.empty(2 * n_experts + 2 + pairs, dtype=_I32, device=dev)
    totals, offsets, row_of = torch.split_with_sizes(block, (n_experts + 1, n_experts + 1, pairs))
    ids, slot_of = torch.empty((2, *shape), dtype=_I32, device=dev).unbind(0)
    weights, loss = torch.empty(shape, dtype=_F32, device=dev), torch.empty((), dtype=_F32, device=dev)
    scratch = _scratch(_lib.load().mb_route_scratch(n, n_experts), logits)
    _launch("mb_route_fwd", _lib.MbRoute, _ROUTE_FMT.pack(
        n, n_experts, top_k, _DTYPES[logits.dtype], renorm, logits.data_ptr(), ld, ptr(valid) or 0, ids.data_ptr(), weights.data_ptr(),
        totals.data_ptr(), loss.data_ptr(), offsets.data_ptr(), row_of.data_ptr(), slot_of.data_ptr(), 0, 0, 0, 0, ptr(scratch) or 0), device)
    return Route(ids, weights, loss, totals, offsets, row_of, slot_of, renorm)


def route_bwd(logits, route: Route, dweights=None, dloss=None):
    """Gradient of the logits from those of the weights [rows, top_k] and of the balance loss (a scalar tensor); None: zero."""
    ids = route.ids
    if ids.dim() != 2:
        raise ValueError(f"route.ids: [rows, top_k] is wanted, got shape {tuple(ids.shape)}")
    top_k = ids.shape[1]
    ld, n, n_experts = _route_args(logits, top_k)
    shape = (n, top_k)
    _take(ids, "route.ids", _I32, shape)
    _take(route.weights, "route.weights", _F32, shape)
    _take(route.totals, "route.totals", _I32, (n_experts + 1,))
    if dweights is not None:
        _take(dweights, "dweights", _F32, shape)
    if dloss is not None:
        if not isinstance(dloss, torch.Tensor) or dloss.dtype != _F32:
            raise TypeError(f"dloss: a float32 tensor is wanted, got {getattr(dloss, 'dtype', type(dloss).__name__)}")
        if dloss.numel() != 1:
            raise ValueError(f"dloss: a scalar is wanted, got shape {tuple(dloss.shape)}")
    device = _here(logits, ids, route.weights, route.totals, dweights, dloss)
    dlogits = torch.empty((n, n_experts), dtype=logits.dtype, device=logits.device)
    _launch("mb_route_bwd", _lib.MbRoute, _ROUTE_FMT.pack(
        n, n_experts, top_k, _DTYPES[logits.dtype], route.renorm, logits.data_ptr(), ld, 0, ids.data_ptr(), route.weights.data_ptr(),
        route.totals.data_ptr(), 0, 0, 0, 0, ptr(dweights) or 0, ptr(dloss) or 0, dlogits.data_ptr(), n_experts, 0), device)
    return dlogits


class ExpertWeights:
    """Weights [experts, n_out, n_in] of the experts' dense layers, laid out once for ``experts_linear`` in both directions:
    two tf32 parts each, w = hi + lo to 2^-23, 16 bytes a weight.  It copies: a later change of ``w`` does not reach it."""

    __slots__ = ("shape", "parts", "ptrs")

    def __init__(self, w: torch.Tensor):
        if not isinstance(w, torch.Tensor) or w.dtype != _F32:
            raise TypeError(f"weights: a float32 tensor is wanted, got {getattr(w, 'dtype', type(w).__name__)}")
        if w.dim() != 3:
            raise ValueError(f"weights: [experts, n_out, n_in] is wanted, got shape {tuple(w.shape)}")
        if not 1 <= w.shape[0] <= 1024:
            raise NotImplementedError(f"1 to 1024 experts, got {w.shape[0]}")
        _expert_widths(w.shape[2], w.shape[1])
        device = _here(w)
        w = w.detach().contiguous()
        self.shape, self.parts = tuple(w.shape), torch.empty((4, w.numel()), dtype=_F32, device=w.device)
        first, step = self.parts.data_ptr(), 4 * w.numel()
        self.ptrs = tuple(first + i * step for i in range(4))  # hi, lo, hi and lo of the transposes
        call("mb_experts_split", *self.shape, w.data_ptr(), first, _stream() if _raw_stream is None else _raw_stream(device))


def _expert_widths(n_in, n_out):
    for n in (n_in, n_out):
        if n % D or not D <= n <= 1024:
            raise NotImplementedError(f"the experts' kernels take widths 128, 256 .. 1024, got {n_in} -> {n_out}")


def _expert_rows(x, idx, n_in, in_act):
    """Row stride and number of rows of an experts' input, and its number of slots."""
    ld = _take_rows(x, "x", _F32, width=n_in, aligned=True)
    n_rows = n_slots = x.shape[0]
    if idx is not None:
        n_slots = _take_vector(idx, "idx")
        if n_slots and not n_rows:
            raise ValueError("idx: there are no rows to take")
    if n_slots >= 1 << 31 or n_rows >= 1 << 31:
        raise NotImplementedError("fewer than 2**31 rows and slots")
    if in_act != 0 and in_act != 1:
        raise ValueError(f"in_act={in_act!r}: 0 (none) or 1 (SiLU)")
    return ld, n_rows, n_slots


def experts_linear(x, weights, offsets, bias=None, idx=None, in_act=0, out_act=0, gate=None, transposed=False, out=None):
    """Dense layers of a mixture of experts on rows grouped by expert: for the slots s of expert e
    y[s] = act(f(x[idx[s]]) W_e^T + bias_e), times SiLU'(gate[s]) where ``gate`` [slots, n_out] is given (idx None: row s itself).

    ``weights``: ExpertWeights, or a [experts, n_out, n_in] tensor that is laid out in the call; ``transposed``: W_e in the place
    of its transpose, the data gradient.  ``in_act`` / ``out_act`` 1: SiLU.  ``offsets``, ``idx``: ``Route.offsets``, ``Route.row_of``.
    Infinities in one operand and NaN give what they give in float32; infinite times infinite or subnormal values give NaN.
    A part of a grouping's offsets with the weights of those experts is a share of the work.  Slots of no expert, ahead of ``offsets[0]`` and
    from ``offsets[-1]`` on, are zero in a returned tensor and left alone in a given ``out``, which does not overlap x or ``gate``."""
    if not isinstance(weights, ExpertWeights):
        weights = ExpertWeights(weights)
    n_experts, n_out, n_in = weights.shape
    w_hi, w_lo = weights.ptrs[:2]
    if transposed:
        n_out, n_in = n_in, n_out
        w_hi, w_lo = weights.ptrs[2:]
    ld, n_rows, n_slots = _expert_rows(x, idx, n_in, in_act)
    if _take_vector(offsets, "offsets") != n_experts + 1:
        raise ValueError(f"offsets: [{n_experts + 1}] is wanted, got {tuple(offsets.shape)}")
    if out_act != 0 and out_act != 1:
        raise ValueError(f"out_act={out_act!r}: 0 (none) or 1 (SiLU)")
    if bias is not None:
        _take(bias, "bias", _F32, (n_experts, n_out))
        if bias.data_ptr() % 16:
            raise ValueError("bias has to start on a 16-byte boundary")
    ld_gate = 0 if gate is None else _take_rows(gate, "gate", _F32, n_slots, n_out, aligned=True)
    ld_y = n_out
    if out is not None:
        ld_y = _take_rows(out, "out", _F32, n_slots, n_out, aligned=True)
        _apart(out, "x", x)
        _apart(out, "gate", gate)
    device = _here(x, weights.parts, offsets, bias, idx, gate, out)
    y = torch.empty((n_slots, n_out), dtype=_F32, device=x.device) if out is None else out
    _launch("mb_experts_linear", _lib.MbExperts, _EXPERTS_FMT.pack(
        n_slots, n_rows, n_experts, n_in, n_out, in_act, out_act, out is None, offsets.data_ptr(), ptr(idx) or 0, x.data_ptr(), ld, w_hi, w_lo,
        ptr(bias) or 0, ptr(gate) or 0, ld_gate, y.data_ptr(), ld_y, 0, 0, 0, 0, 0), device)
    return y


def experts_grad_w(dy, x, offsets, idx=None, in_act=0, want_bias=True):
    """Weight gradients of ``experts_linear``: (dW [experts, n_out, n_in], dbias [experts, n_out] or None) with
    dW_e = sum over the slots of e of dy[s]^T f(x[idx[s]]), summed in a fixed order.  An expert without slots has zeros."""
    ld, n_rows, n_slots = _expert_rows(x, idx, None, in_act)
    ld_dy = _take_rows(dy, "dy", _F32, n_slots, aligned=True)
    n_in, n_out = x.shape[1], dy.shape[1]
    _expert_widths(n_in, n_out)
    n_experts = _take_vector(offsets, "offsets") - 1
    if not 1 <= n_experts <= 1024:
        raise NotImplementedError(f"1 to 1024 experts, got {n_experts}")
    device = _here(dy, x, offsets, idx)
    dw = torch.empty((n_experts, n_out, n_in), dtype=_F32, device=x.device)
    dbias = torch.empty((n_experts, n_out), dtype=_F32, device=x.device) if want_bias else None
    scratch = _scratch(_lib.load().mb_experts_grad_scratch(n_slots, n_experts, n_in, n_out), x)
    _launch("mb_experts_grad_w", _lib.MbExperts, _EXPERTS_FMT.pack(
        n_slots, n_rows, n_experts, n_in, n_out, in_act, 0, 0, offsets.data_ptr(), ptr(idx) or 0, x.data_ptr(), ld, 0, 0, 0, 0, 0, 0, 0,
        dy.data_ptr(), ld_dy, dw.data_ptr(), ptr(dbias) or 0, ptr(scratch) or 0), device)
    return dw, dbias


def _combine_args(y, slot_of, weights):
    """Row stride and shape of the experts' outputs, rows and choices a row."""
    if not isinstance(y, torch.Tensor):
        raise TypeError(f"y: a tensor is wanted, got {type(y).__name__}")
    if y.dim() != 2:
        raise ValueError(f"y: [slots, width] is wanted, got shape {tuple(y.shape)}")
    if not isinstance(slot_of, torch.Tensor) or slot_of.dtype != _I32:
        raise TypeError(f"slot_of: an int32 tensor is wanted, got {getattr(slot_of, 'dtype', type(slot_of).__name__)}")
    if slot_of.dim() != 2 or not slot_of.is_contiguous():
        raise ValueError(f"slot_of: contiguous [rows, top_k] is wanted, got shape {tuple(slot_of.shape)}, strides {slot_of.stride()}")
    (n_slots, width), (n, k) = y.shape, slot_of.shape
    if width % 4 or not width:
        raise NotImplementedError(f"widths that are multiples of 4, got {width}")
    if not 1 <= k <= 32 or n * k >= 1 << 31 or n_slots >= 1 << 31:
        raise NotImplementedError(f"1 to 32 choices a row, fewer than 2**31 in all, got {n} x {k}")
    ld = _take_rows(y, "y", _F32, aligned=True)
    if weights is not None:
        _take(weights, "weights", _F32, (n, k))
    return ld, n_slots, width, n, k


def experts_combine_fwd(y, slot_of, weights=None):
    """The experts' outputs back to their rows: out[t] = sum_j weights[t, j] y[slot_of[t, j]] over the choices with a slot
    (weights None: 1, the sum that the gradient of the gathered rows takes)."""
    ld, n_slots, width, n, k = _combine_args(y, slot_of, weights)
    device = _here(y, slot_of, weights)
    out = torch.empty((n, width), dtype=_F32, device=y.device)
    _launch("mb_experts_combine_fwd", _lib.MbCombine, _COMBINE_FMT.pack(
        n, n_slots, k, width, 0, 0, slot_of.data_ptr(), 0, ptr(weights) or 0, y.data_ptr(), ld, out.data_ptr(), width, 0, 0, 0, 0, 0), device)
    return out


def experts_combine_bwd(dout, y, slot_of, weights=None, offsets=None):
    """Gradients (dy, dweights) of ``experts_combine_fwd``: dy [slots, width], dweights [rows, top_k] (0 for a choice without a
    slot).  With ``offsets``, every slot from ``offsets[0]`` to ``offsets[-1]`` - 1 has to have its choice, as in a Route; the others are
    zero in dy and count as no slot.  Without, dy is cleared first, so that slots that no choice has are zero.  A slot
    is one choice's, as in ``Route.slot_of``: two that name the same one would overwrite each other's dy."""
    ld, n_slots, width, n, k = _combine_args(y, slot_of, weights)
    ld_dout = _take_rows(dout, "dout", _F32, n, width, aligned=True)
    n_experts = 0
    if offsets is not None:
        n_experts = _take_vector(offsets, "offsets") - 1
        if n_experts < 0:
            raise ValueError("offsets: [experts + 1] is wanted, got none")
    device = _here(dout, y, slot_of, weights, offsets)
    dy = (torch.zeros if offsets is None else torch.empty)((n_slots, width), dtype=_F32, device=y.device)
    dweights = torch.empty((n, k), dtype=_F32, device=y.device)
    _launch("mb_experts_combine_bwd", _lib.MbCombine, _COMBINE_FMT.pack(
        n, n_slots, k, width, n_experts, 0, slot_of.data_ptr(), ptr(offsets) or 0, ptr(weights) or 0, y.data_ptr(), ld, 0, 0, dout.data_ptr(),
        ld_dout, dy.data_ptr(), width, dweights.data_ptr()), device)
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
