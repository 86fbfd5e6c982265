"""Tensor-level wrappers of the HIP entry points (one per stage).

Each wrapper validates shapes on the host, allocates outputs that are not
passed in, and enqueues the HIP kernels on ``stream`` (default: torch's
current stream).  There is no CPU path: every function requires the HIP
library and CUDA (ROCm) tensors.
"""
from __future__ import annotations

import ctypes
import functools
import math
from contextlib import nullcontext
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import _lib
from ._lib import call, dtype_code, size_query, stream_handle

C_KEYS = 2048
HEAD_DIM = 128
RANK = 32

_i32, _f16, _f32 = torch.int32, torch.float16, torch.float32


def _dev(t):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError("t2t: expected a GPU tensor")
    return t.device


def _new(stream, *shape, dtype, device):
    """An output of a call on ``stream``: that stream's memory (kernels of the
    current one may still use what it freed), not reused before the current
    stream is done with it either."""
    with torch.cuda.stream(stream):
        t = torch.empty(*shape, dtype=dtype, device=device)
    if stream is not None:
        t.record_stream(torch.cuda.current_stream(device))
    return t


def _ws(nbytes, device, stream=None):
    """A call's scratch, of the stream that it runs on: released at return, the
    memory goes to that stream's later work."""
    with torch.cuda.stream(stream):
        return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


def _ws_for(ws, nbytes, device, stream=None):
    """A caller's workspace if it is a large enough uint8 buffer on ``device``,
    else a fresh one.  Its byte count is passed to the library, which checks it."""
    if ws is not None:
        if (not isinstance(ws, torch.Tensor) or ws.dtype != torch.uint8
                or not ws.is_contiguous() or ws.device != device):
            raise ValueError(f"t2t: ws must be a contiguous uint8 tensor on {device}")
        if ws.numel() >= nbytes:
            return ws
    return _ws(nbytes, device, stream)


_HALF = (torch.float16, torch.bfloat16)


def _check(t, shape, dtype, name, device=None):
    """The kernels take raw pointers and trust these geometries: a tensor of
    another shape, dtype or device would be read or written out of bounds."""
    dtypes = dtype if isinstance(dtype, tuple) else (dtype,)
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"t2t: {name} must be a tensor")
    if (tuple(t.shape) != tuple(shape) or t.dtype not in dtypes or not t.is_contiguous()
            or not t.is_cuda or (device is not None and t.device != device)):
        raise ValueError(f"t2t: {name} must be a contiguous {'/'.join(map(str, dtypes))} "
                         f"{tuple(shape)} tensor on {device or 'the GPU'}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def _rows(t, H, N, D, dtype, name, device):
    """Validate an [H, N, D] view whose rows are contiguous (unit stride along
    D, 16-byte aligned) and return its (head, row) strides in elements: the
    contiguous layout, or e.g. a token-major [N, H, D] tensor seen through
    ``.transpose(0, 1)``."""
    dtypes = dtype if isinstance(dtype, tuple) else (dtype,)
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"t2t: {name} must be a tensor")
    sh, sn = (t.stride(0), t.stride(1)) if t.dim() == 3 else (0, 0)
    if (tuple(t.shape) != (H, N, D) or t.dtype not in dtypes or t.device != device
            or t.stride(2) != 1 or sh % 8 or sn % 8 or sn < D or sh < 0
            or t.data_ptr() % 16):
        raise ValueError(f"t2t: {name} must be a {'/'.join(map(str, dtypes))} [{H}, {N}, {D}] "
                         f"tensor on {device} with contiguous 16-byte aligned rows, got "
                         f"{t.dtype} {tuple(t.shape)} strides {tuple(t.stride())} on {t.device}")
    return sh, sn


def rows_in_place(t):
    """Whether a [H, N, D] GPU tensor can be passed as a strided view."""
    try:
        _rows(t, *t.shape, _HALF, "x", t.device)
    except ValueError:
        return False
    return True


def _check_ns(ns_t, device):
    if not isinstance(ns_t, torch.Tensor) or ns_t.numel() != 1 or ns_t.dtype != _i32 \
            or ns_t.device != device:
        raise ValueError(f"t2t: ns_t must be a one-element int32 tensor on {device}")


def _check_plan(plan, H, N, CQ, device):
    if (not isinstance(plan, torch.Tensor) or plan.dtype != _i32 or not plan.is_contiguous()
            or plan.device != device or plan.numel() < plan_ints(H, N, CQ)):
        raise ValueError(f"t2t: plan must be a contiguous int32 tensor of >= "
                         f"{plan_ints(H, N, CQ)} elements on {device}")


def project(x, U, out=None, stream=None):
    """fp16(x @ U): x [H, N, D] fp16/bf16, U [H, D, 32] fp16 -> [H, N, 32] fp16."""
    H, N, D = x.shape
    dev = _dev(x)
    sxh, sxn = _rows(x, H, N, D, _HALF, "x", dev)
    _check(U, (H, D, RANK), _f16, "U", dev)
    if out is None:
        out = torch.empty(H, N, RANK, dtype=_f16, device=dev)
    _check(out, (H, N, RANK), _f16, "out", dev)
    if not x.is_contiguous():
        call("t2t_project_strided", _lib.RowView(x), dtype_code(x.dtype), U, out, H, N, D, RANK,
             sxh, sxn,
             stream_handle(stream))
        return out
    call("t2t_project", x, dtype_code(x.dtype), U, out, H, N, D, RANK, stream_handle(stream))
    return out


def kmm_ws_bytes(H, N, CQ, CK=C_KEYS):
    return size_query("t2t_kmm_ws_bytes", H, N, CQ, CK)


def kmm_run(QU, KU, V, cq0, ck0, *, pin_tail=0, out=None, ws=None, stream=None,
            write_v_sorted=True):
    """One k-means maintenance call; returns a dict of the outputs.  With
    ``write_v_sorted=False`` V_sorted is neither allocated nor written (its
    entry is None): for callers that read V through kperm."""
    H, N, r = QU.shape
    CQ, CK = cq0.shape[1], ck0.shape[1]
    dev = _dev(QU)
    _check(QU, (H, N, r), _f16, "QU", dev)
    _check(KU, (H, N, r), _f16, "KU", dev)
    _check(cq0, (H, CQ, r), _f16, "cq0", dev)
    _check(ck0, (H, CK, r), _f16, "ck0", dev)
    svh, svn = _rows(V, H, N, HEAD_DIM, _HALF, "V", dev)
    o = dict(out or {})
    o.setdefault("qlab", torch.empty(H, N, dtype=_i32, device=dev))
    o.setdefault("cq2", torch.empty(H, CQ, r, dtype=_f16, device=dev))
    o.setdefault("klab", torch.empty(H, N, dtype=_i32, device=dev))
    o.setdefault("ck2", torch.empty(H, CK, r, dtype=_f32, device=dev))
    o.setdefault("qcounts", torch.empty(H, CQ, dtype=_i32, device=dev))
    o.setdefault("qperm", torch.empty(H, N, dtype=_i32, device=dev))
    o.setdefault("kcounts", torch.empty(H, CK, dtype=_i32, device=dev))
    o.setdefault("kperm", torch.empty(H, N, dtype=_i32, device=dev))
    if write_v_sorted:
        o.setdefault("V_sorted", torch.empty(H, N, HEAD_DIM, dtype=V.dtype, device=dev))
    else:
        o["V_sorted"] = None
    o.setdefault("sumv", torch.empty(H, CK, HEAD_DIM, dtype=_f16, device=dev))
    o.setdefault("lam", torch.empty(H, dtype=_f32, device=dev))
    for name, shape, dt in (("qlab", (H, N), _i32), ("cq2", (H, CQ, r), _f16),
                            ("klab", (H, N), _i32), ("ck2", (H, CK, r), _f32),
                            ("qcounts", (H, CQ), _i32), ("qperm", (H, N), _i32),
                            ("kcounts", (H, CK), _i32), ("kperm", (H, N), _i32),
                            ("V_sorted", (H, N, HEAD_DIM), V.dtype),
                            ("sumv", (H, CK, HEAD_DIM), _f16), ("lam", (H,), _f32)):
        if o[name] is not None or name != "V_sorted":
            _check(o[name], shape, dt, name, dev)
    need = kmm_ws_bytes(H, N, CQ, CK)
    ws = _ws_for(ws, need, dev, stream)
    if V.is_contiguous():
        call("t2t_kmm_run", QU, KU, V, dtype_code(V.dtype), cq0, ck0, o["qlab"], o["cq2"],
             o["klab"], o["ck2"], o["qcounts"], o["qperm"], o["kcounts"], o["kperm"],
             o["V_sorted"], o["sumv"], o["lam"], H, N, CQ, CK, int(pin_tail), ws, ws.numel(),
             stream_handle(stream))
    else:
        call("t2t_kmm_run_strided", QU, KU, _lib.RowView(V), dtype_code(V.dtype), svh, svn, cq0,
             ck0, o["qlab"],
             o["cq2"], o["klab"], o["ck2"], o["qcounts"], o["qperm"], o["kcounts"], o["kperm"],
             o["V_sorted"], o["sumv"], o["lam"], H, N, CQ, CK, int(pin_tail), ws, ws.numel(),
             stream_handle(stream))
    return o


def vstats_ws_bytes(H, N, CK=C_KEYS):
    return size_query("t2t_vstats_ws_bytes", H, N, CK)


def vstats_gather(V, kperm, kcounts, V_sorted=None, sumv=None, lam=None, ws=None, stream=None,
                  write_v_sorted=True):
    """Reuse-call value statistics: V_sorted = V[kperm], sumv, lam.  With
    ``write_v_sorted=False`` only sumv and lam are produced (V_sorted None)."""
    H, N, D = V.shape
    CK = kcounts.shape[1]
    dev = _dev(V)
    if not write_v_sorted:
        V_sorted = None
    elif V_sorted is None:
        V_sorted = torch.empty(H, N, D, dtype=V.dtype, device=dev)
    sumv = torch.empty(H, CK, D, dtype=_f16, device=dev) if sumv is None else sumv
    lam = torch.empty(H, dtype=_f32, device=dev) if lam is None else lam
    svh, svn = _rows(V, H, N, HEAD_DIM, _HALF, "V", dev)
    _check(kperm, (H, N), _i32, "kperm", dev)
    _check(kcounts, (H, CK), _i32, "kcounts", dev)
    if V_sorted is not None:
        _check(V_sorted, (H, N, HEAD_DIM), V.dtype, "V_sorted", dev)
    _check(sumv, (H, CK, HEAD_DIM), _f16, "sumv", dev)
    _check(lam, (H,), _f32, "lam", dev)
    need = vstats_ws_bytes(H, N, CK)
    ws = _ws_for(ws, need, dev, stream)
    if V.is_contiguous():
        call("t2t_kmm_run_vstats_gather", V, dtype_code(V.dtype), kperm, kcounts, V_sorted, sumv,
             lam, H, N, CK, ws, ws.numel(), stream_handle(stream))
    else:
        call("t2t_kmm_run_vstats_gather_strided", _lib.RowView(V), dtype_code(V.dtype), svh, svn,
             kperm, kcounts,
             V_sorted, sumv, lam, H, N, CK, ws, ws.numel(), stream_handle(stream))
    return V_sorted, sumv, lam


def vstats(V_sorted, kcounts, sumv=None, lam=None, ws=None, stream=None):
    H, N, D = V_sorted.shape
    CK = kcounts.shape[1]
    dev = _dev(V_sorted)
    sumv = torch.empty(H, CK, D, dtype=_f16, device=dev) if sumv is None else sumv
    lam = torch.empty(H, dtype=_f32, device=dev) if lam is None else lam
    _check(V_sorted, (H, N, HEAD_DIM), _HALF, "V_sorted", dev)
    _check(kcounts, (H, CK), _i32, "kcounts", dev)
    _check(sumv, (H, CK, HEAD_DIM), _f16, "sumv", dev)
    _check(lam, (H,), _f32, "lam", dev)
    need = vstats_ws_bytes(H, N, CK)
    ws = _ws_for(ws, need, dev, stream)
    call("t2t_kmm_run_vstats", V_sorted, dtype_code(V_sorted.dtype), kcounts, sumv, lam, H, N, CK,
         ws, ws.numel(), stream_handle(stream))
    return sumv, lam


def centroid_finalize(ck2, scale=1.0 / math.sqrt(HEAD_DIM), ck16=None, cks=None, stream=None):
    """(fp16(ck2), fp16(fp32(ck2 * scale)))."""
    H, CK, r = ck2.shape
    dev = _dev(ck2)
    ck16 = torch.empty(H, CK, r, dtype=_f16, device=dev) if ck16 is None else ck16
    cks = torch.empty(H, CK, r, dtype=_f16, device=dev) if cks is None else cks
    _check(ck2, (H, CK, r), _f32, "ck2", dev)
    _check(ck16, (H, CK, r), _f16, "ck16", dev)
    _check(cks, (H, CK, r), _f16, "cks", dev)
    call("t2t_centroid_finalize", ck2, ck16, cks, float(scale), H, CK, r, stream_handle(stream))
    return ck16, cks


def score(QU, cks, out=None, stream=None):
    """gl = fp16(QU @ cks^T): [H, N, 2048] fp16."""
    H, N, r = QU.shape
    CK = cks.shape[1]
    dev = _dev(QU)
    out = torch.empty(H, N, CK, dtype=_f16, device=dev) if out is None else out
    _check(QU, (H, N, r), _f16, "QU", dev)
    _check(cks, (H, CK, r), _f16, "cks", dev)
    _check(out, (H, N, CK), _f16, "out", dev)
    call("t2t_score", QU, cks, out, H, N, CK, r, stream_handle(stream))
    return out


def select_ws_bytes(H, N, CQ):
    return size_query("t2t_select_ws_bytes", H, N, CQ)


def _check_select(dev, H, N, CQ, *, gl=None, kcounts=None, qperm=None, qcounts=None, unip=None,
                  rowcnt=None):
    if gl is not None:
        _check(gl, (H, N, C_KEYS), _f16, "gl", dev)
    _check(kcounts, (H, C_KEYS), _i32, "kcounts", dev)
    _check(qperm, (H, N), _i32, "qperm", dev)
    _check(qcounts, (H, CQ), _i32, "qcounts", dev)
    if unip is not None:
        _check(unip, (H, CQ, C_KEYS // 32), _i32, "unip", dev)
    _check(rowcnt, (H, N), _i32, "rowcnt", dev)


def select_union(gl, kcounts, qperm, qcounts, ns_t, unip=None, rowcnt=None, ws=None,
                 split_cap=0, stream=None):
    """Packed union [H, CQ, 64] int32 and rowcnt [H, N] int32."""
    H, N, CK = gl.shape
    CQ = qcounts.shape[1]
    dev = _dev(gl)
    if CK != C_KEYS:
        raise ValueError("t2t: selection requires 2048 key clusters")
    unip = torch.empty(H, CQ, CK // 32, dtype=_i32, device=dev) if unip is None else unip
    rowcnt = torch.empty(H, N, dtype=_i32, device=dev) if rowcnt is None else rowcnt
    _check_select(dev, H, N, CQ, gl=gl, kcounts=kcounts, qperm=qperm, qcounts=qcounts,
                  unip=unip, rowcnt=rowcnt)
    _check_ns(ns_t, dev)
    need = select_ws_bytes(H, N, CQ)
    ws = _ws_for(ws, need, dev, stream)
    if split_cap:
        call("t2t_select_run_split_packed", gl, kcounts, qperm, qcounts, int(split_cap), ns_t, unip,
             rowcnt, H, N, CQ, ws, ws.numel(), stream_handle(stream))
    else:
        call("t2t_select_run_packed", gl, kcounts, qperm, qcounts, ns_t, unip, rowcnt, H, N, CQ, ws,
             ws.numel(), stream_handle(stream))
    return unip, rowcnt


def score_select(QU, cks, kcounts, qperm, qcounts, ns_t, unip=None, rowcnt=None, ws=None,
                 stream=None):
    """Fused scoring + selection: packed union [H, CQ, 64] int32 and rowcnt
    [H, N], identical to score() followed by select_union()."""
    H, N, r = QU.shape
    CQ = qcounts.shape[1]
    dev = _dev(QU)
    if cks.shape != (H, C_KEYS, RANK):
        raise ValueError("t2t: score_select requires cks [H, 2048, 32]")
    unip = torch.empty(H, CQ, C_KEYS // 32, dtype=_i32, device=dev) if unip is None else unip
    rowcnt = torch.empty(H, N, dtype=_i32, device=dev) if rowcnt is None else rowcnt
    _check(QU, (H, N, RANK), _f16, "QU", dev)
    _check(cks, (H, C_KEYS, RANK), _f16, "cks", dev)
    _check_select(dev, H, N, CQ, kcounts=kcounts, qperm=qperm, qcounts=qcounts, unip=unip,
                  rowcnt=rowcnt)
    _check_ns(ns_t, dev)
    need = select_ws_bytes(H, N, CQ)
    ws = _ws_for(ws, need, dev, stream)
    call("t2t_score_select_packed", QU, cks, kcounts, qperm, qcounts, ns_t, unip, rowcnt, H, N, CQ,
         ws, ws.numel(), stream_handle(stream))
    return unip, rowcnt


def select_union_bytes(gl, kcounts, qperm, qcounts, ns_t, uni=None, rowcnt=None, ws=None,
                       stream=None):
    """Byte-per-cluster union [H, CQ, 2048] uint8 (the reference's `run`)."""
    H, N, CK = gl.shape
    CQ = qcounts.shape[1]
    dev = _dev(gl)
    uni = torch.empty(H, CQ, CK, dtype=torch.uint8, device=dev) if uni is None else uni
    rowcnt = torch.empty(H, N, dtype=_i32, device=dev) if rowcnt is None else rowcnt
    _check(uni, (H, CQ, CK), torch.uint8, "uni", dev)
    _check_select(dev, H, N, CQ, gl=gl, kcounts=kcounts, qperm=qperm, qcounts=qcounts,
                  rowcnt=rowcnt)
    _check_ns(ns_t, dev)
    need = select_ws_bytes(H, N, CQ)
    ws = _ws_for(ws, need, dev, stream)
    call("t2t_select_run", gl, kcounts, qperm, qcounts, ns_t, uni, rowcnt, H, N, CQ, ws, ws.numel(),
         stream_handle(stream))
    return uni, rowcnt


def union_or_last(unip, stream=None):
    H, CQ, W = unip.shape
    _check(unip, (H, CQ, C_KEYS // 32), _i32, "unip")
    call("t2t_union_or_last", unip, H, CQ, W * 32, stream_handle(stream))
    return unip


def fast_gather(x, perm, out=None, stream=None):
    """o[h, i] = x[h, perm[h, i]] for [H, N, D] 16-bit tensors."""
    H, N, D = x.shape
    dev = _dev(x)
    out = torch.empty_like(x) if out is None else out
    _check(x, (H, N, D), _HALF, "x", dev)
    _check(perm, (H, N), _i32, "perm", dev)
    _check(out, (H, N, D), x.dtype, "out", dev)
    call("t2t_fast_gather", x, dtype_code(x.dtype), perm, out, H, N, D, stream_handle(stream))
    return out


def plan_ints(H, N, CQ):
    return size_query("t2t_tile_plan_ints", H, N, CQ)


def tile_plan(qcounts, kcounts, unip, N, plan=None, stream=None):
    H, CQ = qcounts.shape
    dev = _dev(qcounts)
    if plan is None:
        plan = torch.empty(plan_ints(H, N, CQ), dtype=_i32, device=dev)
    _check(qcounts, (H, CQ), _i32, "qcounts", dev)
    _check(kcounts, (H, C_KEYS), _i32, "kcounts", dev)
    _check(unip, (H, CQ, C_KEYS // 32), _i32, "unip", dev)
    _check_plan(plan, H, N, CQ, dev)
    call("t2t_tile_plan", qcounts, kcounts, unip, plan, H, N, CQ, stream_handle(stream))
    return plan


def plan_views(plan, H, N, CQ):
    """Named views of a plan buffer (k_off, kvlen, ntask, tasks)."""
    maxT = CQ + (N + 127) // 128 + 1  # tasks of <= 128 queries
    o = 0
    k_off = plan[o:o + H * 2049].view(H, 2049); o += H * 2049
    kvlen = plan[o:o + H * CQ].view(H, CQ); o += H * CQ
    ntask = plan[o:o + H]; o += H
    tasks = plan[o:o + H * maxT * 4].view(H, maxT, 4)
    return dict(k_off=k_off, kvlen=kvlen, ntask=ntask, tasks=tasks)


def _check_attn(dev, H, N, CQ, *, q=None, kp=None, vp=None, kcounts=None, unip=None, qperm=None,
                plan=None, out=None, lse=None, QU=None, cks=None, sumv=None, lam=None, qlab=None,
                tailw_t=None, qcounts=None, tiles=None, dt=None):
    qs = (H, N, HEAD_DIM)
    for name, t, shape, dtype in (
            ("q", q, qs, _HALF), ("kp", kp, qs, dt), ("vp", vp, qs, dt), ("out", out, qs, dt),
            ("kcounts", kcounts, (H, C_KEYS), _i32), ("qcounts", qcounts, (H, CQ), _i32),
            ("unip", unip, (H, CQ, C_KEYS // 32), _i32), ("qperm", qperm, (H, N), _i32),
            ("qlab", qlab, (H, N), _i32), ("lse", lse, (H, N), _f32),
            ("QU", QU, (H, N, RANK), _f16), ("cks", cks, (H, C_KEYS, RANK), _f16),
            ("sumv", sumv, (H, C_KEYS, HEAD_DIM), _f16), ("lam", lam, (H,), _f32),
            ("tailw_t", tailw_t, (), _f32)):
        if t is not None:
            _check(t, shape, dtype, name, dev)
    if plan is not None:
        _check_plan(plan, H, N, CQ, dev)
    if tiles is not None:
        need = size_query("t2t_centroid_tiles_bytes", H)
        if (not isinstance(tiles, torch.Tensor) or tiles.dtype != torch.uint8
                or not tiles.is_contiguous() or tiles.device != dev or tiles.numel() < need):
            raise ValueError(f"t2t: tiles must be a contiguous uint8 tensor of >= {need} bytes "
                             f"on {dev}")


def tile_attn_exact(q, kp, vp, kcounts, unip, qperm, plan, attn_out=None, lse=None, stream=None):
    """Exact attention over the unions, sorted query order."""
    H, N, D = q.shape
    CQ = unip.shape[1]
    dev = _dev(q)
    attn_out = torch.empty_like(q) if attn_out is None else attn_out
    lse = torch.empty(H, N, dtype=_f32, device=dev) if lse is None else lse
    _check_attn(dev, H, N, CQ, q=q, kp=kp, vp=vp, kcounts=kcounts, unip=unip, qperm=qperm,
                plan=plan, out=attn_out, lse=lse, dt=q.dtype)
    call("t2t_tile_attn_exact", q, kp, vp, dtype_code(q.dtype), kcounts, unip, qperm, plan,
         attn_out, lse, H, N, CQ, stream_handle(stream))
    return attn_out, lse


def tail_merge(attn_out, lse, QU, cks, sumv, kcounts, unip, qlab, qperm, lam, tailw_t, out=None,
               ws=None, stream=None):
    H, N, D = attn_out.shape
    CQ = unip.shape[1]
    dev = _dev(attn_out)
    out = torch.empty_like(attn_out) if out is None else out
    _check_attn(dev, H, N, CQ, q=attn_out, out=out, lse=lse, QU=QU, cks=cks, sumv=sumv,
                kcounts=kcounts, unip=unip, qlab=qlab, qperm=qperm, lam=lam, tailw_t=tailw_t,
                dt=attn_out.dtype)
    need = size_query("t2t_tail_merge_ws_bytes", H)
    ws = _ws_for(ws, need, dev, stream)
    call("t2t_tail_merge", attn_out, lse, QU, cks, sumv, kcounts, unip, qlab, qperm, lam, tailw_t,
         out, dtype_code(attn_out.dtype), H, N, CQ, ws, ws.numel(), stream_handle(stream))
    return out


def centroid_tiles(cks, sumv, tiles=None, stream=None):
    """Tile image of cks / sumv staged by the residual kernel (uint8 bytes)."""
    H = cks.shape[0]
    dev = _dev(cks)
    need = size_query("t2t_centroid_tiles_bytes", H)
    tiles = _ws(need, dev) if tiles is None else tiles
    _check_attn(dev, H, 0, 0, cks=cks, sumv=sumv, tiles=tiles)
    call("t2t_centroid_tiles", cks, sumv, tiles, H, stream_handle(stream))
    return tiles


def tile_attn_exact_orig(q, kp, vp, kcounts, unip, qperm, plan, out, lse, stream=None):
    """Exact attention written at the original rows of out; lse in sorted order."""
    H, N, D = q.shape
    CQ = unip.shape[1]
    _check_attn(_dev(q), H, N, CQ, q=q, kp=kp, vp=vp, kcounts=kcounts, unip=unip, qperm=qperm,
                plan=plan, out=out, lse=lse, dt=q.dtype)
    call("t2t_tile_attn_exact_orig", q, kp, vp, dtype_code(q.dtype), kcounts, unip, qperm, plan,
         out, lse, H, N, CQ, stream_handle(stream))
    return out


def tile_attn_exact_orig_gather(q, k, kperm, vp, kcounts, unip, qperm, plan, out, lse, stream=None):
    """tile_attn_exact_orig reading K in place: k in the original order, key
    position p of the cluster order at row kperm[h, p] (no kp = k[kperm]).
    q, k and out may be strided [H, N, 128] views with contiguous rows (e.g.
    token-major tensors through ``.transpose(0, 1)``)."""
    H, N, D = q.shape
    CQ = unip.shape[1]
    dev = _dev(q)
    sq = _rows(q, H, N, HEAD_DIM, _HALF, "q", dev)
    sk = _rows(k, H, N, HEAD_DIM, q.dtype, "k", dev)
    so = _rows(out, H, N, HEAD_DIM, q.dtype, "out", dev)
    _check_attn(dev, H, N, CQ, vp=vp, kcounts=kcounts, unip=unip, qperm=qperm, plan=plan,
                lse=lse, dt=q.dtype)
    _check(kperm, (H, N), _i32, "kperm", dev)
    if q.is_contiguous() and k.is_contiguous() and out.is_contiguous():
        call("t2t_tile_attn_exact_orig_gather", q, k, kperm, vp, dtype_code(q.dtype), kcounts,
             unip, qperm, plan, out, lse, H, N, CQ, stream_handle(stream))
    else:
        call("t2t_tile_attn_exact_orig_gather_strided", _lib.RowView(q), *sq, _lib.RowView(k),
             *sk, kperm, vp, dtype_code(q.dtype), kcounts, unip, qperm, plan, _lib.RowView(out),
             *so, lse, H, N, CQ, stream_handle(stream))
    return out

def tile_attn_exact_orig_gather_kv(q, k, v, kperm, kcounts, unip, qperm, plan, out, lse,
                                   stream=None):
    """Exact attention with both gathers fused: k and v in the original order,
    key position p of the cluster order at row kperm[h, p] of each (neither
    kp nor V_sorted is stored).  q, k, v and out may be strided [H, N, 128]
    views with contiguous rows."""
    H, N, D = q.shape
    CQ = unip.shape[1]
    dev = _dev(q)
    sq = _rows(q, H, N, HEAD_DIM, _HALF, "q", dev)
    sk = _rows(k, H, N, HEAD_DIM, q.dtype, "k", dev)
    sv = _rows(v, H, N, HEAD_DIM, q.dtype, "v", dev)
    so = _rows(out, H, N, HEAD_DIM, q.dtype, "out", dev)
    _check_attn(dev, H, N, CQ, kcounts=kcounts, unip=unip, qperm=qperm, plan=plan, lse=lse,
                dt=q.dtype)
    _check(kperm, (H, N), _i32, "kperm", dev)
    call("t2t_tile_attn_exact_orig_gather_kv_strided", _lib.RowView(q), *sq, _lib.RowView(k), *sk,
         _lib.RowView(v), *sv, kperm, dtype_code(q.dtype), kcounts, unip, qperm, plan,
         _lib.RowView(out), *so, lse, H, N, CQ, stream_handle(stream))
    return out


def attn_split_ws_bytes(H, N, CQ):
    """Workspace of tile_attn_exact_split (0: these sizes are not split)."""
    return size_query("t2t_tile_attn_split_ws_bytes", H, N, CQ)


def tile_attn_exact_split(q, k, v, kperm, kcounts, unip, qlab, qperm, plan, out, lse, ws=None,
                          stream=None, gather=2):
    """Exact attention at the original rows of out with the tasks of a small
    call split along the keys (fp32 parts in ``ws``).  ``gather`` 2: as
    tile_attn_exact_orig_gather_kv; 1: as tile_attn_exact_orig_gather (v is
    cluster ordered); 0: as tile_attn_exact_orig (k and v are, kperm unused).
    qlab are the labels that qperm sorts."""
    H, N, D = q.shape
    CQ = unip.shape[1]
    dev = _dev(q)
    sq = _rows(q, H, N, HEAD_DIM, _HALF, "q", dev)
    sk = _rows(k, H, N, HEAD_DIM, q.dtype, "k", dev)
    sv = _rows(v, H, N, HEAD_DIM, q.dtype, "v", dev)
    so = _rows(out, H, N, HEAD_DIM, q.dtype, "out", dev)
    _check_attn(dev, H, N, CQ, kcounts=kcounts, unip=unip, qlab=qlab, qperm=qperm, plan=plan,
                lse=lse, dt=q.dtype)
    if gather:
        _check(kperm, (H, N), _i32, "kperm", dev)
    ws = _ws_for(ws, attn_split_ws_bytes(H, N, CQ), dev, stream)
    call("t2t_tile_attn_exact_split", _lib.RowView(q), *sq, _lib.RowView(k), *sk, _lib.RowView(v),
         *sv, kperm if gather else None, int(gather), dtype_code(q.dtype), kcounts, unip, qlab,
         qperm, plan, _lib.RowView(out), *so, lse, H, N, CQ, ws, ws.numel(), stream_handle(stream))
    return out


def resid_merge_inplace(out, lse, QU, tiles, kcounts, unip, qlab, qperm, lam, tailw_t,
                        stream=None):
    """Residual + merge into the exact part held at the original rows of out
    (out may be a strided [H, N, 128] view with contiguous rows)."""
    H, N, D = out.shape
    CQ = unip.shape[1]
    dev = _dev(out)
    so = _rows(out, H, N, HEAD_DIM, _HALF, "out", dev)
    _check_attn(dev, H, N, CQ, lse=lse, QU=QU, tiles=tiles, kcounts=kcounts, unip=unip,
                qlab=qlab, qperm=qperm, lam=lam, tailw_t=tailw_t)
    if out.is_contiguous():
        call("t2t_resid_merge_inplace", out, lse, QU, tiles, kcounts, unip, qlab, qperm, lam,
             tailw_t, dtype_code(out.dtype), H, N, CQ, stream_handle(stream))
    else:
        call("t2t_resid_merge_inplace_strided", _lib.RowView(out), *so, lse, QU, tiles, kcounts,
             unip, qlab,
             qperm, lam, tailw_t, dtype_code(out.dtype), H, N, CQ, stream_handle(stream))
    return out


def attn_ws_bytes(H, N, dtype):
    return size_query("t2t_tile_attn_ws_bytes", H, N, dtype_code(dtype))


def tile_attn_run_planned(q, kp, vp, qcounts, kcounts, unip, QU, cks, sumv, lam, qlab, qperm,
                          tailw_t, out, plan, rebuild, ws=None, stream=None):
    H, N, D = q.shape
    CQ = qcounts.shape[1]
    dev = _dev(q)
    _check_attn(dev, H, N, CQ, q=q, kp=kp, vp=vp, qcounts=qcounts, kcounts=kcounts, unip=unip,
                QU=QU, cks=cks, sumv=sumv, lam=lam, qlab=qlab, qperm=qperm, tailw_t=tailw_t,
                out=out, plan=plan, dt=q.dtype)
    need = attn_ws_bytes(H, N, q.dtype)
    if ws is not None:  # lse and the tile image suffice: nothing is split then
        need = min(need, -(-H * N * 4 // 256) * 256 + size_query("t2t_centroid_tiles_bytes", H))
    ws = _ws_for(ws, need, dev, stream)
    call("t2t_tile_attn_run_planned", q, kp, vp, dtype_code(q.dtype), qcounts, kcounts, unip, QU,
         cks, sumv, lam, qlab, qperm, tailw_t, out, plan, int(bool(rebuild)), H, N, CQ, ws,
         ws.numel(), stream_handle(stream))
    return out


def fast_assign_labels(x, c, out=None, stream=None):
    H, N, D = x.shape
    C = c.shape[1]
    dev = _dev(x)
    out = torch.empty(H, N, dtype=_i32, device=dev) if out is None else out
    _check(x, (H, N, D), _f16, "x", dev)
    _check(c, (H, C, D), _f16, "c", dev)
    _check(out, (H, N), _i32, "out", dev)
    call("t2t_fast_assign", x, c, out, H, N, C, D, stream_handle(stream))
    return out


def det_centroid_update(x, labels, old, stream=None):
    """Deterministic int64 fixed-point centroid update -> (new fp16, counts)."""
    H, N, D = x.shape
    C = old.shape[1]
    dev = _dev(x)
    _check(x, (H, N, D), _f16, "x", dev)
    _check(labels, (H, N), _i32, "labels", dev)
    _check(old, (H, C, D), _f16, "old", dev)
    new = torch.empty(H, C, D, dtype=_f16, device=dev)
    counts = torch.empty(H, C, dtype=_i32, device=dev)
    ws = _ws(size_query("t2t_det_update_ws_bytes", H, N, C), dev, stream)
    call("t2t_det_centroid_update", x, labels, old, new, counts, H, N, C, D, ws, ws.numel(),
         stream_handle(stream))
    return new, counts


def fused_update_vstats(x, labels, old, v=None, stream=None, check_labels=True, half=False):
    """fp32 centroid means (empty clusters keep ``old``), counts, and the
    fp32 per-cluster means of v when given -> (cent fp32 [H, C, D], counts
    int32 [H, C], vmean fp32 [H, C, 128] or None); with ``half`` the means are
    rounded to x's and v's types.  ``check_labels`` raises ValueError for labels
    outside [0, C), which the kernels leave out of every cluster (it reads the
    counts' sum back, a synchronisation); callers whose labels come from an
    assignment kernel pass False."""
    H, N, D = x.shape
    C = old.shape[1]
    dev = _dev(x)
    _check(x, (H, N, D), _f16, "x", dev)
    _check(labels, (H, N), _i32, "labels", dev)
    _check(old, (H, C, D), _f16, "old", dev)
    if v is not None:
        _check(v, (H, N, HEAD_DIM), _HALF, "v", dev)
    cent = torch.empty(H, C, D, dtype=_f16 if half else _f32, device=dev)
    counts = torch.empty(H, C, dtype=_i32, device=dev)
    vmean = None
    if v is not None:
        vmean = torch.empty(H, C, HEAD_DIM, dtype=v.dtype if half else _f32, device=dev)
    ws = _ws(size_query("t2t_det_update_ws_bytes", H, N, C), dev, stream)
    call("t2t_fused_update_vstats16" if half else "t2t_fused_update_vstats", x, labels, old, v,
         dtype_code(v.dtype) if v is not None else 0, cent, counts, vmean, H, N, C, D, ws, ws.numel(),
         stream_handle(stream))
    if check_labels:
        with torch.cuda.stream(stream) if stream is not None else nullcontext():
            rows = int(counts.sum())
        if rows != H * N:
            lo, hi = (int(t) for t in torch.aminmax(labels))
            raise ValueError(f"t2t: labels must lie in [0, {C}), got [{lo}, {hi}]")
    return cent, counts, vmean


def lloyd(x, cen, iters, stream=None):
    """``iters`` warm Lloyd iterations in place on cen [H, C, 32] fp16: the
    labels of fast_assign_labels and the means of fused_update_vstats in fp16."""
    H, N, D = x.shape
    C = cen.shape[1]
    dev = _dev(x)
    _check(x, (H, N, D), _f16, "x", dev)
    _check(cen, (H, C, D), _f16, "cen", dev)
    ws = _ws(size_query("t2t_lloyd_ws_bytes", H, N, C), dev, stream)
    call("t2t_lloyd", x, cen, int(iters), H, N, C, D, ws, ws.numel(), stream_handle(stream))
    return cen


def gram(x, stream=None):
    """x^T x / N per head in fp64: [H, D, D]."""
    H, N, D = x.shape
    _check(x, (H, N, D), _HALF, "x", _dev(x))
    G = torch.empty(H, D, D, dtype=torch.float64, device=_dev(x))
    nws = size_query("t2t_gram_ws_bytes", H, N, D)
    ws = _ws(nws, _dev(x), stream)
    call("t2t_gram", x, dtype_code(x.dtype), G, H, N, D, ws, nws, stream_handle(stream))
    return G


def gram_strided(x, nonfinite=None, stream=None):
    """gram() of any [H, N, D] view with unit stride along D; ``nonfinite``
    ([H] int32, optional) receives 1 for every head holding an inf or NaN."""
    H, N, D = x.shape
    dev = _dev(x)
    if x.dtype not in _HALF or x.stride(2) != 1 or x.stride(1) < D or x.stride(0) < 0:
        raise ValueError(f"t2t: gram_strided needs fp16 or bf16 rows of unit stride, got {x.dtype} "
                         f"{tuple(x.shape)} strides {tuple(x.stride())}")
    if nonfinite is not None:
        _check(nonfinite, (H,), _i32, "nonfinite", dev)
    G = _new(stream, H, D, D, dtype=torch.float64, device=dev)
    nws = size_query("t2t_gram_ws_bytes", H, N, D)
    ws = _ws(nws, dev, stream)
    call("t2t_gram_strided", _lib.RowView(x), dtype_code(x.dtype), x.stride(0), x.stride(1), G,
         nonfinite, H, N, D, ws, nws, stream_handle(stream))
    return G


def fit_chol(Mq, Mk, floor, small, stream=None):
    """Lower Cholesky factor of Mk [H, D, D] fp64; ``small`` ([2, H] int32)
    receives 1 where Mq[h] / Mk[h] has an eigenvalue not above ``floor``."""
    H, D, _ = Mq.shape
    dev = _dev(Mq)
    _check(Mq, (H, D, D), torch.float64, "Mq", dev)
    _check(Mk, (H, D, D), torch.float64, "Mk", dev)
    _check(small, (2, H), _i32, "small", dev)
    L = _new(stream, H, D, D, dtype=torch.float64, device=dev)
    call("t2t_fit_chol", Mq, Mk, L, small, H, D, float(floor), stream_handle(stream))
    return L


# ---------------------------------------------------------------------------
# the block's steps around attention: rotary positions, MXFP4 linear layers
# ---------------------------------------------------------------------------
# (single-token calls are bound by the host: checks are written for few
# operations, and a matrix in MXFP4 is checked once, when it is made)
_functions = {}
_sizes_of = functools.lru_cache(1024)(size_query)  # (of sizes alone)


def _launch(name, dev, stream, tensors, *args):
    """Call an entry point on ``stream`` (default: ``dev``'s current one) with
    ``dev`` current.  On a stream of the caller's choice the memory of
    ``tensors`` is not reused before the stream is done with it."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _launch(name, dev, stream, tensors, *args)
    if stream is None:
        handle = torch._C._cuda_getCurrentRawStream(dev.index)
    else:
        handle = stream.cuda_stream
        for t in tensors:
            if t is not None:
                t.record_stream(stream)
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_lib.lib(), name)
    rc = fn(*args, handle)
    if rc:
        raise RuntimeError(f"{name} failed (code {rc}): "
                           f"{_lib.lib().t2t_last_error().decode(errors='replace')}")


def _on(stream, dev):
    if stream is not None and stream.device != dev:
        raise ValueError(f"t2t: the stream is on {stream.device}, the tensors on {dev}")


def _empty(stream, shape, dtype, dev):
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    return _new(stream, *shape, dtype=dtype, device=dev)


def _is(t, shape, dtype, dev):
    """_check without its message."""
    return (isinstance(t, torch.Tensor) and t.shape == shape and t.dtype == dtype and t.device == dev
            and t.is_contiguous())


def _same_view(a, b):
    return a is b or (a.data_ptr() == b.data_ptr()
                      and all(n < 2 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride())))


def _scattered(t):
    """Whether a view's elements all have an address of their own."""
    if t.is_contiguous():
        return True
    last = 0
    for st, sz in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if st <= last:
            return False
        last += st * (sz - 1)
    return True


def _span(t):
    """First address and the one behind the last of a tensor's elements."""
    p = t.data_ptr()
    if t.is_contiguous():
        return p, p + t.nbytes
    if t.numel() == 0:
        return p, p
    return p, p + (sum(st * (sz - 1) for st, sz in zip(t.stride(), t.shape)) + 1) * t.element_size()


def _in_slots(a, b):
    """Whether the two lie in parts of their own of slots of one stride (the usual
    interleaved views, without the search)."""
    d, ea, eb = b.data_ptr() - a.data_ptr(), a.element_size(), b.element_size()
    da = [(s * ea, n - 1) for s, n in zip(a.stride(), a.shape) if n > 1]
    db = [(s * eb, n - 1) for s, n in zip(b.stride(), b.shape) if n > 1]
    for st, _ in da:
        if st:
            at = d % st
            if (ea + sum(s * n for s, n in da if s % st) <= at
                    and eb + sum(s * n for s, n in db if s % st) <= st - at):
                return True
    return False


def _meet(a, b):
    """Whether two tensors whose spans meet share memory (interleaved views, such
    as q and k of one projection, do not).  An element of each has the same
    address where the difference of the bases is a sum of multiples of all
    strides: the multiples are searched from the largest stride down, within what
    the smaller ones can make up for."""
    if _in_slots(a, b):
        return False
    mul = {1: [1 - b.element_size(), a.element_size() - 1]}  # stride in bytes: lowest, highest multiple
    for t, side in ((a, 1), (b, 0)):
        for st, sz in zip(t.stride(), t.shape):
            if st and sz > 1:
                mul.setdefault(st * t.element_size(), [0, 0])[side] += (sz - 1) if side else (1 - sz)
    strides = sorted(mul, reverse=True)
    low, high = [0], [0]  # reach of the strides from i on
    for st in reversed(strides):
        low.insert(0, low[0] + st * mul[st][0])
        high.insert(0, high[0] + st * mul[st][1])
    work = 4096  # (odd combinations of strides are left to the caller)

    def search(d, i):
        nonlocal work
        if i == len(strides):
            return d == 0
        st = strides[i]
        for k in range(max(mul[st][0], -((high[i + 1] - d) // st)), min(mul[st][1], (d - low[i + 1]) // st) + 1):
            work -= 1
            if work < 0:
                return False
            if search(d - k * st, i + 1):
                return True
        return False

    return search(b.data_ptr() - a.data_ptr(), 0)


def _near(lo, hi, spans):
    """Whether addresses [lo, hi) meet one of spans ((address, bytes) each)."""
    for p, n in spans:
        if p < hi and lo < p + n:
            return True
    return False


def _apart(outs, names, ins):
    """The outputs share no memory with one another or with the inputs, but that
    outs[i] may be ins[i]."""
    at = [(0, 0) if t is None else _span(t) for t in ins]
    to = [at[i] if o is ins[i] else _span(o) for i, o in enumerate(outs)]
    for i, (lo, hi) in enumerate(to):
        o, meets = outs[i], False
        for j, (a, b) in enumerate(at):
            if a < hi and lo < b:
                t = ins[j]
                if t is o if j == i else j < len(outs) and outs[j] is t:
                    continue  # in its own input's place; the place of an output, which comes below
                meets = meets or not (j == i and _same_view(o, t)) and _meet(o, t)
        for j in range(i):
            meets = meets or to[j][0] < hi and lo < to[j][1] and _meet(o, outs[j])
        if meets:
            raise ValueError(f"t2t: {names[i]} shares memory with another argument of the call")


@dataclass(frozen=True)
class RotaryScaling:
    """How the frequencies f[i] = base^(-2 i / d) are stretched for contexts
    ``factor`` times as long as the ``original`` one:

    - ``linear``: f[i] / factor;
    - ``ntk``: base * factor^(d / (d - 2)) in the place of base;
    - ``yarn``: f[i] (1 - r) + f[i] / factor r, r rising from 0 to 1 between
      the pairs that turn ``beta_fast`` and ``beta_slow`` times over the
      original length; cos and sin times ``attention`` (default
      0.1 ln(factor) + 1)."""

    kind: str
    factor: float
    original: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention: float | None = None


class RotaryFrequencies(NamedTuple):
    """Frequencies of every pair (fp64, on the device), the pairs of each
    position axis and the factor of cos and sin."""

    freqs: torch.Tensor
    pairs: tuple[int, ...]
    factor: float


def rotary_frequencies(dims, *, base=10000.0, scaling=None, device):
    """The frequencies of rotated channels ``dims`` (an even number, or one
    for each of up to four position axes), to be kept by the program."""
    given = dims
    try:
        dims = tuple(dims)
    except TypeError:
        dims = (dims,)
    try:
        whole = [int(d) for d in dims]
        fits = 1 <= len(whole) <= 4 and all(w == d and 2 <= w <= 8192 and w % 2 == 0 for w, d in zip(whole, dims))
    except (TypeError, ValueError, OverflowError):
        fits = False
    if not fits:
        raise ValueError(f"t2t: dims must be one to four even numbers in [2, 8192], got {given}")
    dims = tuple(whole)
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError(f"t2t: base must be above 1, got {base}")
    factor = 1.0
    if scaling is not None:
        if scaling.kind not in ("linear", "ntk", "yarn"):
            raise ValueError(f"t2t: scaling kind {scaling.kind!r} (linear, ntk or yarn)")
        if not (math.isfinite(scaling.factor) and scaling.factor >= 1.0):
            raise ValueError(f"t2t: scaling factor must be at least 1, got {scaling.factor}")
        if scaling.kind == "yarn":
            if scaling.original < 1 or not scaling.beta_fast > scaling.beta_slow > 0:
                raise ValueError("t2t: yarn needs the original length and beta_fast > beta_slow > 0")
            factor = scaling.attention
            if factor is None:
                factor = 0.1 * math.log(scaling.factor) + 1.0
    f = []
    for d in dims:
        b = base
        if scaling is not None and scaling.kind == "ntk":
            if d == 2:
                raise ValueError("t2t: ntk scaling needs more than one pair an axis")
            b = base * scaling.factor ** (d / (d - 2.0))
        fd = [b ** (-2.0 * i / d) for i in range(d // 2)]
        if scaling is not None and scaling.kind == "linear":
            fd = [x / scaling.factor for x in fd]
        elif scaling is not None and scaling.kind == "yarn":
            # pair d ln(L / (2 pi t)) / (2 ln base) makes t turns over length L
            lo, hi = (d * math.log(scaling.original / (2.0 * math.pi * t)) / (2.0 * math.log(base))
                      for t in (scaling.beta_fast, scaling.beta_slow))
            lo, hi = math.floor(lo), math.ceil(hi)
            if hi < 0 or lo > d - 1:  # every pair beyond both borders, the slow or the fast one
                r = [1.0 if hi < 0 else 0.0] * (d // 2)
            else:
                lo, hi = max(lo, 0), min(hi, d - 1)
                width = (hi - lo) or 0.001
                r = [min(max((i - lo) / width, 0.0), 1.0) for i in range(d // 2)]
            fd = [x * y / scaling.factor + x * (1.0 - y) for x, y in zip(fd, r)]
        f += fd
    return RotaryFrequencies(torch.tensor(f, dtype=torch.float64, device=device),
                             tuple(d // 2 for d in dims), float(factor))


def rotary_table(positions, frequencies, out=None, stream=None):
    """(cos, sin) of ``positions`` (int32 or int64, [...] for one axis, [...,
    axes] for several) times the frequencies: fp32 [..., pairs] each.  Angles
    are taken in 64 bits; from |position * frequency| = 2^51 on, where they
    are too coarse, the entries are NaN."""
    freqs, pairs, factor = frequencies
    dev = _dev(positions)
    _on(stream, dev)
    lead = tuple(positions.shape)
    if len(pairs) > 1:
        if not lead or lead[-1] != len(pairs):
            raise ValueError(f"t2t: positions must end in {len(pairs)} axes, got {lead}")
        lead = lead[:-1]
    bits = {_i32: 32, torch.int64: 64}.get(positions.dtype)
    if bits is None or not positions.is_contiguous():
        _check(positions, positions.shape, (_i32, torch.int64), "positions", dev)
    shape = (*lead, sum(pairs))
    if not _is(freqs, shape[-1:], torch.float64, dev):
        _check(freqs, shape[-1:], torch.float64, "frequencies", dev)
    if out is None:
        cos, sin = _empty(stream, shape, _f32, dev), _empty(stream, shape, _f32, dev)
    else:
        cos, sin = out
        _check(cos, shape, _f32, "cos", dev)
        _check(sin, shape, _f32, "sin", dev)
        _apart((cos, sin), ("cos", "sin"), (None, None, positions, freqs))
    _launch("t2t_rotary_table", dev, stream, (positions, freqs, cos, sin), positions.data_ptr(),
            bits, math.prod(lead), len(pairs), (ctypes.c_int * len(pairs))(*pairs), freqs.data_ptr(), factor, cos.data_ptr(), sin.data_ptr())
    return cos, sin


_ROPE_LAYOUTS = {"interleaved": 0, "half": 1}
_ROPE_NORMS = {None: 0, "token": 1, "head": 2}


def _rotary_arg(x, out, weight, norm, name, dev, stream, B, N, D, dtype):
    """The argument struct of one tensor, checked (out None: made by the caller)."""
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"t2t: {name} must be a tensor")
    shape, xs = x.shape, x.stride()
    nd = len(shape)
    if (nd not in (3, 4) or x.dtype != dtype or x.device != dev or (shape[0] if nd == 4 else 1) != B
            or shape[-3] != N or shape[-1] != D or not 1 <= shape[-2] <= 65536 or (D > 1 and xs[-1] != 1)):
        raise ValueError(f"t2t: {name} must be a {dtype} [{B}, {N}, heads, {D}] tensor on {dev} with "
                         f"contiguous channels")
    fresh = out is None
    if fresh:
        out = x.new_empty(shape) if stream is None else _empty(stream, shape, dtype, dev)
    os = out.stride() if isinstance(out, torch.Tensor) else ()
    if not fresh and out is not x and (len(os) != nd or out.shape != shape or out.dtype != dtype
                                       or out.device != dev):
        raise ValueError(f"t2t: the output of {name} must be a {dtype} {tuple(shape)} tensor on {dev}")
    if not fresh and ((D > 1 and os[-1] != 1) or not _scattered(out)):
        raise ValueError(f"t2t: the output of {name} must have contiguous channels and no element twice")
    H = x.shape[-2]
    if norm is not None:
        wshape = (H * D,) if norm == "token" else (D,)
        if not _is(weight, wshape, dtype, dev):
            _check(weight, wshape, dtype, f"{name}_weight", dev)
    elif weight is not None:
        raise ValueError(f"t2t: {name}_weight without a norm")
    return out, _lib.ROTARY_TENSOR.pack(x.data_ptr(), xs[0] if nd == 4 else 0, xs[-3], xs[-2], out.data_ptr(),
                                        os[0] if nd == 4 else 0, os[-3], os[-2],
                                        0 if weight is None else weight.data_ptr(), H)


def rotary(q, k, cos, sin, *, layout="interleaved", inverse=False, norm=None, q_weight=None,
           k_weight=None, eps=1e-6, out=None, stream=None):
    """Rotated q [B, N, Hq, D] and k [B, N, Hk, D] (or [N, H, D]; fp16 or bf16;
    any strides with contiguous channels; k may be None), one launch.

    cos, sin fp32 [N, R / 2] or [B, N, R / 2]: the first R <= D channels of every
    head are turned, pairs (2i, 2i + 1) with ``layout`` "interleaved", (i, i +
    R / 2) with "half"; the others pass.  ``inverse`` turns back (the rotation's
    transpose, so also its gradient).  ``norm``: an RMS norm before the turn,
    x * rsqrt(mean(x^2) + eps) * weight, over all heads of a token ("token",
    weight [H * D]) or each head ("head", weight [D]).  fp32 inside, rounded
    once.  ``out``: (out_q, out_k); an output may be its input, and otherwise
    shares no memory with any other argument.  Returns (out_q, out_k)."""
    dev = _dev(q)
    _on(stream, dev)
    if q.dim() not in (3, 4) or q.dtype not in _HALF:
        raise ValueError("t2t: q must be an fp16 or bf16 [B, N, H, D] or [N, H, D] tensor")
    B, (N, _, D) = q.shape[0] if q.dim() == 4 else 1, q.shape[-3:]
    if layout not in _ROPE_LAYOUTS or norm not in _ROPE_NORMS:
        raise ValueError(f"t2t: layout {layout!r} (interleaved or half), norm {norm!r} (None, token or head)")
    if inverse and norm is not None:
        raise ValueError("t2t: the inverse rotation takes no norm")
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError(f"t2t: eps must be at least 0, got {eps}")
    R = 2 * cos.shape[-1] if isinstance(cos, torch.Tensor) and cos.dim() else 0
    if not (1 <= D <= 256 and 2 <= R <= D):
        raise ValueError(f"t2t: {R} of {D} channels rotated (2 <= R <= D <= 256)")
    batched = cos.dim() == 3
    shape = (B, N, R // 2) if batched else (N, R // 2)
    for t, name in ((cos, "cos"), (sin, "sin")):
        if not _is(t, shape, _f32, dev):
            _check(t, shape, _f32, name, dev)
    if B * N >= 2 ** 31:
        raise ValueError(f"t2t: {B} x {N} tokens")
    oq, ok = out if out is not None else (None, None)
    oq, tq = _rotary_arg(q, oq, q_weight, norm, "q", dev, stream, B, N, D, q.dtype)
    tk = None
    if k is not None:
        ok, tk = _rotary_arg(k, ok, k_weight, norm, "k", dev, stream, B, N, D, q.dtype)
    if out is not None:
        _apart((oq,) if k is None else (oq, ok), ("the output of q", "the output of k"),
               (q, k, cos, sin, q_weight, k_weight))
    _launch("t2t_rotary", dev, stream, (q, k, cos, sin, q_weight, k_weight, oq, ok), tq, tk,
            dtype_code(q.dtype), cos.data_ptr(), sin.data_ptr(), batched, B, N, D, R,
            _ROPE_LAYOUTS[layout], bool(inverse), _ROPE_NORMS[norm], eps)
    return oq, ok if k is not None else None


def _mx_bytes(rows, cols):
    """Bytes of the codes and of the scales (t2t_mxfp4_code_bytes, _scale_bytes)."""
    scales = -(-rows // 32) * (-(-cols // 256) * 256)
    return scales * 16, scales


class MxFp4:
    """A matrix [rows, cols] in MXFP4 (``mxfp4_quantize``): E2M1 codes in blocks
    of 32 columns with a power-of-two scale each, in the order of the matrix
    operands (include/t2t_hip.h).  ``codes`` and ``scales`` are the uint8
    buffers on the GPU; they are checked here, once."""

    # (addresses and device are the buffers' at each call: a copied, pickled or loaded matrix has others)
    __slots__ = ("_codes", "_scales", "_rows", "_cols")

    def __init__(self, codes, scales, rows, cols):
        rows, cols = int(rows), int(cols)
        if not (0 <= rows <= 2 ** 30 and 32 <= cols <= 2 ** 27 and cols % 32 == 0):
            raise ValueError(f"t2t: an MXFP4 matrix has columns in multiples of 32, got {rows} x {cols}")
        dev = _dev(codes)
        for t, n, name in zip((codes, scales), _mx_bytes(rows, cols), ("codes", "scales")):
            _check(t, (n,), torch.uint8, name, dev)
            if n and t.data_ptr() % 16:
                raise ValueError(f"t2t: {name} must be 16-byte aligned")
        if _near(*_span(codes), ((scales.data_ptr(), scales.nbytes),)):
            raise ValueError("t2t: scales shares memory with codes")
        self._set(codes, scales, rows, cols)

    def _set(self, codes, scales, rows, cols):
        self._codes, self._scales, self._rows, self._cols = codes, scales, rows, cols
        return self

    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    rows = property(lambda self: self._rows)
    cols = property(lambda self: self._cols)
    shape = property(lambda self: (self._rows, self._cols))
    device = property(lambda self: self._codes.device)

    def __repr__(self):
        return f"MxFp4({self._rows} x {self._cols}, {self.device})"


def _mx_rows(t, name, dev, align):
    """A [..., K] tensor of 16-bit values as rows: (rows, K, row stride)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _HALF or t.device != dev or t.dim() < 1:
        raise ValueError(f"t2t: {name} must be an fp16 or bf16 tensor on {dev}")
    cols = t.shape[-1]
    if t.is_contiguous():
        rows, stride = (t.numel() // cols if cols else 0), cols
    else:
        try:
            v = t.view(math.prod(t.shape[:-1]), cols)
        except RuntimeError:
            raise ValueError(f"t2t: the rows of {name} {tuple(t.shape)} must have one stride, got "
                             f"{tuple(t.stride())}") from None
        rows = v.shape[0]
        stride = v.stride(0) if rows > 1 else cols
        if cols > 1 and v.stride(1) != 1 or stride < cols:
            raise ValueError(f"t2t: {name} must have contiguous rows that do not overlap, got strides "
                             f"{tuple(t.stride())}")
    if t.data_ptr() % align or rows > 1 and stride * 2 % align:
        raise ValueError(f"t2t: the rows of {name} must be {align}-byte aligned, got strides "
                         f"{tuple(t.stride())}")
    return rows, cols, stride


def _mx_dtype(dtype):
    if dtype not in _HALF:
        raise ValueError(f"t2t: the output's type must be torch.float16 or torch.bfloat16, got {dtype}")
    return dtype_code(dtype)


def mxfp4_quantize(x, out=None, stream=None):
    """x [..., K] (fp16 or bf16, contiguous 16-byte aligned rows, K a multiple of
    32) in MXFP4, rows flattened.  A block's scale is 2^(floor(log2 max|x|) - 2)
    (at least 2^-126); values are rounded to nearest, ties to even, and held to
    6 scales; a block with an inf or NaN stands for NaN."""
    dev = _dev(x)
    _on(stream, dev)
    M, K, stride = _mx_rows(x, "x", dev, 16)
    given = out is not None
    if not given:
        if K < 32 or K % 32 or K > 2 ** 27 or M > 2 ** 30:
            raise ValueError(f"t2t: x must have columns in multiples of 32, got {M} x {K}")
        nc, ns = _mx_bytes(M, K)
        out = MxFp4.__new__(MxFp4)._set(_empty(stream, (nc,), torch.uint8, dev),
                                        _empty(stream, (ns,), torch.uint8, dev), M, K)
    elif not isinstance(out, MxFp4) or out.shape != (M, K) or _dev(out._codes) != dev:
        raise ValueError(f"t2t: out must be an MxFp4 matrix {M} x {K} on {dev}, got {out!r}")
    px, codes, scales = x.data_ptr(), out._codes, out._scales
    pc, ps = codes.data_ptr(), scales.data_ptr()
    if given and _near(px, px + 2 * ((M - 1) * stride + K), ((pc, codes.nbytes), (ps, scales.nbytes))):
        _apart((codes, scales), ("out.codes", "out.scales"), (None, None, x))
    _launch("t2t_mxfp4_quantize", dev, stream, (x, codes, scales), px, dtype_code(x.dtype), stride, pc, ps, M, K)
    return out


def mxfp4_dequantize(t, dtype=torch.bfloat16, out=None, stream=None):
    """The values that an MxFp4 matrix stands for, [rows, cols]: exact in the
    type that was quantised, and in bf16 always."""
    if not isinstance(t, MxFp4):
        raise ValueError("t2t: expected an MxFp4 matrix")
    codes, scales = t._codes, t._scales
    dev = codes.device if codes.is_cuda else _dev(codes)
    _on(stream, dev)
    code = _mx_dtype(dtype)
    if out is None:
        out = _empty(stream, t.shape, dtype, dev)
        stride = t._cols
    else:
        M, K, stride = _mx_rows(out, "out", dev, 16)
        if (M, K) != t.shape or out.dtype != dtype:
            raise ValueError(f"t2t: out must be {dtype} {t.shape}, got {out.dtype} {tuple(out.shape)}")
        _apart((out,), ("out",), (None, codes, scales))
    _launch("t2t_mxfp4_dequantize", dev, stream, (codes, scales, out), codes.data_ptr(), scales.data_ptr(),
            out.data_ptr(), code, stride, *t.shape)
    return out


_ACTIVATIONS = {None: 0, "gelu_tanh": 1}


def mxfp4_linear_ws_bytes(M, N, K):
    """Workspace of mxfp4_linear for a 16-bit x of M rows (0 where the product
    quantises them itself)."""
    return size_query("t2t_mxfp4_linear_ws_bytes", M, N, K)


def mxfp4_linear(x, weight, bias=None, *, activation=None, dtype=None, out=None, ws=None, stream=None):
    """act(x W^T + bias) with both operands in MXFP4: x [..., K] fp16 or bf16
    (quantised as by mxfp4_quantize; contiguous 16-byte aligned rows), or an
    MxFp4 matrix that several layers share; weight MxFp4 [N, K]; bias [N] in the
    output's type.  fp32 sums, one rounding to x's type (``dtype``, default
    bf16, for an MxFp4 x) -> [..., N].  ``activation``: None or "gelu_tanh".
    ``out``: contiguous rows; it and ``ws`` share no memory with another argument."""
    if not isinstance(weight, MxFp4):
        raise ValueError("t2t: weight must be an MxFp4 matrix (mxfp4_quantize)")
    wc, wsc = weight._codes, weight._scales
    dev = wc.device if wc.is_cuda else _dev(wc)
    _on(stream, dev)
    N = weight._rows
    shared = isinstance(x, MxFp4)
    if shared:
        xs = x._codes, x._scales
        if xs[0].device != dev:
            raise ValueError(f"t2t: x must be on {dev}")
        M, K = x._rows, x._cols
        shape = (M, N)
        dt = torch.bfloat16 if dtype is None else dtype
    else:
        M, K, stride = _mx_rows(x, "x", dev, 16)
        shape, dt = (*x.shape[:-1], N), x.dtype
        if dtype not in (None, dt):
            raise ValueError(f"t2t: the output of a {dt} input is {dt}, not {dtype}")
    code = _mx_dtype(dt) if shared else dtype_code(dt)
    if K != weight._cols or N < 1:
        raise ValueError(f"t2t: x has {K} columns, weight {N} x {weight._cols}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"t2t: activation {activation!r} (None or gelu_tanh)")
    if bias is not None and not _is(bias, (N,), dt, dev):
        _check(bias, (N,), dt, "bias", dev)
    args = wc.data_ptr(), wsc.data_ptr(), None if bias is None else bias.data_ptr()
    spans = None  # of the inputs, where the caller brings an output or a workspace
    if out is not None or ws is not None:
        spans = [(args[0], wc.nbytes), (args[1], wsc.nbytes)] + [(args[2], 2 * N)] * (bias is not None)
        spans += ([(t.data_ptr(), t.nbytes) for t in xs] if shared else
                  [(x.data_ptr(), 2 * ((M - 1) * stride + K))])
    if out is None:
        out = _empty(stream, shape, dt, dev) if stream is not None or shared else x.new_empty(shape)
        ostride, po = N, out.data_ptr()
    else:
        ostride = _mx_rows(out, "out", dev, 2)[2]
        if tuple(out.shape) != shape or out.dtype != dt:
            raise ValueError(f"t2t: out must be {dt} {shape}, got {out.dtype} {tuple(out.shape)}")
        po = out.data_ptr()
        if _near(po, po + 2 * ((M - 1) * ostride + N), spans):
            _apart((out,), ("out",), (None, *(xs if shared else (x,)), wc, wsc, bias))
    args = *args, _ACTIVATIONS[activation], po
    if shared:
        _launch("t2t_mxfp4_product", dev, stream, (*xs, wc, wsc, bias, out), xs[0].data_ptr(),
                xs[1].data_ptr(), *args, code, ostride, M, N, K)
    else:
        need = mxfp4_linear_ws_bytes(M, N, K)
        if ws is not None:
            ws = _ws_for(ws, need, dev, stream)
            at = ws.data_ptr()
            if need and _near(at, at + need, (*spans, (po, 2 * ((M - 1) * ostride + N)))):
                _apart((ws[:need],), ("ws",), (None, x, wc, wsc, bias, out))
        elif need:
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if stream is None else _ws(need, dev, stream)
        _launch("t2t_mxfp4_linear", dev, stream, (x, wc, wsc, bias, out, ws), x.data_ptr(),
                code, stride, *args, ostride, M, N, K, None if ws is None else ws.data_ptr(),
                0 if ws is None else ws.numel())
    return out


# ---------------------------------------------------------------------------
# 8-bit linear layers
# ---------------------------------------------------------------------------
_I8_MAX_COLS = 2 ** 17 - 1  # the sums stay in 32 bits


class Int8:
    """A matrix [rows, cols] in 8 bits: whole numbers -127 .. 127 and an fp32 scale
    for each row (``int8_quantize``; ``from_codes`` for those of a checkpoint).
    ``codes`` (int8) and ``scales`` are the buffers on the GPU, the codes in the
    order of the products' tiles (include/t2t_hip.h); they are checked here, once."""

    # (addresses and device are the buffers' at each call: a copied, pickled or loaded matrix has others)
    __slots__ = ("_codes", "_scales", "_rows", "_cols")

    def __init__(self, codes, scales, rows, cols):
        rows, cols = int(rows), int(cols)
        if not (0 <= rows <= 2 ** 30 and 1 <= cols <= _I8_MAX_COLS):
            raise ValueError(f"t2t: an 8-bit matrix has 1 to 2^17 - 1 columns, got {rows} x {cols}")
        dev = _dev(codes)
        _check(codes, (_i8_bytes(rows, cols),), torch.int8, "codes", dev)
        _check(scales, (rows,), _f32, "scales", dev)
        if rows and codes.data_ptr() % 16:
            raise ValueError("t2t: codes must be 16-byte aligned")
        if _near(*_span(codes), ((scales.data_ptr(), scales.nbytes),)):
            raise ValueError("t2t: scales shares memory with codes")
        self._set(codes, scales, rows, cols)

    def _set(self, codes, scales, rows, cols):
        self._codes, self._scales, self._rows, self._cols = codes, scales, rows, cols
        return self

    @classmethod
    def from_codes(cls, codes, scales):
        """From whole numbers int8 [rows, cols] in rows and their scales fp32 [rows],
        which are copied."""
        if not isinstance(codes, torch.Tensor) or codes.dtype != torch.int8 or codes.dim() != 2:
            raise ValueError("t2t: codes must be an int8 [rows, cols] tensor")
        if not isinstance(scales, torch.Tensor):
            raise ValueError("t2t: scales must be an fp32 [rows] tensor")
        rows, cols = codes.shape
        if not 1 <= cols <= _I8_MAX_COLS:
            raise ValueError(f"t2t: an 8-bit matrix has 1 to 2^17 - 1 columns, got {rows} x {cols}")
        wide = codes.new_zeros(-(-rows // 16) * 16, -(-cols // 128) * 128)
        wide[:rows, :cols] = codes
        blocks = wide.view(-1, 4, 4, wide.shape[1] // 64, 4, 16)     # row r as (r / 4, r % 4)
        blocks = torch.stack([blocks[:, i][..., [c ^ i for c in range(4)], :] for i in range(4)], 1)
        return cls(blocks.permute(0, 3, 1, 2, 4, 5).contiguous().view(-1), scales.clone(), rows, cols)

    def to_codes(self):
        """The whole numbers in rows, int8 [rows, cols]."""
        blocks = self._codes.view(-(-self._rows // 16), -(-self._cols // 128) * 2, 4, 4, 4, 16)
        blocks = torch.stack([blocks[:, :, i][..., [c ^ i for c in range(4)], :] for i in range(4)], 2)
        wide = blocks.permute(0, 2, 3, 1, 4, 5).reshape(-(-self._rows // 16) * 16, -(-self._cols // 128) * 128)
        return wide[:self._rows, :self._cols].contiguous()

    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    rows = property(lambda self: self._rows)
    cols = property(lambda self: self._cols)
    shape = property(lambda self: (self._rows, self._cols))
    device = property(lambda self: self._codes.device)

    def __repr__(self):
        return f"Int8({self._rows} x {self._cols}, {self.device})"


def _i8_bytes(rows, cols):
    """Bytes of the codes (t2t_int8_code_bytes)."""
    return -(-rows // 16) * 16 * (-(-cols // 128) * 128)


def _x_span(x, rows, cols, stride):
    return x.data_ptr(), 2 * ((rows - 1) * stride + cols)


def int8_quantize(x, out=None, stream=None):
    """x [..., K] (fp16 or bf16, contiguous rows, K < 2^17) in 8 bits, rows
    flattened.  A row's scale is max|x| / 127 in fp32 (at least 2^-120); codes are
    the nearest whole multiples, ties to even; a row with an inf or NaN stands for
    NaN."""
    dev = _dev(x)
    _on(stream, dev)
    M, K, stride = _mx_rows(x, "x", dev, 2)
    if not (1 <= K <= _I8_MAX_COLS and M <= 2 ** 30):
        raise ValueError(f"t2t: x must have 1 to 2^17 - 1 columns, got {M} x {K}")
    given = out is not None
    if not given:
        out = Int8.__new__(Int8)._set(_empty(stream, (_i8_bytes(M, K),), torch.int8, dev),
                                      _empty(stream, (M,), _f32, dev), M, K)
    elif not isinstance(out, Int8) or out.shape != (M, K) or _dev(out._codes) != dev:
        raise ValueError(f"t2t: out must be an Int8 matrix {M} x {K} on {dev}, got {out!r}")
    codes, scales = out._codes, out._scales
    px, pc, ps = x.data_ptr(), codes.data_ptr(), scales.data_ptr()
    if given and _near(px, px + 2 * ((M - 1) * stride + K), ((pc, codes.nbytes), (ps, scales.nbytes))):
        _apart((codes, scales), ("out.codes", "out.scales"), (None, None, x))
    _launch("t2t_int8_quantize", dev, stream, (x, codes, scales), px, dtype_code(x.dtype), stride, pc, ps, M, K)
    return out


def int8_dequantize(t, dtype=torch.bfloat16, out=None, stream=None):
    """The values that an Int8 matrix stands for, [rows, cols] in fp16 or bf16,
    rounded once."""
    if not isinstance(t, Int8):
        raise ValueError("t2t: expected an Int8 matrix")
    codes, scales = t._codes, t._scales
    dev = codes.device if codes.is_cuda else _dev(codes)
    _on(stream, dev)
    code = _mx_dtype(dtype)
    if out is None:
        out = _empty(stream, t.shape, dtype, dev)
        stride = t._cols
    else:
        M, K, stride = _mx_rows(out, "out", dev, 2)
        if (M, K) != t.shape or out.dtype != dtype:
            raise ValueError(f"t2t: out must be {dtype} {t.shape}, got {out.dtype} {tuple(out.shape)}")
        _apart((out,), ("out",), (None, codes, scales))
    _launch("t2t_int8_dequantize", dev, stream, (codes, scales, out), codes.data_ptr(), scales.data_ptr(),
            out.data_ptr(), code, stride, *t.shape)
    return out


def int8_linear_ws_bytes(M, N, K):
    """Workspace of int8_linear for a 16-bit x of M rows (0 where the product
    quantises them itself)."""
    return _sizes_of("t2t_int8_linear_ws_bytes", M, N, K)


def int8_linear(x, weight, bias=None, *, activation=None, dtype=None, out=None, ws=None, stream=None):
    """act(x W^T + bias) with both operands in 8 bits, a scale for each token and
    channel: x [..., K] fp16 or bf16 (quantised as by int8_quantize; contiguous
    rows), or an Int8 matrix that several layers share; weight Int8 [N, K]; bias
    [N] in the output's type.  Integer sums (exact), scales, bias and activation in
    fp32, one rounding to x's type (``dtype``, default bf16, for an Int8 x) ->
    [..., N].  ``activation``: None or "gelu_tanh".  ``out``: contiguous rows; it
    and ``ws`` share no memory with another argument."""
    if not isinstance(weight, Int8):
        raise ValueError("t2t: weight must be an Int8 matrix (int8_quantize)")
    wc, wsc = weight._codes, weight._scales
    dev = wc.device if wc.is_cuda else _dev(wc)
    _on(stream, dev)
    N = weight._rows
    shared = isinstance(x, Int8)
    if shared:
        xs = x._codes, x._scales
        if xs[0].device != dev:
            raise ValueError(f"t2t: x must be on {dev}")
        M, K = x._rows, x._cols
        shape = (M, N)
        dt = torch.bfloat16 if dtype is None else dtype
        code = _mx_dtype(dt)
    else:
        M, K, stride = _mx_rows(x, "x", dev, 2)
        shape, dt = (*x.shape[:-1], N), x.dtype
        if dtype not in (None, dt):
            raise ValueError(f"t2t: the output of a {dt} input is {dt}, not {dtype}")
        code = dtype_code(dt)
    if K != weight._cols or N < 1:
        raise ValueError(f"t2t: x has {K} columns, weight {N} x {weight._cols}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"t2t: activation {activation!r} (None or gelu_tanh)")
    if bias is not None and not _is(bias, (N,), dt, dev):
        _check(bias, (N,), dt, "bias", dev)
    args = wc.data_ptr(), wsc.data_ptr(), None if bias is None else bias.data_ptr()
    spans = None  # of the inputs, where the caller brings an output or a workspace
    if out is not None or ws is not None:
        spans = [(args[0], wc.nbytes), (args[1], wsc.nbytes)] + [(args[2], 2 * N)] * (bias is not None)
        spans += [(t.data_ptr(), t.nbytes) for t in xs] if shared else [_x_span(x, M, K, stride)]
    if out is None:
        out = _empty(stream, shape, dt, dev) if stream is not None or shared else x.new_empty(shape)
        ostride, po = N, out.data_ptr()
    else:
        ostride = _mx_rows(out, "out", dev, 2)[2]
        if tuple(out.shape) != shape or out.dtype != dt:
            raise ValueError(f"t2t: out must be {dt} {shape}, got {out.dtype} {tuple(out.shape)}")
        po = out.data_ptr()
        if _near(po, po + 2 * ((M - 1) * ostride + N), spans):
            _apart((out,), ("out",), (None, *(xs if shared else (x,)), wc, wsc, bias))
    args = *args, _ACTIVATIONS[activation], po
    if shared:
        _launch("t2t_int8_product", dev, stream, (*xs, wc, wsc, bias, out), xs[0].data_ptr(), xs[1].data_ptr(), *args,
                code, ostride, M, N, K)
    else:
        need = int8_linear_ws_bytes(M, N, K)
        if ws is not None:
            ws = _ws_for(ws, need, dev, stream)
            at = ws.data_ptr()
            if need and _near(at, at + need, (*spans, _x_span(out, M, N, ostride))):
                _apart((ws[:need],), ("ws",), (None, x, wc, wsc, bias, out))
        elif need:
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if stream is None else _ws(need, dev, stream)
        _launch("t2t_int8_linear", dev, stream, (x, wc, wsc, bias, out, ws), x.data_ptr(), code, stride, *args,
                ostride, M, N, K, None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel())
    return out


# ---------------------------------------------------------------------------
# paged cache of keys and values
# ---------------------------------------------------------------------------
class PagedCache:
    """Keys and values of tokens in pages: ``k`` and ``v`` fp16 or bf16 [pages,
    page_size, heads, D], D 64 or 128, of the same strides (multiples of 8;
    contiguous channels; both may be views of one tensor), 16-byte aligned.  Slot
    page * page_size + i is row i of a page.  They are checked here, once."""

    __slots__ = ("_k", "_v", "_strides", "_bytes")

    def __init__(self, k, v):
        dev = _dev(k)
        if (k.dtype not in _HALF or k.dim() != 4 or not isinstance(v, torch.Tensor) or v.shape != k.shape
                or v.dtype != k.dtype or v.device != dev):
            raise ValueError(f"t2t: k and v must be fp16 or bf16 [pages, page_size, heads, D] tensors of one shape "
                             f"on {dev}")
        pages, page, heads, D = k.shape
        if D not in (64, 128) or not (1 <= pages < 2 ** 31 and 1 <= page < 2 ** 31 and 1 <= heads <= 65536):
            raise ValueError(f"t2t: a cache of {tuple(k.shape)} (at least one page, row and head, D 64 or 128)")
        st = _cache_strides(k)
        if (st != _cache_strides(v) or k.stride(3) != 1 or v.stride(3) != 1 or any(s % 8 for s in st)
                or (k.data_ptr() | v.data_ptr()) % 16):
            raise ValueError(f"t2t: k and v must have the same strides, in multiples of 8, contiguous channels and "
                             f"16-byte alignment, got {tuple(k.stride())} and {tuple(v.stride())}")
        if (pages - 1) * st[0] + (page - 1) * st[1] >= 2 ** 35:
            raise ValueError("t2t: one head's keys must span less than 64 GiB")
        if not (_scattered(k) and _scattered(v)) or _near(*_span(k), ((_span(v)[0], _span(v)[1] - _span(v)[0]),)) \
                and (_same_view(k, v) or _meet(k, v)):
            raise ValueError("t2t: the cache holds an element twice")
        self._k, self._v, self._strides, self._bytes = k, v, st, _span(k)[1] - _span(k)[0]

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    shape = property(lambda self: tuple(self._k.shape))
    page_size = property(lambda self: self._k.shape[1])
    device = property(lambda self: self._k.device)
    dtype = property(lambda self: self._k.dtype)

    def __repr__(self):
        return f"PagedCache({self.shape}, {self.dtype}, {self.device})"


def _cache_strides(t):
    """Strides of pages, rows and heads (0 where there is one)."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape))


def _cache_of(cache):
    if not isinstance(cache, PagedCache):
        raise ValueError("t2t: cache must be a PagedCache")
    k = cache._k
    return k, cache._v, k.device if k.is_cuda else _dev(k)


_SLOT_BITS = {_i32: 32, torch.int64: 64}


def cache_append(q, k, v, cos, sin, cache, slots, *, layout="interleaved", norm=None, q_weight=None,
                 k_weight=None, eps=1e-6, out=None, stream=None):
    """New tokens' k, normed and rotated as by ``rotary``, and v into their slots of
    a PagedCache, and q (or None) normed and rotated, one launch.  Returns the
    rotated q (``out``, which may be q; else shares no memory with another
    argument).

    q [T, Hq, D], k and v [T, Hk, D] of the cache's type (any strides with
    contiguous channels); cos, sin fp32 [T, R / 2]; slots int32 or int64 [T]: a
    token whose slot lies outside the cache (-1) is stored nowhere; the others'
    must differ.  ``norm`` "token", "head" or None, weights, ``layout`` and eps as
    in ``rotary``."""
    ck, cv, dev = _cache_of(cache)
    _on(stream, dev)
    pages, page, H, D = ck.shape
    dt = ck.dtype
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError("t2t: k must be a [T, heads, D] tensor")
    T = k.shape[0]
    shape, ks = (T, H, D), k.stride()
    if (k.shape != shape or k.dtype != dt or k.device != dev or ks[2] != 1 or not isinstance(v, torch.Tensor)
            or v.shape != shape or v.dtype != dt or v.device != dev or v.stride(2) != 1):
        raise ValueError(f"t2t: k and v must be {dt} [{T}, {H}, {D}] tensors on {dev} with contiguous channels")
    vs = v.stride()
    if layout not in _ROPE_LAYOUTS or norm not in _ROPE_NORMS:
        raise ValueError(f"t2t: layout {layout!r} (interleaved or half), norm {norm!r} (None, token or head)")
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError(f"t2t: eps must be at least 0, got {eps}")
    P = cos.shape[-1] if isinstance(cos, torch.Tensor) and cos.dim() else 0
    if not 1 <= P <= D // 2:
        raise ValueError(f"t2t: {2 * P} of {D} channels rotated (2 <= R <= D)")
    for t, name in ((cos, "cos"), (sin, "sin")):
        if not _is(t, (T, P), _f32, dev):
            _check(t, (T, P), _f32, name, dev)
    if T >= 2 ** 31:
        raise ValueError(f"t2t: {T} tokens")
    bits = _SLOT_BITS.get(slots.dtype) if isinstance(slots, torch.Tensor) else None
    if bits is None or not _is(slots, (T,), slots.dtype, dev):
        _check(slots, (T,), (_i32, torch.int64), "slots", dev)
    if norm is not None:
        wshape = (H * D,) if norm == "token" else (D,)
        if not _is(k_weight, wshape, dt, dev):
            _check(k_weight, wshape, dt, "k_weight", dev)
    elif k_weight is not None:
        raise ValueError("t2t: k_weight without a norm")
    # the cache (and a caller's output) apart from everything that is read
    pk, pv, pck, pcv, pcos, psin, ps = (k.data_ptr(), v.data_ptr(), ck.data_ptr(), cv.data_ptr(), cos.data_ptr(),
                                        sin.data_ptr(), slots.data_ptr())
    kn, n = (T - 1) * ks[0] + (H - 1) * ks[1] + D, 4 * T * P
    at = [(pk, 2 * kn), (pv, 2 * ((T - 1) * vs[0] + (H - 1) * vs[1] + D)), (pcos, n), (psin, n), (ps, T * bits >> 3)]
    pw = None
    if k_weight is not None:
        pw = k_weight.data_ptr()
        at.append((pw, 2 * k_weight.shape[0]))
    cs = cache._strides
    pack = _lib.ROTARY_TENSOR.pack
    oq = tq = None
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError("t2t: q must be a [T, heads, D] tensor")
        oq, tq = _rotary_arg(q, out, q_weight, norm, "q", dev, stream, 1, T, D, dt)
        qs = q.stride()
        at.append((q.data_ptr(), 2 * ((T - 1) * qs[0] + (q.shape[1] - 1) * qs[1] + D)))
        if q_weight is not None:
            at.append((q_weight.data_ptr(), q_weight.nbytes))
    elif out is not None or q_weight is not None:
        raise ValueError("t2t: out and q_weight belong to q")
    ins = (q, k, v, cos, sin, q_weight, k_weight, slots)
    kend, vend = pck + cache._bytes, pcv + cache._bytes
    for p, n in at if out is None and T else ():
        if p < kend and pck < p + n or p < vend and pcv < p + n:
            _apart((ck, cv), ("the cache", "the cache"), (None, None) + ins)
    if out is not None:
        _apart((oq, ck, cv), ("the output of q", "the cache", "the cache"), ins[:1] + (None, None) + ins[1:])
    _launch("t2t_cache_append", dev, stream, (*ins, ck, cv, oq), tq, pack(pk, 0, ks[0], ks[1], pck, *cs, pw or 0, H),
            pack(pv, 0, vs[0], vs[1], pcv, *cs, 0, H), dtype_code(dt), pcos, psin, ps, bits, pages, page, T, D, 2 * P,
            _ROPE_LAYOUTS[layout], _ROPE_NORMS[norm], eps)
    return oq


def cache_attention_ws_bytes(B, T, Hq, cache, width, ragged=False, causal=False, masked=False):
    """Workspace of cache_attention for T rows in all of B sequences (``ragged``: with
    offsets; ``masked``: with a mask) whose page tables are ``width`` pages wide."""
    k = cache._k
    return _sizes_of("t2t_cache_attention_ws_bytes", bool(ragged), 1 if causal else 2 if masked else 0, B, T, Hq,
                     k.shape[2], k.shape[3], width * k.shape[1])


def cache_attention(q, cache, page_table, lengths, *, offsets=None, mask=None, causal=False, scale=None,
                    return_lse=False, out=None, ws=None, stream=None):
    """Attention of new tokens over the cached keys and values of their sequences,
    the new tokens' own among them (``cache_append`` first).

    q [B, N, Hq, D]: N new tokens a sequence, or with ``offsets`` (int32 [B + 1]) [T,
    Hq, D]: rows offsets[b] .. offsets[b + 1] - 1 are sequence b's (rows behind the
    last sequence's stay as they are in ``out``, undefined in a fresh one).  page_table
    int32 [B, width], lengths int32 [B]: the keys of sequence b, positions 0 ..
    lengths[b] - 1, the last ones those of its new tokens, position j in page
    page_table[b, j // page_size].  Query head h reads key head h // (Hq / Hk).

    A token sees all older keys, and of the new ones all, or with ``causal`` those up
    to itself, or those of ``mask`` (bool [B, N, C] or [T, C]: its row's column j is
    the sequence's new token j; none from column C on), such as the tree that drafted
    tokens form or the frames of a chunk.  A token that sees nothing gets zeros.  What
    is not seen has no part whatever it holds; keys in pages outside the cache are not
    seen, and lengths are held to what the table has room for.

    ``scale`` (default D^-0.5) above 0, at most 2.3e38.  fp32 sums and softmax, its weights rounded to
    the type for the second product.  Returns out (of q's shape), or (out, lse) with
    the natural logarithms of the softmax's sums, fp32 [..., Hq].  ``out``: contiguous
    channels, 16-byte aligned rows; it and ``ws`` share no memory with another
    argument.  A ``ws`` (uint8, 16-byte aligned) is never replaced: with fewer bytes
    than cache_attention_ws_bytes a long sequence's keys go to fewer work-groups."""
    ck, cv, dev = _cache_of(cache)
    _on(stream, dev)
    pages, page, Hk, D = ck.shape
    dt = ck.dtype
    ragged = offsets is not None
    if (not isinstance(q, torch.Tensor) or q.dim() != (3 if ragged else 4) or q.dtype != dt or q.device != dev
            or q.shape[-1] != D):
        raise ValueError(f"t2t: q must be a {dt} [{'T' if ragged else 'B, N'}, heads, {D}] tensor on {dev}")
    Hq, N = q.shape[-2], q.shape[-3]
    if Hq < 1 or Hq % Hk or Hq > 65536:
        raise ValueError(f"t2t: {Hq} query heads over {Hk} of keys")
    if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1:
        raise ValueError("t2t: lengths must be an int32 [B] tensor")
    B = lengths.shape[0]
    if not _is(lengths, (B,), _i32, dev):
        _check(lengths, (B,), _i32, "lengths", dev)
    if ragged:
        if not _is(offsets, (B + 1,), _i32, dev):
            _check(offsets, (B + 1,), _i32, "offsets", dev)
        T, lead = N, (N,)
    else:
        if q.shape[0] != B:
            raise ValueError(f"t2t: q of {q.shape[0]} sequences, {B} lengths")
        T, lead = B * N, (B, N)
    if (not isinstance(page_table, torch.Tensor) or page_table.dim() != 2 or page_table.shape[0] != B
            or page_table.dtype != _i32 or page_table.device != dev
            or (page_table.shape[1] > 1 and page_table.stride(1) != 1)):
        raise ValueError(f"t2t: page_table must be an int32 [{B}, width] tensor on {dev} with contiguous rows")
    width = page_table.shape[1]
    if width * page >= 2 ** 31 - 64 or T * Hq >= 2 ** 31 or B > 2 ** 20:
        raise ValueError(f"t2t: {B} sequences of {width} pages of {page}, {T} tokens of {Hq} heads")
    if mask is not None:
        if causal:
            raise ValueError("t2t: a mask and causal")
        if (not isinstance(mask, torch.Tensor) or mask.dtype != torch.bool or mask.device != dev
                or mask.dim() != len(lead) + 1 or tuple(mask.shape[:-1]) != lead
                or (mask.shape[-1] > 1 and mask.stride(-1) != 1) or mask.shape[-1] >= 2 ** 31):
            raise ValueError(f"t2t: mask must be a bool {[*lead, 'columns']} tensor on {dev} with contiguous rows")
    if scale is None:
        scale = D ** -0.5
    elif not 2.0 ** -150 < scale <= 2.3e38:  # (in fp32 above 0, and finite times log2(e))
        raise ValueError(f"t2t: scale must be above 0 and within fp32, got {scale}")
    qs = _attn_strides(q, "q")
    if out is None:
        o = (_empty(stream, q.shape, dt, dev) if stream is not None
             else torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape))
    else:
        o = out
        if not isinstance(o, torch.Tensor) or o.shape != q.shape or o.dtype != dt or o.device != dev:
            raise ValueError(f"t2t: out must be a {dt} {tuple(q.shape)} tensor on {dev}")
        if not _scattered(o):
            raise ValueError("t2t: out holds an element twice")
    os = qs if out is None and q.is_contiguous() else _attn_strides(o, "out")
    lse = _empty(stream, (*lead, Hq), _f32, dev) if return_lse else None
    need = cache_attention_ws_bytes(B, T, Hq, cache, width, ragged, causal, mask is not None) if T and B else 0
    held = 0  # bytes that the launch may use of a caller's workspace
    if ws is not None:
        ws = _ws_for(ws, 0, dev, stream)
        held = min(need, ws.numel())
        if held and ws.data_ptr() % 16:
            raise ValueError("t2t: ws must be 16-byte aligned")
    elif need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if stream is None else _ws(need, dev, stream)
    ins = (q, ck, cv, page_table, lengths, offsets, mask)
    if out is not None:
        _apart((o,), ("out",), (None, *ins))
    if held:
        at = ws.data_ptr()
        if _near(at, at + held, [(p, e - p) for p, e in (_span(t) for t in (*ins, o) if t is not None)]):
            _apart((ws[:held],), ("ws",), (None, *ins, o))
    ms = mask.stride() if mask is not None else (0, 0, 0)
    args = _lib.CACHE_ATTENTION_ARGS.pack(
        _lib.CACHE_ATTENTION_ARGS.size, q.data_ptr(), ck.data_ptr(), cv.data_ptr(), o.data_ptr(),
        0 if lse is None else lse.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
        offsets.data_ptr() if ragged else 0, 0 if mask is None else mask.data_ptr() or q.data_ptr(), *qs, *os,
        *cache._strides, page_table.stride(0), 0 if ragged else ms[0], ms[-2], B, N, Hq, Hk, D, dtype_code(dt),
        pages, page, width, mask.shape[-1] if mask is not None else 0, bool(causal), scale)
    _launch("t2t_cache_attention", dev, stream, (*ins, o, lse, ws), args, None if ws is None else ws.data_ptr(),
            0 if ws is None else ws.numel())
    return (o, lse) if return_lse else o


def _attn_strides(t, name):
    """Strides of sequences, tokens and heads of [B, N, H, D] or [T, H, D]."""
    st = t.stride()
    if t.is_contiguous():
        st = st[:-1]
        bad = t.data_ptr() % 16
    else:
        st = tuple(s if n > 1 else 0 for s, n in zip(st, t.shape))[:-1]
        bad = (t.stride(-1) != 1 or any(s % 8 for s in st) or t.data_ptr() % 16) and t.numel()
    if bad:
        raise ValueError(f"t2t: {name} must have contiguous channels and 16-byte aligned rows, got strides "
                         f"{tuple(t.stride())}")
    return st if len(st) == 3 else (0, *st)
