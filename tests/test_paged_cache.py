"""Paged caches of keys and values: the append with its norm and rotation, and
attention over the cache, against 64-bit forms of their definitions, and what the
entry points refuse."""
import copy
import ctypes
import math
import random

import pytest
import torch

from token2tile_amd import ops

F64, I32 = torch.float64, torch.int32
HALF = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def _half_step(ref, dt):
    fi = torch.finfo(dt)
    return (ref.abs() * (fi.eps / 2)).clamp(min=fi.smallest_normal * fi.eps / 2)


def _cache(g, pages, page, H, D, dt, kind="own", fill=None):
    """A cache in storage of its own, as halves of one tensor, or with heads before rows."""
    if kind == "own":
        k, v = (_randn(g, pages, page, H, D).to(dt) for _ in range(2))
    elif kind == "pairs":
        both = _randn(g, pages, 2, page, H, D).to(dt)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (_randn(g, pages, H, page, D).to(dt).transpose(1, 2) for _ in range(2))
    if fill is not None:
        k.fill_(fill), v.fill_(fill)
    return ops.PagedCache(k, v)


# ---------------------------------------------------------------------------
# refusals before any launch
# ---------------------------------------------------------------------------
def test_entries_reject_bad_arguments():
    from token2tile_amd import _lib
    L = _lib.lib()
    p = ctypes.c_void_p(32)

    def app(q=True, k=True, v=True, dtype=1, bits=32, pages=4, page=16, T=4, D=128, R=128, layout=0, norm=0, heads=2,
            vheads=2, weight=None, x=16, slots=p, cos=p):
        t = _lib.RotaryTensor(x, 0, 0, 0, 16, 0, 0, 0, weight, heads)
        u = _lib.RotaryTensor(x, 0, 0, 0, 16, 0, 0, 0, None, vheads)
        r, s = ctypes.byref(t), ctypes.byref(u)
        return L.t2t_cache_append(r if q else None, r if k else None, s if v else None, dtype, cos, p, slots, bits,
                                  pages, page, T, D, R, layout, norm, 1e-6, None)
    for kw in (dict(k=False), dict(v=False), dict(dtype=2), dict(bits=16), dict(pages=0), dict(page=0), dict(T=-1),
               dict(T=1 << 31), dict(D=257), dict(R=130), dict(R=3), dict(R=0), dict(layout=2), dict(norm=3),
               dict(heads=0), dict(vheads=3), dict(norm=1), dict(x=None), dict(slots=None), dict(cos=None)):
        assert app(**kw) == 1, kw
    assert app(T=0, slots=None) == 0

    def attn(ws=None, nb=0, **kw):
        f = dict(struct_bytes=ctypes.sizeof(_lib.CacheAttentionArgs), q=32, k=32, v=32, out=32, lse=None, table=32,
                 lengths=32, offsets=None, mask=None, q_batch=512, q_row=256, q_head=128, out_batch=512, out_row=256,
                 out_head=128, kv_page=4096, kv_row=256, kv_head=128, table_row=4, mask_batch=0, mask_row=0, B=2, N=2,
                 HQ=2, HK=2, D=128, dtype=1, pages=8, page_size=16, width=4, mask_cols=0, causal=0, scale=0.1)
        f.update(kw)
        return L.t2t_cache_attention(ctypes.byref(_lib.CacheAttentionArgs(**f)), ws, nb, None)
    for kw in (dict(struct_bytes=8), dict(dtype=2), dict(D=96), dict(HK=0), dict(HQ=3), dict(HQ=0), dict(B=-1),
               dict(N=-1), dict(B=1 << 20, N=1 << 20), dict(B=1, N=1 << 30, HQ=4), dict(pages=0), dict(page_size=0),
               dict(width=-1), dict(width=1 << 30), dict(scale=0.0), dict(scale=math.inf), dict(scale=math.nan),
               dict(mask=32, causal=1), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(lengths=None),
               dict(table=None), dict(q=40), dict(out=36), dict(q_row=100), dict(kv_row=4), dict(kv_page=1 << 33),
               dict(kv_page=-256), dict(out_head=60)):
        assert attn(**kw) == 1, kw
    assert L.t2t_cache_attention(None, None, 0, None) == 1
    assert attn(B=0) == 0 and attn(N=0) == 0 and attn(N=0, offsets=32) == 0


def test_workspace_bytes():
    from token2tile_amd import _lib
    f = _lib.lib().t2t_cache_attention_ws_bytes
    assert f(0, 0, 1, 1, 40, 8, 128, 100) == 0               # one part
    assert f(0, 0, 1, 4680, 40, 40, 128, 32768) == 0         # enough rows
    one = f(0, 0, 1, 1, 40, 8, 128, 1 << 16)
    assert one >= 2 * 40 * 130 * 4 and one % (40 * 130 * 4) == 16  # parts, and their size
    assert f(0, 0, 0, 0, 40, 8, 128, 100) == 0 and f(1, 0, 4, 61, 32, 8, 64, 20000) > 0
    assert f(0, 1, 1, 8192, 8, 8, 128, 8192) > f(0, 0, 1, 8192, 8, 8, 128, 8192) == 0  # row blocks that differ


def test_parts_where_they_help():
    """Many sequences are counted by every work-group: no parts where those are many and the keys few."""
    from token2tile_amd import _lib
    f = _lib.lib().t2t_cache_attention_ws_bytes
    for ragged in (0, 1):
        for B, Hk, keys in ((64, 1, 1024), (128, 1, 1024), (256, 1, 1024), (400, 1, 4096), (128, 8, 4096), (1500, 1, 16384)):
            assert f(ragged, 0, B, B, 8, Hk, 128, keys) > 0, (B, Hk, keys)
        for B, Hk, keys in ((400, 1, 2048), (1024, 1, 4096), (2000, 1, 4096), (2000, 1, 16384), (400, 8, 4096), (400, 8, 16384)):
            assert f(ragged, 0, B, B, 8, Hk, 128, keys) == 0, (B, Hk, keys)


def test_cpu_tensors_are_refused():
    z = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="t2t"):
        ops.PagedCache(z, z.clone())
    with pytest.raises(ValueError, match="t2t"):
        ops.cache_attention(z, (z, z), torch.zeros(4, 1, dtype=I32), torch.zeros(4, dtype=I32))


@pytest.fixture
def launches(monkeypatch):
    """CPU tensors in the place of GPU ones; the launches, which are not made."""
    seen = []
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(ops, "_launch", lambda name, dev, stream, tensors, *a: seen.append((name, tensors, a)))
    return seen


def _z(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize("bad", ["type", "types", "shape", "width", "strides", "odd", "align", "channels", "same",
                                 "overlap", "twice", "empty"])
def test_caches_refused(launches, bad):
    buf = _z(1 << 16)
    make = {
        "type": lambda: (_z(4, 16, 2, 64, dtype=torch.float32),) * 2,
        "types": lambda: (_z(4, 16, 2, 64), _z(4, 16, 2, 64, dtype=torch.float16)),
        "shape": lambda: (_z(4, 16, 2, 64), _z(4, 16, 3, 64)),
        "width": lambda: (_z(4, 16, 2, 96), _z(4, 16, 2, 96)),
        "strides": lambda: (_z(4, 16, 2, 64), _z(4, 2, 16, 64).transpose(1, 2)),
        "odd": lambda: (_z(4, 16, 2, 68)[..., :64], _z(4, 16, 2, 68)[..., :64]),
        "align": lambda: (_z(8200)[4:8196].view(4, 16, 2, 64), _z(4, 16, 2, 64)),
        "channels": lambda: (_z(4, 16, 64, 2).transpose(2, 3), _z(4, 16, 64, 2).transpose(2, 3)),
        "same": lambda: (buf[:8192].view(4, 16, 2, 64),) * 2,
        "overlap": lambda: (buf[:8192].view(4, 16, 2, 64), buf[8184:8184 + 8192].view(4, 16, 2, 64)),
        "twice": lambda: (_z(1, 16, 2, 64).expand(4, 16, 2, 64), _z(1, 16, 2, 64).expand(4, 16, 2, 64)),
        "empty": lambda: (_z(0, 16, 2, 64), _z(0, 16, 2, 64))}[bad]
    with pytest.raises(ValueError, match="t2t"):
        ops.PagedCache(*make())


def _append_args(T=6, Hq=4, H=2, D=64, R=64):
    return dict(q=_z(T, Hq, D), k=_z(T, H, D), v=_z(T, H, D), cos=torch.zeros(T, R // 2), sin=torch.zeros(T, R // 2),
                cache=ops.PagedCache(_z(4, 16, H, D), _z(4, 16, H, D)), slots=torch.arange(T))


@pytest.mark.parametrize("bad", ["cache", "k", "k_type", "k_shape", "v_shape", "q_shape", "q_dim", "cos", "sin", "R",
                                 "slots", "slots_type", "layout", "norm", "weight", "no_weight", "eps", "out", "out_q",
                                 "in_cache", "v_in_cache", "q_in_cache", "out_in_cache", "out_in_k"])
def test_append_refused(launches, bad):
    a, kw = _append_args(), {}
    c = a["cache"]
    if bad == "cache": a["cache"] = (c.k, c.v)  # noqa: E701
    elif bad == "k": a["k"] = None  # noqa: E701
    elif bad == "k_type": a["k"] = a["k"].half()  # noqa: E701
    elif bad == "k_shape": a["k"] = _z(6, 3, 64)  # noqa: E701
    elif bad == "v_shape": a["v"] = _z(5, 2, 64)  # noqa: E701
    elif bad == "q_shape": a["q"] = _z(5, 4, 64)  # noqa: E701
    elif bad == "q_dim": a["q"] = _z(1, 6, 4, 64)  # noqa: E701
    elif bad == "cos": a["cos"] = torch.zeros(5, 32)  # noqa: E701
    elif bad == "sin": a["sin"] = torch.zeros(6, 16)  # noqa: E701
    elif bad == "R": a["cos"] = a["sin"] = torch.zeros(6, 33)  # noqa: E701
    elif bad == "slots": a["slots"] = torch.arange(5)  # noqa: E701
    elif bad == "slots_type": a["slots"] = torch.zeros(6)  # noqa: E701
    elif bad == "layout": kw["layout"] = "other"  # noqa: E701
    elif bad == "norm": kw["norm"] = "other"  # noqa: E701
    elif bad == "weight": kw["k_weight"] = _z(64)  # noqa: E701
    elif bad == "no_weight": kw["norm"] = "head"  # noqa: E701
    elif bad == "eps": kw["eps"] = -1.0  # noqa: E701
    elif bad == "out": a["q"], kw["out"] = None, _z(6, 4, 64)  # noqa: E701
    elif bad == "out_q": kw["out"] = _z(6, 4, 32)  # noqa: E701
    elif bad == "in_cache": a["k"] = c.k[0, :6]  # noqa: E701
    elif bad == "v_in_cache": a["v"] = c.v[1, 3:9]  # noqa: E701
    elif bad == "q_in_cache": a["q"] = c.k[0, :12].view(6, 4, 64)  # noqa: E701
    elif bad == "out_in_cache": kw["out"] = c.v[0, :12].view(6, 4, 64)  # noqa: E701
    elif bad == "out_in_k":
        buf = _z(1 << 12)
        a["k"], kw["out"] = buf[:768].view(6, 2, 64), buf[512:512 + 1536].view(6, 4, 64)
    with pytest.raises(ValueError, match="t2t"):
        ops.cache_append(**a, **kw)
    assert not launches
    if bad in ("in_cache", "out"):   # and in good order
        ops.cache_append(**_append_args())
        ops.cache_append(**{**_append_args(), "q": None})
        b = _append_args()
        assert ops.cache_append(**b, out=b["q"]) is b["q"] and len(launches) == 3


def _attend_args(B=3, N=4, Hq=4, H=2, D=64, page=16, width=5):
    return dict(q=_z(B, N, Hq, D), cache=ops.PagedCache(_z(16, page, H, D), _z(16, page, H, D)),
                page_table=torch.zeros(B, width, dtype=I32), lengths=torch.zeros(B, dtype=I32))


@pytest.mark.parametrize("bad", ["cache", "q_type", "q_dim", "q_ragged", "q_width", "heads", "lengths", "lengths_type",
                                 "batch", "table", "table_type", "table_rows", "offsets", "offsets_type", "mask_type",
                                 "mask_shape", "mask_rows", "both", "scale", "scale_nan", "align", "stride", "out",
                                 "out_twice", "out_q", "out_cache", "ws", "ws_q"])
def test_attention_refused(launches, bad):
    a, kw = _attend_args(), {}
    ragged = torch.tensor([0, 4, 8, 12], dtype=I32)
    if bad == "cache": a["cache"] = None  # noqa: E701
    elif bad == "q_type": a["q"] = a["q"].half()  # noqa: E701
    elif bad == "q_dim": a["q"] = _z(12, 4, 64)  # noqa: E701
    elif bad == "q_ragged": kw["offsets"] = ragged  # noqa: E701
    elif bad == "q_width": a["q"] = _z(3, 4, 4, 128)  # noqa: E701
    elif bad == "heads": a["q"] = _z(3, 4, 5, 64)  # noqa: E701
    elif bad == "lengths": a["lengths"] = torch.zeros(3, 1, dtype=I32)  # noqa: E701
    elif bad == "lengths_type": a["lengths"] = torch.zeros(3, dtype=torch.int64)  # noqa: E701
    elif bad == "batch": a["q"] = _z(2, 4, 4, 64)  # noqa: E701
    elif bad == "table": a["page_table"] = torch.zeros(2, 5, dtype=I32)  # noqa: E701
    elif bad == "table_type": a["page_table"] = torch.zeros(3, 5, dtype=torch.int64)  # noqa: E701
    elif bad == "table_rows": a["page_table"] = torch.zeros(5, 3, dtype=I32).t()  # noqa: E701
    elif bad == "offsets": a["q"], kw["offsets"] = _z(12, 4, 64), ragged[:3].clone()  # noqa: E701
    elif bad == "offsets_type": a["q"], kw["offsets"] = _z(12, 4, 64), ragged.long()  # noqa: E701
    elif bad == "mask_type": kw["mask"] = torch.zeros(3, 4, 4, dtype=torch.uint8)  # noqa: E701
    elif bad == "mask_shape": kw["mask"] = torch.zeros(3, 5, 4, dtype=torch.bool)  # noqa: E701
    elif bad == "mask_rows": kw["mask"] = torch.zeros(3, 4, 8, dtype=torch.bool)[..., ::2]  # noqa: E701
    elif bad == "both": kw["mask"], kw["causal"] = torch.zeros(3, 4, 4, dtype=torch.bool), True  # noqa: E701
    elif bad == "scale": kw["scale"] = 0.0  # noqa: E701
    elif bad == "scale_nan": kw["scale"] = math.nan  # noqa: E701
    elif bad == "align": a["q"] = _z(3 * 4 * 4 * 64 + 8)[4:-4].view(3, 4, 4, 64)  # noqa: E701
    elif bad == "stride": a["q"] = _z(3, 4, 4, 68)[..., :64]  # noqa: E701
    elif bad == "out": kw["out"] = _z(3, 4, 4, 32)  # noqa: E701
    elif bad == "out_twice": kw["out"] = _z(3, 4, 1, 64).expand(3, 4, 4, 64)  # noqa: E701
    elif bad == "out_q": kw["out"] = a["q"]  # noqa: E701
    elif bad == "out_cache": kw["out"] = a["cache"].k[:6].view(3, 4, 8, 2, 64)[:, :, :2].reshape(-1)[:0]  # noqa: E701
    elif bad == "ws": kw["ws"] = _z(1 << 16)  # noqa: E701
    elif bad == "ws_q":
        a = _attend_args(width=200)
        need = ops.cache_attention_ws_bytes(3, 12, 4, a["cache"], 200)
        assert need > 0
        buf = torch.zeros(need + 6144, dtype=torch.uint8)
        a["q"], kw["ws"] = buf[:6144].view(torch.bfloat16).view(3, 4, 4, 64), buf[6000:]
    with pytest.raises(ValueError, match="t2t"):
        ops.cache_attention(**a, **kw)
    assert not launches


def test_a_workspace_of_any_size_is_the_one_that_is_used(launches):
    """A caller's workspace is passed on with its own byte count, never replaced."""
    a = _attend_args(width=200)
    need = ops.cache_attention_ws_bytes(3, 12, 4, a["cache"], 200)
    buf = torch.zeros(need + 64, dtype=torch.uint8)
    for n in (0, 1, need // 2, need - 1, need, need + 64):
        ws = buf[:n]
        ops.cache_attention(**a, ws=ws)
        name, tensors, args = launches.pop()
        assert args[1:] == (ws.data_ptr(), n) and any(t is ws for t in tensors)
    with pytest.raises(ValueError, match="aligned"):
        ops.cache_attention(**a, ws=buf[4:])
    # a small one that shares memory with an input
    a["q"] = buf[:6144].view(torch.bfloat16).view(3, 4, 4, 64)
    with pytest.raises(ValueError, match="shares memory"):
        ops.cache_attention(**a, ws=buf[6128:6160])
    ops.cache_attention(**a, ws=buf[6144:6160])
    short = _attend_args(width=1)  # (no workspace asked for: nothing of it is used)
    assert ops.cache_attention_ws_bytes(3, 12, 4, short["cache"], 1) == 0
    ops.cache_attention(**short, ws=buf[4:])


@pytest.mark.parametrize("scale", [1e39, 1e-50, 2.5e38, -1e39, math.inf])
def test_scales_that_fp32_does_not_hold(launches, scale):
    """Not in 32 bits, or not times log2(e): refused before the launch, as every scale that is no number above 0."""
    with pytest.raises(ValueError, match="scale"):
        ops.cache_attention(**_attend_args(), scale=scale)
    assert not launches
    for good in (2.3e38, 1e-45, 1):
        ops.cache_attention(**_attend_args(), scale=good)
    assert len(launches) == 3


def test_the_entry_refuses_a_scale_without_room():
    from token2tile_amd import _lib
    a = _lib.CacheAttentionArgs(struct_bytes=ctypes.sizeof(_lib.CacheAttentionArgs), q=32, k=32, v=32, out=32, table=32,
                                lengths=32, q_batch=512, q_row=256, q_head=128, out_batch=512, out_row=256, out_head=128,
                                kv_page=4096, kv_row=256, kv_head=128, table_row=4, B=2, N=2, HQ=2, HK=2, D=128, dtype=1,
                                pages=8, page_size=16, width=4, scale=2.5e38)
    assert _lib.lib().t2t_cache_attention(ctypes.byref(a), None, 0, None) == 1


@pytest.mark.parametrize("kind", ["k", "v", "page_table", "lengths", "offsets", "mask"])
def test_an_output_apart_from_every_input(launches, kind):
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    at = buf[256:256 + 12 * 4 * 64 * 2].view(torch.bfloat16).view(12, 4, 64)
    a = _attend_args()
    a["q"] = _z(12, 4, 64)
    kw = dict(offsets=torch.zeros(4, dtype=I32), mask=torch.zeros(12, 4, dtype=torch.bool))
    half = buf[:4 * 16 * 2 * 64 * 2].view(torch.bfloat16).view(4, 16, 2, 64)
    if kind in ("k", "v"):
        pair = (half, _z(4, 16, 2, 64)) if kind == "k" else (_z(4, 16, 2, 64), half)
        a["cache"] = ops.PagedCache(*pair)
    elif kind == "page_table":
        a["page_table"] = buf[512:512 + 60].view(I32).view(3, 5)
    elif kind == "lengths":
        a["lengths"] = buf[512:524].view(I32)
    elif kind == "offsets":
        kw["offsets"] = buf[512:528].view(I32)
    else:
        kw["mask"] = buf[512:560].view(torch.bool).view(12, 4)
    with pytest.raises(ValueError, match="shares memory"):
        ops.cache_attention(**a, **kw, out=at)
    assert not launches


def test_every_tensor_of_a_call_is_recorded_on_its_stream(launches):
    a = _append_args()
    stream = type("S", (), {"device": a["k"].device})()
    w = _z(64)
    out = _z(6, 4, 64)
    ops.cache_append(**a, norm="head", q_weight=w, k_weight=w, out=out, stream=stream)
    (_, tensors, _), = launches
    c = a["cache"]
    for t in (a["q"], a["k"], a["v"], a["cos"], a["sin"], a["slots"], w, c.k, c.v, out):
        assert any(u is t for u in tensors)
    launches.clear()
    a = _attend_args(width=200)
    a["q"], ragged = _z(12, 4, 64), torch.zeros(4, dtype=I32)
    mask, out = torch.zeros(12, 4, dtype=torch.bool), _z(12, 4, 64)
    ws = torch.empty(ops.cache_attention_ws_bytes(3, 12, 4, a["cache"], 200, True), dtype=torch.uint8)
    ops.cache_attention(**a, offsets=ragged, mask=mask, out=out, ws=ws, stream=stream)
    (_, tensors, args), = launches
    assert ws.data_ptr() in args
    for t in (a["q"], a["cache"].k, a["cache"].v, a["page_table"], a["lengths"], ragged, mask, out, ws):
        assert any(u is t for u in tensors)


def test_a_copied_cache_is_read_at_its_own_address(launches):
    a = _append_args()
    c = copy.deepcopy(a["cache"])
    assert c.k.data_ptr() != a["cache"].k.data_ptr()
    ops.cache_append(**{**a, "cache": c})
    (_, _, args), = launches
    from token2tile_amd import _lib
    k, v = (_lib.RotaryTensor.from_buffer_copy(x) for x in args[1:3])
    assert k.out == c.k.data_ptr() and v.out == c.v.data_ptr()


def test_arguments_as_bytes_are_the_structs():
    from token2tile_amd import _lib
    for packer, struct in ((_lib.ROTARY_TENSOR, _lib.RotaryTensor),
                           (_lib.CACHE_ATTENTION_ARGS, _lib.CacheAttentionArgs)):
        names = [n for n, _ in struct._fields_]
        values = list(range(1, len(names) + 1))
        a = struct.from_buffer_copy(packer.pack(*values))
        assert packer.size == ctypes.sizeof(struct) and [getattr(a, n) for n in names] == values


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def _tables(g, T, R):
    a = 100 * torch.rand(T, R // 2, generator=g, device=g.device, dtype=F64)
    return a.cos().float(), a.sin().float()


def _turned(x, cos, sin, layout, norm, w, eps=1e-6):
    """(result, bound on the fp32 part) of the norm and rotation of x [T, H, D], in 64 bits."""
    x = x.double()
    if norm == "token":
        x = x / (x.square().mean((-2, -1), keepdim=True) + eps).sqrt() * w.double().view(x.shape[-2:])
    elif norm == "head":
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    R = 2 * cos.shape[-1]
    c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    y, mag = x.clone(), x.abs()
    lo, hi = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    mag[..., lo] = mag[..., hi] = a.abs() + b.abs()
    # the norm's sum by at most 128 additions of 2^-24 (half of that under the root), its root, quotient
    # and products by a few more, the turn by three: 2^-17 of |a| + |b| covers all
    return y, 2.0 ** -17 * mag


def _check_turned(got, x, cos, sin, layout, norm, w):
    ref, tol = _turned(x, cos, sin, layout, norm, w)
    tol = tol + _half_step(ref, x.dtype) * (1 + 2.0 ** -7)
    assert bool(((got.double() - ref).abs() <= tol).all())


APPENDS = [  # T, Hq, Hk, D, R, page
    (1, 40, 40, 128, 128, 64), (4, 12, 2, 128, 128, 16), (5, 1, 1, 64, 2, 1), (33, 5, 5, 64, 32, 7),
    (61, 33, 3, 128, 96, 48), (130, 65, 13, 128, 128, 256), (300, 12, 12, 128, 64, 64), (1100, 3, 3, 64, 64, 16),
    (1203, 32, 8, 128, 128, 48), (40, 130, 130, 128, 128, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("norm", [None, "token", "head"])
@pytest.mark.parametrize("T,Hq,Hk,D,R,page", APPENDS)
def test_append(dev, T, Hq, Hk, D, R, page, norm, layout, dt):
    g, dt = _gen(dev, T + Hq), HALF[dt]
    pages = -(-T // page) + 5
    cache = _cache(g, pages, page, Hk, D, dt, ["own", "pairs", "heads"][T % 3])
    q, k, v = (4 * _randn(g, T, H, D).to(dt) for H in (Hq, Hk, Hk))
    cos, sin = _tables(g, T, R)
    w = [None, None]
    if norm:
        w = [(1 + 0.3 * _randn(g, H * D if norm == "token" else D)).to(dt) for H in (Hq, Hk)]
    slots = torch.randperm(pages * page, generator=g, device=dev)[:T]
    slots[::7] = -1
    if T > 8:
        slots[8] = pages * page            # the first one past the cache
        slots[5] = 1 << 40
    ck, cv = cache.k.clone(), cache.v.clone()
    kw = dict(layout=layout, norm=norm, k_weight=w[1])
    oq = ops.cache_append(q, k, v, cos, sin, cache, slots, q_weight=w[0], **kw)
    _check_turned(oq, q, cos, sin, layout, norm, w[0])
    keep = (slots >= 0) & (slots < pages * page)
    page_of, row = slots[keep] // page, slots[keep] % page
    _check_turned(cache.k[page_of, row], k[keep], cos[keep], sin[keep], layout, norm, w[1])
    # the bits of the rotation alone, values as they are, and every other slot untouched
    rq, rk = ops.rotary(q, k, cos, sin, layout=layout, norm=norm, q_weight=w[0], k_weight=w[1])
    assert torch.equal(oq, rq)
    ck[page_of, row], cv[page_of, row] = rk[keep], v[keep]
    assert torch.equal(cache.k, ck) and torch.equal(cache.v, cv)
    # without q, 32-bit slots
    cache.k.zero_(), cache.v.zero_()
    small = slots.clamp(max=2 ** 31 - 1).to(I32)
    assert ops.cache_append(None, k, v, cos, sin, cache, small, **kw) is None
    assert torch.equal(cache.k[page_of, row], rk[keep]) and torch.equal(cache.v[page_of, row], v[keep])
    assert int((cache.v != 0).any(-1).any(-1).sum()) <= int(keep.sum())


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [None, "token", "head"])
@pytest.mark.parametrize("kind", ["fused", "head_major", "misaligned", "odd_stride", "expanded"])
def test_append_views(dev, kind, norm):
    """Strided inputs give the bits of contiguous ones; q in its own place."""
    g, dt = _gen(dev, 3), torch.bfloat16
    T, Hq, Hk, D, R, page = 37, 6, 2, 128, 96, 16
    cos, sin = _tables(g, T, R)
    w = {None: (None, None), "head": [_randn(g, D).to(dt)] * 2,
         "token": [_randn(g, H * D).to(dt) for H in (Hq, Hk)]}[norm]
    slots = torch.randperm(6 * page, generator=g, device=dev)[:T]
    if kind == "fused":
        buf = _randn(g, T, Hq + 2 * Hk, D).to(dt)
        q, k, v = buf[:, :Hq], buf[:, Hq:Hq + Hk], buf[:, Hq + Hk:]
    else:
        shape = {"head_major": lambda H: _randn(g, H, T, D).to(dt).transpose(0, 1),
                 "misaligned": lambda H: _randn(g, T * H * D + 3).to(dt)[3:].view(T, H, D),
                 "odd_stride": lambda H: _randn(g, T, H, D + 3).to(dt)[..., :D],
                 "expanded": lambda H: _randn(g, 1, H, D).to(dt).expand(T, H, D)}[kind]
        q, k, v = shape(Hq), shape(Hk), shape(Hk)
    call = lambda q, k, v, c, **kw: ops.cache_append(q, k, v, cos, sin, c, slots, layout="half", norm=norm,  # noqa: E731
                                                     q_weight=w[0], k_weight=w[1], **kw)
    c0, c1 = (_cache(g, 6, page, Hk, D, dt, fill=7.0) for _ in range(2))
    want = call(q.contiguous(), k.contiguous(), v.contiguous(), c0)
    kept = (k.clone(), v.clone())
    got = call(q, k, v, c1, out=None if kind == "expanded" else q)
    assert torch.equal(got, want) and torch.equal(c0.k, c1.k) and torch.equal(c0.v, c1.v)
    assert torch.equal(k, kept[0]) and torch.equal(v, kept[1]) and (kind == "expanded" or got is q)


@pytest.mark.gpu
def test_append_of_nothing_and_of_nan(dev):
    g, dt = _gen(dev, 4), torch.float16
    cache = _cache(g, 3, 16, 2, 64, dt)
    k0, v0 = cache.k.clone(), cache.v.clone()
    e = torch.empty(0, 2, 64, device=dev, dtype=dt)
    c = torch.empty(0, 32, device=dev)
    assert ops.cache_append(e, e, e, c, c, cache, torch.empty(0, device=dev, dtype=I32)).shape == (0, 2, 64)
    k, v = _randn(g, 3, 2, 64).to(dt), _randn(g, 3, 2, 64).to(dt)
    v[1, 0, 3] = math.nan
    cos, sin = _tables(g, 3, 64)
    none = torch.full((3,), -5, device=dev)
    ops.cache_append(None, k, v, cos, sin, cache, none)
    assert torch.equal(cache.k, k0) and torch.equal(cache.v, v0)
    ops.cache_append(None, k, v, cos, sin, cache, torch.tensor([0, 17, 47], device=dev))
    assert bool(cache.v[1, 1, 0, 3].isnan()) and torch.equal(cache.v[2, 15], v[2])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _seen(n, L, mask, causal, device):
    """bool [n, L]: what the n last tokens see of L keys."""
    i = torch.arange(n, device=device)[:, None]
    j = torch.arange(L, device=device)[None] - (L - n)
    if causal:
        return j <= i
    if mask is None:
        return torch.ones(n, L, dtype=torch.bool, device=device)
    full = torch.zeros(n, max(n, 1), dtype=torch.bool, device=device)
    c = min(mask.shape[1], n)
    full[:, :c] = mask[:n, :c]
    return (j < 0) | full[i.expand(n, L), j.clamp(0, max(n - 1, 0)).expand(n, L)]


def attention_ref(q, cache, table, lengths, rows, mask=None, causal=False, scale=None):
    """(out, bound, lse, bound) in 64 bits: q and mask by sequences (lists).  Keys
    in pages outside the cache are left out."""
    pages, page, Hk, D = cache.shape
    scale = D ** -0.5 if scale is None else scale
    fi = torch.finfo(cache.dtype)
    outs, tols, lses, ltols = [], [], [], []
    for b, n in enumerate(rows):
        L = min(max(int(lengths[b]), 0), table.shape[1] * page)
        x = q[b].double()
        Hq, G = x.shape[1], x.shape[1] // Hk
        if n == 0 or L == 0:
            for to, value in ((outs, 0.0), (tols, 0.0), (lses, -math.inf), (ltols, 0.0)):
                to.append(torch.full((n, Hq, D)[:2 + (to is outs or to is tols)], value, device=x.device, dtype=F64))
            continue
        pos = torch.arange(L, device=x.device)
        entry = table[b, pos // page].long()
        ok = (entry >= 0) & (entry < pages)
        see = _seen(n, L, None if mask is None else mask[b], causal, x.device) & ok[None]
        k, v = (t[entry.clamp(0, pages - 1), pos % page].double() for t in (cache.k, cache.v))  # [L, Hk, D]
        used = see.any(0)[:, None, None]
        k, v = k.masked_fill(~used, 0.0), v.masked_fill(~used, 0.0)
        k, v = (t.repeat_interleave(G, 1).transpose(0, 1) for t in (k, v))                      # [Hq, L, D]
        x = x.transpose(0, 1)
        s = (x @ k.transpose(1, 2)) * scale
        # a score is a sum of D exact products in fp32 (any order: D additions of half a step each), times the
        # scale; its exponent is taken in fp32 at arguments of the score's size (and of the maximum's)
        ds = (x.abs() @ k.abs().transpose(1, 2)) * scale * (D + 4) * 2.0 ** -24 + 2.0 ** -21 * s.abs().amax().clamp(min=1)
        s = s.masked_fill(~see, -math.inf)
        lse = torch.logsumexp(s, -1)
        p = torch.exp(s - lse.nan_to_num(neginf=0.0)[..., None])
        # a weight: its score's error, and half a step of the type (of the smallest weight kept, 2^-25 where the
        # largest is 2^8 at least in fp16); numerator and denominator; L fp32 additions
        e = ds.exp() - 1 + fi.eps / 2
        small = 2.0 ** -33 if cache.dtype == torch.float16 else 0.0
        y, w = p @ v, p * e + small * see
        wv, ws = w @ v.abs(), w.sum(-1, keepdim=True)
        tol = wv + ws * y.abs() + (L / 16 + 80) * 2.0 ** -23 * (p @ v.abs() + y.abs())
        outs.append(y.transpose(0, 1))
        tols.append(tol.transpose(0, 1))
        lses.append(lse.transpose(0, 1))
        ltols.append((ws[..., 0] * 1.02 + (L / 16 + 80) * 2.0 ** -23 + 2.0 ** -21 * lse.nan_to_num(neginf=0.0).abs()).transpose(0, 1))
    return tuple(torch.cat(t) for t in (outs, tols, lses, ltols))


def _check_attention(got, lse, ref):
    out, tol, rl, ltol = ref
    got, lse = got.reshape(out.shape), lse.reshape(rl.shape)
    tol = tol + _half_step(out, got.dtype) * (1 + 2.0 ** -6)
    bad = ~((got.double() - out).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(),
                                 ((got.double() - out).abs() / tol).nan_to_num(1e9).max().item())
    none = torch.isneginf(rl)
    assert torch.equal(none, torch.isneginf(lse)) and not bool(got[none].any())
    assert bool(((lse.double() - rl).abs() <= ltol)[~none].all())


def _pages(g, lengths, page, spare=2):
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=g, device=g.device).to(I32)
    table = torch.full((len(need), max(need + [1]) + 1), -1, dtype=I32, device=g.device)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return sum(need) + spare, table


def _tree(r, n, cols, empty=()):
    """Ancestors of the tokens of a random tree; rows of ``empty`` see nothing new."""
    m = torch.zeros(n, cols, dtype=torch.bool)
    for i in range(n):
        if i in empty:
            continue
        if i:
            m[i, :n] |= m[r.randrange(i), :n]
        m[i, i] = True
    return m


UNIFORM = [  # lengths, N, Hq, Hk, D, page
    ([1], 1, 1, 1, 128, 1), ([1, 5, 33], 1, 8, 2, 64, 16), ([31, 32, 33, 64, 65], 1, 40, 8, 128, 16),
    ([700, 513, 512, 511, 1], 1, 8, 1, 128, 64), ([5000], 1, 5, 5, 128, 48), ([4097, 100], 3, 12, 3, 64, 7),
    ([61, 200], 61, 4, 2, 128, 16), ([129, 130], 129, 2, 2, 128, 64), ([1000], 300, 4, 4, 128, 64),
    ([90, 1500, 700], 33, 6, 2, 64, 256), ([3000], 1, 40, 1, 128, 16), ([2500], 700, 3, 3, 64, 48),
    ([4200], 1030, 2, 2, 128, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("N,L,Hq,Hk,D,page,frame,cols", [
    (300, 300, 2, 1, 128, 16, 50, 300), (300, 1000, 4, 1, 64, 48, 70, 299), (700, 1500, 3, 3, 128, 64, 64, 700),
    (1300, 1300, 2, 2, 128, 64, 500, 1300), (1100, 900, 2, 2, 64, 16, 300, 1100), (2100, 2500, 2, 1, 128, 256, 33, 2600),
    (900, 5000, 1, 1, 128, 1, 400, 257), (600, 700, 2, 2, 128, 16, 600, 256)])
@pytest.mark.parametrize("kind", ["frames", "window", "holes"])
def test_attention_of_frames(dev, N, L, Hq, Hk, D, page, frame, cols, kind):
    """Masks that most of the new keys pass: tokens see their frame and those before it, or the frame and the one
    before alone, or all but single keys, one of them an inf; rows that see no new key; any byte but 0 is true."""
    g, dt = _gen(dev, 21), torch.bfloat16
    pages, table = _pages(g, [L, L - 1], page)
    cache = _cache(g, pages, page, Hk, D, dt)
    q = _randn(g, 2, N, Hq, D).to(dt)
    f = torch.arange(N, device=dev) // frame
    see = f[:, None] >= f[None]
    if kind == "window":
        see = see & (f[:, None] <= f[None] + 1)
    if kind == "holes":
        see = torch.ones_like(see)
        see[torch.arange(0, N, 7), torch.arange(0, N, 7) * 5 % N] = False
        see[:, N // 2] = False
    see = see[None].repeat(2, 1, 1)
    see[1, N // 3] = False
    byte = torch.randint(1, 256, (2, N, cols + 3), generator=g, device=dev).to(torch.uint8)
    byte[:, :, :min(N, cols)] *= see[:, :, :cols]
    mask = byte.view(torch.bool)[:, :, :cols]            # (rows at any address)
    if kind == "holes" and N // 2 < cols and L >= N:
        at = L - N + N // 2
        cache.v[table[0, at // page], at % page, 0, 3] = math.inf
    lengths = torch.tensor([L, L - 1], dtype=I32, device=dev)
    out, lse = ops.cache_attention(q, cache, table, lengths, mask=mask, return_lse=True)
    full = torch.zeros(2, N, max(cols, N), dtype=torch.bool, device=dev)
    full[:, :, :min(N, cols)] = see[:, :, :cols]
    _check_attention(out, lse, attention_ref(q, cache, table, [L, L - 1], [N, N], full))
    # the same rows, ragged
    off = torch.tensor([0, N, 2 * N], dtype=I32, device=dev)
    again = ops.cache_attention(q.flatten(0, 1), cache, table, lengths, offsets=off, mask=mask.flatten(0, 1))
    _check_attention(again, lse, attention_ref(q, cache, table, [L, L - 1], [N, N], full))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("kind", ["all", "causal", "tree"])
@pytest.mark.parametrize("case", range(len(UNIFORM)))
def test_attention(dev, case, kind, dt):
    lens, N, Hq, Hk, D, page = UNIFORM[case]
    g, dt, r = _gen(dev, case), HALF[dt], random.Random(case)
    pages, table = _pages(g, lens, page)
    cache = _cache(g, pages, page, Hk, D, dt, ["own", "pairs", "heads"][case % 3])
    q = (2 * _randn(g, len(lens), N, Hq, D)).to(dt)
    lengths = torch.tensor(lens, dtype=I32, device=dev)
    mask = torch.stack([_tree(r, N, N) for _ in lens]).to(dev) if kind == "tree" else None
    out, lse = ops.cache_attention(q, cache, table, lengths, mask=mask, causal=kind == "causal", return_lse=True)
    assert out.shape == q.shape and out.dtype == dt
    ref = attention_ref(list(q), cache, table, lens, [N] * len(lens), mask, kind == "causal")
    _check_attention(out, lse, ref)
    assert torch.equal(ops.cache_attention(q, cache, table, lengths, mask=mask, causal=kind == "causal"), out)


RAGGED = [  # (new tokens, keys) of the sequences, Hq, Hk, D, page
    ([(1, 1), (5, 5), (0, 40), (7, 300), (64, 64), (33, 1000)], 4, 2, 128, 16),
    ([(3, 0), (1, 20), (0, 0), (31, 31), (2, 700)], 8, 1, 64, 7),
    ([(128, 128), (1, 129), (200, 3000), (65, 65)], 5, 5, 128, 64),
    ([(10, 4), (1, 5000), (500, 900)], 6, 3, 64, 48)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("kind", ["all", "causal", "tree", "narrow"])
@pytest.mark.parametrize("case", range(len(RAGGED)))
def test_attention_of_ragged_batches(dev, case, kind, dt):
    """Sequences without new tokens or without keys, with fewer keys than new
    tokens, masks with empty rows and too few columns; rows behind the last sequence
    stay as they were, in outputs and inputs of any stride."""
    seqs, Hq, Hk, D, page = RAGGED[case]
    g, dt, r = _gen(dev, case + 50), HALF[dt], random.Random(case)
    rows, lens = [n for n, _ in seqs], [L for _, L in seqs]
    pages, table = _pages(g, lens, page)
    cache = _cache(g, pages, page, Hk, D, dt, ["own", "pairs", "heads"][case % 3])
    T = sum(rows)
    q = (2 * _randn(g, T + 9, Hq, D)).to(dt)
    lengths = torch.tensor(lens, dtype=I32, device=dev)
    offsets = torch.tensor([0] + rows, device=dev).cumsum(0).to(I32)
    masks = mask = None
    if kind in ("tree", "narrow"):
        cols = max(rows) if kind == "tree" else 5
        masks = [_tree(r, n, max(n, cols), empty=(0, 4))[:, :cols].to(dev) for n in rows]
        mask = torch.cat(masks + [torch.ones(9, cols, dtype=torch.bool, device=dev)])
    kw = dict(offsets=offsets, mask=mask, causal=kind == "causal")
    buf = torch.full((T + 9, 2, Hq, D), 7.0, device=dev, dtype=dt)
    out, lse = ops.cache_attention(q, cache, table, lengths, out=buf[:, 1], return_lse=True, **kw)
    qs = [q[a:a + n] for a, n in zip(offsets.tolist(), rows)]
    ref = attention_ref(qs, cache, table, lens, rows, masks, kind == "causal")
    _check_attention(out[:T], lse[:T], ref)
    assert bool((buf[:, 0] == 7.0).all() and (buf[T:] == 7.0).all())
    hq = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.cache_attention(hq, cache, table, lengths, **kw)[:T], out[:T])


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, "lowest"])
@pytest.mark.parametrize("N,L,Hq,Hk", [(1, 45, 4, 4), (5, 700, 4, 2), (150, 300, 2, 2), (40, 40, 8, 1), (300, 900, 2, 2)])
def test_attention_of_what_is_hidden(dev, N, L, Hq, Hk, value):
    """Whatever stands in slots that no one sees, past the length, in the rest of
    the last page, under pages outside the cache, has no part; a key that some rows
    see reaches those alone."""
    g, dt, page, D = _gen(dev, N), torch.bfloat16, 16, 128
    value = torch.finfo(dt).min if value == "lowest" else value
    pages, table = _pages(g, [L], page)
    clean = _cache(g, pages, page, Hk, D, dt)
    q = _randn(g, 1, N, Hq, D).to(dt)
    lengths = torch.tensor([L], dtype=I32, device=dev)
    mask = torch.ones(1, N, N, dtype=torch.bool, device=dev)
    hide = [j for j in (0, N // 2) if N > 1]
    mask[0, :, hide] = False
    bad = 1 if L > 64 else None            # the second page is none of the cache's
    was = None
    if bad is not None:
        was = int(table[0, bad])
        table[0, bad] = pages if N % 2 else -7
    slot = lambda c, j: c[int(table[0, j // page]), j % page]  # noqa: E731
    dirty = ops.PagedCache(torch.full_like(clean.k, value), torch.full_like(clean.v, value))
    for j in range(L):
        if (bad is not None and j // page == bad) or j - (L - N) in hide:
            continue
        slot(dirty.k, j).copy_(slot(clean.k, j))
        slot(dirty.v, j).copy_(slot(clean.v, j))
    want, wl = ops.cache_attention(q, clean, table, lengths, mask=mask, return_lse=True)
    got, gl = ops.cache_attention(q, dirty, table, lengths, mask=mask, return_lse=True)
    assert torch.equal(got, want) and torch.equal(gl, wl)
    ref = attention_ref([q[0]], clean, table, [L], [N], mask)
    _check_attention(got, gl, ref)
    if N > 1 and value != torch.finfo(dt).min:
        # the last row alone sees one of them: its value's channels become that
        mask[0, N - 1, hide[0]] = True
        slot(dirty.k, L - N + hide[0]).copy_(slot(clean.k, L - N + hide[0]))
        v = slot(dirty.v, L - N + hide[0])
        v.zero_()
        v[:, 3] = value
        odd = ops.cache_attention(q, dirty, table, lengths, mask=mask)
        assert torch.equal(odd[:, :N - 1], want[:, :N - 1])
        rest = [d for d in range(D) if d != 3]
        assert bool(torch.isfinite(odd[0, N - 1][:, rest]).all())
        last = odd[0, N - 1, :, 3]
        assert bool(last.isnan().all() if math.isnan(value) else (last == value).all())


@pytest.mark.gpu
@pytest.mark.parametrize("N,causal", [(1, False), (40, True), (200, True)])
def test_attention_shifted_by_a_large_score(dev, N, causal):
    """Scores that rise by hundreds along the keys, and ones far below zero: the
    running maximum moves often, and nothing overflows."""
    for dt, up in ((torch.bfloat16, 1.0), (torch.float16, 1.0), (torch.bfloat16, -1.0), (torch.float16, -1.0)):
        g, L, D, page = _gen(dev, 3), 900, 64, 16
        pages, table = _pages(g, [L], page)
        cache = _cache(g, pages, page, 2, D, dt)
        for j in range(L):
            cache.k[int(table[0, j // page]), j % page, :, 0] = up * (j // 20)
        q = (0.3 * _randn(g, 1, N, 2, D)).to(dt)
        q[..., 0] = 40.0                    # scores up to 45 * 40 / 8 = 225
        lengths = torch.tensor([L], dtype=I32, device=dev)
        out, lse = ops.cache_attention(q, cache, table, lengths, causal=causal, return_lse=True)
        _check_attention(out, lse, attention_ref([q[0]], cache, table, [L], [N], None, causal))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** -100])
@pytest.mark.parametrize("N,L,D,kind", [(1, 900, 64, "all"), (1, 9000, 128, "all"), (40, 900, 128, "causal"),
                                        (200, 900, 64, "mask"), (200, 9000, 128, "all"), (3000, 3000, 64, "causal")])
def test_attention_of_large_and_small_values(dev, N, L, D, kind, size):
    """Scores that rise by hundreds along the keys, over values far from 1 on either side: what is summed stays in
    range (a weight's error and half steps are relative, so the bounds are those of ordinary values)."""
    g, dt, page = _gen(dev, 4), torch.bfloat16, 16
    pages, table = _pages(g, [L], page)
    cache = _cache(g, pages, page, 2, D, dt)
    cache.v.mul_(size)
    at = torch.arange(L, device=dev)
    cache.k[table[0, at // page].long(), at % page, :, 0] = (at * 45 // L).to(dt)[:, None]
    q = (0.3 * _randn(g, 1, N, 2, D)).to(dt)
    q[..., 0] = 40.0
    lengths = torch.tensor([L], dtype=I32, device=dev)
    mask = torch.rand(1, N, N, generator=g, device=dev) < 0.5 if kind == "mask" else None
    out, lse = ops.cache_attention(q, cache, table, lengths, mask=mask, causal=kind == "causal", return_lse=True)
    _check_attention(out, lse, attention_ref([q[0]], cache, table, [L], [N], mask, kind == "causal"))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("N,L", [(1, 1500), (3, 70), (200, 900), (3000, 3000)])
def test_attention_of_scores_as_large_as_documented(dev, N, L, dt):
    """Scores of up to 2^26 in magnitude, the same for all keys of a head: the mean of its values."""
    g, dt, page, D = _gen(dev, 12), HALF[dt], 16, 64
    pages, table = _pages(g, [L], page)
    cache = _cache(g, pages, page, 4, D, dt)
    cache.k.zero_()
    cache.k[..., 0] = torch.tensor([2.0 ** 15, -2.0 ** 15, 2.0 ** 13, -2.0 ** 9], device=dev)
    q = torch.zeros(1, N, 4, D, device=dev)
    q[..., 0] = 2.0 ** 13 * (1 + torch.rand(1, N, 4, generator=g, device=dev))
    q = q.to(dt)
    lengths = torch.tensor([L], dtype=I32, device=dev)
    out, lse = ops.cache_attention(q, cache, table, lengths, return_lse=True)
    at = torch.arange(L, device=dev)
    v = cache.v[table[0, at // page].long(), at % page].double()         # [L, 4, D]
    mean = v.mean(0).expand_as(out[0])
    # equal weights, half a step of the type off their sum; L fp32 additions; the result's half step
    tol = mean.abs() * torch.finfo(dt).eps / 2 + (L + 80) * 2.0 ** -24 * v.abs().mean(0) + _half_step(mean, dt) * (1 + 2.0 ** -6)
    assert bool(((out[0].double() - mean).abs() <= tol).all())
    s = q[0, :, :, 0].double() * cache.k[0, 0, :, 0].double() / 8 + math.log(L)
    assert bool(((lse[0].double() - s).abs() <= 2.0 ** -22 * s.abs() + 1e-3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-6, 0.02, 1.0])
def test_attention_scales(dev, scale):
    g, dt, L = _gen(dev, 8), torch.bfloat16, 333
    pages, table = _pages(g, [L], 16)
    cache = _cache(g, pages, 16, 2, 64, dt)
    q = _randn(g, 1, 70, 2, 64).to(dt)
    lengths = torch.tensor([L], dtype=I32, device=dev)
    out, lse = ops.cache_attention(q, cache, table, lengths, scale=scale, return_lse=True)
    _check_attention(out, lse, attention_ref([q[0]], cache, table, [L], [70], scale=scale))


@pytest.mark.gpu
@pytest.mark.parametrize("N,Hq,Hk", [(1, 8, 2), (3, 4, 4), (70, 2, 2), (300, 2, 2)])
def test_attention_does_not_depend_on_the_company(dev, N, Hq, Hk):
    """A sequence alone and among others, and with more of the table, the same up to
    the rounding of its parts; the same call twice, the same bits; a workspace
    that is too small gives fewer parts."""
    g, dt, page = _gen(dev, 9), torch.bfloat16, 64
    lens = [3000, 700, 3000]
    pages, table = _pages(g, lens, page)
    cache = _cache(g, pages, page, Hk, 128, dt)
    q = _randn(g, 3, N, Hq, 128).to(dt)
    lengths = torch.tensor(lens, dtype=I32, device=dev)
    out = ops.cache_attention(q, cache, table, lengths)
    assert torch.equal(out, ops.cache_attention(q, cache, table, lengths))
    ref = attention_ref(list(q), cache, table, lens, [N] * 3)
    lse = torch.zeros(0)
    for kw in (dict(), dict(ws=torch.empty(1, dtype=torch.uint8, device=dev)),
               dict(ws=torch.empty(3 * N * Hq * 130 * 4 * 2 + 64, dtype=torch.uint8, device=dev))):
        got, lse = ops.cache_attention(q, cache, table, lengths, return_lse=True, **kw)
        _check_attention(got, lse, ref)
    one, l1 = ops.cache_attention(q[1:2], cache, table[1:2, :12], lengths[1:2], return_lse=True)
    _check_attention(one, l1, attention_ref([q[1]], cache, table[1:2, :12], [700], [N]))
    # lengths beyond the table and below zero
    far = torch.tensor([1 << 30, -5, 64], dtype=I32, device=dev)
    got, lse = ops.cache_attention(q, cache, table[:, :3], far, return_lse=True)
    _check_attention(got, lse, attention_ref(list(q), cache, table[:, :3], [192, 0, 64], [N] * 3))
    # an empty table
    got, lse = ops.cache_attention(q, cache, table[:, :0], far, return_lse=True)
    assert not bool(got.any()) and bool(torch.isneginf(lse).all())


@pytest.mark.gpu  # (row blocks of 32, 128 and 256, each in several parts)
@pytest.mark.parametrize("N,Hq,Hk,D,ragged", [(1, 8, 2, 128, False), (7, 4, 2, 64, True), (61, 8, 4, 128, True),
                                              (100, 4, 4, 64, False), (500, 6, 6, 128, False), (500, 4, 4, 64, True)])
def test_attention_with_any_workspace(dev, N, Hq, Hk, D, ragged):
    """The whole workspace, one short of it, those of seven, three and two parts and none (one part): results
    within the bounds, and nothing written outside the bytes that were given."""
    g, dt, page, lens = _gen(dev, 41), torch.bfloat16, 64, [9000, 1, 5000]
    pages, table = _pages(g, lens, page)
    cache = _cache(g, pages, page, Hk, D, dt)
    q = _randn(g, 3, N, Hq, D).to(dt)
    lengths = torch.tensor(lens, dtype=I32, device=dev)
    kw = dict(offsets=torch.arange(0, 3 * N + 1, N, device=dev, dtype=I32)) if ragged else {}
    x = q.flatten(0, 1) if ragged else q
    ref = attention_ref(q, cache, table, lens, [N] * 3)
    need = ops.cache_attention_ws_bytes(3, 3 * N, Hq, cache, table.shape[1], ragged)
    part = 3 * N * Hq * (D + 2) * 4
    assert need >= 2 * part + 16
    for n in (need, need - 1, 7 * part + 16, 3 * part + 16, 2 * part + 16, 2 * part + 15, 1, 0):
        n = min(n, need)
        buf = torch.full((n + 256,), 0xAB, dtype=torch.uint8, device=dev)
        print(N, D, "workspace", n, flush=True)
        out, lse = ops.cache_attention(x, cache, table, lengths, return_lse=True, ws=buf[:n], **kw)
        _check_attention(out, lse, ref)
        assert bool((buf[n:] == 0xAB).all())
        if n < 2 * part + 16:
            assert bool((buf == 0xAB).all())


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,Hq,Hk,D,W,kind", [
    (65, 1, 8, 8, 128, 100, "all"), (300, 1, 8, 1, 128, 250, "all"), (600, 2, 4, 1, 64, 500, "causal"),
    (200, 3, 8, 2, 128, 200, "mask"), (70, 130, 2, 2, 64, 300, "causal"), (1000, 1, 2, 2, 64, 40, "all")])
@pytest.mark.parametrize("ragged", [False, True])
def test_attention_of_many_sequences_of_unequal_lengths(dev, B, N, Hq, Hk, D, W, kind, ragged):
    """More sequences than a wave counts at once, a few of them long, in parts (but for the last)."""
    g, dt, page, r = _gen(dev, 43), torch.bfloat16, 16, random.Random(B)
    cache = _cache(g, 500, page, Hk, D, dt)
    q = _randn(g, B, N, Hq, D).to(dt)
    lens = [r.choice([0, 1, 5, 64, 65, 130]) for _ in range(B)]
    for b in (0, B // 2, B - 1):
        lens[b] = W * page - b % 7
    table = torch.randint(0, 500, (B, W), generator=g, device=dev).to(I32)
    lengths = torch.tensor(lens, dtype=I32, device=dev)
    need = ops.cache_attention_ws_bytes(B, B * N, Hq, cache, W, ragged, kind == "causal", kind == "mask")
    assert (need == 0) == (B == 1000)
    mask = torch.rand(B, N, N, generator=g, device=dev) < 0.5 if kind == "mask" else None
    kw = dict(causal=kind == "causal")
    if ragged:
        kw["offsets"] = torch.arange(0, B * N + 1, N, device=dev, dtype=I32)
    out, lse = ops.cache_attention(q.flatten(0, 1) if ragged else q, cache, table, lengths, return_lse=True,
                                   mask=mask.flatten(0, 1) if ragged and mask is not None else mask, **kw)
    _check_attention(out, lse, attention_ref(q, cache, table, lens, [N] * B, mask, kind == "causal"))


@pytest.mark.gpu
def test_attention_offsets_that_are_no_offsets(dev):
    """Offsets out of order or past the rows: no row out of range is read or
    written (their sequences' results are undefined)."""
    g, dt = _gen(dev, 10), torch.bfloat16
    pages, table = _pages(g, [50] * 4, 16)
    cache = _cache(g, pages, 16, 2, 64, dt)
    buf = torch.full((60, 4, 64), 7.0, device=dev, dtype=dt)
    q = _randn(g, 40, 4, 64).to(dt)
    lengths = torch.full((4,), 50, dtype=I32, device=dev)
    for off in ([0, 100, 5, 1 << 30, -1], [-9, -4, 0, 60, 60], [40, 30, 20, 10, 0]):
        ops.cache_attention(q, cache, table, lengths, offsets=torch.tensor(off, dtype=I32, device=dev), out=buf[10:50])
        assert bool((buf[:10] == 7.0).all() and (buf[50:] == 7.0).all())
    for B in (65, 700):
        many, lens = table[:1].repeat(B, 1), lengths[:1].repeat(B)
        for lo, hi in ((-50, 100), (0, 40), (1 << 30, (1 << 31) - 1), (-(1 << 31), 0)):
            off = torch.randint(lo, hi, (B + 1,), generator=g, device=dev).to(I32)
            for offsets in (off, off.sort(descending=True).values, off.sort().values):
                ops.cache_attention(q, cache, many, lens, offsets=offsets, causal=True, out=buf[10:50])
                assert bool((buf[:10] == 7.0).all() and (buf[50:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,Hq,Hk,D,ragged", [(1, 1, 8, 8, 128, False), (16, 1, 40, 8, 128, False), (16, 2, 8, 2, 64, True),
                                                (70, 1, 8, 8, 64, False), (70, 1, 16, 8, 128, True), (3, 61, 8, 2, 128, True),
                                                (5, 200, 4, 4, 64, False)])
def test_attention_of_unequal_lengths_in_a_captured_call(dev, B, N, Hq, Hk, D, ragged):
    """One long sequence among short ones, tables much wider than they are (behind them entries
    outside the cache), lengths that change from replay to replay, an empty sequence."""
    g, dt, page, W = _gen(dev, 31), torch.bfloat16, 16, 700
    cache = _cache(g, 900, page, Hk, D, dt)
    q = _randn(g, B, N, Hq, D).to(dt)
    kw = dict(offsets=torch.arange(0, B * N + 1, N, device=dev, dtype=I32)) if ragged else {}
    x = q.flatten(0, 1) if ragged else q
    table = torch.empty(B, W, dtype=I32, device=dev)
    lengths = torch.empty(B, dtype=I32, device=dev)
    r = random.Random(B)

    def fill(longest):
        lens = [r.choice([1, 0, 7, 64, 65, 300]) for _ in range(B)]
        lens[r.randrange(B)] = longest
        lengths.copy_(torch.tensor(lens, dtype=I32))
        table.copy_(torch.randint(0, 900, (B, W), generator=g, device=dev))
        table.masked_fill_(torch.arange(W, device=dev)[None] * page >= lengths[:, None], -1)
        return lens
    fill(500)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.cache_attention(x, cache, table, lengths, **kw)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, lse = ops.cache_attention(x, cache, table, lengths, return_lse=True, **kw)
    torch.cuda.synchronize()
    for longest in (11000, 1, 4097, 640):
        lens = fill(longest)
        graph.replay()
        torch.cuda.synchronize()
        _check_attention(out, lse, attention_ref(q, cache, table, lens, [N] * B))
        again, lse2 = ops.cache_attention(x, cache, table, lengths, return_lse=True, **kw)
        assert torch.equal(again, out) and torch.equal(lse2, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("B,most,Hq,Hk,D", [(65, 1, 4, 4, 64), (300, 3, 8, 2, 128), (4100, 1, 2, 2, 64), (130, 40, 10, 5, 128),
                                            (70, 300, 4, 2, 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_many_ragged_sequences(dev, B, most, Hq, Hk, D, causal):
    g, dt, page, r = _gen(dev, 30), torch.bfloat16, 16, random.Random(B)
    rows = [r.choice([0, 1, most, r.randint(0, most)]) for _ in range(B)]
    lens = [n + r.choice([0, 0, 5, 90]) for n in rows]
    rows[-1], lens[-1] = 0, 30
    pages, table = _pages(g, lens, page)
    cache = _cache(g, pages, page, Hk, D, dt)
    T = sum(rows)
    q = _randn(g, T + 3, Hq, D).to(dt)
    offsets = torch.tensor([0] + rows, device=dev).cumsum(0).to(I32)
    buf = torch.full((T + 3, Hq, D), 7.0, device=dev, dtype=dt)
    out, lse = ops.cache_attention(q, cache, table, torch.tensor(lens, dtype=I32, device=dev), offsets=offsets,
                                   causal=causal, out=buf, return_lse=True)
    qs = [q[a:a + n] for a, n in zip(offsets.tolist(), rows)]
    _check_attention(out[:T], lse[:T], attention_ref(qs, cache, table, lens, rows, causal=causal))
    assert bool((buf[T:] == 7.0).all())


@pytest.mark.gpu
def test_attention_of_nothing(dev):
    g, dt = _gen(dev, 11), torch.float16
    cache = _cache(g, 3, 16, 2, 64, dt)
    i = lambda *s: torch.zeros(*s, dtype=I32, device=dev)  # noqa: E731
    q = torch.empty(0, 4, 4, 64, device=dev, dtype=dt)
    assert ops.cache_attention(q, cache, i(0, 3), i(0)).shape == q.shape
    q = torch.empty(2, 0, 4, 64, device=dev, dtype=dt)
    assert ops.cache_attention(q, cache, i(2, 3), i(2)).shape == q.shape
    q = torch.empty(0, 4, 64, device=dev, dtype=dt)
    assert ops.cache_attention(q, cache, i(2, 3), i(2), offsets=i(3)).shape == q.shape
    # a mask without columns hides all new tokens
    q = _randn(g, 1, 3, 4, 64).to(dt)
    none = torch.zeros(1, 3, 0, dtype=torch.bool, device=dev)
    out, lse = ops.cache_attention(q, cache, i(1, 3), torch.tensor([3], dtype=I32, device=dev), mask=none, return_lse=True)
    assert not bool(out.any()) and bool(torch.isneginf(lse).all())


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 40, 150])
def test_attention_on_a_side_stream_and_captured(dev, N):
    """Two graphs that share a workspace, replayed in turn with new lengths, tables
    and inputs and eager work on another stream between."""
    dt, page, Hq, Hk, D = torch.bfloat16, 16, 4, 2, 128
    g = _gen(dev, 12)
    lens = [2000, 900]
    pages, table = _pages(g, lens, page)
    caches = [_cache(g, pages, page, Hk, D, dt) for _ in range(2)]
    q = _randn(g, 2, N, Hq, D).to(dt)
    lengths = torch.tensor(lens, dtype=I32, device=dev)
    need = ops.cache_attention_ws_bytes(2, 2 * N, Hq, caches[0], table.shape[1])
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        for c in caches:
            ops.cache_attention(q, c, table, lengths, ws=ws)
    torch.cuda.current_stream(dev).wait_stream(side)
    graphs, outs = [], []
    for c in caches:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.cache_attention(q, c, table, lengths, causal=True, ws=ws))
        graphs.append(gr)
    for r in range(4):
        q.copy_(_randn(g, 2, N, Hq, D))
        lengths.copy_(torch.tensor([2000 - 400 * r, 150 + 250 * r], dtype=I32))
        table.copy_(table.roll(1, 1))
        side.wait_stream(torch.cuda.current_stream(dev))
        for i in range(2):
            graphs[i].replay()
            want = ops.cache_attention(q, caches[i], table, lengths, causal=True, stream=side)
            torch.cuda.synchronize(dev)
            assert torch.equal(outs[i], want), (r, i)


@pytest.mark.gpu
def test_attention_over_a_cache_beyond_4_gib(dev):
    """Offsets past 32 bits: the last pages of a long cache."""
    g, dt, page, Hk, D = _gen(dev, 13), torch.bfloat16, 256, 8, 128
    pages = (9 << 30) // (2 * page * Hk * D * 2)          # k and v in one tensor of 9 GiB
    both = torch.zeros(pages, 2, page, Hk, D, device=dev, dtype=dt)
    cache = ops.PagedCache(both[:, 0], both[:, 1])
    L = 3 * page - 5
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=I32, device=dev)
    for p in (0, pages - 1, pages - 2):
        both[p] = _randn(g, 2, page, Hk, D).to(dt)
    k, v = (_randn(g, 40, Hk, D).to(dt) for _ in range(2))
    cos, sin = _tables(g, 40, D)
    slots = (pages - 2) * page + torch.arange(40, device=dev) + page - 45   # the last 40 positions
    q = ops.cache_append(_randn(g, 40, 16, D).to(dt), k, v, cos, sin, cache, slots)
    rk = ops.rotary(k, None, cos, sin)[0]
    assert torch.equal(both[pages - 2, 0, page - 45:page - 5], rk) and torch.equal(both[pages - 2, 1, page - 45:page - 5], v)
    for n in (1, 40):
        x = q[None, 40 - n:]
        out, lse = ops.cache_attention(x, cache, table, torch.tensor([L], dtype=I32, device=dev), causal=True, return_lse=True)
        _check_attention(out, lse, attention_ref([x[0]], cache, table, [L], [n], None, True))


# ---------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("chunks", [(7, 1, 1, 40, 3), (130, 130, 130)])
def test_generation_chunk_by_chunk(dev, chunks):
    """Projections in 8 bits, append and attention, chunk after chunk, give what the
    whole sequence gives at once: every chunk sees all before it and itself."""
    g, dt, Hq, Hk, D, page, K = _gen(dev, 14), torch.bfloat16, 6, 2, 64, 16, 200
    N = sum(chunks)
    x = _randn(g, N, K).to(dt)
    W = [ops.int8_quantize((_randn(g, H * D, K) * K ** -0.5).to(dt)) for H in (Hq, Hk, Hk)]
    nw = [(1 + 0.2 * _randn(g, D)).to(dt) for _ in range(2)]
    freqs = ops.rotary_frequencies(D, device=dev)
    pages, table = _pages(g, [N], page)
    cache = _cache(g, pages, page, Hk, D, dt, fill=math.nan)
    kw = dict(norm="head", q_weight=nw[0], k_weight=nw[1])

    def project(x):
        X = ops.int8_quantize(x)
        return (ops.int8_linear(X, w).view(x.shape[0], -1, D) for w in W)
    outs, at = [], 0
    for n in chunks:
        pos = torch.arange(at, at + n, device=dev)
        slots = table[0].long()[pos // page] * page + pos % page
        q, k, v = project(x[at:at + n])
        q = ops.cache_append(q, k, v, *ops.rotary_table(pos, freqs), cache, slots, out=q, **kw)
        at += n
        outs.append(ops.cache_attention(q[None], cache, table, torch.tensor([at], dtype=I32, device=dev))[0])
    # the whole: the same codes, products and rotation, frames as a mask
    q, k, v = project(x)
    q, k = ops.rotary(q, k, *ops.rotary_table(torch.arange(N, device=dev), freqs), **kw)
    pos = torch.arange(N, device=dev)
    at = table[0, pos // page].long(), pos % page
    assert torch.equal(cache.k[at], k) and torch.equal(cache.v[at], v)
    frame = torch.repeat_interleave(torch.arange(len(chunks)), torch.tensor(chunks)).to(dev)
    mask = (frame[None, :, None] >= frame[None, None, :])
    lengths = torch.tensor([N], dtype=I32, device=dev)
    whole, lse = ops.cache_attention(q[None], cache, table, lengths, mask=mask, return_lse=True)
    ref = attention_ref([q], cache, table, [N], [N], mask)
    _check_attention(whole, lse, ref)
    _check_attention(torch.cat(outs), lse, ref)
