"""Rotary positions and MXFP4 linear layers: every operator against plain
64-bit forms of its definition, at the sizes, layouts and values where it can
go wrong, and what the entry points refuse."""
import copy
import ctypes
import io
import math
import pickle
import random

import numpy as np
import pytest
import torch

from token2tile_amd import ops

F64 = torch.float64
HALF = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def _half_step(ref, dt):
    """Half a step of dt around ref: relative eps / 2, in the subnormal range
    half the smallest step."""
    fi = torch.finfo(dt)
    return (ref.abs() * (fi.eps / 2)).clamp(min=fi.smallest_normal * fi.eps / 2)


# ---------------------------------------------------------------------------
# frequencies
# ---------------------------------------------------------------------------
def test_frequencies_of_every_scaling():
    d, base, s, L = 64, 10000.0, 8.0, 4096
    i = torch.arange(d // 2, dtype=F64)
    plain = base ** (-2 * i / d)
    get = lambda sc, **kw: ops.rotary_frequencies(d, base=base, scaling=sc, device="cpu", **kw)  # noqa: E731
    f = get(None)
    assert f.pairs == (32,) and f.factor == 1.0 and torch.allclose(f.freqs, plain, rtol=1e-14)
    assert torch.allclose(get(ops.RotaryScaling("linear", s)).freqs, plain / s, rtol=1e-14)
    ntk = get(ops.RotaryScaling("ntk", s)).freqs
    # the fastest pair keeps its frequency, the slowest is stretched by the factor
    assert abs(float(ntk[0]) - 1) < 1e-14 and abs(float(ntk[-1] * s / plain[-1]) - 1) < 1e-12
    y = get(ops.RotaryScaling("yarn", s, L))
    turns = L * plain / (2 * math.pi)
    fast, slow = turns > 32 * base ** (2 / d), turns < base ** (-2 / d)   # a pair beyond either border
    assert fast.any() and slow.any()
    assert torch.allclose(y.freqs[fast], plain[fast], rtol=1e-14)
    assert torch.allclose(y.freqs[slow], plain[slow] / s, rtol=1e-14)
    assert bool((y.freqs <= plain * (1 + 1e-14)).all() and (y.freqs >= plain / s * (1 - 1e-14)).all())
    assert y.factor == 0.1 * math.log(s) + 1
    assert get(ops.RotaryScaling("yarn", s, L, attention=1.0)).factor == 1.0
    three = ops.rotary_frequencies((44, 42, 42), device="cpu")
    assert three.pairs == (22, 21, 21) and three.freqs.shape == (64,)
    assert three.freqs[22] == 1.0 and three.freqs[43] == 1.0


@pytest.mark.parametrize("dims", [64.0, np.int64(64), (64.0,), [np.int32(64)], torch.tensor(64)])
def test_frequencies_of_whole_numbers_of_any_type(dims):
    f = ops.rotary_frequencies(dims, device="cpu")
    assert f.pairs == (32,) and type(f.pairs[0]) is int
    assert torch.equal(f.freqs, ops.rotary_frequencies(64, device="cpu").freqs)
    for three in (np.array([44, 42, 42]), (d for d in (44, 42, 42)), torch.tensor([44, 42, 42])):
        assert ops.rotary_frequencies(three, device="cpu").pairs == (22, 21, 21)
    for bad in (63.5, "64", None, (64, None), math.nan, math.inf):
        with pytest.raises(ValueError, match="t2t"):
            ops.rotary_frequencies(bad, device="cpu")


@pytest.mark.parametrize("d,base,L,fast,slow", [
    (64, 10000.0, 4096, 32.0, 1.0), (128, 10000.0, 32768, 32.0, 1.0), (96, 500000.0, 8192, 16.0, 2.0),
    (2, 10000.0, 4096, 32.0, 1.0), (42, 10000.0, 81, 32.0, 1.0), (8, 10000.0, 1, 32.0, 1.0),
    (64, 10000.0, 2, 32.0, 1.0), (64, 10000.0, 7, 32.0, 1.0), (16, 100.0, 5_000_000, 32.0, 1.0),
    (16, 100.0, 100_000, 32.0, 1.0), (44, 10000.0, 21, 4.0, 3.9)])
def test_yarn_ramp(d, base, L, fast, slow):
    """The ramp's borders are found by counting turns, pair by pair, not from
    logarithms; a context so short (long) that every pair turns fewer (more)
    times than both borders is stretched (kept) throughout."""
    s = 8.0
    turns = lambda j: L * base ** (-2.0 * j / d) / (2.0 * math.pi)  # noqa: E731
    lo = max(j for j in range(-4 * d, 4 * d) if turns(j) >= fast)
    hi = min(j for j in range(-4 * d, 4 * d) if turns(j) <= slow)
    got = ops.rotary_frequencies(d, base=base, scaling=ops.RotaryScaling("yarn", s, L, fast, slow), device="cpu")
    for i, f in enumerate(got.freqs.tolist()):
        plain = base ** (-2.0 * i / d)
        if hi < 0:
            r = 1.0
        elif lo > d - 1:
            r = 0.0
        else:
            a, b = max(lo, 0), min(hi, d - 1)
            r = min(max((i - a) / (b - a), 0.0), 1.0) if b > a else float(i > a)
        assert abs(f - (plain * (1 - r) + plain / s * r)) <= 1e-13 * plain, (i, lo, hi)


@pytest.mark.parametrize("kw", [
    dict(dims=0), dict(dims=7), dict(dims=()), dict(dims=(2, 2, 2, 2, 2)), dict(dims=64, base=1.0),
    dict(dims=64, base=math.inf), dict(dims=64, scaling=ops.RotaryScaling("other", 2.0)),
    dict(dims=64, scaling=ops.RotaryScaling("linear", 0.5)),
    dict(dims=64, scaling=ops.RotaryScaling("yarn", 2.0)),
    dict(dims=64, scaling=ops.RotaryScaling("yarn", 2.0, 4096, 1.0, 32.0)),
    dict(dims=2, scaling=ops.RotaryScaling("ntk", 2.0))])
def test_frequencies_refused(kw):
    with pytest.raises(ValueError, match="t2t"):
        ops.rotary_frequencies(device="cpu", **kw)


# ---------------------------------------------------------------------------
# refusals before any launch
# ---------------------------------------------------------------------------
def _lib():
    from token2tile_amd import _lib as lib
    return lib, lib.lib()


def test_rotary_entries_reject_bad_arguments():
    lib, L = _lib()
    p = ctypes.c_void_p(16)
    ax = (ctypes.c_int * 4)(8, 8, 8, 8)

    def table(bits=32, T=4, axes=1, pos=p, pairs=ax):
        return L.t2t_rotary_table(pos, bits, T, axes, pairs, p, 1.0, p, p, None)
    assert table(bits=16) == 1 and table(axes=5) == 1 and table(axes=0) == 1 and table(T=-1) == 1
    assert table(pos=None) == 1 and b"null" in L.t2t_last_error()
    assert table(pairs=(ctypes.c_int * 1)(0)) == 1 and table(T=1 << 61) == 1
    assert table(T=0) == 0

    def rot(dtype=1, B=1, N=4, D=128, R=128, layout=0, inverse=0, norm=0, heads=2, q=True, k=True,
            weight=None, x=16):
        t = lib.RotaryTensor(x, 0, 0, 0, 16, 0, 0, 0, weight, heads)
        ref = ctypes.byref(t)
        return L.t2t_rotary(ref if q else None, ref if k else None, dtype, p, p, 0, B, N, D, R, layout,
                            inverse, norm, 1e-6, None)
    assert rot(q=False) == 1 and rot(x=None) == 1
    assert rot(dtype=2) == 1 and b"dtype" in L.t2t_last_error()
    assert rot(D=257) == 1 and rot(D=0, R=0) == 1 and rot(R=130) == 1 and rot(R=3) == 1 and rot(R=0) == 1
    assert rot(layout=2) == 1 and rot(norm=3) == 1 and rot(heads=0) == 1 and rot(N=-1) == 1
    assert rot(norm=1) == 1 and b"weight" in L.t2t_last_error()
    assert rot(norm=1, weight=16, inverse=1) == 1 and b"inverse" in L.t2t_last_error()
    assert rot(B=65536, N=65536) == 1
    assert rot(N=0) == 0 and rot(B=0) == 0


def test_mxfp4_entries_reject_bad_arguments():
    _, L = _lib()
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(8)
    assert L.t2t_mxfp4_code_bytes(33, 32) == 2 * 4096 and L.t2t_mxfp4_scale_bytes(33, 288) == 2 * 512
    assert L.t2t_mxfp4_code_bytes(0, 32) == 0 and L.t2t_mxfp4_scale_bytes(-1, 32) == 0
    for name in ("t2t_mxfp4_quantize", "t2t_mxfp4_dequantize"):
        if name == "t2t_mxfp4_quantize":
            f = lambda x=p, dt=1, rs=64, M=4, K=64, c=p, s=p: L.t2t_mxfp4_quantize(  # noqa: E731
                x, dt, rs, c, s, M, K, None)
        else:
            f = lambda x=p, dt=1, rs=64, M=4, K=64, c=p, s=p: L.t2t_mxfp4_dequantize(  # noqa: E731
                c, s, x, dt, rs, M, K, None)
        assert f(x=None) == 1 and f(c=None) == 1 and f(s=None) == 1 and b"null" in L.t2t_last_error()
        assert f(dt=2) == 1 and f(K=33) == 1 and f(K=0) == 1 and f(M=-1) == 1
        assert f(x=odd) == 1 and f(rs=60) == 1 and f(rs=32) == 1
        assert f(M=0) == 0

    def product(a=p, dt=1, act=0, M=4, N=8, K=64, rs=8):
        return L.t2t_mxfp4_product(a, p, p, p, None, act, p, dt, rs, M, N, K, None)
    assert product(a=None) == 1 and product(dt=9) == 1 and product(act=2) == 1 and product(N=0) == 1
    assert product(K=16) == 1 and product(rs=7) == 1 and product(a=odd) == 1 and product(M=-1) == 1
    assert product(M=0) == 0

    def linear(x=p, dt=1, xs=64, act=0, M=4, N=8, K=64, rs=8, ws=p, nb=1 << 20):
        return L.t2t_mxfp4_linear(x, dt, xs, p, p, None, act, p, rs, M, N, K, ws, nb, None)
    need = L.t2t_mxfp4_linear_ws_bytes(400, 8, 64)
    assert linear(M=400, nb=need - 1) == 2 and b"workspace" in L.t2t_last_error()
    assert linear(M=400, ws=None) == 2 and linear(x=None) == 1 and linear(xs=60) == 1 and linear(dt=3) == 1
    assert linear(act=7) == 1 and linear(rs=4) == 1 and linear(K=31) == 1 and linear(x=odd) == 1
    assert linear(M=0) == 0


@pytest.mark.parametrize("step", [(1, 0), (0, 1)])
def test_the_linear_workspace_never_falls(step):
    _, L = _lib()
    dm, dk = step
    last = 0
    for i in range(1, 3000):
        now = L.t2t_mxfp4_linear_ws_bytes(1 + 13 * dm * i, 5120, 32 + 32 * dk * i)
        assert now >= last
        last = now


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(4, 32)
    for f in (lambda: ops.mxfp4_quantize(x), lambda: ops.rotary(q, None, c, c),
              lambda: ops.rotary_table(torch.arange(4), ops.rotary_frequencies(64, device="cpu")),
              lambda: ops.mxfp4_linear(x, x), lambda: ops.mxfp4_dequantize(x)):
        with pytest.raises(ValueError, match="t2t"):
            f()


def test_calls_run_under_their_tensors_device(monkeypatch):
    """With another GPU current, the launch and its stream are the tensors' GPU's."""
    now, seen = [0], []

    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            self.was, now[0] = now[0], self.device.index

        def __exit__(self, *exc):
            now[0] = self.was

    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setitem(ops._functions, "t2t_probe", lambda *a: seen.append((now[0], a)) or 0)
    ops._launch("t2t_probe", torch.device("cuda", 1), None, (), 5)
    ops._launch("t2t_probe", torch.device("cuda", 0), None, (), 6)
    assert seen == [(1, (5, 101)), (0, (6, 100))] and now == [0]
    with pytest.raises(ValueError, match="stream"):
        ops._on(type("S", (), {"device": torch.device("cuda", 1)})(), torch.device("cuda", 0))


@pytest.fixture
def launches(monkeypatch):
    """CPU tensors in the place of GPU ones; the launches, which are not made:
    (entry point, tensors recorded on the stream, arguments)."""
    seen = []
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(ops, "_launch", lambda name, dev, stream, tensors, *a: seen.append((name, tensors, a)))
    return seen


def _mx_cpu(rows, cols, fill=0):
    n = -(-rows // 32) * -(-cols // 256) * 256
    return ops.MxFp4(torch.full((16 * n,), fill, dtype=torch.uint8), torch.full((n,), fill, dtype=torch.uint8),
                     rows, cols)


def _saved(x):
    f = io.BytesIO()
    torch.save(x, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


COPIES = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda x: pickle.loads(pickle.dumps(x)),
          "save": _saved}


@pytest.mark.parametrize("how", COPIES)
def test_a_copied_matrix_is_read_at_its_own_address(launches, how):
    W = _mx_cpu(40, 64, 3)
    c = COPIES[how](W)
    assert c.shape == (40, 64) and torch.equal(c.codes, W.codes) and torch.equal(c.scales, W.scales)
    assert (c.codes.data_ptr() == W.codes.data_ptr()) == (how == "copy")
    x = torch.zeros(40, 64, dtype=torch.bfloat16)
    ops.mxfp4_dequantize(c)
    ops.mxfp4_quantize(x, out=c)
    ops.mxfp4_linear(x, c)
    ops.mxfp4_linear(c, c)
    mine = [c.codes.data_ptr(), c.scales.data_ptr()]
    at = {"t2t_mxfp4_dequantize": [0], "t2t_mxfp4_quantize": [3], "t2t_mxfp4_linear": [3],
          "t2t_mxfp4_product": [0, 2]}
    assert [name for name, _, _ in launches] == list(at)
    for name, _, args in launches:
        for i in at[name]:
            assert list(args[i:i + 2]) == mine, name


def test_a_matrix_off_the_gpu_is_refused(monkeypatch):
    """A matrix saved on a GPU and loaded to the host goes to no kernel."""
    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "is_cuda", True, raising=False)
        W = _mx_cpu(40, 64)
    monkeypatch.setattr(ops, "_launch", lambda *a: pytest.fail("launched"))
    x = torch.zeros(40, 64, dtype=torch.bfloat16)
    for f in (lambda: ops.mxfp4_dequantize(W), lambda: ops.mxfp4_linear(x, W), lambda: ops.mxfp4_linear(W, W),
              lambda: ops.mxfp4_quantize(x, out=W)):
        with pytest.raises(ValueError, match="t2t"):
            f()


@pytest.mark.parametrize("M", [4, 400])
def test_every_tensor_of_a_call_is_recorded_on_its_stream(launches, M):
    """A caller's workspace too: it may be freed while the stream still writes it."""
    K, N = 64, 40
    dt = torch.bfloat16
    W, x, b, out = _mx_cpu(N, K), torch.zeros(M, K, dtype=dt), torch.zeros(N, dtype=dt), torch.zeros(M, N, dtype=dt)
    ws = torch.empty(max(ops.mxfp4_linear_ws_bytes(M, N, K), 256), dtype=torch.uint8)
    stream = type("S", (), {"device": x.device})()
    ops.mxfp4_linear(x, W, b, out=out, ws=ws, stream=stream)
    (_, tensors, args), = launches
    assert ws.data_ptr() in args
    for t in (x, W.codes, W.scales, b, out, ws):
        assert any(u is t for u in tensors)


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8, "bf16"])
def test_other_output_types_are_refused(launches, dtype):
    W = _mx_cpu(40, 64)
    for f in (lambda: ops.mxfp4_dequantize(W, dtype), lambda: ops.mxfp4_linear(W, W, dtype=dtype)):
        with pytest.raises(ValueError, match="t2t"):
            f()
    assert not launches


def _walk(t):
    """The addresses of a tensor's bytes."""
    at = torch.zeros((), dtype=torch.int64)
    for st, sz in zip(t.stride(), t.shape):
        at = at.unsqueeze(-1) + st * torch.arange(sz)
    e = t.element_size()
    return set((t.data_ptr() + at.reshape(-1, 1) * e + torch.arange(e)).flatten().tolist())


def test_shared_memory_is_found():
    """Random views of one buffer: what the search over the strides says is what
    the lists of addresses say."""
    r = random.Random(3)
    buf = torch.zeros(4000, dtype=torch.bfloat16)
    met = 0
    for _ in range(600):
        views = []
        for _ in range(2):
            shape = [r.randint(1, 4) for _ in range(r.randint(1, 3))] + [r.randint(1, 6)]
            stride = [r.choice([0, 1, 3, 7, 8, 24, 25, 48, 96, 200]) for _ in shape[:-1]] + [1]
            v = buf.as_strided(shape, stride, r.randint(0, 300))
            views.append(v.view(torch.uint8) if r.random() < 0.2 else v)
        a, b = views
        want = bool(_walk(a) & _walk(b))
        met += want
        assert ops._meet(a, b) == want, (a.shape, a.stride(), b.shape, b.stride(), b.data_ptr() - a.data_ptr())
        (lo, hi), at = ops._span(a), _walk(a)
        assert min(at) == lo and max(at) == hi - 1
    assert 100 < met < 500


@pytest.mark.parametrize("kind", ["own", "fused", "slots", "head_major", "moved", "step", "twice", "rows", "table",
                                  "weight", "other", "one", "same", "swapped"])
def test_outputs_of_a_rotation_share_no_memory(launches, kind):
    dt, N, H, D = torch.bfloat16, 6, 4, 32
    buf = torch.zeros(8 * N * H * D, dtype=dt)
    cos = torch.zeros(N, D // 2)
    q, k = torch.zeros(N, H, D, dtype=dt), torch.zeros(N, H, D, dtype=dt)
    view = lambda at, sn=H * D, sh=D: buf.as_strided((N, H, D), (sn, sh, 1), at)  # noqa: E731
    kw, fine = {}, True
    if kind == "own":                # in place
        out = (q, k)
    elif kind == "fused":            # both in place in one projection's rows
        q, k = view(0, 2 * H * D), view(H * D, 2 * H * D)
        out = (q, view(H * D, 2 * H * D))
    elif kind == "slots":            # heads of q and k in turn
        out = (view(0, 2 * H * D, 2 * D), view(D, 2 * H * D, 2 * D))
    elif kind == "head_major":
        out = (view(0, D, 2 * N * D), view(N * D, D, 2 * N * D))
    else:
        fine = False
        if kind == "moved":          # k's rows are q's, one token on
            out = (view(0), view(H * D))
        elif kind == "step":         # an output is its input one token on
            q = view(0)
            out = (view(H * D), k)
        elif kind == "twice":        # in place by another stride
            q = view(0)
            out = (view(0, 2 * H * D), k)
        elif kind == "rows":
            out = (view(0, 2 * H * D), view(H * D - 1, 2 * H * D))
        elif kind == "table":
            cos = buf.view(torch.float32)[:N * D // 2].view(N, D // 2)
            out = (view(0), k)
        elif kind == "weight":
            kw = dict(norm="head", q_weight=buf[:D], k_weight=torch.zeros(D, dtype=dt))
            out = (q, view(0))
        elif kind == "one":          # q for k as well, one of them in place
            k = q
            out = (q, view(0))
        elif kind == "same":
            k = q
            out = (q, q)
        elif kind == "swapped":
            out = (k, q)
        else:                        # the other's input
            k = view(64)
            out = (view(0), torch.zeros(N, H, D, dtype=dt))
    call = lambda: ops.rotary(q, k, cos, torch.zeros(N, D // 2), out=out, **kw)  # noqa: E731
    if fine:
        assert call() == out and len(launches) == 1
    else:
        with pytest.raises(ValueError, match="shares memory"):
            call()
        assert not launches


def test_outputs_of_tables_and_linears_share_no_memory(launches):
    dt, M, K, N = torch.bfloat16, 6, 64, 40
    fr = ops.rotary_frequencies(32, device="cpu")
    pos, c = torch.zeros(M, dtype=torch.int64), torch.zeros(2 * M, 16)
    ops.rotary_table(pos, fr, out=(c[:M], c[M:]))
    buf = torch.zeros(400 * 128, dtype=dt)
    W, x, rows = _mx_cpu(N, K), buf[:M * 128].view(M, 128)[:, :K], buf[:M * 128].view(M, 128)
    ops.mxfp4_linear(x, W, out=rows[:, K:K + N])                 # beside x in its rows
    raw = torch.zeros(1 << 17, dtype=torch.uint8)
    n = ops._mx_bytes(N, K)
    R = ops.MxFp4(raw[:n[0]], raw[n[0]:sum(n)], N, K)
    X = ops.MxFp4(raw[:n[0]], raw[n[0]:sum(n)], N, K)
    big = buf[:400 * K].view(400, K)
    need = ops.mxfp4_linear_ws_bytes(400, N, K)
    assert 0 < need < 1 << 16
    ops.mxfp4_linear(big, W, ws=raw[:need])
    done = len(launches)
    other = raw[1 << 16:].view(dt)
    for f in (lambda: ops.rotary_table(pos, fr, out=(c[:M], c[:M])),
              lambda: ops.rotary_table(pos, fr, out=(c[:M], c[1:M + 1])),
              lambda: ops.mxfp4_linear(x, W, out=rows[:, K - 1:K - 1 + N]),
              lambda: ops.mxfp4_linear(X, W, out=raw[:2 * N * N].view(dt).view(N, N)),
              lambda: ops.mxfp4_linear(other[:M * K].view(M, K), R, out=raw[:2 * M * N].view(dt).view(M, N)),
              lambda: ops.mxfp4_linear(x, W, other[:N], out=other[:M * N].view(M, N)),
              lambda: ops.mxfp4_linear(big, W, ws=buf.view(torch.uint8)),
              lambda: ops.mxfp4_linear(big, W, out=other[:400 * N].view(400, N), ws=raw[(1 << 16):]),
              lambda: ops.MxFp4(raw[:n[0]], raw[n[0] - 16:sum(n) - 16], N, K),
              lambda: ops.mxfp4_dequantize(X, out=raw[:2 * N * K].view(dt).view(N, K)),
              lambda: ops.mxfp4_quantize(raw[:2 * N * K].view(dt).view(N, K), out=X)):
        with pytest.raises(ValueError, match="shares memory"):
            f()
    assert len(launches) == done


@pytest.mark.gpu
@pytest.mark.parametrize("how", COPIES)
def test_a_copied_matrix_outlives_its_source(dev, how):
    g, dt = _gen(dev, 4), torch.bfloat16
    x = _randn(g, 50, 96).to(dt)
    W = ops.mxfp4_quantize(_randn(g, 70, 96).to(dt))
    want = ops.mxfp4_linear(x, W), ops.mxfp4_dequantize(W)
    c = COPIES[how](W)
    if how != "copy":
        W.codes.fill_(0)
        W.scales.fill_(255)
    assert c.device == dev and torch.equal(ops.mxfp4_linear(x, c), want[0])
    assert torch.equal(ops.mxfp4_dequantize(c), want[1])


# ---------------------------------------------------------------------------
# rotary tables
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("pdt", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,dims,scaling,last", [
    (0, 64, None, 10), (1, 64, None, 1 << 20), (3, 2, None, 100), (61, 128, ("yarn", 8.0, 32768), 262143),
    (1000, 80, ("ntk", 4.0), 1 << 20), (777, (44, 42, 42), None, 4096), (1, (16, 56, 56, 8), None, 50),
    (513, 6, ("linear", 2.0), -3000)])
def test_rotary_table(dev, pdt, T, dims, scaling, last):
    g = _gen(dev, T)
    fr = ops.rotary_frequencies(dims, scaling=ops.RotaryScaling(*scaling) if scaling else None, device=dev)
    A = len(fr.pairs)
    pos = torch.randint(min(last, 0), max(last, 0) + 1, (T, A) if A > 1 else (T,), generator=g,
                        device=dev).to(pdt)
    if T:
        pos.view(-1)[0] = last
    cos, sin = ops.rotary_table(pos, fr)
    axis = torch.tensor([a for a, n in enumerate(fr.pairs) for _ in range(n)], device=dev)
    ang = pos.double().view(T, A)[:, axis] * fr.freqs
    # 64-bit sines of both sides are far within a rounding of fp32
    for got, ref in ((cos, fr.factor * ang.cos()), (sin, fr.factor * ang.sin())):
        assert got.shape == (T, sum(fr.pairs)) and got.dtype == torch.float32
        assert bool(((got.double() - ref).abs() <= ref.abs() * 2.0 ** -24 + 2e-15).all())


@pytest.mark.gpu
def test_rotary_table_of_far_positions(dev):
    """Angles beyond 2^31: the host's sine and cosine of the same 64-bit angle;
    beyond 2^51 (half a radian between neighbours) NaN, not some number."""
    fr = ops.rotary_frequencies(64, device=dev)
    pos = [2 ** 31 - 1, 2 ** 31 + 1, 3 * 2 ** 31 + 5, 2 ** 32 + 12345, 5 * 2 ** 32 + 7, 2 ** 40 + 1, -(2 ** 33) - 1,
           -(2 ** 45) - 3, 2 ** 51 - 1, 2 ** 51, -(2 ** 51), 2 ** 53 + 2, 2 ** 62, -(2 ** 63)]
    cos, sin = (t.double().cpu() for t in ops.rotary_table(torch.tensor(pos, device=dev), fr))
    for i, p in enumerate(pos):
        for j, f in enumerate(fr.freqs.tolist()):
            a = float(p) * f
            if abs(a) >= 2.0 ** 51:
                assert math.isnan(cos[i, j]) and math.isnan(sin[i, j]), (p, j)
                continue
            # one rounding to fp32; the reduction's remainder is off by 2^-53, the series by less than
            # 1.2^16 / 16! = 9e-13 (the quotient x 2 / pi is off by up to 0.2, so |r| <= 1.2)
            for got, ref in ((cos[i, j], math.cos(a)), (sin[i, j], math.sin(a))):
                assert abs(float(got) - ref) <= abs(ref) * 2.0 ** -24 + 2e-12, (p, j)


# ---------------------------------------------------------------------------
# rotation and norm
# ---------------------------------------------------------------------------
def _tables(g, shape, R):
    a = 100 * torch.rand(*shape, R // 2, generator=g, device=g.device, dtype=F64)
    return a.cos().float(), a.sin().float()


def _rotary_ref(x, cos, sin, layout, inverse, norm, w, eps):
    """(result, bound on the fp32 part): x [B, N, H, D] in 64 bits."""
    x = x.double()
    if norm == "token":
        x = x / (x.square().mean((-2, -1), keepdim=True) + eps).sqrt() * w.double().view(x.shape[-2:])
    elif norm == "head":
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    R = 2 * cos.shape[-1]
    c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    s = -s if inverse else s
    y, mag = x.clone(), x.abs()
    lo, hi = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    m = a.abs() + b.abs()
    mag[..., lo], mag[..., hi] = m, m
    return y, mag


def _check_rotary(got, x, cos, sin, layout, inverse, norm, w, eps=1e-6):
    ref, mag = _rotary_ref(x, cos, sin, layout, inverse, norm, w, eps)
    # fp32: the norm's sum of squares is off by at most 128 additions of 2^-24 each
    # (half of that under the root), its root, quotient and three products by a few
    # more; the turn's products and sum by three: 2^-17 of |a| + |b| covers all
    tol = _half_step(ref, x.dtype) * (1 + 2.0 ** -7) + 2.0 ** -17 * mag
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), ((got.double() - ref).abs() / tol).max()


ROTARY = [  # B, N, HQ, HK, D, R
    (1, 1, 40, 40, 128, 128), (4, 1, 12, 2, 128, 128), (1, 5, 1, 1, 2, 2), (2, 33, 5, 3, 64, 32),
    (1, 130, 7, 1, 80, 80), (1, 9, 3, 3, 96, 48), (3, 17, 33, 8, 128, 96), (1, 40, 65, 9, 128, 128),
    (1, 7, 4, 2, 256, 256), (1, 7, 4, 2, 256, 64), (1, 6, 2, 2, 88, 24), (1, 6, 3, 1, 77, 20),
    (1, 3, 300, 130, 128, 128), (2, 300, 12, 12, 128, 64), (1, 4, 700, 1, 64, 64), (1, 1501, 3, 1, 64, 32),
    (2, 1100, 1, 1, 40, 40), (1, 1203, 32, 8, 256, 128), (1, 1025, 40, 5, 128, 128), (3, 701, 5, 2, 20, 12),
    (1, 1300, 33, 2, 80, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("norm", [None, "token", "head"])
@pytest.mark.parametrize("B,N,HQ,HK,D,R", ROTARY)
def test_rotary(dev, B, N, HQ, HK, D, R, norm, layout, dt):
    g, dt = _gen(dev, D + HQ), HALF[dt]
    q, k = (4 * _randn(g, B, N, H, D).to(dt) for H in (HQ, HK))
    batched = B > 1
    cos, sin = _tables(g, (B, N) if batched else (N,), R)
    w = [None, None]
    if norm:
        w = [(1 + 0.3 * _randn(g, H * D if norm == "token" else D)).to(dt) for H in (HQ, HK)]
    oq, ok = ops.rotary(q, k, cos, sin, layout=layout, norm=norm, q_weight=w[0], k_weight=w[1])
    _check_rotary(oq, q, cos, sin, layout, False, norm, w[0])
    _check_rotary(ok, k, cos, sin, layout, False, norm, w[1])
    # alone, and back again
    o1, none = ops.rotary(q, None, cos, sin, layout=layout, norm=norm, q_weight=w[0])
    assert none is None and torch.equal(o1, oq)
    if not norm:
        bq, bk = ops.rotary(q, k, cos, sin, layout=layout, inverse=True)
        _check_rotary(bq, q, cos, sin, layout, True, None, None)
        _check_rotary(bk, k, cos, sin, layout, True, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [None, "token", "head"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kind", ["fused", "head_major", "misaligned", "odd_stride", "expanded"])
def test_rotary_views(dev, kind, layout, norm):
    """Strided inputs and outputs give the bits of contiguous ones, and nothing
    but the output's elements is written."""
    g, dt = _gen(dev, 3), torch.bfloat16
    N, HQ, HK, D, R = 37, 6, 2, 128, 96
    cos, sin = _tables(g, (N,), R)
    w = {None: (None, None), "head": [_randn(g, D).to(dt)] * 2,
         "token": [_randn(g, H * D).to(dt) for H in (HQ, HK)]}[norm]
    call = lambda q, k, **kw: ops.rotary(q, k, cos, sin, layout=layout, norm=norm, q_weight=w[0],  # noqa: E731
                                         k_weight=w[1], **kw)
    if kind == "fused":              # q, k, v of one projection: [N, (HQ + 2 HK) D], in place
        buf = _randn(g, N, (HQ + 2 * HK), D).to(dt)
        q, k = buf[:, :HQ], buf[:, HQ:HQ + HK]
        want = call(q.contiguous(), k.contiguous())
        keep = buf[:, HQ + HK:].clone()
        got = call(q, k, out=(q, k))
        assert got[0] is q and torch.equal(buf[:, HQ + HK:], keep)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        return
    shape = {"head_major": lambda H: _randn(g, H, N, D).to(dt).transpose(0, 1),
             "misaligned": lambda H: _randn(g, N * H * D + 3).to(dt)[3:].view(N, H, D),
             "odd_stride": lambda H: _randn(g, N, H, D + 3).to(dt)[..., :D],
             "expanded": lambda H: _randn(g, 1, H, D).to(dt).expand(N, H, D)}[kind]
    q, k = shape(HQ), shape(HK)
    want = call(q.contiguous(), k.contiguous())
    outs = []
    for x in (q, k):
        if kind == "expanded":
            outs.append(torch.empty(N, x.shape[1], D, device=dev, dtype=dt))
            continue
        flat = torch.full((x.untyped_storage().nbytes() // 2,), 7.0, device=dev, dtype=dt)
        outs.append(flat.as_strided(x.shape, x.stride(), x.storage_offset()))
    got = call(q, k, out=tuple(outs))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if kind != "expanded":
        for o in outs:
            flat = torch.as_strided(o, (o.untyped_storage().nbytes() // 2,), (1,), 0).clone()
            flat.as_strided(o.shape, o.stride(), o.storage_offset()).fill_(7.0)
            assert bool((flat == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_rotary_of_more_tokens_than_work_groups(dev, shift):
    """The kernels go through the tokens; the last ones are as the first."""
    g, dt = _gen(dev, shift), torch.float16
    N = 70001
    q = _randn(g, N * 2 * 16 + shift).to(dt)[shift:].view(N, 2, 16)
    cos, sin = _tables(g, (N,), 16)
    w = (1 + 0.3 * _randn(g, 32)).to(dt)
    got = ops.rotary(q, None, cos, sin, norm="token", q_weight=w)[0]
    _check_rotary(got, q, cos, sin, "interleaved", False, "token", w)


@pytest.mark.gpu
def test_rotary_results_do_not_depend_on_the_company(dev):
    """A token's result is the same bits alone and among many, whatever the form
    its call takes."""
    g, dt = _gen(dev, 21), torch.bfloat16
    for D, H, norm in ((128, 40, "token"), (96, 12, "token"), (128, 12, "head"), (64, 70, "token"),
                       (64, 1, "token"), (40, 3, "token"), (20, 2, "head"), (256, 32, "token")):
        q = _randn(g, 2000, H, D).to(dt)
        cos, sin = _tables(g, (2000,), D)
        w = (1 + 0.2 * _randn(g, H * D if norm == "token" else D)).to(dt)
        f = lambda a, b: ops.rotary(q[a:b], None, cos[a:b], sin[a:b], norm=norm, q_weight=w)[0]  # noqa: E731
        whole = f(0, 2000)
        for a, b in ((0, 1), (777, 778), (1500, 1517)):
            assert torch.equal(whole[a:b], f(a, b))


@pytest.mark.gpu
def test_rotary_of_no_tokens_nan_and_far_values(dev):
    c = torch.ones(0, 32, device=dev)
    q = torch.empty(0, 3, 64, device=dev, dtype=torch.float16)
    assert ops.rotary(q, None, c, c)[0].shape == q.shape
    # a NaN stays with its pair (no norm), with its token (norm); others are untouched
    g = _gen(dev, 1)
    q = _randn(g, 4, 3, 64).half()
    cos, sin = _tables(g, (4,), 64)
    w = torch.ones(64, device=dev, dtype=torch.float16)
    clean = ops.rotary(q, None, cos, sin, norm="head", q_weight=w)[0]
    q[2, 1, 5] = float("nan")
    bare = ops.rotary(q, None, cos, sin)[0].isnan().nonzero().tolist()
    assert bare == [[2, 1, 4], [2, 1, 5]]
    got = ops.rotary(q, None, cos, sin, norm="head", q_weight=w)[0]
    assert bool(got[2, 1].isnan().all())
    got[2, 1] = clean[2, 1]
    assert torch.equal(got, clean)
    # a head of zeros stays zero under the norm
    z = torch.zeros(1, 1, 64, device=dev, dtype=torch.float16)
    assert not bool(ops.rotary(z, None, cos[:1], sin[:1], norm="head", q_weight=w)[0].any())


@pytest.mark.gpu
def test_inverse_rotation_is_the_transpose(dev):
    """<rotate(x), y> = <x, rotate back(y)>: the way back of a gradient, and
    against differences of the forward."""
    g = _gen(dev, 2)
    x, y = (_randn(g, 9, 4, 64).to(torch.bfloat16) for _ in range(2))
    cos, sin = _tables(g, (9,), 48)
    for layout in ("interleaved", "half"):
        f = ops.rotary(x, None, cos, sin, layout=layout)[0].double()
        b = ops.rotary(y, None, cos, sin, layout=layout, inverse=True)[0].double()
        n = x.double().norm() * y.double().norm()
        assert abs(float((f * y.double()).sum() - (x.double() * b).sum())) <= 2 * 2.0 ** -8 * float(n)
        # the forward is linear: its difference along a step e is its derivative, and the
        # derivative of <rotate(x), y> along e is <e, rotate back(y)>
        e = torch.zeros_like(x)
        e[3, 2, 7] = 1.0
        d = ops.rotary(e, None, cos, sin, layout=layout)[0].double()
        assert abs(float((d * y.double()).sum() - b[3, 2, 7])) <= 4 * 2.0 ** -8 * float(y[3, 2].double().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", ["cos_shape", "cos_dtype", "sin_shape", "weight_shape", "weight_dtype",
                                 "no_weight", "weight_without_norm", "layout", "norm", "inverse", "k_width",
                                 "k_tokens", "k_type", "channel_stride", "out_shape", "out_twice", "wide",
                                 "eps", "rotated", "out_same", "out_other"])
def test_rotary_refused(dev, bad):
    dt = torch.bfloat16
    z = lambda *s, dtype=dt: torch.zeros(*s, device=dev, dtype=dtype)  # noqa: E731
    q, k, c = z(6, 4, 64), z(6, 2, 64), z(6, 32, dtype=torch.float32)
    a, kw = [q, k, c, c], {}
    if bad == "cos_shape":
        a[2] = z(5, 32, dtype=torch.float32)
    elif bad == "cos_dtype":
        a[2] = z(6, 32)
    elif bad == "sin_shape":
        a[3] = z(6, 31, dtype=torch.float32)
    elif bad == "rotated":
        a[2] = a[3] = z(6, 33, dtype=torch.float32)
    elif bad == "weight_shape":
        kw = dict(norm="token", q_weight=z(256), k_weight=z(64))
    elif bad == "weight_dtype":
        kw = dict(norm="head", q_weight=z(64, dtype=torch.float32), k_weight=z(64))
    elif bad == "no_weight":
        kw = dict(norm="head", q_weight=z(64))
    elif bad == "weight_without_norm":
        kw = dict(q_weight=z(64))
    elif bad in ("layout", "norm"):
        kw = {bad: "other"}
    elif bad == "inverse":
        kw = dict(norm="head", q_weight=z(64), k_weight=z(64), inverse=True)
    elif bad == "eps":
        kw = dict(norm="head", q_weight=z(64), k_weight=z(64), eps=-1.0)
    elif bad == "k_width":
        a[1] = z(6, 2, 80)
    elif bad == "k_tokens":
        a[1] = z(5, 2, 64)
    elif bad == "k_type":
        a[1] = z(6, 2, 64, dtype=torch.float16)
    elif bad == "channel_stride":
        a[0] = z(6, 4, 128)[..., ::2]
    elif bad == "out_shape":
        kw = dict(out=(z(6, 4, 65), z(6, 2, 64)))
    elif bad == "out_same":
        a[1] = z(6, 4, 64)
        kw = dict(out=(z(6, 4, 64),) * 2)
    elif bad == "out_other":
        a[1] = z(6, 4, 64)
        kw = dict(out=(a[1], z(6, 4, 64)))
    elif bad == "out_twice":
        kw = dict(out=(z(1, 4, 64).expand(6, 4, 64), z(6, 2, 64)))
    else:
        a = [z(6, 1, 264), None, z(6, 132, dtype=torch.float32), z(6, 132, dtype=torch.float32)]
    with pytest.raises(ValueError, match="t2t"):
        ops.rotary(*a, **kw)


# ---------------------------------------------------------------------------
# MXFP4
# ---------------------------------------------------------------------------
STEPS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def mx_ref(x):
    """The values that MXFP4 holds for x [M, K], in 64 bits: the nearest of the
    eight magnitudes by distance, an even index on ties."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top)[1].double() - 3).clamp(min=-126)
    t = (b.abs() / torch.exp2(e)).clamp(max=6.0)   # exp2 is exact here; pow(2, e) on the GPU is not
    best, near = torch.zeros_like(t), t.clone()
    for i, s in enumerate(STEPS[1:], 1):
        d = (t - s).abs()
        take = (d < near) | ((d == near) & (i % 2 == 0))
        best, near = torch.where(take, torch.full_like(t, s), best), torch.where(take, d, near)
    v = torch.copysign(best * torch.exp2(e), b)
    return v.masked_fill(~b.isfinite().all(-1, keepdim=True), math.nan).flatten(-2)


def _same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("M,K", [(1, 32), (1, 5120), (2, 64), (31, 96), (32, 256), (33, 288), (257, 1536),
                                 (1000, 160)])
def test_quantize(dev, M, K, dt):
    g, dt = _gen(dev, M + K), HALF[dt]
    x = (_randn(g, M, K) * torch.exp(2 * _randn(g, K))).to(dt)
    t = ops.mxfp4_quantize(x)
    assert t.shape == (M, K) and t.codes.numel() == -(-M // 32) * -(-K // 256) * 4096
    assert _same(ops.mxfp4_dequantize(t, dt).double(), mx_ref(x))
    # as the layout says, padding included
    G = -(-K // 256)
    rows = -(-M // 32) * 32
    v = torch.zeros(rows, G * 256, device=dev, dtype=F64)
    v[:M, :K] = mx_ref(x)
    c = t.codes.view(-1, G, 4, 2, 32, 16).permute(0, 4, 1, 2, 3, 5).reshape(rows, -1).long()
    tab = torch.tensor(STEPS, device=dev, dtype=F64)
    m = torch.stack((c & 15, c >> 4), -1).flatten(1)
    s = t.scales.view(-1, G, 2, 32, 4).permute(0, 3, 1, 4, 2).reshape(rows, -1).double()
    got = tab[m & 7] * torch.where(m > 7, -1.0, 1.0) * torch.exp2(s - 127).repeat_interleave(32, 1)
    assert _same(got, v)
    assert not bool(t.codes.view(-1, G, 4, 2, 32, 16)[-1, :, :, :, (M - 1) % 32 + 1:].any())


@pytest.mark.gpu
def test_quantize_more_tiles_than_work_groups(dev):
    g = _gen(dev, 1)
    x = _randn(g, 65537 * 32 + 5, 32).to(torch.float16)
    y = ops.mxfp4_dequantize(ops.mxfp4_quantize(x), torch.float16)
    for part in (slice(0, 4096), slice(-4096, None)):
        assert _same(y[part].double(), mx_ref(x[part]))
    assert bool(((y - x).abs() <= x.abs().amax(1, keepdim=True) / 4).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
def test_quantize_every_value(dev, dt):
    """Every 16-bit value once under each other value's scale range: blocks of
    one magnitude with random mates below it; ties, infs, NaN, subnormals."""
    dt = HALF[dt]
    g = _gen(dev, 0)
    bits = torch.arange(65536, device=dev, dtype=torch.int32).to(torch.int16)
    x = bits.view(dt)[:, None].repeat(1, 32)
    # mates: the value shifted down by 0 .. 7 binades, random low bits (finite: below it)
    mate = (bits.int() & 0x7fff)[:, None] - torch.randint(0, 8 << (7 if dt == torch.bfloat16 else 10),
                                                          (65536, 31), generator=g, device=dev)
    x[:, 1:] = mate.clamp(min=0).to(torch.int16).view(dt)
    x[:, 5] = -x[:, 5]
    t = ops.mxfp4_quantize(x)
    assert _same(ops.mxfp4_dequantize(t, dt).double(), mx_ref(x))


@pytest.mark.gpu
def test_quantize_ties_and_saturation(dev):
    row = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.96875, -0.25, -0.75, -5.0, -7.0, 0.2490234375,
           0.2509765625, 0.0, -0.0, 4.0, 6.0, 3.0]
    want = [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0, 0.0, -1.0, -4.0, -6.0, 0.0, 0.5, 0.0, 0.0, 4.0, 6.0,
            3.0]
    x = torch.zeros(3, 32, device=dev, dtype=torch.float16)
    x[1, :len(row)] = torch.tensor(row, dtype=torch.float16)
    y = ops.mxfp4_dequantize(ops.mxfp4_quantize(x), torch.float16)
    assert y[1, :len(row)].tolist() == want and not bool(y[::2].any())


@pytest.mark.gpu
def test_quantize_views_and_buffers(dev):
    g = _gen(dev, 5)
    big = _randn(g, 70, 3, 96).to(torch.bfloat16)
    want = ops.mxfp4_dequantize(ops.mxfp4_quantize(big[:, 1].contiguous()))
    t = ops.mxfp4_quantize(big[:, 1])                            # row stride 288
    assert torch.equal(ops.mxfp4_dequantize(t), want)
    t.codes.fill_(255)
    t.scales.fill_(255)
    assert ops.mxfp4_quantize(big[:, 1], out=t) is t             # every byte is written, padding too
    assert torch.equal(ops.mxfp4_dequantize(t), want)
    buf = torch.full((72, 200), 9.0, device=dev, dtype=torch.bfloat16)
    ops.mxfp4_dequantize(t, out=buf[1:71, 8:104])
    assert torch.equal(buf[1:71, 8:104], want)
    buf[1:71, 8:104] = 9.0
    assert bool((buf == 9.0).all())
    e = ops.mxfp4_quantize(big[:0, 0])
    assert e.shape == (0, 96) and ops.mxfp4_dequantize(e).shape == (0, 96)
    assert ops.mxfp4_quantize(big.view(7, 10, 3, 96)).shape == (210, 96)


def _linear_ref(x, w, b, act):
    """(result, bound on the fp32 part) from the values of both operands."""
    a, w = mx_ref(x), mx_ref(w)
    y = a @ w.t()
    mag = a.abs() @ w.abs().t()
    if b is not None:
        y = y + b.double()
        mag = mag + b.double().abs()
    # fp32 sums of K products in any order, 2^-23 of the terms' magnitudes an addition:
    # chains of at most K / 32 + 64
    tol = (x.shape[1] / 32 + 64) * 2.0 ** -23 * mag
    if act:
        u = math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
        # |gelu'| <= 1.13; e^-2u is off by 2 |u| 2^-23 and a few roundings, y / (1 + e) by as much
        # where e counts: 2^-18 of |y| covers it
        tol = 1.13 * tol + 2.0 ** -18 * y.abs()
        y = 0.5 * y * (1 + torch.tanh(u))
    return y, tol


def _check_linear(got, x, w, b, act):
    ref, tol = _linear_ref(x, w, b, act)
    tol = tol + _half_step(ref, got.dtype) * (1 + 2.0 ** -7)
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


# (33, 20481, 256) and on: 128 x 128 tiles; (16385, 1030, 1056) and on: 256 x 256 tiles
SIZES = [(1, 1, 32), (1, 64, 64), (1, 5120, 512), (2, 33, 96), (5, 96, 256), (31, 100, 288), (32, 32, 1568),
         (33, 257, 512), (64, 640, 2048), (100, 72, 5120), (129, 130, 160), (257, 513, 256), (600, 1000, 320),
         (1000, 1536, 1536), (2049, 776, 64), (4099, 2041, 1568),
         (33, 20481, 256), (700, 1100, 512), (300, 1700, 800), (16385, 1030, 1056), (4100, 4200, 1024),
         (70000, 1025, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
@pytest.mark.parametrize("dt,bias", [("bf16", True), ("fp16", False)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(dev, M, N, K, dt, bias, act):
    g, dt = _gen(dev, M + N + K), HALF[dt]
    x = (_randn(g, M, K) * torch.exp(0.5 * _randn(g, K))).to(dt)
    w = (_randn(g, N, K) * K ** -0.5).to(dt)
    b = _randn(g, N).to(dt) if bias else None
    W = ops.mxfp4_quantize(w)
    y = ops.mxfp4_linear(x, W, b, activation=act)
    assert y.shape == (M, N) and y.dtype == dt
    _check_linear(y, x, w, b, act)
    # the product of an already quantised x: the same sums
    z = ops.mxfp4_linear(ops.mxfp4_quantize(x), W, b, activation=act, dtype=dt)
    _check_linear(z, x, w, b, act)
    assert torch.equal(ops.mxfp4_linear(x, W, b, activation=act), y)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_views_and_buffers(dev, M):
    g, dt = _gen(dev, M), torch.bfloat16
    K, N = 192, 72
    big = _randn(g, 2 * M, 2, K).to(dt)
    x = big.view(2, M, 2, K)[:, :, 1]                            # [2, M, K], row stride 2 K
    w = _randn(g, N, K).to(dt)
    W = ops.mxfp4_quantize(w)
    b = _randn(g, N).to(dt)
    y = ops.mxfp4_linear(x, W, b)
    assert y.shape == (2, M, N)
    _check_linear(y.view(-1, N), x.reshape(-1, K), w, b, None)
    for off, width in ((8, 96), (3, 77)):                        # aligned rows, odd ones
        buf = torch.full((2 * M + 2, width), 5.0, device=dev, dtype=dt)
        out = buf[1:2 * M + 1, off:off + N].unflatten(0, (2, M))
        ws = torch.empty(ops.mxfp4_linear_ws_bytes(2 * M, N, K), dtype=torch.uint8, device=dev)
        assert ops.mxfp4_linear(x, W, b, out=out, ws=ws) is out
        assert torch.equal(out, y)
        out.fill_(5.0)
        assert bool((buf == 5.0).all())
    # one-dimensional and empty inputs
    assert torch.equal(ops.mxfp4_linear(x[0, 0].contiguous(), W, b),
                       ops.mxfp4_linear(x[0, :1].contiguous(), W, b)[0])
    assert ops.mxfp4_linear(x[:, :0], W, b).shape == (2, 0, N)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 48), (40, 48), (700, 600)])
def test_linear_of_nonfinite_blocks(dev, M, N):
    """An inf or NaN turns its row (x) or column (weight) of the result to NaN
    and leaves the rest; a row of zeros gives the bias."""
    g, dt, K = _gen(dev, 9), torch.float16, 320
    x, w, b = _randn(g, M, K).to(dt), _randn(g, N, K).to(dt), _randn(g, N).to(dt)
    x[0] = 0
    clean = ops.mxfp4_linear(x, ops.mxfp4_quantize(w), b)
    assert torch.equal(clean[0], b)
    w[7, 300] = float("inf")
    if M > 1:
        x[M - 1, 40] = float("nan")
    y = ops.mxfp4_linear(x, ops.mxfp4_quantize(w), b)
    bad = torch.zeros(M, N, device=dev, dtype=torch.bool)
    bad[:, 7] = True
    if M > 1:
        bad[M - 1] = True
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], clean[~bad])


@pytest.mark.gpu
def test_linear_of_long_sums(dev):
    """Magnitudes that 16-bit sums would lose: 13,824 products of one sign."""
    K = 13824
    x = torch.full((3, K), 6.0, device=dev, dtype=torch.bfloat16)
    w = torch.full((40, K), 0.5, device=dev, dtype=torch.bfloat16)
    x[1] = 1.5
    y = ops.mxfp4_linear(x, ops.mxfp4_quantize(w))
    # 41,472 and 10,368: rounded once to bf16 (steps of 256 and 64)
    want = (torch.tensor([3.0, 0.75, 3.0], device=dev) * K).to(torch.bfloat16)
    assert torch.equal(y, want[:, None].expand(3, 40))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", ["k", "cols", "stride", "align", "type", "bias", "bias_type", "act", "dtype",
                                 "out", "out_type", "out_twice", "weight", "buffers", "ws", "rows", "out_mx"])
def test_mxfp4_refused(dev, bad):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device=dev, dtype=dtype)  # noqa: E731
    W, x = ops.mxfp4_quantize(z(40, 64)), z(6, 64)
    calls = {
        "k": lambda: ops.mxfp4_linear(z(6, 96), W),
        "cols": lambda: ops.mxfp4_quantize(z(6, 40)),
        "stride": lambda: ops.mxfp4_quantize(z(64, 6).t()),
        "align": lambda: ops.mxfp4_quantize(z(6 * 64 + 8)[1:385].view(6, 64)),
        "type": lambda: ops.mxfp4_quantize(z(6, 64, dtype=torch.float32)),
        "bias": lambda: ops.mxfp4_linear(x, W, z(41)),
        "bias_type": lambda: ops.mxfp4_linear(x, W, z(40, dtype=torch.float32)),
        "act": lambda: ops.mxfp4_linear(x, W, activation="relu"),
        "dtype": lambda: ops.mxfp4_linear(x, W, dtype=torch.float16),
        "out": lambda: ops.mxfp4_linear(x, W, out=z(6, 41)),
        "out_type": lambda: ops.mxfp4_linear(x, W, out=z(6, 40, dtype=torch.float16)),
        "out_twice": lambda: ops.mxfp4_linear(x, W, out=z(1, 40).expand(6, 40)),
        "weight": lambda: ops.mxfp4_linear(x, z(40, 64)),
        "buffers": lambda: ops.mxfp4_dequantize(ops.MxFp4(W.codes[:-1], W.scales, 40, 64)),
        "ws": lambda: ops.mxfp4_linear(x, W, ws=z(1 << 16)),
        "rows": lambda: ops.mxfp4_quantize(z(6, 2, 3, 64)[:, :, 1]),
        "out_mx": lambda: ops.mxfp4_quantize(x, out=W)}
    if bad == "rows":   # [6, 2, 64] with strides (384, 192, 1): one row stride, accepted
        assert calls[bad]().shape == (12, 64)
        calls[bad] = lambda: ops.mxfp4_quantize(z(6, 3, 3, 64)[:, :2, 1])
    with pytest.raises(ValueError, match="t2t"):
        calls[bad]()


# 128 x 128 tiles (32 x 48 blocks; the last group of 256 columns padded in the second), 256 x 256 tiles
# (17 x 17 of them, the last ones with a single block of rows or one of 96 columns)
TILES = [(1000, 1536, 512), (1000, 1531, 800), (4100, 4200, 1024), (4100, 4195, 1056)]


def _operands(dev, M, N, K, dt, seed):
    g = _gen(dev, seed)
    return _randn(g, M, K).to(dt), (_randn(g, N, K) * K ** -0.5).to(dt), _randn(g, N).to(dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,act", [("bf16", "gelu_tanh"), ("fp16", None)])
@pytest.mark.parametrize("M,N,K", TILES)
def test_tiles_into_views(dev, M, N, K, dt, act):
    """Outputs of any stride and address get the bits of a contiguous one, and
    nothing around them is written."""
    dt = HALF[dt]
    x, w, b = _operands(dev, M, N, K, dt, M + N)
    W = ops.mxfp4_quantize(w)
    y = ops.mxfp4_linear(x, W, b, activation=act)
    _check_linear(y, x, w, b, act)
    X = ops.mxfp4_quantize(x)
    # aligned rows, an address off by 8 bytes, an odd stride, an odd stride and address
    for off, width in ((16, N + 24 - N % 8), (4, N + 24 - N % 8), (8, N + 17 - N % 2), (3, N + 17 - N % 2)):
        buf = torch.full((M + 2, width), 5.0, device=dev, dtype=dt)
        out = buf[1:M + 1, off:off + N]
        for src in (x, X):
            assert ops.mxfp4_linear(src, W, b, activation=act, dtype=dt, out=out) is out
            assert torch.equal(out, y), (off, width)
            out.fill_(5.0)
            assert bool((buf == 5.0).all()), (off, width)


@pytest.mark.gpu
@pytest.mark.parametrize("col", [40, 168, -1])
@pytest.mark.parametrize("M,N,K", TILES)
def test_tiles_of_nonfinite_blocks(dev, M, N, K, col):
    """In an even stage of 128 columns, an odd one and the last: an inf or NaN
    turns its row or column of the result to NaN and leaves the rest; a row of
    zeros gives the bias."""
    x, w, b = _operands(dev, M, N, K, torch.float16, col + 2)
    x[0] = 0
    clean = ops.mxfp4_linear(x, ops.mxfp4_quantize(w), b)
    assert torch.equal(clean[0], b)
    bad = torch.zeros(M, N, device=dev, dtype=torch.bool)
    for r in (7, N // 2, N - 1):
        w[r, col] = float("inf")
        bad[:, r] = True
    for r in (130, M - 1):
        x[r, col] = float("nan")
        bad[r] = True
    y = ops.mxfp4_linear(x, ops.mxfp4_quantize(w), b)
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], clean[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(600, 1000), (4100, 4200)])
def test_tiles_of_long_sums(dev, M, N):
    """13,824 products of one sign, as in the split form."""
    K = 13824
    x = torch.full((M, K), 6.0, device=dev, dtype=torch.bfloat16)
    w = torch.full((N, K), 0.5, device=dev, dtype=torch.bfloat16)
    x[1::2] = 1.5
    y = ops.mxfp4_linear(x, ops.mxfp4_quantize(w))
    want = (torch.tensor([3.0, 0.75], device=dev) * K).to(torch.bfloat16)
    assert torch.equal(y, want.repeat(M // 2)[:, None].expand(M, N))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", TILES)
def test_tiles_on_a_side_stream_and_captured(dev, M, N, K):
    """Two graphs that share a workspace, replayed in turn with new inputs and
    eager work on another stream between, against the eager results."""
    dt = torch.bfloat16
    x, w, b = _operands(dev, M, N, K, dt, 3)
    W = [ops.mxfp4_quantize(w), ops.mxfp4_quantize(w.flip(0))]
    ws = torch.empty(ops.mxfp4_linear_ws_bytes(M, N, K), dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        for i in range(2):
            ops.mxfp4_linear(x, W[i], b, ws=ws)
    torch.cuda.current_stream(dev).wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.mxfp4_linear(x, W[i], b, activation="gelu_tanh", ws=ws))
        graphs.append(gr)
    for r in range(3):
        x.copy_(_randn(_gen(dev, r), M, K))
        side.wait_stream(torch.cuda.current_stream(dev))
        for i in range(2):
            graphs[i].replay()
            want = ops.mxfp4_linear(x, W[i], b, activation="gelu_tanh", stream=side)
            torch.cuda.synchronize(dev)
            assert torch.equal(outs[i], want), (r, i)


# ---------------------------------------------------------------------------
# streams, captures and the operators together
# ---------------------------------------------------------------------------
@pytest.mark.gpu
def test_operators_on_a_side_stream(dev):
    """On a given stream the calls follow that stream's work, and their
    workspaces and outputs are its own."""
    g, dt = _gen(dev, 11), torch.bfloat16
    x0, w, b = _randn(g, 700, 512).to(dt), _randn(g, 256, 512).to(dt), _randn(g, 256).to(dt)
    cos, sin = _tables(g, (700,), 128)
    W = ops.mxfp4_quantize(w)
    want = ops.mxfp4_linear(x0, W, b)
    wq = ops.rotary(want.view(700, 2, 128), None, cos, sin)[0]
    torch.cuda.synchronize(dev)
    side = torch.cuda.Stream(dev)
    for _ in range(3):
        x = torch.zeros_like(x0)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            x.copy_(x0)
        y = ops.mxfp4_linear(x, W, b, stream=side)
        q = ops.rotary(y.view(700, 2, 128), None, cos, sin, stream=side)[0]
        v = ops.mxfp4_dequantize(ops.mxfp4_quantize(x, stream=side), stream=side)
        side.synchronize()
        assert torch.equal(y, want) and torch.equal(q, wq) and _same(v.double(), mx_ref(x0))


@pytest.mark.gpu
def test_the_chain_captured_and_replayed(dev):
    """Tables, quantisation, products, norm and rotation in two graphs that share
    a workspace, replayed in turn with new inputs and eager work between."""
    g, dt = _gen(dev, 12), torch.bfloat16
    N, K, H = 96, 512, 4
    W = [ops.mxfp4_quantize(_randn(g, H * 64, K).to(dt)) for _ in range(2)]
    wn = (1 + 0.1 * _randn(g, H * 64)).to(dt)
    fr = ops.rotary_frequencies(64, device=dev)
    x = _randn(g, N, K).to(dt)
    pos = torch.arange(N, device=dev)
    ws = torch.empty(ops.mxfp4_linear_ws_bytes(N, H * 64, K), dtype=torch.uint8, device=dev)

    def chain(i):
        cos, sin = ops.rotary_table(pos, fr)
        q = ops.mxfp4_linear(x, W[i], ws=ws).view(N, H, 64)
        k = ops.mxfp4_linear(ops.mxfp4_quantize(x), W[1 - i]).view(N, H, 64)
        return ops.rotary(q, k, cos, sin, norm="token", q_weight=wn, k_weight=wn)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        chain(0), chain(1)
    torch.cuda.current_stream(dev).wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(chain(i))
        graphs.append(gr)
    for r in range(4):
        x.copy_(_randn(g, N, K))
        pos.copy_(torch.randint(0, 5000, (N,), generator=g, device=dev))
        for i in range(2):
            graphs[i].replay()
            torch.cuda.synchronize(dev)
            want = chain(i)
            assert torch.equal(outs[i][0], want[0]) and torch.equal(outs[i][1], want[1]), (r, i)


@pytest.mark.gpu
def test_projection_to_attention_input(dev):
    """One block's way from the activations to the attention call: tables of a
    latent grid, x quantised once for three projections, norm and rotation,
    against the definitions in 64 bits on the same roundings."""
    g, dt = _gen(dev, 13), torch.bfloat16
    f, h, w = 3, 7, 9
    N, H, D, K = f * h * w, 6, 128, 768
    t = torch.arange(N, device=dev)
    pos = torch.stack((t // (h * w), t // w % h, t % w), -1)
    cos, sin = ops.rotary_table(pos, ops.rotary_frequencies((44, 42, 42), device=dev))
    x = _randn(g, 1, N, K).to(dt)
    wt = [(_randn(g, H * D, K) * K ** -0.5).to(dt) for _ in range(3)]
    bt = [_randn(g, H * D).to(dt) for _ in range(3)]
    nw = [(1 + 0.2 * _randn(g, H * D)).to(dt) for _ in range(2)]
    X = ops.mxfp4_quantize(x)
    q, k, v = (ops.mxfp4_linear(X, ops.mxfp4_quantize(wi), bi).view(1, N, H, D) for wi, bi in zip(wt, bt))
    for y, wi, bi in zip((q, k, v), wt, bt):
        _check_linear(y.view(N, -1), x[0], wi, bi, None)
    oq, ok = ops.rotary(q, k, cos, sin, norm="token", q_weight=nw[0], k_weight=nw[1])
    _check_rotary(oq, q, cos, sin, "interleaved", False, "token", nw[0])
    _check_rotary(ok, k, cos, sin, "interleaved", False, "token", nw[1])
