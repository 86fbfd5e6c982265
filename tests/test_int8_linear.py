"""8-bit linear layers: quantisation by rows, the values back and the product
against 64-bit forms of their definitions, and what the entry points refuse."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

from token2tile_amd import ops

F64 = torch.float64
HALF = {"bf16": torch.bfloat16, "fp16": torch.float16}
LOWEST = 2.0 ** -120


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def _half_step(ref, dt):
    fi = torch.finfo(dt)
    return (ref.abs() * (fi.eps / 2)).clamp(min=fi.smallest_normal * fi.eps / 2)


def i8_ref(x):
    """(codes, scales) in 64 bits: the scale rounded to fp32, the exact quotient to
    the nearest whole number, the even one on ties (a quotient of 11 by 24 bits that
    is no tie is at least 2^-36 away from one, so 64 bits decide it)."""
    x = x.double()
    bad = ~torch.isfinite(x).all(-1)
    s = (x.abs().amax(-1) / 127).float().double().clamp(min=LOWEST)
    t = x / s[:, None]
    low = t.floor()
    n = low + ((t - low > 0.5) | ((t - low == 0.5) & (low % 2 != 0)))
    n[bad] = 0
    s[bad] = math.nan
    return n, s


def _check_codes(t, x):
    n, s = i8_ref(x)
    M, K = x.shape
    assert t.shape == (M, K) and torch.equal(t.scales.double().nan_to_num(-1.0), s.nan_to_num(-1.0))
    wide = _rows(t)
    assert torch.equal(wide[:M, :K].double(), n) and not bool(wide[:M, K:].any())
    assert torch.equal(t.to_codes(), wide[:M, :K])


def _rows(t):
    """All codes of a matrix in rows, by the layout's definition: chunk c of row r at
    place c ^ ((r >> 2) & 3) of its block of 16 rows x 64 columns."""
    M, K = -(-t.rows // 16) * 16, -(-t.cols // 128) * 128
    r, c = torch.arange(M)[:, None], torch.arange(K)[None]
    at = ((r // 16 * (K // 64) + c // 64) * 16 + r % 16) * 64 + ((c // 16 % 4) ^ (r // 4 % 4)) * 16 + c % 16
    return t.codes[at.to(t.codes.device)]


# ---------------------------------------------------------------------------
# refusals before any launch
# ---------------------------------------------------------------------------
def test_entries_reject_bad_arguments():
    from token2tile_amd import _lib
    L = _lib.lib()
    p, odd = ctypes.c_void_p(32), ctypes.c_void_p(40)
    bytes_of = L.t2t_int8_code_bytes
    assert [bytes_of(1, k) for k in (0, 1, 128, 129, 131071, 131072)] == [0, 2048, 2048, 4096, 16 * 131072, 0]
    assert [bytes_of(m, 100) for m in (-1, 0, 16, 17)] == [0, 0, 2048, 4096]

    def quant(x=p, dtype=1, stride=300, codes=p, scales=p, M=4, K=300):
        return L.t2t_int8_quantize(x, dtype, stride, codes, scales, M, K, None)
    assert quant(dtype=7) == 1 and quant(stride=299) == 1 and quant(codes=odd) == 1 and quant(scales=ctypes.c_void_p(6)) == 1
    assert quant(K=0) == 1 and quant(K=1 << 17, stride=1 << 17) == 1
    assert quant(M=-1) == 1 and quant(M=(1 << 30) + 1) == 1
    assert quant(scales=None) == 1 and b"null" in L.t2t_last_error() and quant(x=None) == 1
    assert quant(M=0, x=None) == 0

    def deq(dtype=1, stride=300, out=p, codes=p):
        return L.t2t_int8_dequantize(codes, p, out, dtype, stride, 4, 300, None)
    assert deq(dtype=2) == 1 and deq(stride=299) == 1 and deq(out=None) == 1 and deq(codes=odd) == 1

    def prod(a=p, w=p, act=0, out=p, dtype=1, ldo=40, M=4, N=40, K=300):
        return L.t2t_int8_product(a, p, w, p, None, act, out, dtype, ldo, M, N, K, None)
    assert prod(act=2) == 1 and prod(dtype=3) == 1 and prod(ldo=39) == 1 and prod(N=0) == 1 and prod(w=None) == 1
    assert prod(a=odd) == 1 and prod(w=odd) == 1 and prod(out=None) == 1
    assert prod(M=0, a=None, out=None) == 0

    def lin(ws=p, nb=1 << 20, M=40, K=300, x=p):
        return L.t2t_int8_linear(x, 1, 300, p, p, None, 0, p, 40, M, 40, K, ws, nb, None)
    assert lin(ws=None) == 2 and lin(nb=100) == 2 and b"workspace" in L.t2t_last_error()
    assert lin(ws=odd) == 1 and lin(x=None) == 1 and lin(M=0, ws=None) == 0


@pytest.mark.parametrize("step", [(1, 0), (0, 1), (3, 2)])
def test_the_workspace_never_falls(step):
    from token2tile_amd import _lib
    L = _lib.lib()
    last = 0
    for i in range(1, 3000):
        now = L.t2t_int8_linear_ws_bytes(1 + 13 * step[0] * i, 5120, 32 + 20 * step[1] * i)
        assert now >= last
        last = now


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for f in (lambda: ops.int8_quantize(x), lambda: ops.int8_linear(x, x), lambda: ops.int8_dequantize(x),
              lambda: ops.Int8.from_codes(torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4))):
        with pytest.raises(ValueError, match="t2t"):
            f()


@pytest.fixture
def launches(monkeypatch):
    """CPU tensors in the place of GPU ones; the launches, which are not made."""
    seen = []
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(ops, "_launch", lambda name, dev, stream, tensors, *a: seen.append((name, tensors, a)))
    return seen


def _cpu(rows, cols, fill=3):
    n = -(-rows // 16) * 16 * (-(-cols // 128) * 128)
    return ops.Int8(torch.full((n,), fill, dtype=torch.int8), torch.ones(rows), rows, cols)


@pytest.mark.parametrize("how", ["copy", "deepcopy", "pickle"])
def test_a_copied_matrix_is_read_at_its_own_address(launches, how):
    W = _cpu(40, 100)
    c = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda t: pickle.loads(pickle.dumps(t))}[how](W)
    assert c.shape == (40, 100) and (c.codes.data_ptr() == W.codes.data_ptr()) == (how == "copy")
    x = torch.zeros(40, 100, dtype=torch.bfloat16)
    ops.int8_dequantize(c)
    ops.int8_quantize(x, out=c)
    ops.int8_linear(x, c)
    ops.int8_linear(c, c)
    mine = [c.codes.data_ptr(), c.scales.data_ptr()]
    at = {"t2t_int8_dequantize": [0], "t2t_int8_quantize": [3], "t2t_int8_linear": [3], "t2t_int8_product": [0, 2]}
    assert [name for name, _, _ in launches] == list(at)
    for name, _, args in launches:
        for i in at[name]:
            assert list(args[i:i + 2]) == mine, name


def test_every_tensor_of_a_call_is_recorded_on_its_stream(launches):
    M, K, N, dt = 50, 100, 40, torch.bfloat16
    W, x, b, out = _cpu(N, K), torch.zeros(M, K, dtype=dt), torch.zeros(N, dtype=dt), torch.zeros(M, N, dtype=dt)
    ws = torch.empty(ops.int8_linear_ws_bytes(M, N, K) + 64, dtype=torch.uint8)
    ops.int8_linear(x, W, b, out=out, ws=ws, stream=type("S", (), {"device": x.device})())
    (_, tensors, args), = launches
    assert ws.data_ptr() in args
    for t in (x, W.codes, W.scales, b, out, ws):
        assert any(u is t for u in tensors)


@pytest.mark.parametrize("bad", ["k", "type", "stride", "none", "bias", "bias_type", "act", "dtype", "dtype_q", "out",
                                 "out_type", "out_twice", "weight", "ws", "out_q", "codes", "cols", "size", "scales",
                                 "scales_shape", "align", "rows", "code_type", "code_dim", "code_cols", "in_x", "in_w",
                                 "in_bias", "ws_x", "ws_out", "q_in_x", "d_in_codes", "apart"])
def test_refused(launches, bad):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    i8, f32 = torch.int8, torch.float32
    W, V, x = _cpu(40, 100), _cpu(10, 100), z(6, 100)
    buf = z(4000)
    big = torch.zeros(1 << 14, dtype=torch.uint8)
    calls = {
        "k": lambda: ops.int8_linear(z(6, 96), W),
        "type": lambda: ops.int8_quantize(z(6, 64, dtype=f32)),
        "stride": lambda: ops.int8_quantize(z(64, 6).t()),
        "none": lambda: ops.int8_quantize(z(6, 0)),
        "bias": lambda: ops.int8_linear(x, W, z(41)),
        "bias_type": lambda: ops.int8_linear(x, W, z(40, dtype=f32)),
        "act": lambda: ops.int8_linear(x, W, activation="relu"),
        "dtype": lambda: ops.int8_linear(x, W, dtype=torch.float16),
        "dtype_q": lambda: ops.int8_linear(W, W, dtype=f32),
        "out": lambda: ops.int8_linear(x, W, out=z(6, 41)),
        "out_type": lambda: ops.int8_linear(x, W, out=z(6, 40, dtype=torch.float16)),
        "out_twice": lambda: ops.int8_linear(x, W, out=z(1, 40).expand(6, 40)),
        "weight": lambda: ops.int8_linear(x, z(40, 100)),
        "ws": lambda: ops.int8_linear(x, W, ws=z(1 << 16)),
        "out_q": lambda: ops.int8_quantize(x, out=W),
        "codes": lambda: ops.Int8(z(2048), torch.zeros(4), 4, 100),
        "cols": lambda: ops.Int8(z(1 << 21, dtype=i8), torch.zeros(4), 4, 1 << 17),
        "size": lambda: ops.Int8(z(2048, dtype=i8), torch.zeros(4), 4, 129),
        "scales": lambda: ops.Int8(z(2048, dtype=i8), torch.zeros(4, dtype=F64), 4, 100),
        "scales_shape": lambda: ops.Int8(z(2048, dtype=i8), torch.zeros(4, 1), 4, 100),
        "align": lambda: ops.Int8(z(2056, dtype=i8)[8:], torch.zeros(4), 4, 100),
        "rows": lambda: ops.Int8(z(2048, dtype=i8), torch.zeros(4), -1, 100),
        "code_type": lambda: ops.Int8.from_codes(z(4, 100), torch.zeros(4)),
        "code_dim": lambda: ops.Int8.from_codes(z(400, dtype=i8), torch.zeros(4)),
        "code_cols": lambda: ops.Int8.from_codes(z(4, 0, dtype=i8), torch.zeros(4)),
        "in_x": lambda: ops.int8_linear(buf[:600].view(6, 100), W, out=buf[500:740].view(6, 40)),
        "in_w": lambda: ops.int8_linear(x, W, out=W.codes.view(torch.bfloat16)[:240].view(6, 40)),
        "in_bias": lambda: ops.int8_linear(x, W, buf[:40], out=buf[39:279].view(6, 40)),
        "ws_x": lambda: ops.int8_linear(big[:1800].view(torch.bfloat16).view(9, 100), W, ws=big[512:]),
        "ws_out": lambda: ops.int8_linear(z(9, 100), W, out=big[:720].view(torch.bfloat16).view(9, 40), ws=big[256:]),
        "q_in_x": lambda: ops.int8_quantize(
            buf[:256].view(2, 128), out=ops.Int8(buf[128:1152].view(i8), torch.zeros(2), 2, 128)),
        "d_in_codes": lambda: ops.int8_dequantize(V, out=V.codes.view(torch.bfloat16)[:1000].view(10, 100)),
        "apart": lambda: ops.Int8(big[:2048].view(i8), big[:16].view(f32), 4, 128)}
    with pytest.raises(ValueError, match="t2t"):
        calls[bad]()
    assert not launches


@pytest.mark.parametrize("scales", [None, [1.0] * 4, 1.0])
def test_scales_of_a_checkpoint_are_a_tensor(launches, scales):
    with pytest.raises(ValueError, match="t2t"):
        ops.Int8.from_codes(torch.zeros(4, 100, dtype=torch.int8), scales)
    W = ops.Int8.from_codes(torch.zeros(4, 100, dtype=torch.int8), torch.arange(8.0)[::2])  # (of any stride)
    assert W.scales.tolist() == [0.0, 2.0, 4.0, 6.0] and W.scales.is_contiguous()


# ---------------------------------------------------------------------------
# quantisation
# ---------------------------------------------------------------------------
# every count of values a thread, the borders between them, rows of one value and of odd widths
WIDTHS = [1, 2, 7, 8, 9, 127, 128, 129, 511, 513, 1023, 1531, 2048, 2049, 4096, 4097, 5120, 6145, 8192, 8200, 16385,
          32769, 131071]
MANY = [300, 1000, 1531, 2041, 5120, 16000]  # of rows enough that fewer threads take each


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("K", MANY)
def test_quantize_many_rows(dev, K, dt):
    g, dt, M = _gen(dev, K), HALF[dt], 1027
    x = (_randn(g, M, K) * torch.exp(2 * _randn(g, M, 1))).to(dt)
    x[5, K // 2] = math.inf
    t = ops.int8_quantize(x)
    few = ops.int8_quantize(x[1000:])
    assert bool(t.scales[5].isnan()) and not bool(t.to_codes()[5].any())
    assert torch.equal(t.to_codes()[1000:], few.to_codes()) and torch.equal(t.scales[1000:], few.scales)
    x[5] = 0
    t.scales[5] = 2.0 ** -120
    n, s = i8_ref(x)
    assert torch.equal(t.to_codes().double(), n) and torch.equal(t.scales.double(), s)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("K", WIDTHS)
def test_quantize(dev, K, dt):
    g, dt = _gen(dev, K), HALF[dt]
    M = 37 if K < 20000 else 5
    x = (_randn(g, M, K) * torch.exp(2 * _randn(g, M, 1))).to(dt)
    x[0] = 0
    t = ops.int8_quantize(x)
    _check_codes(t, x)
    v = ops.int8_dequantize(t, dt)
    n, s = i8_ref(x)
    # one fp32 product of 8 and 24 bits, rounded to the type
    ref = n * s[:, None]
    assert bool(((v.double() - ref).abs() <= _half_step(ref, dt) * (1 + 2.0 ** -12) + ref.abs() * 2.0 ** -24).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
def test_quantize_values_on_and_beside_the_borders(dev, dt):
    """Rows whose quotients are ties or the type's neighbours of ties, under scales
    that are powers of two and that are not."""
    dt = HALF[dt]
    n = torch.arange(-126.5, 127.0, 0.5, device=dev)
    rows = []
    for s in (1.0, 0.25, 2.0 ** -10, 3.0, 1.1, 0.0123, 7e-5):
        base = (n * s).to(dt)
        up = torch.nextafter(base, torch.full_like(base, math.inf))
        down = torch.nextafter(base, torch.full_like(base, -math.inf))
        top = torch.tensor([127.0 * s], device=dev).to(dt)
        rows += [torch.cat((t.clamp(-top, top), top)) for t in (base, up, down)]
    x = torch.stack(rows)
    _check_codes(ops.int8_quantize(x), x)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
def test_quantize_every_value(dev, dt):
    """All finite bit patterns, a binade of them a row: subnormal rows too."""
    dt = HALF[dt]
    x = torch.arange(-(1 << 15), 1 << 15, device=dev).to(torch.int16).view(dt)
    x = x[torch.isfinite(x)]
    order = x.double().abs().sort(stable=True).indices
    x = x[order][:x.numel() // 256 * 256].view(-1, 256)
    _check_codes(ops.int8_quantize(x), x)


@pytest.mark.gpu
def test_quantize_nonfinite_rows_views_and_buffers(dev):
    g, dt = _gen(dev, 5), torch.bfloat16
    big = _randn(g, 70, 3, 203).to(dt)
    x = big[:, 1, 2:202]                       # rows 609 apart, an odd address
    big[3, 1, 7], big[9, 1, 100], big[11, 1, 201] = math.inf, math.nan, -math.inf
    t = ops.int8_quantize(x)
    _check_codes(t, x)
    assert bool(t.scales[[3, 9, 11]].isnan().all()) and bool(ops.int8_dequantize(t)[9].isnan().all())
    # into a caller's matrix: rows behind the last stay as they were; values into a strided view
    out = ops.Int8(torch.full((80 * 256,), 9, device=dev, dtype=torch.int8), torch.empty(70, device=dev), 70, 200)
    assert ops.int8_quantize(x, out=out) is out
    _check_codes(out, x)
    assert bool((_rows(out)[70:] == 9).all()) and torch.equal(out.scales.nan_to_num(7), t.scales.nan_to_num(7))
    buf = torch.full((72, 301), 9.0, device=dev, dtype=dt)
    ops.int8_dequantize(t, out=buf[1:71, 5:205])
    assert torch.equal(buf[1:71, 5:205].nan_to_num(3), ops.int8_dequantize(t).nan_to_num(3))
    buf[1:71, 5:205] = 9.0
    assert bool((buf == 9.0).all())
    assert ops.int8_quantize(big[:0, 0]).shape == (0, 203)
    assert ops.int8_dequantize(ops.int8_quantize(big[:0, 0])).shape == (0, 203)
    assert ops.int8_quantize(big).shape == (210, 203) and ops.int8_quantize(big[0, 0]).shape == (1, 203)


@pytest.mark.gpu
def test_quantize_more_rows_than_work_groups(dev):
    x = _randn(_gen(dev, 1), 1 << 20, 8).half()
    x = torch.cat((x, x, x, x, x[:37]))
    t = ops.int8_quantize(x)
    codes = t.to_codes()
    n, s = i8_ref(x[:1 << 20])
    for i in range(4):
        assert torch.equal(codes[i << 20:(i + 1) << 20].double(), n)
    assert torch.equal(codes[4 << 20:].double(), n[:37]) and torch.equal(t.scales[4 << 20:].double(), s[:37])


# ---------------------------------------------------------------------------
# linear layers
# ---------------------------------------------------------------------------
def _linear_ref(a, sa, w, sw, b, act):
    """(result, bound on the fp32 part) from codes and scales in 64 bits."""
    y = (a.double() @ w.double().t()) * sw.double() * sa.double()[:, None]
    # the exact sum to fp32 and two products (the second one's fused with the bias): one rounding each
    tol = 3 * 2.0 ** -24 * y.abs()
    if b is not None:
        y = y + b.double()
    tol = tol + 2.0 ** -24 * y.abs()
    if act:
        u = math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
        # |gelu'| <= 1.13; e^-2u is off by 2 |u| 2^-23 and a few roundings, y / (1 + e) by as much
        # where e counts: 2^-18 of |y| covers it
        tol = 1.13 * tol + 2.0 ** -18 * y.abs()
        y = 0.5 * y * (1 + torch.tanh(u))
    return y, tol


def _check_linear(got, x, W, b, act):
    """x: what came in (quantised here by the definition), or an Int8 matrix."""
    a, sa = (x.to_codes(), x.scales) if isinstance(x, ops.Int8) else i8_ref(x)
    ref, tol = _linear_ref(a, sa, W.to_codes(), W.scales, b, act)
    tol = tol + _half_step(ref, got.dtype) * (1 + 2.0 ** -7)
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


def _operands(dev, M, N, K, dt, seed):
    g = _gen(dev, seed)
    x = (_randn(g, M, K) * torch.exp(0.5 * _randn(g, K))).to(dt)
    return x, (_randn(g, N, K) * K ** -0.5).to(dt), _randn(g, N).to(dt)


SIZES = [(1, 1, 1), (1, 64, 64), (1, 5000, 33000), (3, 70, 10001), (8, 100, 4097), (9, 100, 4097), (1, 5120, 512), (2, 33, 95), (5, 96, 256), (16, 48, 1024), (17, 31, 300),
         (31, 100, 288), (32, 32, 1571), (33, 257, 512), (64, 640, 2048), (100, 72, 5120), (129, 130, 161),
         (257, 513, 256), (600, 1000, 321), (1000, 1536, 1536), (2049, 776, 64), (4099, 2041, 1571),
         (33, 20481, 256), (700, 1100, 512), (16385, 1030, 1057), (4100, 4200, 1024), (70000, 1025, 96),
         (3900, 4091, 1057), (3969, 4096, 320), (8000, 4060, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
@pytest.mark.parametrize("dt,bias", [("bf16", True), ("fp16", False)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(dev, M, N, K, dt, bias, act):
    dt = HALF[dt]
    x, w, b = _operands(dev, M, N, K, dt, M + N + K)
    b = b if bias else None
    W = ops.int8_quantize(w)
    y = ops.int8_linear(x, W, b, activation=act)
    assert y.shape == (M, N) and y.dtype == dt
    _check_linear(y, x, W, b, act)
    # an x that was quantised before: the same codes, the same bits
    assert torch.equal(ops.int8_linear(ops.int8_quantize(x), W, b, activation=act, dtype=dt), y)


# forms of every size of tile, ragged in both directions
TILES = [(3, 40, 96), (40, 100, 700), (1000, 1536, 512), (1000, 1531, 800), (4100, 4200, 1024), (4100, 4195, 1057),
         (3900, 4088, 512), (3969, 4091, 705)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt,act", [("bf16", "gelu_tanh"), ("fp16", None)])
@pytest.mark.parametrize("M,N,K", TILES)
def test_linear_into_views(dev, M, N, K, dt, act):
    """Outputs of any stride and address get the bits of a contiguous one, nothing
    around them is written, and what stands behind the last rows of the operands has
    no part."""
    dt = HALF[dt]
    x, w, b = _operands(dev, M, N, K, dt, M + N)
    W = ops.int8_quantize(w)
    y = ops.int8_linear(x, W, b, activation=act)
    _check_linear(y, x, W, b, act)
    X = ops.int8_quantize(x)
    assert torch.equal(ops.int8_linear(ops.int8_quantize(x), ops.Int8.from_codes(W.to_codes(), W.scales), b,
                                       activation=act, dtype=dt), y)
    full = []
    for t in (X, W):
        wide = _rows(t)
        wide[t.rows:] = 77
        codes = ops.Int8.from_codes(wide, torch.ones(wide.shape[0], device=dev)).codes
        full.append(ops.Int8(codes, t.scales, *t.shape))
    assert torch.equal(ops.int8_linear(*full, b, activation=act, dtype=dt), y)
    for off, width in ((16, N + 24 - N % 8), (4, N + 24 - N % 8), (8, N + 17 - N % 2), (3, N + 17 - N % 2)):
        buf = torch.full((M + 2, width), 5.0, device=dev, dtype=dt)
        out = buf[1:M + 1, off:off + N]
        for src in (x, X):
            assert ops.int8_linear(src, W, b, activation=act, dtype=dt, out=out) is out
            assert torch.equal(out, y), (off, width)
            out.fill_(5.0)
            assert bool((buf == 5.0).all()), (off, width)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", TILES)
def test_linear_of_nonfinite_rows(dev, M, N, K):
    """An inf or NaN turns its row (x) or column (weight) of the result to NaN and
    leaves the rest; a row of zeros gives the bias."""
    x, w, b = _operands(dev, M, N, K, torch.float16, 2)
    x[0] = 0
    clean = ops.int8_linear(x, ops.int8_quantize(w), b)
    assert torch.equal(clean[0], b)
    bad = torch.zeros(M, N, device=dev, dtype=torch.bool)
    for r in (7, N // 2, N - 1):
        w[r, 40] = math.inf
        bad[:, r] = True
    for r in {M // 2, M - 1}:
        x[r, -1] = math.nan
        bad[r] = True
    y = ops.int8_linear(x, ops.int8_quantize(w), b)
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], clean[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(2, 40), (40, 200), (600, 1000), (4100, 4200), (3900, 4090)])
def test_linear_of_the_longest_sums(dev, M, N):
    """Codes of the largest magnitude over the longest rows, -128 among them: the
    sums fill 31 bits and are exact."""
    K = 131071 if M < 1000 else 20001
    full = lambda n, code: torch.full((n, K), code, device=dev, dtype=torch.int8)  # noqa: E731
    ones = lambda n: torch.ones(n, device=dev)  # noqa: E731
    a = full(M, -128)
    a[1::2] = 127
    A = ops.Int8.from_codes(a, 2.0 ** -20 * ones(M))
    for code, values in ((-128, (16384, -16256)), (127, (-16256, 16129))):
        y = ops.int8_linear(A, ops.Int8.from_codes(full(N, code), ones(N)), dtype=torch.bfloat16)
        for i, v in enumerate(values):
            want = torch.tensor(float(v * K), dtype=F64).float().mul(2.0 ** -20).to(torch.bfloat16)
            assert bool((y[i::2] == want.to(dev)).all())


@pytest.mark.gpu
def test_linear_scales_of_every_size(dev):
    """Rows far apart in scale keep their bits: the result is the same times the
    power of two."""
    g, dt = _gen(dev, 6), torch.bfloat16
    x, w = _randn(g, 7, 300).to(dt), ops.int8_quantize(_randn(g, 70, 300).to(dt))
    y = ops.int8_linear(x, w)
    e = torch.tensor([-100.0, -60, -20, 0, 20, 60, 100], device=dev)
    z = ops.int8_linear((x.double() * torch.exp2(e.double())[:, None]).to(dt), w)
    assert torch.equal(z.double(), y.double() * torch.exp2(e.double())[:, None])


@pytest.mark.gpu
def test_linear_shapes(dev):
    g, dt = _gen(dev, 7), torch.bfloat16
    K, N = 200, 72
    big = _randn(g, 4, 3, 2, K).to(dt)
    W, b = ops.int8_quantize(_randn(g, N, K).to(dt)), _randn(g, N).to(dt)
    x = big[:, :, 1]
    y = ops.int8_linear(x, W, b)
    assert y.shape == (4, 3, N)
    _check_linear(y.view(-1, N), x.reshape(-1, K), W, b, None)
    assert torch.equal(ops.int8_linear(x[0, 0], W, b), y[0, 0]) and ops.int8_linear(x[:, :0], W, b).shape == (4, 0, N)
    assert ops.int8_linear(ops.int8_quantize(x), W).shape == (12, N)
    ws = torch.empty(ops.int8_linear_ws_bytes(12, N, K) + 100, dtype=torch.uint8, device=dev)
    assert torch.equal(ops.int8_linear(x, W, b, ws=ws), y)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", TILES)
def test_on_a_side_stream_and_captured(dev, M, N, K):
    """Two graphs that share a workspace, replayed in turn with new inputs and eager
    work on another stream between, against the eager results."""
    dt = torch.bfloat16
    x, w, b = _operands(dev, M, N, K, dt, 3)
    W = [ops.int8_quantize(w), ops.int8_quantize(w.flip(0))]
    ws = torch.empty(ops.int8_linear_ws_bytes(M, N, K), dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        for i in range(2):
            ops.int8_linear(x, W[i], b, ws=ws)
    torch.cuda.current_stream(dev).wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.int8_linear(x, W[i], b, activation="gelu_tanh", ws=ws))
        graphs.append(gr)
    for r in range(3):
        x.copy_(_randn(_gen(dev, r), M, K))
        side.wait_stream(torch.cuda.current_stream(dev))
        for i in range(2):
            graphs[i].replay()
            want = ops.int8_linear(x, W[i], b, activation="gelu_tanh", stream=side)
            torch.cuda.synchronize(dev)
            assert torch.equal(outs[i], want), (r, i)
