"""Performance cases of the block operators around the attention call: the
rotary tables, the RMS norm and rotation of q and k, MXFP4 quantisation and
the MXFP4 linear layer.

With ``own`` false, ``run`` computes each operator in its plain form, out of
elementary torch operations; with ``own`` true it makes the calls of
``token2tile_amd.ops`` that ``token2tile_amd/dit.py`` makes.

``kind`` of a case:
  table     ``rotary_table``: cos / sin of a set of positions
  rotary    ``rotary``: q and k of one call, normed and rotated
  quantize  ``mxfp4_quantize`` and ``mxfp4_dequantize``: the values that the
            4-bit codes and their scales stand for
  linear    ``mxfp4_linear``: a 16-bit input, a weight kept in MXFP4
"""
import math

import torch

own = False

DEV = torch.device("cuda", 0)
F32, F64 = torch.float32, torch.float64
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
GRIDS = {75600: (21, 45, 80), 32760: (21, 30, 52)}  # latent frames x height x width


def _table(name, T, dims, scaling, last):
    """dims: channels per position axis, as text; last: the highest position
    (one axis; three axes take the positions of a latent grid of T tokens)."""
    return dict(name=name, kind="table", T=T, dims=dims, scaling=scaling, last=last)


def _rotary(name, B, N, HQ, HK, D, R, layout, norm, dtype="bf16", inverse=False):
    return dict(name=name, kind="rotary", B=B, N=N, HQ=HQ, HK=HK, D=D, R=R, layout=layout, norm=norm,
                dtype=dtype, inverse=inverse)


def _quantize(name, M, K, dtype="bf16"):
    return dict(name=name, kind="quantize", M=M, K=K, dtype=dtype)


def _linear(name, M, N, K, act="none", bias=True, dtype="bf16"):
    return dict(name=name, kind="linear", M=M, N=N, K=K, act=act, bias=bias, dtype=dtype)


def listed():
    return [
        # the tables of a 720p request: three position axes, built once a request
        _table("table_720p", 75600, "44,42,42", "none", 0),
        # a serving batch of single tokens far into a context stretched eightfold
        _table("table_tokens", 61, "128", "yarn", 262143),
        # a batch of four single tokens: all heads normed together, latency
        _rotary("rotary_token", 4, 1, 40, 40, 128, 128, "interleaved", "token"),
        # q and k of one 720p block, as the block stack makes them
        _rotary("rotary_720p", 1, 75600, 40, 40, 128, 128, "interleaved", "token"),
        # shared key heads, norm of each head, part of the head rotated, odd length
        _rotary("rotary_part", 2, 10007, 32, 8, 128, 96, "half", "head", "fp16"),
        # keys of a 480p call turned back: the rotation's transpose, no norm
        _rotary("rotary_back_480p", 1, 32760, 12, 12, 128, 128, "half", "none", "bf16", True),
        # the activations that enter the projections of a 720p block
        _quantize("quantize_720p", 75600, 5120),
        # ragged rows at the small model's width
        _quantize("quantize_odd", 4099, 1536, "fp16"),
        # one row through a projection: a single token, weight reading
        _linear("linear_token", 1, 5120, 5120),
        # keys of the text context: 512 tokens, a launch that fills the chip badly
        _linear("linear_context", 512, 5120, 5120),
        # ragged in every size, no bias
        _linear("linear_odd", 4099, 2041, 1568, "none", False, "fp16"),
        # the first feed-forward layer of a 720p block
        _linear("linear_ffn_720p", 75600, 13824, 5120, "gelu"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["table", "rotary", "rotary", "rotary", "quantize", "quantize", "linear", "linear",
                       "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        if kind == "table":
            if rng.random() < 0.4:
                T = rng.choice(sorted(GRIDS))
                d = rng.choice([64, 96, 128])
                dims = "%d,%d,%d" % (d - 4 * (d // 6), 2 * (d // 6), 2 * (d // 6))
                c = _table("", T, dims, "none", 0)
            else:
                c = _table("", _log(rng, 1, 75600), str(rng.choice([32, 64, 80, 96, 128])),
                           rng.choice(["none", "linear", "ntk", "yarn"]), _log(rng, 1000, 1 << 20))
        elif kind == "rotary":
            HQ = rng.choice([1, 2, 5, 7, 12, 16, 24, 32, 40])
            HK = rng.choice([HQ, max(1, HQ // 4), 1])
            D = rng.choice([64, 80, 96, 128, 128, 128, 256])
            R = rng.choice([D, D, D // 2])
            B = rng.choice([1, 1, 2, 3])
            N = _log(rng, 1, 75600)
            if B * N * (HQ + HK) * D > 75600 * 80 * 128:
                continue
            norm = rng.choice(["token", "token", "head", "none"])
            c = _rotary("", B, N, HQ, HK, D, R, rng.choice(["interleaved", "half"]), norm, dtype,
                        norm == "none" and rng.random() < 0.5)
        elif kind == "quantize":
            c = _quantize("", _log(rng, 1, 75600), 32 * _log(rng, 1, 160), dtype)
        else:
            M, N, K = _log(rng, 1, 75600), _log(rng, 64, 13824), 32 * _log(rng, 4, 432)
            if M * N * K > 75600 * 13824 * 5120:
                continue
            c = _linear("", M, N, K, rng.choice(["none", "gelu"]), rng.random() < 0.7, dtype)
        del c["name"]
        return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=F32)


def _activations(g, rows, cols, dt):
    """Rows whose channels have scales of their own, a few far above the rest."""
    scale = torch.exp(0.5 * _randn(g, cols))
    scale[torch.randint(0, cols, (max(1, cols // 256),), generator=g, device=DEV)] *= 20.0
    return _randn(g, rows, cols).mul_(scale).to(dt)


def _positions(case, g):
    dims = case["dims"].split(",")
    if len(dims) == 1:
        return torch.randint(0, case["last"] + 1, (case["T"],), generator=g, device=DEV)
    f, h, w = GRIDS[case["T"]]
    t = torch.arange(f * h * w, device=DEV)
    start = torch.randint(0, 64, (1,), generator=g, device=DEV)  # a window of a longer video
    return torch.stack((t // (h * w) + start, t // w % h, t % w), dim=-1)


def _frequencies(case):
    """Frequencies [R / 2] in 64 bits and the factor of cos and sin."""
    base, out, factor = 10000.0, [], 1.0
    for d in map(int, case["dims"].split(",")):
        s, L = 8.0, 32768
        f = [base ** (-2.0 * i / d) for i in range(d // 2)]
        if case["scaling"] == "linear":
            f = [x / s for x in f]
        elif case["scaling"] == "ntk":
            b = base * s ** (d / (d - 2.0))
            f = [b ** (-2.0 * i / d) for i in range(d // 2)]
        elif case["scaling"] == "yarn":
            at = [d * math.log(L / (2 * math.pi * b)) / (2 * math.log(base)) for b in (32.0, 1.0)]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
            r = [min(max((i - lo) / ((hi - lo) or 0.001), 0.0), 1.0) for i in range(d // 2)]
            f = [x * y / s + x * (1.0 - y) for x, y in zip(f, r)]
            factor = 0.1 * math.log(s) + 1.0
        out += f
    return torch.tensor(out, dtype=F64, device=DEV), factor


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    if case["kind"] == "table":
        st["pos"] = _positions(case, g)
        if own:
            from token2tile_amd import ops
            scaling = None
            if case["scaling"] != "none":
                scaling = ops.RotaryScaling(case["scaling"], 8.0, 32768)
            dims = tuple(map(int, case["dims"].split(",")))
            st["freqs"] = ops.rotary_frequencies(dims if len(dims) > 1 else dims[0], base=10000.0,
                                                 scaling=scaling, device=DEV)
        else:
            st["freqs"] = _frequencies(case)
        return st
    dt = DT[case["dtype"]]
    if case["kind"] == "rotary":
        B, N, D, R = case["B"], case["N"], case["D"], case["R"]
        for x, H in (("q", case["HQ"]), ("k", case["HK"])):
            st[x] = _activations(g, B * N, H * D, dt).view(B, N, H, D)
            if case["norm"] != "none":
                n = H * D if case["norm"] == "token" else D
                st["w" + x] = (1.0 + 0.2 * _randn(g, n)).to(dt)
        # consecutive positions of each sequence, one starting point a sequence
        pos = torch.randint(0, 4096, (B, 1), generator=g, device=DEV) + torch.arange(N, device=DEV)
        freq = 10000.0 ** (-2.0 * torch.arange(R // 2, device=DEV, dtype=F64) / R)
        ang = pos[..., None].double() * freq
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
    elif case["kind"] == "quantize":
        st["x"] = _activations(g, case["M"], case["K"], dt)
    else:
        M, N, K = case["M"], case["N"], case["K"]
        st["x"] = _activations(g, M, K, dt)
        w = (_randn(g, N, K) * K ** -0.5).to(dt)
        st["b"] = (0.1 * _randn(g, N)).to(dt) if case["bias"] else None
        if own:  # a program keeps its weights in MXFP4 ...
            from token2tile_amd import ops
            st["w"] = ops.mxfp4_quantize(w)
        else:    # ... or the 16-bit values that those stand for
            st["w"] = _values(w).to(dt)
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _values(x):
    """The values in 32 bits that MXFP4 holds for x [M, K]: blocks of 32, a
    power of two that brings the largest magnitude to [4, 8), each quotient
    rounded to 0, .5, 1, 1.5, 2, 3, 4 or 6, ties to the even code."""
    M, K = x.shape
    y = x.float().view(M, K // 32, 32)
    top = y.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top)[1] - 3).clamp_(min=-126)
    scale = torch.exp2(e.float())
    y = y / scale
    a = y.abs()
    v = 0.5 * (a > 0.25) + 0.5 * (a >= 0.75) + 0.5 * (a > 1.25) + 0.5 * (a >= 1.75)
    v += 1.0 * (a > 2.5) + 1.0 * (a >= 3.5)
    v += 2.0 * (a > 5.0)
    v = torch.where(y < 0, -v, v).mul_(scale)
    return torch.where(torch.isfinite(top), v, torch.full_like(v, math.nan)).view(M, K)


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))


def _turn(st, x, w, case):
    y = x.float()
    if case["norm"] == "token":
        f = y.flatten(2)
        y = (f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + EPS) * w.float()).view(y.shape)
    elif case["norm"] == "head":
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * w.float()
    R = case["R"]
    c, s = st["cos"][:, :, None], st["sin"][:, :, None]
    if case["inverse"]:
        s = -s
    r, rest = y[..., :R], y[..., R:]
    if case["layout"] == "half":
        a, b = r[..., :R // 2], r[..., R // 2:]
        r = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    return torch.cat((r, rest), dim=-1).to(x.dtype)


def _plain(st, case):
    if case["kind"] == "table":
        freq, factor = st["freqs"]
        dims = list(map(int, case["dims"].split(",")))
        pos = st["pos"][:, None] if len(dims) == 1 else st["pos"]
        axis = torch.cat([torch.full((d // 2,), a, device=DEV) for a, d in enumerate(dims)])
        ang = pos[:, axis].double() * freq
        return (factor * ang.cos()).float(), (factor * ang.sin()).float()
    if case["kind"] == "rotary":
        return _turn(st, st["q"], st.get("wq"), case), _turn(st, st["k"], st.get("wk"), case)
    if case["kind"] == "quantize":
        return _values(st["x"]).to(st["x"].dtype)
    y = torch.matmul(_values(st["x"]), st["w"].float().t())
    if st["b"] is not None:
        y += st["b"].float()
    if case["act"] == "gelu":
        y = _gelu(y)
    return y.to(st["x"].dtype)


def run(state):
    case = state["case"]
    if not own:
        return _plain(state, case)
    from token2tile_amd import ops
    if case["kind"] == "table":
        return ops.rotary_table(state["pos"], state["freqs"])
    if case["kind"] == "rotary":
        return ops.rotary(state["q"], state["k"], state["cos"], state["sin"], layout=case["layout"],
                          inverse=case["inverse"], norm=None if case["norm"] == "none" else case["norm"],
                          q_weight=state.get("wq"), k_weight=state.get("wk"), eps=EPS)
    if case["kind"] == "quantize":
        return ops.mxfp4_dequantize(ops.mxfp4_quantize(state["x"]), state["x"].dtype)
    return ops.mxfp4_linear(state["x"], state["w"], state["b"],
                            activation="gelu_tanh" if case["act"] == "gelu" else None)


# ---------------------------------------------------------------------------
# definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_mx(x):
    """Nearest of the eight magnitudes by distance, an even index on ties."""
    steps = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=F64, device=x.device)
    out = torch.empty(x.shape, dtype=F64, device=x.device)
    for r0 in range(0, x.shape[0], 8192):
        b = x[r0:r0 + 8192].double().unflatten(-1, (-1, 32))
        amax = b.abs().max(-1, keepdim=True).values
        e = torch.where(amax > 0, torch.floor(torch.log2(amax)), torch.full_like(amax, -1e9)) - 2.0
        s = torch.exp2(e.clamp(min=-126.0))  # exact, which pow(2, e) is not on the GPU
        t = (b.abs() / s).clamp(max=6.0)
        best, near = torch.zeros_like(t), t.clone()
        for i in range(1, 8):
            d = (t - steps[i]).abs()
            take = (d < near) | ((d == near) & (i % 2 == 0))
            best, near = torch.where(take, steps[i], best), torch.where(take, d, near)
        v = torch.copysign(best * s, b)
        v = v.masked_fill(~torch.isfinite(b).all(-1, keepdim=True), math.nan)
        out[r0:r0 + 8192] = v.flatten(-2)
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "table":
        dims = list(map(int, case["dims"].split(",")))
        freq, factor = st["freqs"]
        cos, sin, at = [], [], 0
        for a, d in enumerate(dims):
            p = (st["pos"] if len(dims) == 1 else st["pos"][:, a]).to(F64)
            turn = torch.outer(p, freq[at:at + d // 2])
            cos.append(torch.cos(turn) * factor)
            sin.append(torch.sin(turn) * factor)
            at += d // 2
        return torch.cat(cos, 1), torch.cat(sin, 1)
    if case["kind"] == "rotary":
        R, outs = case["R"], []
        phase = torch.complex(st["cos"].double(), st["sin"].double()).unsqueeze(2)
        if case["inverse"]:
            phase = phase.conj().resolve_conj()
        for name in ("q", "k"):
            x = st[name].to(F64)
            if case["norm"] != "none":
                w = st["w" + name].to(F64)
                over = (-2, -1) if case["norm"] == "token" else (-1,)
                x = x / torch.sqrt((x * x).mean(over, keepdim=True) + EPS)
                x *= w.view(x.shape[2:]) if case["norm"] == "token" else w
            i = torch.arange(R // 2, device=DEV)
            re, im = (i, i + R // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., re], x[..., im]) * phase
            x[..., re], x[..., im] = z.real, z.imag
            outs.append(x)
        return tuple(outs)
    if case["kind"] == "quantize":
        return _exact_mx(st["x"])
    if 2.0 * case["M"] * case["N"] * case["K"] > 2.2e13:
        return None
    y = _exact_mx(st["x"]) @ st["w"].to(F64).t()
    if st["b"] is not None:
        y += st["b"].to(F64)
    if case["act"] == "gelu":
        y *= 0.5 + 0.5 * torch.tanh(0.7978845608028654 * y * (1.0 + 0.044715 * y ** 2))
    return y


def work(case):
    if case["kind"] == "table":
        dims = list(map(int, case["dims"].split(",")))
        n = case["T"] * sum(dims) // 2
        return {"bytes": 8 * case["T"] * len(dims) + 4 * sum(dims) + 8 * n, "flops": 3 * n}
    if case["kind"] == "rotary":
        T, H = case["B"] * case["N"], case["HQ"] + case["HK"]
        n = T * H * case["D"]
        w = {"token": 2 * H * case["D"], "head": 4 * case["D"], "none": 0}[case["norm"]]
        return {"bytes": 4 * n + 4 * T * case["R"] + w,
                "flops": 3 * T * H * case["R"] + (4 * n if case["norm"] != "none" else 0)}
    if case["kind"] == "quantize":
        return {"bytes": 4 * case["M"] * case["K"], "flops": 2 * case["M"] * case["K"]}
    M, N, K = case["M"], case["N"], case["K"]
    return {"bytes": 2 * M * K + N * K // 2 + N * K // 32 + 2 * N * case["bias"] + 2 * M * N,
            "flops": 2 * M * N * K}
