"""The DiT harness with MXFP4 linear layers and the fused norm and rotary
embedding: the blocks call the operators as documented, the defaults are what
they were, and the whole stack runs both ways."""
import copy
import io
import math

import pytest
import torch

from token2tile_amd import dit, ops

CFG = dict(blocks=2, hidden=768, heads=6, ffn=1056, context_tokens=40, grid=(3, 8, 10))


def _model(dev, seed=0, **kw):
    torch.manual_seed(seed)
    return dit.WanDiT(dit.DiTConfig(**CFG, **kw), sparse=False, device=dev)


def _inputs(dev, cfg):
    g = torch.Generator(device=dev).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=dev, dtype=torch.bfloat16)  # noqa: E731
    return r(1, cfg.tokens, cfg.hidden), 0.1 * r(1, cfg.hidden), r(1, cfg.context_tokens, cfg.hidden)


def test_defaults_are_the_plain_forms():
    cfg = dit.DiTConfig()
    assert not cfg.mxfp4 and not cfg.fused_rope
    torch.manual_seed(0)
    blk = dit.Block(dit.DiTConfig(blocks=1, hidden=256, heads=2, ffn=64, context_tokens=4, grid=(2, 3, 4)), 0)
    rope = dit.rope_tables(blk.cfg, "cpu")
    x = torch.randn(1, 24, 256)
    q, k, v = blk.qkv(x, rope)
    want = dit.apply_rope(dit.rms_norm(blk.q(x), blk.norm_q, 1e-6).view(1, 24, 2, 128), *rope)
    assert torch.equal(q, want) and torch.equal(v, blk.v(x).view(1, 24, 2, 128)) and k.shape == q.shape


def _layer(dev, dtype, bias, seed=0):
    torch.manual_seed(seed)
    return dit.MxFp4Linear(torch.nn.Linear(64, 40, bias=bias).to(dev, dtype))


@pytest.mark.parametrize("bias", [True, False])
def test_the_layer_is_a_module(monkeypatch, bias):
    """Its weight is saved, loaded, copied and moved with it, and its output's
    type follows the module's (CPU tensors in the place of GPU ones)."""
    seen = []
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(ops, "_launch", lambda name, dev, stream, tensors, *a: seen.append((name, a)))
    a, b = _layer("cpu", torch.float16, bias), _layer("cpu", torch.float16, bias)
    a.weight.codes.fill_(3), a.weight.scales.fill_(4)
    assert {t.data_ptr() for t in a.state_dict().values()} >= {a.weight.codes.data_ptr(), a.weight.scales.data_ptr()}
    b.load_state_dict(a.state_dict())
    c = copy.deepcopy(a)
    for m in (b, c):
        assert torch.equal(m.weight.codes, a.weight.codes) and torch.equal(m.weight.scales, a.weight.scales)
        assert m.weight.codes.data_ptr() != a.weight.codes.data_ptr() and m.weight.shape == (40, 64)
    X = ops.MxFp4(*(torch.zeros(n, dtype=torch.uint8) for n in ops._mx_bytes(6, 64)), 6, 64)
    assert a(X).dtype == torch.float16 and a.to(torch.bfloat16)(X).dtype == torch.bfloat16
    assert c(torch.zeros(2, 3, 64, dtype=torch.float16)).shape == (2, 3, 40)
    assert seen[-1][0] == "t2t_mxfp4_linear" and c.weight.codes.data_ptr() in seen[-1][1]
    c.to("meta")
    assert c.weight_codes.device.type == "meta" and c.weight_scales.device.type == "meta"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bias", [(torch.float16, False), (torch.bfloat16, True)])
def test_a_saved_and_moved_layer_gives_the_same(dev, dtype, bias):
    a, b = _layer(dev, dtype, bias), _layer(dev, dtype, bias, seed=1)
    x = torch.randn(2, 9, 64, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(dtype)
    want = a(x)
    assert a(ops.mxfp4_quantize(x)).dtype == dtype
    f = io.BytesIO()
    torch.save(a.state_dict(), f)
    f.seek(0)
    b.load_state_dict(torch.load(f, weights_only=True))
    c = copy.deepcopy(a)
    a.weight.codes.fill_(0)
    assert torch.equal(b(x), want) and torch.equal(c(x), want)
    c.cpu()
    with pytest.raises(ValueError, match="t2t"):
        c(x)
    assert torch.equal(c.to(dev)(x), want)


@pytest.mark.gpu
def test_fused_tables_equal_the_harness_tables(dev):
    cfg = dit.DiTConfig(**CFG)
    for a, b in zip(dit.rope_tables(cfg, dev), dit.rope_tables(dit.DiTConfig(**CFG, fused_rope=True), dev)):
        # two 64-bit angles, each rounded once to fp32 (half a step each)
        assert bool(((a - b).abs() <= a.abs() * 2.0 ** -23 + 1e-12).all())


@pytest.mark.gpu
def test_fused_rope_block(dev):
    """q and k of a block against the 64-bit norm and rotation of its own
    projections, one rounding."""
    model = _model(dev, fused_rope=True)
    blk = model.blocks[0]
    x, _, _ = _inputs(dev, model.cfg)
    with torch.no_grad():
        q, k, v = blk.qkv(x, model.rope)
        cos, sin = (t.double()[None, :, None] for t in model.rope)
        for y, lin, w in ((q, blk.q, blk.norm_q), (k, blk.k, blk.norm_k)):
            f = lin(x).double()
            f = (f / (f.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()).view(y.shape)
            a, b = f[..., 0::2], f[..., 1::2]
            ref = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
            # a bf16 rounding of the result, fp32 inside (2^-17 of the pair)
            mag = torch.stack((a.abs() + b.abs(),) * 2, -1).flatten(-2)
            assert bool(((y.double() - ref).abs() <= ref.abs() * 2.0 ** -8 + 2.0 ** -17 * mag).all())
        assert torch.equal(v, blk.v(x).view(v.shape))


@pytest.mark.gpu
def test_mxfp4_block_calls(dev):
    """The quantised block's layers are the operators on the model's weights."""
    plain, model = _model(dev), _model(dev, mxfp4=True)
    x, _, ctx = _inputs(dev, model.cfg)
    with torch.no_grad():
        for name in ("q", "k", "v", "o", "cq", "ck", "cv", "co", "ffn1", "ffn2"):
            lin, mx = getattr(plain.blocks[1], name), getattr(model.blocks[1], name)
            assert isinstance(mx, dit.MxFp4Linear) and mx.weight.shape == tuple(lin.weight.shape)
            assert torch.equal(ops.mxfp4_dequantize(mx.weight),
                               ops.mxfp4_dequantize(ops.mxfp4_quantize(lin.weight.detach())))
        blk = model.blocks[1]
        q, k, v = blk.qkv(x, model.rope)
        assert torch.equal(v, blk.v(x).view(v.shape))           # shared or own quantisation: the same
        f = dit.rms_norm(blk.q(x), blk.norm_q, model.cfg.eps).view(q.shape)
        assert torch.equal(q, dit.apply_rope(f, *model.rope))


LAYERS = ("q", "k", "v", "o", "cq", "ck", "cv", "co", "ffn1", "ffn2")


def _check_layer(layer, x, got, gelu=False):
    """A layer's output against the values of its weight and input in 64 bits."""
    if not isinstance(x, ops.MxFp4):
        x = ops.mxfp4_quantize(x)
    a, w = ops.mxfp4_dequantize(x).double(), ops.mxfp4_dequantize(layer.weight).double()
    b = layer.bias.double()
    y, mag = a @ w.t() + b, a.abs() @ w.abs().t() + b.abs()
    # fp32 sums: chains of at most K / 32 + 64 additions, 2^-23 of the terms' magnitudes each; the
    # activation (slope up to 1.13) adds 2^-18 of its argument; one rounding to bf16
    tol = (x.cols / 32 + 64) * 2.0 ** -23 * mag
    if gelu:
        u = math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
        tol, y = 1.13 * tol + 2.0 ** -18 * y.abs(), 0.5 * y * (1 + torch.tanh(u))
    tol = tol + y.abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + 1e-30
    assert bool(((got.double().view(y.shape) - y).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
def test_every_layer_of_a_quantised_block(dev, fused):
    """Each linear layer is called once, on what the block's definition makes of
    the layers before it (bit for bit), gives the product of its own weight, and
    the block's output is the sum of all three parts."""
    model = _model(dev, mxfp4=True, fused_rope=fused)
    blk, cfg = model.blocks[1], model.cfg
    x, t, ctx = _inputs(dev, cfg)
    B, N, D = x.shape
    calls = {n: [] for n in LAYERS}
    for n in LAYERS:   # (outputs as they were: the fused rotation works in place)
        getattr(blk, n).register_forward_hook(lambda m, a, y, n=n: calls[n].append((a[0], y.clone())))
    with torch.no_grad():
        out = blk(x, t, ctx, model.rope, None)
        assert all(len(c) == 1 for c in calls.values())
        src, y = ({n: c[0][i] for n, c in calls.items()} for i in range(2))
        for n in LAYERS:
            _check_layer(getattr(blk, n), src[n], y[n], gelu=n == "ffn1")

        def quantised(n, want):
            q = ops.mxfp4_quantize(want)
            assert torch.equal(src[n].codes, q.codes) and torch.equal(src[n].scales, q.scales), n

        heads = lambda z: z.reshape(B, -1, cfg.heads, cfg.head_dim)  # noqa: E731
        attend = lambda q, k, v: torch.nn.functional.scaled_dot_product_attention(  # noqa: E731
            q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)).transpose(1, 2).reshape(B, N, D)
        e = (blk.modulation + t[:, None, :]).chunk(6, dim=1)
        h = torch.nn.functional.layer_norm(x, (D,), eps=cfg.eps) * (1 + e[1]) + e[0]
        for n in "qkv":
            quantised(n, h)
        if fused:
            q, k = ops.rotary(heads(y["q"]), heads(y["k"]), *model.rope, norm="token", q_weight=blk.norm_q,
                              k_weight=blk.norm_k, eps=cfg.eps)
        else:
            q, k = (dit.apply_rope(heads(dit.rms_norm(z, g, cfg.eps)), *model.rope)
                    for z, g in ((y["q"], blk.norm_q), (y["k"], blk.norm_k)))
        assert torch.equal(src["o"], attend(q, k, heads(y["v"])))
        x1 = x + y["o"] * e[2]
        assert torch.equal(src["cq"], blk.norm3(x1))
        for n in ("ck", "cv"):
            quantised(n, ctx)
        q, k = (heads(dit.rms_norm(z, g, cfg.eps)) for z, g in ((y["cq"], blk.cnorm_q), (y["ck"], blk.cnorm_k)))
        assert torch.equal(src["co"], attend(q, k, heads(y["cv"])))
        x2 = x1 + y["co"]
        assert torch.equal(src["ffn1"],
                           torch.nn.functional.layer_norm(x2, (D,), eps=cfg.eps) * (1 + e[4]) + e[3])
        assert torch.equal(src["ffn2"], y["ffn1"])
        assert torch.equal(out, x2 + y["ffn2"] * e[5])
        # every part counts: none is lost in the residual's rounding
        for part in (y["o"] * e[2], y["co"], y["ffn2"] * e[5]):
            assert float(part.float().norm()) > 2.0 ** -8 * float(x.float().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(fused_rope=True), dict(mxfp4=True), dict(mxfp4=True, fused_rope=True)])
def test_stack_runs(dev, kw):
    plain, model = _model(dev), _model(dev, **kw)
    args = _inputs(dev, model.cfg)
    y, z = plain(*args), model(*args)
    assert z.shape == y.shape and z.dtype == y.dtype and bool(torch.isfinite(z).all())
    assert torch.equal(model(*args), z)
    c = torch.nn.functional.cosine_similarity(y.float().flatten(), z.float().flatten(), dim=0)
    assert c > (0.9 if kw.get("mxfp4") else 0.99)


@pytest.mark.gpu
def test_sparse_attention_takes_the_fused_rows(dev):
    """The chain into the sparse attention call: MXFP4 projections, fused norm
    and rotation, the T2T backend's rebuilding and reuse steps."""
    cfg = dit.DiTConfig(blocks=1, hidden=12 * 128, heads=12, ffn=2048, context_tokens=64, grid=(4, 32, 32),
                        mxfp4=True, fused_rope=True)
    budget = dict(ns_base=4096, dense_prefix_steps=1, cq=32, ck=2048, step_profile=(1.0,) * 4,
                  layer_profile=(1.0,) * 6, cfg_mult=(1.0, 1.0))
    from token2tile_amd.backend.t2t_attn import T2TAttentionMetadataBuilder, T2TRequestCache
    torch.manual_seed(0)
    model = dit.WanDiT(cfg, sparse=True, device=dev)
    x, t, ctx = _inputs(dev, cfg)
    b, cache = T2TAttentionMetadataBuilder(), T2TRequestCache()
    outs = []
    for step in range(3):
        md = b.build(step_index=step, total_steps=50, cache=cache, profile_name="manual", **budget)
        outs.append(model(x, t, ctx, lambda i, m=md: m).float())
    # a budget of every key: the sparse steps are dense attention up to bf16 roundings of its output
    # (2^-8 of it twice), which the block's MXFP4 layers then carry on
    for y in outs[1:]:
        assert bool(torch.isfinite(y).all())
        assert torch.nn.functional.cosine_similarity(y.flatten(), outs[0].flatten(), dim=0) > 0.99
    assert math.isfinite(float(outs[0].abs().max()))
