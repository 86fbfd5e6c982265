"""The DiT harness with 8-bit linear layers and generation chunk by chunk: the
blocks call the operators as documented and the whole stack runs both ways."""
import copy
import math

import pytest
import torch

from token2tile_amd import dit, ops

CFG = dict(blocks=2, hidden=768, heads=6, ffn=1056, context_tokens=40, grid=(5, 8, 10))


def _model(dev, seed=0, **kw):
    torch.manual_seed(seed)
    return dit.WanDiT(dit.DiTConfig(**CFG, **kw), sparse=False, device=dev)


def _inputs(dev, cfg):
    g = torch.Generator(device=dev).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=dev, dtype=torch.bfloat16)  # noqa: E731
    return r(1, cfg.tokens, cfg.hidden), 0.1 * r(1, cfg.hidden), r(1, cfg.context_tokens, cfg.hidden)


def test_defaults_and_refusals(monkeypatch):
    assert not dit.DiTConfig().int8
    with pytest.raises(ValueError, match="not both"):
        dit.WanDiT(dit.DiTConfig(**CFG, int8=True, mxfp4=True), False, "cpu")
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    cfg = dit.DiTConfig(**CFG)
    c = dit.ChunkCache(cfg, "cpu", tokens=70, page_size=16)
    assert len(c.blocks) == 2 and c.blocks[0].shape == (5, 16, 6, 128) and c.table.tolist() == [[0, 1, 2, 3, 4]]
    for start, n in ((-1, 2), (0, 0), (0, 71), (70, 1), (60, 11)):
        with pytest.raises(ValueError, match="cache for 70"):
            c.at(start, n)
    c.at(66, 4)
    assert c.slots.tolist() == [66, 67, 68, 69] and c.lengths.tolist() == [70]


@pytest.mark.parametrize("bias", [True, False])
def test_the_layer_is_a_module(monkeypatch, bias):
    """Its weight is saved, loaded, copied and moved with it; a conversion changes
    its output's type and leaves the scales (CPU tensors in the place of GPU ones)."""
    seen = []
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(ops, "_launch", lambda name, dev, stream, tensors, *a: seen.append((name, a)))
    a, b = (dit.Int8Linear(torch.nn.Linear(64, 40, bias=bias).to(torch.float16)) for _ in range(2))
    a.weight.codes.fill_(3), a.weight.scales.fill_(1 + 2.0 ** -20)
    b.load_state_dict(a.state_dict())
    c = copy.deepcopy(a)
    for m in (b, c):
        assert torch.equal(m.weight.codes, a.weight.codes) and torch.equal(m.weight.scales, a.weight.scales)
        assert m.weight.codes.data_ptr() != a.weight.codes.data_ptr() and m.weight.shape == (40, 64)
    X = ops.Int8(torch.zeros(ops._i8_bytes(6, 64), dtype=torch.int8), torch.zeros(6), 6, 64)
    assert a(X).dtype == torch.float16 and a.to(torch.bfloat16)(X).dtype == torch.bfloat16
    assert a.weight.scales.dtype == torch.float32 and bool((a.weight.scales == 1 + 2.0 ** -20).all())
    assert c(torch.zeros(2, 3, 64, dtype=torch.float16), activation="gelu_tanh").shape == (2, 3, 40)
    assert seen[-1][0] == "t2t_int8_linear" and c.weight.codes.data_ptr() in seen[-1][1]
    c.to("meta")
    assert c.weight_codes.device.type == "meta" and c.weight_scales.device.type == "meta"


LAYERS = ("q", "k", "v", "o", "cq", "ck", "cv", "co", "ffn1", "ffn2")


def _check_layer(layer, x, got, gelu):
    """A layer's output against the values of its weight and input in 64 bits."""
    if isinstance(x, torch.Tensor):
        x = ops.int8_quantize(x)
    a, w = x.to_codes().double(), layer.weight.to_codes().double()
    y = (a @ w.t()) * x.scales.double()[:, None] * layer.weight.scales.double() + layer.bias.double()
    # exact sums; the scales' product, the sum's conversion and its scaling, the bias: half a step of fp32 each
    tol = 4 * 2.0 ** -24 * (y.abs() + layer.bias.double().abs())
    if gelu:  # (slope up to 1.13, 2^-18 of the argument)
        tol = 1.13 * tol + 2.0 ** -18 * y.abs()
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    tol = tol + y.abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + 1e-30
    assert bool(((got.double().view(y.shape) - y).abs() <= tol).all())


@pytest.mark.gpu
def test_every_layer_of_a_block_in_8_bits(dev):
    plain, model = _model(dev), _model(dev, int8=True)
    blk, was = model.blocks[1], plain.blocks[1]
    x, t, ctx = _inputs(dev, model.cfg)
    calls = {n: [] for n in LAYERS}
    for n in LAYERS:
        getattr(blk, n).register_forward_hook(lambda m, a, y, n=n: calls[n].append((a[0], y.clone())))
    with torch.no_grad():
        out = blk(x, t, ctx, model.rope, None)
        for n in LAYERS:
            layer, want = getattr(blk, n), ops.int8_quantize(getattr(was, n).weight.detach())
            assert isinstance(layer, dit.Int8Linear)
            assert torch.equal(layer.weight.codes, want.codes) and torch.equal(layer.weight.scales, want.scales)
            (src, y), = calls[n]
            _check_layer(layer, src, y, n == "ffn1")
        e = (blk.modulation + t[:, None, :]).chunk(6, dim=1)
        y = {n: c[0][1] for n, c in calls.items()}
        x2 = x + y["o"] * e[2] + y["co"]
        assert torch.equal(out, x2 + y["ffn2"] * e[5])
        for n in "qkv":  # one quantisation for the three
            assert calls[n][0][0] is calls["q"][0][0]


@pytest.mark.gpu
@pytest.mark.parametrize("chunks", [[2, 2, 1], [1, 4], [5]])
def test_attention_of_the_chunks(dev, chunks):
    """What every block's output layer gets is the attention in 64 bits of the chunk's
    queries over the keys and values of the chunks up to it."""
    model = _model(dev)
    cfg, frame = model.cfg, 80
    x, t, ctx = _inputs(dev, cfg)
    cache = dit.ChunkCache(cfg, dev, page_size=48)
    for c in cache.blocks:   # (what no chunk has written yet plays no part)
        c.k.fill_(math.nan), c.v.fill_(math.nan)
    calls = {}
    for i, blk in enumerate(model.blocks):
        for n in "qkvo":
            getattr(blk, n).register_forward_hook(
                lambda m, a, y, at=(i, n): calls.setdefault(at, []).append((a[0] if at[1] == "o" else y).clone()))
    start, outs = 0, []
    for n in chunks:
        outs.append(model.forward_chunk(x[:, start:start + n * frame], t, ctx, cache, start))
        start += n * frame
    heads = lambda y: y.view(-1, cfg.heads, cfg.head_dim)  # noqa: E731
    with torch.no_grad():
        for i, blk in enumerate(model.blocks):
            q, k, v, o = (heads(torch.cat(calls[i, n], 1)[0]) for n in "qkvo")
            q, k = ops.rotary(q, k, *model.rope, norm="token", q_weight=blk.norm_q, k_weight=blk.norm_k, eps=cfg.eps)
            own = cache.blocks[i]
            assert torch.equal(own.k.flatten(0, 1)[:cfg.tokens], k) and torch.equal(own.v.flatten(0, 1)[:cfg.tokens], v)
            at = 0
            for n in chunks:
                end = at + n * frame
                Q, K, V = (y.double().transpose(0, 1) for y in (q[at:end], k[:end], v[:end]))
                scale = cfg.head_dim ** -0.5
                s = Q @ K.transpose(1, 2) * scale
                p = s.softmax(-1)
                want = p @ V
                # scores: sums of 128 exact products in fp32, exponents at arguments of their size; weights rounded
                # to bf16 (half a step, 2^-8) and to fp32 in the sum; 400 additions at most; one rounding
                ds = Q.abs() @ K.abs().transpose(1, 2) * scale * 132 * 2.0 ** -24 + 2.0 ** -21 * s.abs().amax().clamp(min=1)
                w = p * (ds.exp() - 1 + 2.0 ** -8)
                tol = w @ V.abs() + w.sum(-1, keepdim=True) * want.abs()
                tol = tol + 105 * 2.0 ** -23 * (p @ V.abs() + want.abs()) + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -6)
                got = o[at:end].double().transpose(0, 1)
                assert bool(((got - want).abs() <= tol).all())
                at = end
    # a chunk again (the next step of its denoising) writes the same slots and gives the same
    start = (sum(chunks) - chunks[-1]) * frame
    assert torch.equal(model.forward_chunk(x[:, start:], t, ctx, cache, start), outs[-1])


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_one_chunk_is_the_whole_video(dev, int8):
    plain, model = _model(dev), _model(dev, int8=int8)
    args = _inputs(dev, model.cfg)
    y = plain(*args)
    z = model.forward_chunk(*args, dit.ChunkCache(model.cfg, dev), 0)
    assert z.shape == y.shape and z.dtype == y.dtype and bool(torch.isfinite(z).all())
    assert torch.nn.functional.cosine_similarity(y.float().flatten(), z.float().flatten(), dim=0) > 0.99
