"""Wan2.1-architecture DiT forward with the Token2Tile attention backend.

End-to-end harness for the operator: a diffusion transformer with the Wan2.1
block structure (adaLN modulation, q/k RMSNorm, 3-D rotary embedding,
cross-attention to a text context, GELU feed-forward) and random bf16 weights.
Its self-attention runs either dense (torch SDPA) or through
``token2tile_amd.backend.t2t_attn.T2TAttentionImpl`` with the backend's budget
profile, dense prefix and mask-refresh reuse, so one denoising step can be
timed both ways on the same weights and inputs.

With ``mxfp4`` the blocks' linear layers run on MXFP4 operands, with ``int8`` on
8-bit ones, and with ``fused_rope`` the RMSNorm and rotary embedding of q and k in
one launch.  A ``ChunkCache`` generates a video chunk by chunk: each chunk's tokens
attend to their own and the earlier chunks' keys in a paged cache.

``python -m token2tile_amd.dit`` prints one JSON line with the per-step times
at the Wan2.1-14B 720p shape (40 blocks, hidden 5120, 40 heads, FFN 13824,
75,600 latent tokens, 512 context tokens).
"""
from __future__ import annotations

import argparse
import json
import math
import sys
import time
from dataclasses import dataclass

import torch
import torch.nn.functional as F


@dataclass
class DiTConfig:
    """Block structure of Wan2.1-T2V-14B."""

    blocks: int = 40
    hidden: int = 5120
    heads: int = 40
    ffn: int = 13824
    context_tokens: int = 512
    grid: tuple[int, int, int] = (21, 45, 80)  # latent frames x height x width (720p)
    eps: float = 1e-6
    mxfp4: bool = False       # the blocks' linear layers in MXFP4 (ops.mxfp4_linear)
    int8: bool = False        # the blocks' linear layers in 8 bits (ops.int8_linear)
    fused_rope: bool = False  # q/k RMSNorm and rotary embedding in one launch (ops.rotary)

    @property
    def head_dim(self) -> int:
        return self.hidden // self.heads

    @property
    def tokens(self) -> int:
        f, h, w = self.grid
        return f * h * w


def rope_tables(cfg: DiTConfig, device) -> tuple[torch.Tensor, torch.Tensor]:
    """cos / sin [N, head_dim / 2] of the 3-D rotary embedding: the rotary
    pairs of a head are split between the frame, height and width positions
    (d - 4 (d // 6), 2 (d // 6), 2 (d // 6) channels, as in Wan2.1)."""
    d = cfg.head_dim
    parts = [d - 4 * (d // 6), 2 * (d // 6), 2 * (d // 6)]
    f, h, w = cfg.grid
    pos = torch.stack(torch.meshgrid(torch.arange(f), torch.arange(h), torch.arange(w),
                                     indexing="ij"), dim=-1).reshape(-1, 3).to(device)
    if cfg.fused_rope:
        from token2tile_amd import ops
        return ops.rotary_table(pos, ops.rotary_frequencies(parts, device=device))
    angles = []
    for axis, ch in enumerate(parts):
        inv = 1.0 / (10000.0 ** (torch.arange(0, ch, 2, device=device, dtype=torch.float64) / ch))
        angles.append(pos[:, axis:axis + 1].double() * inv[None])
    ang = torch.cat(angles, dim=1)                  # [N, d / 2]
    return ang.cos().float(), ang.sin().float()


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [B, N, H, d]: rotate channel pairs (2i, 2i + 1) by the position angles."""
    xf = x.float().unflatten(-1, (-1, 2))
    x0, x1 = xf[..., 0], xf[..., 1]
    c, s = cos[None, :, None, :], sin[None, :, None, :]
    out = torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), dim=-1).flatten(-2)
    return out.to(x.dtype)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype) * weight


class _FewBitLinear(torch.nn.Module):
    """A linear layer whose weight is kept in fewer bits (its codes and scales are
    buffers: moved, copied, saved and loaded with the module); its input is
    quantised at the call, or comes as a matrix that several layers share (the
    output's leading dimensions are then flattened)."""

    def __init__(self, linear: torch.nn.Linear):
        super().__init__()
        w = self.quantize(linear.weight.detach())
        self.out_features, self.in_features = w.shape
        self.register_buffer("weight_codes", w.codes)
        self.register_buffer("weight_scales", w.scales)
        # of the outputs' type, which the module's conversions change with the bias
        self.register_buffer("_like", linear.weight.detach().new_empty(0), persistent=False)
        self.bias = linear.bias

    def _dtype(self, x):
        return None if isinstance(x, torch.Tensor) else self._like.dtype


class MxFp4Linear(_FewBitLinear):
    """In MXFP4, input and weight (``ops.MxFp4``)."""

    @staticmethod
    def quantize(x):
        from token2tile_amd import ops
        return ops.mxfp4_quantize(x)

    @property
    def weight(self):
        from token2tile_amd import ops
        return ops.MxFp4(self.weight_codes, self.weight_scales, self.out_features, self.in_features)

    def forward(self, x, activation=None):
        from token2tile_amd import ops
        return ops.mxfp4_linear(x, self.weight, self.bias, activation=activation, dtype=self._dtype(x))


class Int8Linear(_FewBitLinear):
    """In 8 bits, a scale for each token and channel (``ops.Int8``)."""

    def _apply(self, fn, *args, **kw):
        # conversions of the module to a 16-bit type leave the scales in 32 bits, as they are
        scales = self.weight_scales
        super()._apply(fn, *args, **kw)
        if self.weight_scales.dtype != scales.dtype:
            self.weight_scales = scales.to(self.weight_scales.device)
        return self

    @staticmethod
    def quantize(x):
        from token2tile_amd import ops
        return ops.int8_quantize(x)

    @property
    def weight(self):
        from token2tile_amd import ops
        return ops.Int8(self.weight_codes, self.weight_scales, self.out_features, self.in_features)

    def forward(self, x, activation=None):
        from token2tile_amd import ops
        return ops.int8_linear(x, self.weight, self.bias, activation=activation, dtype=self._dtype(x))


def _shared(x, layer):
    """x as ``layer`` and its neighbours take it: in few bits once for all of them."""
    return layer.quantize(x) if isinstance(layer, _FewBitLinear) else x


class ChunkCache:
    """The keys and values of a stack's self-attention for generation chunk by
    chunk: a paged cache for each block, with room for ``tokens`` (default: the
    configuration's), and the positions of the chunk at hand."""

    def __init__(self, cfg: DiTConfig, device, dtype=torch.bfloat16, tokens=None, page_size=64):
        from token2tile_amd import ops
        self.tokens = cfg.tokens if tokens is None else tokens
        pages = -(-self.tokens // page_size)
        self.blocks = []
        for _ in range(cfg.blocks):
            k, v = torch.zeros(2, pages, page_size, cfg.heads, cfg.head_dim, dtype=dtype, device=device)
            self.blocks.append(ops.PagedCache(k, v))
        self.table = torch.arange(pages, dtype=torch.int32, device=device)[None]
        self.slots = self.lengths = None

    def at(self, start, n):
        """Tokens ``start`` .. ``start + n - 1`` come next (again, at each step of a
        chunk's denoising): their slots are theirs, and they see all before them."""
        if not (0 <= start and 1 <= n and start + n <= self.tokens):
            raise ValueError(f"tokens {start} .. {start + n - 1} of a cache for {self.tokens}")
        dev = self.table.device
        self.slots = torch.arange(start, start + n, dtype=torch.int32, device=dev)
        self.lengths = torch.full((1,), start + n, dtype=torch.int32, device=dev)


class Block(torch.nn.Module):
    def __init__(self, cfg: DiTConfig, index: int, attn_impl=None):
        super().__init__()
        D, Fh = cfg.hidden, cfg.ffn
        self.cfg = cfg
        self.index = index
        self.modulation = torch.nn.Parameter(torch.randn(1, 6, D) / D ** 0.5)
        self.q = torch.nn.Linear(D, D)
        self.k = torch.nn.Linear(D, D)
        self.v = torch.nn.Linear(D, D)
        self.o = torch.nn.Linear(D, D)
        self.norm_q = torch.nn.Parameter(torch.ones(D))
        self.norm_k = torch.nn.Parameter(torch.ones(D))
        self.norm3 = torch.nn.LayerNorm(D, eps=cfg.eps)
        self.cq = torch.nn.Linear(D, D)
        self.ck = torch.nn.Linear(D, D)
        self.cv = torch.nn.Linear(D, D)
        self.co = torch.nn.Linear(D, D)
        self.cnorm_q = torch.nn.Parameter(torch.ones(D))
        self.cnorm_k = torch.nn.Parameter(torch.ones(D))
        self.ffn1 = torch.nn.Linear(D, Fh)
        self.ffn2 = torch.nn.Linear(Fh, D)
        self.attn_impl = attn_impl  # None: dense SDPA

    def quantize_(self, layer=MxFp4Linear):
        """The block's linear layers as ``layer``, in the place of the 16-bit ones."""
        for name in ("q", "k", "v", "o", "cq", "ck", "cv", "co", "ffn1", "ffn2"):
            setattr(self, name, layer(getattr(self, name)))

    def qkv(self, x, rope):
        """q, k (normed and rotated) and v [B, N, H, d] of the self-attention."""
        B, N, D = x.shape
        H, d = self.cfg.heads, self.cfg.head_dim
        x = _shared(x, self.q)
        q, k, v = self.q(x), self.k(x), self.v(x).view(B, N, H, d)
        if self.cfg.fused_rope:
            from token2tile_amd import ops
            q, k = q.view(B, N, H, d), k.view(B, N, H, d)
            q, k = ops.rotary(q, k, *rope, norm="token", q_weight=self.norm_q, k_weight=self.norm_k,
                              eps=self.cfg.eps, out=(q, k))
            return q, k, v
        q = rms_norm(q, self.norm_q, self.cfg.eps).view(B, N, H, d)
        k = rms_norm(k, self.norm_k, self.cfg.eps).view(B, N, H, d)
        return apply_rope(q, *rope), apply_rope(k, *rope), v

    def chunk_attention(self, x, rope, cache):
        """The self-attention of a chunk, behind the chunks that the cache holds."""
        from token2tile_amd import ops
        B, N, D = x.shape
        H, d = self.cfg.heads, self.cfg.head_dim
        x = _shared(x, self.q)
        q, k, v = (y(x).view(N, H, d) for y in (self.q, self.k, self.v))
        own = cache.blocks[self.index]
        q = ops.cache_append(q, k, v, *rope, own, cache.slots, norm="token", q_weight=self.norm_q,
                             k_weight=self.norm_k, eps=self.cfg.eps, out=q)
        o = ops.cache_attention(q.view(B, N, H, d), own, cache.table, cache.lengths)
        return self.o(o.view(B, N, D))

    def self_attention(self, x, rope, attn_metadata):
        B, N, D = x.shape
        q, k, v = self.qkv(x, rope)
        if self.attn_impl is None:
            o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2),
                                               v.transpose(1, 2)).transpose(1, 2)
        else:
            o = self.attn_impl.forward(q, k, v, attn_metadata)
        return self.o(o.reshape(B, N, D))

    def cross_attention(self, x, ctx):
        B, N, D = x.shape
        H, d = self.cfg.heads, self.cfg.head_dim
        q = rms_norm(self.cq(x), self.cnorm_q, self.cfg.eps).view(B, N, H, d).transpose(1, 2)
        ctx = _shared(ctx, self.ck)
        k = rms_norm(self.ck(ctx), self.cnorm_k, self.cfg.eps).view(B, -1, H, d).transpose(1, 2)
        v = self.cv(ctx).view(B, -1, H, d).transpose(1, 2)
        o = F.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(B, N, D)
        return self.co(o)

    def forward(self, x, t_emb, ctx, rope, attn_metadata, cache=None):
        e = (self.modulation + t_emb[:, None, :]).chunk(6, dim=1)  # 6 x [B, 1, D]
        D = self.cfg.hidden
        h = F.layer_norm(x, (D,), eps=self.cfg.eps) * (1 + e[1]) + e[0]
        a = self.self_attention(h, rope, attn_metadata) if cache is None else self.chunk_attention(h, rope, cache)
        x = x + a * e[2]
        x = x + self.cross_attention(self.norm3(x), ctx)
        h = F.layer_norm(x, (D,), eps=self.cfg.eps) * (1 + e[4]) + e[3]
        if isinstance(self.ffn1, _FewBitLinear):
            y = self.ffn1(h, activation="gelu_tanh")
        else:
            y = F.gelu(self.ffn1(h), approximate="tanh")
        x = x + self.ffn2(y) * e[5]
        return x


class WanDiT(torch.nn.Module):
    """The block stack (patch embedding, time embedding MLP and the output
    head are outside the attention path and omitted; the latent enters as
    [1, N, hidden] tokens)."""

    def __init__(self, cfg: DiTConfig, sparse: bool, device, dtype=torch.bfloat16, tie=0.0):
        super().__init__()
        if cfg.mxfp4 and cfg.int8:
            raise ValueError("linear layers in MXFP4 or in 8 bits, not both")
        self.cfg = cfg
        impls = [None] * cfg.blocks
        if sparse:
            from token2tile_amd.backend.t2t_attn import T2TAttentionImpl
            impls = [T2TAttentionImpl(cfg.heads, cfg.head_dim, False, 1.0 / math.sqrt(cfg.head_dim),
                                      prefix=f"blocks.{i}.self_attn.attn") for i in range(cfg.blocks)]
        with torch.device(device):
            self.blocks = torch.nn.ModuleList(Block(cfg, i, impls[i]) for i in range(cfg.blocks))
        for m in self.modules():
            if isinstance(m, torch.nn.Linear):
                torch.nn.init.normal_(m.weight, std=m.in_features ** -0.5)
                torch.nn.init.zeros_(m.bias)
        if tie > 0:
            # self-attention key weights tied to the query weights (same scale):
            # W_k = tie W_q + sqrt(1 - tie^2) W_k, so q_i . k_j is large for
            # similar tokens and attention follows the latent's structure
            with torch.no_grad():
                for blk in self.blocks:
                    blk.k.weight.mul_(math.sqrt(1.0 - tie * tie)).add_(tie * blk.q.weight)
        self.to(dtype)
        if cfg.mxfp4 or cfg.int8:
            for blk in self.blocks:
                blk.quantize_(MxFp4Linear if cfg.mxfp4 else Int8Linear)
        self.rope = rope_tables(cfg, device)

    @torch.no_grad()
    def forward(self, x, t_emb, ctx, metadata_for_layer=None):
        for blk in self.blocks:
            md = metadata_for_layer(blk.index) if metadata_for_layer is not None else None
            x = blk(x, t_emb, ctx, self.rope, md)
        return x

    @torch.no_grad()
    def forward_chunk(self, x, t_emb, ctx, cache: ChunkCache, start):
        """Tokens ``start`` .. of the video (x [1, n, hidden]; by whole frames, for
        chunks that see all of themselves) behind those the cache holds."""
        n = x.shape[1]
        cache.at(start, n)
        rope = tuple(t[start:start + n] for t in self.rope)
        for blk in self.blocks:
            x = blk(x, t_emb, ctx, rope, None, cache)
        return x


def smooth_latent(cfg: DiTConfig, g, device, components=32, noise=0.3):
    """[1, N, hidden] tokens that vary smoothly over the (frame, height,
    width) grid: a sum of low-frequency plane waves, each along its own
    random direction of the hidden space, plus white noise."""
    f, h, w = cfg.grid
    pos = torch.stack(torch.meshgrid(torch.arange(f), torch.arange(h), torch.arange(w),
                                     indexing="ij"), dim=-1).reshape(-1, 3).to(device).float()
    pos = pos / torch.tensor([f, h, w], device=device, dtype=torch.float32)
    freq = 3.0 * torch.randn(3, components, generator=g, device=device)
    phase = 2 * math.pi * torch.rand(components, generator=g, device=device)
    dirs = torch.randn(components, cfg.hidden, generator=g, device=device)
    waves = torch.sin(2 * math.pi * pos @ freq + phase)                 # [N, components]
    x = waves @ dirs / math.sqrt(components)
    x += noise * torch.randn(x.shape, generator=g, device=device)
    return x[None].to(torch.bfloat16)


def run(cfg: DiTConfig, steps, device, *, sparse: bool, profile="auto", budget_kw=None, seed=0,
        structured=False):
    """Time one forward (one CFG branch) of the block stack per denoising step
    index in ``steps``; returns {step: ms}.  With ``sparse`` the self-attention
    goes through the T2T backend, whose dense prefix, budget windows and
    mask-refresh schedule follow the step index.  ``structured``: key weights
    tied to the query weights (0.9) and a spatially smooth latent, so that
    attention is local, as in trained video models (random weights and white
    noise give near-uniform attention, whose unions hold most keys)."""
    torch.manual_seed(seed)
    model = WanDiT(cfg, sparse, device, tie=0.9 if structured else 0.0)
    g = torch.Generator(device=device).manual_seed(seed + 1)
    if structured:
        x = smooth_latent(cfg, g, device)
    else:
        x = torch.randn(1, cfg.tokens, cfg.hidden, generator=g, device=device, dtype=torch.bfloat16)
    ctx = torch.randn(1, cfg.context_tokens, cfg.hidden, generator=g, device=device,
                      dtype=torch.bfloat16)
    t_emb = 0.1 * torch.randn(1, cfg.hidden, generator=g, device=device, dtype=torch.bfloat16)
    builder = cache = None
    if sparse:
        from token2tile_amd.backend.t2t_attn import T2TAttentionMetadataBuilder, T2TRequestCache
        builder, cache = T2TAttentionMetadataBuilder(), T2TRequestCache()
    times = {}
    for step in steps:
        md = None
        if sparse:
            md = builder.build(step_index=step, total_steps=50, cache=cache, profile_name=profile,
                               **(budget_kw or {}))
        torch.cuda.synchronize(device)
        t0 = time.perf_counter()
        y = model(x, t_emb, ctx, (lambda i, m=md: m) if sparse else None)
        torch.cuda.synchronize(device)
        times[step] = (time.perf_counter() - t0) * 1e3
        print(f"[dit] {'t2t' if sparse else 'dense'} step {step}: {times[step]:.1f} ms",
              file=sys.stderr, flush=True)
        assert bool(torch.isfinite(y).all()), "non-finite DiT output"
    return times


def run_chunks(cfg: DiTConfig, frames, device, steps=2, seed=0):
    """Time the block stack over a video in chunks of ``frames`` latent frames, each
    ``steps`` times (its denoising steps); returns the ms of each chunk's last."""
    torch.manual_seed(seed)
    model = WanDiT(cfg, False, device)
    g = torch.Generator(device=device).manual_seed(seed + 1)
    r = lambda *shape: torch.randn(*shape, generator=g, device=device, dtype=torch.bfloat16)  # noqa: E731
    x, ctx, t_emb = r(1, cfg.tokens, cfg.hidden), r(1, cfg.context_tokens, cfg.hidden), 0.1 * r(1, cfg.hidden)
    cache, n = ChunkCache(cfg, device), frames * cfg.grid[1] * cfg.grid[2]
    times = []
    for start in range(0, cfg.tokens, n):
        for _ in range(steps):
            torch.cuda.synchronize(device)
            t0 = time.perf_counter()
            y = model.forward_chunk(x[:, start:start + n], t_emb, ctx, cache, start)
            torch.cuda.synchronize(device)
            ms = (time.perf_counter() - t0) * 1e3
        times.append(ms)
        print(f"[dit] tokens {start} .. {min(start + n, cfg.tokens) - 1}: {ms:.1f} ms", file=sys.stderr, flush=True)
        assert bool(torch.isfinite(y).all()), "non-finite DiT output"
    return times


WINDOWS = ((12, 21), (21, 31), (31, 41), (41, 50))  # the backend's budget windows


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--blocks", type=int, default=40)
    p.add_argument("--per-window", type=int, default=4,
                   help="sparse steps timed per budget window (after the initial step 12)")
    p.add_argument("--structured", action="store_true",
                   help="tied q/k weights and a smooth latent (local attention); default: random")
    p.add_argument("--mxfp4", action="store_true",
                   help="the blocks' linear layers in MXFP4; default: bf16")
    p.add_argument("--int8", action="store_true",
                   help="the blocks' linear layers in 8 bits; default: bf16")
    p.add_argument("--chunk", type=int, default=0, metavar="FRAMES",
                   help="time generation in chunks of that many latent frames (dense attention over a paged cache) "
                        "instead of whole steps")
    p.add_argument("--fused-rope", action="store_true",
                   help="q/k norm and rotary embedding in one launch; default: torch")
    args = p.parse_args(argv)
    if not torch.cuda.is_available():
        sys.exit("the DiT harness needs a ROCm GPU")
    dev = torch.device("cuda", 0)
    if args.mxfp4 and args.int8:
        p.error("--mxfp4 or --int8")
    cfg = DiTConfig(blocks=args.blocks, mxfp4=args.mxfp4, int8=args.int8, fused_rope=args.fused_rope)
    linear = {"linear": "mxfp4"} if cfg.mxfp4 else {"linear": "int8"} if cfg.int8 else {}
    if args.chunk:
        if not 1 <= args.chunk <= cfg.grid[0]:
            p.error(f"--chunk: 1 to {cfg.grid[0]} frames")
        times = run_chunks(cfg, args.chunk, dev)
        print(json.dumps({"metric": "Wan2.1-14B DiT denoising step of a chunk (one CFG branch), ms",
                          "config": {"blocks": cfg.blocks, "hidden": cfg.hidden, "heads": cfg.heads, "ffn": cfg.ffn,
                                     "tokens": cfg.tokens, "chunk_frames": args.chunk, "dtype": "bf16",
                                     "weights": "random"},
                          **linear, "chunk_ms": [round(t, 1) for t in times]}), flush=True)
        return
    dense = run(cfg, [0, 1, 2], dev, sparse=False, structured=args.structured)
    d_ms = (dense[1] + dense[2]) / 2
    torch.cuda.empty_cache()
    # step 12 fits the projections and centroids (init_state) and rebuilds;
    # then a run of consecutive steps per window, so the mask-refresh
    # schedule (one structure rebuild per 4 steps) is what gets timed
    steps = [12]
    for lo, hi in WINDOWS:
        first = lo + 1 if lo == 12 else lo
        steps += list(range(first, min(hi, first + args.per_window)))
    sparse = run(cfg, steps, dev, sparse=True, structured=args.structured)
    win_ms = []
    for lo, hi in WINDOWS:
        ts = [sparse[s] for s in steps if lo <= s < hi and s != 12]
        win_ms.append(sum(ts) / len(ts))
    n_steps = [hi - lo for lo, hi in WINDOWS]
    # step 12 (the fit + first rebuild) at its measured time, the other
    # sparse steps at their window's mean
    n_steps[0] -= 1
    t2t_total = 12 * d_ms + sparse[12] + sum(n * w for n, w in zip(n_steps, win_ms))
    out = {"metric": "Wan2.1-14B DiT denoising step (one CFG branch), ms",
           "config": {"blocks": cfg.blocks, "hidden": cfg.hidden, "heads": cfg.heads,
                      "ffn": cfg.ffn, "tokens": cfg.tokens, "context_tokens": cfg.context_tokens,
                      "dtype": "bf16",
                      "weights": "random, k tied to q (0.9), smooth latent" if args.structured
                      else "random", "attention_profile": "auto"},
           **linear, **({"rope": "fused"} if cfg.fused_rope else {}),
           "dense_ms_per_step": round(d_ms, 1),
           "t2t_step_ms": {str(k): round(v, 1) for k, v in sparse.items()},
           "t2t_ms_per_step_by_window": [round(w, 1) for w in win_ms],
           "init_step_ms": round(sparse[12], 1),
           "schedule_50_steps_s": {"dense": round(50 * d_ms / 1e3, 2),
                                   "t2t": round(t2t_total / 1e3, 2)},
           "schedule_speedup_50_steps": round(50 * d_ms / t2t_total, 3)}
    print(json.dumps(out), flush=True)


if __name__ == "__main__":
    main()
