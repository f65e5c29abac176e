"""SD1.5-architecture conditional UNet (anythingv3), channels-last, inference only.

Implied compute of the anythingv3 Cog container (template
``templates/anythingv3.json:1``): 4 resolution levels (320/640/1280/1280),
2 ResBlocks per down level, 3 per up level, Transformer2D blocks with
self-attention (8 heads), cross-attention to 77x768 CLIP tokens, GEGLU FF.

MI355X-first choices (not a translation of any reference code - the reference
has none, inference lives in an external container):
  * NHWC everywhere; 1x1 proj_in/proj_out are plain GEMMs over [B*HW, C].
  * Q/K/V of self-attention are ONE fused GEMM; K/V of cross-attention one
    GEMM; the attention kernel reads q/k/v through strides (no reshapes).
  * out-projections and FF down-projections fuse the residual add into the
    GEMM (addmm, beta=1).
  * all 22 ResBlock time-embedding projections are ONE batched GEMM per step.
  * GroupNorm+SiLU is one HIP kernel; the nearest-x2 upsample is fused into
    the following conv's input indexing.
"""
from __future__ import annotations

import threading
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch
import torch.nn as nn

from .. import ops
from .layers import Conv2d, GroupNorm, LayerNorm, Linear, timestep_embedding


@dataclass
class UNetConfig:
    in_channels: int = 4
    out_channels: int = 4
    block_channels: Tuple[int, ...] = (320, 640, 1280, 1280)
    attn_levels: Tuple[bool, ...] = (True, True, True, False)
    layers_per_block: int = 2
    heads: int = 8
    head_dim: Optional[int] = None  # if set, heads = C // head_dim (SD2-style)
    cross_dim: int = 768
    groups: int = 32
    eps: float = 1e-5
    time_dim: int = 320  # == block_channels[0]

    @staticmethod
    def sd15():
        return UNetConfig()

    @staticmethod
    def tiny():
        return UNetConfig(block_channels=(32, 64, 64, 64), heads=2, cross_dim=32, groups=8, time_dim=32)


class SelfAttention(nn.Module):
    def __init__(self, dim, heads):
        super().__init__()
        self.heads = heads
        self.to_qkv = Linear(dim, 3 * dim, bias=False)
        self.to_out = Linear(dim, dim)

    def forward(self, x, residual, ln=None):
        """``ln``: the block's LayerNorm of x, folded into the QKV GEMM (x is then its input)."""
        B, N, C = x.shape
        H = self.heads
        qkv = (ln.linear(x, self.to_qkv) if ln is not None else self.to_qkv(x)).view(B, N, 3, H, C // H)
        o = ops.attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2])
        return self.to_out(o.reshape(B, N, C), residual=residual)


# Cross-attention K/V hoisting: the text context is constant over a task's denoising steps, so
# the graphed UNet computes every cross-attention K/V projection once per context (a separate
# small hipGraph, "produce") and the per-step graph reads them ("consume").  Thread-local: the
# modules are shared by the pipeline forks, each fork owns its K/V buffers.
_KV = threading.local()


class cross_kv_mode:
    """``with cross_kv_mode("produce" | "consume", table): ...`` - see ``_KV`` above."""

    def __init__(self, mode, table):
        self.mode, self.table = mode, table

    def __enter__(self):
        self.prev = (getattr(_KV, "mode", None), getattr(_KV, "table", None))
        _KV.mode, _KV.table = self.mode, self.table
        return self

    def __exit__(self, *exc):
        _KV.mode, _KV.table = self.prev


class CrossAttention(nn.Module):
    def __init__(self, dim, ctx_dim, heads):
        super().__init__()
        self.heads = heads
        self.to_q = Linear(dim, dim, bias=False)
        self.to_kv = Linear(ctx_dim, 2 * dim, bias=False)
        self.to_out = Linear(dim, dim)

    def context_kv(self, ctx):
        return self.to_kv(ctx)

    def forward(self, x, ctx, residual, ln=None):
        B, N, C = x.shape
        H = self.heads
        q = (ln.linear(x, self.to_q) if ln is not None else self.to_q(x)).view(B, N, H, C // H)
        mode = getattr(_KV, "mode", None)
        if mode == "consume":
            kv = _KV.table[id(self)]
        else:
            kv = self.to_kv(ctx)
            if mode == "produce":
                _KV.table[id(self)] = kv
        kv = kv.view(B, ctx.shape[1], 2, H, C // H)
        o = ops.attention(q, kv[:, :, 0], kv[:, :, 1])
        return self.to_out(o.reshape(B, N, C), residual=residual)


class FeedForward(nn.Module):
    """GEGLU FF: C -> 8C (value|gate) -> gelu-gated 4C -> C."""

    def __init__(self, dim, mult=4):
        super().__init__()
        self.proj = Linear(dim, 2 * mult * dim)
        self.out = Linear(mult * dim, dim)

    def forward(self, x, residual, ln=None):
        # GEGLU fused into the projection GEMM's epilogue on the GPU (ops.linear_geglu); ``ln``: the
        # block's LayerNorm of x folded into the same GEMM
        h = ln.linear_geglu(x, self.proj) if ln is not None else self.proj.geglu(x)
        return self.out(h, residual=residual)


class BasicTransformerBlock(nn.Module):
    def __init__(self, dim, ctx_dim, heads):
        super().__init__()
        self.norm1 = LayerNorm(dim)
        self.attn1 = SelfAttention(dim, heads)
        self.norm2 = LayerNorm(dim)
        self.attn2 = CrossAttention(dim, ctx_dim, heads)
        self.norm3 = LayerNorm(dim)
        self.ff = FeedForward(dim)

    def forward(self, h, ctx):
        # pre-LN: each LayerNorm feeds only its GEMM, so it is folded into that GEMM (ops.ln_linear)
        h = self.attn1(h, residual=h, ln=self.norm1)
        h = self.attn2(h, ctx, residual=h, ln=self.norm2)
        h = self.ff(h, residual=h, ln=self.norm3)
        return h


class Transformer2D(nn.Module):
    def __init__(self, dim, ctx_dim, heads, groups):
        super().__init__()
        self.norm = GroupNorm(groups, dim, eps=1e-6)
        self.proj_in = Linear(dim, dim)
        self.block = BasicTransformerBlock(dim, ctx_dim, heads)
        self.proj_out = Linear(dim, dim)

    def forward(self, x, ctx):
        B, H, W, C = x.shape
        h = self.proj_in.forward_norm(x.view(B, H * W, C), self.norm.table(x))  # GN fused into proj_in
        h = self.block(h, ctx)
        return self.proj_out(h, residual=x.view(B, H * W, C)).view(B, H, W, C)


class ResBlock(nn.Module):
    def __init__(self, cin, cout, temb_dim, groups, eps):
        super().__init__()
        self.norm1 = GroupNorm(groups, cin, eps, silu=True)
        self.conv1 = Conv2d(cin, cout, 3)
        self.temb_proj = Linear(temb_dim, cout, hoisted=True) if temb_dim else None
        self.norm2 = GroupNorm(groups, cout, eps, silu=True)
        self.conv2 = Conv2d(cout, cout, 3)
        self.shortcut = Conv2d(cin, cout, 1) if cin != cout else None
        self.cout = cout

    def forward(self, x, temb_out=None):
        """temb_out: this block's projected time embedding [B, cout] (batched GEMM)."""
        # GroupNorm+SiLU run as the convs' operand prologue (table of per-(b, c) affines);
        # time-embedding add and residual are fused into the epilogues.
        h = self.conv1(x, temb=temb_out, norm=self.norm1.table(x))
        skip = self.shortcut(x) if self.shortcut is not None else ops.materialize(x)
        return self.conv2(h, residual=skip, norm=self.norm2.table(h))


class Downsample(nn.Module):
    def __init__(self, c):
        super().__init__()
        self.conv = Conv2d(c, c, 3, stride=2, padding=1)

    def forward(self, x):
        return self.conv(x)


class Upsample(nn.Module):
    def __init__(self, c):
        super().__init__()
        self.conv = Conv2d(c, c, 3)

    def forward(self, x):
        return self.conv(x, upsample=True)


class UNet2DCondition(nn.Module):
    def __init__(self, cfg: UNetConfig = None):
        super().__init__()
        cfg = cfg or UNetConfig()
        self.cfg = cfg
        ch = cfg.block_channels
        tdim = cfg.time_dim * 4
        self.conv_in = Conv2d(cfg.in_channels, ch[0], 3)
        self.time_lin1 = Linear(cfg.time_dim, tdim)
        self.time_lin2 = Linear(tdim, tdim)

        def heads_for(c):
            return c // cfg.head_dim if cfg.head_dim else cfg.heads

        self.down = nn.ModuleList()
        skip_ch = [ch[0]]
        cur = ch[0]
        for lvl, c in enumerate(ch):
            blk = nn.Module()
            blk.resnets = nn.ModuleList()
            blk.attns = nn.ModuleList()
            for _ in range(cfg.layers_per_block):
                blk.resnets.append(ResBlock(cur, c, tdim, cfg.groups, cfg.eps))
                cur = c
                if cfg.attn_levels[lvl]:
                    blk.attns.append(Transformer2D(c, cfg.cross_dim, heads_for(c), cfg.groups))
                skip_ch.append(c)
            blk.downsample = Downsample(c) if lvl < len(ch) - 1 else None
            if blk.downsample is not None:
                skip_ch.append(c)
            self.down.append(blk)

        self.mid_res1 = ResBlock(cur, cur, tdim, cfg.groups, cfg.eps)
        self.mid_attn = Transformer2D(cur, cfg.cross_dim, heads_for(cur), cfg.groups)
        self.mid_res2 = ResBlock(cur, cur, tdim, cfg.groups, cfg.eps)

        self.up = nn.ModuleList()
        rch = list(reversed(ch))
        rattn = list(reversed(cfg.attn_levels))
        for lvl, c in enumerate(rch):
            blk = nn.Module()
            blk.resnets = nn.ModuleList()
            blk.attns = nn.ModuleList()
            for _ in range(cfg.layers_per_block + 1):
                s = skip_ch.pop()
                blk.resnets.append(ResBlock(cur + s, c, tdim, cfg.groups, cfg.eps))
                cur = c
                if rattn[lvl]:
                    blk.attns.append(Transformer2D(c, cfg.cross_dim, heads_for(c), cfg.groups))
            blk.upsample = Upsample(c) if lvl < len(rch) - 1 else None
            self.up.append(blk)

        self.norm_out = GroupNorm(cfg.groups, ch[0], cfg.eps, silu=True)
        self.conv_out = Conv2d(ch[0], cfg.out_channels, 3)
        self._temb_cache = None

    # ---- batched time-embedding projection for all ResBlocks -------------------------------
    def _resblocks(self) -> List[ResBlock]:
        return [m for m in self.modules() if isinstance(m, ResBlock)]

    def _temb_weights(self):
        rbs = self._resblocks()
        key = tuple(r.temb_proj.weight.data_ptr() for r in rbs)
        if self._temb_cache is None or self._temb_cache[0] != key:
            w = torch.cat([r.temb_proj.weight for r in rbs], dim=0)
            b = torch.cat([r.temb_proj.bias for r in rbs], dim=0)
            ops.derived_ready(w)
            self._temb_cache = (key, w, b, [r.cout for r in rbs])
        return self._temb_cache[1:]

    def time_embed(self, t, batch, dtype):
        """t: scalar / [B] timestep -> per-ResBlock projected embeddings (dict)."""
        if not torch.is_tensor(t):
            t = torch.tensor([t], dtype=torch.float32)
        t = t.reshape(-1).to(self.conv_in.weight.device)
        if t.numel() == 1:
            t = t.expand(batch)
        emb = timestep_embedding(t, self.cfg.time_dim).to(dtype)
        emb = self.time_lin2(ops.silu(self.time_lin1(emb)))
        w, b, couts = self._temb_weights()
        allp = ops.linear(ops.silu(emb), w, b)  # one GEMM for every ResBlock
        return dict(zip(self._resblocks(), torch.split(allp, couts, dim=1)))

    def forward(self, x, t, ctx, temb=None):
        """x [B, H, W, 4] latent (channels-last), t timestep, ctx [B, 77, cross_dim]."""
        if temb is None:
            temb = self.time_embed(t, x.shape[0], x.dtype)
        h = self.conv_in(x)
        skips = [h]
        for blk in self.down:
            for i, rb in enumerate(blk.resnets):
                h = rb(h, temb[rb])
                if len(blk.attns):
                    h = blk.attns[i](h, ctx)
                skips.append(h)
            if blk.downsample is not None:
                h = blk.downsample(h)
                skips.append(h)
        h = self.mid_res1(h, temb[self.mid_res1])
        h = self.mid_attn(h, ctx)
        h = self.mid_res2(h, temb[self.mid_res2])
        for blk in self.up:
            for i, rb in enumerate(blk.resnets):
                h = ops.cat_channels(h, skips.pop())      # read in place by GN stats/apply + shortcut
                h = rb(h, temb[rb])
                if len(blk.attns):
                    h = blk.attns[i](h, ctx)
            if blk.upsample is not None:
                h = blk.upsample(h)
        return self.conv_out(h, norm=self.norm_out.table(h))
