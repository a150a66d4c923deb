"""Attention blocks for the U-Net's bottleneck, between the last Down and the first Up block (the reference's trunk has none there,
core/models/trunks/unet.py:33-46): every pixel of the deepest feature map sees every other one, with a learned bias for their distance.

A block, on tokens x (one for each pixel, channels last, no copy):

    h = N_pre(x)
    q, k, v = conv(h);  g = conv(h)                           1x1 convolutions without bias, on the trunk's MFMA kernels
    f = conv(attention(q, k, v; bias table of the block))     "relative": softmax attention; "differential": the difference of two maps
    x = x + scale * sigmoid(g) * N_post(f)

The last line and the next block's N_pre are one pass over the tokens (attn_ops.norm_gate_residual)."""
import math

import torch
import torch.nn as nn

from ... import _pkg  # noqa: F401
from .... import attn_ops, nn_ops
from .unet_parts import _cdt

KINDS = ("relative", "differential")


class AttentionBlock(nn.Module):
    """the parameters of one block; AttentionBottleneck runs it"""

    def __init__(self, channels, kind, heads, buckets, index):
        super().__init__()
        self.heads = heads
        self.pre_weight = nn.Parameter(torch.ones(channels))
        self.qkv = nn.Conv2d(channels, 3 * channels, kernel_size=1, bias=False)
        self.gate = nn.Conv2d(channels, channels, kernel_size=1, bias=False)
        self.table = nn.Parameter(torch.zeros(buckets, buckets, heads))
        # the second map starts with little weight in the first block and more in later ones
        self.lam = nn.Parameter(torch.full((heads,), 0.8 - 0.6 * math.exp(-0.3 * index))) if kind == "differential" else None
        self.proj = nn.Conv2d(channels, channels, kernel_size=1, bias=False)
        self.post_weight = nn.Parameter(torch.ones(channels))
        self.scale = nn.Parameter(torch.full((channels,), 0.1))


class AttentionBottleneck(nn.Module):
    """`blocks` attention blocks on a [B, C, H, W] feature map, which keeps its shape.  kind: "relative" | "differential"; heads: C / 64 unless
    given; buckets: of the bias table, for each axis; distances from max_distance on share a bucket."""

    def __init__(self, channels, kind="relative", blocks=1, heads=None, buckets=16, max_distance=64):
        super().__init__()
        if kind not in KINDS:
            raise ValueError(f"attention must be one of {KINDS} or None, got {kind!r}")
        if blocks < 1:
            raise ValueError(f"attention blocks: at least 1, got {blocks}")
        heads = max(1, channels // 64) if heads is None else heads
        maps = 2 if kind == "differential" else 1
        if channels % 32 or heads < 1 or channels % (8 * heads * maps) or channels // heads > 128:
            raise ValueError(f"{channels} channels do not divide into {heads} heads of {maps} map(s): a multiple of 32, and up to 128 channels a head in "
                             f"multiples of {8 * maps}")
        attn_ops.bucket_thresholds(buckets, max_distance)
        self.kind, self.max_distance = kind, max_distance
        self.blocks = nn.ModuleList([AttentionBlock(channels, kind, heads, buckets, i) for i in range(blocks)])
        self.compute_dtype = None

    def forward(self, x):
        cdt = _cdt(self)
        t = nn_ops.nhwc(nn_ops.materialize(x), cdt)
        b, gh, gw, c = t.shape

        def conv(layer, tokens):
            return nn_ops.nhwc(nn_ops.Conv1x1.apply(nn_ops.nchw(tokens.reshape(b, gh, gw, -1)), layer.weight, None, cdt)).view(b, gh * gw, -1)
        t = t.reshape(b, gh * gw, c)
        h = attn_ops.token_norm(t, self.blocks[0].pre_weight)
        for i, blk in enumerate(self.blocks):
            a = attn_ops.grid_self_attention(conv(blk.qkv, h), blk.heads, blk.table, (gh, gw), lam=blk.lam, max_distance=self.max_distance)
            following = self.blocks[i + 1].pre_weight if i + 1 < len(self.blocks) else None
            t, h = attn_ops.norm_gate_residual(t, conv(blk.proj, a), gate=conv(blk.gate, h), scale=blk.scale, post_weight=blk.post_weight,
                                               pre_weight=following)
        return nn_ops.nchw(t.view(b, gh, gw, c))
