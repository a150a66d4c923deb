"""What the attention bottleneck's operators settle without a GPU: bucket borders and refusals at the C entries and in Python."""
import ctypes
import math

import pytest
import torch

from im2im_uq_amd import attn_ops
from im2im_uq_amd._lib import AttentionDesc, AttentionGrads, Im2ImError, NormGateDesc, lib

N = ctypes.byref


@pytest.mark.parametrize("n", [2, 4, 6, 8, 12, 16, 32, 64])
@pytest.mark.parametrize("m", [17, 20, 33, 64, 100, 128, 1000, 4096])
def test_bucket_borders(n, m):
    """the borders are where floor(e + (half - e) log(t / e) / log(m / e)) steps, computed in 64 bits and nudged over exact borders"""
    half = n // 2
    e = max(1, half // 2)
    thr = attn_ops.bucket_thresholds(n, m)
    assert len(thr) == half - 1 and list(thr) == sorted(thr)
    for t in list(range(0, 300)) + [m - 1, m, m + 1, 3 * m]:
        b = t if t < e else min(half - 1, e + math.floor((half - e) * math.log(t / e) / math.log(m / e) + 1e-9))
        assert sum(t >= x for x in thr) == min(b, half - 1), t


def test_bucket_refusals():
    assert attn_ops.bucket_thresholds(1, 0) == () and attn_ops.bucket_thresholds(2, 0) == ()
    for n, m in ((0, 64), (3, 64), (66, 64), (-2, 64), (8, 2), (64, 16), (8, 1 << 25)):
        with pytest.raises(Im2ImError):
            attn_ops.bucket_thresholds(n, m)


def test_cpu_tensors_are_refused():
    t = torch.zeros(1, 4, 2, 8)
    with pytest.raises(Im2ImError, match="GPU"):
        attn_ops.grid_attention(t, t, t, torch.zeros(2, 2, 2), (2, 2))
    with pytest.raises(Im2ImError, match="GPU"):
        attn_ops.norm_gate_residual(t, t, post_weight=torch.ones(8))


def desc(**kw):
    p = AttentionDesc()
    base = dict(q=4096, k=4096, v=4096, line=4096, B=2, Lq=6, Lk=6, H=2, D=16, maps=1, gh=2, gw=3, q_start=0, dtype=0, ny=2, nx=2, scale=0.25)
    for k, v in {**base, **kw}.items():
        setattr(p, k, v)
    for s in (p.q_stride, p.k_stride, p.v_stride):
        s[:] = kw.get("stride", (192, 32, 16))
    return p


def test_attention_entry_refusals():
    """every one is turned away on the host: the pointers are no memory"""
    assert lib.im2im_attention_fwd_workspace_bytes(N(desc())) == 0
    for kw in (dict(q=0), dict(line=0), dict(dtype=2), dict(maps=3), dict(maps=2), dict(B=0), dict(Lq=0), dict(Lk=0), dict(H=0), dict(D=12), dict(D=136),
               dict(maps=2, lam=4096, D=72), dict(gh=0), dict(gh=2, gw=513), dict(Lk=7), dict(q_start=1), dict(q_start=-1), dict(gh=1 << 13, gw=1 << 13),
               dict(q=4104), dict(stride=(190, 32, 16)), dict(stride=(-192, 32, 16)), dict(scale=math.inf), dict(scale=math.nan)):
        p = desc(**kw)
        assert lib.im2im_attention_fwd(N(p), 4096, None, None, None, 0, None) == -1, kw
        assert b"invalid argument" in lib.im2im_last_error()
        assert lib.im2im_attention_fwd_workspace_bytes(N(p)) == -1 and lib.im2im_attention_bwd_workspace_bytes(N(p), 1) == -1
        assert lib.im2im_attention_bwd(N(p), N(AttentionGrads()), 4096, 1 << 30, None) == -1
    assert lib.im2im_attention_fwd(None, 4096, None, None, None, 0, None) == -1
    assert lib.im2im_attention_fwd(N(desc()), None, None, None, None, 0, None) == -1
    assert lib.im2im_attention_fwd(N(desc()), 4096, 4096, None, None, 0, None) == -1              # one of the two saved tensors
    long_ = desc(Lq=1, Lk=4096, gh=64, gw=64)
    need = lib.im2im_attention_fwd_workspace_bytes(N(long_))
    assert need > 0
    assert lib.im2im_attention_fwd(N(long_), 4096, None, None, None, 0, None) == -1               # no workspace
    assert lib.im2im_attention_fwd(N(long_), 4096, None, None, 4096, need - 1, None) == -1
    token = dict(Lq=1, line=0, table=4096)                                                         # one query, its bias from the table
    assert lib.im2im_attention_fwd_workspace_bytes(N(desc(**token))) == 0
    for kw in (dict(table=0), dict(Lq=2), dict(ny=0), dict(nx=3), dict(ny=66), dict(nx=8)):
        assert lib.im2im_attention_fwd(N(desc(**{**token, **kw})), 4096, None, None, None, 0, None) == -1, kw
    assert lib.im2im_attention_fwd(N(desc(**token)), 4096, 4096, 4096, None, 0, None) == -1       # nothing to save
    assert lib.im2im_attention_bwd(N(desc(**token)), N(AttentionGrads()), 4096, 1 << 30, None) == -1
    g = AttentionGrads()
    for name in ("dout", "lse", "map_out", "dq", "dk", "dv", "dtable"):
        setattr(g, name, 4096)
    for s in (g.dq_stride, g.dk_stride, g.dv_stride):
        s[:] = (192, 32, 16)
    need = lib.im2im_attention_bwd_workspace_bytes(N(desc()), 1)
    for n in (0, 3, 66):
        assert lib.im2im_attention_bwd(N(desc(ny=n)), N(g), 4096, need, None) == -1
    assert lib.im2im_attention_bwd(N(desc(ny=8)), N(g), 4096, need, None) == -1                   # no borders
    assert lib.im2im_attention_bwd(N(desc()), N(g), 4096, 512, None) == -1                        # not enough for one image at a time either
    assert lib.im2im_attention_bwd(N(desc()), N(g), None, need, None) == -1
    assert lib.im2im_attention_bwd(N(desc(maps=2, lam=4096)), N(g), 4096, 1 << 30, None) == -1    # no dlam
    g.dq_stride[1] = 0
    assert lib.im2im_attention_bwd(N(desc()), N(g), 4096, need, None) == -1
    assert lib.im2im_relpos_line_len(20, 20) == 39 * 39 and lib.im2im_relpos_line_len(0, 4) == -1
    for args in ((None, 2, 2, 1, None, None, 2, 2, 4096), (4096, 3, 2, 1, None, None, 2, 2, 4096), (4096, 4, 2, 1, None, None, 2, 2, 4096),
                 (4096, 2, 2, 0, None, None, 2, 2, 4096), (4096, 2, 2, 1, None, None, 0, 2, 4096), (4096, 2, 2, 1, None, None, 2, 2, None)):
        assert lib.im2im_relpos_line(*args, None) == -1


def test_norm_entry_refusals():
    def p(**kw):
        d = NormGateDesc()
        for k, v in {**dict(x=4096, f=4096, post_weight=4096, pre_weight=4096, rows=4, C=16, x_stride=16, f_stride=16, norm=0, dtype=0, eps=1e-6), **kw}.items():
            setattr(d, k, v)
        return d

    def fwd(d, y=4096, h=4096):
        return lib.im2im_norm_gate_fwd(N(d), y, h, None)
    for kw in (dict(x=0), dict(rows=0), dict(C=0), dict(C=8193), dict(dtype=2), dict(norm=2), dict(post_weight=0), dict(pre_weight=0, pre_bias=4096),
               dict(post_bias=4096), dict(pre_bias=4096), dict(eps=0.0), dict(eps=math.nan), dict(x_stride=-1), dict(pre_weight=4100), dict(f=0)):
        assert fwd(p(**kw)) == -1, kw
    assert fwd(p(), y=None) == -1 and fwd(p(), h=None) == -1
    assert fwd(p(f=0, post_weight=0), y=4096) == -1
    n = lib.im2im_norm_gate_bwd_workspace_bytes(4, 16)
    assert n > 0 and lib.im2im_norm_gate_bwd_workspace_bytes(0, 16) == -1 and lib.im2im_norm_gate_bwd_workspace_bytes(4, 8193) == -1
    none = [None] * 8

    def bwd(d, dy, dh, outs=none, ws=4096, size=n):
        return lib.im2im_norm_gate_bwd(N(d), dy, dh, *outs, ws, size, None)
    assert bwd(p(), None, None) == -1 and bwd(p(), 4096, 4096, ws=None) == -1 and bwd(p(), 4096, 4096, size=n - 1) == -1
    assert bwd(p(pre_weight=0), 4096, 4096) == -1 and bwd(p(f=0, post_weight=0), 4096, 4096) == -1
    assert bwd(p(), 4096, 4096, [None, None, 4096] + [None] * 5) == -1                            # a gradient of a gate that is not there
    assert bwd(p(), 4096, None, none[:6] + [4096, None]) == -1                                    # of a norm that no gradient came through
