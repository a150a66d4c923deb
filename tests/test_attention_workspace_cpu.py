"""How much memory the attention backward asks for, without a GPU."""
import ctypes

import pytest

from im2im_uq_amd._lib import AttentionDesc, lib


def need(gh, gw, heads, d, batch=1, maps=1, dtype=1, table=1):
    n = gh * gw
    p = AttentionDesc()
    for k, v in dict(q=4096, k=4096, v=4096, line=4096, lam=4096, B=batch, Lq=n, Lk=n, H=heads, D=d, maps=maps, gh=gh, gw=gw, dtype=dtype, ny=2, nx=2, scale=1.0).items():
        setattr(p, k, v)
    c = heads * maps * d
    for s in (p.q_stride, p.k_stride):
        s[:] = (n * c, c, d)
    p.v_stride[:] = (n * c, c, d * maps)
    return lib.im2im_attention_bwd_workspace_bytes(ctypes.byref(p), table)


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("gh,gw,heads,batch", [(20, 20, 8, 78), (128, 128, 8, 1), (128, 128, 8, 4), (256, 256, 8, 1), (512, 512, 8, 1), (512, 512, 1, 3), (32768, 512, 2, 1),
                                               (1, 65536, 8, 1), (1, 1 << 24, 1, 1), (1 << 24, 1, 4, 1)])
def test_memory_grows_with_the_tokens(gh, gw, heads, batch, maps):
    """the table's gradient: at most 1 GiB of lines, or one of all heads where that is more, beside its 64-bit sum; D and lam's parts: four bytes a query
    and map, and less; parts of few workgroups: up to 256 MiB"""
    tokens, line = gh * gw, heads * (2 * gh - 1) * (2 * gw - 1)
    most = max(1 << 30, 4 * line) + 8 * line + batch * heads * tokens * (4 * maps + 4) + (256 << 20)
    assert 0 < need(gh, gw, heads, 32, batch, maps) <= most
    assert 0 < need(gh, gw, heads, 32, batch, maps, table=0) <= batch * heads * tokens * (4 * maps + 4) + (256 << 20)


def test_usual_sizes_are_as_they_were():
    """20x20 at batch 78: one image a workgroup"""
    assert need(20, 20, 8, 64, 78) > 78 * 4 * 8 * 39 * 39 * 4
    assert need(20, 20, 8, 64, 78) < 78 * 4 * 8 * 39 * 39 * 4 + (2 << 20)


def test_calls_over_a_launch_are_refused():
    """2^32 work-items: a batch and its heads of up to 2^24 - 1 workgroups, one token or key each, are described; from there on refused"""
    def tokens(batch, heads, lq, lk):
        p = AttentionDesc()
        for k, v in dict(q=4096, k=4096, v=4096, line=4096, B=batch, Lq=lq, Lk=lk, H=heads, D=8, maps=1, gh=1, gw=512, ny=2, nx=2, scale=1.0).items():
            setattr(p, k, v)
        c = heads * 8
        p.q_stride[:], p.k_stride[:], p.v_stride[:] = (lq * c, c, 8), (lk * c, c, 8), (lk * c, c, 8)
        return lib.im2im_attention_fwd_workspace_bytes(ctypes.byref(p)), lib.im2im_attention_bwd_workspace_bytes(ctypes.byref(p), 0)
    assert min(tokens((1 << 21) - 1, 8, 1, 1)) >= 0 and min(tokens((1 << 19) - 1, 8, 1, 512)) >= 0 and min(tokens((1 << 19) - 1, 8, 512, 1)) >= 0
    for sizes in ((1 << 21, 8, 1, 1), (1 << 19, 8, 1, 512), (1 << 19, 8, 512, 1), (1 << 20, 16, 1, 1)):
        assert tokens(*sizes) == (-1, -1), sizes
