"""norm_gate_residual / token_norm on the GPU against 64 bits, with bounds that follow the arithmetic: each step's error from its operands'
errors, 2^-24 of the result for each 32-bit rounding (2^-8 for a stored bf16), and for a sum over a row's C channels, chains of at most
16 additions in a thread and 10 across threads, K = 32 times 2^-24 of the sum of magnitudes."""
import math

import pytest
import torch

from im2im_uq_amd import attn_ops
from im2im_uq_amd._lib import Im2ImError

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"
U32, U16, K = 2.0 ** -24, 2.0 ** -8, 32
EPS = 1e-5


def operands(rows, c, dtype, norm, gate=True, scale=True, post=True, pre=True, bias=True, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    vec = lambda mean=0.0: rnd(c) * 0.3 + mean  # noqa: E731
    o = {"x": (rnd(rows, c) + shift).to(dtype), "f": (rnd(rows, c) * 2 + shift).to(dtype) if post else None, "gate": rnd(rows, c).to(dtype) if gate and post else None,
         "scale": vec(0.5) if scale and post else None, "post_weight": vec(1.0) if post else None,
         "post_bias": vec() if post and bias and norm == "layer" else None, "pre_weight": vec(1.0) if pre else None,
         "pre_bias": vec() if pre and bias and norm == "layer" else None}
    o = {k: None if t is None else t.to(DEV) for k, t in o.items()}
    dy, dh = rnd(rows, c).to(dtype).to(DEV), rnd(rows, c).to(dtype).to(DEV)
    return o, dy if post else None, dh if pre else None


def call(o, norm):
    if o["f"] is None:
        return None, attn_ops.token_norm(o["x"], o["pre_weight"], o["pre_bias"], norm=norm, eps=EPS)
    return attn_ops.norm_gate_residual(**o, norm=norm, eps=EPS)


def train(o, norm, dy, dh):
    leaves = {k: t.detach().requires_grad_(True) for k, t in o.items() if t is not None}
    y, h = call({**o, **leaves}, norm)
    pairs = [(a, b) for a, b in ((y, dy), (h, dh)) if a is not None and b is not None]
    grads = torch.autograd.grad([a for a, _ in pairs], list(leaves.values()), [b for _, b in pairs], allow_unused=True)
    return {**({} if y is None else {"y": y}), **({} if h is None else {"h": h}), **{"d" + k: t for k, t in zip(leaves, grads)}}


def normed(v, err, w, b, layer):
    """(z, its error, reciprocal deviation, result, its error) of a row with elementwise error `err`"""
    mag = v.abs().mean(1, keepdim=True)
    mean = v.mean(1, keepdim=True) if layer else torch.zeros_like(mag)
    mean_err = (err.mean(1, keepdim=True) + K * U32 * mag) * layer
    r = 1 / ((v - mean).pow(2).mean(1, keepdim=True) + EPS).sqrt()
    z = (v - mean) * r
    lin = (err + mean_err + 2 * U32 * (v.abs() + mean.abs())) * r
    r_err = (lin * z.abs()).mean(1, keepdim=True) + (lin ** 2).mean(1, keepdim=True) + (K + 8) * U32       # relative
    z_err = lin * (1 + r_err) + z.abs() * (r_err + 2 * U32)
    n = z * w + (0 if b is None else b)
    return z, z_err, r, r_err, n, z_err * w.abs() + 3 * U32 * (z * w).abs() + U32 * n.abs()


def back(u, u_err, z, z_err, r, r_err, layer):
    """L(u) = r (u - mean u - z mean(u z)) and its error"""
    m, mag = u.mean(1, keepdim=True) * layer, u.abs().mean(1, keepdim=True)
    m_err = (u_err.mean(1, keepdim=True) + K * U32 * mag) * layer
    a, a_mag = (u * z).mean(1, keepdim=True), (u * z).abs().mean(1, keepdim=True)
    a_err = (u_err * z.abs() + u.abs() * z_err).mean(1, keepdim=True) + K * U32 * a_mag
    g = r * (u - m - z * a)
    parts = u.abs() + m.abs() + (z * a).abs()
    return g, r * (u_err + m_err + z_err * a.abs() + z.abs() * a_err + (4 * U32 + r_err) * parts)


def reference(o, norm, dy, dh):
    last = U16 if o["x"].dtype == BF16 else U32
    layer = norm == "layer"
    d = {k: None if t is None else t.detach().double() for k, t in o.items()}
    rows = d["x"].shape[0]
    x, out = d["x"], {}
    y, y_err = x, torch.zeros_like(x)
    s = 1.0 if d["scale"] is None else d["scale"]
    s_abs = abs(s) if d["scale"] is None else s.abs()
    if d["f"] is not None:
        zf, zf_err, rf, rf_err, n, n_err = normed(d["f"], torch.zeros_like(x), d["post_weight"], d["post_bias"], layer)
        a = torch.sigmoid(d["gate"]) if d["gate"] is not None else torch.ones_like(x)
        a_err = U32 * (8 + 2 * d["gate"].abs()) * a if d["gate"] is not None else torch.zeros_like(x)      # the exponent's rounding among them
        u = s * a * n
        u_err = s_abs * (a * n_err + a_err * n.abs()) + 3 * U32 * u.abs()
        y, y_err = x + u, u_err + U32 * (x + u).abs()
        out["y"] = (y, y_err + last * y.abs())
    du, du_err = (torch.zeros_like(x),) * 2
    if d["pre_weight"] is not None:
        zy, zy_err, ry, ry_err, h, h_err = normed(y, y_err, d["pre_weight"], d["pre_bias"], layer)
        out["h"] = (h, h_err + last * h.abs())
        if dh is not None:
            g = dh.double()
            du, du_err = back(g * d["pre_weight"], U32 * (g * d["pre_weight"]).abs(), zy, zy_err, ry, ry_err, layer)
            sums(out, "dpre_weight", g * zy, g.abs() * zy_err, rows)
            if d["pre_bias"] is not None:
                sums(out, "dpre_bias", g, torch.zeros_like(g), rows)
    if dy is not None:
        du = du + dy.double()
        du_err = du_err + U32 * du.abs()
    out["dx"] = (du, du_err + last * du.abs())
    if d["f"] is not None:
        ug, ug_err = du * a, du_err * a + du.abs() * a_err + U32 * (du * a).abs()
        if d["scale"] is not None:
            sums(out, "dscale", ug * n, ug_err * n.abs() + ug.abs() * n_err, rows)
        dn, dn_err = ug * s, ug_err * s_abs + U32 * (ug * s).abs()
        if d["gate"] is not None:
            dg = dn * n * (1 - a)
            err = (dn_err * n.abs() + dn.abs() * n_err) * (1 - a) + (dn * n).abs() * (a_err + U32) + 3 * U32 * dg.abs()
            out["dgate"] = (dg, err + last * dg.abs())
        sums(out, "dpost_weight", dn * zf, dn_err * zf.abs() + dn.abs() * zf_err, rows)
        if d["post_bias"] is not None:
            sums(out, "dpost_bias", dn, dn_err, rows)
        df, df_err = back(dn * d["post_weight"], dn_err * d["post_weight"].abs() + U32 * (dn * d["post_weight"]).abs(), zf, zf_err, rf, rf_err, layer)
        out["df"] = (df, df_err + last * df.abs())
    return out


def sums(out, name, terms, err, rows):
    chain = math.ceil(rows / 512) + 34                       # a thread's own rows at most, the block's 32; then 64 bits
    v = terms.sum(0)
    out[name] = (v, err.sum(0) + (chain + 2) * U32 * terms.abs().sum(0) + U32 * v.abs())


def check(got, want):
    assert set(got) == set(want)
    for name, (value, bound) in want.items():
        off = (got[name].detach().double() - value).abs()
        bad = ~(off <= bound + 1e-30)
        assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds, worst {float((off / (bound + 1e-30)).nan_to_num(math.inf).max()):.3g} x its bound"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 7), (65, 64), (33, 65), (130, 128), (7, 200), (50, 333), (1000, 512), (2049, 520), (17, 1024),
                                    (9, 1031), (40, 2048), (5, 3000), (6, 4096), (3, 5001), (2, 8192)])
def test_seam(rows, c, norm, dtype):
    o, dy, dh = operands(rows, c, dtype, norm, seed=c)
    check(train(o, norm, dy, dh), reference(o, norm, dy, dh))


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("absent", ["gate", "scale", "bias", "pre", "post", "gate scale", "gate scale bias pre"])
def test_parts_left_out(absent, norm):
    o, dy, dh = operands(77, 96, BF16, norm, seed=1, **{k: False for k in absent.split()})
    got = train(o, norm, dy, dh)
    check(got, reference(o, norm, dy, dh))
    y, h = call(o, norm)
    assert (h is None or torch.equal(h, got["h"])) and (y is None or torch.equal(y, got["y"]))


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("which", ["y", "h"])
def test_gradient_through_one_result(which, norm):
    o, dy, dh = operands(70, 100, F32, norm, seed=2)
    dy, dh = (dy, None) if which == "y" else (None, dh)
    want = reference(o, norm, dy, dh)
    got = train(o, norm, dy, dh)
    for n in ("y", "h"):
        got.pop(n), want.pop(n)
    for n in [n for n in got if n not in want]:              # the second norm's weights where only y is used
        assert which == "y" and n in ("dpre_weight", "dpre_bias") and (got[n] is None or (got[n] == 0).all())
        got.pop(n)
    check(got, want)


def test_large_mean():
    """channels around 1000: the variance survives the mean"""
    o, dy, dh = operands(64, 512, F32, "layer", seed=3, shift=1000.0)
    check(train(o, "layer", dy, dh), reference(o, "layer", dy, dh))


def test_strides_and_broadcast():
    """a slice of wider rows, head-major rows, one gate row for an image: the dense copies' bits; an expanded operand's gradient is the sum"""
    o, dy, dh = operands(48, 64, BF16, "layer", seed=4)
    dense = train(o, "layer", dy, dh)
    wide = torch.zeros(48, 200, dtype=BF16, device=DEV)
    wide[:, 3:67] = o["f"]
    got = train(dict(o, f=wide[:, 3:67], x=o["x"].t().contiguous().t()), "layer", dy.t().contiguous().t(), dh)
    assert all(torch.equal(got[n], dense[n]) for n in dense)
    x3, f3 = o["x"].view(6, 8, 64), o["f"].view(6, 8, 64).transpose(0, 1).contiguous().transpose(0, 1)
    gate = o["gate"][:6].clone().view(6, 1, 64).requires_grad_(True)
    full = gate.detach().expand(6, 8, 64).contiguous().requires_grad_(True)
    got = []
    for g in (gate.expand(6, 8, 64), full):
        y, h = attn_ops.norm_gate_residual(x3, f3, g, o["scale"], o["post_weight"], o["post_bias"], o["pre_weight"], o["pre_bias"], norm="layer")
        got.append((y, h, torch.autograd.grad((y, h), gate if g is not full else full, (dy.view_as(y), dh.view_as(h)))[0]))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert torch.equal(got[0][2], got[1][2].sum(1, keepdim=True))


def test_same_bits_and_graph():
    o, dy, dh = operands(5000, 256, BF16, "rms", seed=5)
    first = train(o, "rms", dy, dh)
    assert all(torch.equal(t, first[n]) for n, t in train(o, "rms", dy, dh).items())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x = o["x"].clone()
    with torch.cuda.stream(side):
        train(dict(o, x=x), "rms", dy, dh)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = train(dict(o, x=x), "rms", dy, dh)
    for scale in (2.0, 0.5, 1.0):
        x.copy_(o["x"] * scale)
        want = train(dict(o, x=x.clone()), "rms", dy, dh)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_no_rows():
    o, _, _ = operands(0, 16, F32, "rms")
    y, h = call(o, "rms")
    assert y.shape == h.shape == (0, 16)


def test_refusals():
    o, _, _ = operands(4, 16, F32, "layer")

    def refused(match, norm="layer", **kw):
        with pytest.raises(Im2ImError, match=match):
            attn_ops.norm_gate_residual(**dict(o, **kw), norm=norm)
    refused("GPU", x=o["x"].cpu())
    refused("fp32 or bf16", x=o["x"].half())
    refused("as x", f=o["f"].to(BF16))
    refused("as x", f=o["f"][:1])
    refused("as x", gate=o["gate"][:, :8])
    refused("GPU", gate=o["gate"].cpu())
    refused("fp32", scale=o["scale"].to(BF16))
    refused("fp32", post_weight=o["post_weight"][:8])
    refused("post_weight", post_weight=None)
    refused("pre_bias", pre_weight=None)
    refused("no bias", norm="rms")
    refused("norm must", norm="batch")
    for eps in (0.0, -1.0, math.inf, math.nan, 1e-60):
        refused("eps", eps=eps)
    with pytest.raises(Im2ImError, match="channels"):
        attn_ops.token_norm(torch.zeros(2, 8193, device=DEV), torch.ones(8193, device=DEV))
    with pytest.raises(Im2ImError, match="weight"):
        attn_ops.token_norm(o["x"], None)
