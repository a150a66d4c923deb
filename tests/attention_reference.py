"""Plain attention on a grid in 64 bits, and how far 32-bit and bf16 arithmetic may be from it.

Bounds: a product of n terms in 32 bits is off by at most n 2^-24 of the sum of its terms' magnitudes; a rounding by 2^-24 of the value (bf16:
2^-8).  With rho the relative error of a probability (twice the score's error, since the row's sum carries one too, and the sum's own)
    out    2^-8 (sum P|v| + |out|)        P rounded for the product, the result rounded                       (bf16)   + rho sum P|v|
    dS     E = P (rho |dP - D| + delta_dP + delta_D), and 2^-8 |dS| where it is rounded for a product        (bf16)
so every bound below is a sum over the same pairs as the value it belongs to, with magnitudes in the place of values."""
import math

import torch

from im2im_uq_amd.attn_ops import bucket_thresholds

U32, U16 = 2.0 ** -24, 2.0 ** -8


def axis_bucket(delta, n, max_distance):
    if n == 1:
        return torch.zeros_like(delta)
    side, m = n // 2, torch.zeros_like(delta)
    for t in bucket_thresholds(n, max_distance):
        m = m + (delta.abs() >= t)
    return m + side * (delta > 0)


def attention(q, k, v, table, grid, max_distance=64, lam=None, lengths=None, q_start=0, scale=None, dout=None):
    """{name: (value, bound)} in float64: out, and with dout: dq, dk, dv, dtable, dlam.  q [B, Lq, H * maps, D] and so on, any type."""
    bf16 = q.dtype == torch.bfloat16
    r = U16 if bf16 else 0.0                                 # roundings of products' operands
    last = U16 if bf16 else U32                              # and of results
    maps = 1 if lam is None else 2
    b, lq, hm, d = q.shape
    h, lk, gw = hm // maps, k.shape[1], grid[1]
    dev = q.device
    q, k, v = (t.detach().double() for t in (q, k, v))
    tab = table.detach().double()
    sc = 1 / math.sqrt(d) if scale is None else scale
    i, j = torch.arange(q_start, q_start + lq, device=dev), torch.arange(lk, device=dev)
    my, mx = max_distance if isinstance(max_distance, tuple) else (max_distance, max_distance)
    by = axis_bucket((j // gw)[None] - (i // gw)[:, None], table.shape[0], my)
    bx = axis_bucket((j % gw)[None] - (i % gw)[:, None], table.shape[1], mx)
    row = (by * table.shape[1] + bx).reshape(-1)
    bias = tab.reshape(-1, h)[row].view(lq, lk, h).permute(2, 0, 1)[None, :, None]
    ok = torch.ones(b, lk, dtype=torch.bool, device=dev) if lengths is None else j[None] < lengths.clamp(0, lk)[:, None]
    ok5 = ok[:, None, None, None, :]
    k = torch.where(ok[:, :, None, None], k, 0.0)
    v = torch.where(ok[:, :, None, None], v, 0.0)
    q5 = q.view(b, lq, h, maps, d).permute(0, 2, 3, 1, 4)
    k5 = k.view(b, lk, h, maps, d).permute(0, 2, 3, 1, 4)
    v4, kt, vt = v.permute(0, 2, 1, 3), k5.transpose(3, 4), v.permute(0, 2, 3, 1)
    s = (q5 @ kt * sc + bias).masked_fill(~ok5, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    # a score: d products, the scale and the bias (a handful of roundings, in units of log2 again); with it go the exponential's argument
    # and result, and the row's sum
    size = q5.abs() @ kt.abs() * sc + torch.where(bias.isfinite(), bias, 0.0).abs()
    size = torch.where(p > 0, size, 0.0).amax(-1, keepdim=True)
    rho = U32 * (2 * (d + 8) * size + lk / 16 + 32)
    weight = torch.ones(1, 1, 1, 1, 1, dtype=torch.float64, device=dev) if maps == 1 else torch.stack(
        (torch.ones_like(lam, dtype=torch.float64), -lam.detach().double()), 1).view(1, h, 2, 1, 1)
    mixed, mixed_abs = (weight * p).sum(2), (weight.abs() * p).sum(2)
    mixed_err = (weight.abs() * p * rho).sum(2)
    out = mixed @ v4
    out_err = (mixed_err + r * mixed_abs + (lk + 8) * U32 * mixed_abs) @ v4.abs() + last * out.abs()
    got = {"out": (out.permute(0, 2, 1, 3), out_err.permute(0, 2, 1, 3))}
    if dout is None:
        return got
    g = dout.detach().double().permute(0, 2, 1, 3)
    dv = mixed.transpose(2, 3) @ g
    dv_err = (mixed_err + r * mixed.abs() + (lq + 8) * U32 * mixed_abs).transpose(2, 3) @ g.abs() + last * dv.abs()
    dp0 = (g @ vt)[:, :, None]
    dp0_err = (d * maps + 4) * U32 * (g.abs() @ vt.abs())[:, :, None]
    dp, dp_err = weight * dp0, weight.abs() * (dp0_err + 2 * U32 * dp0.abs())
    dd = (p * dp).sum(-1, keepdim=True)
    # D comes from the saved result of the map: its probabilities enter as bf16 hi + lo (2^-8 of 2^-8)
    own, own_abs = p @ v4[:, :, None], p @ v4.abs()[:, :, None]
    dd_err = weight.abs() * ((g.abs()[:, :, None] * (own_abs * (r * r + rho + (lk + 8) * U32) + (d * maps + 8) * U32 * own.abs())).sum(-1, keepdim=True))
    ds = p * (dp - dd)
    ds_err = p * (rho * (dp - dd).abs() + dp_err + dd_err + 4 * U32 * (dp.abs() + dd.abs()))
    dq = ds @ k5 * sc
    dq_err = (ds_err + (r + (lk + 8) * U32) * ds.abs()) @ k5.abs() * sc + last * dq.abs()
    dk = ds.transpose(3, 4) @ q5 * sc
    dk_err = (ds_err + (r + (lq + 8) * U32) * ds.abs()).transpose(3, 4) @ q5.abs() * sc + last * dk.abs()
    flat = lambda t, n: t.permute(0, 3, 1, 2, 4).reshape(b, n, hm, d)  # noqa: E731
    got.update(dq=(flat(dq, lq), flat(dq_err, lq)), dk=(flat(dk, lk), flat(dk_err, lk)), dv=(dv.permute(0, 2, 1, 3), dv_err.permute(0, 2, 1, 3)))
    # the table: 32-bit chains of at most 2 x 32 queries, 8 copies, the images of a workgroup and the two maps, then 64 bits
    by_pair, err_pair = ds.sum((0, 2)).reshape(h, -1), (ds_err + (80 + b) * U32 * ds.abs()).sum((0, 2)).reshape(h, -1)
    rows = lambda t: torch.zeros(h, table.shape[0] * table.shape[1], dtype=torch.float64, device=dev).index_add_(1, row, t).t().reshape(  # noqa: E731
        table.shape)
    dt = rows(by_pair)
    got["dtable"] = (dt, rows(err_pair) + U32 * dt.abs())
    if maps == 2:
        terms, terms_err = p[:, :, 1] * dp0[:, :, 0], p[:, :, 1] * (rho[:, :, 1] * dp0[:, :, 0].abs() + dp0_err[:, :, 0])
        chain = (b * lk / 2 + 80) * U32                       # a lane's own chain of additions, then the workgroup's
        dl = -terms.sum((0, 2, 3))
        got["dlam"] = (dl, (terms_err + chain * terms.abs()).sum((0, 2, 3)) + U32 * dl.abs())
    return got


def check(got, want, names=None):
    """every element within its bound (and no NaN)"""
    for name, (value, bound) in want.items():
        if names is not None and name not in names:
            continue
        x = got[name].detach().double()
        assert x.shape == value.shape, (name, tuple(x.shape), tuple(value.shape))
        off = (x - value).abs()
        floor = 1e-30
        bad = ~(off <= bound + floor)
        assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds, worst {float((off / (bound + floor)).nan_to_num(math.inf).max()):.3g} x its bound"
