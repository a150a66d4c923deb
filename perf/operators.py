"""The token operators of a U-Net's attention bottleneck: what is timed, and their plain forms.

Three operators act on the bottleneck feature map read as one token per pixel (channels last, no copy):

* ``attn``   softmax attention over an image grid with a learned relative position bias by buckets,
* ``diff``   differential attention on the same grid: the difference of two softmax maps with a learned weight per head,
* ``norm``   the norms behind and before a block, fused with the block's gate, its residual scale and the residual sum.

``own = False``: ``run`` computes them with elementary torch operations in 32 bits.  ``own = True``: ``run`` makes the calls
that a user makes of ``im2im_uq_amd.attn_ops``.
"""
import math

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
_DTYPE = {"bf16": BF16, "fp32": F32}


# ------------------------------------------------------------------------------------------------------------- the cases
def _attention(name, op, grid, b, heads, d, buckets, dtype, train, lq=None, q_start=0, ragged=False):
    c = {"op": op, "gh": grid[0], "gw": grid[1], "b": b, "heads": heads, "d": d, "ny": buckets[0], "nx": buckets[1], "max_distance": 64,
         "dtype": dtype, "train": train, "lq": grid[0] * grid[1] if lq is None else lq, "q_start": q_start, "ragged": ragged}
    return dict(c, name=name) if name else c


def _norm(name, rows, c, kind, dtype, train, gate=True):
    k = {"op": "norm", "rows": rows, "c": c, "kind": kind, "dtype": dtype, "train": train, "gate": gate}
    return dict(k, name=name) if name else k


def listed():
    return [
        # one pixel of a 1024 x 1024 image's 64 x 64 bottleneck is asked for again: one query, the whole grid as keys
        _attention("attn token of 64x64", "attn", (64, 64), 1, 8, 64, (32, 32), "bf16", False, lq=1, q_start=2080),
        # training on 320 x 320 images, four levels: a 20 x 20 grid of 512 channels; 10 images is one GPU's share of a batch of 78
        _attention("attn train 20x20 b10", "attn", (20, 20), 10, 8, 64, (16, 16), "bf16", True),
        # the whole batch of 78 on one GPU
        _attention("attn train 20x20 b78", "attn", (20, 20), 78, 8, 64, (16, 16), "bf16", True),
        # 1024 x 1024 images, five levels: a 32 x 32 grid of 1024 channels
        _attention("attn train 32x32 b8", "attn", (32, 32), 8, 8, 128, (32, 32), "bf16", True),
        # parity mode (32 bits), an odd grid, padded images: one of them empty
        _attention("attn train 17x23 fp32 ragged", "attn", (17, 23), 3, 5, 40, (8, 16), "fp32", True, ragged=True),
        # differential heads in the 320 x 320 network
        _attention("diff train 20x20 b10", "diff", (20, 20), 10, 8, 32, (16, 16), "bf16", True),
        # inference one level higher up: a 40 x 40 grid, padded images
        _attention("diff 40x40 b16 ragged", "diff", (40, 40), 16, 4, 64, (16, 16), "bf16", False, ragged=True),
        # one token against a long row of tokens (a flattened volume)
        _attention("diff token of 1x16384 b4", "diff", (1, 16384), 4, 8, 32, (1, 32), "bf16", False, lq=1, q_start=16383, ragged=True),
        # parity mode
        _attention("diff train 24x24 fp32", "diff", (24, 24), 4, 4, 32, (16, 16), "fp32", True),
        # between two blocks of the bottleneck, training at batch 78: 78 * 400 tokens of 512 channels
        _norm("norm train 31200x512", 31200, 512, "rms", "bf16", True),
        # the same seam at inference, one image
        _norm("norm 400x512", 400, 512, "layer", "bf16", False),
        # parity mode with a channel count that no vector width divides
        _norm("norm train 4097x333 fp32", 4097, 333, "layer", "fp32", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attn", "attn", "diff", "diff", "norm"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    train = rng.random() < 0.6
    if op == "norm":
        c = rng.choice((_log_int(rng, 32, 2048), 8 * _log_int(rng, 4, 256)))
        return _norm(None, _log_int(rng, 16, 16384), c, rng.choice(("rms", "layer")), dtype, train, gate=rng.random() < 0.75)
    d = 8 * rng.randint(1, 16) if op == "attn" else 8 * rng.randint(1, 8)
    heads, buckets = rng.randint(1, 8), (rng.choice((8, 16, 32)), rng.choice((8, 16, 32)))
    if train:
        grid = (rng.randint(5, 32), rng.randint(5, 32))
        most = max(1, min(32, int(1.2e7 / (grid[0] * grid[1]) ** 2 / (1 if dtype == "bf16" else 4))))
        return _attention(None, op, grid, _log_int(rng, 1, most), heads, d, buckets, dtype, True, ragged=rng.random() < 0.4)
    if rng.random() < 0.5:  # single tokens and a few of them
        grid = (_log_int(rng, 8, 96), _log_int(rng, 8, 96)) if rng.random() < 0.6 else (1, _log_int(rng, 64, 16384))
        if grid[0] == 1:
            buckets = (1, buckets[1])
        lq = rng.choice((1, 1, 1, rng.randint(2, 40)))
        return _attention(None, op, grid, _log_int(rng, 1, 8), heads, d, buckets, dtype, False, lq=lq,
                          q_start=rng.randint(0, grid[0] * grid[1] - lq), ragged=rng.random() < 0.5)
    grid = (rng.randint(7, 40), rng.randint(7, 40))
    return _attention(None, op, grid, _log_int(rng, 1, 8), heads, d, buckets, dtype, False, ragged=rng.random() < 0.4)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        n, c = case["rows"] * case["c"], case["c"]
        wide = 3 if case["gate"] else 2                                    # x, f and the gate's logits
        fwd = (wide + 2) * n * e + 5 * c * 4                               # ... in; y and h out
        bwd = (wide + 2) * n * e + wide * n * e + 10 * c * 4               # the same inputs, dy and dh in; dx, df, dgate out
        return {"bytes": fwd + (bwd if case["train"] else 0), "flops": n * (20 + (50 if case["train"] else 0))}
    b, h, d, lq, lk = case["b"], case["heads"], case["d"], case["lq"], case["gh"] * case["gw"]
    maps = 2 if case["op"] == "diff" else 1
    dv = maps * d
    q, kk, o = b * lq * h * maps * d * e, b * lk * h * maps * d * e, b * lq * h * dv * e
    v = b * lk * h * dv * e
    pair = 2 * b * h * lq * lk                                             # one multiply-add per pair, head and channel
    fwd, mm = q + kk + v + o, pair * maps * (d + dv)
    if not case["train"]:
        return {"bytes": fwd, "flops": mm}
    # backward: the scores again, the values' products once for both maps, dq and dk of each map, dv once
    return {"bytes": fwd + 2 * (q + kk + v) + o, "flops": mm + pair * (maps * d + dv + 2 * maps * d + dv)}


# ------------------------------------------------------------------------------------------------------------ the inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    dt = _DTYPE[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dtype)

    s = {"case": dict(case)}
    if case["op"] == "norm":
        n, c = case["rows"], case["c"]
        s["x"] = normal(n, c) + normal(1, c, std=0.5)                      # a residual stream with channel means
        s["f"] = normal(n, c, std=2.0) + normal(1, c)
        s["gate"] = normal(n, c, std=1.5) if case["gate"] else None
        s["scale"] = normal(c, std=0.2, mean=0.5, dtype=F32)
        s["post_weight"], s["pre_weight"] = normal(c, std=0.2, mean=1.0, dtype=F32), normal(c, std=0.2, mean=1.0, dtype=F32)
        both = case["kind"] == "layer"
        s["post_bias"], s["pre_bias"] = (normal(c, std=0.2, dtype=F32), normal(c, std=0.2, dtype=F32)) if both else (None, None)
        s["dy"], s["dh"] = normal(n, c), normal(n, c)
        leaves = ("x", "f", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")
    else:
        b, h, d, lq, lk = case["b"], case["heads"], case["d"], case["lq"], case["gh"] * case["gw"]
        maps = 2 if case["op"] == "diff" else 1
        s["q"], s["k"], s["v"] = normal(b, lq, h * maps, d), normal(b, lk, h * maps, d), normal(b, lk, h, maps * d)
        s["table"] = normal(case["ny"], case["nx"], h, std=0.5, dtype=F32)
        s["lam"] = torch.rand(h, generator=g, device=dev) * 0.6 + 0.2 if maps == 2 else None
        s["lengths"] = None
        if case["ragged"]:                                                 # padded images; with several of them, the last is empty
            lengths = torch.randint((lk + 1) // 2, lk + 1, (b,), generator=g, device=dev, dtype=torch.int32)
            if b > 2:
                lengths[-1] = 0
            s["lengths"] = lengths
        s["dout"] = normal(b, lq, h, maps * d)
        leaves = ("q", "k", "v", "table", "lam")
    if case["train"]:
        for name in leaves:
            if s[name] is not None:
                s[name].requires_grad_(True)
    s["leaves"] = [n for n in leaves if s[n] is not None]
    return s


# ------------------------------------------------------------------------------------------------------- the plain forms
def _thresholds(n, max_distance):
    """Smallest distances of the buckets 1, 2, ... of one sign: exact up to half of them, then even in the distance's logarithm."""
    half = max(1, n // 2)
    e = max(1, half // 2)
    # bucket >= m  <=>  (half - e) log(t / e) >= (m - e) log(max_distance / e), in whole numbers
    thr = []
    for m in range(1, half):
        t = min(m, e)
        while m > e and t ** (half - e) * e ** (m - e) < max_distance ** (m - e) * e ** (half - e):
            t += 1
        thr.append(t)
    return half, thr


def _axis_bucket(delta, n, max_distance):
    if n == 1:
        return torch.zeros_like(delta)
    half, thr = _thresholds(n, max_distance)
    reached = delta.abs()[..., None] >= torch.tensor(thr, dtype=delta.dtype, device=delta.device)
    return reached.sum(-1) + half * (delta > 0)


def _bucket_index(case, dev):
    """[Lq, Lk]: the row of the table (ny * nx rows) that belongs to each query and key."""
    gw = case["gw"]
    i = torch.arange(case["q_start"], case["q_start"] + case["lq"], device=dev)
    j = torch.arange(case["gh"] * gw, device=dev)
    dy = torch.arange(-(case["gh"] - 1), case["gh"], device=dev)           # key minus query, once for each distance
    dx = torch.arange(-(gw - 1), gw, device=dev)
    by, bx = _axis_bucket(dy, case["ny"], case["max_distance"]), _axis_bucket(dx, case["nx"], case["max_distance"])
    row = (j // gw)[None, :] - (i // gw)[:, None] + case["gh"] - 1
    col = (j % gw)[None, :] - (i % gw)[:, None] + gw - 1
    return by[row] * case["nx"] + bx[col]


def _members(size, n, max_distance, dev):
    """[size * size, n]: 1 where the pair (query, key) of positions on one axis belongs to the bucket."""
    at = torch.arange(size, device=dev)
    bucket = _axis_bucket(at[None, :] - at[:, None], n, max_distance).reshape(-1)
    return (bucket[:, None] == torch.arange(n, device=dev)).to(torch.float64)


def _attention_plain(s):
    c = s["case"]
    maps = 2 if c["op"] == "diff" else 1
    dt = _DTYPE[c["dtype"]]
    b, h, d, lq, lk = c["b"], c["heads"], c["d"], c["lq"], c["gh"] * c["gw"]
    q, k, v, table = (s[n].detach().to(F32) for n in ("q", "k", "v", "table"))
    sm = 1.0 / math.sqrt(d)
    q = q.view(b, lq, h, maps, d).permute(0, 2, 3, 1, 4).contiguous()      # [B, H, maps, Lq, D]
    k = k.view(b, lk, h, maps, d).permute(0, 2, 3, 1, 4).contiguous()
    v = v.permute(0, 2, 1, 3).contiguous()                                 # [B, H, Lk, Dv]
    index = _bucket_index(c, q.device)
    bias = table.view(-1, h)[index.reshape(-1)].view(lq, lk, h).permute(2, 0, 1)
    scores = torch.matmul(q, k.transpose(3, 4).contiguous()) * sm + bias[None, :, None]
    if s["lengths"] is not None:
        masked = torch.arange(lk, device=q.device)[None, :] >= s["lengths"][:, None]
        scores = scores.masked_fill(masked[:, None, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)         # a row without keys: zeros
    if maps == 2:
        lam = s["lam"].detach()[None, :, None, None]
        a = p[:, :, 0] - lam * p[:, :, 1]
    else:
        a = p[:, :, 0]
    out = torch.matmul(a, v).permute(0, 2, 1, 3).contiguous().to(dt)
    if not c["train"]:
        return {"out": out}
    dout = s["dout"].to(F32).permute(0, 2, 1, 3).contiguous()              # [B, H, Lq, Dv]
    dv = torch.matmul(a.transpose(2, 3).contiguous(), dout)
    dp = torch.matmul(dout, v.transpose(2, 3).contiguous())                # of the map that is added; the other's is -lam times it
    got = {"out": out, "dv": dv.permute(0, 2, 1, 3).contiguous().to(dt)}
    dp = dp[:, :, None]
    if maps == 2:
        got["dlam"] = -(p[:, :, 1] * dp[:, :, 0]).sum((2, 3), dtype=torch.float64).sum(0).to(F32)
        dp = torch.cat((dp, -lam[:, :, None] * dp), 2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    got["dq"] = (torch.matmul(ds, k) * sm).permute(0, 3, 1, 2, 4).reshape(b, lq, h * maps, d).to(dt)
    got["dk"] = (torch.matmul(ds.transpose(3, 4).contiguous(), q) * sm).permute(0, 3, 1, 2, 4).reshape(b, lk, h * maps, d).to(dt)
    # long sums, over the pairs of each bucket: pairs of rows and pairs of columns of the grid, one product for each axis
    gh, gw = c["gh"], c["gw"]
    pairs = ds.sum((0, 2), dtype=torch.float64).view(h, gh, gw, gh, gw).permute(0, 1, 3, 2, 4).reshape(h, gh * gh, gw * gw)
    by_column = torch.matmul(pairs, _members(gw, c["nx"], c["max_distance"], q.device))
    rows = torch.matmul(_members(gh, c["ny"], c["max_distance"], q.device).t().contiguous(), by_column)
    got["dtable"] = rows.permute(1, 2, 0).contiguous().to(F32)
    return got


def _normalised(v, kind, eps):
    v = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    rstd = 1.0 / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
    return v * rstd, rstd


def _norm_back(g, z, rstd, kind):
    g = g - g.mean(-1, keepdim=True) if kind == "layer" else g
    return rstd * (g - z * (g * z).mean(-1, keepdim=True))


def _norm_plain(s):
    c = s["case"]
    dt, kind, eps = _DTYPE[c["dtype"]], c["kind"], 1e-6
    x, f = s["x"].detach().to(F32), s["f"].detach().to(F32)
    scale, wp, wq = (s[n].detach() for n in ("scale", "post_weight", "pre_weight"))
    z, rf = _normalised(f, kind, eps)
    n = z * wp if s["post_bias"] is None else z * wp + s["post_bias"].detach()
    a = 1.0 / (1.0 + torch.exp(-s["gate"].detach().to(F32))) if s["gate"] is not None else torch.ones_like(x)
    y = x + scale * a * n
    zy, ry = _normalised(y, kind, eps)
    h = zy * wq if s["pre_bias"] is None else zy * wq + s["pre_bias"].detach()
    got = {"y": y.to(dt), "h": h.to(dt)}
    if not c["train"]:
        return got
    dy, dh = s["dy"].to(F32), s["dh"].to(F32)
    total = lambda t: t.sum(0, dtype=torch.float64).to(F32)  # noqa: E731   long sums
    du = dy + _norm_back(dh * wq, zy, ry, kind)
    dn = du * scale * a
    got.update(dx=du.to(dt), df=_norm_back(dn * wp, z, rf, kind).to(dt), dscale=total(du * a * n), dpost_weight=total(dn * z),
               dpre_weight=total(dh * zy))
    if s["gate"] is not None:
        got["dgate"] = (du * scale * n * a * (1.0 - a)).to(dt)
    if kind == "layer":
        got.update(dpost_bias=total(dn), dpre_bias=total(dh))
    return got


# --------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if not own:
        return _norm_plain(s) if c["op"] == "norm" else _attention_plain(s)
    from im2im_uq_amd import attn_ops
    if c["op"] == "norm":
        y, h = attn_ops.norm_gate_residual(s["x"], s["f"], gate=s["gate"], scale=s["scale"], post_weight=s["post_weight"],
                                           post_bias=s["post_bias"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"],
                                           norm=c["kind"], eps=1e-6)
        got, outs, douts = {"y": y, "h": h}, (y, h), (s["dy"], s["dh"])
    else:
        at = dict(grid=(c["gh"], c["gw"]), max_distance=c["max_distance"], lengths=s["lengths"], q_start=c["q_start"])
        if c["op"] == "diff":
            out = attn_ops.diff_grid_attention(s["q"], s["k"], s["v"], s["lam"], s["table"], **at)
        else:
            out = attn_ops.grid_attention(s["q"], s["k"], s["v"], s["table"], **at)
        got, outs, douts = {"out": out}, (out,), (s["dout"],)
    if c["train"]:
        for name, grad in zip(s["leaves"], torch.autograd.grad(outs, [s[n] for n in s["leaves"]], douts)):
            got["d" + name] = grad
    return got


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_lookup(table, case):
    """The bias of every query and key from the buckets' definition: logarithms in 64 bits, nudged over the borders they meet exactly."""
    def axis(rel, n):
        if n == 1:
            return rel * 0
        side = max(1, n // 2)
        few = max(1, side // 2)
        t = rel.abs().double()
        far = few + torch.floor(torch.log(t.clamp(min=1) / few) / math.log(case["max_distance"] / few) * (side - few) + 1e-9)
        one = torch.where(t < few, t, far.clamp(max=side - 1)).long().clamp(max=side - 1)
        return one + torch.where(rel > 0, side, 0)
    at = torch.arange(case["gh"] * case["gw"], device=table.device)
    ys, xs = torch.div(at, case["gw"], rounding_mode="floor"), at % case["gw"]
    mine = slice(case["q_start"], case["q_start"] + case["lq"])
    return axis(ys[None, :] - ys[mine, None], case["ny"]), axis(xs[None, :] - xs[mine, None], case["nx"])


def _exact_attention(s):
    c = s["case"]
    maps, d = (2 if c["op"] == "diff" else 1), c["d"]
    q, k, v, table = (s[n].detach().double() for n in ("q", "k", "v", "table"))
    dout = s["dout"].double()
    lam = s["lam"].detach().double() if maps == 2 else None
    by, bx = _exact_lookup(table, c)
    rows = by * c["nx"] + bx
    out, dq, dk, dv = torch.zeros_like(dout), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dtable = torch.zeros(c["ny"] * c["nx"], c["heads"], dtype=torch.float64, device=q.device)
    dlam = torch.zeros(c["heads"], dtype=torch.float64, device=q.device)
    for b in range(c["b"]):
        n = k.shape[1] if s["lengths"] is None else int(s["lengths"][b])
        if n == 0:
            continue
        for h in range(c["heads"]):
            bias = table[by[:, :n], bx[:, :n], h]
            vv, dd = v[b, :n, h], dout[b, :, h]
            probs = [torch.softmax(q[b, :, maps * h + m] @ k[b, :n, maps * h + m].T / math.sqrt(d) + bias, -1) for m in range(maps)]
            weight = [1.0, -float(lam[h])][:maps] if maps == 2 else [1.0]
            mixed = sum(w * p for w, p in zip(weight, probs))
            out[b, :, h] = mixed @ vv
            if not c["train"]:
                continue
            dv[b, :n, h] = mixed.T @ dd
            dmix = dd @ vv.T
            for m, (w, p) in enumerate(zip(weight, probs)):
                g = p * (w * dmix - (p * (w * dmix)).sum(-1, keepdim=True))
                dq[b, :, maps * h + m] = g @ k[b, :n, maps * h + m] / math.sqrt(d)
                dk[b, :n, maps * h + m] = g.T @ q[b, :, maps * h + m] / math.sqrt(d)
                dtable[:, h].index_add_(0, rows[:, :n].reshape(-1), g.reshape(-1))
            if maps == 2:
                dlam[h] -= (probs[1] * dmix).sum()
    got = {"out": out}
    if c["train"]:
        got.update(dq=dq, dk=dk, dv=dv, dtable=dtable.view(c["ny"], c["nx"], -1))
        if maps == 2:
            got["dlam"] = dlam
    return got


def _exact_norm(s):
    c = s["case"]
    names = s["leaves"]
    t = {n: s[n].detach().double().requires_grad_(c["train"]) for n in names}

    def normed(v, w, b):
        if c["kind"] == "layer":
            v = v - v.mean(1, keepdim=True)
        v = v / (v.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * t[w]
        return v + t[b] if b in t else v

    u = normed(t["f"], "post_weight", "post_bias") * t["scale"]
    y = t["x"] + (u * torch.sigmoid(t["gate"]) if "gate" in t else u)
    h = normed(y, "pre_weight", "pre_bias")
    got = {"y": y.detach(), "h": h.detach()}
    if c["train"]:
        grads = torch.autograd.grad((y, h), [t[n] for n in names], (s["dy"].double(), s["dh"].double()))
        got.update(("d" + n, g) for n, g in zip(names, grads))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["op"] == "norm" else _exact_attention(s)
