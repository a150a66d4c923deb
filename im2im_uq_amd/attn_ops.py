"""Operators of an attention bottleneck over the HIP kernels (C ABI in include/im2im_uq.h): attention on an image grid with a learned
relative position bias, its differential form, and the norms between blocks fused with their gate and residual.

Tokens are the pixels of a feature map in raster order: a channels-last [B, C, H, W] activation read as [B, H * W, C] is a view.  The reference's
trunk has no attention (core/models/trunks/unet.py:33-46); `UNet(attention=...)` puts these between its last Down and its first Up block.

All operators take and return GPU tensors in fp32 or bf16 with fp32 parameters (as the convolutions do), launch on torch's current stream,
allocate what they need there, never synchronise, and can be captured into a HIP graph.  Softmax statistics and every sum are 32-bit or
wider, in one fixed order: a repeated call gives the same bits.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib
from ._lib import AttentionDesc, AttentionGrads, Im2ImError, NormGateDesc, check, lib

F32, BF16 = torch.float32, torch.bfloat16
_DT = {F32: 0, BF16: 1}
_NORM = {"rms": 0, "layer": 1}
MAX_BUCKETS = 64           # of one axis
MAX_GRID_WIDTH = 512       # of a grid with more than one row
MAX_NORM_CHANNELS = 8192


@functools.lru_cache(maxsize=256)
def bucket_thresholds(n: int, max_distance: int):
    """smallest distances of the buckets 1, 2, ... of one direction of an axis with `n` buckets (see grid_attention): distances below
    half of a direction's buckets have one each, the others share the rest evenly in the distance's logarithm up to `max_distance`.
    Decided in whole numbers: bucket >= m iff (t / e) ** (half - e) >= (max_distance / e) ** (m - e)."""
    if n != 1 and (n < 2 or n % 2 or n > MAX_BUCKETS):
        raise Im2ImError(f"buckets of an axis: 1 or an even number up to {MAX_BUCKETS}, got {n}")
    half = max(1, n // 2)
    e = max(1, half // 2)
    if half > e and not e < max_distance <= 1 << 24:
        raise Im2ImError(f"max_distance must lie over {e} (the exact buckets of {n}) and be at most 2**24, got {max_distance}")
    thr = []
    for m in range(1, half):
        lo, hi = min(m, e), max(m, max_distance)
        if m > e:
            bound = max_distance ** (m - e) * e ** (half - e)
            while lo < hi:                                   # the first t with t ** (half - e) * e ** (m - e) >= bound
                mid = (lo + hi) // 2
                lo, hi = (lo, mid) if mid ** (half - e) * e ** (m - e) >= bound else (mid + 1, hi)
        thr.append(lo)
    return tuple(thr)


@functools.lru_cache(maxsize=256)
def _thresholds_arg(n, max_distance):
    thr = bucket_thresholds(n, max_distance)
    return (ctypes.c_int32 * len(thr))(*thr) if thr else None


def _fail(what):
    raise Im2ImError(what)


def _on_gpu(name, t, device=None):
    if not isinstance(t, torch.Tensor):
        _fail(f"{name}: expected a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        _fail(f"{name} must live on the GPU; the HIP path has no CPU fallback (got {t.device})")
    if device is not None and t.device != device:
        _fail(f"{name} is on {t.device}, the other operands on {device}")


def _parameter(name, t, shape, device):
    _on_gpu(name, t, device)
    if t.dtype != F32 or tuple(t.shape) != shape:
        _fail(f"{name}: expected fp32 {list(shape)}, got {t.dtype} {list(t.shape)}")


def _rows16(t):
    """`t` with its last index dense and every row at 16 bytes, as the kernels read it (a copy only where it is not)"""
    e = t.element_size()
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s * e % 16 == 0 for s in t.stride()[:-1])
    return t if ok else _dense16(t)


def _dense16(t):
    t = t if t.is_contiguous() else t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _on:
    """the operands' device as the current one, for the launches (torch.cuda.device only where it is another)"""
    __slots__ = ("idx", "guard")

    def __init__(self, device):
        self.idx = device.index

    def __enter__(self):
        self.guard = None
        if self.idx != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.idx)
            self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


class _Plan:
    """the whole numbers of a call"""
    __slots__ = ("heads", "d", "maps", "gh", "gw", "my", "mx", "q_start", "scale")


def _describe(plan, q, k, v, line, lengths, lam):
    p = AttentionDesc()
    p.q, p.k, p.v, p.line = q.data_ptr(), k.data_ptr(), v.data_ptr(), line.data_ptr()
    p.lengths = None if lengths is None else lengths.data_ptr()
    p.lam = None if lam is None else lam.data_ptr()
    p.q_stride[:], p.k_stride[:], p.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    p.B, p.Lq, p.Lk, p.H, p.D, p.maps = q.shape[0], q.shape[1], k.shape[1], plan.heads, plan.d, plan.maps
    p.gh, p.gw, p.q_start, p.dtype, p.scale = plan.gh, plan.gw, plan.q_start, _DT[q.dtype], plan.scale
    return p


def _forward(plan, q, k, v, table, lam, lengths, keep):
    """(out, line, lse, map_out); the last two only with `keep`"""
    dev = q.device
    b, lq, h, maps = q.shape[0], q.shape[1], plan.heads, plan.maps
    dv = plan.d * maps
    out = torch.empty((b, lq, h, dv), dtype=q.dtype, device=dev)
    ny, nx = table.shape[0], table.shape[1]
    line = torch.empty((h, (2 * plan.gh - 1) * (2 * plan.gw - 1)), dtype=F32, device=dev)
    lse = torch.empty((b * h, maps, lq), dtype=F32, device=dev) if keep else None
    map_out = torch.empty((b * h, lq, maps, dv), dtype=F32, device=dev) if keep else None
    with _on(dev) as stream:
        check(lib.im2im_relpos_line(table.data_ptr(), ny, nx, h, _thresholds_arg(ny, plan.my), _thresholds_arg(nx, plan.mx), plan.gh, plan.gw,
                                    line.data_ptr(), stream), "im2im_relpos_line")
        p = _describe(plan, q, k, v, line, lengths, lam)
        n = lib.im2im_attention_fwd_workspace_bytes(ctypes.byref(p))
        if n < 0:
            check(-1, "im2im_attention_fwd")
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        check(lib.im2im_attention_fwd(ctypes.byref(p), out.data_ptr(), lse.data_ptr() if keep else None, map_out.data_ptr() if keep else None,
                                      ws.data_ptr() if n else None, n, stream), "im2im_attention_fwd")
    return out, line, lse, map_out


def _backward(plan, q, k, v, table_shape, line, lam, lengths, lse, map_out, dout, dq, dk, dv, want_table):
    """fills dq, dk, dv ([B, L, heads, D] views); returns (dtable | None, dlam | None)"""
    dev = q.device
    dout = _dense16(dout if dout.dtype == q.dtype else dout.to(q.dtype))
    dtable = torch.empty(table_shape, dtype=F32, device=dev) if want_table else None
    dlam = torch.empty(plan.heads, dtype=F32, device=dev) if plan.maps == 2 else None
    with _on(dev) as stream:
        p = _describe(plan, q, k, v, line, lengths, lam)
        g = AttentionGrads()
        g.dout, g.lse, g.map_out = dout.data_ptr(), lse.data_ptr(), map_out.data_ptr()
        g.dq, g.dk, g.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        g.dq_stride[:], g.dk_stride[:], g.dv_stride[:] = dq.stride()[:3], dk.stride()[:3], dv.stride()[:3]
        g.dtable, g.dlam = dtable.data_ptr() if want_table else None, dlam.data_ptr() if dlam is not None else None
        ty, tx = _thresholds_arg(table_shape[0], plan.my), _thresholds_arg(table_shape[1], plan.mx)
        g.thr_y, g.thr_x = ctypes.cast(ty, ctypes.c_void_p), ctypes.cast(tx, ctypes.c_void_p)
        g.ny, g.nx = table_shape[0], table_shape[1]
        n = lib.im2im_attention_bwd_workspace_bytes(ctypes.byref(p), int(want_table))
        if n < 0:
            check(-1, "im2im_attention_bwd")
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        check(lib.im2im_attention_bwd(ctypes.byref(p), ctypes.byref(g), ws.data_ptr(), n, stream), "im2im_attention_bwd")
    return dtable, dlam


class _GridAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, lam, lengths, plan, keep):
        table, lam = table.contiguous(), None if lam is None else lam.contiguous()
        out, line, lse, map_out = _forward(plan, q, k, v, table, lam, lengths, keep)
        if keep:
            ctx.plan, ctx.table_shape = plan, tuple(table.shape)
            ctx.save_for_backward(q, k, v, line, lam, lengths, lse, map_out)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, line, lam, lengths, lse, map_out = ctx.saved_tensors
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        dtable, dlam = _backward(ctx.plan, q, k, v, ctx.table_shape, line, lam, lengths, lse, map_out, dout, dq, dk, dv, ctx.needs_input_grad[3])
        return dq, dk, dv, dtable, dlam, None, None, None


class _GridSelfAttention(torch.autograd.Function):
    """q, k and v side by side in one tensor: their gradients leave in one tensor too, without the copies that three slices would cost"""

    @staticmethod
    def forward(ctx, qkv, table, lam, plan, keep):
        table, lam = table.contiguous(), None if lam is None else lam.contiguous()
        qkv = _rows16(qkv)
        out, line, lse, map_out = _forward(plan, *_split_qkv(qkv, plan), table, lam, None, keep)
        if keep:
            ctx.plan, ctx.table_shape = plan, tuple(table.shape)
            ctx.save_for_backward(qkv, line, lam, lse, map_out)
        return out.view(out.shape[0], out.shape[1], -1)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, line, lam, lse, map_out = ctx.saved_tensors
        plan = ctx.plan
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        dout = dout.reshape(qkv.shape[0], qkv.shape[1], plan.heads, plan.d * plan.maps)
        dtable, dlam = _backward(plan, *_split_qkv(qkv, plan), ctx.table_shape, line, lam, None, lse, map_out, dout, *_split_qkv(dqkv, plan),
                                 ctx.needs_input_grad[1])
        return dqkv, dtable, dlam, None, None


def _split_qkv(t, plan):
    b, n, c3 = t.shape
    c = c3 // 3
    q, k, v = t[..., :c], t[..., c:2 * c], t[..., 2 * c:]
    maps, h, d = plan.maps, plan.heads, plan.d
    return q.unflatten(2, (h * maps, d)), k.unflatten(2, (h * maps, d)), v.unflatten(2, (h, d * maps))


def _make_plan(maps, heads, d, dtype, table, lam, grid, max_distance, lk, lq, q_start, scale, device):
    if dtype not in _DT:
        _fail(f"q, k, v: fp32 or bf16, got {dtype}")
    if heads < 1 or d < 8 or d % 8 or d * maps > 128:
        _fail(f"head size: a multiple of 8 up to {128 // maps} with {maps} map(s), got {d} ({heads} heads)")
    p = _Plan()
    try:
        p.gh, p.gw = (int(x) for x in grid)
        p.my, p.mx = (int(x) for x in max_distance) if isinstance(max_distance, (tuple, list)) else (int(max_distance),) * 2
    except (TypeError, ValueError):
        _fail(f"grid = (height, width) and max_distance = a number or (vertical, horizontal), got {grid!r}, {max_distance!r}")
    if p.gh < 1 or p.gw < 1 or p.gh * p.gw > 1 << 24 or (p.gh > 1 and p.gw > MAX_GRID_WIDTH):
        _fail(f"grid {grid}: at least 1 x 1, at most 2**24 tokens, and at most {MAX_GRID_WIDTH} wide unless it is one row")
    if lk > p.gh * p.gw:
        _fail(f"{lk} keys do not fit the grid {grid}")
    if q_start < 0 or q_start + lq > p.gh * p.gw:
        _fail(f"queries {q_start} .. {q_start + lq - 1} are not tokens of the grid {grid}")
    _on_gpu("table", table, device)
    if table.dtype != F32 or table.dim() != 3 or table.shape[2] != heads:
        _fail(f"table: expected fp32 [vertical buckets, horizontal buckets, {heads}], got {table.dtype} {list(table.shape)}")
    bucket_thresholds(table.shape[0], p.my)
    bucket_thresholds(table.shape[1], p.mx)
    if maps == 2:
        _parameter("lam", lam, (heads,), device)
    p.heads, p.d, p.maps, p.q_start = heads, d, maps, q_start
    p.scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not math.isfinite(p.scale):
        _fail(f"scale must be finite, got {scale}")
    return p


def _attend(maps, q, k, v, lam, table, grid, max_distance, lengths, q_start, scale):
    _on_gpu("q", q)
    _on_gpu("k", k, q.device)
    _on_gpu("v", v, q.device)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        _fail(f"q, k, v: expected [batch, tokens, heads, channels], got {list(q.shape)}, {list(k.shape)}, {list(v.shape)}")
    if not q.dtype == k.dtype == v.dtype:
        _fail(f"q, k, v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    b, lq, hm, d = q.shape
    lk, h = k.shape[1], v.shape[2]
    if hm != h * maps or tuple(k.shape) != (b, lk, hm, d) or tuple(v.shape) != (b, lk, h, d * maps):
        _fail(f"shapes do not belong together: q {list(q.shape)}, k {list(k.shape)}, v {list(v.shape)} with {maps} map(s): k [batch, keys, "
              f"{maps} * heads, D], v [batch, keys, heads, {maps} * D]")
    plan = _make_plan(maps, h, d, q.dtype, table, lam, grid, max_distance, lk, lq, q_start, scale, q.device)
    if lengths is not None:
        _on_gpu("lengths", lengths, q.device)
        if lengths.dtype != torch.int32 or tuple(lengths.shape) != (b,):
            _fail(f"lengths: expected int32 [{b}], got {lengths.dtype} {list(lengths.shape)}")
        lengths = lengths.contiguous()
    needs = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or table.requires_grad
                                         or (lam is not None and lam.requires_grad))
    if b * lq == 0:                                          # nothing is asked for
        return v.new_empty((b, lq, h, d * maps)) + 0 * q.sum() if needs else v.new_empty((b, lq, h, d * maps))
    if lk == 0:
        _fail("k, v: no keys (lengths may be 0, the tensors not)")
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    if not needs:
        return _forward(plan, q, k, v, table.contiguous(), None if lam is None else lam.contiguous(), lengths, False)[0]
    return _GridAttention.apply(q, k, v, table, lam, lengths, plan, True)


def grid_attention(q, k, v, table, grid, max_distance=64, lengths=None, q_start=0, scale=None):
    """softmax attention over the pixels of an image grid with a learned relative position bias by buckets

        out_i = sum_j softmax_j(scale q_i . k_j + table[by(y_j - y_i), bx(x_j - x_i), head]) v_j

    q [B, Lq, heads, D], k, v [B, Lk, heads, D], fp32 or bf16; D a multiple of 8 up to 128; any strides (rows that do not start at 16
    bytes are copied).  Returns [B, Lq, heads, D] in their type.
    grid = (height, width): token t is the pixel (t // width, t % width).  The keys are the tokens 0 .. Lk - 1, the queries the tokens
    q_start .. q_start + Lq - 1 (all pixels, a band of them, or a single one).  (1, n): a row of n tokens.
    table [ny, nx, heads] fp32: ny and nx buckets for the two axes (each 1, or an even number up to 64: the lower half for distances
    <= 0, the upper half for those > 0; bucket_thresholds has the borders; from `max_distance` on they share the last one).
    An entry of -inf masks its pairs.
    lengths [B] int32 (on the GPU, clipped to 0 .. Lk): keys from there on take no part, whatever they hold; with none left a
    row gives zeros.  scale: 1 / sqrt(D) unless given.
    Gradients: q, k, v, table."""
    return _attend(1, q, k, v, None, table, grid, max_distance, lengths, q_start, scale)


def diff_grid_attention(q, k, v, lam, table, grid, max_distance=64, lengths=None, q_start=0, scale=None):
    """differential attention on the grid: the difference of two softmax maps, out = (P_0 - lam[head] P_1) v

    q, k [B, L, 2 * heads, D] (map m of head h is their head 2 h + m), v [B, Lk, heads, 2 * D], D a multiple of 8 up to 64, lam [heads] fp32;
    both maps of a head share its bias.  Returns [B, Lq, heads, 2 * D].  Everything else as in grid_attention.
    Gradients: q, k, v, lam, table."""
    return _attend(2, q, k, v, lam, table, grid, max_distance, lengths, q_start, scale)


def grid_self_attention(qkv, heads, table, grid, lam=None, max_distance=64, scale=None):
    """grid_attention (lam given: diff_grid_attention) of a whole grid with itself from one projection: qkv [B, height * width, 3 C] holds q, k
    and v side by side, C = heads * D (differential: C = heads * 2 * D), and so does its gradient.  Returns [B, height * width, C]."""
    _on_gpu("qkv", qkv)
    maps = 1 if lam is None else 2
    if qkv.dim() != 3 or heads < 1 or qkv.shape[2] % (3 * heads * maps):
        _fail(f"qkv: expected [batch, tokens, 3 * C] with C a multiple of {heads} heads x {maps} map(s), got {list(qkv.shape)}")
    b, n, c3 = qkv.shape
    plan = _make_plan(maps, heads, c3 // (3 * heads * maps), qkv.dtype, table, lam, grid, max_distance, n, n, 0, scale, qkv.device)
    if n != plan.gh * plan.gw:
        _fail(f"{n} tokens are not the grid {grid}")
    if b == 0:
        return qkv[..., :c3 // 3]
    keep = torch.is_grad_enabled() and (qkv.requires_grad or table.requires_grad or (lam is not None and lam.requires_grad))
    return _GridSelfAttention.apply(qkv, table, lam, plan, keep)


# ---------------------------------------------------------------------------------------------------------------------- norms
class _Seam:
    """what a norm_gate_residual call is, beside its tensors"""
    __slots__ = ("norm", "eps", "rows", "c", "shape")


def _rows_of(t, shape):
    """`t` as [rows, C] with dense channels and one stride between its rows, and that stride (a copy only where there is none)"""
    if t.stride(-1) == 1 or shape[-1] == 1:
        stride, size, ok = None, 1, True
        for n, s in zip(reversed(shape[:-1]), reversed(t.stride()[:-1])):
            if n == 1:
                continue
            stride = s if stride is None else stride
            ok = ok and s == stride * size
            size *= n
        if ok and (stride is None or stride >= 0):
            return t, shape[-1] if stride is None else stride
    return t.contiguous(), shape[-1]


def _seam_desc(s, x, f, gate, params):
    p = NormGateDesc()
    for name, t in (("x", x), ("f", f), ("gate", gate)):
        if t is not None:
            t, stride = t
            setattr(p, name, t.data_ptr())
            setattr(p, name + "_stride", stride)
    p.scale, p.post_weight, p.post_bias, p.pre_weight, p.pre_bias = (None if t is None else t.data_ptr() for t in params)
    p.rows, p.C, p.norm, p.dtype, p.eps = s.rows, s.c, s.norm, _DT[x[0].dtype], s.eps
    return p


def _seam_forward(s, x, f, gate, params):
    x, f, gate = (None if t is None else _rows_of(t, s.shape) for t in (x, f, gate))
    params = [None if t is None else _dense16(t) for t in params]
    dev, dt = x[0].device, x[0].dtype
    y = torch.empty(s.shape, dtype=dt, device=dev) if f is not None else None
    h = torch.empty(s.shape, dtype=dt, device=dev) if params[3] is not None else None
    with _on(dev) as stream:
        check(lib.im2im_norm_gate_fwd(ctypes.byref(_seam_desc(s, x, f, gate, params)), None if y is None else y.data_ptr(),
                                      None if h is None else h.data_ptr(), stream), "im2im_norm_gate_fwd")
    return y, h


class _NormGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s, x, f, gate, *params):
        ctx.s = s
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, f, gate, *params)
        y, h = _seam_forward(s, x, f, gate, params)
        return (y, h) if f is not None and h is not None else h if f is None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        s = ctx.s
        x, f, gate, *params = ctx.saved_tensors
        has_y, has_h = f is not None, params[3] is not None
        dy, dh = grads if has_y and has_h else (grads[0], None) if has_y else (None, grads[0])
        if dy is None and dh is None:
            return (None,) * 9
        dev, dt = x.device, x.dtype
        dy, dh = (None if t is None else (t if t.dtype == dt else t.to(dt)).contiguous() for t in (dy, dh))
        need = ctx.needs_input_grad[1:]
        rows = [torch.empty(s.shape, dtype=dt, device=dev) if t is not None and n else None for t, n in zip((x, f, gate), need)]
        want = [t is not None and n for t, n in zip(params, need[3:])]
        sums = [torch.empty(s.c, dtype=F32, device=dev) if w and (i < 3 or dh is not None) else None for i, w in enumerate(want)]
        params = [None if t is None else _dense16(t) for t in params]
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        with _on(dev) as stream:
            n = lib.im2im_norm_gate_bwd_workspace_bytes(s.rows, s.c)
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            desc = _seam_desc(s, *(None if t is None else _rows_of(t, s.shape) for t in (x, f, gate)), params)
            check(lib.im2im_norm_gate_bwd(ctypes.byref(desc), ptr(dy), ptr(dh), *(ptr(t) for t in rows), *(ptr(t) for t in sums), ws.data_ptr(), n,
                                          stream), "im2im_norm_gate_bwd")
        sums = [torch.zeros(s.c, dtype=F32, device=dev) if w and t is None else t for w, t in zip(want, sums)]
        return (None, *rows, *sums)


def norm_gate_residual(x, f, gate=None, scale=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, norm="rms", eps=1e-6):
    """the seam between two blocks in one pass:  y = x + scale * sigmoid(gate) * N_post(f),  h = N_pre(y)

    x: the residual stream, f: the block's output, gate: its gate's logits (or None), all [..., C] of one type (fp32 or bf16) and shape, any
    strides (expanded ones too: their gradient is the sum).  scale, the weights and biases: fp32 [C]; scale (residual scale), the biases
    and pre_weight may be None.  N: "rms" (root mean square, no bias) or "layer" over the last index, C <= 8192; h is taken from y before y is rounded.
    Returns (y, h); h is None without pre_weight.  Gradients: everything that is a tensor."""
    return _seam(x, f, gate, scale, post_weight, post_bias, pre_weight, pre_bias, norm, eps)


def token_norm(x, weight, bias=None, norm="rms", eps=1e-6):
    """N_pre of norm_gate_residual alone: the norm in front of the first block"""
    return _seam(x, None, None, None, None, None, weight, bias, norm, eps)


def _seam(x, f, gate, scale, post_weight, post_bias, pre_weight, pre_bias, norm, eps):
    _on_gpu("x", x)
    if norm not in _NORM:
        _fail(f"norm must be 'rms' or 'layer', got {norm!r}")
    if x.dtype not in _DT or x.dim() < 1:
        _fail(f"x: expected fp32 or bf16 [..., C], got {x.dtype} {list(x.shape)}")
    if not (isinstance(eps, (int, float)) and 0 < eps < math.inf and ctypes.c_float(eps).value > 0):
        _fail(f"eps must be a positive number, got {eps!r}")
    c = x.shape[-1]
    if not 1 <= c <= MAX_NORM_CHANNELS:
        _fail(f"x: 1 to {MAX_NORM_CHANNELS} channels, got {c}")
    for name, t in (("f", f), ("gate", gate)):
        if t is not None:
            _on_gpu(name, t, x.device)
            if t.dtype != x.dtype or t.shape != x.shape:
                _fail(f"{name}: expected {x.dtype} {list(x.shape)} as x, got {t.dtype} {list(t.shape)}")
    params = (scale, post_weight, post_bias, pre_weight, pre_bias)
    for name, t in zip(("scale", "post_weight", "post_bias", "pre_weight", "pre_bias"), params):
        if t is not None:
            _parameter(name, t, (c,), x.device)
    if f is None and pre_weight is None:
        _fail("weight is missing")
    if f is not None and post_weight is None:
        _fail("f needs post_weight")
    if norm == "rms" and (post_bias is not None or pre_bias is not None):
        _fail("a root-mean-square norm has no bias")
    if pre_bias is not None and pre_weight is None:
        _fail("pre_bias needs pre_weight")
    s = _Seam()
    s.norm, s.eps, s.c, s.shape, s.rows = _NORM[norm], float(eps), c, tuple(x.shape), x.numel() // c
    if s.rows == 0:
        y = None if f is None else x + 0 * f
        h = None if pre_weight is None else x * pre_weight.to(x.dtype)
        return h if f is None else (y, h)
    tensors = (x, f, gate, *params)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        got = _NormGate.apply(s, *tensors)
        return got if f is None or pre_weight is not None else (got, None)
    y, h = _seam_forward(s, x, f, gate, params)
    return h if f is None else (y, h)

