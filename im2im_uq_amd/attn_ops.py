"""Operators of an attention bottleneck over the HIP kernels (C ABI in include/im2im_uq.h): attention on an image grid with a learned
relative position bias, its differential form, and the norms between blocks fused with their gate and residual.

Tokens are the pixels of a feature map in raster order: a channels-last [B, C, H, W] activation read as [B, H * W, C] is a view.  The reference's
trunk has no attention (core/models/trunks/unet.py:33-46); `UNet(attention=...)` puts these between its last Down and its first Up block.

All operators take and return GPU tensors in fp32 or bf16 with fp32 parameters (as the convolutions do), launch on torch's current stream,
allocate what they need there, never synchronise, and can be captured into a HIP graph.  Softmax statistics and every sum are 32-bit or
wider, in one fixed order: a repeated call gives the same bits; a bf16 result is 32-bit arithmetic that is rounded once.  Second derivatives and forward-mode tangents
are refused.
"""
from __future__ import annotations

import ctypes
import functools
import math
import operator

import torch
from torch.autograd import forward_ad

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


def _is(t, dtype, shape, device):
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device


def _parameter(name, t, shape, device):
    if _is(t, F32, shape, device):
        return
    _on_gpu(name, t, device)
    if t.dtype != F32 or tuple(t.shape) != shape:
        _fail(f"{name}: expected fp32 {list(shape)}, got {t.dtype} {list(t.shape)}")


def _dense16(t):
    """`t` dense and at 16 bytes"""
    t = t if t.is_contiguous() else t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows16(t):
    """`t` with its last index dense and every row at 16 bytes, as the kernels read it (a copy only where it is not)"""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():                                # heads are multiples of 16 bytes long
            return t
        e, strides = t.element_size(), t.stride()
        if strides[-1] == 1 and all(s * e % 16 == 0 for s in strides[:-1]) and strides[1] * e < 1 << 25:
            return t
    return _dense16(t)


def _like(t):
    """a dense tensor of t's shape (for a dense t empty_like is the shorter call; the strides that it keeps of sizes of one are never read)"""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _guard(device):
    """the operands' device made the current one for the launches; None where it is already"""
    if device.index == torch._C._cuda_getDevice():
        return None
    guard = torch.cuda.device(device.index)
    guard.__enter__()
    return guard


class _Plan:
    """what a call is, beside its tensors: settled once for each combination of sizes (plain numbers only)"""
    __slots__ = ("heads", "d", "maps", "batch", "grid", "desc", "desc_qkv", "grads", "grads_qkv", "table_shape", "thr", "out_shape", "save", "fwd_ws",
                 "bwd_ws", "lse_at", "map_at")


@functools.lru_cache(maxsize=1024)
def _plan(maps, q_shape, k_shape, v_shape, dtype, table_shape, grid, max_distance, scale):
    if dtype not in _DT:
        _fail(f"q, k, v: fp32 or bf16, got {dtype}")
    if not len(q_shape) == len(k_shape) == len(v_shape) == 4:
        _fail(f"q, k, v: expected [batch, tokens, heads, channels], got {list(q_shape)}, {list(k_shape)}, {list(v_shape)}")
    b, lq, hm, d = q_shape
    lk, heads = k_shape[1], v_shape[2]
    if hm != heads * maps or tuple(k_shape) != (b, lk, hm, d) or tuple(v_shape) != (b, lk, heads, d * maps):
        _fail(f"shapes do not belong together: q {list(q_shape)}, k {list(k_shape)}, v {list(v_shape)} with {maps} map(s): k [batch, keys, "
              f"{maps} * heads, D], v [batch, keys, heads, {maps} * D]")
    if heads < 1 or d < 8 or d % 8 or d * maps > 128:
        _fail(f"head size: a multiple of 8 up to {128 // maps} with {maps} map(s), got {d} ({heads} heads)")
    try:
        gh, gw = (int(x) for x in grid)
        my, mx = (int(x) for x in max_distance) if isinstance(max_distance, tuple) else (int(max_distance),) * 2
    except (TypeError, ValueError):
        _fail(f"grid = (height, width) and max_distance = a number or (vertical, horizontal), got {grid!r}, {max_distance!r}")
    if gh < 1 or gw < 1 or gh * gw > 1 << 24 or (gh > 1 and gw > MAX_GRID_WIDTH):
        _fail(f"grid {grid}: at least 1 x 1, at most 2**24 tokens, and at most {MAX_GRID_WIDTH} wide unless it is one row")
    if lk > gh * gw:
        _fail(f"{lk} keys do not fit the grid {grid}")
    if lq > gh * gw:
        _fail(f"{lq} queries are not tokens of the grid {grid}")
    if len(table_shape) != 3 or table_shape[2] != heads:
        _fail(f"table: expected fp32 [vertical buckets, horizontal buckets, {heads}], got {list(table_shape)}")
    p = _Plan()
    p.thr = _thresholds_arg(table_shape[0], my), _thresholds_arg(table_shape[1], mx)
    p.heads, p.d, p.maps, p.table_shape, p.out_shape = heads, d, maps, tuple(table_shape), (b, lq, heads, d * maps)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not math.isfinite(scale):
        _fail(f"scale must be finite, got {scale}")
    if b * lq and lk == 0:
        _fail("k, v: no keys (lengths may be 0, the tensors not)")
    p.desc, p.batch, p.grid = None, b, (gh, gw)
    if b * lq == 0:
        return p
    # the description of dense operands with the pointers left open, and the sizes that follow from it
    t = p.desc = AttentionDesc()
    t.B, t.Lq, t.Lk, t.H, t.D, t.maps, t.gh, t.gw, t.dtype, t.scale = b, lq, lk, heads, d, maps, gh, gw, _DT[dtype], scale
    t.q = t.k = t.v = t.line = t.lam = 16
    t.ny, t.nx = table_shape[:2]
    t.thr_y, t.thr_x = (ctypes.cast(x, ctypes.c_void_p) for x in p.thr)
    c = heads * maps * d
    t.q_stride[:], t.k_stride[:], t.v_stride[:] = (lq * c, c, d), (lk * c, c, d), (lk * c, c, d * maps)
    p.fwd_ws = lib.im2im_attention_fwd_workspace_bytes(ctypes.byref(t))
    p.bwd_ws = [lib.im2im_attention_bwd_workspace_bytes(ctypes.byref(t), w) for w in (0, 1)]
    if p.fwd_ws < 0 or min(p.bwd_ws) < 0:
        check(-1, "im2im_attention_fwd")
    g = p.grads = AttentionGrads()
    g.dq_stride[:], g.dk_stride[:], g.dv_stride[:] = t.q_stride, t.k_stride, t.v_stride
    # the same for q, k and v side by side in one tensor
    p.desc_qkv, p.grads_qkv = AttentionDesc.from_buffer_copy(t), AttentionGrads.from_buffer_copy(g)
    for x in (p.desc_qkv.q_stride, p.desc_qkv.k_stride, p.grads_qkv.dq_stride, p.grads_qkv.dk_stride):
        x[:] = 3 * lk * c, 3 * c, d
    for x in (p.desc_qkv.v_stride, p.grads_qkv.dv_stride):
        x[:] = 3 * lk * c, 3 * c, d * maps
    # one buffer for the bias of every displacement (its begin) and what the backward needs; places in bytes, at 16
    up = lambda n: (4 * n + 15) // 16 * 16  # noqa: E731
    p.lse_at = up(heads * (2 * gh - 1) * (2 * gw - 1))
    p.map_at = p.lse_at + up(2 * b * heads * maps * lq)
    p.save = p.map_at + up(b * heads * lq * maps * d * maps)
    return p


def _describe(plan, q, k, v, lengths, lam, q_start):
    p = AttentionDesc.from_buffer_copy(plan.desc)
    p.q_start = q_start
    p.q, p.k, p.v, p.lengths, p.lam = q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(lengths), _ptr(lam)
    if not q.is_contiguous():
        p.q_stride[:] = q.stride()[:3]
    if not k.is_contiguous():
        p.k_stride[:] = k.stride()[:3]
    if not v.is_contiguous():
        p.v_stride[:] = v.stride()[:3]
    return p


def _describe_qkv(plan, qkv, lam):
    p = AttentionDesc.from_buffer_copy(plan.desc_qkv)
    at, step = qkv.data_ptr(), plan.heads * plan.maps * plan.d * qkv.element_size()
    p.q, p.k, p.v, p.lam = at, at + step, at + 2 * step, _ptr(lam)
    return p


def _forward(plan, p, dtype, dev, table, keep):
    """(out, saved) for the description `p` (its line is filled in): `saved` holds the line, the rows' references and log-sums, and map results"""
    out = torch.empty(plan.out_shape, dtype=dtype, device=dev)
    ws = torch.empty(plan.fwd_ws, dtype=torch.uint8, device=dev) if plan.fwd_ws else None
    guard = _guard(dev)
    try:
        stream = torch._C._cuda_getCurrentRawStream(dev.index)
        if not keep and plan.out_shape[1] == 1:              # one query: its bias comes from the table itself
            p.line, p.table = None, table.data_ptr()
            check(lib.im2im_attention_fwd(ctypes.byref(p), out.data_ptr(), None, None, _ptr(ws), plan.fwd_ws, stream), "im2im_attention_fwd")
            return out, None
        saved = torch.empty(plan.save if keep else plan.lse_at, dtype=torch.uint8, device=dev)
        p.line = line = saved.data_ptr()
        ny, nx, heads = plan.table_shape
        check(lib.im2im_relpos_line(table.data_ptr(), ny, nx, heads, plan.thr[0], plan.thr[1], plan.grid[0], plan.grid[1], line, stream), "im2im_relpos_line")
        check(lib.im2im_attention_fwd(ctypes.byref(p), out.data_ptr(), line + plan.lse_at if keep else None, line + plan.map_at if keep else None,
                                      _ptr(ws), plan.fwd_ws, stream), "im2im_attention_fwd")
    finally:
        if guard is not None:
            guard.__exit__(None, None, None)
    return out, saved


def _backward(plan, p, g, saved, dout, want_table):
    """launches the backward of the description `p`; `g` has the pointers of dq, dk, dv.  Returns (dtable | None, dlam | None)"""
    dev = saved.device
    line = saved.data_ptr()
    dtable = dlam = None
    g.dout, g.lse, g.map_out = dout.data_ptr(), line + plan.lse_at, line + plan.map_at
    if want_table:
        dtable = torch.empty(plan.table_shape, dtype=F32, device=dev)
        g.dtable = dtable.data_ptr()
    if plan.maps == 2:
        dlam = torch.empty(plan.heads, dtype=F32, device=dev)
        g.dlam = dlam.data_ptr()
    n = plan.bwd_ws[want_table]
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    guard = _guard(dev)
    try:
        check(lib.im2im_attention_bwd(ctypes.byref(p), ctypes.byref(g), ws.data_ptr(), n, torch._C._cuda_getCurrentRawStream(dev.index)), "im2im_attention_bwd")
    finally:
        if guard is not None:
            guard.__exit__(None, None, None)
    return dtable, dlam


def _once(backward):
    """once_differentiable, whose bookkeeping a first-order pass (no gradient mode in its backward) goes without"""
    strict = torch.autograd.function.once_differentiable(backward)
    return lambda ctx, *grads: strict(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)


class _GridAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, lam, lengths, plan, q_start):
        lam = None if lam is None else lam.contiguous()
        p = _describe(plan, q, k, v, lengths, lam, q_start)
        out, saved = _forward(plan, p, q.dtype, q.device, table.contiguous(), True)
        ctx.plan, ctx.q_start = plan, q_start
        ctx.save_for_backward(q, k, v, lam, lengths, saved)
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        q, k, v, lam, lengths, saved = ctx.saved_tensors
        plan = ctx.plan
        dq, dk, dv = _like(q), _like(k), _like(v)
        p = _describe(plan, q, k, v, lengths, lam, ctx.q_start)
        p.line = saved.data_ptr()
        g = AttentionGrads.from_buffer_copy(plan.grads)
        g.dq, g.dk, g.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        dout = _dense16(dout)
        dtable, dlam = _backward(plan, p, g, saved, dout, ctx.needs_input_grad[3])
        return dq, dk, dv, dtable, dlam, None, None, None


class _GridSelfAttention(torch.autograd.Function):
    """q, k and v side by side in one tensor: their gradients leave in one tensor too, without the copies that three slices would cost"""

    @staticmethod
    def forward(ctx, qkv, table, lam, plan):
        qkv = _dense16(qkv)
        lam = None if lam is None else lam.contiguous()
        out, saved = _forward(plan, _describe_qkv(plan, qkv, lam), qkv.dtype, qkv.device, table.contiguous(), True)
        ctx.plan = plan
        ctx.save_for_backward(qkv, lam, saved)
        return out.view(out.shape[0], out.shape[1], -1)

    @staticmethod
    @_once
    def backward(ctx, dout):
        qkv, lam, saved = ctx.saved_tensors
        plan = ctx.plan
        dqkv = _like(qkv)
        p = _describe_qkv(plan, qkv, lam)
        p.line = saved.data_ptr()
        g = AttentionGrads.from_buffer_copy(plan.grads_qkv)
        at, step = dqkv.data_ptr(), plan.heads * plan.maps * plan.d * dqkv.element_size()
        g.dq, g.dk, g.dv = at, at + step, at + 2 * step
        dout = _dense16(dout)
        dtable, dlam = _backward(plan, p, g, saved, dout, ctx.needs_input_grad[1])
        return dqkv, dtable, dlam, None


def _integers(name, x):
    """`x`, a number or a pair of them, as plain ints: nothing that could change enters a plan's key"""
    if type(x) is int or (type(x) is tuple and len(x) == 2 and type(x[0]) is int and type(x[1]) is int):
        return x
    try:
        return tuple(operator.index(n) for n in x) if isinstance(x, (tuple, list)) else operator.index(x)
    except (TypeError, RuntimeError):
        _fail(f"{name}: expected whole numbers, got {x!r}")


def _number(name, x):
    if x is None or type(x) is float:
        return x
    if isinstance(x, torch.Tensor):
        _fail(f"{name}: expected a number, got a tensor")
    try:
        return float(x)
    except (TypeError, ValueError):
        _fail(f"{name}: expected a number, got {x!r}")


def _needs_grad(*tensors):
    """whether autograd has a part in the call: a gradient is wanted, or an operand carries a forward-mode tangent (it need not require a gradient), which
    the autograd functions refuse"""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _nothing(out, needs, *tensors):
    """an empty result; where a gradient is wanted, one that every operand has a gradient of zeros through"""
    return sum((t[:0].sum() for t in tensors if t is not None), out).to(out.dtype) if needs else out


def _attend(maps, q, k, v, lam, table, grid, max_distance, lengths, q_start, scale):
    _on_gpu("q", q)
    dev = q.device
    _on_gpu("k", k, dev)
    _on_gpu("v", v, dev)
    _on_gpu("table", table, dev)
    if not q.dtype is k.dtype is v.dtype:
        _fail(f"q, k, v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    if table.dtype != F32:
        _fail(f"table: expected fp32, got {table.dtype}")
    plan = _plan(maps, q.shape, k.shape, v.shape, q.dtype, table.shape, _integers("grid", grid), _integers("max_distance", max_distance),
                 _number("scale", scale))
    q_start = _integers("q_start", q_start)                  # no part of the plan: token after token has another one
    (gh, gw), lq = plan.grid, plan.out_shape[1]
    if isinstance(q_start, tuple) or not 0 <= q_start <= gh * gw - lq:
        _fail(f"q_start = {q_start}: {lq} queries from there on are not tokens of the grid {grid}")
    if maps == 2:
        _parameter("lam", lam, (plan.heads,), dev)
    if lengths is not None:
        _on_gpu("lengths", lengths, dev)
        if lengths.dtype != torch.int32 or lengths.shape != (plan.batch,):
            _fail(f"lengths: expected int32 [{plan.batch}], got {lengths.dtype} {list(lengths.shape)}")
        lengths = lengths.contiguous()
    needs = _needs_grad(q, k, v, table, lam)
    if plan.desc is None:                                    # nothing is asked for
        return _nothing(v.new_empty(plan.out_shape), needs, q, k, v, table, lam)
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    if needs:
        return _GridAttention.apply(q, k, v, table, lam, lengths, plan, q_start)
    table, lam = table.contiguous(), None if lam is None else lam.contiguous()
    return _forward(plan, _describe(plan, q, k, v, lengths, lam, q_start), q.dtype, dev, table, False)[0]


def grid_attention(q, k, v, table, grid, max_distance=64, lengths=None, q_start=0, scale=None):
    """softmax attention over the pixels of an image grid with a learned relative position bias by buckets

        out_i = sum_j softmax_j(scale q_i . k_j + table[by(y_j - y_i), bx(x_j - x_i), head]) v_j

    q [B, Lq, heads, D], k, v [B, Lk, heads, D], fp32 or bf16; D a multiple of 8 up to 128; any strides (rows that do not start at 16
    bytes are copied).  Returns [B, Lq, heads, D] in their type.
    grid = (height, width): token t is the pixel (t // width, t % width).  The keys are the tokens 0 .. Lk - 1, the queries the tokens
    q_start .. q_start + Lq - 1 (all pixels, a band of them, or a single one).  (1, n): a row of n tokens.
    table [ny, nx, heads] fp32: ny and nx buckets for the two axes (each 1, or an even number up to 64: the lower half for distances
    <= 0, the upper half for those > 0; bucket_thresholds has the borders; from `max_distance` on they share the last one).
    An entry of -inf masks its pairs; every finite one is a bias, the type's lowest and largest among them.
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
    if qkv.dim() != 3 or not isinstance(heads, int) or heads < 1 or qkv.shape[2] % (3 * heads * maps):
        _fail(f"qkv: expected [batch, tokens, 3 * C] with C a multiple of {heads} heads x {maps} map(s), got {list(qkv.shape)}")
    _on_gpu("table", table, qkv.device)
    if table.dtype != F32:
        _fail(f"table: expected fp32, got {table.dtype}")
    if lam is not None:
        _parameter("lam", lam, (heads,), qkv.device)
    b, n, c3 = qkv.shape
    d = c3 // (3 * heads * maps)
    shape, grid = (b, n, heads * maps, d), _integers("grid", grid)
    plan = _plan(maps, shape, shape, (b, n, heads, d * maps), qkv.dtype, table.shape, grid, _integers("max_distance", max_distance), _number("scale", scale))
    if n != plan.grid[0] * plan.grid[1]:
        _fail(f"{n} tokens are not the grid {grid}")
    needs = _needs_grad(qkv, table, lam)
    if plan.desc is None:
        return _nothing(qkv.new_empty((b, n, c3 // 3)), needs, qkv, table, lam)
    if needs:
        return _GridSelfAttention.apply(qkv, table, lam, plan)
    qkv, table, lam = _dense16(qkv), table.contiguous(), None if lam is None else lam.contiguous()
    return _forward(plan, _describe_qkv(plan, qkv, lam), qkv.dtype, qkv.device, table, False)[0].view(b, n, c3 // 3)


# ---------------------------------------------------------------------------------------------------------------------- norms
class _Seam:
    """what a norm_gate_residual call is, beside its tensors"""
    __slots__ = ("norm", "eps", "rows", "c", "shape")


def _rows_of(t, shape):
    """`t` as [rows, C] with dense channels and one stride between its rows, and that stride (a copy only where there is none)"""
    if t.is_contiguous():
        return t, shape[-1]
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
    """the description of a call, its operands (they have to outlive the launch)"""
    params = [None if t is None else _dense16(t) for t in params]
    (x, xs), (f, fs), (gate, gs) = rows = [(None, 0) if t is None else _rows_of(t, s.shape) for t in (x, f, gate)]
    return NormGateDesc(x.data_ptr(), _ptr(f), _ptr(gate), *[None if t is None else t.data_ptr() for t in params], s.rows, xs, fs, gs,
                        s.c, s.norm, _DT[x.dtype], s.eps), (rows, params)


def _seam_forward(s, x, f, gate, params):
    dev = x.device
    desc, operands = _seam_desc(s, x, f, gate, params)
    y = _like(x) if f is not None else None
    h = _like(x) if params[3] is not None else None
    guard = _guard(dev)
    try:
        check(lib.im2im_norm_gate_fwd(ctypes.byref(desc), _ptr(y), _ptr(h), torch._C._cuda_getCurrentRawStream(dev.index)), "im2im_norm_gate_fwd")
    finally:
        if guard is not None:
            guard.__exit__(None, None, None)
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
    @_once
    def backward(ctx, *grads):
        s = ctx.s
        x, f, gate, *params = ctx.saved_tensors
        dy, dh = grads if len(grads) == 2 else (grads[0], None) if f is not None else (None, grads[0])
        if dy is None and dh is None:
            return (None,) * 9
        dev, dt, c = x.device, x.dtype, s.c
        dy, dh = (None if t is None else (t if t.dtype == dt else t.to(dt)).contiguous() for t in (dy, dh))
        _, need_x, need_f, need_gate, *need = ctx.needs_input_grad
        dx = _like(x) if need_x else None
        df = _like(x) if need_f and f is not None else None
        dgate = _like(x) if need_gate and gate is not None else None
        want = [n and t is not None for n, t in zip(need, params)]
        wanted = sum(want)
        if wanted and c % 4 == 0:                            # one buffer, each row at 16 bytes
            spare = list(torch.empty((wanted, c), dtype=F32, device=dev).unbind())
        else:
            spare = [torch.empty(c, dtype=F32, device=dev) for _ in range(wanted)]
        sums = [spare.pop() if w else None for w in want]
        if dh is None:                                       # no gradient came through the second norm
            for t in sums[3:]:
                if t is not None:
                    t.zero_()
        out = sums if dh is not None else [*sums[:3], None, None]
        n = lib.im2im_norm_gate_bwd_workspace_bytes(s.rows, c)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        desc, operands = _seam_desc(s, x, f, gate, params)
        guard = _guard(dev)
        try:
            check(lib.im2im_norm_gate_bwd(ctypes.byref(desc), _ptr(dy), _ptr(dh), _ptr(dx), _ptr(df), _ptr(dgate), *map(_ptr, out), ws.data_ptr(), n,
                                          torch._C._cuda_getCurrentRawStream(dev.index)), "im2im_norm_gate_bwd")
        finally:
            if guard is not None:
                guard.__exit__(None, None, None)
        return (None, dx, df, dgate, *sums)


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
    dev, shape = x.device, x.shape
    c = shape[-1]
    if not 1 <= c <= MAX_NORM_CHANNELS:
        _fail(f"x: 1 to {MAX_NORM_CHANNELS} channels, got {c}")
    for name, t in (("f", f), ("gate", gate)):
        if t is not None:
            if not _is(t, x.dtype, shape, dev):
                _on_gpu(name, t, dev)
                _fail(f"{name}: expected {x.dtype} {list(x.shape)} as x, got {t.dtype} {list(t.shape)}")
    params = (scale, post_weight, post_bias, pre_weight, pre_bias)
    for name, t in zip(("scale", "post_weight", "post_bias", "pre_weight", "pre_bias"), params):
        if t is not None:
            _parameter(name, t, (c,), dev)
    if f is None and pre_weight is None:
        _fail("weight is missing")
    if f is not None and post_weight is None:
        _fail("f needs post_weight")
    if norm == "rms" and (post_bias is not None or pre_bias is not None):
        _fail("a root-mean-square norm has no bias")
    if pre_bias is not None and pre_weight is None:
        _fail("pre_bias needs pre_weight")
    s = _Seam()
    s.norm, s.eps, s.c, s.shape, s.rows = _NORM[norm], float(eps), c, shape, x.numel() // c
    tensors = (x, f, gate, *params)
    needs = _needs_grad(*tensors)
    if s.rows == 0:
        y = None if f is None else _nothing(x.new_empty(shape), needs, *tensors[:6])
        h = None if pre_weight is None else _nothing(x.new_empty(shape), needs, *tensors)
        return h if f is None else (y, h)
    if needs:
        got = _NormGate.apply(s, *tensors)
        return got if f is None or pre_weight is not None else (got, None)
    y, h = _seam_forward(s, x, f, gate, params)
    return h if f is None else (y, h)

