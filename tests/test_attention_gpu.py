"""Grid attention and its differential form on the GPU against a plain implementation in 64 bits (tests/attention_reference.py: values and
error bounds), at the sizes, masks and strides where they can go wrong, and their refusals."""
import math

import pytest
import torch

from attention_reference import attention, check
from im2im_uq_amd import attn_ops
from im2im_uq_amd._lib import Im2ImError

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def operands(maps, dtype, grid, b, heads, d, buckets, lq=None, lk=None, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    n = grid[0] * grid[1]
    lq, lk = n if lq is None else lq, n if lk is None else lk
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    o = {"q": (rnd(b, lq, heads * maps, d) * spread).to(dtype), "k": rnd(b, lk, heads * maps, d).to(dtype), "v": rnd(b, lk, heads, d * maps).to(dtype),
         "table": rnd(buckets[0], buckets[1], heads) * 0.7, "lam": torch.rand(heads, generator=g) if maps == 2 else None,
         "dout": rnd(b, lq, heads, d * maps).to(dtype)}
    return {k: None if t is None else t.to(DEV) for k, t in o.items()}


def call(o, grid, **kw):
    if o["lam"] is None:
        return attn_ops.grid_attention(o["q"], o["k"], o["v"], o["table"], grid, **kw)
    return attn_ops.diff_grid_attention(o["q"], o["k"], o["v"], o["lam"], o["table"], grid, **kw)


def train(o, grid, **kw):
    names = [n for n in ("q", "k", "v", "table", "lam") if o[n] is not None]
    leaves = {n: o[n].detach().requires_grad_(True) for n in names}
    out = call({**o, **leaves, **({"lam": None} if o["lam"] is None else {})}, grid, **kw)
    grads = torch.autograd.grad(out, [leaves[n] for n in names], o["dout"])
    return {"out": out, **{"d" + n: t for n, t in zip(names, grads)}}


def reference(o, grid, with_grads=True, **kw):
    return attention(o["q"], o["k"], o["v"], o["table"], grid, lam=o["lam"], dout=o["dout"] if with_grads else None, **kw)


# maps, grid, batch, heads, D, buckets
SHAPES = [
    (1, (1, 1), 1, 1, 8, (2, 2)), (1, (1, 2), 2, 1, 16, (1, 4)), (1, (3, 5), 2, 3, 24, (4, 6)), (1, (8, 8), 1, 2, 32, (8, 8)),
    (1, (5, 13), 2, 2, 40, (16, 8)), (1, (20, 20), 2, 2, 64, (16, 16)), (1, (9, 15), 1, 2, 72, (1, 16)), (1, (12, 11), 1, 1, 128, (32, 2)),
    (1, (1, 129), 1, 2, 64, (1, 32)), (1, (64, 2), 1, 1, 64, (64, 2)), (1, (130, 1), 1, 1, 32, (16, 1)), (1, (2, 300), 1, 1, 64, (8, 64)),
    (2, (1, 1), 1, 1, 8, (2, 2)), (2, (3, 5), 2, 3, 24, (4, 6)), (2, (20, 20), 2, 2, 32, (16, 16)), (2, (7, 19), 2, 2, 40, (8, 8)),
    (2, (12, 11), 1, 2, 64, (32, 2)), (2, (1, 193), 2, 1, 64, (1, 32)),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,grid,b,heads,d,buckets", SHAPES)
def test_forward_and_gradients(maps, grid, b, heads, d, buckets, dtype):
    o = operands(maps, dtype, grid, b, heads, d, buckets)
    want = reference(o, grid, max_distance=(20, 40))
    check(train(o, grid, max_distance=(20, 40)), want)
    check({"out": call(o, grid, max_distance=(20, 40))}, want, ("out",))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,d", [(1, 32), (1, 64), (1, 80), (1, 128), (2, 24), (2, 32), (2, 64)])
@pytest.mark.parametrize("grid,b", [((5, 7), 64), ((4, 8), 64), ((12, 12), 33), ((9, 15), 33)])
def test_many_images(grid, b, maps, d, dtype):
    """enough work for a workgroup of 128 queries or keys each (small calls share 32 of them between two waves), widths that are and are not a
    multiple of four"""
    o = operands(maps, dtype, grid, b, 8, d, (8, 8), seed=b + d)
    lengths = torch.full((b,), grid[0] * grid[1], dtype=torch.int32, device=DEV)
    lengths[1::3] = grid[0] * grid[1] // 2 + 1
    lengths[2] = 0
    want = reference(o, grid, lengths=lengths)
    check(train(o, grid, lengths=lengths), want)
    check({"out": call(o, grid, lengths=lengths)}, want, ("out",))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,d", [(1, 128), (2, 64)])
def test_widest_grid(maps, d, dtype):
    """512 wide: the largest window and accumulators in LDS"""
    grid = (2, 512)
    o = operands(maps, dtype, grid, 1, 1, d, (2, 64), seed=31)
    check(train(o, grid, max_distance=300), reference(o, grid, max_distance=300))


@pytest.mark.parametrize("maps,d", [(1, 32), (2, 32)])
@pytest.mark.parametrize("grid", [(8, 12), (7, 9), (1, 300)])
def test_small_workspace(grid, maps, d, monkeypatch):
    """a workspace for fewer lines than images: workgroups take several images in turn and add to their line"""
    o = operands(maps, BF16, grid, 7, 2, d, (8, 8), seed=33)
    want = reference(o, grid)
    lengths = torch.tensor([0, 40, 63, 5, 1, 64, 33], dtype=torch.int32, device=DEV)
    want_ragged = reference(o, grid, lengths=lengths)
    full = train(o, grid)
    real = attn_ops.lib.im2im_attention_bwd
    for images in (2, 3, 7):
        def smaller(p, g, ws, n, stream, images=images):
            line = 2 * (2 * grid[0] - 1) * (2 * grid[1] - 1) * 4 * ((grid[0] * grid[1] + 63) // 64)
            return real(p, g, ws, n - (7 - -(-7 // images)) * (line - 256), stream)
        monkeypatch.setattr(attn_ops.lib, "im2im_attention_bwd", smaller)
        check(train(o, grid), want)
        check(train(o, grid, lengths=lengths), want_ragged)
    monkeypatch.undo()
    assert all(torch.equal(full[n], t) for n, t in train(o, grid).items())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,d", [(1, 32), (1, 64), (1, 104), (2, 32), (2, 56)])
@pytest.mark.parametrize("grid,lq,q_start", [((17, 23), None, 0), ((1, 700), None, 0), ((3, 256), 100, 300), ((3, 256), 1, 767), ((9, 30), 260, 10)])
def test_few_images(grid, lq, q_start, maps, d, dtype):
    """so few workgroups that the keys (and queries) are shared out to more of them, whose parts are joined; lengths that end before, at and behind
    the ends of those parts"""
    o = operands(maps, dtype, grid, 4, 1, d, (8, 8), lq=lq, seed=41)
    n = grid[0] * grid[1]
    for lengths in (None, [0, 1, 128, n], [129, n - 1, 64, 256]):
        lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
        got = train(o, grid, q_start=q_start, lengths=lengths)
        check(got, reference(o, grid, q_start=q_start, lengths=lengths))
        assert all(torch.equal(got[k], t) for k, t in train(o, grid, q_start=q_start, lengths=lengths).items())


def test_far_apart_rows():
    """offsets that pass 32 bits: tokens 16 MiB apart"""
    grid, step = (1, 300), 1 << 23
    o = operands(1, BF16, grid, 1, 1, 32, (1, 8), seed=35)
    far = torch.empty(300 * step, dtype=BF16, device=DEV)
    s = dict(o)
    for n, at in (("q", 0), ("k", 64), ("v", 128)):
        s[n] = far.as_strided((1, 300, 1, 32), (300 * step, step, 32, 1), at)
        s[n].copy_(o[n])
    got, want = train(s, grid), train(o, grid)
    assert s["k"].data_ptr() == far.data_ptr() + 128 and all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,d", [(1, 64), (1, 40), (2, 32), (2, 64)])
@pytest.mark.parametrize("lengths", [[0, 1, 63], [64, 65, 128], [129, 130, 1000], [130, -5, 64]])
def test_lengths(maps, d, dtype, lengths):
    """padded images: what lies behind a length is NaN and infinity; an empty image gives zeros everywhere"""
    grid = (10, 13)
    o = operands(maps, dtype, grid, 3, 2, d, (8, 8), seed=3)
    for b, n in enumerate(lengths):
        o["k"][b, max(n, 0):] = math.nan
        o["v"][b, max(n, 0):] = math.inf
    t = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = train(o, grid, lengths=t)
    check(got, reference(o, grid, lengths=t))
    for b, n in enumerate(lengths):
        assert (got["dk"][b, max(n, 0):] == 0).all() and (got["dv"][b, max(n, 0):] == 0).all()
        if n <= 0:
            assert (got["out"][b] == 0).all() and (got["dq"][b] == 0).all()
    check({"out": call(o, grid, lengths=t)}, reference(o, grid, False, lengths=t))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("grid,lq,q_start,lk", [((1, 4097), 1, 4096, None), ((64, 64), 1, 2080, None), ((64, 64), 1, 0, 4000), ((16, 33), 5, 40, None),
                                                ((16, 33), 33, 495, 66), ((40, 30), 200, 700, 1199), ((1, 700), 3, 0, 1)])
def test_few_queries(maps, dtype, grid, lq, q_start, lk):
    """single tokens and bands of the grid against all of its keys, or its first ones: the keys split over workgroups"""
    o = operands(maps, dtype, grid, 2, 2, 32, (8, 16), lq=lq, lk=lk, seed=5)
    n = o["k"].shape[1]
    lengths = torch.tensor([n, n // 2], dtype=torch.int32, device=DEV)
    check({"out": call(o, grid, q_start=q_start, lengths=lengths)}, reference(o, grid, False, q_start=q_start, lengths=lengths))
    check(train(o, grid, q_start=q_start), reference(o, grid, q_start=q_start))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,d,heads,b,grid,buckets", [
    (1, 64, 2, 2, (5, 7), (4, 6)), (1, 40, 1, 1, (1, 1), (1, 1)), (1, 32, 8, 64, (9, 15), (64, 64)), (1, 128, 2, 1, (130, 1), (32, 1)),
    (1, 24, 3, 1, (1, 300), (1, 64)), (2, 32, 2, 2, (5, 7), (6, 4)), (2, 64, 1, 2, (17, 33), (16, 8)), (2, 16, 9, 57, (2, 65), (2, 2))])
def test_single_token(maps, d, heads, b, grid, buckets, dtype):
    """one query at the grid's ends and inside, with lengths that leave no key, one key and half a tile, and masks in its table"""
    n = grid[0] * grid[1]
    for at in sorted({0, n // 3, n - 1}):
        o = operands(maps, dtype, grid, b, heads, d, buckets, lq=1, seed=at)
        o["table"][0, 0, 0], o["table"][-1, -1, -1] = -math.inf, torch.finfo(F32).min
        lengths = torch.tensor([(n, 0, 1, 33)[x % 4] for x in range(b)], dtype=torch.int32, device=DEV)
        check({"out": call(o, grid, q_start=at, lengths=lengths)}, reference(o, grid, False, q_start=at, lengths=lengths))
        whole = operands(maps, dtype, grid, b, heads, d, buckets, seed=at)
        alone = call({**o, "q": whole["q"][:, at:at + 1]}, grid, q_start=at)
        check({"out": alone}, reference({**o, "q": whole["q"][:, at:at + 1]}, grid, False, q_start=at))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps", [1, 2])
def test_table_masks(maps, dtype):
    """entries of -infinity mask their pairs, a row of the grid loses all its keys to them; the type's lowest value is a bias like others"""
    grid, low = (6, 11), torch.finfo(F32).min
    o = operands(maps, dtype, grid, 2, 2, 32, (2, 8), seed=7)
    o["table"][0, :, 0] = -math.inf                          # head 0: no key above or beside; the last row of the grid has no key at all
    o["table"][1, 3:, 1] = -math.inf
    want = reference(o, grid)
    got = train(o, grid)
    check(got, want)
    assert (got["out"][:, 55:, 0] == 0).all() and (got["dq"][:, 55:, :maps] == 0).all()
    assert (got["dtable"][0, :, 0] == 0).all()
    o["table"][:, :, 0] = low                                # all keys at the same enormous bias: in the limits of 32 bits an even softmax
    got = train(o, grid)
    assert all(t.isfinite().all() for t in got.values())
    weight = 1.0 if maps == 1 else 1 - o["lam"][0].item()
    mean = o["v"][:, :, 0].double().mean(1, keepdim=True) * weight
    assert (got["out"][:, :, 0].double() - mean).abs().max() <= 3 * 2.0 ** -8 * o["v"].double().abs().max()


def test_one_large_score():
    """scores in the thousands: one key takes all, and nothing overflows on the way"""
    grid = (9, 9)
    o = operands(1, F32, grid, 1, 1, 32, (4, 4), seed=9, spread=4000.0)
    got = train(o, grid)
    assert all(t.isfinite().all() for t in got.values())
    s = (o["q"][0, :, 0].double() @ o["k"][0, :, 0].double().T) / math.sqrt(32)
    best = s.topk(2).values
    clear = best[:, 0] - best[:, 1] > 64                     # more than the bias and the scores' rounding can turn
    assert clear.sum() > 40
    assert torch.allclose(got["out"][0, clear, 0], o["v"][0, s.argmax(1)[clear], 0], rtol=2.0 ** -20, atol=0)


@pytest.mark.parametrize("maps", [1, 2])
def test_strides_and_alignment(maps):
    """head-major tensors, slices of a wider one, expanded batches and rows off 16 bytes give the bits of their dense copies"""
    grid, d = (7, 9), 32
    o = operands(maps, BF16, grid, 3, 2, d, (8, 8), seed=11)
    dense = train(o, grid)
    wide = torch.randn(3, 63, 4, 2 * maps * d + 24, device=DEV).to(BF16)
    off = torch.empty(o["v"].numel() + 1, dtype=BF16, device=DEV)[1:].view(o["v"].shape)
    off.copy_(o["v"])
    wide[:, :, :2 * maps, 8:8 + d] = o["q"]
    s = dict(o, q=wide[:, :, :2 * maps, 8:8 + d], k=o["k"].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3), v=off,
             dout=o["dout"].transpose(1, 2).contiguous().transpose(1, 2))
    got = train(s, grid)
    assert all(torch.equal(got[n], dense[n]) for n in dense)
    one = {n: t[:1].as_strided(t[:1].shape, (0, *t.stride()[1:])) if n in ("q", "k", "v") else None if t is None else t[:1] if n == "dout" else t
           for n, t in o.items()}                            # a batch of one whose stride says nothing
    assert torch.equal(train(one, grid)["dq"], dense["dq"][:1])
    s = dict(o, k=o["k"][:1].expand(3, -1, -1, -1), v=o["v"][..., ::2].repeat_interleave(2, -1)[..., ::2].repeat_interleave(2, -1))
    check(train(s, grid), reference(s, grid))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps", [1, 2])
def test_one_projection(maps, dtype):
    """q, k and v side by side in one tensor: the bits of the three, the gradient in one tensor"""
    grid, heads, d = (8, 11), 2, 32
    o = operands(maps, dtype, grid, 2, heads, d, (8, 8), seed=13)
    want = train(o, grid)
    qkv = torch.cat([o[n].flatten(2) for n in ("q", "k", "v")], 2).requires_grad_(True)
    table, lam = o["table"].requires_grad_(True), o["lam"]
    out = attn_ops.grid_self_attention(qkv, heads, table, grid, lam=lam)
    dqkv, dtable = torch.autograd.grad(out, (qkv, table), o["dout"].flatten(2))
    assert torch.equal(out, want["out"].flatten(2)) and torch.equal(dtable, want["dtable"])
    assert torch.equal(dqkv, torch.cat([want["d" + n].flatten(2) for n in ("q", "k", "v")], 2))


@pytest.mark.parametrize("maps", [1, 2])
def test_same_bits_again(maps):
    """many images for each workgroup of the queries' gradients; repeated calls, with other work between them, give the same bits"""
    grid = (12, 12)
    o = operands(maps, BF16, grid, 40, 16, 32, (8, 8), seed=15)
    first = train(o, grid)
    for _ in range(5):
        torch.randn(1 << 20, device=DEV).sort()
        again = train(o, grid)
        assert all(torch.equal(first[n], again[n]) for n in first)
    check(first, reference(o, grid))


def test_gradients_by_differences():
    """a step along a random direction changes the loss by the gradient's product with it (64-bit differences of the plain form apart, these
    are the kernel's own values: 32 bits leave about 2^-24 |loss| / step)"""
    grid = (4, 6)
    o = operands(2, F32, grid, 1, 2, 16, (4, 4), seed=17)
    got = train(o, grid)
    names = ("q", "k", "v", "table", "lam")
    step = 2.0 ** -7
    for n in names:
        u = torch.randn_like(o[n])
        u /= u.norm()
        loss = [float((call(dict(o, **{n: o[n] + e * step * u}), grid).double() * o["dout"].double()).sum()) for e in (1, -1)]
        scale = float(o["dout"].double().norm() * got["out"].detach().double().norm())
        slope = float((got["d" + n].double() * u.double()).sum())
        # third derivatives are of the loss's own size here: step^2 of it; rounding of the 32-bit values: 2^-20 of it over the step
        assert abs((loss[0] - loss[1]) / (2 * step) - slope) <= scale * (step ** 2 + 2.0 ** -20 / step), n


@pytest.mark.parametrize("maps", [1, 2])
def test_captured_graph(maps):
    """forward and backward in a HIP graph, replayed on new inputs between eager calls: the eager bits each time"""
    grid = (10, 10)
    sets = [operands(maps, BF16, grid, 2, 4, 32, (8, 8), seed=20 + n) for n in range(3)]
    want = [train(o, grid) for o in sets]
    static = {n: None if t is None else t.clone() for n, t in sets[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(static, grid)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = train(static, grid)
    for n in (1, 2, 0, 1):
        for name, t in static.items():
            if t is not None:
                t.copy_(sets[n][name])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(got[name], want[n][name]) for name in got)
        train(sets[2], grid)


def test_on_another_stream():
    grid = (16, 16)
    o = operands(1, BF16, grid, 4, 4, 64, (8, 8), seed=23)
    want = train(o, grid)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [train(o, grid) for _ in range(4)]
    want2 = train(o, grid)                                   # at the same time on the first stream
    side.synchronize()
    assert all(torch.equal(g[n], want[n]) for g in got for n in want) and all(torch.equal(want2[n], want[n]) for n in want)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one GPU")
def test_on_another_device():
    grid = (6, 7)
    o = operands(1, F32, grid, 2, 2, 32, (8, 8), seed=25)
    want = train(o, grid)
    got = train({n: None if t is None else t.to("cuda:1") for n, t in o.items()}, grid)
    assert all(torch.equal(got[n].cpu(), want[n].cpu()) for n in want)


def test_numbers_of_other_kinds():
    """numpy's and torch's whole numbers and lists are taken as they are at the call, whatever becomes of them later"""
    import numpy as np
    grid = (6, 7)
    o = operands(1, F32, grid, 1, 1, 16, (4, 4), lq=1)
    at = torch.tensor(3)
    for t in (3, 11, 40):
        at.fill_(t)
        want = call(o, grid, q_start=t, max_distance=16, scale=0.5)
        assert torch.equal(call(o, [np.int64(6), np.int32(7)], q_start=at, max_distance=[16, np.int16(16)], scale=np.float32(0.5)), want)
        check({"out": want}, reference(o, grid, False, q_start=t, max_distance=16, scale=0.5))


@pytest.mark.parametrize("maps", [1, 2])
def test_no_second_derivatives(maps):
    """create_graph gives the same gradients and refuses to be differentiated again, rather than giving a gradient of nothing"""
    grid = (5, 7)
    o = operands(maps, F32, grid, 2, 2, 32, (4, 4))
    names = [n for n in o if n != "dout" and o[n] is not None]
    for n in names:
        o[n] = o[n].detach().requires_grad_()
    leaves = [o[n] for n in names]
    plain = torch.autograd.grad(call(o, grid), leaves, o["dout"])
    graph = torch.autograd.grad(call(o, grid), leaves, o["dout"], create_graph=True)
    for a, b in zip(plain, graph):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="does not require grad"):
        graph[0].sum().backward()
    graph = torch.autograd.grad(call(o, grid), leaves, o["dout"].clone().requires_grad_(), create_graph=True)
    for a, b in zip(plain, graph):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        graph[0].sum().backward()


def test_nothing_asked_for():
    o = operands(1, F32, (2, 3), 2, 2, 8, (2, 2))
    t = o["q"][:0].requires_grad_(True)
    out = attn_ops.grid_attention(t, o["k"][:0], o["v"][:0], o["table"], (2, 3))
    assert out.shape == (0, 6, 2, 8)
    out.sum().backward()
    assert t.grad.shape == t.shape
    assert attn_ops.grid_attention(o["q"][:, :0], o["k"], o["v"], o["table"], (2, 3)).shape == (2, 0, 2, 8)


def test_refusals():
    grid = (4, 5)
    o = operands(1, F32, grid, 2, 2, 16, (4, 4))
    o2 = operands(2, F32, grid, 2, 2, 16, (4, 4))

    def refused(match, base=o, where=grid, **kw):
        tensors = {k: kw.pop(k) for k in list(kw) if k in base}
        with pytest.raises(Im2ImError, match=match):
            call(dict(base, **tensors), where, **kw)

    refused("GPU", q=o["q"].cpu())
    refused("one type", k=o["k"].to(BF16))
    refused("fp32 or bf16", **{n: o[n].half() for n in ("q", "k", "v")})
    refused("belong together", v=o["v"][:, :-1])
    refused("belong together", k=o["k"][..., :8])
    refused("belong together", q=o["q"][:1])
    refused("expected \\[batch", q=o["q"][0])
    refused("head size", **{n: o[n][..., :12] for n in ("q", "k", "v")})
    big = operands(1, F32, grid, 1, 1, 136, (4, 4))
    refused("head size", base=big)
    refused("head size", base=operands(2, F32, grid, 1, 1, 72, (4, 4)))
    refused("table", table=o["table"][..., :1])
    refused("table", table=o["table"].to(BF16))
    refused("buckets of an axis", table=torch.zeros(3, 4, 2, device=DEV))
    refused("buckets of an axis", table=torch.zeros(4, 66, 2, device=DEV))
    refused("max_distance", table=torch.zeros(64, 4, 2, device=DEV), max_distance=16)
    refused("do not fit", where=(3, 5))
    refused("not tokens", where=(4, 5), q_start=1)
    refused("not tokens", where=(4, 5), q_start=-1)
    refused("grid", where=(0, 5))
    refused("grid", where=(2, 513))
    refused("grid =", where=20)
    refused("whole numbers", where=(4.0, 5))
    refused("whole numbers", q_start=0.5)
    refused("whole numbers", q_start=None)
    refused("not tokens", q_start=(0, 1))
    refused("whole numbers", max_distance="far")
    refused("a tensor", scale=torch.tensor(0.5))
    refused("a number", scale="one")
    refused("lengths", lengths=torch.zeros(2, dtype=torch.int64, device=DEV))
    refused("lengths", lengths=torch.zeros(3, dtype=torch.int32, device=DEV))
    refused("GPU", lengths=torch.zeros(2, dtype=torch.int32))
    refused("scale", scale=math.inf)
    refused("lam", base=o2, lam=o2["lam"][:1])
    refused("no keys", k=o["k"][:, :0], v=o["v"][:, :0])
    qkv = torch.zeros(2, 20, 96, device=DEV)
    with pytest.raises(Im2ImError, match="qkv"):
        attn_ops.grid_self_attention(qkv[..., :95], 2, o["table"], grid)
    with pytest.raises(Im2ImError, match="not the grid"):
        attn_ops.grid_self_attention(qkv[:, :19], 2, o["table"], grid)
    torch.cuda.synchronize()
