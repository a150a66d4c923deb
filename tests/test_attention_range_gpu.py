"""Grid attention on the GPU with biases over the whole range of their type and with NaN among the keys: values and gradients against 64 bits."""
import math

import pytest
import torch

from attention_reference import U16, U32, attention, axis_bucket, check
from test_attention_gpu import DEV, call, operands, train

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
LOW, HIGH = torch.finfo(F32).min, torch.finfo(F32).max

# maps, grid, batch, heads, D, lq, q_start: calls of half and whole workgroups, of split keys and queries, of odd widths, of one query
CALLS = [(1, (20, 20), 2, 2, 32, None, 0), (1, (4, 8), 64, 8, 64, None, 0), (1, (9, 15), 1, 2, 128, None, 0), (1, (64, 64), 1, 2, 32, 1, 2080),
         (2, (20, 20), 2, 2, 32, None, 0), (2, (5, 7), 64, 8, 64, None, 0), (2, (40, 30), 1, 1, 40, 70, 600)]


def swallowed(o, grid, **kw):
    """reference where finite biases lie so far apart that a score plus its bias is the bias in 32 bits: each entry by its rank, 800 apart (the others'
    share, e^-800, is nothing in 64 bits either), and scores of nothing: q as 2^-60 of itself, the keys' gradients as much larger"""
    rank = torch.searchsorted(o["table"].unique(), o["table"]).float() * 800
    table = torch.where(o["table"] == -math.inf, o["table"], rank - rank.max())
    want = attention(o["q"] * 2.0 ** -60, o["k"], o["v"], table, grid, lam=o["lam"], dout=o["dout"], **kw)
    want["dk"] = tuple(t * 2.0 ** 60 for t in want["dk"])
    return want


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bias", [1.0, -1e6, -1e7, -1e8, -1e9, LOW, 1e7, 1e9, 2e38])
@pytest.mark.parametrize("maps,grid,b,heads,d,lq,q_start", CALLS)
def test_a_common_bias_cancels(maps, grid, b, heads, d, lq, q_start, bias, dtype):
    """every query's probabilities sum to one in the backward too, so that the values' gradients of an image sum to its output gradients (two
    maps: 1 - lam times); where the bias swallows the scores, every gradient is that of an even softmax"""
    o = operands(maps, dtype, grid, b, heads, d, (8, 8), lq=lq, seed=1)
    o["table"].fill_(bias)
    n = grid[0] * grid[1]
    lengths = torch.tensor([(n, n // 2 + 1, 1, 0)[x % 4] for x in range(b)], dtype=torch.int32, device=DEV)
    got = train(o, grid, lengths=lengths, q_start=q_start)
    dv, dout, lam = got["dv"].double(), o["dout"].double(), 0.0 if maps == 1 else o["lam"].double()[:, None]
    dout = torch.where(lengths[:, None, None, None] > 0, dout, 0.0)
    # each dv is rounded once, P for its product (bf16), exponentials, the row's sum and the chains over queries in 32 bits
    bf16 = dtype == BF16
    bound = (U16 if bf16 else U32) * dv.abs().sum(1) + ((U16 if bf16 else 0) + (dout.shape[1] + n / 16 + 64) * U32) * (1 + lam) * dout.abs().sum(1)
    off = (dv.sum(1) - (1 - lam) * dout.sum(1)).abs()
    assert (off <= bound).all(), float((off / bound.clamp(min=1e-30)).max())
    if abs(bias) >= 1e9:
        check(got, swallowed(o, grid, lengths=lengths, q_start=q_start))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,grid,b,heads,d,lq,q_start", CALLS)
def test_a_key_of_nan(maps, grid, b, heads, d, lq, q_start, dtype):
    """a NaN in one key makes its head's probabilities NaN, all of them: no value that comes from them is a number, and nothing else changes"""
    o = operands(maps, dtype, grid, b, heads, d, (8, 8), lq=lq, seed=2)
    n = grid[0] * grid[1]
    length = n - 3
    lengths = torch.full((b,), length, dtype=torch.int32, device=DEV)
    want = train(o, grid, lengths=lengths, q_start=q_start)
    o["k"][0, length // 2, 0, d - 1] = math.nan
    got = train(o, grid, lengths=lengths, q_start=q_start)
    assert got["out"][0, :, 0].isnan().all() and got["dq"][0, :, 0].isnan().all()
    assert got["dk"][0, :length, 0].isnan().all() and got["dv"][0, :length, 0].isnan().all()
    assert (got["dk"][0, length:, 0] == 0).all() and (got["dv"][0, length:, 0] == 0).all()
    assert call(o, grid, lengths=lengths, q_start=q_start)[0, :, 0].isnan().all()
    for name in ("out", "dq", "dk", "dv"):
        t, w = got[name].clone(), want[name].clone()
        h = 0 if name in ("out", "dv") or maps == 1 else slice(0, 2)
        t[0, :, h] = w[0, :, h] = 0
        assert torch.equal(t, w), name
    if heads > 1:
        assert torch.equal(got["dtable"][..., 1:], want["dtable"][..., 1:])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,grid,b,heads,d,lq,q_start", CALLS)
@pytest.mark.parametrize("entries", [(LOW, -2e38, -2.5e38), (HIGH, 2.3e38, 2.4e38, -1e38), (LOW, HIGH, 1e38, 2e38), (LOW, -math.inf, -3e38), (LOW, 1e9, -1e9)])
def test_the_ends_of_the_range(maps, grid, b, heads, d, lq, q_start, entries, dtype):
    """table entries of any finite size are ordered as they are: the largest that a row reaches takes it, alone or in even shares"""
    o = operands(maps, dtype, grid, b, heads, d, (8, 8), lq=lq, seed=3)
    pick = torch.randint(len(entries), o["table"].shape, generator=torch.Generator().manual_seed(4))
    o["table"].copy_(torch.tensor(entries)[pick])
    want = swallowed(o, grid, q_start=q_start)
    check(train(o, grid, q_start=q_start), want)
    check({"out": call(o, grid, q_start=q_start)}, want, ("out",))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("entry", [math.nan, math.inf])
@pytest.mark.parametrize("maps,d,grid,b,heads,lq,q_start", [(1, 32, (16, 33), 2, 2, 5, 40), (1, 64, (16, 16), 2, 2, 70, 30), (1, 128, (12, 20), 1, 1, 33, 0),
                                                            (1, 64, (9, 15), 64, 8, 40, 0), (2, 32, (16, 33), 2, 2, 5, 40), (2, 64, (12, 20), 33, 8, 33, 10)])
def test_entries_that_no_pair_has(maps, d, grid, b, heads, lq, q_start, entry, dtype):
    """what the table holds for distances that no query of a band has to any key changes nothing, and has no gradient"""
    o = operands(maps, dtype, grid, b, heads, d, (16, 32), lq=lq, seed=7)
    i, j = torch.arange(q_start, q_start + lq, device=DEV), torch.arange(grid[0] * grid[1], device=DEV)
    row = axis_bucket((j // grid[1])[None] - (i // grid[1])[:, None], 16, 16) * 32 + axis_bucket((j % grid[1])[None] - (i % grid[1])[:, None], 32, 40)
    free = torch.ones(16 * 32, dtype=torch.bool, device=DEV)
    free[row.flatten().unique()] = False
    free = free.view(16, 32)
    assert free.sum() > 16
    want = train(o, grid, q_start=q_start, max_distance=(16, 40))
    out = call(o, grid, q_start=q_start, max_distance=(16, 40))
    o["table"][free] = entry
    got = train(o, grid, q_start=q_start, max_distance=(16, 40))
    assert torch.equal(call(o, grid, q_start=q_start, max_distance=(16, 40)), out)
    for name in want:
        assert torch.equal(got[name], want[name]), name
    assert (got["dtable"][free] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,d,grid,b,heads,lq,q_start", [(1, 64, (16, 16), 2, 2, 70, 30), (1, 64, (9, 15), 64, 8, 40, 0), (2, 32, (16, 33), 2, 2, 5, 40)])
@pytest.mark.parametrize("name", ["q", "v", "dout"])
def test_a_last_query_of_nan(name, maps, d, grid, b, heads, lq, q_start, dtype):
    """NaN in the last query (its gradient, a value of the first head): no bucket that none of the queries reaches has a gradient, no other head has NaN"""
    o = operands(maps, dtype, grid, b, heads, d, (16, 32), lq=lq, seed=8)
    i, j = torch.arange(q_start, q_start + lq, device=DEV), torch.arange(grid[0] * grid[1], device=DEV)
    row = axis_bucket((j // grid[1])[None] - (i // grid[1])[:, None], 16, 16) * 32 + axis_bucket((j % grid[1])[None] - (i % grid[1])[:, None], 32, 40)
    free = torch.ones(16 * 32, dtype=torch.bool, device=DEV)
    free[row.flatten().unique()] = False
    free = free.view(16, 32)
    want = train(o, grid, q_start=q_start, max_distance=(16, 40))
    o[name][0, -1, 0] = math.nan
    got = train(o, grid, q_start=q_start, max_distance=(16, 40))
    assert got["dtable"][..., 0].isnan().any() and (got["dtable"][free] == 0).all()
    assert torch.equal(got["dtable"][..., 1:], want["dtable"][..., 1:])
    if maps == 2:                                            # lam weighs the second map, which the first one's query is no part of
        assert got["dlam"][0].isnan() if name != "q" else got["dlam"][0] == want["dlam"][0]
        assert torch.equal(got["dlam"][1:], want["dlam"][1:])
