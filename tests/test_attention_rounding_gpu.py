"""bf16 attention is 32-bit arithmetic that is rounded once: P and dS enter their products as two bf16, whose sum has 16 bits of them, so that what
they lose is far below the rounding of a result, also of one that is small beside its terms."""
import pytest
import torch

import attention_reference
from attention_reference import U16, U32, attention, check
from test_attention_gpu import DEV, SHAPES, call, operands, train

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
# maps, grid, batch, heads, D, buckets: whole and half workgroups, split keys and queries
CASES = SHAPES + [(1, (20, 20), 10, 8, 64, (16, 16)), (1, (17, 23), 16, 4, 8, (8, 8)), (1, (17, 23), 16, 4, 16, (8, 8)), (1, (16, 16), 33, 8, 32, (8, 8)),
                  (1, (9, 15), 33, 8, 24, (8, 8)), (1, (32, 32), 2, 2, 128, (32, 32)), (2, (20, 20), 10, 8, 32, (16, 16)), (2, (17, 23), 16, 4, 8, (8, 8)),
                  (2, (17, 23), 9, 4, 64, (8, 8))]


def rounded_once(o, grid, monkeypatch, **kw):
    """attention's values with the bounds of one rounding.  With u a bf16's, its bounds are A + u (M + |value|) + u^2 N: 32-bit arithmetic, operands of
    products rounded, the result, what is left of hi + lo; three evaluations give the parts, and operands of 16 bits leave A + u |value| + u^2 (M + N)"""
    wide = {n: t.float() if t is not None and t.dtype == BF16 else t for n, t in o.items()}

    def bounds(x, u=U16):
        with monkeypatch.context() as m:
            m.setattr(attention_reference, "U16", u)
            return attention(x["q"], x["k"], x["v"], x["table"], grid, lam=x["lam"], dout=x["dout"], **kw)
    exact, one, half = bounds(wide), bounds(o), bounds(o, U16 / 2)
    want = {}
    for name, (value, bound) in one.items():
        if name in ("dtable", "dlam"):
            want[name] = (value, bound)
            continue
        a = exact[name][1] - U32 * value.abs()
        square = (2 * (bound - 2 * half[name][1] + a)).clamp(min=0)
        m = ((bound - a - square) / U16 - value.abs()).clamp(min=0)
        want[name] = (value, a + U16 * value.abs() + U16 ** 2 * m + square)
    return want


@pytest.mark.parametrize("maps,grid,b,heads,d,buckets", CASES)
def test_one_rounding(maps, grid, b, heads, d, buckets, monkeypatch):
    o = operands(maps, BF16, grid, b, heads, d, buckets, seed=61)
    n = grid[0] * grid[1]
    lengths = torch.randint((n + 1) // 2, n + 1, (b,), generator=torch.Generator().manual_seed(6), dtype=torch.int32).to(DEV)
    want = rounded_once(o, grid, monkeypatch, lengths=lengths)
    check(train(o, grid, lengths=lengths), want)
    check({"out": call(o, grid, lengths=lengths)}, want, ("out",))


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("grid,lq,q_start", [((1, 4097), 1, 4096), ((64, 64), 1, 2080), ((16, 33), 5, 40), ((40, 30), 200, 700)])
def test_one_rounding_of_few_queries(maps, grid, lq, q_start, monkeypatch):
    o = operands(maps, BF16, grid, 2, 2, 32, (8, 16), lq=lq, seed=63)
    want = rounded_once(o, grid, monkeypatch, q_start=q_start)
    check(train(o, grid, q_start=q_start), want)
    check({"out": call(o, grid, q_start=q_start)}, want, ("out",))
