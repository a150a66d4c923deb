"""The attention backward in a smaller workspace than it asks for: workgroups that take several images in turn and add to their line, and a pass over the
queries in several launches, with whole and half workgroups, both ring sizes, many key tiles an image and lengths."""
import pytest
import torch

from attention_reference import check
from im2im_uq_amd import attn_ops
from test_attention_gpu import DEV, operands, reference, train

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
BLANK = 0xAB


def up(n):
    return (n + 255) // 256 * 256


class Smaller:
    """lib.im2im_attention_bwd with a workspace for `images` images a workgroup and `tiles` query tiles a launch.  What it wrote of its lines shows that
    these were used."""

    def __init__(self, real, grid, b, heads, maps, images, tiles=None):
        n = grid[0] * grid[1]
        self.real = real
        self.rows = 64 if b * heads * -(-n // 128) < 256 else 128
        nq, groups = -(-n // self.rows), -(-b // images)
        tiles = nq if tiles is None else tiles
        assert tiles == nq or groups == 1
        line = heads * (2 * grid[0] - 1) * (2 * grid[1] - 1) * 4
        self.at = up(b * heads * maps * n * 4) + up(2 * line)
        self.line, self.slots = line, groups * tiles
        self.size = self.at + up(self.slots * line) + up(groups * nq * heads * 4)
        self.calls = 0

    def __call__(self, p, g, ws, n, stream):
        assert self.size < n
        torch.cuda.synchronize()
        ws = torch.full((self.size + self.line + 4096,), BLANK, dtype=torch.uint8, device=DEV)
        rc = self.real(p, g, ws.data_ptr(), self.size, stream)
        torch.cuda.synchronize()
        assert (ws[self.size:] == BLANK).all()
        lines = ws[self.at:self.at + up(self.slots * self.line)]
        written = int((lines != BLANK).nonzero().max())
        assert (self.slots - 1) * self.line <= written < self.slots * self.line
        self.calls += 1
        return rc


def ragged(b, n):
    t = torch.randint(0, n + 1, (b,), generator=torch.Generator().manual_seed(b), dtype=torch.int32)
    t[0], t[1 % b], t[-1] = 0, n, n // 2 + 1
    return t.to(DEV)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,d", [(1, 32), (1, 64), (1, 128), (2, 32), (2, 64)])
@pytest.mark.parametrize("grid,b,heads", [((17, 23), 16, 6), ((20, 20), 16, 6), ((2, 300), 7, 8), ((12, 27), 5, 2), ((1, 333), 5, 2)])
def test_images_in_turn(grid, b, heads, maps, d, dtype, monkeypatch):
    o = operands(maps, dtype, grid, b, heads, d, (8, 8), seed=51)
    n = grid[0] * grid[1]
    lengths = ragged(b, n)
    want, want_ragged = reference(o, grid), reference(o, grid, lengths=lengths)
    real = attn_ops.lib.im2im_attention_bwd
    for images in (2, 3, b):
        call = Smaller(real, grid, b, heads, maps, images)
        monkeypatch.setattr(attn_ops.lib, "im2im_attention_bwd", call)
        got = train(o, grid)
        check(got, want)
        check(train(o, grid, lengths=lengths), want_ragged)
        assert all(torch.equal(got[k], t) for k, t in train(o, grid).items()) and call.calls == 3


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("maps,d", [(1, 32), (1, 128), (2, 64)])
@pytest.mark.parametrize("grid,b,heads", [((17, 23), 16, 6), ((2, 300), 7, 8), ((24, 40), 3, 2), ((1, 700), 2, 3)])
def test_queries_in_several_launches(grid, b, heads, maps, d, dtype, monkeypatch):
    o = operands(maps, dtype, grid, b, heads, d, (8, 8), seed=53)
    n = grid[0] * grid[1]
    lengths = ragged(b, n)
    want, want_ragged = reference(o, grid), reference(o, grid, lengths=lengths)
    real = attn_ops.lib.im2im_attention_bwd
    for tiles in (1, 2):
        call = Smaller(real, grid, b, heads, maps, b, tiles)
        monkeypatch.setattr(attn_ops.lib, "im2im_attention_bwd", call)
        got = train(o, grid)
        check(got, want)
        check(train(o, grid, lengths=lengths), want_ragged)
        assert all(torch.equal(got[k], t) for k, t in train(o, grid).items()) and call.calls == 3
