"""The attention operators and autograd: tangents are refused, never dropped, and calls of no tokens are part of the graph."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from im2im_uq_amd import attn_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def calls():
    """(name, function, its tensors)"""
    r = lambda *s: torch.randn(*s, device=DEV)  # noqa: E731
    grid, vec = (3, 4), lambda: r(16)  # noqa: E731
    return [
        ("grid", lambda q, k, v, t: attn_ops.grid_attention(q, k, v, t, grid), [r(2, 12, 2, 8), r(2, 12, 2, 8), r(2, 12, 2, 8), r(2, 2, 2)]),
        ("token", lambda q, k, v, t: attn_ops.grid_attention(q, k, v, t, grid, q_start=5), [r(2, 1, 2, 8), r(2, 12, 2, 8), r(2, 12, 2, 8), r(2, 2, 2)]),
        ("diff", lambda q, k, v, t, lam: attn_ops.diff_grid_attention(q, k, v, lam, t, grid),
         [r(2, 12, 4, 8), r(2, 12, 4, 8), r(2, 12, 2, 16), r(2, 2, 2), r(2)]),
        ("self", lambda qkv, t: attn_ops.grid_self_attention(qkv, 2, t, grid), [r(2, 12, 48), r(2, 2, 2)]),
        ("self diff", lambda qkv, t, lam: attn_ops.grid_self_attention(qkv, 2, t, grid, lam=lam), [r(2, 12, 96), r(2, 2, 2), r(2)]),
        ("norm", lambda x, w, b: attn_ops.token_norm(x, w, b, norm="layer"), [r(5, 16), vec(), vec()]),
        ("seam", lambda x, f, g, s, pw, pb, qw, qb: torch.cat(attn_ops.norm_gate_residual(x, f, g, s, pw, pb, qw, qb, norm="layer")),
         [r(5, 16), r(5, 16), r(5, 16), vec(), vec(), vec(), vec(), vec()]),
        ("residual", lambda x, f, pw: attn_ops.norm_gate_residual(x, f, post_weight=pw)[0], [r(5, 16), r(5, 16), vec()]),
    ]


@pytest.mark.parametrize("which", range(8))
@pytest.mark.parametrize("leaf", [False, True])
def test_tangents_are_refused(which, leaf):
    """forward-mode differentiation of any operand is an error, whether or not anything requires a gradient; without tangents a call inside a
    dual level gives what it gives outside"""
    _, fn, tensors = calls()[which]
    with torch.no_grad():
        want = fn(*tensors)
    for at in range(len(tensors)):
        with fwad.dual_level():
            assert torch.equal(fn(*tensors), want)
            args = [t.detach().requires_grad_(leaf) for t in tensors]
            args[at] = fwad.make_dual(args[at], torch.ones_like(args[at]))
            with pytest.raises(RuntimeError, match="jvp"):
                fn(*args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                fn(*args)
            if at == 0:                                      # through a view of a dual tensor
                args[0] = args[0].flip(0)
                with pytest.raises(RuntimeError, match="jvp"):
                    fn(*args)


def test_calls_of_nothing_are_in_the_graph():
    """no batch, no query, no row: every operand's gradient is there, and zero"""
    r = lambda *s: torch.randn(*s, device=DEV)  # noqa: E731
    w = lambda: r(16)  # noqa: E731
    nan = torch.full((2, 2, 2), float("nan"), device=DEV)
    cases = [
        (lambda q, k, v, t: attn_ops.grid_attention(q, k, v, t, (3, 4)), [r(0, 12, 2, 8), r(0, 12, 2, 8), r(0, 12, 2, 8), nan]),
        (lambda q, k, v, t: attn_ops.grid_attention(q, k, v, t, (3, 4)), [r(2, 0, 2, 8), r(2, 12, 2, 8) * float("inf"), r(2, 12, 2, 8), r(2, 2, 2)]),
        (lambda q, k, v, t, lam: attn_ops.diff_grid_attention(q, k, v, lam, t, (3, 4)), [r(2, 0, 4, 8), r(2, 12, 4, 8), r(2, 12, 2, 16), r(2, 2, 2), r(2)]),
        (lambda qkv, t: attn_ops.grid_self_attention(qkv, 2, t, (3, 4)), [r(0, 12, 48), r(2, 2, 2)]),
        (lambda qkv, t, lam: attn_ops.grid_self_attention(qkv, 2, t, (3, 4), lam=lam), [r(0, 12, 96), r(2, 2, 2), r(2)]),
        (lambda x, p, q: attn_ops.token_norm(x, p, q, norm="layer"), [r(0, 16), w(), w()]),
        (lambda x, f, g, s, pw, pb, qw, qb: sum(t.sum() for t in attn_ops.norm_gate_residual(x, f, g, s, pw, pb, qw, qb, norm="layer")),
         [r(0, 16), r(0, 16), r(0, 16), w(), w(), w(), w(), w()]),
        (lambda x, f, pw: attn_ops.norm_gate_residual(x.bfloat16(), f.bfloat16(), post_weight=pw)[0], [r(3, 0, 16), r(3, 0, 16), w()]),
    ]
    for fn, tensors in cases:
        for at in [*range(len(tensors)), None]:              # each alone, and all
            args = [t.detach().clone().requires_grad_(at is None or n == at) for n, t in enumerate(tensors)]
            leaves = [t for t in args if t.requires_grad]
            grads = torch.autograd.grad(fn(*args).sum(), leaves)
            assert all(g.shape == t.shape and (g == 0).all() for g, t in zip(grads, leaves))
        with torch.no_grad():
            fn(*tensors)
