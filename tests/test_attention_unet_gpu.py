"""The attention operators together, as the U-Net runs them: AttentionBottleneck against plain 64-bit torch, UNet(attention=...) through a training
step, the graphed training loop, evaluation, a checkpoint and the router."""
import math
import os

import pytest
import torch
import yaml
from torch.utils.data import TensorDataset

from attention_reference import axis_bucket
from conftest import ROOT

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PARAMS = dict(uncertainty_type="quantiles", q_lo=0.05, q_hi=0.95, q_lo_weight=1, q_hi_weight=1, mse_weight=1, alpha=0.1, delta=0.1, num_lambdas=50,
              rcps_loss="fraction_missed", minimum_lambda=0, maximum_lambda=6, device=DEV, dataset="synthetic", batch_size=4, lr=1e-3,
              input_normalization="standard", output_normalization="min-max", num_validation_images=2)


@pytest.fixture(autouse=True)
def _restore_dtype():
    from im2im_uq_amd import nn_ops
    yield
    nn_ops.set_compute_dtype("bf16")


def plain_bottleneck(module, p, x):
    """the same blocks from their formulas, on parameters `p` and an input of any type"""
    b, c, gh, gw = x.shape
    t = x.permute(0, 2, 3, 1).reshape(b, gh * gw, c)
    rms = lambda v, w: v / (v.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w  # noqa: E731
    at = torch.arange(gh * gw, device=x.device)
    y, xx = at // gw, at % gw
    for i, blk in enumerate(module.blocks):
        g = lambda n: p[f"blocks.{i}.{n}"]  # noqa: E731, B023
        lin = lambda v, n: v @ g(n + ".weight").flatten(1).T  # noqa: E731
        h = rms(t, g("pre_weight"))
        maps, heads = (2 if blk.lam is not None else 1), blk.heads
        d = c // (heads * maps)
        q, k, v = lin(h, "qkv").chunk(3, -1)
        q, k = (u.reshape(b, -1, heads, maps, d).permute(0, 2, 3, 1, 4) for u in (q, k))
        v = v.reshape(b, -1, heads, maps * d).permute(0, 2, 1, 3)
        n = blk.table.shape[0]
        bias = g("table")[axis_bucket(y[None] - y[:, None], n, module.max_distance), axis_bucket(xx[None] - xx[:, None], n, module.max_distance)]
        s = torch.softmax(q @ k.transpose(3, 4) / math.sqrt(d) + bias.permute(2, 0, 1)[None, :, None], -1)
        a = s[:, :, 0] - g("lam")[None, :, None, None] * s[:, :, 1] if maps == 2 else s[:, :, 0]
        f = lin((a @ v).permute(0, 2, 1, 3).reshape(b, -1, c), "proj")
        t = t + g("scale") * torch.sigmoid(lin(h, "gate")) * rms(f, g("post_weight"))
    return t.reshape(b, gh, gw, c).permute(0, 3, 1, 2)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("kind,blocks,channels,grid", [("relative", 1, 64, (6, 9)), ("relative", 2, 128, (8, 8)), ("differential", 2, 128, (5, 12))])
def test_bottleneck(kind, blocks, channels, grid, mode):
    """Norm-relative bounds.  fp32: a block is eight steps of 32-bit sums of at most C products, (C + 8) 2^-24 of their magnitudes each, twice that
    many in the backward, doubled for what cancels in a gradient.  bf16: sixteen stored roundings of 2^-8 a block forward and backward."""
    from im2im_uq_amd import nn_ops
    from im2im_uq_amd.core.models.trunks.attention import AttentionBottleneck
    nn_ops.set_compute_dtype(mode)
    torch.manual_seed(0)
    m = AttentionBottleneck(channels, kind, blocks).to(DEV)
    with torch.no_grad():
        for n, q in m.named_parameters():
            if n.endswith("table") or n.endswith("scale"):
                q.copy_(torch.randn_like(q) * 0.5)
    x = torch.randn(2, channels, *grid, device=DEV)
    x = x.to(nn_ops.get_compute_dtype()).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    out = m(x)
    assert out.shape == x.shape and out.dtype == x.dtype and out.permute(0, 2, 3, 1).is_contiguous()
    g = torch.randn_like(out)
    grads = torch.autograd.grad(out, [x, *m.parameters()], g)
    x64 = x.detach().double().requires_grad_(True)
    p64 = {k: v.detach().double().requires_grad_(True) for k, v in m.named_parameters()}
    ref = plain_bottleneck(m, p64, x64)
    want = torch.autograd.grad(ref, [x64, *p64.values()], g.double())
    bound = blocks * (2 * 3 * 8 * (channels + 8) * 2.0 ** -24 if mode == "fp32" else 16 * 2.0 ** -8)
    for name, a, b in zip(["out", "x", *p64], [out, *grads], [ref, *want]):
        off = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        assert off <= bound, (name, off, bound)


def test_default_network_is_the_same():
    from im2im_uq_amd.core.models.trunks.unet import UNet
    torch.manual_seed(3)
    plain = UNet(1, 1, depth=2, base=32).state_dict()
    torch.manual_seed(3)
    with_ = UNet(1, 1, depth=2, base=32, attention="relative", attention_blocks=2).state_dict()
    assert list(plain) == [k for k in with_ if not k.startswith("attention.")]
    assert all(torch.equal(plain[k], with_[k]) for k in plain)
    for bad in (dict(attention="global"), dict(attention="relative", attention_blocks=0)):
        with pytest.raises(ValueError):
            UNet(1, 1, depth=2, base=32, **bad)


def _model(kind, norm="batch", blocks=2):
    from im2im_uq_amd.core.models.add_uncertainty import add_uncertainty
    from im2im_uq_amd.core.models.trunks.unet import UNet
    torch.manual_seed(1)
    return add_uncertainty(UNet(1, 1, depth=2, base=32, norm=norm, attention=kind, attention_blocks=blocks), dict(PARAMS)).to(DEV)


@pytest.mark.parametrize("norm", ["batch", "group"])
@pytest.mark.parametrize("kind", ["relative", "differential"])
def test_training_step_and_eval(kind, norm):
    """every parameter of the blocks gets a finite gradient, a step changes them, the same step gives the same bits; eval runs without a graph"""
    from im2im_uq_amd import nn_ops
    g = torch.Generator().manual_seed(5)
    x, y = torch.randn(3, 1, 36, 44, generator=g).to(DEV), torch.rand(3, 1, 36, 44, generator=g).to(DEV)
    results = []
    for _ in range(2):
        m = _model(kind, norm).train()
        opt = nn_ops.FusedAdam(m.parameters(), lr=1e-3)
        before = {n: p.detach().clone() for n, p in m.named_parameters() if ".attention." in n}
        assert len(before) == 2 * (8 if kind == "differential" else 7)
        m.loss_fn(m(x), y).backward()
        nn_ops.join_side_streams()
        for n, p in m.named_parameters():
            if ".attention." in n:
                assert p.grad is not None and p.grad.isfinite().all(), n
        opt.step()
        assert all(not torch.equal(before[n], p) for n, p in m.named_parameters() if n in before)
        results.append({n: p.detach().clone() for n, p in m.named_parameters()})
        with torch.no_grad():
            out = m.eval()(x)
        assert out.shape == (3, 3, 1, 36, 44) and out.isfinite().all()
    assert all(torch.equal(results[0][n], results[1][n]) for n in results[0])


def test_graphed_training_equals_eager(tmp_path):
    """train_net with the step in a HIP graph (a short last batch among the steps) ends in the eager loop's parameters, and its checkpoint loads"""
    from im2im_uq_amd.core.scripts.train import train_net
    g = torch.Generator().manual_seed(7)
    data = TensorDataset(torch.randn(18, 1, 32, 32, generator=g), torch.rand(18, 1, 32, 32, generator=g))
    got = []
    for graph in (False, True):
        m = _model("differential")
        cfg = dict(PARAMS, hip_graph=graph, checkpoint_dir=str(tmp_path / str(graph)))
        torch.manual_seed(11)
        m = train_net(m, data, data, DEV, 3, 4, 1e-3, False, cfg["checkpoint_dir"], 3, 100, cfg)
        got.append({n: p.detach().clone() for n, p in m.named_parameters()})
    assert all(torch.equal(got[0][n], got[1][n]) for n in got[0])
    name = [f for f in os.listdir(tmp_path / "True") if f.startswith("CP_epoch3")][0]
    from im2im_uq_amd.compat import load_reference_checkpoint
    again = load_reference_checkpoint(str(tmp_path / "True" / name)).to(DEV)
    assert all(torch.equal(got[1][n], p.detach().to(DEV)) for n, p in again.named_parameters())


def test_router_with_attention(tmp_path):
    from im2im_uq_amd.core.scripts.router import expand_sweep, run_experiment
    params = expand_sweep(yaml.safe_load(open(os.path.join(ROOT, "experiments", "synthetic_fastmri", "config.yml"))))[0]
    params.update(output_dir=str(tmp_path / "out"), checkpoint_dir=str(tmp_path / "ckpt"), num_images=16, side_length=48, epochs=1, batch_size=4,
                  num_lambdas=50, num_validation_images=1, attention="relative", attention_blocks=2)
    res = run_experiment(params)
    assert res["spatial_miscoverage"].shape == (48, 48) and 0.0 <= float(res["risk"]) <= 1.0
