"""Files of runs that differ in their attention blocks have different names, those of the reference's network the reference's."""
import itertools

BASE = dict(dataset="synthetic", uncertainty_type="quantiles", batch_size=16, lr=0.001, input_normalization="standard", output_normalization="min-max")


def test_names_tell_the_networks_apart():
    from im2im_uq_amd.core.scripts.router import _suffix
    from im2im_uq_amd.core.scripts.train import _ckpt_name
    runs = [dict(BASE, attention=kind, attention_blocks=n) for kind, n in itertools.product(("relative", "differential"), (1, 2, 12))] + [BASE]
    assert len({_suffix(p) for p in runs}) == len({_ckpt_name("c", 3, p) for p in runs}) == len(runs)
    for same in (dict(BASE, attention=None), dict(BASE, attention=None, attention_blocks=4)):
        assert _suffix(same) == _suffix(BASE) == "synthetic_quantiles_16_0.001_standard_min-max"
        assert _ckpt_name("c", 3, same) == "c/CP_epoch3_synthetic_quantiles_16_0.001_standard_min-max.pth"
    assert _suffix(dict(BASE, attention="relative")) == _suffix(dict(BASE, attention="relative", attention_blocks=1))
