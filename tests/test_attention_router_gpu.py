"""Runs of several networks into the same folders: each trains, stores its own results and is found again."""
import os

import pytest
import yaml

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_networks_share_their_folders(tmp_path):
    from im2im_uq_amd import nn_ops
    from im2im_uq_amd.core.scripts.router import expand_sweep, run_experiment
    before = nn_ops.get_compute_dtype()
    params = expand_sweep(yaml.safe_load(open(os.path.join(ROOT, "experiments", "synthetic_fastmri", "config.yml"))))[0]
    params.update(output_dir=str(tmp_path / "out"), checkpoint_dir=str(tmp_path / "ckpt"), num_images=16, side_length=48, epochs=1, batch_size=4,
                  num_lambdas=50, num_validation_images=1, checkpoint_every=1, load_from_checkpoint=True)
    networks = [dict(), dict(attention="relative"), dict(attention="relative", attention_blocks=2), dict(attention="differential")]
    try:
        for extra in networks:
            res = run_experiment(dict(params, **extra))
            assert res is not None and 0.0 <= float(res["risk"]) <= 1.0, extra
        for extra in networks:
            assert run_experiment(dict(params, **extra)) is None                 # stored before
    finally:
        nn_ops.set_compute_dtype("bf16" if before.itemsize == 2 else "fp32")
    files = os.listdir(tmp_path / "out")
    assert sum(f.startswith("results_") for f in files) == sum(f.startswith("loss_table_") for f in files) == len(networks)
    assert len([f for f in os.listdir(tmp_path / "ckpt") if f.startswith("CP_epoch1_")]) == len(networks)
