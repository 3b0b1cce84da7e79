"""Opacity dropout beside what else a training run does: the statistics of density control, the blend's limit of alpha, the executor."""
import pytest
import torch

from litegs_amd import densify as D
from litegs_amd.statistics import STATS
from litegs_amd.trainer import SyntheticTrainer

pytestmark = pytest.mark.gpu


# ---- statistics ----------------------------------------------------------------------------------------------------------------------
def _evidence(mode, p):
    """what density control decides by after a statistics epoch of one frame -> (flagged for pruning, times visible, score > 0)"""
    tr = SyntheticTrainer(4096, 128, 96, 120.0, n_frames=1, fused=False)
    try:
        tr.opacity_dropout, tr.opacity_dropout_seed = p, 7
        ctl = tr.enable_densify(D.DensifyParams(densify_from=0, densify_until=20, densification_interval=5, prune_mode=mode), 40, 1.0)
        opacity = tr.params[5].detach().clone().reshape(1, -1)          # (before the step)
        with tr.begin_epoch(0):
            assert STATS.active
            tr.step(0)
        return ctl.prune_mask(opacity.sigmoid()), STATS.visible_count.clone(), ctl.score(opacity) > 0
    finally:
        STATS.reset(0, 128, lambda epoch: False)
        tr.close()


@pytest.mark.parametrize("mode", ["weight", "threshold"])
def test_a_dropped_gaussian_is_not_taken_for_an_invisible_one(mode):
    plain, dropped = _evidence(mode, 0.0), _evidence(mode, 0.9)
    assert not plain[0].all() and plain[1].any()
    assert torch.equal(dropped[0], plain[0]) and torch.equal(dropped[1], plain[1]) and torch.equal(dropped[2], plain[2])
