"""Opacity dropout beside what else a training run does: the statistics of density control, the blend's limit of alpha, the executor."""
import numpy as np
import pytest
import torch

from litegs_amd import densify as D
from litegs_amd import render as R
from litegs_amd.statistics import STATS
from litegs_amd.synthetic import orbit_cameras
from litegs_amd.trainer import SyntheticTrainer
from tests import stochastic_reference as ref

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


# ---- opacities above one -------------------------------------------------------------------------------------------------------------
P, SEED, OFFSET = 0.5, 3, 1


def _one_gaussian():
    """a cloud of one visible Gaussian in front of a camera, white, 20 pixels wide, opacity 0.95: 1.9 where dropout keeps it"""
    kept = int(np.flatnonzero(ref.kept(np.arange(128), P, SEED, OFFSET))[0])
    view, proj, planes = [torch.from_numpy(x).cuda() for x in orbit_cameras(1, 160, 128, 150.0, 150.0, 4.0)[0]]
    xyz = torch.zeros(3, 1, 128)
    scale = torch.full((3, 1, 128), 20.0 * 4.0 / 150.0).log()
    rot = torch.zeros(4, 1, 128)
    rot[0] = 1
    sh_0 = torch.full((1, 3, 1, 128), 0.4 / 0.28209479177387814)          # colour 0.9
    sh_rest = torch.zeros(15, 3, 1, 128)
    opacity = torch.full((1, 1, 128), -20.0)
    opacity[0, 0, kept] = 2.9444389
    params = [t.cuda().requires_grad_(True) for t in (xyz, scale, rot, sh_0, sh_rest, opacity)]
    pp = R.PipelineParams(sparse_grad=False)

    def render(params):
        out = R.render_preprocess(None, None, planes, view, *params, None, None, pp, 0, (P, SEED, OFFSET))
        assert out[-1].max() > 1.8
        img, *_ = R.render(view, proj, *out[2:], out[1] * pp.cluster_size, None, None, 0, (128, 160), pp, limit_opacity=True)
        return img

    return params, render


def _difference(params, render, loss, k, h):
    values = []
    with torch.no_grad():
        for s in (h, -h):
            moved = [p.detach() + s if i == k else p.detach() for i, p in enumerate(params)]
            values.append(loss(render(moved)).double().item())
    return (values[0] - values[1]) / (2 * h)


def test_gradients_of_opacities_above_one_are_those_of_the_image():
    """against central differences.  With k = -ln G of a pixel in (0.05, 0.6), G(s) = exp(-k e^(-2 s)) over s = ln scale has a third derivative
    of at most 8 (k + 3 k^2 + k^3) G < 16, so that a step of 2^-7 is off by 16 / 6 * 2^-14 = 1.6e-4 for a derivative 2 k G >= 0.09: 0.2 %; the image's
    roundings, 2^-23 of 1 over 2^-6, are below that.  One per cent holds both and what the blend's own sum rounds"""
    params, render = _one_gaussian()
    img = render(params)
    alpha = img.detach()[0, 0] / 0.9
    rim = (alpha > 0.57) & (alpha < 0.95)                              # inside the core that an opacity of 1.9 would saturate
    assert 0.98 < alpha.max() <= 1.0 and rim.sum() > 100
    loss = lambda im: im[0, 0][rim].sum()
    grads = torch.autograd.grad(loss(img), params)
    assert (grads[5] == 0).all() and _difference(params, render, loss, 5, 0.05) == 0
    want = _difference(params, render, loss, 1, 2.0 ** -7)
    assert want > 1 and abs(grads[1].sum().item() - want) <= 0.01 * want


def test_training_steps_limit_opacities(monkeypatch):
    seen = []
    real = R.wrapper.GaussiansRasterFunc.apply
    monkeypatch.setattr(R.wrapper.GaussiansRasterFunc, "apply", lambda *a: (seen.append(a[5].detach().max().item()), real(*a))[1])
    tr = SyntheticTrainer(4096, 128, 96, 120.0, n_frames=1, fused=False)
    try:
        tr.opacity_dropout = 0.9
        tr.step(0)
        assert seen == [1.0]
    finally:
        tr.close()


# ---- the executor --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fused,drop,warned", [(True, 0.1, True), (False, 0.1, False), (True, 0.0, False)])
def test_start_says_that_it_leaves_the_executor(fused, drop, warned, tmp_path):
    import os
    import sys
    import warnings
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tools"))
    import make_colmap_scene as M
    from litegs_amd import arguments as A
    from litegs_amd import training
    M.make(str(tmp_path / "scene"), points=1024, frames=2, width=96, height=64, focal=80.0, sfm_fraction=0.6, seed=3)
    lp, op, pp, dp = A.get_default_arg()
    lp.source_path, lp.model_path, lp.eval, lp.resolution = str(tmp_path / "scene"), str(tmp_path / "m"), False, 1
    op.iterations, op.opacity_dropout = 2, drop
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        trainer, _ = training.start(lp, op, pp, dp, fused=fused, log=lambda *a: None)
    assert any("without the native executor" in str(w.message) for w in seen) == warned
    assert trainer.fused == (fused and not drop)
    trainer.close()
