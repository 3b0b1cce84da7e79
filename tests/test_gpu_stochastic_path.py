"""The random draws where the framework uses them: opacity dropout of training steps, the density controller's counter sampler, a chain of
them on another stream and in captured graphs."""
import os
import sys

import numpy as np
import pytest
import torch

from litegs_amd import densify as D
from litegs_amd import optimizer as opt_mod
from litegs_amd import render as R
from litegs_amd import stochastic
from litegs_amd import wrapper
from tests import stochastic_reference as ref
from tests.util import case

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tools"))


# ---- opacity dropout -----------------------------------------------------------------------------------------------------------------
def _render(c, params, drop):
    """-> (img, culled opacity, visible chunk ids, their number) of one view"""
    pp = R.PipelineParams()
    view, proj, planes = [torch.from_numpy(x).cuda() for x in (c["view"], c["proj"], c["planes"])]
    out = R.render_preprocess(None, None, planes, view, *params, None, None, pp, c["degree"], *(() if drop is None else (drop,)))
    img, *_ = R.render(view, proj, *out[2:], out[1] * pp.cluster_size, None, None, c["degree"], (c["H"], c["W"]), pp)
    return img, out[-1], out[0], out[1]


def _params(c):
    return [torch.nn.Parameter(torch.from_numpy(p).cuda()) for p in c["params"]]


def test_dropped_opacities_are_those_of_the_whole_cloud():
    c = case("small")
    params = _params(c)
    opacity = params[5]
    with torch.no_grad():
        _, plain, ids, num = _render(c, params, None)
        img, dropped, ids2, _ = _render(c, params, (0.4, 11, 5))
    n = int(num.item())
    assert torch.equal(ids[:n], ids2[:n])
    keep = torch.from_numpy(ref.kept(np.arange(opacity.numel()), 0.4, 11, 5)).cuda().view(opacity.shape[-2:])
    m = keep[ids[:n]].reshape(-1)
    want = torch.where(m, plain[0, : n * 128] * torch.tensor(1 / 0.6, device="cuda"), torch.zeros((), device="cuda"))
    assert torch.equal(dropped[0, : n * 128], want)
    # ... and the image is that of a cloud without the dropped Gaussians: the same as with their opacities put to nothing by hand
    pp = R.PipelineParams()
    view, proj, planes = [torch.from_numpy(x).cuda() for x in (c["view"], c["proj"], c["planes"])]
    out = R.render_preprocess(None, None, planes, view, *params, None, None, pp, c["degree"])
    by_hand = torch.zeros_like(out[-1])
    by_hand[0, : n * 128] = want
    img2, *_ = R.render(view, proj, *out[2:-1], by_hand, out[1] * pp.cluster_size, None, None, c["degree"], (c["H"], c["W"]), pp)
    assert torch.equal(img, img2)


def test_dropout_without_chunks_draws_the_same_mask():
    c = case("small")
    flat = [p.detach().reshape(*p.shape[:-2], -1).contiguous() for p in _params(c)]
    pp = R.PipelineParams(cluster_size=0)
    view, _, planes = [torch.from_numpy(x).cuda() for x in (c["view"], c["proj"], c["planes"])]
    out = R.render_preprocess(None, None, planes, view, *flat, None, None, pp, c["degree"], (0.4, 11, 5))
    keep = torch.from_numpy(ref.kept(np.arange(flat[5].shape[-1]), 0.4, 11, 5)).cuda()
    assert torch.equal(out[-1][0] > 0, keep)


def test_gradients_of_a_render_with_dropout():
    """against the same render with the mask applied by elementary operations: the blend backward adds in no fixed order, so the two runs of
    the same kernels agree to 1e-4 of the largest gradient; a dropped Gaussian has no opacity gradient at all"""
    c = case("small")
    w = torch.from_numpy(np.random.default_rng(1).standard_normal((1, 3, c["H"], c["W"])).astype(np.float32)).cuda()
    grads = []
    for by_hand in (False, True):
        params = _params(c)
        opacity = params[5]
        if by_hand:
            keep = torch.from_numpy(ref.kept(np.arange(opacity.numel()), 0.3, 2, 9)).cuda().view(opacity.shape[-2:])
            real = stochastic.dropout
            try:
                stochastic.dropout = lambda x, p, seed, offset, chunk_ids: x * (keep[chunk_ids].to(x.dtype) / (1 - p))
                img, _, ids, num = _render(c, params, (0.3, 2, 9))
            finally:
                stochastic.dropout = real
        else:
            img, _, ids, num = _render(c, params, (0.3, 2, 9))
        (img * w).sum().backward()
        n = int(num.item())
        grads.append([p.grad.to_dense(n) for p in params])
    for a, b in zip(*grads):
        assert a.isfinite().all() and (a - b).abs().max() <= 1e-4 * b.abs().max()
    dropped = ~torch.from_numpy(ref.kept(np.arange(opacity.numel()), 0.3, 2, 9)).cuda().view(opacity.shape)
    assert (grads[0][5][dropped] == 0).all() and (grads[0][5][~dropped] != 0).any()


def test_training_steps_draw_new_masks_and_evaluation_none():
    from litegs_amd.trainer import SyntheticTrainer
    tr = SyntheticTrainer(4096, 128, 96, 120.0, n_frames=2, fused=False)
    tr.opacity_dropout, tr.opacity_dropout_seed = 0.25, 7
    seen, real = [], stochastic.dropout

    def spy(x, p, seed, offset, **kw):
        y = real(x, p, seed, offset, **kw)
        seen.append((p, seed, offset, (y == 0).float().mean().item()))
        return y

    try:
        stochastic.dropout = spy
        before = [p.detach().clone() for p in tr.params]
        for k in range(3):
            assert torch.isfinite(tr.step(k)).item()
        tr.forward_only(0)
    finally:
        stochastic.dropout = real
    assert [s[:3] for s in seen] == [(0.25, 7, 0), (0.25, 7, 1), (0.25, 7, 2)]
    assert all(abs(s[3] - 0.25) < 0.1 for s in seen)
    assert all(p.isfinite().all() for p in tr.params) and any((a != b).any() for a, b in zip(before, tr.params))
    tr.close()
    tr = SyntheticTrainer(4096, 128, 96, 120.0, n_frames=2)
    tr.opacity_dropout = 0.25
    with pytest.raises(RuntimeError, match="operator path"):
        tr.step(0)
    tr.close()


def test_start_trains_with_dropout_and_counter_sampler(tmp_path, monkeypatch):
    import make_colmap_scene as M
    from litegs_amd import arguments as A
    from litegs_amd import training
    M.make(str(tmp_path / "scene"), points=2048, frames=8, width=192, height=128, focal=170.0, sfm_fraction=0.6, seed=3)
    lp, op, pp, dp = A.get_default_arg()
    lp.source_path, lp.model_path, lp.eval, lp.resolution = str(tmp_path / "scene"), str(tmp_path / "m"), True, 1
    op.iterations, op.opacity_dropout = 7 * 6, 0.1
    dp.target_primitives, dp.densify_from, dp.densification_interval, dp.opacity_reset_interval, dp.sampler, dp.densify_until = 6000, 2, 3, 6, "counter", 6
    keys = []                                                        # (seed, offset) of every draw of the run

    def spy(name, at):
        real = getattr(stochastic, name)
        monkeypatch.setattr(stochastic, name, lambda *a, **kw: (keys.append(tuple(a[at:at + 2])), real(*a, **kw))[1])

    for name, at in (("dropout", 2), ("uniform", 1), ("normal", 1)):
        spy(name, at)
    trainer, hist = training.start(lp, op, pp, dp, test_epochs=[0, 5], log=lambda *a: None)
    assert len(keys) > 42 and len(set(keys)) == len(keys) and len({k[0] for k in keys}) == 2
    assert not trainer.fused and trainer.training_steps == 42 and type(trainer.controller.sampler) is D.CounterSampler
    assert all(p.isfinite().all() for p in trainer.params) and hist[-1]["points_after"] > hist[0]["points"]
    op.opacity_dropout = 1.0
    with pytest.raises(ValueError, match="opacity_dropout"):
        training.start(lp, op, pp, dp, log=lambda *a: None)


# ---- density control -----------------------------------------------------------------------------------------------------------------
class Evidence:
    """statistics of a made-up epoch: half of the Gaussians have an error score"""

    def __init__(self, n, positive=0.5):
        g = torch.Generator(device="cuda").manual_seed(5)
        self.err = torch.rand(n, generator=g, device="cuda")
        self.cnt = (torch.rand(n, generator=g, device="cuda") < positive).float()

    def var(self, key):
        return self.err, self.cnt

    def mean(self, key):
        return None

    def all_reduce(self, group=None):
        pass

    def reset(self, *a, **k):
        pass


def _grown(n_chunks=40, positive=0.5, epoch=5, **dp):
    g = torch.Generator(device="cuda").manual_seed(1)
    shape = dict(xyz=(3,), scale=(3,), rot=(4,), sh_0=(1, 3), sh_rest=(15, 3), opacity=(1,))
    ps = {n: torch.nn.Parameter(torch.randn((*shape[n], n_chunks, 128), generator=g, device="cuda")) for n in D.PARAM_NAMES}
    opt, _ = opt_mod.get_optimizer(*[ps[n] for n in D.PARAM_NAMES], 1.0, opt_mod.OptimizationParams())
    params = D.DensifyParams(densify_until=41, target_primitives=20000, sampler="counter", **dp)
    ctl = D.DensityController(1.0, params, 128, n_chunks * 128, Evidence(n_chunks * 128, positive), D.make_sampler(params, 3))
    return ps, ctl, ctl.step(opt, epoch)


def test_counter_sampler_decides_the_same_every_time():
    (_, ctl, a), (_, _, b), (_, _, other) = _grown(), _grown(), _grown(epoch=10)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert ctl.last["split"] + ctl.last["clone"] == ctl.last["budget"] and ctl.last["appended"] > 0
    assert a[0].shape != other[0].shape or not torch.equal(a[0], other[0])


def test_counter_sampler_is_the_definition():
    s = D.CounterSampler(9, temperature=0.5, top_p=0.9)
    score = torch.rand(5000, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").square()
    score[::3] = 0
    s.begin(4, score.device)
    picked = s.multinomial(score, 700)
    u = np.minimum(((ref.words(np.arange(5000), 9, 4 << 8) + 0.5) / 2.0 ** 32).astype(np.float32), np.float32(1 - 2.0 ** -24))
    want = ref.distinct_row(score.double().cpu().numpy(), u, 700, False, 0.5, 0, 0.9, 0.0, 3e38)
    assert np.array_equal(picked.cpu().numpy(), want[want >= 0]) and (score[picked] > 0).all()


def test_counter_sampler_with_little_or_no_evidence():
    for positive in (0.0, 0.01):
        ps, ctl, out = _grown(positive=positive)
        assert all(o.isfinite().all() for o in out)
        assert ctl.last["split"] + ctl.last["clone"] <= int((ctl.score(ps["opacity"].detach().reshape(1, -1)) > 0).sum())


def test_more_gaussians_than_torch_draws_from():
    n = (1 << 24) + 77777
    g = torch.Generator(device="cuda").manual_seed(3)
    score = torch.rand(n, generator=g, device="cuda").square()
    s = D.CounterSampler(1)
    s.begin(0, score.device)
    picked = s.multinomial(score, 200000)
    u = np.minimum(((ref.words(np.arange(n), 1, 0) + 0.5) / 2.0 ** 32).astype(np.float32), np.float32(1 - 2.0 ** -24))
    x = score.double().cpu().numpy()
    with np.errstate(divide="ignore"):
        key = np.log(x) - np.log(-np.log1p(-u.astype(np.float64)))
    want = np.sort(np.argpartition(-key, 200000)[:200000])
    assert np.array_equal(picked.cpu().numpy(), want)


# ---- together, on other streams and in graphs ----------------------------------------------------------------------------------------
def _chain(score, x, step):
    """what an epoch's end and a step draw, in order"""
    u = stochastic.uniform(score.shape, 3, step)
    few = stochastic.sample_distinct(score, u, 500, logits=False, temperature=0.8, top_p=0.95)
    again = stochastic.sample(score, u[:, :300], logits=False, top_k=score.shape[-1] // 2)
    shift = stochastic.normal(score[:, :3001], 4, step)
    return [few, again, shift, stochastic.dropout(x, 0.3, 5, step, shared=1)]


@pytest.mark.parametrize("V", [9000, 120000])
def test_chain_on_another_stream(V):
    score, x = torch.rand((2, V), device="cuda"), torch.randn((3, V), device="cuda")
    want = _chain(score, x, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _chain(score, x, 8)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("V", [9000, 120000])
def test_chain_in_captured_graphs(V):
    """two graphs over one counter that the graphs advance themselves: every replay draws what an eager call with the same count draws"""
    score, x = torch.rand((2, V), device="cuda"), torch.randn((3, V), device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    graphs = []
    for _ in range(2):
        _chain(score, x, step)                                       # (warm: everything that is loaded once is loaded)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step.add_(1)
            out = _chain(score, x, step)
        graphs.append((graph, out))
    step.zero_()
    count = 0
    for k in (0, 1, 1, 0, 1):
        graph, out = graphs[k]
        graph.replay()
        count += 1
        torch.cuda.synchronize()
        assert int(step) == count
        eager = _chain(score, x, count)
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), (k, count)
        score.mul_(0.99)                                             # other inputs for the next replay, in place
        assert not torch.equal(eager[3], _chain(score, x, count + 1)[3])


def test_forward_and_backward_in_a_captured_graph():
    x, dy = torch.randn((4, 5, 128), device="cuda", requires_grad=True), torch.randn((4, 5, 128), device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                                    # warm up off the capturing stream
        torch.autograd.grad(stochastic.dropout(x, 0.5, 1, step, shared=1), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = stochastic.dropout(x, 0.5, 1, step, shared=1)
        (dx,) = torch.autograd.grad(y, x, dy)
    for k in (3, 4, 9):
        step.fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        m = torch.from_numpy(ref.kept(np.arange(640).reshape(5, 128), 0.5, 1, k)).cuda()
        assert torch.equal(y, torch.where(m, 2 * x, torch.zeros((), device="cuda"))) and torch.equal(dx, torch.where(m, 2 * dy, torch.zeros((), device="cuda")))
        torch.cuda.synchronize()
