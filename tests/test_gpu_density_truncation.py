"""Density control appends whole chunks: which of the counter sampler's picks that leaves out."""
import pytest
import torch

from litegs_amd import densify as D
from litegs_amd import stochastic
from tests.test_gpu_stochastic_path import _grown

pytestmark = pytest.mark.gpu


def _lost(monkeypatch, percent_dense):
    """-> (picks, ascending; those of them that were not appended)"""
    seen = []
    real = stochastic.sample_distinct
    monkeypatch.setattr(stochastic, "sample_distinct", lambda *a, **kw: (seen.append(real(*a, **kw)), seen[-1])[1])
    ps, ctl, out = _grown(positive=1.0, epoch=10, percent_dense=percent_dense)                 # 2741 picks, 21 chunks: 53 are left out
    (picked,) = seen
    n = ps["sh_0"].shape[-2] * ps["sh_0"].shape[-1]
    colour, new = ps["sh_0"].detach().reshape(3, -1), out[3].detach().reshape(3, -1)
    assert ctl.last["appended"] > 0 and picked.numel() - ctl.last["appended"] > 20
    # (nothing is pruned here: the appended ones, whose colours are their parents', are the last)
    child = new[:, n:]
    gone = [i for i in picked.tolist() if not (child == colour[:, i:i + 1]).all(dim=0).any()]
    assert child.shape[1] == ctl.last["appended"] and len(gone) == picked.numel() - ctl.last["appended"]
    return picked, torch.tensor(gone)


@pytest.mark.parametrize("percent_dense", [1e9, 0.0])                  # all of them cloned, all of them split
def test_picks_lost_to_whole_chunks_are_spread_over_the_cloud(percent_dense, monkeypatch):
    """at random, n of the picks lie in the lower half of the index range with a standard deviation of sqrt(n) / 2 at most: five of them"""
    picked, gone = _lost(monkeypatch, percent_dense)
    n, half = gone.numel(), picked[picked.numel() // 2].item()
    assert abs(int((gone < half).sum()) - n / 2) <= 2.5 * n ** 0.5


def test_the_mixed_order_is_a_permutation_of_the_counter_alone():
    s = D.CounterSampler(3)
    orders = []
    for _ in range(2):
        s.begin(7, torch.device("cuda"))
        orders.append([s.mixed(torch.arange(1000, device="cuda")) for _ in range(2)])
    (a, b), (c, d) = orders
    assert torch.equal(a, c) and torch.equal(b, d) and not torch.equal(a, b)
    assert torch.equal(a.sort().values, torch.arange(1000, device="cuda"))
    assert s.mixed(torch.zeros(0, dtype=torch.int64, device="cuda")).numel() == 0


def test_torchs_order_is_left_alone():
    x = torch.tensor([5, 2, 9])
    assert D.Sampler(1).mixed(x) is x
