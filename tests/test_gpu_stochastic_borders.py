"""The samplers where the masses before and behind a category differ by many powers of two, and at the ends of the range of ``u``: against
the 64-bit forms, index for index."""
import math

import numpy as np
import pytest
import torch

from litegs_amd import stochastic
from tests import stochastic_reference as ref
from tests.test_gpu_stochastic import DEV, TYPES, check_sample, rule, scores_of

pytestmark = pytest.mark.gpu

SMALL = [0.0, -1.0, math.nan, 1e-45, 1e-38, 1e-30, 1e-20, 1e-12, 1e-6]


def numbers(values, R):
    return torch.tensor(values, dtype=torch.float32, device=DEV).expand(R, len(values))


def test_a_far_larger_mass_behind_does_not_hide_a_small_one():
    """the threads of a workgroup hold four scores each: 1 lies in the first one's, 7 and 11 at the ends of the others'.  The masses are
    e^-40 = 4.2e-18, 1 and 1, so that 1e-18 of their total, 2e-18, still lies in the first"""
    x = torch.full((1, 12), -math.inf, device=DEV)
    x[0, 1], x[0, 7], x[0, 11] = -40.0, 0.0, 0.0
    assert stochastic.sample(x, numbers([0.0, -1.0, math.nan, 1e-45, 1e-18, 0.25, 0.75], 1)).tolist() == [[1, 1, 1, 1, 1, 7, 11]]


@pytest.mark.parametrize("V", [5, 12, 64, 300, 1000, 1024, 1025, 4096, 4097, 9000, 12288])
@pytest.mark.parametrize("T", [0.05, 0.1, 1.0])
def test_small_numbers_in_short_rows(V, T):
    for dtype in TYPES:
        for seed in range(4):
            x = scores_of("masked", 16, V, dtype, True, seed=seed)
            for kw in (dict(), dict(top_k=V // 2 + 65), dict(top_p=0.9999), dict(min_p=1e-30)):
                check_sample(x, numbers(SMALL, 16), logits=True, temperature=T, **kw)
        x = scores_of("steps", 16, V, dtype, False, seed=V)             # weights over the whole range of the type
        for kw in (dict(), dict(temperature=0.5), dict(top_k=V // 2 + 65)):
            check_sample(x, numbers(SMALL, 16), logits=False, **kw)


# A long row's masses are added up tile by tile (4096 scores), four tiles a thread
TILE = 4096


def test_a_far_larger_tile_behind_does_not_hide_a_small_one():
    x = torch.full((1, 9 * TILE), -math.inf, device=DEV)
    x[0, 5], x[0, 4 * TILE + 9], x[0, 7 * TILE + 3] = -80.0, -80.0 + math.log(1.5), 0.0
    p = math.exp(-80.0)
    assert stochastic.sample(x, numbers([0.5 * p, 1.2 * p, 2.0 * p, 3.0 * p], 1)).tolist() == [[5, 4 * TILE + 9, 4 * TILE + 9, 7 * TILE + 3]]


@pytest.mark.parametrize("V", [12289, 40000, 300001])
@pytest.mark.parametrize("T", [0.05, 0.1, 1.0])
def test_small_numbers_in_long_rows(V, T):
    """masses that fall by tiles and rise again, so that a thread's tiles hold sums far apart"""
    for dtype in TYPES:
        x = scores_of("masked", 3, V, dtype, True, seed=V)
        far = torch.rand(3, (V + TILE - 1) // TILE, generator=torch.Generator(device=DEV).manual_seed(V), device=DEV).mul(-60.0)
        y = (x.float() + far.repeat_interleave(TILE, dim=1)[:, :V] * T).to(dtype)
        for z in (x, y):
            for kw in (dict(), dict(top_k=V // 2), dict(top_p=0.9999), dict(min_p=1e-20)):
                check_sample(z, numbers(SMALL, 3), logits=True, temperature=T, **kw)


@pytest.mark.parametrize("V", [12, 12288, 12289, 5 * TILE])
@pytest.mark.parametrize("logits", [True, False])
def test_a_mass_below_the_least_number_is_none(V, logits):
    """masses are exp(l - max l) in 64 bits, whatever lies next to a score: exp(-750) is 0, exp(-100) is not"""
    T = 0.01
    x = torch.full((1, V), -math.inf if logits else 0.0, device=DEV)
    x[0, 1], x[0, 3], x[0, V - 1] = (-7.5, -1.0, 0.0) if logits else (math.exp(-7.5), math.exp(-1.0), 1.0)
    assert stochastic.sample(x, numbers([0.0, -1.0, math.nan, 1e-45, 0.5], 1), logits=logits, temperature=T).tolist() == [[3, 3, 3, 3, V - 1]]


@pytest.mark.parametrize("V", [300, 9000, 12289, 40000])
@pytest.mark.parametrize("T", [1e-30, 1e-3, 0.004, 0.01, 0.03])
def test_nothing_without_a_mass_is_drawn_by_a_small_number(V, T):
    for dtype in TYPES:
        for kind in ("normal", "masked", "ties"):
            x = scores_of(kind, 3, V, dtype, True, seed=V)
            for kw in (dict(), dict(top_k=V // 2), dict(top_p=0.99)):
                check_sample(x, numbers(SMALL, 3), logits=True, temperature=T, **kw)


@pytest.mark.parametrize("V", [12, 300, 4097, 12288, 12289, 40000, 300001])
@pytest.mark.parametrize("T", [1e-30, 0.004, 0.03, 0.1, 1.0])
def test_numbers_from_one_on_draw_the_last(V, T):
    """... with a mass, however small: what follows the large ones does not move their sum.  (The 64-bit form rounds the total, and what is
    above the rounded one is found before the last: from one on the answer is the definition's own, the last category with a mass.)"""
    def check(x, logits, **kw):
        a = rule(kw, logits)
        got = stochastic.sample(x, numbers([1.0, 1.5, math.inf], x.shape[0]), **a).cpu()
        for r, row in zip(x.double().cpu().numpy(), got.tolist()):
            who, _, mass = ref.filtered(r, big=torch.finfo(x.dtype).max, **a)
            assert row == [int(who[mass > 0][-1])] * 3, (x.shape, x.dtype, kw)
        check_sample(x, numbers([1.0 - 2.0 ** -24], x.shape[0]), logits=logits, **kw)

    for dtype in TYPES:
        for kind in ("normal", "masked"):
            x = scores_of(kind, 3, V, dtype, True, seed=V)
            x[0, V // 3], x[1, 0] = 30.0, 30.0
            for kw in (dict(), dict(top_k=V // 2), dict(top_k=min(V // 2, 50)), dict(top_p=0.99), dict(min_p=1e-30)):
                check(x, True, temperature=T, **kw)
        check(scores_of("steps", 3, V, dtype, False, seed=V), False)
