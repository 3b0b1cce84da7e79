"""Random draws, the parts that need no GPU: the generator's published answers, the reference forms' own properties, refusals."""
import numpy as np
import pytest
import torch

from litegs_amd import stochastic
from litegs_amd._lib import lib
from tests import stochastic_reference as ref

INVALID = 1          # hipErrorInvalidValue


def test_generator_known_answers():
    """the three published vectors of Philox4x32-10 (Salmon et al. 2011, the authors' test set)"""
    M = 0xFFFFFFFF
    for counter, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
            ((M, M, M, M), (M, M), (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
            ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
        got = ref.philox(np.array([counter], dtype=np.uint64), key)[0]
        assert tuple(int(v) for v in got) == want


def test_words_are_a_function_of_the_index():
    i = np.array([0, 1, 5, 2 ** 32 + 3, 2 ** 34, 2 ** 62 - 1])
    w = ref.words(i, 2 ** 64 - 3, 2 ** 40 + 9)
    assert all(int(ref.words(np.array([k]), 2 ** 64 - 3, 2 ** 40 + 9)[0]) == int(v) for k, v in zip(i, w))
    assert len(set(int(v) for v in w)) == len(w)


def test_reference_draws_follow_the_masses():
    rng = np.random.default_rng(0)
    x = np.array([0.0, 1.0, 2.0, -np.inf, np.nan, 3.0])
    u = rng.random(200000).astype(np.float32)
    got = np.bincount(ref.sample_row(x, u, True, 1.0, 0, 1.0, 0.0, 3e38), minlength=6) / len(u)
    p = np.exp(x); p[np.isnan(p)] = 0; p /= p.sum()
    assert np.abs(got - p).max() < 5 * np.sqrt(0.25 / len(u))
    # without replacement: the first of one draw follows the masses too
    one = np.array([ref.distinct_row(x, rng.random(6).astype(np.float32), 1, True, 1.0, 0, 1.0, 0.0, 3e38)[0] for _ in range(20000)])
    assert np.abs(np.bincount(one, minlength=6) / 20000 - p).max() < 5 * np.sqrt(0.25 / 20000)


def test_no_cpu_path():
    x = torch.zeros(4, 8)
    for call in (lambda: stochastic.dropout(x, 0.5, 1), lambda: stochastic.normal(x, 1), lambda: stochastic.sample(x, torch.zeros(4, 1)),
                 lambda: stochastic.sample_distinct(x, x, 2), lambda: stochastic.uniform((4,), 1, device=torch.device("cpu"))):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("bad", [-1, 1 << 64, 1.0, True, None])
def test_seed_is_refused(bad):
    with pytest.raises(ValueError):
        stochastic._key(bad, 0, torch.device("cuda", 0), "draw")


@pytest.mark.parametrize("bad", [-1, 1 << 63, 0.5, torch.zeros(2, dtype=torch.int64), torch.zeros(1), torch.zeros(1, dtype=torch.int64)])
def test_offset_is_refused(bad):
    with pytest.raises(ValueError):
        stochastic._key(0, bad, torch.device("cuda", 0), "draw")


def test_largest_seed_keeps_its_bits():
    assert stochastic._key((1 << 64) - 1, 7, torch.device("cuda", 0), "draw") == (-1, 7, None)
    assert stochastic._key(1 << 63, 7, torch.device("cuda", 0), "draw")[0] == -(1 << 63)


def _sample(**kw):
    a = dict(scores=16, dtype=0, ss=8, u=16, us=8, R=1, V=8, n=2, distinct=0, logits=1, T=1.0, k=0, p=1.0, m=0.0, out=16, temp=16, tb=1 << 40)
    a.update(kw)
    return lib().lg_sample(a["scores"], a["dtype"], a["ss"], a["u"], a["us"], a["R"], a["V"], a["n"], a["distinct"], a["logits"], a["T"], a["k"],
                           a["p"], a["m"], a["out"], a["temp"], a["tb"], None)


@pytest.mark.parametrize("kw", [dict(T=0.0), dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")), dict(k=-1), dict(p=0.0), dict(p=1.5), dict(p=float("nan")),
                                dict(m=-0.1), dict(m=1.1), dict(m=float("nan")), dict(dtype=3), dict(dtype=-1), dict(scores=None), dict(u=None),
                                dict(out=None), dict(R=-1), dict(V=-1), dict(n=-1), dict(V=1 << 31), dict(distinct=1, n=9), dict(R=1 << 31)])
def test_c_entry_refuses_bad_sampling_arguments(kw):
    assert _sample(**kw) == INVALID


def test_c_entry_of_empty_calls():
    assert _sample(R=0) == 0 and _sample(n=0) == 0
    assert lib().lg_dropout(None, None, 0, 0, 8, 0.5, 0, 0, None, None, 1, None) == 0
    assert lib().lg_random_draw(None, None, 0, 0, 0, 0, None, None) == 0


@pytest.mark.parametrize("kw", [dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(dtype=7), dict(x=None), dict(y=None), dict(ids=16, S=0), dict(ids=16, S=3)])
def test_c_entry_refuses_bad_dropout_arguments(kw):
    a = dict(x=16, y=16, dtype=0, p=0.5, ids=None, S=1)
    a.update(kw)
    assert lib().lg_dropout(a["x"], a["y"], a["dtype"], 1, 8, a["p"], 0, 0, None, a["ids"], a["S"], None) == INVALID


def test_c_entry_refuses_a_bad_draw():
    assert lib().lg_random_draw(None, None, 0, 8, 0, 0, None, None) == INVALID
    assert lib().lg_random_draw(None, 16, 5, 8, 0, 0, None, None) == INVALID


# ---- where the framework takes them from ----------------------------------------------------------------------------------------------
def test_sampler_of_the_density_controller_is_chosen_by_its_parameters():
    from types import SimpleNamespace
    from litegs_amd import densify as D
    assert type(D.make_sampler(D.DensifyParams(), 3)) is D.Sampler and type(D.make_sampler(SimpleNamespace(), 3)) is D.Sampler
    s = D.make_sampler(D.DensifyParams(sampler="counter", sample_top_p=0.9, sample_temperature=0.5), 3)
    assert type(s) is D.CounterSampler and s.seed == 3 and s.rule == dict(temperature=0.5, top_k=0, top_p=0.9, min_p=0.0)
    for bad in (dict(sampler="other"), dict(sample_top_k=5), dict(sample_min_p=0.1), dict(sample_temperature=2.0)):
        with pytest.raises(ValueError):
            D.make_sampler(D.DensifyParams(**bad))


@pytest.mark.parametrize("bad", [dict(seed=-1), dict(seed=1 << 63), dict(temperature=0.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=1.5), dict(top_p=0.0),
                                 dict(top_p=1.5), dict(min_p=-0.1)])
def test_counter_sampler_refuses_bad_options_before_training(bad):
    from litegs_amd import densify as D
    with pytest.raises(ValueError):
        D.CounterSampler(**bad)


def test_every_draw_of_a_run_has_a_counter_of_its_own():
    from litegs_amd import densify as D
    s, seen = D.CounterSampler(1), []
    for epoch in range(3):
        s.begin(epoch, torch.device("cpu"))
        seen += [s._next() for _ in range(4)]
    assert len(set(seen)) == len(seen)
    s.begin(1, torch.device("cpu"))
    assert s._next() == seen[4]                                      # ... and a repeated epoch the same ones


def test_command_line_carries_the_options():
    from argparse import ArgumentParser
    from litegs_amd import arguments as A
    parser = ArgumentParser()
    A.add_cmdline_args(parser)
    _, op, _, dp = A.extract(parser.parse_args(["--opacity_dropout", "0.1", "--sampler", "counter", "--sample_top_p", "0.95", "--sample_top_k", "7"]))
    assert op.opacity_dropout == 0.1 and (dp.sampler, dp.sample_top_p, dp.sample_top_k) == ("counter", 0.95, 7)
    _, op, _, dp = A.extract(parser.parse_args([]))
    assert op.opacity_dropout == 0.0 and dp.sampler == "torch"
