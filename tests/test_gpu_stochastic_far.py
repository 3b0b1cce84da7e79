"""Sampling without replacement where the approximate race keys decide little: temperatures that flatten or magnify everything, numbers that
repeat.  Against the 64-bit form, index for index."""
import pytest
import torch

from tests.test_gpu_stochastic import DEV, TYPES, check_distinct, draws_of, scores_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1e-30, 1e-20, 1e-8, 1e-5, 1e-3, 1e20, 1e30])
@pytest.mark.parametrize("V", [300, 9000, 70001])
@pytest.mark.parametrize("logits", [True, False])
def test_distinct_at_far_temperatures(T, V, logits):
    """slopes that spread nothing, or so much that the approximate keys end at the largest number: what is near the border goes by exact keys"""
    for dtype in TYPES:
        for kind in ("ties", "normal", "masked"):
            x = scores_of(kind, 2, V, dtype, logits, seed=8)
            for n in (1, V // 10, V // 2):
                check_distinct(x, draws_of((2, V)), n, logits=logits, temperature=T)
            check_distinct(x, draws_of((2, V)), 20, logits=logits, temperature=T, top_p=0.8)


@pytest.mark.parametrize("V", [300, 9000, 70001, 1200000])
def test_distinct_with_few_different_numbers(V):
    """whole parts of a row with one key: by numbers of three bits, by one for all, by numbers so small that they are clamped"""
    x = scores_of("ties", 1, V, torch.float32, True, seed=2)
    u = draws_of((1, V))
    for v in ((u * 8).floor() / 8, torch.full_like(u, 0.3), u * 1e-12, 1.0 - u * 2.0 ** -26):
        for T in (1.0, 1e-4):
            check_distinct(x, v, V // 7 + 1, logits=True, temperature=T)


def test_race_keys_next_to_the_series():
    """1 - u loses most where the series for small u ends (2^-6): keys of equal weights follow the numbers alone, in their order"""
    V = 60000
    step = torch.arange(V, device=DEV, dtype=torch.float32)
    u = (2.0 ** -6 + (step - V // 2) * 2.0 ** -29)[None]               # neighbours one or two floats apart, on either side of the border
    u = u[:, torch.randperm(V, generator=torch.Generator().manual_seed(1)).to(DEV)].contiguous()
    for n in (V // 2 - 50, V // 2, V // 2 + 50, V // 2 + 5000):
        check_distinct(torch.zeros_like(u), u, n, logits=True)
