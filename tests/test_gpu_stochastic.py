"""Random draws on the GPU against plain 64-bit forms (tests/stochastic_reference.py): indices and masks are equal, values as close as their
roundings allow."""
import itertools
import math

import numpy as np
import pytest
import torch

from litegs_amd import stochastic
from tests import stochastic_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(t):
    return torch.finfo(t).eps / 2


# ---- dropout -------------------------------------------------------------------------------------------------------------------------
def scaled(x, p):
    """x / (1 - p) as one product in 32 bits, rounded once: what the definition's kept elements are, bit for bit"""
    return (x.float() * torch.tensor(1.0 / (1.0 - p), dtype=torch.float32, device=x.device)).to(x.dtype)


def check_dropout(x, p, seed, offset, index, **kw):
    m = torch.from_numpy(np.asarray(ref.kept(index, p, seed, offset))).to(DEV).expand(x.shape)
    y = stochastic.dropout(x, p, seed, offset, **kw)
    assert y.dtype == x.dtype and y.shape == x.shape
    want = torch.where(m, scaled(x, p) if p < 1 else x, torch.zeros((), dtype=x.dtype, device=DEV))
    assert torch.equal(torch.nan_to_num(y.detach(), nan=7.0), torch.nan_to_num(want.detach(), nan=7.0))
    return m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,shared", [((1,), 0), ((3,), 0), ((4,), 0), ((5, 7), 0), ((5, 7), 1), ((2, 3, 129), 2), ((45, 2, 128), 1), ((17, 4, 12), 1),
                                          ((1, 1023), 0), ((9, 1), 1), ((3, 4), 2), ((1000, 8), 1), ((1, 40, 128), 0), ((0, 4), 0), ((4, 0), 1)])
def test_dropout_matches_the_definition(shape, shared, dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(shape, generator=g, device=DEV).to(dtype)
    tail = shape[shared:]
    index = np.arange(math.prod(tail), dtype=np.int64).reshape(tail)
    for p, seed, offset in ((0.3, 5, 0), (0.9, 2 ** 64 - 1, 2 ** 63 - 1), (0.0, 0, 1), (1.0, 3, 2), (1e-9, 1, 2 ** 33)):
        check_dropout(x, p, seed, offset, index, shared=shared)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,A,S", [((), 5, 128), ((1,), 1, 128), ((15, 3), 4, 128), ((2,), 6, 7), ((), 3, 1), ((9,), 5, 12)])
def test_dropout_by_chunk_id(lead, A, S, dtype):
    rng = np.random.default_rng(2)
    ids = np.sort(rng.choice(10 ** 9, A, replace=False))
    ids[-1] = 2 ** 40 + 1                                          # index far behind 32 bits
    x = torch.randn((*lead, A, S), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).to(dtype)
    index = ids[:, None] * S + np.arange(S)
    check_dropout(x, 0.4, 77, 3, index, chunk_ids=torch.from_numpy(ids).to(DEV))


def test_dropout_of_a_chunk_is_the_same_in_every_slot():
    """compacted differently, a Gaussian keeps its decision -- and it is the decision of the whole cloud's mask"""
    x = torch.ones((1, 20, 128), device=DEV)
    whole = stochastic.dropout(x, 0.5, 9, 4)
    for ids in ([3, 4, 19], [0, 3, 7, 19]):
        t = torch.tensor(ids, device=DEV)
        assert torch.equal(stochastic.dropout(x[:, : len(ids)], 0.5, 9, 4, chunk_ids=t), whole[:, t])


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_of_views(dtype):
    """strides and alignment other than a fresh tensor's"""
    base = torch.randn((7, 33, 20), device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)).to(dtype)
    for x in (base.transpose(0, 2), base[:, 1:, 3:], base.reshape(-1)[1:], base.reshape(-1)[2:402], base[::2], base[:1].expand(4, 33, 20)):
        index = np.arange(x.numel(), dtype=np.int64).reshape(x.shape)
        check_dropout(x, 0.5, 11, 5, index)


def test_dropped_elements_are_zero_whatever_they_held():
    x = torch.tensor([math.nan, math.inf, -math.inf, 1.0] * 64, device=DEV)
    m = check_dropout(x, 0.5, 1, 1, np.arange(256))
    y = stochastic.dropout(x, 0.5, 1, 1)
    assert (y[~m] == 0).all() and torch.isnan(y[m & x.isnan()]).all() and (y[m & x.isinf()] == x[m & x.isinf()]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("by_chunk", [False, True])
def test_dropout_gradient(dtype, by_chunk):
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randn((4, 3, 128), generator=g, device=DEV).to(dtype).requires_grad_(True)
    dy = torch.randn((4, 3, 128), generator=g, device=DEV).to(dtype)
    ids = torch.tensor([5, 6, 90], device=DEV)
    kw = dict(chunk_ids=ids) if by_chunk else dict(shared=1)
    index = (ids.cpu().numpy()[:, None] if by_chunk else np.arange(3)[:, None]) * 128 + np.arange(128)
    y = stochastic.dropout(x, 0.35, 8, 21, **kw)
    for grad in (dy, dy.transpose(0, 2).contiguous().transpose(0, 2), dy[:1].expand_as(dy)):
        (dx,) = torch.autograd.grad(y, x, grad, retain_graph=True)
        m = torch.from_numpy(ref.kept(index, 0.35, 8, 21)).to(DEV)
        assert torch.equal(dx, torch.where(m, scaled(grad, 0.35), torch.zeros((), dtype=dtype, device=DEV)))
    # differences: the map is linear; a step of a power of two moves a kept element by step / (1 - p) up to the roundings of its two values
    h = 0.25
    with torch.no_grad():
        up, down = (stochastic.dropout(x + s * h, 0.35, 8, 21, **kw).float() for s in (1, -1))
        step = ((x + h).float() - (x - h).float())
        (unit,) = torch.autograd.grad(y, x, torch.ones_like(y))
        got, want = up - down, unit.float() * step
        bound = half_step(dtype) * (up.abs() + down.abs() + 2 * want.abs()) + 2.0 ** -22 * (up.abs() + down.abs())
        assert ((got - want).abs() <= bound + 1e-30).all()


def test_dropout_second_derivatives():
    x = torch.randn(64, device=DEV, requires_grad=True)
    g = torch.randn(64, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad(stochastic.dropout(x * x, 0.5, 1), x, g, create_graph=True)          # 2 x g m / (1 - p)
    m2 = 2.0 * torch.from_numpy(ref.kept(np.arange(64), 0.5, 1, 0)).to(DEV)
    dxx, dxg = torch.autograd.grad(dx.sum(), (x, g))
    assert torch.equal(dxx, 2 * g * m2) and torch.equal(dxg, 2 * x * m2)


def test_dropout_in_autograd():
    x = torch.randn((3, 40), device=DEV, requires_grad=True)
    with torch.no_grad():
        assert not stochastic.dropout(x, 0.4, 3).requires_grad
    with torch.inference_mode():
        assert stochastic.dropout(x, 0.4, 3).is_inference()
    assert not stochastic.dropout(x.detach(), 0.4, 3).requires_grad
    step = torch.tensor([7], device=DEV)
    y = stochastic.dropout(x * 2, 0.4, 3, step)
    (a,) = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    (b,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(a, b) and torch.equal(a != 0, y != 0) and torch.equal(y.detach(), x.detach() * a)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x, torch.ones_like(y))
    z = stochastic.dropout(x, 0.4, 3)                                # an output that the loss does not use, a gradient with strides of zero
    (c,) = torch.autograd.grad(z.sum(), x)
    assert torch.equal(c != 0, z != 0)
    (d,) = torch.autograd.grad((stochastic.dropout(x, 0.4, 3) * 0 + x).sum(), x)
    assert torch.equal(d, torch.ones_like(d))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
        stochastic.dropout(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)), 0.4, 3)


def test_offset_tensor_and_its_guard():
    x = torch.randn((1, 7, 128), device=DEV, requires_grad=True)
    step = torch.tensor([41], device=DEV)
    y = stochastic.dropout(x, 0.5, 13, step)
    assert torch.equal(y, stochastic.dropout(x, 0.5, 13, 41))
    step += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()                                          # the mask of step 41 is gone: reported, not replaced by step 42's
    assert torch.equal(stochastic.uniform((9,), 13, step), stochastic.uniform((9,), 13, 42))
    assert torch.equal(stochastic.normal(x.detach(), 13, step), stochastic.normal(x.detach(), 13, 42))


def test_dropout_refusals():
    x = torch.zeros((2, 4, 8), device=DEV)
    ids = torch.zeros(4, dtype=torch.int64, device=DEV)
    for kw in (dict(p=-0.1), dict(p=1.01), dict(p=math.nan), dict(p="a"), dict(seed=-1), dict(offset=-1), dict(shared=4), dict(shared=-1), dict(chunk_ids=ids[:3]),
               dict(chunk_ids=ids.int()), dict(chunk_ids=ids.cpu()), dict(chunk_ids=ids, shared=2), dict(offset=ids), dict(offset=ids[:1].cpu())):
        a = dict(p=0.5, seed=1)
        a.update(kw)
        with pytest.raises(ValueError):
            stochastic.dropout(x, **a)
    with pytest.raises(ValueError, match="columns"):
        stochastic.dropout(x[:1, 0, :1].expand(1, 2 ** 32 + 8), 0.5, 1, chunk_ids=ids[:1])
    with pytest.raises(RuntimeError):
        stochastic.dropout(x.double(), 0.5, 1)
    with pytest.raises(RuntimeError):
        stochastic.dropout(x.cpu(), 0.5, 1)


# ---- uniform, normal -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [0, 1, 2, 3, 4, 5, 1000, 4097, 300001])
def test_uniform_matches_the_definition(n, dtype):
    for seed, offset in ((0, 0), (2 ** 63 + 5, 2 ** 62 + 1)):
        u = stochastic.uniform((n,), seed, offset, dtype=dtype)
        w = ref.words(np.arange(n), seed, offset).astype(np.float64)
        want = torch.from_numpy(((w + 0.5) / 2.0 ** 32).astype(np.float32)).to(dtype).clamp(max=1.0 - half_step(dtype))
        assert torch.equal(u.cpu(), want)
        assert (u < 1).all()


def test_uniform_behind_32_bits():
    n = 2 ** 32 + 11
    u = stochastic.uniform((n,), 3, 4, dtype=torch.float16)
    w = ref.words(np.arange(n - 32, n), 3, 4).astype(np.float64)
    assert torch.equal(u[-32:].cpu(), torch.from_numpy(((w + 0.5) / 2.0 ** 32).astype(np.float32)).half().clamp(max=1 - 2.0 ** -11))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 6, 7, 1001, 400003])
def test_normal_matches_the_definition(n, dtype):
    """r = sqrt(-2 ln a) in 32 bits: the argument's rounding (2^-24) against |ln a| >= ln 2 and a logarithm good to two steps give 4 steps of
    -ln a, the root halves them and adds one: 3 * 2^-24 r.  cos / sin: the angle (<= pi/4) is rounded twice and its polynomial evaluated in
    32 bits: 4 * 2^-24 absolute.  Product and std: 2 steps of the value.  Then one rounding to the type."""
    std = torch.rand(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(7)).add(0.5).to(dtype)
    got = stochastic.normal(std, 99, 2 ** 35).double().cpu().numpy()
    z, r = ref.normals(n, 99, 2 ** 35)
    s = std.double().cpu().numpy()
    f = 2.0 ** -24
    bound = s * f * (4 * r + 8 * np.abs(z))
    if dtype != torch.float32:
        bound = bound + half_step(dtype) * (np.abs(s * z) + bound) + 2.0 ** -25 * (dtype == torch.float16)
    assert (np.abs(got - s * z) <= bound).all()


def test_normal_is_normal():
    n = 1 << 20
    z = stochastic.normal(torch.ones(n, device=DEV), 5).double()
    assert abs(z.mean().item()) < 5 / math.sqrt(n) and abs(z.square().mean().item() - 1) < 5 * math.sqrt(2 / n)
    assert abs((z[0::2] * z[1::2]).mean().item()) < 5 / math.sqrt(n / 2)


def test_normal_special_values():
    std = torch.tensor([0.0, math.inf, math.nan, 1.0], device=DEV)
    z = stochastic.normal(std, 1)
    assert z[0] == 0 and z[1].isinf() and z[2].isnan() and z[3].isfinite()


# ---- sampling ------------------------------------------------------------------------------------------------------------------------
RULES = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=13), dict(top_p=0.8), dict(min_p=0.05), dict(temperature=1.7, top_k=40, top_p=0.9, min_p=0.01),
         dict(temperature=0.05, top_p=0.999)]


def rule(kw, logits):
    a = dict(logits=logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    a.update(kw)
    return a


def scores_of(kind, R, V, dtype, logits, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = torch.randn((R, V), generator=g, device=DEV) * 3
    hole = torch.rand((R, V), generator=g, device=DEV)
    if kind == "ties":
        z = torch.randint(-2, 3, (R, V), generator=g, device=DEV).float()
    elif kind == "equal":
        z = torch.full((R, V), 0.75, device=DEV)
    elif kind == "wide":
        z = z * 20
    elif kind == "steps":                                           # powers of two over the whole range of float32, either sign
        z = torch.where(hole < 0.5, -1.0, 1.0) * torch.exp2(torch.randint(-140, 120, (R, V), generator=g, device=DEV).float())
    elif kind == "near":                                            # floats next to each other, around one and around zero
        z = torch.where(hole < 0.5, 1.0 + (z * 3).round() * 2.0 ** -23, (z * 3).round() * 2.0 ** -149)
    if not logits:
        z = z.abs() if kind in ("steps", "near") else z.clamp(-40, 40).exp()
    z = z.to(dtype)
    if kind == "masked":
        z = torch.where(hole < 0.5, torch.tensor(-math.inf if logits else 0.0, dtype=dtype, device=DEV), z)
    elif kind == "lowest":                                          # masks of the type's lowest value; a weight below zero is no weight
        z = torch.where(hole < 0.5, torch.tensor(torch.finfo(dtype).min, dtype=dtype, device=DEV), z)
    elif kind == "nan":
        z = torch.where(hole < 0.3, torch.tensor(math.nan, dtype=dtype, device=DEV), z)
        z = torch.where(hole > 0.9, torch.tensor(-math.inf, dtype=dtype, device=DEV), z)
    elif kind == "inf":
        z = torch.where(hole < 0.01, torch.tensor(math.inf, dtype=dtype, device=DEV), z)
    elif kind == "zeros":
        z = torch.where(hole < 0.5, torch.tensor(-0.0, dtype=dtype, device=DEV), torch.zeros_like(z))
    elif kind == "empty":
        z = z.clone()
        z[R // 2] = -math.inf if logits else -1.0
    elif kind == "tiny":
        z = (z.float() * 1e-42).to(dtype)
    return z


def draws_of(shape, seed=1):
    return torch.rand(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def check_sample(x, u, **kw):
    a = rule({k: v for k, v in kw.items() if k != "logits"}, kw["logits"])
    got = stochastic.sample(x, u, **a)
    big = torch.finfo(x.dtype).max
    want = np.stack([ref.sample_row(r, v, big=big, **a) for r, v in zip(x.double().cpu().numpy(), u.cpu().numpy())])
    assert got.dtype == torch.int64 and np.array_equal(got.cpu().numpy(), want), (x.shape, x.dtype, kw)


def check_distinct(x, u, n, **kw):
    a = rule({k: v for k, v in kw.items() if k != "logits"}, kw["logits"])
    got = stochastic.sample_distinct(x, u, n, **a)
    big = torch.finfo(x.dtype).max
    want = np.stack([ref.distinct_row(r, v, n, big=big, **a) for r, v in zip(x.double().cpu().numpy(), u.cpu().numpy())])
    assert got.dtype == torch.int64 and np.array_equal(got.cpu().numpy(), want), (x.shape, x.dtype, n, kw)


LENGTHS = [1, 2, 63, 64, 65, 1000, 1024, 1025, 4095, 4096, 4097, 9000, 12288, 12289, 20001]


@pytest.mark.parametrize("V", LENGTHS)
@pytest.mark.parametrize("logits", [True, False])
def test_sample_lengths(V, logits):
    for dtype, kw in zip(itertools.cycle(TYPES), RULES):
        x = scores_of("normal", 3, V, dtype, logits, seed=V)
        check_sample(x, draws_of((3, 9), V), logits=logits, **kw)


@pytest.mark.parametrize("V", LENGTHS)
@pytest.mark.parametrize("logits", [True, False])
def test_distinct_lengths(V, logits):
    for dtype, kw in zip(itertools.cycle(TYPES), RULES):
        x = scores_of("normal", 2, V, dtype, logits, seed=V)
        for n in sorted({1, (V + 2) // 3, V}):
            check_distinct(x, draws_of((2, V), V), n, logits=logits, **kw)


KINDS = ["ties", "equal", "wide", "steps", "near", "masked", "lowest", "nan", "inf", "zeros", "empty", "tiny"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("logits", [True, False])
@pytest.mark.parametrize("V", [300, 70001])
def test_sampling_of_special_scores(kind, logits, V):
    for dtype in TYPES:
        x = scores_of(kind, 2, V, dtype, logits, seed=3)
        for kw in RULES if V < 1000 else RULES[:1] + RULES[5:7]:
            check_sample(x, draws_of((2, 50)), logits=logits, **kw)
            check_distinct(x, draws_of((2, V)), V // 4, logits=logits, **kw)


@pytest.mark.parametrize("kind", ["normal", "ties", "masked", "nan", "wide", "inf", "near", "empty", "tiny"])
@pytest.mark.parametrize("V", [64, 65, 130, 1025, 5000, 12288])
@pytest.mark.parametrize("logits", [True, False])
def test_top_k_around_a_wave(kind, V, logits):
    """top-k of up to 64 is finished by one wave, unless equal scores at the border are too many for it"""
    for k, dtype in zip((1, 2, 50, 63, 64, 65), itertools.cycle(TYPES)):
        x = scores_of(kind, 3, V, dtype, logits, seed=k)
        if kind == "masked":
            x[1, : V - 20] = -math.inf if logits else 0.0             # fewer left than k
        for kw in (dict(), dict(top_p=0.7), dict(min_p=0.2), dict(temperature=0.6, top_p=0.9, min_p=0.05)):
            check_sample(x, draws_of((3, 40), k), logits=logits, top_k=k, **kw)
            for n in (1, 20, 64):
                check_distinct(x, draws_of((3, V), k), n, logits=logits, top_k=k, **kw)
    check_sample(x[:1], draws_of((1, 5000)), logits=logits, top_k=40, top_p=0.9)      # draws shared by workgroups


@pytest.mark.parametrize("T", [1e-30, 1e-20, 1e-14, 1e-8, 1e-3, 0.7, 1.7, 1e20, 1e30])
@pytest.mark.parametrize("V", [300, 9000, 70001])
@pytest.mark.parametrize("logits", [True, False])
def test_far_temperatures(T, V, logits):
    """equal scores have equal masses however far T magnifies what a logarithm rounds; scores that differ have 2^-24 between them at least"""
    for kind, dtype in itertools.product(("ties", "normal"), TYPES):
        x = scores_of(kind, 2, V, dtype, logits, seed=8)
        for kw in (dict(), dict(top_p=0.8), dict(min_p=0.5), dict(min_p=1e-3), dict(top_k=20, top_p=0.9)):
            check_sample(x, draws_of((2, 20)), logits=logits, temperature=T, **kw)


@pytest.mark.parametrize("V", [5, 5000, 90000])
def test_sampling_with_special_numbers(V):
    x = scores_of("ties", 2, V, torch.float32, True)
    odd = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan, 1e-45, 0.5], device=DEV)
    check_sample(x, odd.expand(2, 8), logits=True)
    check_sample(scores_of("masked", 2, V, torch.float32, False), odd.expand(2, 8), logits=False)
    u = draws_of((2, V))
    for k, v in enumerate(odd):
        u[:, k % V :: 11] = v
    check_distinct(x, u, V // 2, logits=True)
    check_distinct(x, torch.full_like(u, 0.25), V // 2, logits=True)            # nothing but ties: lowest indices of the best scores
    check_distinct(torch.zeros_like(x), torch.full_like(u, 0.25), V // 3 + 1, logits=True)


def test_sample_borders_are_exact():
    """integer weights: u * total falls on a border exactly, and the draw is the category behind it"""
    w = torch.tensor([[0.0, 1, 0, 2, 1, 0, 4, 0]], device=DEV)
    u = torch.arange(8, device=DEV).float().div(8)[None]
    assert stochastic.sample(w, u, logits=False).tolist() == [[1, 3, 3, 4, 6, 6, 6, 6]]


def test_top_p_and_top_k_cut_ties_at_the_lowest_index():
    x = torch.zeros((1, 1000), device=DEV)
    assert stochastic.sample_distinct(x, draws_of((1, 1000)), 1000, top_k=7)[0, :8].tolist() == [0, 1, 2, 3, 4, 5, 6, -1]
    assert stochastic.sample_distinct(x, draws_of((1, 1000)), 1000, top_p=0.5)[0, 499:501].tolist() == [499, -1]
    assert stochastic.sample_distinct(x, draws_of((1, 1000)), 1000, min_p=1.0)[0, 999].item() == 999


@pytest.mark.parametrize("R", [1, 5, 300])
def test_rows_with_strides(R):
    base = scores_of("normal", R, 2100, torch.bfloat16, True)
    u = draws_of((R, 2100))
    check_sample(base[:, 7:2003], u[:, 1:4], logits=True, top_p=0.9)
    check_distinct(base[:, 7:2003], u[:, 3:1999], 20, logits=True, top_k=100)
    check_sample(base.t()[:R].t() if R <= 2100 else base, u[:, :2], logits=True)
    one = stochastic.sample(base[0], u[0, :3])
    assert torch.equal(one, stochastic.sample(base[:1], u[:1, :3])[0])
    three = stochastic.sample_distinct(base.reshape(R, 3, 700), u.reshape(R, 3, 700), 5)
    assert torch.equal(three.reshape(-1, 5), stochastic.sample_distinct(base.reshape(-1, 700), u.reshape(-1, 700), 5))


@pytest.mark.parametrize("R,V", [(2, 700), (2, 11000), (1, 50000), (3, 50000), (260, 13000), (300, 20000)])
def test_many_rows_and_many_draws(R, V):
    """several workgroups a row and one, shares of the draws, 16-bit scores in more rows than their histogram of all keys is made for"""
    for dtype in (torch.float32, torch.bfloat16):
        x = scores_of("normal", R, V, dtype, True, seed=R)
        n = 9000 if R < 10 else 5
        check_sample(x, draws_of((R, n)), logits=True, top_k=V // 3, top_p=0.9)
        check_sample(x, draws_of((R, n)), logits=True, top_k=300, min_p=1e-4)
        check_distinct(x, draws_of((R, V)), 50, logits=True, top_k=V // 3, top_p=0.9, min_p=1e-3)


@pytest.mark.parametrize("equal", [2500, 5000])
def test_distinct_with_many_candidates_next_to_the_border(equal):
    """more elements of one race key than a workgroup ranks pairwise, then more than the list holds; the rest on either side of it"""
    V = 60000
    x = torch.zeros((2, V), device=DEV)
    u = draws_of((2, V)) * 0.2 + 0.4
    u[:, 7::23] = 0.1                                               # (a small u wins)
    some = torch.randperm(V, generator=torch.Generator().manual_seed(1))[:equal].to(DEV)
    u[:, some] = 0.25
    ahead = int((u[0] < 0.25).sum())
    for n in (ahead, ahead + 1, ahead + equal // 2, ahead + equal, ahead + equal + 1):
        check_distinct(x, u, n, logits=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("logits,small", [(True, -21.0), (True, -14.0), (False, 2.0 ** -31 * 1.5), (False, 2.0 ** -20)])
@pytest.mark.parametrize("V", [12000, 2000001])
def test_top_p_ends_inside_a_long_tail(V, logits, small, dtype):
    """one large mass and a tail of equal small ones, cut in its middle: (1 + j m) < top_p (1 + (V - 1) m) holds up to j = V / 2, half a
    mass away from the border, so that top_p's own rounding (2^-53 of about one: at most 2^-53 / m = 2e-7 of an element here) cannot matter"""
    if not logits and dtype == torch.float16:
        small = max(small, 2.0 ** -20)
    m = math.exp(small) if logits else small
    x = torch.full((1, V), small, device=DEV).to(dtype)
    x[0, V // 3] = 0.0 if logits else 1.0
    assert float(x[0, 0]) == small
    j = V // 2
    top_p = (1.0 + (j - 0.5) * m) / (1.0 + (V - 1) * m)
    last = stochastic.sample(x, torch.ones((1, 1), device=DEV), top_p=top_p, logits=logits)
    assert int(last) == j                                            # the large one at V / 3, and the first j of the others: 0 ... j


def test_rows_of_two_gigabytes_and_more():
    V = 2 ** 31 - 1
    x = torch.full((1, V), -math.inf, dtype=torch.bfloat16, device=DEV)
    x[0, 5], x[0, 2 ** 30], x[0, V - 1] = 1.0, 0.5, 1.0
    u = torch.tensor([[0.0, 0.3, 0.5, 0.99]], device=DEV)             # masses e, sqrt(e), e: borders at 0.38 and 0.62
    for dtype in (torch.bfloat16, torch.float32):
        x = x.to(dtype)
        for kw, want in ((dict(), [5, 5, 2 ** 30, V - 1]), (dict(top_k=2), [5, 5, V - 1, V - 1]), (dict(top_p=0.9), [5, 5, 2 ** 30, V - 1]), (dict(top_p=0.5), [5, 5, V - 1, V - 1]),
                         (dict(top_k=20000, min_p=0.9), [5, 5, V - 1, V - 1])):
            got = stochastic.sample(x, u, **kw).tolist()[0]
            assert got == want, (dtype, kw, got)
    del x
    torch.cuda.empty_cache()
    w = torch.zeros((1, V), dtype=torch.bfloat16, device=DEV)
    w[0, 3], w[0, 2 ** 30 + 1], w[0, V - 2] = 1.0, 0.5, 2.0
    uu = torch.full((1, V), 0.5, device=DEV)
    assert stochastic.sample_distinct(w, uu, 2, logits=False).tolist() == [[3, V - 2]]
    assert stochastic.sample_distinct(w, uu, 4, logits=False).tolist() == [[3, 2 ** 30 + 1, V - 2, -1]]


def test_more_rows_than_a_launch_has_threads_for():
    few, R = 1000, 2 ** 24 + 5                                       # (256 threads a row: more than 2^32)
    x, u = scores_of("normal", few, 3, torch.float32, True), draws_of((few, 3))
    rows = torch.arange(R, device=DEV) % few
    for got, want in ((stochastic.sample(x[rows], u[rows][:, :1]), stochastic.sample(x, u[:, :1])), (stochastic.sample_distinct(x[rows], u[rows], 2), stochastic.sample_distinct(x, u, 2))):
        assert torch.equal(got, want[rows])


def test_dropout_behind_32_bits():
    lead, M = 9, 2 ** 29 + 4
    x = torch.ones((lead, M), dtype=torch.bfloat16, device=DEV)
    y = stochastic.dropout(x, 0.5, 11, 3, shared=1)
    for at in (0, M - 1000):
        keep = torch.from_numpy(ref.kept(np.arange(at, at + 1000), 0.5, 11, 3)).to(DEV)
        assert ((y[:, at:at + 1000] != 0) == keep).all()
    del y
    y = stochastic.dropout(x, 0.5, 11, 3)                            # an index of its own for each
    keep = torch.from_numpy(ref.kept(np.arange(lead * M - 1000, lead * M), 0.5, 11, 3)).to(DEV)
    assert ((y[-1, -1000:] != 0) == keep).all()


def test_sample_of_more_tiles_than_a_workgroup_keeps():
    V = 9000001
    x = scores_of("masked", 1, V, torch.float32, False, seed=4)
    u = draws_of((1, 3000))
    u[0, 0], u[0, 1] = 0.0, 1.0
    check_sample(x, u, logits=False)
    check_sample(x, u, logits=False, temperature=0.7, top_p=0.8)


def test_distinct_of_more_tiles_than_are_counted_in_lds():
    V, n = 34000000, 100000
    g = torch.Generator(device=DEV).manual_seed(8)
    x, u = torch.rand((1, V), generator=g, device=DEV), torch.rand((1, V), generator=g, device=DEV)
    got = stochastic.sample_distinct(x, u, n, logits=False)[0].cpu().numpy()
    key = torch.log(x.double()) - torch.log(-torch.log1p(-u.double().clamp(2.0 ** -33, 1 - 2.0 ** -24)))
    want = key[0].topk(n).indices.sort().values.cpu().numpy()       # (keys differ: 2^-24 steps of either number meet in few places, far from the border)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("distinct", [False, True])
@pytest.mark.parametrize("R,V,n", [(1, 5, 3), (3, 4096, 17), (2, 12289, 333), (1, 100003, 1000), (300, 13001, 4)])
def test_nothing_is_written_outside(distinct, R, V, n):
    """the C entry with its output and its workspace inside larger buffers: what lies around them stays as it was"""
    from litegs_amd._lib import lib
    L = lib()
    for code, dtype in enumerate(TYPES):
        for top_k, top_p in ((0, 1.0), (9, 0.9), (V // 2, 0.9)):
            x, u = scores_of("normal", R, V, dtype, True), draws_of((R, V if distinct else n))
            need = L.lg_sample_temp_bytes(R, V, n, code, int(distinct), top_k, top_p)
            out = torch.full((R * n + 512,), -77, dtype=torch.int64, device=DEV)
            temp = torch.full((need + 8192,), 0xC1, dtype=torch.uint8, device=DEV)
            rc = L.lg_sample(x.data_ptr(), code, V, u.data_ptr(), u.shape[1], R, V, n, int(distinct), 1, 1.0, top_k, top_p, 0.0, out.data_ptr() + 256 * 8,
                             temp.data_ptr() + 4096, need, torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            assert (out[:256] == -77).all() and (out[256 + R * n:] == -77).all() and (out[256:256 + R * n] >= -1).all()
            assert (temp[:4096] == 0xC1).all() and (temp[4096 + need:] == 0xC1).all()
            if need:                                                # a workspace that is too small or missing is refused
                assert L.lg_sample(x.data_ptr(), code, V, u.data_ptr(), u.shape[1], R, V, n, int(distinct), 1, 1.0, top_k, top_p, 0.0, out.data_ptr(),
                                   temp.data_ptr(), need - 1, None) != 0
                assert L.lg_sample(x.data_ptr(), code, V, u.data_ptr(), u.shape[1], R, V, n, int(distinct), 1, 1.0, top_k, top_p, 0.0, out.data_ptr(),
                                   None, 0, None) != 0


def test_two_streams_at_once():
    x, u = scores_of("normal", 4, 60000, torch.float32, True), draws_of((4, 60000))
    want = [stochastic.sample_distinct(x, u, 100, top_p=0.9), stochastic.sample(x, u[:, :500], top_k=20000)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([stochastic.sample_distinct(x, u, 100, top_p=0.9), stochastic.sample(x, u[:, :500], top_k=20000)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))


def test_empty_calls():
    z = torch.zeros((2, 0), device=DEV)
    assert stochastic.sample(z, draws_of((2, 3))).tolist() == [[-1] * 3] * 2
    assert stochastic.sample(torch.zeros((2, 5), device=DEV), z).shape == (2, 0)
    assert stochastic.sample_distinct(torch.zeros((2, 5), device=DEV), draws_of((2, 5)), 0).shape == (2, 0)
    assert stochastic.sample_distinct(z, z, 0).shape == (2, 0)
    assert stochastic.sample(torch.zeros((0, 5), device=DEV), draws_of((0, 3))).shape == (0, 3)


def test_too_many_rows_or_draws_are_refused():
    x, u = torch.zeros((1, 1), device=DEV), torch.zeros((1, 1), device=DEV)
    with pytest.raises(ValueError, match="too many"):
        stochastic.sample(x.expand(2 ** 21, 13000), u.expand(2 ** 21, 1))
    with pytest.raises(ValueError, match="too many"):
        stochastic.sample(x.expand(2 ** 12, 13000), u.expand(2 ** 12, 2 ** 20))


def test_sampling_refusals():
    x, u = torch.zeros((2, 8), device=DEV), draws_of((2, 8))
    for kw in (dict(temperature=0.0), dict(temperature=-1), dict(temperature=math.inf), dict(temperature=math.nan), dict(top_k=-1), dict(top_k=2.0), dict(top_p=0.0),
               dict(top_p=1.1), dict(min_p=-0.1), dict(min_p=1.1)):
        with pytest.raises(ValueError):
            stochastic.sample(x, u, **kw)
        with pytest.raises(ValueError):
            stochastic.sample_distinct(x, u, 2, **kw)
    for n in (-1, 9, 1.0, None):
        with pytest.raises(ValueError):
            stochastic.sample_distinct(x, u, n)
    for a, b in ((x, u[:1]), (x, u[0]), (x[0, 0], u[0, 0])):
        with pytest.raises(ValueError):
            stochastic.sample(a, b)
    with pytest.raises(ValueError):
        stochastic.sample_distinct(x, u[:, :7], 2)
    for a, b in ((x.double(), u), (x, u.double()), (x.cpu(), u.cpu()), (x, u.cpu()), (x.long(), u)):
        with pytest.raises(RuntimeError):
            stochastic.sample(a, b)


# ---- the two bindings ----------------------------------------------------------------------------------------------------------------
def test_compiled_and_ctypes_bindings_agree(monkeypatch):
    assert stochastic._C is not None, "the compiled binding is built by litegs_amd.build"
    x = torch.randn((3, 5, 128), device=DEV, requires_grad=True)
    dy, ids, step = torch.randn_like(x), torch.tensor([9, 4, 2, 8, 70], device=DEV), torch.tensor([6], device=DEV)
    z, u = scores_of("normal", 2, 40000, torch.float16, True), draws_of((2, 40000))

    def everything():
        out = []
        for kw in (dict(), dict(shared=1), dict(chunk_ids=ids), dict(offset=step)):
            y = stochastic.dropout(x, 0.4, 2 ** 64 - 1, **kw)
            out += [y, torch.autograd.grad(y, x, dy)[0]]
        out += [stochastic.uniform((7, 3), 5, 6), stochastic.normal(x, 5, step), stochastic.normal(x.detach(), 5, 6)]
        out += [stochastic.sample(z, u[:, :9], top_p=0.9), stochastic.sample_distinct(z, u, 77, top_k=500), stochastic.sample(z[:, :50], u[:, :3])]
        return out

    compiled = everything()
    monkeypatch.setattr(stochastic, "_C", None)
    for a, b in zip(compiled, everything()):
        assert torch.equal(a, b) and a.requires_grad == b.requires_grad
