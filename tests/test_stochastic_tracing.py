"""The random draws under torch's tracers: refused, not recorded as empty tensors.  (The refusal comes before the look at the device, so that
it shows without a GPU.)"""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from litegs_amd import stochastic

CALLS = {"dropout": lambda x: stochastic.dropout(x, 0.5, 1), "uniform": lambda x: stochastic.uniform((3,), 1) + x, "normal": lambda x: stochastic.normal(x, 1),
         "sample": lambda x: stochastic.sample(x[None], x[None]), "sample_distinct": lambda x: stochastic.sample_distinct(x, x, 2)}


class Module(torch.nn.Module):
    def __init__(self, f):
        super().__init__()
        self.f = f

    def forward(self, x):
        return self.f(x)


def fake(f, x):
    with FakeTensorMode() as mode:
        return f(mode.from_tensor(x))


TRACERS = {"jit": lambda f, x: torch.jit.trace(f, x, check_trace=False), "fx": lambda f, x: make_fx(f)(x), "fx fake": lambda f, x: make_fx(f, tracing_mode="fake")(x),
           "fx before dispatch": lambda f, x: make_fx(f, pre_dispatch=True)(x), "fake": fake,
           "export": lambda f, x: torch.export.export(Module(f), (x,), strict=False)}


@pytest.fixture(params=["compiled", "ctypes"])
def binding(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(stochastic, "_C", None)
    elif stochastic._C is None:
        pytest.skip("the compiled binding is not built")


@pytest.mark.parametrize("tracer", TRACERS)
@pytest.mark.parametrize("call", CALLS)
def test_tracing_is_refused(call, tracer, binding):
    with pytest.raises(RuntimeError, match=f"{call}: cannot be traced"):
        TRACERS[tracer](CALLS[call], torch.ones(3))
    with pytest.raises(RuntimeError, match="no CPU path|HIP GPUs|CUDA"):              # (and outside it is the device again)
        if torch.cuda.is_available():
            raise RuntimeError("no CPU path")
        CALLS[call](torch.ones(3))


def test_other_modes_are_not(binding):
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False):
        stochastic._not_traced("draw")
    stochastic._not_traced("draw")


# ---- on the GPU ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("tracer", TRACERS)
@pytest.mark.parametrize("call", CALLS)
def test_tracing_is_refused_with_gpu_tensors(call, tracer, binding):
    x = torch.rand(3, device="cuda")
    want = CALLS[call](x)
    with pytest.raises(RuntimeError, match=f"{call}: cannot be traced"):
        TRACERS[tracer](CALLS[call], x)
    assert torch.equal(CALLS[call](x), want)


@pytest.mark.gpu
def test_tracing_a_backward_pass_is_refused(binding):
    x = torch.rand(64, device="cuda", requires_grad=True)
    y = stochastic.dropout(x, 0.5, 1)
    grad = lambda g: torch.autograd.grad(y, x, g, retain_graph=True)[0]
    want = grad(torch.ones_like(y))
    with pytest.raises(RuntimeError, match="dropout: cannot be traced"):
        make_fx(grad)(torch.ones_like(y))
    assert torch.equal(grad(torch.ones_like(y)), want)


@pytest.mark.gpu
def test_compiled_functions_call_the_kernels():
    """torch.compile leaves the calls out of its graphs and makes them as they stand"""
    def f(x, u):
        y = stochastic.dropout(x * 2, 0.5, 3) + 1
        return y, stochastic.sample(y.detach()[None], u[None]), stochastic.normal(x.detach(), 4), stochastic.uniform((5,), 9)

    x, u = torch.rand(64, device="cuda", requires_grad=True), torch.rand(4, device="cuda")
    g = torch.compile(f, backend="eager")
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(g(x, u), f(x, u)))
    (a,), (b,) = (torch.autograd.grad(h(x, u)[0].sum(), x) for h in (g, f))
    assert torch.equal(a, b) and (a != 0).any()
