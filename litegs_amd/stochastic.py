"""Random draws of training: counter-based dropout and noise, sampling with and without replacement (csrc/draws.hip, csrc/sample.hip).

Every random number here is either an argument (the ``u`` of the two samplers) or a function of ``(seed, offset, index)`` alone: word
``i`` of a draw is word ``i % 4`` of the Philox4x32-10 block with counter ``(i // 4, offset)`` under key ``seed``.  Nothing depends on the
launch, the device or the rank, so replicas that call with the same numbers take identical decisions, a dropout mask is drawn again in the
backward pass instead of being stored, and a run can be repeated from any step.  Take a new ``offset`` for every draw (a step number); as
an int64 tensor of one element on the device it is read by the kernel, and a captured graph draws anew on every replay that changes it.

The reference draws with ``torch.multinomial`` (at most 2^24 categories) and ``torch.normal`` (litegs/training/densify.py:296-310); it has
no dropout.  GPU tensors only; everything runs on the current stream.  The calls are no operators of torch's dispatcher: a trace
(``torch.jit.trace``, ``make_fx``, ``torch.export``) or a fake-tensor mode would not see the kernels, and is refused.
"""
from __future__ import annotations

import math
import numbers
from contextlib import nullcontext
from typing import Optional, Tuple, Union

import torch

from ._lib import check, lib
from .binding import load_compiled

_C = load_compiled("_stochastic_C")          # None: the same calls through ctypes (litegs_amd/binding.py)
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
Offset = Union[int, torch.Tensor]


def _s() -> int:
    return torch.cuda.current_stream().cuda_stream


def _on(device: torch.device):
    """launches go to the tensor's device, whichever is current"""
    return nullcontext() if device.index is None or device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _traced() -> bool:
    """the compiled binding's ``traced`` (csrc/ext/stochastic_ext.cpp)"""
    c = torch._C
    if c._get_tracing_state() is not None or c._dispatch_tls_is_dispatch_key_included(c.DispatchKey.PreDispatch):
        return True
    keys = c._TorchDispatchModeKey
    return c._len_torch_dispatch_stack() > 0 and any(c._get_dispatch_mode(k) is not None for k in (keys.PROXY, keys.FAKE, keys.FUNCTIONAL))


def _not_traced(what: str) -> None:
    if _traced() if _C is None else _C.traced():
        raise RuntimeError(f"{what}: cannot be traced (the kernel would not be part of the trace)")


def _float_tensor(t, what: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _DTYPES:
        raise RuntimeError(f"{what}: float32, float16 or bfloat16 GPU tensor required (no CPU path)")


def _integer(v, what: str, name: str, lo: int, hi: int) -> int:
    """v as an int in [lo, hi)"""
    if (type(v) is not int and (isinstance(v, bool) or not isinstance(v, numbers.Integral))) or not lo <= int(v) < hi:
        raise ValueError(f"{what}: {name} must be an integer in [{lo}, {hi}), got {v!r}")
    return int(v)


def _real(v, what: str, name: str, lo: float, hi: float) -> float:
    """v as a float in [lo, hi]"""
    if (type(v) is not float and (isinstance(v, bool) or not isinstance(v, numbers.Real))) or not lo <= float(v) <= hi:
        raise ValueError(f"{what}: {name} must be a number in [{lo}, {hi}], got {v!r}")
    return float(v)


def _key(seed, offset: Offset, device: torch.device, what: str) -> Tuple[int, int, Optional[torch.Tensor]]:
    """-> (seed as the int64 of the same bits, host offset, device offset or None)"""
    seed = _integer(seed, what, "seed", 0, 1 << 64)
    seed -= (seed >> 63) << 64
    if isinstance(offset, torch.Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1 or offset.device != device:
            raise ValueError(f"{what}: an offset tensor must be one int64 on {device}")
        return seed, 0, offset
    return seed, _integer(offset, what, "offset", 0, 1 << 63), None


class _Dropout(torch.autograd.Function):
    """a linear map that is its own transpose: the gradient is the same call on the gradient, to any order"""

    @staticmethod
    def forward(ctx, x, lead, M, p, seed, offset, offset_dev, chunk_ids, S):
        _not_traced("dropout")
        ctx.meta = (lead, M, p, seed, offset, S)
        ctx.save_for_backward(offset_dev, chunk_ids)        # a step counter advanced in between is reported by autograd, not used
        x = x.contiguous()
        y = torch.empty_like(x)
        with _on(x.device):
            check(lib().lg_dropout(x.data_ptr(), y.data_ptr(), _DTYPES[x.dtype], lead, M, p, seed, offset,
                                   None if offset_dev is None else offset_dev.data_ptr(),
                                   None if chunk_ids is None else chunk_ids.data_ptr(), S, _s()), "dropout")
        return y

    @staticmethod
    def backward(ctx, grad):
        lead, M, p, seed, offset, S = ctx.meta
        return (_Dropout.apply(grad, lead, M, p, seed, offset, *ctx.saved_tensors, S),) + (None,) * 8


def dropout(x: torch.Tensor, p: float, seed: int, offset: Offset = 0, shared: int = 0, chunk_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x / (1 - p)`` where the element is kept, 0 where it is dropped (whatever it held); differentiable.

    The element of index ``i`` is kept when ``word(i) >= round(p * 2^32)``.  ``i`` counts the elements of ``x`` in row-major order; with
    ``shared = k`` it counts those of the trailing dimensions behind the first ``k``, which all share one mask (``shared=2`` on ``sh_rest``
    [R,3,chunks,S] drops whole Gaussians).  ``chunk_ids`` int64 [A] for ``x`` [..., A, S]: column ``s`` of slot ``a`` belongs to Gaussian
    ``chunk_ids[a] * S + s``, and that is its index, shared by all leading dimensions -- a Gaussian's decision is the same in every view,
    whatever slot its chunk was compacted to.  ``p = 1`` drops everything."""
    _not_traced("dropout")
    _float_tensor(x, "dropout")
    p = _real(p, "dropout", "p", 0.0, 1.0)
    key = _key(seed, offset, x.device, "dropout")
    shared = _integer(shared, "dropout", "shared", 0, x.dim() + 1)
    S = 1
    if chunk_ids is not None:
        if not isinstance(chunk_ids, torch.Tensor) or x.dim() < 2 or chunk_ids.dtype != torch.int64 or chunk_ids.device != x.device or tuple(chunk_ids.shape) != (x.shape[-2],):
            raise ValueError("dropout: chunk_ids must be int64 [A] on the device of x [..., A, S]")
        if shared not in (0, x.dim() - 2):
            raise ValueError("dropout: chunk_ids share the mask over all leading dimensions")
        if x.shape[-1] >= 1 << 31:
            raise ValueError("dropout: a chunk has at most 2^31 - 1 columns")
        shared, S, chunk_ids = x.dim() - 2, x.shape[-1], chunk_ids.contiguous()
    M = math.prod(x.shape[shared:])
    lead = math.prod(x.shape[:shared])
    return (_Dropout.apply if _C is None else _C.dropout)(x, lead, M, p, *key, chunk_ids, S)


def _draw(std, out, seed, offset, offset_dev, what: str) -> None:
    if _C is not None:
        _C.random_draw(std, out, seed, offset, offset_dev)
        return
    with _on(out.device):
        check(lib().lg_random_draw(None if std is None else std.data_ptr(), out.data_ptr(), _DTYPES[out.dtype], out.numel(), seed, offset,
                                   None if offset_dev is None else offset_dev.data_ptr(), _s()), what)


def uniform(shape, seed: int, offset: Offset = 0, dtype: torch.dtype = torch.float32, device: Optional[torch.device] = None) -> torch.Tensor:
    """``(word(i) + 1/2) / 2^32`` rounded to ``dtype`` and kept below one: in (0, 1) in float32 (in half width the smallest round to 0)"""
    _not_traced("uniform")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.type != "cuda" or dtype not in _DTYPES:
        raise RuntimeError("uniform: float32, float16 or bfloat16 on a GPU (no CPU path)")
    out = torch.empty(shape, dtype=dtype, device=device)
    seed, offset, offset_dev = _key(seed, offset, out.device, "uniform")
    _draw(None, out, seed, offset, offset_dev, "uniform")
    return out


def normal(std: torch.Tensor, seed: int, offset: Offset = 0) -> torch.Tensor:
    """``std * N(0,1)``, element for element (Box-Muller: the words 2j and 2j + 1 give the elements 2j and 2j + 1); not differentiable"""
    _not_traced("normal")
    _float_tensor(std, "normal")
    seed, offset, offset_dev = _key(seed, offset, std.device, "normal")
    std = std.detach().contiguous()
    out = torch.empty_like(std)
    _draw(std, out, seed, offset, offset_dev, "normal")
    return out


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., K] -> [R, K] with a contiguous innermost dimension (a view where the strides allow one)"""
    if t.dim() == 2 and t.stride(1) == 1:
        return t
    t = t.detach().reshape(-1, t.shape[-1]) if t.shape[-1] else t.new_empty((math.prod(t.shape[:-1]), 0))
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def check_rule(what: str, temperature, top_k, top_p, min_p) -> Tuple[float, int, float, float]:
    """the samplers' options as numbers, or ValueError"""
    temperature = _real(temperature, what, "temperature", 1e-30, 1e30)
    top_k = _integer(top_k, what, "top_k", 0, 1 << 62)
    top_p = _real(top_p, what, "top_p", 0.0, 1.0)
    min_p = _real(min_p, what, "min_p", 0.0, 1.0)
    if top_p == 0.0:
        raise ValueError(f"{what}: top_p must be more than 0")
    return temperature, top_k, top_p, min_p


def _sample(what: str, scores, u, n: int, distinct: bool, temperature, top_k, top_p, min_p, logits) -> torch.Tensor:
    V = scores.shape[-1]
    if V >= 1 << 31:
        raise ValueError(f"{what}: at most 2^31 - 1 categories")
    temperature, top_k, top_p, min_p = check_rule(what, temperature, top_k, top_p, min_p)
    R = math.prod(scores.shape[:-1])
    if V > 12288 and (R * ((V + 8191) // 8192) >= 1 << 22 or R * ((n + 255) // 256) >= 1 << 24):
        raise ValueError(f"{what}: {R} rows of {V} categories and {n} draws are too many for one call")
    x, uu = _rows(scores), _rows(u)
    out = torch.empty((*scores.shape[:-1], n), dtype=torch.int64, device=x.device)
    if _C is not None:
        _C.sample(x, uu, out, n, distinct, bool(logits), temperature, top_k, top_p, min_p)
        return out
    L = lib()
    tb = L.lg_sample_temp_bytes(R, V, n, _DTYPES[x.dtype], int(distinct), top_k, top_p)
    temp = torch.empty((max(tb, 1),), dtype=torch.uint8, device=x.device)
    with _on(x.device):
        check(L.lg_sample(x.data_ptr(), _DTYPES[x.dtype], x.stride(0), uu.data_ptr(), uu.stride(0), R, V, n, int(distinct), int(bool(logits)),
                          temperature, top_k, top_p, min_p, out.data_ptr(), temp.data_ptr(), tb, _s()), what)
    return out


def _check_scores(scores, u, what: str) -> None:
    _not_traced(what)
    _float_tensor(scores, what)
    if not isinstance(u, torch.Tensor) or u.dtype != torch.float32 or u.device != scores.device:
        raise RuntimeError(f"{what}: u must be float32 on the device of the scores")
    if scores.dim() < 1 or u.dim() != scores.dim() or u.shape[:-1] != scores.shape[:-1]:
        raise ValueError(f"{what}: scores [..., V] and u [..., K] must have the same leading dimensions")


def sample(scores: torch.Tensor, u: torch.Tensor, *, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0,
           logits: bool = True) -> torch.Tensor:
    """Categories drawn with replacement: ``scores`` [..., V], ``u`` [..., n] float32 in [0, 1) -> int64 [..., n].

    The mass of a category is ``exp(x / temperature)`` (``logits``) or ``x ** (1 / temperature)`` (weights).  NaN, ``-inf`` and weights that
    are not positive are excluded; ``+inf`` counts as the type's largest value.  In this order: ``top_k`` keeps the k best (ties: lowest index first), ``top_p`` the
    shortest prefix of those, best first, that carries ``top_p`` of their mass, ``min_p`` what has at least ``min_p`` of the best mass.
    Draw ``j`` is the first category, in index order, up to which the kept masses add to more than ``u[j]`` of their total (``u`` below
    zero or NaN counts as 0, from one on it draws the last).  A row with nothing to draw from gives -1.  ``top_k=1`` is greedy."""
    _check_scores(scores, u, "sample")
    return _sample("sample", scores, u, u.shape[-1], False, temperature, top_k, top_p, min_p, logits)


def sample_distinct(scores: torch.Tensor, u: torch.Tensor, n: int, *, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                    min_p: float = 0.0, logits: bool = True) -> torch.Tensor:
    """``n`` different categories drawn one after the other without replacement, in ascending order: ``scores`` and ``u`` [..., V] -> int64 [..., n].

    The filters are those of ``sample``.  The winners are the ``n`` largest ``log(mass) - log(-log(1 - u))`` (ties: lowest index first; ``u`` is
    clamped to [2^-33, 1 - 2^-24], NaN to its upper end), which is distributed as drawing from the masses n times, each time without those
    drawn before.  Where fewer than ``n`` categories are left, the row ends in -1."""
    _check_scores(scores, u, "sample_distinct")
    if u.shape != scores.shape:
        raise ValueError("sample_distinct: one u for every score")
    n = _integer(n, "sample_distinct", "n", 0, scores.shape[-1] + 1)
    return _sample("sample_distinct", scores, u, n, True, temperature, top_k, top_p, min_p, logits)
