"""Row softmax; same surface as the reference's ``kernels/softmax/__init__.py:15-35``.

``sample_tokens`` (additive) draws a token from each row's softmax after temperature, top-k, top-p and
min-p, with the random numbers given.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _native as N


def online_softmax(
    x: torch.Tensor,
    *,
    is_causal: bool = False,
    log: bool = False,
    backend: Optional[str] = None,
) -> torch.Tensor:
    """Softmax (or log-softmax) along the last dim of ``x``, any leading shape.

    ``is_causal`` treats the last two dims as a square score matrix and masks
    ``col > row``; non-square input raises ``ValueError`` as in the reference
    (``kernels/softmax/triton_softmax.py:146-164,190-195``).
    """
    N.check_backend(backend)
    if is_causal:
        if x.dim() < 2 or x.shape[-2] != x.shape[-1]:
            raise ValueError(
                "causal mode requires square input (last two dims equal); "
                f"got {tuple(x.shape)}."
            )
    dev = N.require_cuda("online_softmax", x)
    n = x.shape[-1]
    x2 = x.reshape(-1, n).contiguous()
    y = torch.empty_like(x2)
    a = N.SoftmaxArgs(x=N.ptr(x2), y=N.ptr(y), rows=x2.shape[0], n=n, is_causal=int(is_causal), log=int(log),
                      dtype=N.dtype_code(x2), stream=N.stream_handle(dev))
    N.call("rfx_online_softmax", a, dev)
    return y.reshape(x.shape)


_INF = float("inf")
_MOST = torch.finfo(torch.float32).max
_sample = N.Entry("rfx_sample_tokens", N.SampleArgs)


def _setting(name, what, value, B, dtype, low, high):
    """``(tensor or None, number)`` of a sampling setting; only numbers are checked against their range."""
    if isinstance(value, torch.Tensor):
        if value.shape != (B,):
            raise ValueError(f"{name}: {what} must be a number or [{B}], got {tuple(value.shape)}")
        if value.dtype != dtype:
            if dtype == torch.int32 and value.dtype == torch.int64:
                value = value.clamp(-1, 2**31 - 1)
            value = value.to(dtype)
        return value.contiguous(), 0
    if not low <= value <= high:
        raise ValueError(f"{name}: {what} must be between {low} and {high}, got {value}")
    return None, value


def sample_tokens(
    logits: torch.Tensor,
    uniform: torch.Tensor,
    *,
    temperature: Union[float, torch.Tensor] = 1.0,
    top_k: Union[int, torch.Tensor] = 0,
    top_p: Union[float, torch.Tensor] = 1.0,
    min_p: Union[float, torch.Tensor] = 0.0,
    out: Optional[torch.Tensor] = None,
    backend: Optional[str] = None,
) -> torch.Tensor:
    """One token per row of ``logits`` ``[B, vocab]`` from the numbers ``uniform`` ``[B]`` in [0, 1); returns
    int64 ``[B]`` (``out`` if given).

    Every setting is a number or a tensor ``[B]``. In this order: ``top_k`` keeps the k largest logits (0:
    all); of their softmax at ``temperature`` ``top_p`` keeps the likeliest tokens while the mass before
    them is below ``top_p``; ``min_p`` keeps those at least ``min_p`` times as likely as the likeliest. Equal
    logits rank by index, the likeliest token always stays. The token is the lowest index at which the
    running sum of the kept probabilities, in index order, exceeds ``uniform`` times their sum. Temperature 0
    takes the largest logit. NaN counts as -inf; a row without a finite logit (or +inf) gives -1. Logits
    may be strided by row; float64 settings and ``uniform`` are rounded to float32. The result depends on
    the arguments alone, not on the batch, the launch or the order of threads; a running sum is off by less than 2**-26 of the
    total (2**-29 up to 131072 tokens or a ``top_k`` that small). ``vocab`` is at most 2**24.
    """
    N.check_backend(backend)
    name = "sample_tokens"
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"{name}: logits must be [B, vocab], got {tuple(logits.shape)}")
    B, vocab = logits.shape
    if uniform.shape != (B,):
        raise ValueError(f"{name}: uniform must be [{B}], got {tuple(uniform.shape)}")
    temperature, temperature_all = _setting(name, "temperature", temperature, B, torch.float32, 0.0, _INF)
    top_k, top_k_all = _setting(name, "top_k", top_k, B, torch.int32, 0, _INF)
    top_p, top_p_all = _setting(name, "top_p", top_p, B, torch.float32, 0.0, 1.0)
    min_p, min_p_all = _setting(name, "min_p", min_p, B, torch.float32, 0.0, 1.0)
    index = N.same_device(name, logits, uniform, temperature, top_k, top_p, min_p, out)
    if vocab > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    if uniform.dtype != torch.float32:
        uniform = uniform.to(torch.float32)
    uniform = uniform.contiguous()
    if out is None:
        out = logits.new_empty(B, dtype=torch.int64)
    elif out.shape != (B,) or out.dtype != torch.int64 or not out.is_contiguous():
        raise ValueError(f"{name}: out must be contiguous int64 [{B}]")
    _sample(index, logits.data_ptr(), uniform.data_ptr(), 0 if temperature is None else temperature.data_ptr(),
            0 if top_k is None else top_k.data_ptr(), 0 if top_p is None else top_p.data_ptr(),
            0 if min_p is None else min_p.data_ptr(), out.data_ptr(), B, vocab, logits.stride(0),
            _INF if temperature_all > _MOST else temperature_all, int(min(top_k_all, vocab)), top_p_all, min_p_all, N.dtype_code(logits),
            N.stream_of(index))
    return out


# The reference's surface; sample_tokens is an addition, imported by name.
__all__ = ["online_softmax"]
