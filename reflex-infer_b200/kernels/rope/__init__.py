"""RoPE; same surface as the reference's ``kernels/rope/__init__.py``.

``apply_rope`` returns a new tensor, ``apply_rope_`` rotates in place, and
``build_rope_tables`` builds the cos/sin tables on the device. Rounding follows the
reference's torch path: each multiply / add is rounded to the activation dtype
(``kernels/rope/triton_rope.py:230-240``), so 16-bit outputs match it bit for bit when
the tables carry the activation dtype (the way every reference test builds them,
``tests/test_rope.py:25-27``).

``qk_norm_rope`` / ``qk_norm_rope_`` (additive) norm every query and key head before they rotate it,
in one pass and in fp32 with a single rounding.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native as N


def _resolve_layout(x: torch.Tensor, layout: str):
    if x.dim() != 4:
        raise ValueError(f"x must be 4-D, got {tuple(x.shape)}")
    if layout == "bshd":
        B, S, H, D = x.shape
        sb, ss, sh, sd = x.stride()
    elif layout == "bhsd":
        B, H, S, D = x.shape
        sb, sh, ss, sd = x.stride()
    else:
        raise ValueError(f"unknown layout {layout!r}; want 'bshd' or 'bhsd'")
    return (B, S, H, D), (sb, ss, sh, sd)


def _tables_for(x, cos, sin, S, D):
    if cos.shape != (S, D) or sin.shape != (S, D):
        raise ValueError(f"cos/sin must be [{S}, {D}], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    # The kernels work in the activation dtype (see module docstring).
    if cos.dtype != x.dtype:
        cos = cos.to(x.dtype)
    if sin.dtype != x.dtype:
        sin = sin.to(x.dtype)
    if cos.stride(1) != 1:
        cos = cos.contiguous()
    if sin.stride() != cos.stride():
        sin = sin.contiguous()
        cos = cos.contiguous()
    return cos, sin


def _launch(x, y, cos, sin, interleaved, layout):
    dev = N.require_cuda("apply_rope", x, y, cos, sin)
    (B, S, H, D), (xsb, xss, xsh, _) = _resolve_layout(x, layout)
    _, (ysb, yss, ysh, _) = _resolve_layout(y, layout)
    if D % 2 != 0:
        raise ValueError("head_dim must be even for RoPE")
    cos, sin = _tables_for(x, cos, sin, S, D)
    a = N.RopeArgs(
        x=N.ptr(x), y=N.ptr(y), cos=N.ptr(cos), sin=N.ptr(sin),
        batch=B, seq=S, heads=H, head_dim=D,
        x_stride_b=xsb, x_stride_s=xss, x_stride_h=xsh,
        y_stride_b=ysb, y_stride_s=yss, y_stride_h=ysh,
        table_stride_s=cos.stride(0),
        interleaved=int(bool(interleaved)), dtype=N.dtype_code(x), stream=N.stream_handle(dev),
    )
    N.call("rfx_rope_apply", a, dev)


def apply_rope(
    x: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    interleaved: bool = False,
    layout: str = "bshd",
    backend: Optional[str] = None,
) -> torch.Tensor:
    """Apply RoPE to ``x``; returns a new contiguous tensor.

    ``x``: ``[B, S, H, D]`` (``bshd``) or ``[B, H, S, D]`` (``bhsd``); ``cos``/``sin``: ``[S, D]``;
    row ``s`` rotates sequence index ``s``. ``interleaved`` pairs ``(2i, 2i+1)``, otherwise
    ``(i, i + D/2)``.
    """
    N.check_backend(backend)
    _resolve_layout(x, layout)
    if x.stride(-1) != 1:
        x = x.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _launch(x, y, cos, sin, interleaved, layout)
    return y


def apply_rope_(
    x: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    interleaved: bool = False,
    layout: str = "bshd",
    backend: Optional[str] = None,
) -> torch.Tensor:
    """In-place RoPE. Returns the (mutated) input tensor.

    ``x`` may be any strided view whose last axis is contiguous; a view that is not
    raises instead of silently rotating a copy (the reference's Triton path does the
    latter, ``kernels/rope/triton_rope.py:172-173``).
    """
    N.check_backend(backend)
    _resolve_layout(x, layout)
    if x.stride(-1) != 1:
        raise ValueError("apply_rope_: the head_dim axis must be contiguous to rotate in place")
    _launch(x, x, cos, sin, interleaved, layout)
    return x


def build_rope_tables(
    seq_len: int,
    head_dim: int,
    *,
    base: float = 10000.0,
    device: Optional[torch.device] = None,
    dtype: torch.dtype = torch.float32,
    interleaved: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Build the cos/sin tables ``[seq_len, head_dim]`` on the device.

    Same recipe as the reference (``kernels/rope/triton_rope.py:247-285``): inverse
    frequencies ``1/base**(i/half)`` in fp32, angle = position * frequency in fp32,
    cos/sin, duplicated to width ``head_dim`` (concatenated halves, or repeated pairs when
    ``interleaved``), cast to ``dtype``. The ``half``-long frequency vector is formed with
    the very torch expression the reference uses and handed to the kernel, so the angles
    are bit-identical; cos/sin are correctly rounded on the device, within 1 fp32 ulp of
    torch's CPU values.
    """
    if head_dim % 2 != 0:
        raise ValueError("head_dim must be even for RoPE")
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise RuntimeError(f"build_rope_tables builds on a CUDA device (got {dev}); there is no CPU path")
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    half = head_dim // 2
    inv_freq = (1.0 / (base ** (torch.arange(0, half, dtype=torch.float32) / half))).to(dev)
    cos = torch.empty((seq_len, head_dim), dtype=dtype, device=dev)
    sin = torch.empty_like(cos)
    a = N.RopeTableArgs(cos=N.ptr(cos), sin=N.ptr(sin), inv_freq=N.ptr(inv_freq), seq_len=seq_len,
                        head_dim=head_dim, base=float(base), interleaved=int(bool(interleaved)),
                        dtype=N.dtype_code(cos), stream=N.stream_handle(dev))
    N.call("rfx_rope_build_tables", a, dev)
    return cos, sin


_dense = N.Entry("rfx_qk_norm_rope", N.QkNormRopeArgs)


def _norm_inputs(name, q, k, q_weight, k_weight, cos, sin, positions, eps):
    """The checks that the dense form and the append share; returns ``(n, H_kv, D, H_q, dtype, cos, sin,
    positions, q_weight, k_weight, table_f32)`` as the kernel takes them. ``q`` may be ``None`` (no query
    heads). Every attribute is read once: for a decode step this costs more than the kernel."""
    shape, dtype, hq = k.shape, k.dtype, 0
    if q is not None:
        q_shape = q.shape
        if len(q_shape) != 3 or len(shape) != 3 or q_shape[0] != shape[0] or q_shape[2] != shape[2]:
            raise ValueError(f"{name}: q must be [N, H_q, D] and k [N, H_kv, D]; got {tuple(q_shape)} and {tuple(shape)}")
        if q.dtype != dtype:
            raise RuntimeError(f"{name}: q dtype {q.dtype} differs from k dtype {dtype}")
        hq = q_shape[1]
    elif len(shape) != 3:
        raise ValueError(f"{name}: k must be [N, H_kv, D], got {tuple(shape)}")
    n, hkv, D = shape
    if D % 2 != 0:
        raise ValueError("head_dim must be even for RoPE")
    for w in (q_weight, k_weight):
        if w.shape != (D,):
            raise ValueError(f"{name}: weights must be [{D}], got {tuple(w.shape)}")
        if w.dtype != dtype:
            raise RuntimeError(f"{name}: weight dtype {w.dtype} differs from the activations' {dtype}")
    rows = cos.shape
    if len(rows) != 2 or rows[1] != D or sin.shape != rows:
        raise ValueError(f"{name}: cos/sin must both be [rows, {D}], got {tuple(rows)} and {tuple(sin.shape)}")
    table = cos.dtype
    if (table != torch.float32 and table != dtype) or sin.dtype != table:
        cos, sin, table = cos.to(dtype), sin.to(dtype), dtype
    strides = cos.stride()
    if strides[1] != 1 or sin.stride() != strides:
        cos, sin = cos.contiguous(), sin.contiguous()
    if positions is not None:
        if positions.shape != (n,):
            raise ValueError(f"{name}: positions must be [N]={n}, got {tuple(positions.shape)}")
        if positions.dtype != torch.int32:
            if positions.dtype == torch.int64:
                positions = positions.clamp(-1, 2**31 - 1)
            positions = positions.to(torch.int32)
        positions = positions.contiguous()
    elif n > rows[0]:
        raise ValueError(f"{name}: {n} tokens without positions need as many table rows, got {rows[0]}")
    if not 0.0 <= eps < 3e38:
        raise ValueError(f"{name}: eps must not be negative, got {eps}")
    return (n, hkv, D, hq, dtype, cos, sin, positions, q_weight.contiguous(), k_weight.contiguous(),
            1 if table == torch.float32 else 0)


def _rows(t):
    """``t`` and its token and head strides, its last axis contiguous (a copy where it is not)."""
    st = t.stride()
    if st[-1] != 1:
        t = t.contiguous()
        st = t.stride()
    return t, st[0], st[1]


def _norm_rope(name, q, k, in_place, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    index = N.same_device(name, k, q, q_weight, k_weight, cos, sin, positions)
    n, hkv, D, hq, _, cos, sin, positions, q_weight, k_weight, f32 = _norm_inputs(
        name, q, k, q_weight, k_weight, cos, sin, positions, eps)
    code = N.dtype_code(k)
    q, q_sn, q_sh = _rows(q)
    k, k_sn, k_sh = _rows(k)
    if in_place:
        q_out, k_out, qo_sn, qo_sh, ko_sn, ko_sh = q, k, q_sn, q_sh, k_sn, k_sh
    else:
        q_out, k_out = q.new_empty((n, hq, D)), k.new_empty((n, hkv, D))
        qo_sn, qo_sh, ko_sn, ko_sh = hq * D, D, hkv * D, D
    _dense(index,
           q.data_ptr(), k.data_ptr(), 0, q_out.data_ptr(), k_out.data_ptr(), 0, 0,
           0, 0 if positions is None else positions.data_ptr(), cos.data_ptr(), sin.data_ptr(),
           q_weight.data_ptr(), k_weight.data_ptr(),
           n, hq, hkv, D, 0, 0, cos.shape[0],
           q_sn, q_sh, k_sn, k_sh, 0, 0, qo_sn, qo_sh, ko_sn, ko_sh, 0, 0, 0, cos.stride(0),
           eps, 1 if interleaved else 0, f32, code, 0, 0, 0, N.stream_of(index))
    return q_out, k_out


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    positions: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    backend: Optional[str] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q`` and ``k``, then its rotation; returns new contiguous tensors.

    ``q``: ``[N, H_q, D]``, ``k``: ``[N, H_kv, D]``, any token and head strides (views of a packed
    projection are read in place); ``q_weight``/``k_weight``: ``[D]`` in the activations' dtype;
    ``cos``/``sin``: ``[rows, D]`` in float32 or the activations' dtype (others are cast to the latter);
    ``positions``: ``[N]`` table row of each token (default: token ``n`` has row ``n``). ``D`` is even and
    at most 512. A head is ``x / sqrt(mean(x^2) + eps) * weight``, rotated in pairs ``(i, i + D/2)`` or
    (``interleaved``) ``(2i, 2i + 1)``; all in fp32, rounded once. A token whose position lies outside
    the tables gives zeros.
    """
    N.check_backend(backend)
    return _norm_rope("qk_norm_rope", q, k, False, q_weight, k_weight, cos, sin, positions, eps, interleaved)


def qk_norm_rope_(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    positions: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    backend: Optional[str] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``qk_norm_rope`` in place; returns ``(q, k)``. The last axis of both must be contiguous and their
    rows distinct memory (no expanded views). A token whose position lies outside the tables is left as
    it is."""
    N.check_backend(backend)
    for t in (q, k):
        if t.stride(-1) != 1:
            raise ValueError("qk_norm_rope_: the head_dim axis must be contiguous to work in place")
        if any(st == 0 and size > 1 for st, size in zip(t.stride(), t.shape)):
            raise ValueError("qk_norm_rope_: an expanded view has no rows of its own to work in place")
    return _norm_rope("qk_norm_rope_", q, k, True, q_weight, k_weight, cos, sin, positions, eps, interleaved)


# The reference's surface; qk_norm_rope and qk_norm_rope_ are additions, imported by name.
__all__ = [
    "apply_rope",
    "apply_rope_",
    "build_rope_tables",
]
