"""Refusals of the norm + rotation, page and sampling entry points at the C boundary, without a GPU: a wrong
argument is a status and a message before any launch, an empty problem succeeds."""
from __future__ import annotations

import ctypes as C

import pytest


def _norm(native, **kw):
    base = dict(q=256, k=256, v=256, q_out=256, k_out=256, k_cache=256, v_cache=256, slot_mapping=256, positions=256,
                cos=256, sin=256, q_weight=256, k_weight=256, n_tokens=2, num_q_heads=2, num_kv_heads=1, head_dim=64,
                num_blocks=2, block_size=4, table_rows=8, eps=1e-6, dtype=1)
    return native.QkNormRopeArgs(**{**base, **kw})


@pytest.mark.parametrize("kw,text", [
    (dict(head_dim=63), b"even"), (dict(head_dim=0), b"even"), (dict(head_dim=514), b"512"), (dict(dtype=7), b"dtype"),
    (dict(n_tokens=-1), b"bad sizes"), (dict(num_q_heads=-1), b"bad sizes"), (dict(eps=-1.0), b"eps"),
    (dict(eps=float("nan")), b"eps"), (dict(cos=0), b"null"), (dict(k_weight=0), b"null"), (dict(q_out=0), b"null")])
def test_qk_norm_refusals(native, kw, text):
    lib = native.lib()
    for fn in (lib.rfx_qk_norm_rope, lib.rfx_qk_norm_rope_append):
        assert fn(C.byref(_norm(native, **kw))) == native.RFX_INVALID_ARGUMENT
        assert text in lib.rfx_last_error()


def test_qk_norm_refusals_of_one_form(native):
    lib = native.lib()
    assert lib.rfx_qk_norm_rope(None) == native.RFX_INVALID_ARGUMENT
    assert lib.rfx_qk_norm_rope(C.byref(_norm(native, k_out=0))) == native.RFX_INVALID_ARGUMENT
    for kw in (dict(num_blocks=0), dict(block_size=0), dict(num_kv_heads=0), dict(v=0), dict(k_cache=0),
               dict(slot_mapping=0), dict(positions=0), dict(kv_int8=1)):
        assert lib.rfx_qk_norm_rope_append(C.byref(_norm(native, **kw))) == native.RFX_INVALID_ARGUMENT, kw
    assert lib.rfx_qk_norm_rope(C.byref(_norm(native, n_tokens=0))) == native.RFX_SUCCESS
    assert lib.rfx_qk_norm_rope_append(C.byref(_norm(native, n_tokens=0))) == native.RFX_SUCCESS
