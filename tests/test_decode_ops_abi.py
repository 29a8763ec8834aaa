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


def test_page_refusals(native):
    lib, bad = native.lib(), native.RFX_INVALID_ARGUMENT
    fork = dict(block_table=256, context_lens=256, parents=256, ref_counts=256, child_table=256, src_pages=256,
                dst_pages=256, copy_rows=256, n_children=1, batch=1, max_blocks=2, bt_stride_b=2, num_blocks=4, block_size=4)
    for kw in (dict(n_children=-1), dict(num_blocks=0), dict(num_blocks=1 << 31), dict(block_size=0), dict(batch=-1),
               dict(parents=0), dict(ref_counts=0), dict(child_table=0), dict(block_table=0), dict(context_lens=0),
               dict(dst_pages=0)):
        assert lib.rfx_kv_fork(C.byref(native.KvForkArgs(**{**fork, **kw}))) == bad, kw
    assert lib.rfx_kv_fork(C.byref(native.KvForkArgs(**{**fork, "n_children": 0}))) == native.RFX_SUCCESS
    free = dict(block_table=256, rows=256, ref_counts=256, n_rows=1, batch=1, max_blocks=2, bt_stride_b=2, num_blocks=4)
    for kw in (dict(n_rows=-1), dict(num_blocks=0), dict(rows=0), dict(block_table=0), dict(ref_counts=0)):
        assert lib.rfx_kv_free(C.byref(native.KvFreeArgs(**{**free, **kw}))) == bad, kw
    assert lib.rfx_kv_free(C.byref(native.KvFreeArgs(**{**free, "n_rows": 0}))) == native.RFX_SUCCESS
    need = lib.rfx_kv_compact_workspace_bytes(5000)
    assert need >= 8 and need % 256 == 0 and lib.rfx_kv_compact_workspace_bytes(0) == 0
    compact = dict(block_table=256, ref_counts=256, page_map=256, src_pages=256, dst_pages=256, n_moves=256, batch=1,
                   max_blocks=2, bt_stride_b=2, num_blocks=5000, workspace=256, workspace_bytes=need)
    for kw in (dict(num_blocks=0), dict(page_map=0), dict(n_moves=0), dict(block_table=0), dict(batch=-1)):
        assert lib.rfx_kv_compact(C.byref(native.KvCompactArgs(**{**compact, **kw}))) == bad, kw
    for kw in (dict(workspace=0), dict(workspace_bytes=need - 1)):
        assert lib.rfx_kv_compact(C.byref(native.KvCompactArgs(**{**compact, **kw}))) == native.RFX_WORKSPACE_TOO_SMALL
    for fn in (lib.rfx_kv_fork, lib.rfx_kv_free, lib.rfx_kv_compact, lib.rfx_kv_copy_pages):
        assert fn(None) == bad
    ptrs, none = (native.vp * 1)(256), (native.vp * 1)(None)
    copy = dict(k_caches=ptrs, v_caches=ptrs, src_pages=256, dst_pages=256, n_layers=1, n_pairs=1, num_kv_heads=1,
                head_dim=8, num_blocks=4, block_size=4, cache_stride_blk=32, cache_stride_h=32, cache_stride_pos=8, dtype=1)
    for kw in (dict(dtype=9), dict(n_pairs=-1), dict(num_kv_heads=0), dict(block_size=0), dict(src_pages=0),
               dict(k_caches=none), dict(kv_int8=1), dict(head_dim=0)):
        assert lib.rfx_kv_copy_pages(C.byref(native.KvCopyArgs(**{**copy, **kw}))) == bad, kw
    for kw in (dict(n_pairs=0), dict(n_layers=0)):
        assert lib.rfx_kv_copy_pages(C.byref(native.KvCopyArgs(**{**copy, **kw}))) == native.RFX_SUCCESS


def test_sample_refusals(native):
    lib = native.lib()
    good = dict(logits=256, uniform=256, tokens=256, batch=1, vocab=8, row_stride=8, temperature_all=1.0, top_p_all=1.0, dtype=1)
    for kw in (dict(dtype=5), dict(batch=-1), dict(vocab=0), dict(vocab=-3), dict(vocab=(1 << 24) + 1), dict(logits=0),
               dict(uniform=0), dict(tokens=0), dict(logits=257)):
        assert lib.rfx_sample_tokens(C.byref(native.SampleArgs(**{**good, **kw}))) == native.RFX_INVALID_ARGUMENT, kw
    assert lib.rfx_sample_tokens(None) == native.RFX_INVALID_ARGUMENT
    assert lib.rfx_sample_tokens(C.byref(native.SampleArgs(**{**good, "batch": 0}))) == native.RFX_SUCCESS
