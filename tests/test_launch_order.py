"""Kernels that are launched programmatically may start while the kernels ahead of them still run. What each may do
before its wait is read from the source here: a kernel that breaks the rule would race on a GPU only now and then."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "reflex-infer_b200" / "csrc"
WAIT, TRIGGER = "ptx::pdl_wait()", "ptx::pdl_trigger()"


def _code(name):
    """The file without its comments."""
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def _bodies(name):
    """``{kernel: text of its definition}`` of a file."""
    parts = re.split(r"__global__", _code(name))[1:]
    return {re.search(r"(\w+_kernel)\s*\(", p).group(1): p for p in parts}


def test_the_plan_writes_nothing_before_its_wait():
    body = _bodies("plan.cu")["plan_kernel"]
    assert body.count(WAIT) == 1
    inside = body[body.index("{"):]
    before, after = inside.split(WAIT)
    for name in ("hdr", "pair_item_begin", "pair_counter", "part_first", "items", "item_prow"):
        assert not re.search(rf"\b{name}\s*\[", before), name
        assert re.search(rf"\b{name}\s*\[", after), name
    # (unit_order as a pointer only: whether there is a list)
    assert not re.search(r"\bunit_order\s*\[", before) and re.search(r"\bunit_order\s*\[", after)


@pytest.mark.parametrize("name", ["qk_norm.cuh", "kv_pages.cu", "sample.cu"])
def test_kernels_wait_before_they_let_the_next_one_start(name):
    kernels = _bodies(name)
    assert kernels
    for kernel, body in kernels.items():
        assert body.count(WAIT) == 1, kernel
        if TRIGGER in body:
            assert body.index(WAIT) < body.index(TRIGGER), kernel
        assert not re.search(r"->|\[", body[body.index("{"):body.index(WAIT)]), kernel  # nothing is read or written first


def test_kernels_that_write_32_bit_words_do_not_let_the_next_one_start_early():
    """The plan reads context lengths before its wait; these kernels' outputs may be such lengths."""
    kernels = _bodies("kv_pages.cu")
    for kernel in ("kv_fork_small_kernel", "kv_fork_table_kernel", "kv_free_kernel", "kv_compact_small_kernel",
                   "kv_compact_apply_kernel"):
        assert TRIGGER not in kernels[kernel], kernel
