"""The C entry of the list's divergence knows four forms of what the list leaves."""

from __future__ import annotations


def test_forms_that_there_are_not_are_refused():
    from rte_amd import _lib

    lib, buf = _lib.load(), 1 << 20
    for tail in (-1, 4):
        assert lib.rte_topk_distill_fwd(buf, 64, 1, 4, 64, buf, buf, 8, 1.0, tail, buf, buf, buf, buf, buf, 1 << 40, None) != 0
        assert b"tail" in lib.rte_last_error()
