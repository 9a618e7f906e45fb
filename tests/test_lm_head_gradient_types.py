"""The C entry of the head's gradients in fp32 or bf16, without a device."""

from __future__ import annotations


def test_types_and_workspaces():
    from rte_amd import _lib

    lib, buf = _lib.load(), 1 << 20
    for flags in (-1, 4):
        assert lib.rte_lm_head_logprobs_bwd(buf, buf, 100, 128, 1000, buf, 1.0, buf, buf, buf, buf, 256, buf, buf, flags, buf,
                                            1 << 40, None) != 0
        assert b"grads_f32" in lib.rte_last_error()
    # fp32 gradients of several ranges are summed where they are wanted; a single range needs no room either way
    size = lib.rte_lm_head_logprobs_bwd_workspace_bytes
    assert size(100, 128, 1024, 256, 1, 1) - size(100, 128, 1024, 256, 2, 1) == 100 * 128 * 4
    assert size(100, 128, 1024, 1024, 1, 1) == size(100, 128, 1024, 1024, 2, 1)
