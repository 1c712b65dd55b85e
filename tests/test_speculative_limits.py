"""Operators of speculative decoding without a GPU: sizes past what a launch can take."""
import torch


def test_batches_past_a_launch_are_refused():
    """The deciding launch has 1024 threads a sequence, and a launch fewer than 2^32: the call is
    refused as a whole, before its first pass has run."""
    from llm_cuda import _native

    lib = _native.load()
    buf = torch.zeros(1 << 12, dtype=torch.uint8)
    base = (buf.data_ptr() + 255) // 256 * 256

    for B in (1 << 22, (1 << 24) - 1):
        need = lib.lc_verify_draft_tokens_workspace_bytes(B, 0, 10)
        rc = lib.lc_verify_draft_tokens(base, 10, 10, None, 0, 0, None, base, None, None, 1.0, B, 0, 10, base, base,
                                        base, need, 0, None)
        assert rc < 0 and b"sequences" in lib.lc_last_error(), (B, rc, lib.lc_last_error())
