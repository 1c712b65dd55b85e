"""Beam operators without a GPU: sizes past the kernels' index arithmetic, and what calls share."""
import threading

import torch


def test_tables_past_32_bits_are_refused():
    """The kernel counts the entries of a group's table in 32 bits: 256 beams of 2^23 columns wrap."""
    from llm_cuda import _native

    lib = _native.load()
    buf = torch.zeros(1 << 12, dtype=torch.uint8)
    base = (buf.data_ptr() + 255) // 256 * 256

    def reorder(W, M):
        # (out on the far side of a table of that size: refused before anything is read)
        return lib.lc_paged_kv_reorder(base, base, 2048, 256, 128, 16, 1, 8, base, M, base + (1 << 40), M, M,
                                       base, base, 1, W, 2, 16, 8, 0, None)

    for W, M in ((256, 1 << 23), (128, 1 << 24), (255, (1 << 31) // 255), (256, (1 << 27) - 1)):
        assert reorder(W, M) < 0, (W, M)
        assert b"2^31 entries" in lib.lc_last_error()


def test_first_calls_of_two_threads_share_their_tickets(monkeypatch):
    """Two threads that both find no tickets for a stream launch with the same buffer, the one
    that is kept: the other's memory is free for any tensor as soon as it is dropped."""
    from llm_cuda.kernels import _ops

    both, zeros, got = threading.Barrier(2), torch.zeros, []

    def zeros_together(*args, **kw):
        buf = zeros(*args, **kw)
        try:
            both.wait(5)  # the other thread has found none either
        except threading.BrokenBarrierError:
            pass
        return buf

    monkeypatch.setattr(_ops, "_JOIN_COUNTERS", {})
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    monkeypatch.setattr(torch, "zeros", zeros_together)
    cpu = torch.device("cpu")
    threads = [threading.Thread(target=lambda: got.append(_ops._join_counters("beam_select", cpu, 0)))
               for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    (kept,) = _ops._JOIN_COUNTERS.values()
    assert got == [kept.data_ptr()] * 2
