"""Beam operators without a GPU: sizes past the kernels' index arithmetic, and what calls share."""
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
