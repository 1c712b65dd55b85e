"""A pooled cache whose batch grew past the one that its pool was made for: a fork that finds too
few free pages raises and leaves the cache as it was, however many rows it asks for."""
import pytest
import torch

from llm_cuda.kernels import _ops
from llm_cuda.models.llama3.kv_cache import PooledKVCache
from oracle import speculative as oracle

I64 = torch.int64


def on_the_cpu(monkeypatch):
    """The pool's operators by the oracle."""
    def stands_in(name, results):
        def call(key_pages, value_pages, *args):
            got = getattr(oracle, f"kv_{name}")(key_pages, value_pages, *args)
            key_pages.copy_(got[-2])
            value_pages.copy_(got[-1])
            return got[:results]
        monkeypatch.setattr(_ops, f"paged_kv_{name}", call)

    stands_in("resize", 3)
    stands_in("fork", 4)


def grow(cache, tokens):
    """A step whose tokens' contents do not matter."""
    cache.reserve(tokens)
    cache.seq_lens_all.add_(tokens)
    cache.appended(len(cache.layer_caches) - 1, tokens)


def forks_down_from_a_full_pool(dev):
    cache = PooledKVCache(1, 1, 2, 8, 4, dev, torch.float32, batch_size=2)  # 6 pages
    grow(cache, 3)
    cache.fork(torch.tensor([0, 0, 1], dtype=I64, device=dev))
    grow(cache, 4)  # 3 rows of 7 tokens: all pages
    assert cache.pages_in_use() == cache.num_pages
    state = {k: getattr(cache, k).clone() for k in ("block_table", "page_refs", "seq_lens_all")}
    with pytest.raises(RuntimeError, match="1 short"):
        cache.fork(torch.tensor([0, 0], dtype=I64, device=dev))
    assert cache.batch_size == 3 and all(torch.equal(getattr(cache, k), t) for k, t in state.items())
    # without a second child, and once a row has left, there is room
    cache.fork(torch.tensor([0, 2], dtype=I64, device=dev))
    assert cache.pages_in_use() == 4
    cache.fork(torch.tensor([0, 0], dtype=I64, device=dev))
    lens = cache.seq_lens.tolist()
    table = cache.block_table.tolist()
    assert lens == [7, 7] and table[0][0] == table[1][0] and table[0][1] != table[1][1]
    assert min(min(r) for r in table) >= 0


def test_fork_of_a_batch_that_has_grown(monkeypatch):
    on_the_cpu(monkeypatch)
    forks_down_from_a_full_pool(torch.device("cpu"))


@pytest.mark.gpu
def test_fork_of_a_batch_that_has_grown_on_the_gpu(cuda):
    forks_down_from_a_full_pool(cuda)
