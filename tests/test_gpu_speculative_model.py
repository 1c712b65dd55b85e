"""Speculative decoding of a small model: greedy runs equal the model's own greedy decoding,
samples share pages, and the cache's counts stay those of its table."""
import pytest
import torch

from llm_cuda.models.llama3.config import Llama3Config
from llm_cuda.models.llama3.kv_cache import PooledKVCache
from llm_cuda.models.llama3.model import Llama3ForCausalLM

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def build(dev, dtype=F32, seed=0, layers=2, hidden=256, heads=8, kv=2, vocab=500):
    torch.manual_seed(seed)
    cfg = Llama3Config(vocab_size=vocab, hidden_size=hidden, intermediate_size=384, num_hidden_layers=layers,
                       num_attention_heads=heads, num_key_value_heads=kv, initializer_range=0.2)
    return Llama3ForCausalLM(cfg).to(dtype).to(dev).eval()


def prompts(dev, N=3, S=19, vocab=500, seed=1):
    return torch.randint(0, vocab, (N, S), generator=torch.Generator().manual_seed(seed)).to(dev)


def counts_match(cache):
    torch.cuda.synchronize()
    lens, P = cache.seq_lens.cpu(), cache.page_size
    held = torch.arange(cache.max_pages) < ((lens + P - 1) // P).unsqueeze(1)
    named = cache.block_table.cpu()[held].long()
    assert (named >= 0).all()
    assert torch.equal(torch.bincount(named, minlength=cache.num_pages).int(), cache.page_refs.cpu())


@pytest.mark.parametrize("page_size", [16, 64])
@pytest.mark.parametrize("K", [1, 3, 6])
def test_greedy_equals_generate(cuda, K, page_size):
    """fp32: the steps' logits differ by rounding (1e-5) where the choices of random models are
    apart by more."""
    model, draft = build(cuda, seed=0), build(cuda, seed=7, layers=1)
    ids = prompts(cuda)
    want = model.generate(ids, max_new_tokens=21, use_paged_kv=True)
    got, steps = model.speculative_generate(ids, draft, max_new_tokens=21, num_draft_tokens=K, page_size=page_size)
    assert got.shape == (3, 1, 40) and torch.equal(got[:, 0], want)
    assert steps <= 21


def test_a_perfect_draft_needs_few_steps(cuda):
    model = build(cuda)
    ids = prompts(cuda, N=2, S=33)
    got, steps = model.speculative_generate(ids, model, max_new_tokens=20, num_draft_tokens=4)
    assert torch.equal(got[:, 0], model.generate(ids, max_new_tokens=20, use_paged_kv=True))
    assert steps == 5  # the prompt's token, then 5 a round


@pytest.mark.parametrize("K", [2, 5, 9])
def test_sequences_that_end_in_different_rounds(cuda, K):
    """A draft model near the target: sequences overshoot the end by up to K while others go on."""
    import copy

    model = build(cuda)
    draft = copy.deepcopy(model)
    g = torch.Generator(device=cuda).manual_seed(0)
    with torch.no_grad():
        for p in draft.parameters():
            p.add_(0.04 * p.std() * torch.randn(p.shape, generator=g, device=cuda))
    ids = prompts(cuda, N=9, S=15)
    got, steps = model.speculative_generate(ids, draft, max_new_tokens=13, num_draft_tokens=K, page_size=16)
    assert torch.equal(got[:, 0], model.generate(ids, max_new_tokens=13, use_paged_kv=True))
    assert steps < 13


def test_draft_model_of_another_type(cuda):
    model, draft = build(cuda, BF16), build(cuda, F32, seed=2, layers=1)
    got, _ = model.speculative_generate(prompts(cuda), draft, max_new_tokens=9, num_draft_tokens=3, temperature=0.8)
    assert got.shape == (3, 1, 28)


def test_one_token_prompts_and_one_new_token(cuda):
    model, draft = build(cuda), build(cuda, seed=3)
    for S, T in ((1, 9), (5, 1), (1, 1)):
        ids = prompts(cuda, N=2, S=S)
        got, _ = model.speculative_generate(ids, draft, max_new_tokens=T, num_draft_tokens=2, page_size=16)
        assert torch.equal(got[:, 0], model.generate(ids, max_new_tokens=T, use_paged_kv=True))


def test_eos_ends_a_sequence(cuda):
    model, draft = build(cuda), build(cuda, seed=5)
    ids = prompts(cuda, N=4, S=12)
    plain = model.generate(ids, max_new_tokens=24, use_paged_kv=True)
    eos = int(plain[1, 17])
    got, _ = model.speculative_generate(ids, draft, max_new_tokens=24, num_draft_tokens=3, eos_token_id=eos)
    for b in range(4):
        want = plain[b].tolist()
        if eos in want[12:]:
            end = 12 + want[12:].index(eos)
            want[end:] = [eos] * (len(want) - end)
        assert got[b, 0].tolist() == want


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_samples(cuda, dtype):
    model, draft = build(cuda, dtype), build(cuda, dtype, seed=2, layers=1)
    ids = prompts(cuda, N=2, S=30)
    g = torch.Generator(device=cuda).manual_seed(4)
    got, steps = model.speculative_generate(ids, draft, max_new_tokens=17, num_draft_tokens=3, temperature=1.0,
                                            num_samples=5, generator=g, page_size=16)
    assert got.shape == (2, 5, 47) and torch.equal(got[:, :, :30], ids.unsqueeze(1).expand(2, 5, 30))
    assert (got >= 0).all() and (got < 500).all() and 1 < steps <= 17
    assert len({tuple(r) for r in got.view(10, -1).tolist()}) > 5
    again, _ = model.speculative_generate(ids, draft, max_new_tokens=17, num_draft_tokens=3, temperature=1.0,
                                          num_samples=5, generator=g.manual_seed(4), page_size=16)
    assert torch.equal(got, again)


def test_cache_follows_growth_forks_truncation_and_compaction(cuda):
    """Logits of continued sequences equal those of the whole text, whatever the pages went through."""
    model = build(cuda)
    ids = prompts(cuda, N=3, S=21)
    cache = model._pooled_cache(6, 64, 16, cuda)
    cache.fork(torch.arange(3, device=cuda))
    model._pooled_step(ids, cache)
    parents = torch.tensor([2, 0, 0, 2, 1], device=cuda)
    cache.fork(parents)
    counts_match(cache)
    text = ids[parents]
    more = prompts(cuda, N=5, S=7, seed=9)
    model._pooled_step(more, cache)
    counts_match(cache)
    keep = torch.tensor([28, 23, 20, 16, 1], dtype=torch.int32, device=cuda)
    cache.truncate(keep, 28)
    counts_match(cache)
    before = cache.pages_in_use()
    page_map = cache.compact()
    counts_match(cache)
    assert cache.pages_in_use() == before and int(cache.block_table.max()) == before - 1
    assert int((page_map >= 0).sum()) == before
    text = torch.cat([text, more], 1)
    last = prompts(cuda, N=5, S=3, seed=10)
    logits = model.lm_head(model._pooled_step(last, cache))
    counts_match(cache)
    for b in range(5):
        whole = torch.cat([text[b, :int(keep[b])], last[b]]).unsqueeze(0)
        want = model(whole)["logits"][0, -3:]
        assert (logits[b] - want).abs().max() <= 1e-4 * want.abs().max()


def test_small_pools_refuse_and_stay(cuda):
    model = build(cuda)
    cache = PooledKVCache(2, 2, 32, 64, 16, cuda, F32, batch_size=2, num_pages=4)
    model._pooled_step(prompts(cuda, N=2, S=30), cache)
    table, refs = cache.block_table.clone(), cache.page_refs.clone()
    with pytest.raises(RuntimeError, match="2 short"):
        cache.reserve(3)
    with pytest.raises(RuntimeError, match="short"):
        cache.fork(torch.tensor([0, 0, 1], device=cuda))
    assert torch.equal(cache.block_table, table) and torch.equal(cache.page_refs, refs)
    cache.fork(torch.tensor([1], device=cuda))
    model._pooled_step(prompts(cuda, N=1, S=20), cache)
    counts_match(cache)


def test_refusals(cuda):
    model = build(cuda)
    ids = prompts(cuda)
    for kw in (dict(num_draft_tokens=0), dict(num_draft_tokens=256), dict(max_new_tokens=0), dict(num_samples=0),
               dict(eos_token_id=500), dict(draft_model=build(cuda, vocab=400))):
        args = dict(draft_model=model)
        args.update(kw)
        with pytest.raises(ValueError):
            model.speculative_generate(ids, **args)
    with pytest.raises(ValueError):
        model.speculative_generate(ids[0], model)
    got, steps = model.speculative_generate(ids[:0], model, max_new_tokens=4)
    assert got.shape == (0, 1, 23) and steps == 0
    cache = model._pooled_cache(3, 32, 16, cuda)
    with pytest.raises(ValueError):
        model.model(ids, past_key_values=cache, use_cache=True)  # nothing reserved
    cache.reserve(19)
    for call in (lambda: cache.reserve(1), lambda: cache.truncate(cache.seq_lens, 0),
                 lambda: cache.fork(torch.arange(3, device=cuda)), cache.compact,
                 lambda: model.model(ids, past_key_values=cache),
                 lambda: model.model(ids[:, :5], past_key_values=cache, use_cache=True)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        model.model(ids, attention_mask=torch.zeros(1, 1, 19, 19, device=cuda), past_key_values=cache, use_cache=True)
    model.model(ids, past_key_values=cache, use_cache=True)
    with pytest.raises(ValueError):
        cache.reserve(14)
