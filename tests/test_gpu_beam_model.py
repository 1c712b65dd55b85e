"""Beam search of whole models: the operators together, over the shared cache.

The oracle recomputes every beam in fp32 at every step. Its candidates are kept at
least 1e-3 apart (asserted), an fp32 model's summed log-probabilities being off by
less (hidden sizes of a few hundred: 1e-4 in the logits, as for the other model
tests), so ids have to be equal.
"""
import pytest
import torch

from oracle import beam as oracle

pytestmark = pytest.mark.gpu


def make(dtype=torch.float32, seed=3, sharp=12.0, **kw):
    from llm_cuda.models.llama3.config import Llama3Config
    from llm_cuda.models.llama3.model import Llama3ForCausalLM

    torch.manual_seed(seed)
    base = dict(vocab_size=300, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
                num_attention_heads=8, num_key_value_heads=4, max_position_embeddings=256)
    base.update(kw)
    cfg = Llama3Config(**base)
    model = Llama3ForCausalLM(cfg).eval()
    with torch.no_grad():
        for p in model.model.layers.parameters():
            if p.dim() == 2:
                p.mul_(6.0)
        model.lm_head.weight.mul_(sharp)
    return cfg, model.to(dtype)


@pytest.mark.parametrize("N,S,W,T,page,eos", [
    (1, 7, 4, 9, 8, None), (2, 9, 3, 12, 8, None), (2, 17, 5, 6, 16, None), (1, 5, 8, 20, 64, None),
    (2, 8, 4, 10, 8, 17), (1, 1, 3, 6, 8, None), (1, 6, 4, 1, 8, None), (1, 6, 4, 2, 8, None),
    (1, 6, 3, 8, 6, None)])  # (the last: pages that are no power of two)
def test_equals_the_oracle(cuda, N, S, W, T, page, eos):
    cfg, model = make()
    g = torch.Generator().manual_seed(N * 100 + S * 10 + W + T)
    ids = torch.randint(0, cfg.vocab_size, (N, S), generator=g)
    want, scores, gap = oracle.beam_search(model.state_dict(), cfg, ids, W, T, eos)
    assert gap > 1e-3, f"candidates only {gap:.1e} apart"
    got, got_scores = model.to(cuda).beam_search(ids.to(cuda), W, T, page_size=page, eos_token_id=eos)
    torch.cuda.synchronize()
    assert got.shape == (N, W, S + T) and got_scores.dtype == torch.float32
    assert torch.equal(got.cpu(), want)
    assert (got_scores.double().cpu() - scores).abs().max().item() <= 1e-3


def test_finished_beams_keep_their_score(cuda):
    """A frequent end token: finished beams end in it and their score is that of the
    tokens up to the first one."""
    cfg, model = make()
    ids = torch.randint(0, cfg.vocab_size, (2, 6), generator=torch.Generator().manual_seed(0))
    free, _, _ = oracle.beam_search(model.state_dict(), cfg, ids, 4, 6)
    eos = int(free[0, 0, 8])  # a token that the best beam produces
    want, _, _ = oracle.beam_search(model.state_dict(), cfg, ids, 4, 10, eos)
    assert (want[:, :, 6:] == eos).any()
    got, got_scores = model.to(cuda).beam_search(ids.to(cuda), 4, 10, page_size=8, eos_token_id=eos)
    got, got_scores = got.cpu(), got_scores.double().cpu()
    assert (got[:, :, 6:] == eos).any()
    for n in range(2):
        for w in range(4):
            row = got[n, w, 6:].tolist()
            end = row.index(eos) + 1 if eos in row else len(row)
            assert all(t == eos for t in row[end:])
            logits = oracle_logits(model, cfg, got[n, w:w + 1, :6 + end])
            lp = torch.log_softmax(logits.double(), -1)[0]
            total = sum(lp[5 + i, row[i]].item() for i in range(end))
            assert abs(total - got_scores[n, w].item()) <= 1e-3


def oracle_logits(model, cfg, ids):
    from oracle.model import forward

    return forward({k: v.cpu() for k, v in model.state_dict().items()}, cfg, ids)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_beam_is_greedy(cuda, dtype):
    cfg, model = make(dtype, hidden_size=256, vocab_size=1000)
    model = model.to(cuda)
    ids = torch.randint(0, cfg.vocab_size, (3, 11), device=cuda)
    got, _ = model.beam_search(ids, 1, 8)
    if dtype == torch.float32:
        assert torch.equal(got[:, 0], model.generate(ids, max_new_tokens=8, use_paged_kv=True))
    else:
        # bf16 roundings differ between the two attention paths: each token has to be the
        # argmax of the model's own logits up to their rounding (2^-8 relative, two ways)
        logits = model(got[:, 0])["logits"].float()
        step = logits[:, 10:-1]
        best = step.max(-1).values
        took = torch.gather(step, 2, got[:, 0, 11:].unsqueeze(-1)).squeeze(-1)
        assert ((best - took) <= 0.1 * best.abs().clamp(min=1)).all()


@pytest.mark.parametrize("dtype,N,W,T,eos", [
    (torch.float32, 2, 3, 9, None), (torch.bfloat16, 2, 8, 12, 5), (torch.bfloat16, 1, 40, 6, None),
    (torch.bfloat16, 2, 4, 2, None), (torch.float16, 1, 4, 20, None)])
def test_graph_replays_equal_eager_steps(cuda, dtype, N, W, T, eos):
    cfg, model = make(dtype, hidden_size=512, intermediate_size=1024, vocab_size=2000,
                      num_key_value_heads=2)
    model = model.to(cuda)
    ids = torch.randint(0, cfg.vocab_size, (N, 9), device=cuda)
    eager, scores = model.beam_search(ids, W, T, page_size=8, eos_token_id=eos)
    for _ in range(2):
        got, got_scores = model.beam_search(ids, W, T, page_size=8, eos_token_id=eos, use_graph=True)
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.equal(got_scores, scores)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-3), (torch.bfloat16, 0.6)])
def test_scores_are_the_models_own(cuda, dtype, tol):
    """A beam's score is the sum of the log-probabilities that a full forward of its ids
    gives (bf16: 12 tokens whose logits of size about 10 are off by some 2^-8 each way)."""
    cfg, model = make(dtype, hidden_size=512, intermediate_size=1024, vocab_size=2000,
                      num_key_value_heads=2)
    model = model.to(cuda)
    ids = torch.randint(0, cfg.vocab_size, (2, 40), device=cuda)
    got, scores = model.beam_search(ids, 6, 12, page_size=16)
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    flat = got.view(12, 52)
    assert torch.unique(flat, dim=0).shape[0] == 12
    with torch.no_grad():
        lp = torch.log_softmax(model(flat)["logits"].double(), -1)
    total = torch.gather(lp[:, 39:-1], 2, flat[:, 40:].unsqueeze(-1)).sum((1, 2)).view(2, 6)
    assert (total - scores.double()).abs().max().item() <= tol


def test_refusals(cuda):
    from llm_cuda import BeamKVCache

    cfg, model = make()
    model = model.to(cuda)
    ids = torch.zeros(1, 4, dtype=torch.int64, device=cuda)
    for args, kw in (((0,), {}), ((65,), {}), ((2, 0), {}), ((2,), dict(eos_token_id=300)),
                     ((2,), dict(eos_token_id=-1)), ((2,), dict(page_size=0))):
        with pytest.raises(ValueError):
            model.beam_search(ids, *args, **kw)
    with pytest.raises(ValueError):
        model.beam_search(ids[0], 2)
    none, scores = model.beam_search(ids[:0], 2, 3)
    assert none.shape == (0, 2, 7) and scores.shape == (0, 2)
    cache = BeamKVCache(2, 4, 16, 1, 2, 4, 1, 8, cuda, torch.float32)
    mask = torch.zeros(1, 1, 4, 4, device=cuda)
    with torch.no_grad():
        with pytest.raises(NotImplementedError):
            model.model(ids, attention_mask=mask, past_key_values=cache, use_cache=True)
        with pytest.raises(ValueError):
            model.model(ids, past_key_values=cache)
        with pytest.raises(ValueError):
            model.model(ids.repeat(1, 2), past_key_values=cache, use_cache=True)  # too long
        model.model(ids, past_key_values=cache, use_cache=True)
        with pytest.raises(ValueError):
            model.model(ids, past_key_values=cache, use_cache=True)  # not one token of two beams
        step = torch.zeros(2, 1, dtype=torch.int64, device=cuda)
        model.model(step, past_key_values=cache, use_cache=True)
        with pytest.raises(ValueError):
            model.model(step, past_key_values=cache, use_cache=True)  # past max_new_len
    with pytest.raises(ValueError):
        cache.reorder(torch.zeros(2, 1, dtype=torch.int64, device=cuda))
