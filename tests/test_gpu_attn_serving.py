"""PagedGenerator on a tiny random-init fp16 Llama (head_dim 128) against the
model's own forward: the bar is the one of the one-sequence generator's test
(2e-2 on logits of order one, fp16)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tiny_llama(n_q=4, n_kv=2, vocab=500, seed=0):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(seed)
    cfg = LlamaConfig(vocab_size=vocab, hidden_size=n_q * 128, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=n_q, num_key_value_heads=n_kv, head_dim=128, max_position_embeddings=1024,
                      rope_theta=500000.0)
    return LlamaForCausalLM(cfg).half().to(DEV).eval()


def want_logits(m, ids):
    with torch.no_grad():
        return m(torch.tensor([ids], device=DEV)).logits[0].float()


def prompts_of(ns, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 500, (n,), generator=g).tolist() for n in ns]


def test_requests_of_many_lengths_match_the_model():
    from kvr_b200 import PagedGenerator
    m = tiny_llama()
    gen = PagedGenerator(m, n_pages=60, page=16, max_requests=6, chunk=64)
    prompts = prompts_of([150, 1, 64, 333])
    rows = gen.add(prompts)
    seqs = {b: list(p) for b, p in zip(rows, prompts)}
    for b in rows:
        assert torch.allclose(gen.last[b], want_logits(m, seqs[b])[-1], rtol=2e-2, atol=2e-2), b
    # a fifth prompt arrives while the others decode: a chunk and single tokens in one step
    late = prompts_of([90], 2)[0]
    new = {b: [7 + b] for b in rows}
    new[4] = late
    got = gen.step(new)
    for b in rows:
        seqs[b].append(7 + b)
    seqs[4] = late
    for b, s in seqs.items():
        assert torch.allclose(got[b], want_logits(m, s)[-1], rtol=2e-2, atol=2e-2), b
    # greedy tokens: each is a best one of the model's own logits, up to the bar
    out = gen.generate([0, 4], 5)
    for b in (0, 4):
        for t in out[b]:
            w = want_logits(m, seqs[b])[-1]
            assert w[t] >= w.max() - 4e-2, b
            seqs[b].append(t)
    used = gen.cache.n_free.item()
    gen.drop([3, 4])
    assert gen.cache.n_free.item() == used + -(-len(seqs[3]) // 16) + -(-len(seqs[4]) // 16)


def test_score_matches_the_model():
    from kvr_b200 import PagedGenerator
    m = tiny_llama(n_q=8, n_kv=1)
    gen = PagedGenerator(m, n_pages=4, page=16, max_requests=1)
    prompts = prompts_of([3, 200, 1, 77])
    for p, got in zip(prompts, gen.score(prompts)):
        assert torch.allclose(got, want_logits(m, p), rtol=2e-2, atol=2e-2), len(p)


def test_refusals_leave_the_cache_usable():
    from kvr_b200 import PagedGenerator
    m = tiny_llama()
    gen = PagedGenerator(m, n_pages=4, page=16, max_requests=2, max_len=256)
    rows = gen.add(prompts_of([40]))
    with pytest.raises(RuntimeError, match="does not fit"):
        gen.step({1: prompts_of([50], 3)[0]})
    with pytest.raises(RuntimeError, match="free rows"):
        gen.add(prompts_of([1, 1]))
    with pytest.raises(ValueError, match="at least one"):
        gen.step({0: []})
    gen.drop(rows)
    p = prompts_of([50], 3)[0]
    rows = gen.add([p])
    assert torch.allclose(gen.last[rows[0]], want_logits(m, p)[-1], rtol=2e-2, atol=2e-2)
