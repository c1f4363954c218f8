"""PagedGenerator's beam search, dense and with sparse MLPs, on tiny random-init
models against the model's own forward: the selection, the reordering of shared
pages, attention over them and the sparse MLP together.

The bar for logits is the one of the generator's other tests (2e-2 on logits of
order one, fp16).  A continuation of n tokens adds up n log-probabilities, each
off by twice that at most (a logit and the log-sum-exp), so scores divided by n
are compared at 4e-2."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BAR = 2e-2


def tiny(sparse, seed=0, layers=2, experts=12, top_k=3):
    import transformers as T
    torch.manual_seed(seed)
    kw = dict(vocab_size=300, hidden_size=256, intermediate_size=512, num_hidden_layers=layers, num_attention_heads=4,
              num_key_value_heads=2, head_dim=128, max_position_embeddings=512)
    if sparse:
        cfg = T.Qwen3MoeConfig(**kw, moe_intermediate_size=72, num_experts=experts, num_experts_per_tok=top_k, norm_topk_prob=sparse == "norm")
        m = T.Qwen3MoeForCausalLM(cfg)
        for layer in m.model.layers:  # (weights that tell experts apart)
            for p in layer.mlp.parameters():
                torch.nn.init.normal_(p, std=0.1)
    else:
        m = T.LlamaForCausalLM(T.LlamaConfig(**kw))
    torch.nn.init.normal_(m.lm_head.weight, std=0.2)
    return m.half().to(DEV).eval()


def want_logits(m, ids):
    with torch.no_grad():
        return m(torch.tensor([ids], device=DEV)).logits[0].float()


def prompts_of(ns, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 300, (n,), generator=g).tolist() for n in ns]


def score_of(m, prompt, q):
    lp = want_logits(m, prompt + q)[len(prompt) - 1:-1].double().log_softmax(-1)
    return sum(lp[i, t].item() for i, t in enumerate(q))


def plain_beams(m, prompt, k, steps, eos):
    """Beam search on the model's own forward; also the least gap between what was kept and what was not."""
    beams, ended, gap = [(0.0, [])], [], math.inf
    for t in range(1, steps + 1):
        cand = []
        for s, q in beams:
            lp = want_logits(m, prompt + q)[-1].double().log_softmax(-1)
            top = lp.topk(2 * k)
            cand += [(s + v, q + [i]) for v, i in zip(top.values.tolist(), top.indices.tolist())]
        cand.sort(key=lambda c: -c[0])
        gap = min([gap] + [a[0] - b[0] for a, b in zip(cand[:2 * k], cand[1:2 * k + 1])])
        ended += [(s / t, q) for s, q in cand[:k] if q[-1] == eos]
        ended = sorted(ended, key=lambda e: -e[0])[:k]
        beams = [(s, q) for s, q in cand if q[-1] != eos][:k]
        if len(ended) == k and ended[-1][0] >= beams[0][0] / t:
            return ended, gap
    ended += [(s / len(q), q) for s, q in beams]
    return sorted(ended, key=lambda e: -e[0])[:k], gap


@pytest.mark.parametrize("sparse", [False, "norm", "plain"])
def test_beam_search_against_the_model(sparse):
    from kvr_b200 import PagedGenerator
    from kvr_b200 import kernels as K
    m = tiny(sparse)
    k, steps, eos = 4, 20, 7
    prompts = prompts_of([40, 1, 64, 133])
    gen = PagedGenerator(m, n_pages=90, page=16, max_requests=18, chunk=64)
    other = gen.add(prompts_of([30], 9))[0]  # a request beside them, whose pages nobody touches
    before = gen.cache.n_free.item()
    got = gen.beam_search(prompts, k, steps, eos=eos)
    K.attn_status()
    K.moe_status()
    assert gen.cache.n_free.item() == before and list(gen.last) == [other]
    assert gen.cache.shared.eq(0).all()
    for p, found in zip(prompts, got):
        assert 1 <= len(found) <= k and len({tuple(q) for q, _ in found}) == len(found)
        for q, s in found:
            assert 1 <= len(q) <= steps and eos not in q[:-1]
            assert abs(s - score_of(m, p, q) / len(q)) <= 2 * BAR, (s, score_of(m, p, q) / len(q))
        want, gap = plain_beams(m, p, k, steps, eos)
        # the best found is as good as the plain search's, up to what logits may be off by
        assert found[0][1] >= want[0][0] - 2 * BAR * 2
        # after t tokens two candidates' scores are off from one another by 4 BAR t at most: where the plain search never
        # had two as close as that, the same are kept
        if gap > 4 * BAR * steps:
            assert [q for q, _ in found] == [q for q, _ in want]
    # the other request goes on as if nothing had been
    text = prompts_of([30], 9)[0]
    step = gen.step({other: [5]})[other]
    assert torch.allclose(step, want_logits(m, text + [5])[-1], rtol=BAR, atol=BAR)


def exact_logits(m, ids):
    """The model in fp32: logits, and for each token how far the last expert chosen is from the first left out, at the
    least of all layers (and of the tokens before, which it sees)."""
    import copy
    big, gaps = copy.deepcopy(m).float(), []

    def look(gate, args, out):
        if gate.top_k == gate.weight.shape[0]:
            gaps.append(torch.full((len(ids),), math.inf, device=DEV))
            return
        z = (args[0].reshape(-1, gate.weight.shape[1]) @ gate.weight.t()).sort(-1, descending=True)[0]
        gaps.append(z[:, gate.top_k - 1] - z[:, gate.top_k])
    hooks = [layer.mlp.gate.register_forward_hook(look) for layer in big.model.layers]
    with torch.no_grad():
        out = big(torch.tensor([ids], device=DEV)).logits[0]
    for h in hooks:
        h.remove()
    return out.double(), torch.stack(gaps).min(0)[0].cummin(0)[0]


def check_logits(got, want, gap):
    """Rows of logits whose experts are the same either way: a router's logits, of order one like the others, are off by the
    bar at most, so a choice is safe where its gap is twice that."""
    safe = gap > 2 * BAR
    scale = want.std().item()
    if safe.any():
        assert ((got.double() - want)[safe].abs() <= BAR * (scale + want[safe].abs())).all(), (got.double() - want)[safe].abs().max()
    return int(safe.sum())


@pytest.mark.parametrize("experts,top_k", [(5, 5), (12, 3)])
def test_sparse_model_steps_and_chunks(experts, top_k):
    """Chunks of more tokens than the sparse operator takes go through the model's module, single tokens through the
    operator.  With all experts chosen no choice is close, and every row of logits says something."""
    from kvr_b200 import PagedGenerator
    m = tiny("norm", seed=3, experts=experts, top_k=top_k)
    gen = PagedGenerator(m, n_pages=60, page=16, max_requests=4, chunk=200)
    prompts = prompts_of([300, 17, 90])
    rows = gen.add(prompts)
    seqs = {b: list(p) for b, p in zip(rows, prompts)}
    seen = 0
    for t in range(4):
        for b in rows:
            want, gap = exact_logits(m, seqs[b])
            seen += check_logits(gen.last[b][None], want[-1:], gap[-1:])
            seqs[b].append(11 * t + b)
        gen.step({b: seqs[b][-1:] for b in rows})
    for p, got in zip(prompts[1:], gen.score(prompts[1:])):
        seen += check_logits(got, *exact_logits(m, p))
    assert seen >= (12 + 17 + 90 if experts == top_k else 4)  # (after a close choice no later token says anything)


def test_forked_rows_go_their_own_ways():
    """Rows forked from one prompt share its pages, go on with other tokens, fork again, and give back only what is theirs."""
    from kvr_b200 import PagedGenerator
    m = tiny(False, seed=4)
    gen = PagedGenerator(m, n_pages=24, page=16, max_requests=5, chunk=64)
    text = prompts_of([85])[0]
    (a,) = gen.add([text])
    n = gen.cache.n_free.item()
    assert gen.cache.reorder([[a, 3, 4]], [[0, 0, 0]]).tolist() == [0, 2, 0, 0]
    assert gen.cache.n_free.item() == n - 2  # five full pages are shared, the sixth copied twice
    seqs = {a: list(text), 3: list(text), 4: list(text)}
    for t in range(30):
        new = {b: [10 * b + t] for b in seqs}
        got = gen.step(new)
        for b in seqs:
            seqs[b] += new[b]
        if t % 9 == 0:
            for b in seqs:
                assert torch.allclose(got[b], want_logits(m, seqs[b])[-1], rtol=BAR, atol=BAR), (t, b)
        if t == 12:
            gen.cache.reorder([[a, 3, 4]], [[1, 1, 2]])
            seqs[a] = list(seqs[3])
    gen.drop([3])
    got = gen.step({a: [1], 4: [2]})
    for b, t in ((a, 1), (4, 2)):
        assert torch.allclose(got[b], want_logits(m, seqs[b] + [t])[-1], rtol=BAR, atol=BAR), b
    gen.drop([a, 4])
    assert gen.cache.n_free.item() == 24 and gen.cache.shared.eq(0).all()
    assert sorted(gen.cache.free_pages.tolist()) == list(range(24))


def test_beam_search_without_pages_gives_all_back():
    from kvr_b200 import PagedGenerator
    m = tiny(False, seed=5)
    gen = PagedGenerator(m, n_pages=8, page=16, max_requests=8, chunk=64)
    with pytest.raises(RuntimeError, match="not fit"):
        gen.beam_search(prompts_of([90]), 4, 10)  # six pages and three copies of the last
    assert gen.cache.n_free.item() == 8 and not gen.last and gen.cache.ctx_len.eq(0).all()
    gen.cache.check()  # (what was lost has been told)
    assert len(gen.beam_search(prompts_of([30]), 2, 3)[0]) == 2
