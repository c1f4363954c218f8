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


class Step:
    """A decode step of two requests of three beams as one chain on the device: pages, writes, attention, a sparse MLP,
    logits, selection, reordering.  Nothing is read on the host, so it can be captured."""

    G, K, H, LAYERS = 2, 3, 256, 2

    def __init__(self):
        from kvr_b200 import PagedKVCache
        g = torch.Generator(device=DEV).manual_seed(1)
        n = lambda *s: (torch.randn(*s, device=DEV, generator=g) / s[-1] ** 0.5).half()  # noqa: E731
        self.emb = n(500, self.H) * 16
        self.o = [n(self.H, 4 * 128) for _ in range(self.LAYERS)]
        self.moe = [(n(10, self.H) * 2, n(10, 2 * 72, self.H), n(10, self.H, 72)) for _ in range(self.LAYERS)]
        self.qkv = [n(8 * 128, self.H) for _ in range(self.LAYERS)]
        a = torch.outer(torch.arange(256, device=DEV).float(), 10000.0 ** (-torch.arange(0, 128, 2, device=DEV).float() / 128))
        self.cos, self.sin = torch.cat([a.cos()] * 2, 1), torch.cat([a.sin()] * 2, 1)
        self.cache = PagedKVCache(self.LAYERS, 4, 2, 80, page=8, max_requests=self.G * self.K, max_len=256, dtype=torch.float16)
        i32 = dict(dtype=torch.int32, device=DEV)
        self.rows = torch.tensor([[4, 0, 2], [1, 5, 3]], **i32)
        self.new = torch.ones(self.G * self.K, **i32)
        self.tokens = torch.tensor([[7] * 3, [9] * 3], **i32)   # by beam
        self.scores = torch.tensor([[0.0] + [-float("inf")] * 2] * 2, device=DEV)
        self.by_row = torch.empty(self.G * self.K, **i32)

    def __call__(self):
        from kvr_b200 import kernels as K
        c = self.cache
        # (a beam without a token goes on with token 0: its score keeps it out)
        self.by_row[self.rows.view(-1).long()] = self.tokens.clamp(min=0).view(-1)
        h = self.emb[self.by_row.long()]
        c.begin(self.new, self.G * self.K)
        for i in range(self.LAYERS):
            q, k, v = (h @ self.qkv[i].t()).view(-1, 8, 128).split([4, 2, 2], 1)
            q = c.write(i, q, k, v, self.cos, self.sin)
            h = h + c.attend(i, q).view(-1, 4 * 128) @ self.o[i].t()
            x = torch.nn.functional.rms_norm(h, (self.H,))
            h = h + K.moe_layer(x, *self.moe[i], 3)
        c.commit()
        logits = (torch.nn.functional.rms_norm(h, (self.H,)) @ self.emb.t())[self.rows.view(-1).long()]
        st = K.beam_select(logits, self.scores)
        c.reorder(self.rows, st.next_beams)
        self.tokens.copy_(st.next_tokens)
        self.scores.copy_(st.next_scores)


def test_whole_step_in_a_graph():
    from kvr_b200 import kernels as K
    eager, captured = Step(), Step()
    for s in (eager, captured):
        s()  # (and what a first call sets up)
        s()
    state = lambda s: [s.tokens, s.scores, s.cache.block_table, s.cache.ctx_len, s.cache.shared, s.cache.n_free, s.cache.free_pages,  # noqa: E731
                       s.cache.k, s.cache.v]
    keep = [t.clone() for t in state(captured)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured()
    for t, b in zip(state(captured), keep):
        t.copy_(b)
    for i in range(40):
        eager()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(state(eager), state(captured))), i
    eager.cache.check()
    K.moe_status()
    K.attn_status()
    assert eager.cache.ctx_len.eq(42).all() and eager.scores.isfinite().all()
    held = {p for r in eager.cache.block_table.tolist() for p in r[:6]}
    free = eager.cache.free_pages[:eager.cache.n_free.item()].tolist()
    assert sorted(held | set(free)) == list(range(80)) and len(free) + len(held) == 80
    assert eager.cache.shared.sum().item() == 6 * 6 - len(held)


def test_host_threads_at_once():
    """Threads on one stream and on streams of their own: every call has its own workspace."""
    import threading

    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(2)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g).half()  # noqa: E731
    w = (n(16, 256), n(16, 192, 256) / 16, n(16, 256, 96) / 10)
    xs, logits = [n(t, 256) for t in (1, 5, 40, 128)], [n(6, 5000 + 900 * i) for i in range(4)]
    scores = -torch.rand(2, 3, device=DEV, generator=g)
    want = [(K.moe_layer(x, *w, 4), K.beam_select(z, scores, eos=(1,)).tokens) for x, z in zip(xs, logits)]
    torch.cuda.synchronize()
    bad = []

    def work(i, stream):
        with torch.cuda.stream(stream):
            for _ in range(60):
                y, t = K.moe_layer(xs[i], *w, 4), K.beam_select(logits[i], scores, eos=(1,)).tokens
                if not (torch.equal(y, want[i][0]) and torch.equal(t, want[i][1])):
                    bad.append(i)

    for streams in ([torch.cuda.current_stream()] * 4, [torch.cuda.Stream() for _ in range(4)]):
        threads = [threading.Thread(target=work, args=(i, s)) for i, s in enumerate(streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    torch.cuda.synchronize()
    K.moe_status()
    assert not bad


def test_a_sparse_mlp_that_gave_up_ends_the_step(monkeypatch):
    """A wait that ran out (the self-test's, on the word that the call was given): the step, and what is built on it, raise
    before anything counts as cached; it can be tried again."""
    from kvr_b200 import PagedGenerator
    from kvr_b200 import _native as N
    from kvr_b200 import kernels as K
    m = tiny("norm", seed=6)
    gen = PagedGenerator(m, n_pages=40, page=16, max_requests=6, chunk=64)
    (a,) = gen.add(prompts_of([30]))
    K.moe_status()
    kept = [gen.cache.ctx_len.clone(), gen.cache.n_free.clone(), gen.last[a].clone()]
    real = K.moe_layer

    def gave_up(x, *args, status=None, **kw):
        y = real(x, *args, status=status, **kw)
        word = K._moe_status(x.device) if status is None else status
        N.call("kvr_selftest_bounded_wait", word.data_ptr(), 1000, N.stream())
        return y

    monkeypatch.setattr(K, "moe_layer", gave_up)
    for broken in (lambda: gen.step({a: [5]}), lambda: gen.generate([a], 2), lambda: gen.beam_search(prompts_of([20, 9]), 2, 4),
                   lambda: gen.add(prompts_of([12])), lambda: gen.score(prompts_of([40, 11]))):
        with pytest.raises(N.KvrError, match="gave up"):
            broken()
        now = [gen.cache.ctx_len, gen.cache.n_free, gen.last[a]]
        assert all(torch.equal(x, y) for x, y in zip(kept, now)) and list(gen.last) == [a] and gen.cache.step is None
    K.moe_status()  # (nobody else's word was set)
    monkeypatch.setattr(K, "moe_layer", real)
    text = prompts_of([30])[0]
    assert torch.allclose(gen.step({a: [5]})[a], want_logits(m, text + [5])[-1], rtol=BAR, atol=BAR)


def test_release_of_many_rows_that_share_pages():
    """More rows than one reordering takes, all of them holders of one page."""
    from kvr_b200 import PagedKVCache
    c = PagedKVCache(1, 4, 2, 9010, page=8, max_requests=9000, max_len=24, dtype=torch.float16)
    n = torch.arange(9000, dtype=torch.int32, device=DEV)
    c.block_table[:, 0] = 5                  # rows forked from one prompt
    c.block_table[:, 1] = n + 6
    c.ctx_len.fill_(12)
    c.shared[5] = 8999
    c.free_pages[:10] = torch.tensor([0, 1, 2, 3, 4, 9006, 9007, 9008, 9009, 0], dtype=torch.int32)
    c.n_free.fill_(9)
    c.reorder([[0, 1]], [[0, 1]])            # (nothing changes)
    c.release(range(0, 8998))
    assert c.n_free.item() == 9 + 8998 and c.shared[5].item() == 1 and c.shared.sum().item() == 1
    assert c.free_pages[9:9007].tolist() == list(range(6, 9004))
    c.release([8998, 8999])
    assert sorted(c.free_pages[:c.n_free.item()].tolist()) == list(range(9010)) and c.shared.eq(0).all()
    assert c.ctx_len.eq(0).all() and c.block_table.eq(-1).all()
    c.check()


def test_release_counts_holders_however_rows_came_to_share():
    """kernels.paged_reorder on a cache's own tensors, then release: the other rows' pages stay theirs."""
    from kvr_b200 import PagedKVCache
    from kvr_b200 import kernels as K
    c = PagedKVCache(2, 4, 2, 20, page=16, max_requests=4, max_len=128, dtype=torch.bfloat16)
    c.begin([50, 0, 3, 0], 53)
    c.commit()
    assert c.n_free.item() == 15
    i32 = lambda *x: torch.tensor([x], dtype=torch.int32, device=DEV)  # noqa: E731
    K.paged_reorder(c.block_table, c.ctx_len, c.shared, c.free_pages, c.n_free, i32(0, 1, 3), i32(0, 0, 0), c.k, c.v)
    assert c.n_free.item() == 13 and c.ctx_len.tolist() == [50, 50, 3, 50]
    c.begin([0, 0, 9, 20], 29)               # row 3 writes a page of its own
    c.step = None                            # and the step is given up
    for rows, left in (([1, 2], 15), ([3], 16), ([0], 20)):
        c.release(rows)
        assert c.n_free.item() == left, rows
        held = {p for r, m in zip(c.block_table.tolist(), c.ctx_len.tolist()) for p in r[:-(-m // 16)]}
        assert sorted(held | set(c.free_pages[:left].tolist())) == list(range(20)) and len(held) == 20 - left
        assert c.block_table[rows].eq(-1).all() and c.ctx_len[rows].eq(0).all()
    assert c.shared.eq(0).all()


@pytest.mark.parametrize("sparse", [False, True])
def test_beam_search_keeps_what_its_logits_say(sparse):
    """Every logit that the search used, by the text of its row, is the model's for that text; and the plain search on those
    logits finds the same sequences.  Nothing is close but for ties: a score is off by the log-sum-exp's error and a rounding
    to fp32 a step, 2^-21 + 2^-24 40 + 300 / 256 2^-24 < 4e-6, so where no two of the plain search's candidates lie within
    2e-4 (12 steps, both of them, twice) the order is the same."""
    from kvr_b200 import PagedGenerator
    m = tiny("norm", seed=8, experts=5, top_k=5) if sparse else tiny(False, seed=8)  # (all experts: no choice is close)
    k, steps, eos = 4, 12, 7
    prompts = prompts_of([40, 1, 64, 133, 17, 90], 12)
    gen = PagedGenerator(m, n_pages=90, page=16, max_requests=26, chunk=64)
    text, seen = [[] for _ in range(26)], {}
    step, reorder = gen.step, gen.cache.reorder

    def noted_step(new):
        out = step(new)
        for b, ids in new.items():
            text[b] += ids
            seen[tuple(text[b])] = out[b].clone()
        return out

    def noted_reorder(rows, parents):
        old = [list(t) for t in text]
        for g, ps in zip(rows, parents):
            for b, p in zip(g, ps):
                text[b] = list(old[g[p]]) if p >= 0 else []
        return reorder(rows, parents)

    gen.step, gen.cache.reorder = noted_step, noted_reorder
    got = gen.beam_search(prompts, k, steps, eos=eos)
    compared = 0
    for p, found in zip(prompts, got):
        for t in [t for t in seen if t[:len(p)] == tuple(p)]:
            # What a hidden state is off by, e of its size, goes through the rows of lm_head as the state itself does, so logits
            # are off by e of their spread: sqrt(256) 0.2 = 3.2 here, not one.  (e: some ten roundings to fp16 on the way, each
            # 2^-11 / sqrt(3) of an element at most, 9e-4 rms; the largest of 50 texts' 300 logits is 4.3 times that, and
            # two such computations differ by 1.4 times that: 5.4e-3, a quarter of the bar.)
            want = want_logits(m, list(t))[-1]
            assert ((seen[t] - want).abs() <= BAR * (want.std() + want.abs())).all(), (seen[t] - want).abs().max()
        beams, ended, gap = [(0.0, [])], [], math.inf
        for t in range(1, steps + 1):
            cand = []
            for s, q in beams:
                lp = seen[tuple(p + q)].double().log_softmax(-1)
                top = lp.topk(2 * k + 1)
                cand += [(s + v, q + [i]) for v, i in zip(top.values.tolist(), top.indices.tolist())]
            cand.sort(key=lambda c: -c[0])
            gap = min([gap] + [a[0] - b[0] for a, b in zip(cand[:2 * k], cand[1:2 * k + 1])])
            if gap <= 2e-4:
                break  # (from here on the beams may be others, whose texts nobody has seen)
            ended = sorted(ended + [(s / t, q) for s, q in cand[:k] if q[-1] == eos], key=lambda e: -e[0])[:k]
            beams = [(s, q) for s, q in cand if q[-1] != eos][:k]
            if len(ended) == k and ended[-1][0] >= beams[0][0] / t:
                beams = []
                break
        if gap <= 2e-4:
            continue
        want = sorted(ended + [(s / len(q), q) for s, q in beams], key=lambda e: -e[0])[:k]
        gap = min([math.inf] + [a[0] - b[0] for a, b in zip(want, want[1:])])
        if gap > 1e-5:
            assert [q for q, _ in found] == [q for _, q in want]
            assert all(abs(a - b) < 1e-4 for (_, a), (b, _) in zip(found, want))
            compared += 1
    assert compared >= 2, compared


def test_host_threads_first_calls_at_once():
    """As above, from the first call on (no status word, no kernel attributes of a warm-up), and a thread that raises is seen."""
    import concurrent.futures

    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(2)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g).half()  # noqa: E731
    w = (n(16, 256), n(16, 192, 256) / 16, n(16, 256, 96) / 10)
    xs, logits = [n(t, 256) for t in (1, 5, 40, 128)], [n(6, 5000 + 900 * i) for i in range(4)]
    scores = -torch.rand(2, 3, device=DEV, generator=g)
    torch.cuda.synchronize()
    K._MOE_STATUS.clear()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = [(K.moe_layer(xs[i], *w, 4), K.beam_select(logits[i], scores, eos=(1,)).tokens) for _ in range(60)]
            torch.cuda.current_stream().synchronize()
            return out

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        got = [f.result() for f in [pool.submit(work, i) for i in range(4)]]
    assert len(K._MOE_STATUS) == 1
    K.moe_status()
    for i, runs in enumerate(got):
        assert len(runs) == 60
        y, t = K.moe_layer(xs[i], *w, 4), K.beam_select(logits[i], scores, eos=(1,)).tokens
        assert all(torch.equal(a, y) and torch.equal(b, t) for a, b in runs)
