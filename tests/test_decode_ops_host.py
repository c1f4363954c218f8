"""CPU checks of beam selection, reordering and the sparse MLP: what the Python
calls hand to the native ones, what both refuse, and the host logic of
PagedKVCache.reorder and PagedGenerator.beam_search."""
import numpy as np
import pytest
import torch

from oracle import decode_ref as R

PTR = 4096  # a pointer that no refused call follows


@pytest.fixture
def native(monkeypatch):
    """The calls that would reach a GPU, recorded: name -> arguments of the last."""
    from kvr_b200 import _native as N
    from kvr_b200 import kernels as K
    seen, real = {}, N.call

    def call(name, *args):
        if name.endswith("_bytes"):
            return real(name, *args)
        seen[name] = args
        return 0

    monkeypatch.setattr(K, "call", call)
    monkeypatch.setattr(K, "_on_current_gpu", lambda *t: None)
    monkeypatch.setattr(K, "_moe_status", lambda device: torch.zeros(256, dtype=torch.uint8))
    monkeypatch.setattr(K, "stream", lambda: 0)
    return seen


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


# ---------------------------------------------------------------- select --


def test_select_hands_on_strides_and_ends(native):
    from kvr_b200 import kernels as K
    wide = torch.zeros(6, 100)
    st = K.beam_select(wide[:, :77], torch.zeros(2, 3), eos=[5, 9])
    a = native["kvr_beam_select"]
    assert a[1:6] == (0, 100, 2, 3, 77) and a[7] == 9 and a[9] == 2 and list(a[8])[:2] == [5, 9]
    assert st.scores.shape == st.beams.shape == st.tokens.shape == (2, 9) and st.next_beams.shape == (2, 3)
    assert st.scores.dtype is torch.float32 and st.tokens.dtype is torch.int32
    # rows that all beams of a request share
    K.beam_select(torch.zeros(1, 77, dtype=torch.bfloat16).expand(3, 77), torch.zeros(1, 3), n=4)
    assert native["kvr_beam_select"][1:6] == (2, 0, 1, 3, 77) and native["kvr_beam_select"][7] == 4
    K.beam_select(torch.zeros(2, 3, 50), torch.zeros(2, 3))
    assert native["kvr_beam_select"][2] == 50


def test_select_refusals(native):
    from kvr_b200 import kernels as K
    x, s = torch.zeros(6, 50), torch.zeros(2, 3)
    for bad in (dict(logits=x[:5]), dict(scores=torch.zeros(6)), dict(n=2), dict(logits=x[:, :0]), dict(logits=torch.zeros(50)),
                dict(eos=(1 << 31,)), dict(eos=[-1])):
        with pytest.raises(ValueError):
            K.beam_select(**{"logits": x, "scores": s, **bad})
    with pytest.raises(TypeError):
        K.beam_select(x, s.double())
    with pytest.raises(TypeError):
        K.beam_select(x.double(), s)
    assert not native


def select_call(**kw):
    from kvr_b200 import _native as N
    a = dict(logits=PTR, dtype=0, stride=50, batch=2, beams=3, vocab=50, cum=PTR, n=6, eos=None, n_eos=0, out=PTR, ws=PTR,
             ws_bytes=1 << 20)
    a.update(kw)
    return N.call("kvr_beam_select", a["logits"], a["dtype"], a["stride"], a["batch"], a["beams"], a["vocab"], a["cum"], a["n"],
                  a["eos"], a["n_eos"], a["out"], PTR, PTR, PTR, PTR, PTR, a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=7), "dtype"), (dict(n=2), "shape"), (dict(vocab=0), "shape"), (dict(beams=0), "shape"), (dict(beams=33, n=40), "at most"),
    (dict(n=129), "at most"), (dict(n_eos=9), "at most"), (dict(logits=None), "null"), (dict(ws=None), "null"),
    (dict(n_eos=1), "null"), (dict(ws_bytes=8), "workspace"), (dict(logits=PTR + 2), "aligned"), (dict(stride=-50), "stride"),
    (dict(batch=-1), "shape")])
def test_select_c_refusals(kw, match):
    from kvr_b200._native import KvrError
    with pytest.raises(KvrError, match=match):
        select_call(**kw)


def test_no_requests_is_no_call():
    assert select_call(batch=0, logits=None) == 0


# --------------------------------------------------------------- reorder --


def reorder_args():
    k = torch.zeros(2, 9, 16, 2, 128, dtype=torch.float16)
    return dict(block_table=torch.zeros(4, 6, dtype=torch.int32), ctx_len=i32(0, 0, 0, 0), shared=torch.zeros(9, dtype=torch.int32),
                free_pages=torch.zeros(9, dtype=torch.int32), n_free=i32(0), rows=i32(0, 1).view(1, 2), parents=i32(0, 0).view(1, 2),
                k_pages=k, v_pages=k.clone())


def test_reorder_hands_on_layouts(native):
    from kvr_b200 import kernels as K
    a = reorder_args()
    K.paged_reorder(**a)
    c = native["kvr_paged_reorder"]
    assert c[1:4] == (6, 4, 6) and c[5] == 16 and c[7] == 9 and c[13:15] == (1, 2)
    assert c[17:24] == (1, 2, 2, 128, 9 * 16 * 256, 16 * 256, 256)
    kv = torch.zeros(9, 2, 16, 2, 128, dtype=torch.float16)  # one layer, K and V of a page in one tensor
    K.paged_reorder(**{**a, "k_pages": kv[:, 0], "v_pages": kv[:, 1]})
    assert native["kvr_paged_reorder"][17:24] == (1, 1, 2, 128, 0, 2 * 16 * 256, 256)


def test_reorder_refusals(native):
    from kvr_b200 import kernels as K
    a = reorder_args()
    k = a["k_pages"]
    for bad in (dict(v_pages=k[:1]), dict(v_pages=k.bfloat16()), dict(k_pages=k[..., :64]), dict(k_pages=k.transpose(2, 3)),
                dict(shared=torch.zeros(8, dtype=torch.int32)), dict(n_free=i32(1, 2)), dict(ctx_len=i32(0, 0, 0, 0, 0)),
                dict(block_table=torch.zeros(1, 6, dtype=torch.int32).expand(4, 6)), dict(rows=torch.zeros(1, 0, dtype=torch.int32),
                                                                                        parents=torch.zeros(1, 0, dtype=torch.int32))):
        with pytest.raises(ValueError):
            K.paged_reorder(**{**a, **bad})
    for bad in (dict(rows=a["rows"].long()), dict(parents=i32(0, 0)), dict(parents=i32(0, 0, 0).view(1, 3)),
                dict(shared=a["shared"].long()), dict(block_table=a["block_table"].long())):
        with pytest.raises(TypeError):
            K.paged_reorder(**{**a, **bad})
    assert not native


def reorder_call(**kw):
    from kvr_b200 import _native as N
    a = dict(table=PTR, stride=6, rows=4, width=6, ctx=PTR, page=16, shared=PTR, pages=9, free=PTR, cap=9, n_free=PTR, r=PTR, p=PTR,
             groups=1, beams=2, k=PTR, v=PTR, dtype=1, layers=2, n_kv=2, d=128, ls=9 * 16 * 256, ps=16 * 256, ts=256, info=PTR,
             ws=PTR, ws_bytes=1 << 20)
    a.update(kw)
    return N.call("kvr_paged_reorder", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(beams=0), "groups"), (dict(beams=33), "at most"), (dict(groups=2000, beams=4), "at most"), (dict(rows=1 << 17), "at most"),
    (dict(page=0), "page"), (dict(width=0), "table"), (dict(stride=5), "table"), (dict(pages=0), "pool"), (dict(cap=9, free=None), "free"),
    (dict(d=64), "head_dim"), (dict(dtype=0), "fp16"), (dict(k=None), "null"), (dict(info=None), "null"), (dict(r=None), "null"),
    (dict(ts=128), "contiguous"), (dict(ps=16 * 256 + 4), "aligned"), (dict(v=PTR + 8), "aligned"), (dict(ws_bytes=16), "workspace"),
    (dict(layers=0), "contiguous"), (dict(width=1 << 20, stride=1 << 20, groups=1000, ws_bytes=1 << 40), "too long")])
def test_reorder_c_refusals(kw, match):
    from kvr_b200._native import KvrError
    with pytest.raises(KvrError, match=match):
        reorder_call(**kw)


def cache():
    from kvr_b200 import PagedKVCache
    return PagedKVCache(1, 8, 2, 10, page=16, max_requests=4, max_len=64, device="cpu")


def test_reorder_refuses_pages_beyond_its_arithmetic():
    from kvr_b200._native import KvrError
    with pytest.raises(KvrError, match="32 GB"):
        reorder_call(page=1 << 20, n_kv=128, ts=128 * 128, ps=1 << 37, ls=1 << 42)


def test_cache_reorder_refusals(native):
    c = cache()
    for rows, parents in (([[0, 0]], [[0, 0]]), ([[0, 1], [2]], [[0, 0], [0]]), ([[0, 4]], [[0, 0]]), ([[-1, 0]], [[0, 0]]),
                          ([], []), ([[0, 1]], [[0, 2]]), ([[0, 1]], [[0, -2]])):
        with pytest.raises(ValueError):
            c.reorder(rows, parents)
    with pytest.raises(TypeError):
        c.reorder([[0, 1]], [[0, 0], [0, 0]])
    c.step = object()
    with pytest.raises(RuntimeError, match="commit"):
        c.reorder([[0, 1]], [[0, 0]])
    assert "kvr_paged_reorder" not in native


def test_release_after_sharing_counts_holders(native):
    """Pages that another row holds too must not go back to the list: release then empties rows by reorder."""
    c = cache()
    c.reorder([[0, 1, 2]], [[0, 0, 0]])
    native.clear()
    c.release([2, 0])
    assert native["kvr_paged_reorder"][13:15] == (2, 1)
    native.clear()
    c.release([])
    assert not native


# ------------------------------------------------------------------- moe --


def moe_args(T=3, H=64, I=24, E=4, dt=torch.bfloat16):
    return dict(x=torch.zeros(T, H, dtype=dt), router=torch.zeros(E, H, dtype=dt), gate_up=torch.zeros(E, 2 * I, H, dtype=dt),
                down=torch.zeros(E, H, I, dtype=dt), top_k=2)


def test_moe_hands_on_strides(native):
    from kvr_b200 import kernels as K
    a = moe_args()
    wide = torch.zeros(3, 128, dtype=torch.bfloat16)
    K.moe_layer(**{**a, "x": wide[:, :64], "down": torch.zeros(4, 64, 40, dtype=torch.bfloat16)[:, :, :24]}, norm_topk=False, scale=2.0)
    c = native["kvr_moe_layer"]
    assert c[1:5] == (2, 3, 64, 128) and c[6] == 64 and c[8:10] == (48 * 64, 64) and c[11:13] == (64 * 40, 40)
    assert c[13:18] == (4, 24, 2, 0, 2.0)


def test_moe_refusals(native):
    from kvr_b200 import kernels as K
    a = moe_args()
    for bad in (dict(router=a["router"][:3]), dict(gate_up=a["gate_up"][:, :40]), dict(down=a["down"][:3]), dict(x=a["x"][0]),
                dict(gate_up=a["gate_up"].transpose(1, 2).contiguous().transpose(1, 2)), dict(out=torch.zeros(3, 64)),
                dict(router=torch.zeros(64, 4, dtype=torch.bfloat16).t())):
        with pytest.raises(ValueError):
            K.moe_layer(**{**a, **bad})
    for bad in (dict(x=a["x"].half()), dict(down=a["down"].float())):
        with pytest.raises(TypeError):
            K.moe_layer(**{**a, **bad})
    assert not native


def moe_call(**kw):
    from kvr_b200 import _native as N
    a = dict(x=PTR, dtype=2, T=3, H=64, xs=64, router=PTR, rs=64, gu=PTR, ge=48 * 64, gr=64, down=PTR, de=64 * 24, dr=24, E=4, I=24,
             k=2, norm=1, scale=1.0, y=2 * PTR, ids=PTR, w=PTR, ws=PTR, ws_bytes=1 << 24, status=PTR)
    a.update(kw)
    return N.call("kvr_moe_layer", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(T=129), "at most"), (dict(E=513), "at most"), (dict(E=32, k=17), "at most"), (dict(k=5), "shape"), (dict(k=0), "shape"),
    (dict(dtype=0), "fp16"), (dict(H=60, xs=64), "multiples of 8"), (dict(I=20), "multiples of 8"), (dict(x=None), "null"), (dict(status=None), "null"),
    (dict(xs=32), "share"), (dict(ge=40 * 64), "share"), (dict(dr=16), "share"), (dict(xs=68), "aligned"), (dict(down=PTR + 8), "aligned"),
    (dict(ws=PTR + 16), "aligned"), (dict(ws_bytes=64), "workspace"), (dict(y=PTR + 64), "lie in x"), (dict(y=1 << 20, gu=(1 << 20) - 512), "weights"), (dict(y=1 << 20, router=(1 << 20) + 128), "weights"), (dict(H=1 << 17, xs=1 << 17, rs=1 << 17,
                                                                                                              gr=1 << 17, ge=1 << 24), "too large")])
def test_moe_c_refusals(kw, match):
    from kvr_b200._native import KvrError
    with pytest.raises(KvrError, match=match):
        moe_call(**kw)


def test_moe_refuses_rows_beyond_its_arithmetic():
    from kvr_b200._native import KvrError
    with pytest.raises(KvrError, match="too far apart"):
        moe_call(xs=(1 << 28) + 8)


def test_no_tokens_is_no_call():
    assert moe_call(T=0, x=None) == 0


def test_operators_refuse_cpu_tensors(monkeypatch):
    from kvr_b200 import kernels as K
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    for f, a in ((K.paged_reorder, reorder_args()), (K.moe_layer, moe_args()), (K.beam_select, dict(logits=torch.zeros(3, 9), scores=torch.zeros(1, 3)))):
        with pytest.raises(ValueError, match="CUDA"):
            f(**a)


def tiny_moe(**kw):
    import transformers as T
    torch.manual_seed(0)
    cfg = T.Qwen3MoeConfig(**{"vocab_size": 50, "hidden_size": 64, "intermediate_size": 64, "moe_intermediate_size": 24, "num_hidden_layers": 1,
                              "num_attention_heads": 2, "num_key_value_heads": 1, "head_dim": 128, "num_experts": 4, "num_experts_per_tok": 2,
                              "max_position_embeddings": 64, **kw})
    return T.Qwen3MoeForCausalLM(cfg).half().eval()


def test_generator_takes_sparse_models_it_can_compute(native):
    from kvr_b200 import PagedGenerator
    from kvr_b200 import kvr_paged as P
    m = tiny_moe()
    gen = PagedGenerator(m, n_pages=4, page=16, max_requests=1, max_len=40)
    x = torch.zeros(5, 64, dtype=torch.float16)
    gen._mlp(m.model.layers[0].mlp, x)
    assert native["kvr_moe_layer"][13:17] == (4, 24, 2, 0)
    native.clear()
    y = gen._mlp(m.model.layers[0].mlp, torch.randn(129, 64).half())  # more tokens: the model's own
    assert not native and y.shape == (129, 64)
    with pytest.raises(NotImplementedError, match="gelu"):
        PagedGenerator(tiny_moe(hidden_act="gelu"), n_pages=4, page=16, max_requests=1, max_len=40)
    m.model.layers[0].mlp.shared_expert = torch.nn.Linear(64, 64)
    with pytest.raises(NotImplementedError, match="shared_expert"):
        P._sparse(m.model.layers[0].mlp)


# ----------------------------------------------------------- beam search --


class Toy:
    """A language model of a few tokens, whose logits depend on the whole text."""

    def __init__(self, vocab, seed):
        self.vocab, self.seed = vocab, seed

    def logits(self, text):
        return 2 * np.random.default_rng([self.seed, len(text)] + list(text)).standard_normal(self.vocab).astype(np.float32)


def toy_generator(toy, rows, monkeypatch):
    """A PagedGenerator whose cache holds texts, and whose kernels are their specification."""
    from kvr_b200 import kernels as K
    from kvr_b200 import PagedGenerator
    gen = object.__new__(PagedGenerator)

    class Cache:
        max_requests = rows

        def __init__(self):
            self.text = [[] for _ in range(rows)]

        def reorder(self, r, parents):
            old = [list(t) for t in self.text]
            for g, ps in zip(r, parents):
                for b, p in zip(g, ps):
                    self.text[b] = list(old[g[p]]) if p >= 0 else []

        def check(self):
            pass

        def release(self, r):
            for b in r:
                self.text[b] = []

    gen.cache, gen.last, gen.device, gen.chunk = Cache(), {}, torch.device("cpu"), 3

    def step(new):
        for b, t in new.items():
            gen.cache.text[b] += t
        out = {b: torch.tensor(toy.logits(gen.cache.text[b])) for b in new}
        gen.last.update(out)
        return out

    def select(logits, scores, n=None, eos=()):
        B, k = scores.shape
        x = logits.reshape(B, k, -1).numpy()
        want = R.beam_select(x, scores.numpy(), k * (1 + len(eos)) if n is None else n, eos)
        st = K.BeamStep()
        for f, v in want.items():
            setattr(st, f, torch.tensor(v, dtype=torch.float32 if "scores" in f else torch.int32))
        return st

    gen.step = step
    monkeypatch.setattr(K, "beam_select", select)
    return gen


def plain_beams(toy, prompt, k, steps, eos, penalty):
    beams, ended = [(0.0, [])], []
    for t in range(1, steps + 1):
        cand = []
        for s, q in beams:
            x = toy.logits(prompt + q).astype(np.float64)
            lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
            cand += [(s + lp[v], q + [v]) for v in range(toy.vocab)]
        cand.sort(key=lambda c: -c[0])
        ended += [(s / t ** penalty, q) for s, q in cand[:k] if q[-1] in eos]
        ended = sorted(ended, key=lambda e: -e[0])[:k]
        beams = [(s, q) for s, q in cand if q[-1] not in eos][:k]
        if not beams or (len(ended) == k and ended[-1][0] >= beams[0][0] / t ** penalty):
            return ended
    ended += [(s / len(q) ** penalty, q) for s, q in beams]
    return sorted(ended, key=lambda e: -e[0])[:k]


@pytest.mark.parametrize("k,steps,eos,penalty", [(1, 5, (), 1.0), (3, 6, (2,), 1.0), (4, 7, (0, 5), 0.6), (2, 1, (1,), 1.0), (5, 9, (3,), 2.0),
                                                 (3, 4, tuple(range(6)), 1.0)])
def test_beam_search_matches_the_plain_one(k, steps, eos, penalty, monkeypatch):
    toy = Toy(6 if len(eos) < 6 else 7, 11 + k)
    prompts = [[1, 2, 3, 4], [5], [0, 0]]
    gen = toy_generator(toy, 3 * k + 2, monkeypatch)
    gen.last[1] = torch.zeros(6)  # a row in use is left alone
    gen.cache.text[1] = [9]
    got = gen.beam_search(prompts, k, steps, eos=eos, length_penalty=penalty)
    for p, found in zip(prompts, got):
        want = plain_beams(toy, p, k, steps, eos, penalty)
        assert [q for q, _ in found] == [q for _, q in want], p
        assert np.allclose([s for _, s in found], [s for s, _ in want], rtol=0, atol=1e-5)
    assert list(gen.last) == [1] and gen.cache.text[1] == [9] and sum(map(len, gen.cache.text)) == 1


def test_beam_search_refusals_and_cleanup(monkeypatch):
    gen = toy_generator(Toy(6, 1), 6, monkeypatch)
    with pytest.raises(RuntimeError, match="free rows"):
        gen.beam_search([[1], [2]], 4, 3)
    for bad in (dict(n_beams=0), dict(max_new_tokens=0)):
        with pytest.raises(ValueError):
            gen.beam_search([[1]], **{"n_beams": 2, "max_new_tokens": 2, **bad})
    with pytest.raises(ValueError, match="at least one"):
        gen.beam_search([[1], []], 2, 3)
    assert gen.beam_search([], 2, 3) == [] and not gen.last

    def fails():
        raise RuntimeError("committed steps did not fit")
    gen.cache.check = fails
    with pytest.raises(RuntimeError, match="not fit"):
        gen.beam_search([[1], [2]], 2, 3)
    assert not gen.last and not any(gen.cache.text)


@pytest.mark.parametrize("tokens,experts,top_k,hidden,inter,router,own", [
    (1, 4, 2, 16, 8, torch.bfloat16, True), (128, 512, 16, 16, 8, torch.bfloat16, True),
    (129, 4, 2, 16, 8, torch.bfloat16, False), (2, 513, 2, 16, 8, torch.bfloat16, False), (2, 32, 17, 16, 8, torch.bfloat16, False),
    (2, 4, 2, 20, 8, torch.bfloat16, False), (2, 4, 2, 16, 12, torch.bfloat16, False), (2, 4, 2, 16, 8, torch.float32, False)])
def test_sparse_mlps_that_the_call_does_not_take_stay_the_models(native, tokens, experts, top_k, hidden, inter, router, own):
    from kvr_b200.kvr_paged import PagedGenerator

    class Sparse(torch.nn.Module):
        def __init__(self):
            super().__init__()
            zeros = lambda *s, dtype=torch.bfloat16: torch.nn.Parameter(torch.zeros(*s, dtype=dtype), requires_grad=False)
            self.gate, self.experts = torch.nn.Module(), torch.nn.Module()
            self.gate.weight, self.gate.top_k = zeros(experts, hidden, dtype=router), top_k
            self.experts.gate_up_proj = zeros(experts, 2 * inter, hidden)
            self.experts.down_proj = zeros(experts, hidden, inter)

        def forward(self, x):
            return x + 1

    y = PagedGenerator._mlp(Sparse(), torch.zeros(tokens, hidden, dtype=torch.bfloat16))
    assert y.shape == (tokens, hidden) and ("kvr_moe_layer" in native) == own
    assert own or bool((y == 1).all())


# ------------------------------------------- last pages that rows share --


def whole_pool(table, ctx, shared, free, n_free, page):
    """Each page of the pool is held or free, once; counts are what the rows hold."""
    held = [int(p) for r, c in zip(table, ctx) for p in r[:-(-int(c) // page)] if p >= 0]
    assert sorted(set(held) | {int(p) for p in free[:n_free]}) == list(range(len(shared))) and n_free + len(set(held)) == len(shared)
    assert [int(x) for x in shared] == [max(held.count(p) - 1, 0) for p in range(len(shared))]


# rows 0, 1 and 2 hold page 1, which is not full, behind page 0; row 3 has pages of its own
SHARED_LAST = [([[0, 1, 2]], [[0, 1, 2]]), ([[0, 1, 2]], [[0, 1, 1]]), ([[2, 3, 1, 0]], [[0, 2, 2, 3]]), ([[0], [1], [2]], [[0]] * 3),
               ([[1], [2]], [[0]] * 2), ([[0, 3], [1, 2]], [[0, 0], [1, 0]]), ([[0, 3], [1, 2]], [[1, 1], [1, 0]]),
               ([[1, 2], [3, 0]], [[-1, 1], [0, -1]]), ([[3], [2]], [[0]] * 2)]


def shared_last(free):
    table = np.array([[0, 1, -1], [0, 1, -1], [0, 1, -1], [2, 3, -1]], np.int32)
    shared = np.array([2, 2] + [0] * (2 + free), np.int32)
    return table, np.array([20, 20, 25, 18], np.int32), shared, np.array(list(range(4, 4 + free)) + [0] * 4, np.int32), free


@pytest.mark.parametrize("free", [0, 1, 8])
@pytest.mark.parametrize("rows,parents", SHARED_LAST)
def test_no_shared_last_page_is_lost(rows, parents, free):
    """The first place that a last page of several rows falls to keeps it, unless a row outside of the call has it."""
    table, ctx, shared, free_pages, n = shared_last(free)
    w = R.reorder(table, ctx, shared, free_pages, n, rows, parents, 16)
    whole_pool(w["table"], w["ctx"], w["shared"], w["free"], w["n_free"], 16)
    last = [w["table"][r, 1] for r in range(4) if w["ctx"][r] > 16]
    named = {r for g in rows for r in g}
    if named >= {0, 1, 2}:
        assert len(set(last)) == len(last)  # nobody writes where another reads
    else:  # row 0 goes on with it: the others do not
        assert w["table"][0, 1] == 1 and 1 not in [w["table"][r, 1] for r in named]


# ---------------------------------------------------- the status word --


def test_status_word_is_seen_when_it_is_zeroed(monkeypatch):
    """Two host threads' first calls: one word for both, that none of them gets before its zeros are there."""
    import threading
    from kvr_b200 import kernels as K
    entered, go, got = threading.Event(), threading.Event(), []

    class Stream:
        def synchronize(self):
            entered.set()
            assert go.wait(20)

    monkeypatch.setattr(K, "_MOE_STATUS", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    threads = [threading.Thread(target=lambda: got.append(K._moe_status(torch.device("cpu")))) for _ in range(2)]
    threads[0].start()
    assert entered.wait(20)
    threads[1].start()
    threads[1].join(0.5)
    early = list(got)
    go.set()
    for t in threads:
        t.join()
    assert not early and got[0] is got[1] and K._moe_status(torch.device("cpu")) is got[0]


# --------------------------------------------- release where rows share --


def test_release_of_many_rows_after_sharing(native, monkeypatch):
    """As many rows as the cache has, of tables of any width: in calls of what one of them takes."""
    from kvr_b200 import PagedKVCache
    from kvr_b200 import kernels as K
    calls = []
    monkeypatch.setattr(K, "paged_reorder", lambda table, ctx, shared, free, n_free, rows, parents, k, v: (
        calls.append((rows.clone(), parents.clone())), torch.zeros(4, dtype=torch.int32))[1])
    c = PagedKVCache(1, 8, 2, 10, page=16, max_requests=9000, max_len=32, device="cpu")
    c.reorder([[0, 1]], [[0, 0]])
    calls.clear()
    c.release(range(8999, -1, -1))
    assert [r.shape[1] for r, _ in calls] == [1] * len(calls) and max(len(r) for r, _ in calls) <= 4096
    assert torch.cat([r[:, 0] for r, _ in calls]).tolist() == list(range(8999, -1, -1))
    assert all(p.eq(-1).all() for _, p in calls)
    wide = PagedKVCache(1, 8, 2, 10, page=8, max_requests=1200, max_len=1 << 23, device="cpu")  # 2^20 columns
    wide.reorder([[0, 1]], [[0, 0]])
    calls.clear()
    wide.release(range(1200))
    assert sum(len(r) for r, _ in calls) == 1200 and max(len(r) for r, _ in calls) * (1 << 20) < 1 << 30


# ------------------------------------------------- limits of beam search --


@pytest.mark.parametrize("kw,match", [
    (dict(n_beams=33), "32 beams"), (dict(eos=tuple(range(9))), "8 ends"), (dict(n_beams=32, eos=(1, 2, 3, 4)), "128"),
    (dict(n_beams=16, eos=tuple(range(8))), "128"), (dict(eos=(-1,)), "token ids"), (dict(eos=1 << 31), "token ids"),
    (dict(prompts=[[1]] * 2049, n_beams=2), "4096")])
def test_beam_search_refuses_before_it_computes(kw, match, monkeypatch):
    """What the selection or the reordering would refuse is refused before the prompts are computed."""
    gen = toy_generator(Toy(6, 1), 5000, monkeypatch)
    gen.step = lambda new: pytest.fail("computed a step")
    with pytest.raises(ValueError, match=match):
        gen.beam_search(**{"prompts": [[1, 2]], "n_beams": 2, "max_new_tokens": 3, **kw})
    assert not gen.last


def test_beam_search_counts_an_end_once(monkeypatch):
    gen = toy_generator(Toy(6, 3), 40, monkeypatch)
    once = gen.beam_search([[1, 2]], 32, 2, eos=[4, 1])
    assert gen.beam_search([[1, 2]], 32, 2, eos=[4, 1, 4, 1, 1, 4, 4, 4, 4]) == once


def test_select_takes_ends_by_value(native):
    """Ends in objects that change between calls (an element of a tensor): each call's own values."""
    from kvr_b200 import kernels as K
    end = torch.tensor(5)
    for t in (5, 9, 2):
        end.fill_(t)
        K.beam_select(torch.zeros(3, 50), torch.zeros(1, 3), eos=[end])
        assert list(native["kvr_beam_select"][8]) == [t]
    K.beam_select(torch.zeros(3, 50), torch.zeros(1, 3), eos=np.array([7, 8]))
    assert list(native["kvr_beam_select"][8]) == [7, 8] and native["kvr_beam_select"][7] == 9


def test_routing_does_not_keep_the_workspace(native):
    """ids and weights that a caller collects over layers and steps hold their own bytes, not a call's h and partial rows."""
    from kvr_b200 import kernels as K
    a = moe_args(T=100, H=512, I=256, E=8)
    y, ids, w = K.moe_layer(**a, return_routing=True)
    assert ids.shape == w.shape == (100, 2) and ids.dtype is torch.int32 and w.dtype is torch.float32
    for t in (ids, w):
        assert t.untyped_storage().nbytes() <= 100 * 2 * 8 + 256
    c = native["kvr_moe_layer"]
    assert c[19] == ids.data_ptr() and c[20] == w.data_ptr() and c[21] % 64 == 0 and c[22] > 100 * 2 * 256 * 4


@pytest.mark.parametrize("change,own", [
    (None, True), ("wide rows", True), ("experts fp32", False), ("down fp32", False), ("gate_up off", False), ("down off", False),
    ("router off", False), ("router 36 apart", False), ("down transposed", False), ("experts expanded", False), ("all fp32", False)])
def test_sparse_mlps_laid_out_otherwise_stay_the_models(native, change, own):
    """Types, places in memory and strides that the call refuses: the model's own module, no error."""
    from kvr_b200.kvr_paged import PagedGenerator
    E, H, I = 4, 32, 24
    bf = torch.bfloat16
    off = lambda *s: torch.zeros(int(np.prod(s)) + 1, dtype=bf)[1:].view(*s)  # noqa: E731

    class Sparse(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate, self.experts = torch.nn.Module(), torch.nn.Module()
            self.gate.top_k = 2
            gate, gu, down = torch.zeros(E, H, dtype=bf), torch.zeros(E, 2 * I, H, dtype=bf), torch.zeros(E, H, I, dtype=bf)
            if change == "wide rows":
                down = torch.zeros(E, H, 40, dtype=bf)[:, :, :I]
            elif change == "experts fp32":
                gu, down = gu.float(), down.float()
            elif change == "all fp32":
                gate, gu, down = gate.float(), gu.float(), down.float()
            elif change == "down fp32":
                down = down.float()
            elif change == "gate_up off":
                gu = off(E, 2 * I, H)
            elif change == "down off":
                down = off(E, H, I)
            elif change == "router off":
                gate = off(E, H)
            elif change == "router 36 apart":
                gate = torch.zeros(E, 36, dtype=bf)[:, :H]
            elif change == "down transposed":
                down = torch.zeros(E, I, H, dtype=bf).transpose(1, 2)
            elif change == "experts expanded":
                gu = gu[:1].expand(E, -1, -1)
            p = lambda t: torch.nn.Parameter(t, requires_grad=False)  # noqa: E731
            self.gate.weight, self.experts.gate_up_proj, self.experts.down_proj = p(gate), p(gu), p(down)

        def forward(self, x):
            return x + 1

    x = torch.zeros(3, H, dtype=torch.float32 if change == "all fp32" else bf)
    y = PagedGenerator._mlp(Sparse(), x)
    assert y.shape == (3, H) and ("kvr_moe_layer" in native) == own
    assert own or bool((y == 1).all())
