"""CPU checks of the paged-cache operators and classes: what the Python calls
hand to the native ones, what they refuse, and the host logic of PagedKVCache
and PagedGenerator."""
import pytest
import torch


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


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
    monkeypatch.setattr(K, "ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(K, "_on_gpu", lambda *t: None)
    monkeypatch.setattr(K, "stream", lambda: 0)
    monkeypatch.setattr(K, "_attn_workspace", lambda device: (256, 1 << 30, 0))
    return seen


def test_block_tables_whose_rows_share_memory_are_refused(native):
    """A table of one row expanded to several has the stride 0: the kernels would
    follow another stride past its storage."""
    from kvr_b200 import kernels as K
    pool = torch.zeros(4, 16, 2, 128, dtype=torch.float16)
    q = torch.zeros(3, 8, 128, dtype=torch.float16)
    plan = K.attn_plan(i32(0, 1, 2, 3), 3, 8, 2, kv_len=i32(5, 5, 5))
    flat = torch.zeros(20, dtype=torch.int32)
    for table in (flat[:4].expand(3, 4), flat.as_strided((3, 4), (2, 1))):
        with pytest.raises(ValueError, match="share memory"):
            K.paged_map(i32(5, 5, 5), i32(1, 1, 1), table, i32(0, 1, 2), i32(3), 16, 3)
        with pytest.raises(ValueError, match="share memory"):
            K.paged_attn(q, pool, pool, table, plan)
    assert "kvr_paged_map" not in native and "kvr_paged_attn" not in native
    # the stride of a view is handed on; that of a single row means nothing
    K.paged_map(i32(5, 5, 5), i32(1, 1, 1), flat.as_strided((3, 4), (6, 1)), i32(0, 1, 2), i32(3), 16, 3)
    assert native["kvr_paged_map"][6:8] == (6, 4)
    K.paged_map(i32(5), i32(1), flat.as_strided((1, 4), (2, 1)), i32(0, 1, 2), i32(3), 16, 1)
    assert native["kvr_paged_map"][6:8] == (4, 4)
    K.paged_attn(q, pool, pool, flat.as_strided((3, 4), (6, 1)), plan)
    assert native["kvr_paged_attn"][15:17] == (6, 4)


def held_cache():
    """Row 0 holds pages 0, 1, row 1 pages 2, 3, 4."""
    from kvr_b200 import PagedKVCache
    c = PagedKVCache(1, 8, 2, 10, page=16, max_requests=3, max_len=64, device="cpu")
    c.block_table[0, :2] = i32(0, 1)
    c.block_table[1, :3] = i32(2, 3, 4)
    c.ctx_len[:] = i32(17, 48, 0)
    c.n_free.fill_(5)
    return c


@pytest.mark.parametrize("rows", [[1, 1], [1, 0, 1], [0, 0, 1, 1, 2, 2]])
def test_release_counts_a_row_once(rows):
    c = held_cache()
    c.release(rows)
    n = c.n_free.item()
    assert n == (8 if 0 not in rows else 10)
    free = c.free_pages[:n].tolist()
    assert len(set(free)) == n  # a page given out twice would be two requests' memory
    held = [p for row, m in zip(c.block_table.tolist(), c.ctx_len.tolist()) for p in row[:-(-m // 16)]]
    assert sorted(free + held) == list(range(10))


@pytest.mark.parametrize("rows", [[3], [-1], [0, 7]])
def test_release_refuses_rows_that_do_not_exist(rows):
    c = held_cache()
    with pytest.raises(ValueError, match="rows must be in"):
        c.release(rows)
    assert c.n_free.item() == 5 and c.ctx_len.tolist() == [17, 48, 0]
    c.release([])
    assert c.n_free.item() == 5


def tiny(cls="Llama", n_q=2, n_kv=1, layers=1, **kw):
    import transformers as T
    torch.manual_seed(0)
    kw = {"vocab_size": 50, "hidden_size": 64, "intermediate_size": 64, "num_hidden_layers": layers,
          "num_attention_heads": n_q, "num_key_value_heads": n_kv, "head_dim": 128, "max_position_embeddings": 64, **kw}
    return getattr(T, cls + "ForCausalLM")(getattr(T, cls + "Config")(**kw)).half().eval()


def generator(model=None, **kw):
    from kvr_b200 import PagedGenerator
    return PagedGenerator(model or tiny(), **{"n_pages": 10, "page": 16, "max_requests": 3, "max_len": 40, **kw})


def test_score_refuses_prompts_past_the_rope_tables(native):
    """Positions past the tables would be an index out of range on the device."""
    gen = generator()
    with pytest.raises(ValueError, match="longer than max_len"):
        gen.score([[1] * 41, [2]])
    assert not native


def test_generator_refuses_rows_that_do_not_exist_or_come_twice(native):
    """Row -1 would read the last row's length, and that row would get its tokens."""
    gen = generator()
    for new in ({-1: [5], 2: [6]}, {3: [1]}, {0: [1], 7: [2]}):
        with pytest.raises(ValueError, match="rows must be in"):
            gen.step(new)
    gen.last = {0: torch.zeros(50), 1: torch.zeros(50)}
    with pytest.raises(ValueError, match="twice"):
        gen.generate([0, 1, 0], 2)
    assert not native


HEAP = 1 << 40  # addresses that are only compared: every call below is refused before any CUDA call


def prompt_args(**kw):
    """kvr_prompt_attn of 16 tokens, 8 query heads on 8: every tensor takes 32 KB, all apart."""
    a = dict(q=HEAP, k=HEAP + (1 << 20), v=HEAP + (2 << 20), out=HEAP + (3 << 20), lse=None)
    a.update(kw)
    return [a["q"], a["k"], a["v"], 1, 16, 16, 2, 8, 8, 128, 1024, 1024, 1024, HEAP + (4 << 20), 1 << 15, 0.0, a["out"],
            a["lse"], HEAP + (5 << 20), 1 << 40, None]


def paged_args(**kw):
    """kvr_paged_attn of 16 tokens over 4 pages of 16, 8 heads: the pools take 128 KB each."""
    a = dict(q=HEAP, k=HEAP + (1 << 20), v=HEAP + (2 << 20), out=HEAP + (3 << 20), lse=None)
    a.update(kw)
    return [a["q"], 1, 16, 2, 8, 8, 128, 1024, a["k"], a["v"], 4, 16, 16384, 1024, HEAP + (6 << 20), 4, 4, HEAP + (4 << 20),
            1 << 15, 0.0, a["out"], a["lse"], HEAP + (5 << 20), 1 << 40, None]


@pytest.mark.parametrize("name,args,size", [("kvr_prompt_attn", prompt_args, 32768), ("kvr_paged_attn", paged_args, 131072)])
@pytest.mark.parametrize("over", ["q", "k", "v"])
@pytest.mark.parametrize("what", ["out", "lse"])
def test_output_over_an_input_is_refused(name, args, size, over, what):
    """CTAs store finished rows while others still read."""
    from kvr_b200 import _native as N
    at = {"q": HEAP, "k": HEAP + (1 << 20), "v": HEAP + (2 << 20)}[over]
    size = 32768 if over == "q" else size
    for p in (at, at + size - 512, at + 512):
        if what == "out" and p == at + 512:
            p = at - 512  # the end of out in the input's first row
        with pytest.raises(N.KvrError, match="must not") as e:
            N.call(name, *args(**{what: p}))
        assert e.value.code == 1


def test_output_over_the_log_sum_exps_is_refused():
    from kvr_b200 import _native as N
    for name, args in (("kvr_prompt_attn", prompt_args), ("kvr_paged_attn", paged_args)):
        with pytest.raises(N.KvrError, match="overlap"):
            N.call(name, *args(lse=HEAP + (3 << 20) + 32768 - 4))


def test_prompt_keys_must_be_the_queries_tokens_without_cu_k(native):
    """Fewer keys than tokens would be made up with zeros that take part in the softmax."""
    from kvr_b200 import kernels as K
    q, kv = torch.zeros(6, 8, 128, dtype=torch.float16), torch.zeros(9, 2, 128, dtype=torch.float16)
    plan = K.attn_plan(i32(0, 2, 6), 6, 8, 2)
    for n in (5, 7):
        with pytest.raises(ValueError, match="no cu_k"):
            K.prompt_attn(q, kv[:n], kv[:n], plan)
    assert "kvr_prompt_attn" not in native
    K.prompt_attn(q, kv[:6], kv[:6], plan)
    K.prompt_attn(q, kv, kv, K.attn_plan(i32(0, 2, 6), 6, 8, 2, cu_k=i32(0, 4, 9)))
    assert native["kvr_prompt_attn"][5] == 9


def test_write_with_half_of_the_rope_arguments_is_refused(native):
    """A sine table alone would leave q and k unrotated."""
    from kvr_b200 import kernels as K
    pool, x = torch.zeros(4, 16, 2, 128, dtype=torch.float16), torch.zeros(3, 2, 128, dtype=torch.float16)
    slots, pos, tab = torch.zeros(3, dtype=torch.int64), i32(0, 1, 2), torch.zeros(8, 128)
    for kw in (dict(sin=tab), dict(cos=tab, positions=pos), dict(sin=tab, positions=pos), dict(cos=tab, sin=tab)):
        with pytest.raises(ValueError, match="both tables"):
            K.paged_write(x, x, x, pool, pool, slots, **kw)
    assert not native


def write_args(**kw):
    """kvr_paged_write of 16 tokens, 8 query heads on 8, 4 pages of 16: tensors all apart."""
    a = dict(q=HEAP, k=HEAP + (1 << 20), v=HEAP + (2 << 20), kp=HEAP + (3 << 20), vp=HEAP + (4 << 20), q_out=HEAP + (5 << 20),
             qs=1024)
    a.update(kw)
    return [a["q"], a["k"], a["v"], 1, 16, 8, 8, 128, a["qs"], 1024, 1024, None, None, 0, 0, None, HEAP + (6 << 20), a["q_out"],
            a["kp"], a["vp"], 4, 16, 16384, 1024, None]


@pytest.mark.parametrize("kw", [
    dict(q_out=HEAP + 512), dict(q_out=HEAP - 512), dict(qs=2048, q_out=HEAP), dict(q_out=HEAP + (1 << 20)),
    dict(q_out=HEAP + (2 << 20) + 32256), dict(q_out=HEAP + (3 << 20) + 131072 - 256), dict(q_out=HEAP + (4 << 20) - 256)])
def test_rotated_queries_over_an_input_are_refused(kw):
    """Another warp may not have read it yet."""
    from kvr_b200 import _native as N
    with pytest.raises(N.KvrError, match="q_out must"):
        N.call("kvr_paged_write", *write_args(**kw))


@pytest.fixture
def cpu_map(monkeypatch):
    """kernels.paged_map by its CPU specification."""
    from kvr_b200 import kernels as K
    from oracle import paged_ref as R

    def paged_map(ctx_len, new_len, block_table, free_pages, n_free, page, n_tokens, **kw):
        m = R.page_map(ctx_len.tolist(), new_len.tolist(), block_table.numpy(), free_pages.tolist(), n_free.item(), page, n_tokens)
        block_table.copy_(torch.from_numpy(m["table"]))
        st = K.PagedStep()
        st.cu_q, st.kv_len, st.positions, st.slots, st.info = (
            torch.from_numpy(m[k]) for k in ("cu_q", "kv_len", "positions", "slots", "info"))
        st.n_free, st.n_tokens, st.plan = i32(m["n_free"]), n_tokens, None
        return st

    monkeypatch.setattr(K, "paged_map", paged_map)


def test_max_len_within_a_page(cpu_map):
    """The table's rows hold whole pages: 48 tokens where max_len is 40."""
    from kvr_b200 import PagedKVCache
    c = PagedKVCache(1, 8, 2, 10, page=16, max_requests=2, max_len=40, device="cpu")
    for new, fits in (([39, 5], True), ([1, 0], True), ([1, 3], False), ([0, 33], True), ([0, 32], False)):
        c.begin(new, sum(new))
        if fits:
            before = c.ctx_len.tolist()
            c.check()
            c.commit()
            assert c.ctx_len.tolist() == [a + b for a, b in zip(before, new)]
        else:
            with pytest.raises(RuntimeError, match="1 longer than max_len"):
                c.check()
            c.step = None
    # a step committed all the same (as a captured loop does) leaves the length at max_len
    c.begin([5, 0], 5)
    c.commit()
    assert c.ctx_len.tolist() == [40, 38]


def test_step_that_fails_in_the_model_leaves_no_open_step(cpu_map, monkeypatch):
    from kvr_b200 import kernels as K
    gen = generator()
    monkeypatch.setattr(K, "paged_write", lambda *a: (_ for _ in ()).throw(RuntimeError("out of memory")))
    with pytest.raises(RuntimeError, match="out of memory"):
        gen.step({1: [1, 2, 3]})
    gen.drop([1])
    assert gen.cache.n_free.item() == 10 and gen.last == {}


def test_add_takes_all_prompts_or_none(cpu_map, monkeypatch):
    """Prompts of 3 and 2 pages in a cache of 3: the second chunk does not fit."""
    from kvr_b200 import kernels as K
    monkeypatch.setattr(K, "paged_write", lambda q, *a: q)
    monkeypatch.setattr(K, "paged_attn", lambda q, *a, **kw: q)
    gen = generator(n_pages=3, chunk=16)
    with pytest.raises(RuntimeError, match="does not fit"):
        gen.add([[1] * 40, [2] * 20])
    assert gen.cache.n_free.item() == 3 and gen.last == {} and gen.cache.ctx_len.tolist() == [0, 0, 0]
    assert sorted(gen.cache.free_pages.tolist()) == [0, 1, 2]
    assert gen.add([[1] * 30]) == [0]
    assert gen.cache.n_free.item() == 1 and set(gen.last) == {0}


def test_add_refuses_an_empty_prompt(cpu_map):
    """It would return a row that has no logits to go on from."""
    gen = generator()
    for prompts in ([[]], [[1, 2], []]):
        with pytest.raises(ValueError, match="at least one token"):
            gen.add(prompts)
    assert gen.last == {} and gen.cache.n_free.item() == 10 and gen.add([]) == []


@pytest.mark.parametrize("cls,kw,match", [
    ("Granite", dict(head_dim=None, hidden_size=256, residual_multiplier=0.5), "granite"),
    ("Olmo2", dict(hidden_size=256, head_dim=None), "olmo2"),
    ("Llama", dict(rope_parameters={"rope_type": "dynamic", "factor": 2.0, "rope_theta": 1e4}), "dynamic"),
    ("Qwen2", dict(layers=2, use_sliding_window=True, sliding_window=8, max_window_layers=1, hidden_size=256), "window")])
def test_models_with_parts_that_are_not_applied_are_refused(cls, kw, match):
    kw = {k: v for k, v in kw.items() if v is not None}
    m = tiny(cls, **kw)
    with pytest.raises(NotImplementedError, match=match):
        generator(m)


def test_models_of_another_type_are_refused():
    with pytest.raises(ValueError, match="fp16 or bf16"):
        generator(tiny().float())


@pytest.mark.parametrize("cls,kw,own,given,want", [
    ("Llama", {}, 0, 0, 0), ("Llama", {}, 0, 7, 7), ("Mistral", dict(sliding_window=20), 20, 0, 20),
    ("Mistral", dict(sliding_window=20), 20, 7, 7), ("Mistral", dict(sliding_window=20), 20, 30, 20),
    ("Mistral", dict(sliding_window=40), 0, 0, 0), ("Mistral", dict(sliding_window=None), 0, 0, 0),
    ("Qwen3", dict(sliding_window=20, use_sliding_window=False), 0, 0, 0),
    ("Qwen3", dict(sliding_window=20, use_sliding_window=True, max_window_layers=0), 20, 0, 20)])
def test_window_of_the_model(cls, kw, own, given, want):
    from kvr_b200 import kvr_paged
    m = tiny(cls, **kw)
    assert kvr_paged._model_window(m, 40) == own
    assert generator(m, window=given).cache.window == want


def test_oracle_map_counts_the_keys_that_have_pages():
    # pages of 4, rows of 2 entries: request 0 runs past its row, request 1 past the free list, request 2 needs nothing
    import numpy as np
    from oracle import paged_ref as R
    t = np.full((3, 2), -1, np.int32)
    t[0, 0], t[2, 0] = 9, 8
    m = R.page_map([3, 0, 2], [9, 7, 1], t, [4, 5], 2, 4, 17)
    assert m["table"].tolist() == [[9, 5], [4, -1], [8, -1]] and m["n_free"] == 0
    assert m["kv_len"].tolist() == [8, 4, 3] and m["cu_q"].tolist() == [0, 9, 16, 17]
    assert m["slots"].tolist() == [39, 20, 21, 22, 23, -1, -1, -1, -1, 16, 17, 18, 19, -1, -1, -1, 34]
    assert m["info"].tolist() == [2, 0, 1, 0]  # request 1's second page, and request 0's third


@pytest.mark.parametrize("max_len,new,match", [
    (40, [41, 0], "0 pages missing, 0 requests cut at n_tokens, 1 longer"), (48, [49, 0], "1 longer"), (48, [48, 30], "1 pages missing"),
    (48, [30, 5], None)])
def test_a_committed_step_without_room_is_reported_later(cpu_map, max_len, new, match):
    """A loop of captured steps checks none of them on the host."""
    from kvr_b200 import PagedKVCache
    c = PagedKVCache(1, 8, 2, 4, page=16, max_requests=2, max_len=max_len, device="cpu")
    c.check()
    c.begin(new, sum(new))
    c.commit()
    c.begin([0, 0], 3)
    c.check()  # the open step has nothing to report
    c.commit()
    if match:
        with pytest.raises(RuntimeError, match="committed steps did not fit: .*" + match):
            c.check()
    c.check()  # once


def test_a_step_cut_at_n_tokens_is_reported_later(cpu_map):
    from kvr_b200 import PagedKVCache
    c = PagedKVCache(1, 8, 2, 9, page=16, max_requests=3, max_len=64, device="cpu")
    for _ in range(2):
        c.begin([3, 3, 3], 4)
        c.commit()
    with pytest.raises(RuntimeError, match="4 requests cut"):
        c.check()
    assert c.ctx_len.tolist() == [6, 2, 0]


def test_host_threads_on_one_workspace_take_turns(native, monkeypatch):
    """A call is two launches and ctypes lets other threads run meanwhile: attention,
    attention, join, join would join the wrong rows."""
    import threading
    import time
    from kvr_b200 import kernels as K
    inside, most = [0], [0]
    other, others = [0], [0]

    def slow(name, *args):
        if not name.endswith("_attn"):
            return 16
        n, m = (other, others) if args[-3] == 512 else (inside, most)
        n[0] += 1
        m[0] = max(m[0], n[0])
        time.sleep(0.01)
        n[0] -= 1
        return 0

    monkeypatch.setattr(K, "call", slow)
    at = threading.local()
    monkeypatch.setattr(K, "_attn_workspace", lambda device: (getattr(at, "ws", 256), 1 << 30, 0))
    q, kv = torch.zeros(2, 8, 128, dtype=torch.float16), torch.zeros(2, 2, 128, dtype=torch.float16)
    pool, table = torch.zeros(1, 16, 2, 128, dtype=torch.float16), torch.zeros(1, 1, dtype=torch.int32)
    packed, paged = K.attn_plan(i32(0, 2), 2, 8, 2), K.attn_plan(i32(0, 2), 2, 8, 2, kv_len=i32(2))

    def work(k):
        at.ws = 512 if k == 4 else 256
        for _ in range(5):
            K.prompt_attn(q, kv, kv, packed) if k % 2 else K.paged_attn(q, pool, pool, table, paged)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(5)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert most == [1] and others == [1]


def test_captured_calls_have_a_workspace_of_their_own(monkeypatch):
    """What a graph has baked in must not be what later calls on the stream use: the
    graph may be replayed on another stream beside them."""
    from types import SimpleNamespace
    from kvr_b200 import kernels as K
    now = {"stream": 7, "capturing": False}
    monkeypatch.setattr(K, "_ATTN_WS", {})
    monkeypatch.setattr(K, "stream", lambda: now["stream"])
    monkeypatch.setattr(K.N, "workspace", lambda tag, nbytes, device: torch.zeros(1))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: SimpleNamespace(synchronize=lambda: None))

    def address(stream, capturing):
        now.update(stream=stream, capturing=capturing)
        return K._attn_workspace("dev")[0]

    with pytest.raises(RuntimeError, match="outside of a graph capture"):
        address(7, True)
    eager = [address(7, False), address(9, False)]
    captured = [address(7, True), address(9, True), address(11, True)]
    assert len(set(eager + captured)) == 5
    assert address(12, True) == captured[2]  # streams without a call outside of captures share the device's
    assert [address(7, False), address(9, False)] == eager and address(7, True) == captured[0]


def test_calls_without_tokens_take_an_output(native):
    from kvr_b200 import kernels as K
    q, kv, pool = (torch.zeros(*s, 128, dtype=torch.float16) for s in ((0, 8), (0, 2), (1, 16, 2)))
    out = torch.empty_like(q)
    assert K.prompt_attn(q, kv, kv, K.attn_plan(i32(0, 0), 0, 8, 2), out=out) is out
    plan = K.attn_plan(i32(0, 0), 0, 8, 2, kv_len=i32(5))
    assert K.paged_attn(q, pool, pool, torch.zeros(1, 1, dtype=torch.int32), plan, out=out) is out
