"""The paged-cache serving operators at the ends of their ranges: what a call
must not write, and what it must refuse.  Plain 64-bit forms and tolerances as
in test_gpu_attn_paged.py unless said."""
import pytest
import torch

from test_gpu_attn_paged import BF16, DEV, F16, exact, i32, offsets

pytestmark = pytest.mark.gpu


def read_plan(buf):
    """Plan buffer -> (header words, pieces (n, 8)) on the host."""
    w = buf.cpu().view(torch.int32)
    return w[:64].tolist(), w[64:64 + 8 * w[7].item()].view(-1, 8)


# More items than a list has extra room for (512), all as long as the longest, in bins of more than one length: from
# 1024 K/V tiles on.  None may be cut then, and nothing may be written behind the plan.
@pytest.mark.parametrize("new,kv,n_q,n_kv,causal", [
    ([1] * 600, [131072] * 600, 4, 1, True),
    ([1] * 600, [131072 - 128] * 600, 4, 1, True),   # 1023 tiles: one length a bin
    ([1] * 513, [262400] * 513, 8, 8, True),         # 2050 tiles, four lengths a bin
    ([70000], [131072], 4, 1, False),
    ([1] * 300 + [2000], [131072] * 300 + [140000], 2, 2, True)])
def test_plan_of_many_equally_long_items_stays_in_its_buffer(new, kv, n_q, n_kv, causal):
    from kvr_b200 import _native as N
    n = sum(new)
    nbytes = N.call("kvr_attn_plan_bytes", n, len(new), n_q, n_kv)
    buf = torch.full((nbytes + (1 << 20),), 0xA5, dtype=torch.uint8, device=DEV)
    cu, kvl = offsets(new), i32(kv)
    N.call("kvr_attn_plan", N.ptr(cu), N.ptr(kvl), None, len(new), n, n_q, n_kv, int(causal), 0, N.ptr(buf), nbytes,
           N.stream())
    assert (buf[nbytes:] == 0xA5).all()
    head, pieces = read_plan(buf)
    per = 2 * (128 // (n_q // n_kv))
    items = sum(-(-m // per) for m in new)
    assert head[10] == 0 and head[11] == 0
    assert head[7] <= items + 512 and head[8] <= 512 and head[9] * n_kv <= 75776
    # every item's K/V tiles lie in its pieces once
    tiles = {}
    for q, n_tok, first, length, req, t0, t1, part in pieces.tolist():
        tiles.setdefault((q, n_tok, first, length, req), []).append((t0, t1))
    assert len(tiles) == items
    for (q, n_tok, first, length, req), got in tiles.items():
        got.sort()
        end = min(length, first + n_tok - 1) if causal else length
        assert got[0][0] == 0 and got[-1][1] == -(-end // 128)
        assert all(a[1] == b[0] for a, b in zip(got, got[1:]))


def test_plan_of_items_times_heads_past_32_bits():
    """2^23 items for each of 256 KV heads: far more than CTAs, whatever their
    product is in 32 bits."""
    from kvr_b200 import _native as N
    n, n_q, n_kv = 1 << 24, 128 * 256, 256
    nbytes = N.call("kvr_attn_plan_bytes", n, 1, n_q, n_kv)
    buf = torch.full((nbytes + (1 << 20),), 0xA5, dtype=torch.uint8, device=DEV)
    cu, kvl = i32([0, n]), i32([64])
    N.call("kvr_attn_plan", N.ptr(cu), N.ptr(kvl), None, 1, n, n_q, n_kv, 1, 0, N.ptr(buf), nbytes, N.stream())
    assert (buf[nbytes:] == 0xA5).all()
    head = buf[:256].cpu().view(torch.int32).tolist()
    assert head[7:12] == [n // 2, 0, 0, 0, 0]
    pieces = buf[256:256 + 32 * (n // 2)].view(torch.int32).view(-1, 8)
    starts, order = pieces[:, 0].sort()
    assert torch.equal(starts, torch.arange(0, n, 2, dtype=torch.int32, device=DEV)) and (pieces[:, 1] == 2).all()
    first = pieces[order, 2]
    assert torch.equal(first, 64 - n + 1 + starts)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_paged_attn_many_requests_of_131072_keys(dtype):
    """530 requests that share their pages.  Sums over n keys: the tensor core adds
    n / 16 products into an fp32 accumulator, each rounded by at most 2^-23 of A,
    beside the bound of the shorter cases."""
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(31)
    b, n, page = 530, 131072, 64
    k = torch.randn(n, 1, 128, device=DEV, generator=g).to(dtype)
    ramp = torch.linspace(-1, 1, n, device=DEV)[:, None, None]  # values that tell where a key lies
    v = (ramp + 0.1 * torch.randn(n, 1, 128, device=DEV, generator=g)).to(dtype)
    q = torch.randn(b, 2, 128, device=DEV, generator=g).to(dtype)
    order = torch.randperm(n // page, device=DEV, generator=g)
    kp, vp = torch.empty(n // page, page, 1, 128, device=DEV, dtype=dtype), torch.empty(n // page, page, 1, 128, device=DEV, dtype=dtype)
    kp[order], vp[order] = k.view(-1, page, 1, 128), v.view(-1, page, 1, 128)
    table = order.to(torch.int32).expand(b, -1).contiguous()
    plan = K.attn_plan(offsets([1] * b), b, 2, 1, kv_len=i32([n] * b))
    out, lse = K.paged_attn(q, kp, vp, table, plan, return_lse=True)
    K.attn_status()
    want, lse_x, tol, tol_l = exact(q, k, v, causal=False)
    tol = tol + n / 16 * 2.0 ** -23 * v.double().abs().max()
    assert ((out.double() - want).abs() <= tol).all()
    assert ((lse.double() - lse_x).abs() <= tol_l + n / 16 * 2.0 ** -23).all()


def test_write_in_place():
    """q_out may be q itself."""
    from kvr_b200 import kernels as K
    from test_gpu_attn_paged import tables
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = (torch.randn(33, h, 128, device=DEV, generator=g).half() for h in (8, 2, 2))
    kp, vp = torch.zeros(4, 16, 2, 128, device=DEV, dtype=F16), torch.zeros(4, 16, 2, 128, device=DEV, dtype=F16)
    slots, pos = torch.arange(33, device=DEV), torch.arange(33, device=DEV, dtype=torch.int32)
    want = K.paged_write(q, k, v, kp, vp, slots, pos, *tables(40))
    got = K.paged_write(q, k, v, kp, vp, slots, pos, *tables(40), q_out=q)
    assert got is q and torch.equal(got, want)


def test_generator_up_to_a_max_len_that_is_not_whole_pages():
    from kvr_b200 import PagedGenerator
    from test_gpu_attn_serving import prompts_of, tiny_llama, want_logits
    m = tiny_llama()
    gen = PagedGenerator(m, n_pages=12, page=16, max_requests=3, max_len=40, chunk=32)
    ids = prompts_of([40])[0]
    rows = gen.add([ids[:37]])
    for n in (38, 39, 40):
        got = gen.step({rows[0]: ids[n - 1:n]})[rows[0]]
        assert torch.allclose(got, want_logits(m, ids[:n])[-1], rtol=2e-2, atol=2e-2), n
    with pytest.raises(RuntimeError, match="longer than max_len"):
        gen.step({rows[0]: [1]})
    with pytest.raises(RuntimeError, match="longer than max_len"):
        gen.step({1: ids + [2]})
    assert torch.allclose(gen.score([ids])[0], want_logits(m, ids), rtol=2e-2, atol=2e-2)


@pytest.mark.parametrize("cls,kw", [
    ("Qwen3", {}), ("Qwen2", {}), ("Llama", dict(attention_bias=True, mlp_bias=True)), ("Mistral", dict(sliding_window=20)),
    ("Qwen3", dict(sliding_window=33, use_sliding_window=True, max_window_layers=0)),
    ("Llama", dict(rope_parameters={"rope_type": "yarn", "factor": 4.0, "rope_theta": 1e4,
                                    "original_max_position_embeddings": 128}))])
def test_generator_serves_models_with_norms_biases_and_windows(cls, kw):
    """Against the model's own forward, at the bar of the one-sequence generator's
    test (2e-2 on logits of order one, fp16)."""
    import transformers as T
    from kvr_b200 import PagedGenerator
    from test_gpu_attn_serving import prompts_of, want_logits
    torch.manual_seed(3)
    cfg = getattr(T, cls + "Config")(vocab_size=500, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                                     num_attention_heads=4, num_key_value_heads=2, head_dim=128, max_position_embeddings=512, **kw)
    m = getattr(T, cls + "ForCausalLM")(cfg)
    for layer in m.model.layers:  # weights that tell whether a part is applied
        for name, w in layer.self_attn.named_parameters():
            if "norm" in name:
                torch.nn.init.uniform_(w, 0.5, 2.0)
            elif name.endswith("bias"):
                torch.nn.init.normal_(w, std=0.5)
            else:
                torch.nn.init.normal_(w, std=0.06)  # scores far from flat, so that windows and norms show
    m = m.half().to(DEV).eval()
    prompts = prompts_of([90, 1, 37])
    gen = PagedGenerator(m, n_pages=30, page=16, max_requests=3, chunk=48)
    rows = gen.add(prompts)
    for b, p in zip(rows, prompts):
        assert torch.allclose(gen.last[b], want_logits(m, p)[-1], rtol=2e-2, atol=2e-2), b
    got = gen.step({b: [5 + b] for b in rows})
    for b, p in zip(rows, prompts):
        assert torch.allclose(got[b], want_logits(m, p + [5 + b])[-1], rtol=2e-2, atol=2e-2), b
    for p, x in zip(prompts, gen.score(prompts)):
        assert torch.allclose(x, want_logits(m, p), rtol=2e-2, atol=2e-2), len(p)


def test_requests_without_room_keep_what_is_stored():
    """A step that passes max_len and the free list, committed as a captured loop
    does: no page is lost, the keys that were stored (and only they) are attended,
    and the requests go on when pages are free again."""
    from kvr_b200 import PagedKVCache
    from test_gpu_attn_paged import check, exact
    g = torch.Generator(device=DEV).manual_seed(17)
    c = PagedKVCache(1, 8, 2, 6, page=16, max_requests=3, max_len=64, dtype=F16)
    held = [[], [], []]  # keys and values that a request has in the cache

    def step(new, stored, info):
        x = torch.randn(sum(new), 12, 128, device=DEV, generator=g).half()
        q, k, v = x.split([8, 2, 2], 1)
        st = c.begin(new, sum(new))
        out, lse = c.attend(0, c.write(0, q, k, v), return_lse=True)
        c.commit()
        assert st.info.tolist() == info and c.ctx_len.tolist() == stored
        at = 0
        for b, n in enumerate(new):
            had = sum(len(y[0]) for y in held[b])
            kept = stored[b] - had
            held[b].append((k[at:at + kept], v[at:at + kept]))
            if kept:
                kk, vv = (torch.cat([y[i] for y in held[b]]) for i in (0, 1))
                check(out[at:at + kept], lse[at:at + kept], exact(q[at:at + kept], kk, vv), (b, new))
            at += n
        assert torch.isfinite(out).all()
        pages = [p for row, m in zip(c.block_table.tolist(), stored) for p in row[:-(-m // 16)]]
        assert sorted(pages + c.free_pages[:c.n_free.item()].tolist()) == list(range(6))
        return out, lse

    step([30, 20, 0], [30, 20, 0], [0, 0, 0, 0])
    out, lse = step([40, 1, 10], [64, 21, 0], [2, 0, 1, 0])
    assert (out[41:] == 0).all() and (lse[41:] == -torch.inf).all()  # request 2 got no page: it sees nothing
    step([1, 0, 0], [64, 21, 0], [1, 0, 1, 0])
    c.release([0])
    held[0] = []
    step([0, 1, 10], [0, 22, 10], [0, 0, 0, 0])
    step([20, 12, 6], [20, 34, 16], [0, 0, 0, 0])  # pages 2 + 3 + 1: all
    step([0, 9, 0], [20, 43, 16], [0, 0, 0, 0])
    step([13, 8, 0], [32, 48, 16], [2, 0, 0, 0])   # 33 and 51 tokens would take a page more each


def test_map_plans_like_attn_plan():
    """The step's plan and attn_plan over its lengths give the same bits."""
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(18)
    ctx, new = [700, 0, 33, 1500], [90, 130, 0, 1]
    table = torch.full((4, 110), -1, dtype=torch.int32, device=DEV)
    table[:, :100] = torch.randperm(400, device=DEV, generator=g).view(4, 100).int()
    free = torch.arange(400, 440, dtype=torch.int32, device=DEV)
    kp, vp = (torch.randn(440, 16, 2, 128, device=DEV, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(230, 8, 128, device=DEV, generator=g).bfloat16()
    for window in (0, 200):
        st = K.paged_map(i32(ctx), i32(new), table, free, i32([40]), 16, 230, n_q=8, n_kv=2, window=window)
        plan = K.attn_plan(st.cu_q, 230, 8, 2, kv_len=st.kv_len, window=window)
        a, b = (K.paged_attn(q, kp, vp, table, p, return_lse=True) for p in (st.plan, plan))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_replayed_steps_without_room_are_reported():
    """A captured decode step, replayed past the pages there are."""
    from kvr_b200 import PagedKVCache
    c = PagedKVCache(1, 8, 2, 3, page=16, max_requests=2, max_len=64, dtype=F16)
    x = torch.randn(2, 12, 128, device=DEV).half()
    lens = i32([1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        q, k, v = x.split([8, 2, 2], 1)
        c.begin(lens, 2)
        out = c.attend(0, c.write(0, q, k, v))
        c.commit()
        return out

    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for _ in range(15):
            graph.replay()
        c.check()
        assert c.ctx_len.tolist() == [16, 16]
        graph.replay()  # two pages wanted, one left
        with pytest.raises(RuntimeError, match="1 pages missing"):
            c.check()
        assert c.ctx_len.tolist() == [17, 16]
        for _ in range(3):
            graph.replay()
        with pytest.raises(RuntimeError, match="3 pages missing"):
            c.check()
        c.check()
        assert c.ctx_len.tolist() == [20, 16]
    torch.cuda.current_stream().wait_stream(side)


def test_offsets_that_overlap_past_the_list_are_reported():
    """40 requests that all claim all tokens: the plan's list has room for some of
    their items only.  The call leaves its output alone and says so."""
    from kvr_b200 import _native as N
    from kvr_b200 import kernels as K
    q = torch.randn(640, 8, 128, device=DEV).half()
    kv = torch.randn(640, 2, 128, device=DEV).half()
    cu = i32([640, 0] * 20 + [640])
    plan = K.attn_plan(cu, 640, 8, 2)
    head, _ = read_plan(plan.buf)
    assert head[10] == 1
    K.attn_status()
    out = torch.full_like(q, 7)
    K.prompt_attn(q, kv, kv, plan, out=out)
    with pytest.raises(N.KvrError, match="offsets overlap"):
        K.attn_status()
    assert (out == 7).all()
    K.attn_status()


def test_host_threads_on_one_stream():
    """Calls whose pieces are joined by a second kernel, from four threads."""
    import threading
    from kvr_b200 import kernels as K
    from test_gpu_attn_paged import make_pages
    g = torch.Generator(device=DEV).manual_seed(19)
    jobs = []
    for kv in ([5000], [3000, 9000], [7777], [4096, 100]):
        kp, vp, table, _ = make_pages(g, kv, 2, 16, F16)
        q = torch.randn(len(kv), 8, 128, device=DEV, generator=g).half()
        plan = K.attn_plan(offsets([1] * len(kv)), len(kv), 8, 2, kv_len=i32(kv))
        jobs.append((q, kp, vp, table, plan, K.paged_attn(q, kp, vp, table, plan)))
    torch.cuda.synchronize()
    wrong, done = [], []

    def work(k):
        *args, want = jobs[k]
        outs = [K.paged_attn(*args) for _ in range(200)]
        wrong.extend(k for o in outs if not torch.equal(o, want))
        done.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and sorted(done) == [0, 1, 2, 3]
    K.attn_status()


@pytest.mark.parametrize("what", ["paged", "prompt"])
def test_attention_as_a_host_threads_first_call(what):
    """A thread whose memory comes from torch's cache has no CUDA context of its own yet."""
    import threading
    from kvr_b200 import kernels as K
    q, k, v = torch.randn(40, 12, 128, device=DEV).half().split([8, 2, 2], 1)
    if what == "prompt":
        plan = K.attn_plan(i32([0, 40]), 40, 8, 2)
        call = lambda: K.prompt_attn(q, k, v, plan)  # noqa: E731
    else:
        plan = K.attn_plan(i32([0, 40]), 40, 8, 2, kv_len=i32([40]))
        kp, vp, table = torch.randn(3, 16, 2, 128, device=DEV).half(), torch.randn(3, 16, 2, 128, device=DEV).half(), i32([2, 0, 1])[None]
        call = lambda: K.paged_attn(q, kp, vp, table, plan)  # noqa: E731
    want, got = call(), []
    call()  # its output goes back to the cache
    t = threading.Thread(target=lambda: got.append(call()))
    t.start()
    t.join()
    assert len(got) == 1 and torch.equal(got[0], want)


def test_graph_replayed_beside_calls_on_its_capture_stream():
    """Captured on one stream, replayed on another while that one has calls of its own."""
    from kvr_b200 import kernels as K
    from test_gpu_attn_paged import make_pages
    g = torch.Generator(device=DEV).manual_seed(23)
    jobs = []
    for kv in ([6000], [9000]):  # pieces joined through the workspace
        kp, vp, table, _ = make_pages(g, kv, 2, 16, BF16)
        q = torch.randn(1, 8, 128, device=DEV, generator=g).bfloat16()
        plan = K.attn_plan(offsets([1]), 1, 8, 2, kv_len=i32(kv))
        jobs.append((q, kp, vp, table, plan))
    want = [K.paged_attn(*j) for j in jobs]
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (one, two):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(one):
        K.paged_attn(*jobs[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=one):
            outs = [K.paged_attn(*jobs[1]) for _ in range(40)]
    two.wait_stream(one)
    beside = []
    for _ in range(10):
        with torch.cuda.stream(two):
            graph.replay()
        with torch.cuda.stream(one):
            beside += [K.paged_attn(*jobs[0]) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[1]) for o in outs)
    assert all(torch.equal(o, want[0]) for o in beside)


@pytest.mark.parametrize("own_stream", [False, True])
def test_status_covers_replayed_graphs(own_stream):
    """A graph whose plan is of other shapes by the time it is replayed."""
    from kvr_b200 import _native as N
    from kvr_b200 import kernels as K
    q = torch.randn(6, 8, 128, device=DEV).half()
    kv = torch.randn(6, 2, 128, device=DEV).half()
    plan, other = K.attn_plan(i32([0, 6]), 6, 8, 2), K.attn_plan(i32([0, 3, 6]), 6, 8, 2)
    keep = plan.buf[:64].clone()
    K.prompt_attn(q, kv, kv, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.prompt_attn(q, kv, kv, plan)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, **({"stream": side} if own_stream else {})):
            K.prompt_attn(q, kv, kv, plan)
        graph.replay()
        K.attn_status()
        plan.buf[:64].copy_(other.buf[:64])
        graph.replay()
        with pytest.raises(N.KvrError, match="plan"):
            K.attn_status()
        K.attn_status("cuda")
        plan.buf[:64].copy_(keep)
        graph.replay()
        K.attn_status(torch.device("cuda"))
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_attn_of_queries_without_any_keys(causal):
    from kvr_b200 import kernels as K
    q, kv = torch.randn(70, 8, 128, device=DEV).half(), torch.empty(0, 2, 128, device=DEV, dtype=F16)
    plan = K.attn_plan(i32([0, 40, 70]), 70, 8, 2, cu_k=i32([0, 0, 0]), causal=causal)
    out, lse = K.prompt_attn(q, kv, kv, plan, return_lse=True)
    K.attn_status()
    assert (out == 0).all() and (lse == -torch.inf).all()


def test_calls_without_tokens():
    from kvr_b200 import kernels as K
    q, kv = torch.empty(0, 8, 128, device=DEV, dtype=F16), torch.empty(0, 2, 128, device=DEV, dtype=F16)
    out = torch.empty_like(q)
    assert K.prompt_attn(q, kv, kv, K.attn_plan(i32([0, 0]), 0, 8, 2), out=out) is out
    pool = torch.zeros(2, 16, 2, 128, device=DEV, dtype=F16)
    st = K.paged_map(i32([5, 0]), i32([0, 0]), torch.zeros(2, 3, dtype=torch.int32, device=DEV), i32([1]), i32([1]), 16, 0, n_q=8, n_kv=2)
    assert K.paged_write(q, kv, kv, pool, pool.clone(), st.slots).shape == q.shape
    out, lse = K.paged_attn(q, pool, pool, torch.zeros(2, 3, dtype=torch.int32, device=DEV), st.plan, return_lse=True)
    assert out.shape == q.shape and lse.shape == (0, 8) and st.kv_len.tolist() == [5, 0]
    K.attn_status()


def test_log_sum_exps_merge_with_attention_over_other_keys():
    """Keys in two caches: attention over each, merged as rows [lse, 1, out] by the
    sequence split's merge, is attention over all.  Each part brings its own bound."""
    from kvr_b200 import kernels as K
    from test_gpu_attn_paged import make_pages
    g = torch.Generator(device=DEV).manual_seed(29)
    kv, n_q, n_kv = [333, 90, 1200], 8, 2
    old = [200, 0, 1100]  # keys that lie elsewhere; request 1 has none there
    q = torch.randn(3, n_q, 128, device=DEV, generator=g).half()
    parts, keys = [], []
    for lens in (old, [a - b for a, b in zip(kv, old)]):
        kp, vp, table, rows = make_pages(g, lens, n_kv, 16, F16)
        plan = K.attn_plan(offsets([1, 1, 1]), 3, n_q, n_kv, kv_len=i32(lens), causal=False)
        parts.append(K.paged_attn(q, kp, vp, table, plan, return_lse=True))
        keys.append([(kp[r], vp[r]) for r in rows])
    rows = torch.stack([torch.cat([lse[..., None], torch.ones_like(lse)[..., None], out.float()], -1) for out, lse in parts])
    got = K.lse_merge(rows.view(2, 3 * n_q, 130)).view(3, n_q, 128)
    for b in range(3):
        k, v = (torch.cat([part[b][i] for part in keys]) for i in (0, 1))
        want, lse, tol, tol_l = exact(q[b:b + 1], k, v, causal=False)
        # a part off by tol, weights off by e^(2 tol_l): the output moves by 2 tol_l of the parts' sizes
        size = torch.stack([p[0][b:b + 1].double().abs() for p in parts]).amax(0)
        part_tol = [exact(q[b:b + 1], *part[b], causal=False)[2] for part in keys if len(part[b][0])]
        bound = torch.stack(part_tol).amax(0) + tol + 4 * tol_l[..., None] * size
        assert ((got[b:b + 1].double() - want).abs() <= bound).all(), b


def test_cache_step_against_the_keys_it_holds():
    """Steps of chunks and single tokens: each output against the 64-bit form over
    the rotated queries and the pages as they are, so no rotation's rounding has to
    be allowed for; and the rotation against the CPU specification."""
    from kvr_b200 import PagedKVCache
    from oracle import paged_ref as R
    from test_gpu_attn_paged import HALF_STEP, U, check, tables
    g = torch.Generator(device=DEV).manual_seed(30)
    cos, sin = tables(512)
    for dtype in (F16, BF16):
        c = PagedKVCache(1, 8, 2, 60, page=16, max_requests=3, max_len=512, dtype=dtype)
        done = [0, 0, 0]
        for new in ([100, 37, 0], [1, 1, 200], [260, 1, 1], [1, 0, 1]):
            x = torch.randn(sum(new), 12, 128, device=DEV, generator=g).to(dtype)
            q, k, v = x.split([8, 2, 2], 1)
            st = c.begin(new, sum(new))
            turned = c.write(0, q, k, v, cos, sin)
            out, lse = c.attend(0, turned, return_lse=True)
            pos = st.positions.long()
            want = torch.from_numpy(R.rope(q.double().cpu().numpy(), *(t[pos].double().cpu().numpy() for t in (cos, sin)))).to(DEV)
            y = torch.cat([q[..., 64:], q[..., :64]], -1)
            tol = U[dtype] * want.abs() + 2.0 ** -22 * (q.double().abs() + y.double().abs()) + HALF_STEP[dtype]
            assert ((turned.double() - want).abs() <= tol).all()
            c.commit()
            done = [a + b for a, b in zip(done, new)]
            at = 0
            for b, n in enumerate(new):
                pages = c.block_table[b, :-(-done[b] // 16)].long()
                kk, vv = (p[0][pages].reshape(-1, 2, 128)[:done[b]] for p in (c.k, c.v))
                if n:
                    check(out[at:at + n], lse[at:at + n], exact(turned[at:at + n], kk, vv), (dtype, new, b))
                at += n
        # one request once more against the CPU specification of attention
        b, n = 1, 39
        kk, vv = (p[0][c.block_table[b, :3].long()].reshape(-1, 2, 128)[:n].double().cpu().numpy() for p in (c.k, c.v))
        qq = torch.randn(2, 8, 128, device=DEV, generator=g).to(dtype)
        x_out, x_lse, _ = R.attention(qq.double().cpu().numpy(), kk, vv, 2, n)
        mine = exact(qq, *(torch.from_numpy(t).to(DEV) for t in (kk, vv)))
        assert (mine[0].cpu() - torch.from_numpy(x_out)).abs().max() < 1e-12
        assert (mine[1].cpu() - torch.from_numpy(x_lse)).abs().max() < 1e-12
