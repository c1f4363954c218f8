"""Beam selection and the reordering of paged rows on the GPU against their
64-bit specification.

Tolerance of a score: its rounding to fp32 (2^-24 of it) and the error of the
log-sum-exp.  A sum of V exponentials e^(x - m), each within 2^-21 (the exponent's
rounding for |x - m| up to 64 with a base-2 exponential of 2^-22), added up in fp32
by each thread (at most V / 256 + 9 additions, 2^-24 each) and joined in 64
bits: an absolute error of lse below 2^-21 + (V / 256 + 9) 2^-24."""
import numpy as np
import pytest
import torch

from oracle import decode_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def lse_error(V):
    return 2.0 ** -21 + (V / 256 + 9) * 2.0 ** -24


def check_select(logits, cum, n=None, eos=(), given=None):
    from kvr_b200 import kernels as K
    B, k = cum.shape
    V = logits.shape[-1]
    got = K.beam_select(logits if given is None else given, cum, n=n, eos=eos)
    n = k * (1 + len(eos)) if n is None else n
    want = R.beam_select(logits.double().cpu().numpy().reshape(B, k, V), cum.cpu().numpy(), n, eos)
    for name in ("beams", "tokens", "next_beams", "next_tokens"):
        assert np.array_equal(getattr(got, name).cpu().numpy(), want[name]), name
        assert getattr(got, name).dtype is torch.int32
    for name in ("scores", "next_scores"):
        a, w = getattr(got, name).double().cpu().numpy(), want[name]
        assert np.array_equal(np.isfinite(a), np.isfinite(w))
        f = np.isfinite(w)
        assert (np.abs(a[f] - w[f]) <= lse_error(V) + 2.0 ** -23 * np.abs(w[f])).all(), np.abs(a[f] - w[f]).max()
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,k,V,pad", [(1, 1, 1, 0), (1, 4, 32000, 0), (3, 5, 50257, 0), (2, 3, 1009, 7), (1, 32, 2049, 1),
                                       (7, 2, 7, 1), (40, 8, 4100, 0), (1, 1, 200001, 0),
                                       (700, 1, 300, 0), (3, 31, 16, 3)])
def test_select(dtype, B, k, V, pad):
    g = torch.Generator(device=DEV).manual_seed(V + k)
    wide = (3 * torch.randn(B * k, V + pad, device=DEV, generator=g)).to(DT[dtype])
    cum = -5 * torch.rand(B, k, device=DEV, generator=g)
    check_select(wide[:, :V], cum)


@pytest.mark.parametrize("n,eos", [(4, ()), (128, ()), (12, (5, 9)), (8, (0,)), (36, tuple(range(8)))])
def test_select_ends_and_counts(n, eos):
    g = torch.Generator(device=DEV).manual_seed(n)
    logits = 2 * torch.randn(8, 700, device=DEV, generator=g)
    logits[:, list(eos)] += 6
    check_select(logits, -torch.rand(2, 4, device=DEV, generator=g), n, eos)


def test_select_equal_logits_by_beam_and_token():
    # every logit the same; and values that repeat many times, in any order of threads
    for V in (40, 5000, 70000):
        cum = torch.zeros(2, 3, device=DEV)
        check_select(torch.full((6, V), 1.5, device=DEV), cum)
        g = torch.Generator(device=DEV).manual_seed(V)
        few = torch.randint(0, 4, (6, V), device=DEV, generator=g).to(torch.bfloat16)
        few[3:] = few[:3]
        check_select(few, cum)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_select_sorted_rows(dtype):
    """Every step of a rising row passes the threshold: the list is cut again and again."""
    V = 30000
    up = (torch.arange(V, device=DEV) / 97).to(DT[dtype])
    rows = torch.stack([up, up.flip(0), up - 1, torch.roll(up, 777)])
    check_select(rows, torch.tensor([[0.0, -0.3, 0.7, 0.1]], device=DEV), 64)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_select_masks(dtype):
    """Masked by -inf and by the type's lowest value; rows without a token; beams that do not count; infinities and NaN."""
    dt = DT[dtype]
    g = torch.Generator(device=DEV).manual_seed(3)
    V = 9001
    x = torch.randn(12, V, device=DEV, generator=g).to(dt)
    x[0, :] = -float("inf")                       # nothing allowed
    x[1, 5:] = -float("inf")                      # five tokens
    x[2, :] = torch.finfo(dt).min                 # all at the lowest value
    x[3, 3:] = torch.finfo(dt).min
    x[4, 100] = float("nan")                      # no candidates from these
    x[5, 8000] = float("inf")
    x[6, :] = float("nan")
    x[7, 1:] = -float("inf")                      # one token: its score is the beam's
    cum = torch.tensor([[0.0, -1, -2], [-3, 0, -1], [0, -2, -float("inf")], [float("nan"), float("inf"), -1]], device=DEV)
    check_select(x, cum, 40, (1, 3))
    # a request without any continuation
    none = check_select(torch.full((4, 50), -float("inf"), device=DEV, dtype=dt), torch.zeros(2, 2, device=DEV))
    assert none.next_tokens.eq(-1).all() and none.next_scores.eq(-float("inf")).all()


def test_select_first_step_from_one_row():
    """All beams of a request see its prompt's logits: expanded rows, and only the first beam counts."""
    g = torch.Generator(device=DEV).manual_seed(4)
    one = torch.randn(3, 1, 5003, device=DEV, generator=g)
    cum = torch.full((3, 4), -float("inf"), device=DEV)
    cum[:, 0] = 0
    check_select(one.expand(3, 4, -1).reshape(12, -1), cum, eos=(2,), given=one.expand(3, 4, -1))
    same = torch.randn(1, 5003, device=DEV, generator=g)
    check_select(same.expand(4, -1).contiguous(), cum[:1], given=same.expand(4, -1))


@pytest.mark.parametrize("V", [9, 4100, 128256])
def test_select_beams_that_there_are_not(V):
    """Their rows mean nothing, whatever stands in them: no candidates, and no request's other beams change."""
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = 2 * torch.randn(5 * 4, V, device=DEV, generator=g)
    cum = -torch.rand(5, 4, device=DEV, generator=g)
    inf = float("inf")
    cum[0, 1:], cum[1, :3], cum[2, 2], cum[3] = -inf, -inf, float("nan"), -inf
    cum[4, 0] = inf
    dead = ~cum.isfinite().flatten()
    plain = check_select(logits.clone(), cum)
    for fill in (float("nan"), inf, -inf, 3e38):
        logits[dead] = fill
        got = check_select(logits.clone(), cum)
        assert torch.equal(got.tokens, plain.tokens) and torch.equal(got.scores, plain.scores)
    assert (plain.beams[3] == -1).all() and (plain.next_scores[3] == -inf).all()


def test_select_in_a_graph_and_on_another_stream():
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(5)
    x, cum = torch.randn(8, 33000, device=DEV, generator=g), -torch.rand(2, 4, device=DEV, generator=g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = K.beam_select(x, cum, eos=(3,))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b = K.beam_select(x, cum, eos=(3,))
    for seed in (6, 7):
        x.copy_(torch.randn(8, 33000, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)))
        graph.replay()
        c = K.beam_select(x, cum, eos=(3,))
        for name in ("scores", "beams", "tokens", "next_scores", "next_beams", "next_tokens"):
            assert torch.equal(getattr(b, name), getattr(c, name))
    assert a.scores.isfinite().all()


# ----------------------------------------------------------------- reorder --


def make_cache(groups, beams, lens, page, seed, spare=0, n_kv=2, layers=2, dtype=torch.float16, strided=False):
    """Rows of several groups with pages of their own and pages that beams share.
    lens[g][i]: tokens of row i of group g; the shared part is the shortest's full pages of the first half of the rows."""
    rng = np.random.default_rng(seed)
    n_rows = groups * beams + 2
    width = max(max(-(-n // page) for g in lens for n in g), 1) + 2
    total = sum(-(-n // page) for g in lens for n in g) + spare
    ids = rng.permutation(total).astype(np.int32)
    table = np.full((n_rows, width), -1, np.int32)
    ctx = np.zeros(n_rows, np.int32)
    rows = rng.permutation(n_rows)[:groups * beams].reshape(groups, beams)
    at = 0
    for g in range(groups):
        common = min(lens[g]) // page  # columns whose pages all rows of the group may share
        upto = int(rng.integers(0, common + 1))
        for i, n in enumerate(lens[g]):
            r = rows[g, i]
            ctx[r] = n
            for j in range(-(-n // page)):
                if i and j < upto:
                    table[r, j] = table[rows[g, 0], j]
                else:
                    table[r, j] = ids[at]
                    at += 1
    held = [p for r in range(n_rows) for p in table[r, :-(-ctx[r] // page)]]
    shared = np.maximum(np.bincount(np.array(held, dtype=np.int64), minlength=max(total, 1)) - 1, 0).astype(np.int32)
    free = np.concatenate([ids[at:], ids[:at]]).astype(np.int32)
    if total == 0:
        free = np.zeros(1, np.int32)
    g = torch.Generator(device=DEV).manual_seed(seed)
    if strided:  # K and V of a page in one tensor
        kv = torch.randn(layers, max(total, 1), 2, page, n_kv, 128, device=DEV, generator=g).to(dtype)
        k, v = kv[:, :, 0], kv[:, :, 1]
    else:
        k, v = (torch.randn(layers, max(total, 1), page, n_kv, 128, device=DEV, generator=g).to(dtype) for _ in range(2))
    return table, ctx, shared, free, total - at, rows, k, v


def check_reorder(cache, parents, page):
    from kvr_b200 import kernels as K
    table, ctx, shared, free, n_free, rows, k, v = cache
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731
    want = R.reorder(table, ctx, shared, free, n_free, rows.tolist(), parents.tolist(), page)
    t, c, s, f, n = i32(table), i32(ctx), i32(shared), i32(free), i32([n_free])
    want_k, want_v = k.clone(), v.clone()
    for a, b, m in want["copies"]:
        want_k[:, b, :m], want_v[:, b, :m] = k[:, a, :m], v[:, a, :m]
    info = K.paged_reorder(t, c, s, f, n, i32(rows), i32(parents), k, v)
    assert np.array_equal(info.cpu().numpy(), want["info"]), (info.tolist(), want["info"])
    assert np.array_equal(c.cpu().numpy(), want["ctx"])
    assert np.array_equal(t.cpu().numpy(), want["table"])
    assert np.array_equal(s.cpu().numpy(), want["shared"])
    assert n.item() == want["n_free"]
    assert np.array_equal(f.cpu().numpy(), want["free"])
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    return want


@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("groups,beams", [(1, 2), (3, 4), (5, 7), (2, 32), (1, 1), (30, 5)])
def test_reorder(groups, beams, page):
    rng = np.random.default_rng(groups * 100 + beams)
    lens = [[int(rng.integers(0, 9 * page + 1)) for _ in range(beams)] for _ in range(groups)]
    if groups > 1:
        lens[1] = [page * 4 + 3] * beams  # as beam search has them: of one length
        lens[0] = [page * 5] * beams      # at a page's end
    cache = make_cache(groups, beams, lens, page, 7, spare=groups * beams, strided=page == 16)
    parents = rng.integers(-1, beams, (groups, beams))
    check_reorder(cache, parents, page)


def test_reorder_fork_keep_and_empty():
    page = 16
    for lens, parents in [([[100, 0, 0, 0]], [[0, 0, 0, 0]]),      # a prompt becomes four beams
                          ([[100, 90, 80, 70]], [[0, 1, 2, 3]]),    # nothing changes
                          ([[100, 90, 80, 70]], [[-1, -1, -1, -1]]),
                          ([[100, 90, 80, 70]], [[3, 2, 1, 0]]),
                          ([[100, 90, 80, 70]], [[1, 9, -7, 0]]),   # no such parent: emptied
                          ([[0, 0, 0]], [[2, 1, 0]]), ([[1, 1, 1]], [[1, 1, 1]]), ([[16, 16, 16]], [[1, 1, 1]])]:
        check_reorder(make_cache(1, len(lens[0]), lens, page, 3, spare=4), np.array(parents), page)


@pytest.mark.parametrize("spare", [0, 1, 2])
def test_reorder_without_pages(spare):
    """A fork with too few free pages: what finds none keeps its full pages."""
    page = 16
    w = check_reorder(make_cache(1, 4, [[100, 0, 0, 0]], page, 5, spare=spare), np.zeros((1, 4), int), page)
    assert w["info"][0] == 3 - spare


@pytest.mark.parametrize("groups,beams", [(128, 32), (4096, 1), (819, 5)])
def test_reorder_most_rows(groups, beams):
    page = 8
    rng = np.random.default_rng(groups)
    lens = [[int(rng.integers(0, 5 * page))] * beams for _ in range(groups)]
    cache = make_cache(groups, beams, lens, page, groups, spare=groups * beams // 2, n_kv=1, layers=1)
    check_reorder(cache, rng.integers(-1, beams, (groups, beams)), page)


@pytest.mark.parametrize("beams", [3, 8])
def test_reorder_long_tables(beams):
    """More 32-column units than warps, and rows that share all but the end."""
    page, n = 8, 20000
    lens = [[n + 5 * g] * beams for g in range(6)]
    rng = np.random.default_rng(beams)
    check_reorder(make_cache(6, beams, lens, page, 9, spare=40, n_kv=1, layers=1), rng.integers(0, beams, (6, beams)), page)


def test_reorder_pages_shared_by_groups():
    """A page that rows of two groups give up goes back once; one that a third row holds stays."""
    page = 16
    table = np.array([[0, 1, 2], [0, 1, 3], [0, 4, 5], [6, 7, -1]], np.int32)
    ctx = np.array([48, 48, 48, 32], np.int32)
    for rows, parents in [([[0], [1], [2]], [[-1], [-1], [-1]]), ([[0], [1]], [[-1], [-1]]), ([[0, 3], [1, 2]], [[1, 1], [1, 1]])]:
        shared = np.zeros(9, np.int32)
        shared[0], shared[1] = 2, 1
        g = torch.Generator(device=DEV).manual_seed(1)
        k, v = (torch.randn(1, 9, page, 1, 128, device=DEV, generator=g).half() for _ in range(2))
        free = np.array([8, 0, 0, 0, 0, 0, 0, 0, 0], np.int32)
        check_reorder((table, ctx, shared, free, 1, np.array(rows), k, v), np.array(parents), page)


def test_reorder_rows_that_do_not_exist():
    """Rows outside of the table are passed over; nothing is written for them."""
    from kvr_b200 import kernels as K
    table, ctx, shared, free, n_free, rows, k, v = make_cache(1, 3, [[40, 30, 20]], 16, 2, spare=5)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731
    t, c, s, f, n = i32(table), i32(ctx), i32(shared), i32(free), i32([n_free])
    rows = rows.copy()
    lost = rows[0, 2]
    rows[0, 2] = 99
    info = K.paged_reorder(t, c, s, f, n, i32(rows), i32([[0, 0, 0]]), k, v)
    assert info.tolist()[:2] == [0, 1] and c[lost].item() == 20 and c[rows[0, 1]].item() == 40
    held = [p for r in range(5) for p in t[r, :-(-c[r].item() // 16)].tolist()]
    assert sorted(set(held) | set(f[:n.item()].tolist())) == list(range(k.shape[1]))


def test_reorder_in_a_graph():
    from kvr_b200 import kernels as K
    page, beams = 16, 4
    cache = make_cache(2, beams, [[70] * 4, [33] * 4], page, 11, spare=10)
    table, ctx, shared, free, n_free, rows, k, v = cache
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731
    state = [i32(table), i32(ctx), i32(shared), i32(free), i32([n_free])]
    eager = [x.clone() for x in state]
    k2, v2 = k.clone(), v.clone()
    parents, r = i32([[0, 1, 2, 3]] * 2), i32(rows)
    keep = [x.clone() for x in state]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        info = K.paged_reorder(*state, r, parents, k, v)
    for a, b in zip(state, keep):
        a.copy_(b)
    for p in ([[1, 1, 0, 2], [3, 3, 3, 3]], [[0, 0, 0, 1], [2, 1, 0, -1]], [[3, 2, 2, 0], [0, 0, 1, 1]]):
        parents.copy_(i32(p))
        graph.replay()
        other = K.paged_reorder(*eager, r, parents, k2, v2)
        assert torch.equal(info, other) and all(torch.equal(a, b) for a, b in zip(state, eager))
        assert torch.equal(k, k2) and torch.equal(v, v2)


@pytest.mark.parametrize("free", [0, 1, 8])
def test_reorder_last_pages_that_rows_share(free):
    """A last page of several rows, in one group under several parents, in several groups, with a row outside of the call."""
    from test_decode_ops_host import SHARED_LAST, shared_last, whole_pool
    g = torch.Generator(device=DEV).manual_seed(1)
    for rows, parents in SHARED_LAST:
        table, ctx, shared, free_pages, n = shared_last(free)
        k, v = (torch.randn(2, len(shared), 16, 1, 128, device=DEV, generator=g).half() for _ in range(2))
        w = check_reorder((table, ctx, shared, free_pages, n, np.array(rows), k, v), np.array(parents), 16)
        whole_pool(w["table"], w["ctx"], w["shared"], w["free"], w["n_free"], 16)


@pytest.mark.parametrize("groups,beams,free", [(3000, 1, 0), (3000, 1, 700), (3000, 1, 2000), (1024, 3, 3000), (4096, 1, 5000)])
def test_reorder_last_pages_shared_by_distant_groups(groups, beams, free):
    """More places than threads: what one place does to a page's count is nothing that a later one goes by."""
    from test_decode_ops_host import whole_pool
    rng = np.random.default_rng(groups + free)
    rows = groups * beams + 10           # ten of them not in the call
    pages = groups
    of = rng.integers(0, pages, rows)    # whose last page a row has
    n = pages + 1 + free                 # (page 0 in front of all)
    of = np.unique(of, return_inverse=True)[1]  # each one held
    n -= pages - (of.max() + 1)
    table = np.full((rows, 2), -1, np.int32)
    table[:, 0], table[:, 1] = 0, of + 1
    shared = (np.bincount(table.reshape(-1), minlength=n) - 1).clip(min=0).astype(np.int32)
    lists = np.concatenate([np.arange(of.max() + 2, n), np.zeros(n, np.int64)])[:n].astype(np.int32)
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(1, n, 16, 1, 128, device=DEV, generator=g).half() for _ in range(2))
    ctx = rng.integers(17, 32, rows).astype(np.int32)
    where = rng.permutation(rows)[:groups * beams].reshape(groups, beams)
    w = check_reorder((table, ctx, shared, lists, n - of.max() - 2, where, k, v), rng.integers(0, beams, (groups, beams)), 16)
    whole_pool(w["table"], w["ctx"], w["shared"], w["free"], w["n_free"], 16)


def test_select_scores_beyond_fp32():
    """A masked token of a beam that came by a masked token: a sum below all of fp32 is no continuation, in any of the outputs."""
    low = torch.finfo(torch.float32).min
    x = torch.full((4, 600), low, device=DEV)
    x[:, :2] = torch.randn(4, 2, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    x[3] = 1.0
    cum = torch.tensor([[-1.0, low], [low / 2, low]], device=DEV)
    got = check_select(x, cum, 12, (0,))
    assert got.scores.isfinite().eq(got.beams >= 0).all() and got.next_scores.isfinite().eq(got.next_tokens >= 0).all()
    # request 0: two tokens of each beam, and the masked ones of beam 0; none of beam 1's masked ones
    assert got.beams[0].tolist() == [0] * 12
    one = check_select(x[1:2], cum[:1, 1:], 5)
    assert one.tokens[0, 2:].tolist() == [-1] * 3 and one.scores[0, :2].isfinite().all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("k,n,eos", [(32, 64, (3,)), (32, 128, (3, 5, 9)), (32, 33, ()), (16, 32, (7,)), (31, 93, (1, 2))])
def test_select_many_beams_of_equal_scores(k, n, eos, dtype):
    """Beams whose scores and rows are alike: the best of all lie in all lists, at equal ranks.

    Rows of 20011 logits lie at different places within 16 bytes, so the sums of equal rows are added up in different orders,
    and each log-sum-exp may be off by lse_error on its own.  Scores that differ by less than twice that have no order by
    the sums' accuracy: among such candidates of different beams any order is right, within a beam (one log-sum-exp) only
    that of the logits, then the tokens."""
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(k + n)
    cum = torch.zeros(1, k, device=DEV)
    x = (2 * torch.randn(k, 20011, device=DEV, generator=g)).to(DT[dtype])
    check_select(x, cum, n, eos)
    x[:] = x[:1]
    got = K.beam_select(x, cum, n, eos)
    lp = x[0].double().log_softmax(0)  # the score of a token, in every beam
    order = lp.sort(descending=True, stable=True)[1]
    beams, tokens, scores = got.beams[0].tolist(), got.tokens[0].tolist(), got.scores[0].double()
    close = lse_error(20011) + 2.0 ** -23 * lp[order[:n]].abs().max()
    assert len(set(zip(beams, tokens))) == n and (scores.diff() <= 0).all()
    assert ((scores - lp[got.tokens[0].long()]).abs() <= close).all()
    best = lp[order].repeat_interleave(k)[:n]  # each token of all beams, from the best on
    assert ((scores - best).abs() <= 2 * close).all()
    for b in range(k):  # a beam's own are its best, in order
        mine = [t for o, t in zip(beams, tokens) if o == b]
        assert mine == order[:len(mine)].tolist()
    on = [i for i in range(n) if tokens[i] not in eos][:k]
    assert got.next_beams[0].tolist()[:len(on)] == [beams[i] for i in on] and got.next_tokens[0].tolist()[:len(on)] == [tokens[i] for i in on]
