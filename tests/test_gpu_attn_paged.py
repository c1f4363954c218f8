"""Paged-cache serving operators on the GPU against plain 64-bit forms.

Tolerances, from the number formats: outputs are rounded to the tensors' type
(unit roundoff u) and so are the softmax weights that enter the tensor cores;
scores are 128-term fp32 sums, so a score is off by at most 2^-16 of S = the
largest sum_c |q_c k_c| / scale of the row (128 roundings of 2^-24, doubled);
an exponential may be off by 2^-14 (a 16-bit weight keeps no more).  With A =
sum_j p_j |v_j|:
  |out - exact| <= u |exact| + (u + 2 (2^-16 S + 2^-14)) A + 2^-20 max|v|
  |lse - exact| <= 2^-16 S + 2^-14 + 2^-22 |exact|.
"""
import numpy as np
import pytest
import torch

from oracle import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
HALF_STEP = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # of the subnormal range, where u does not hold
F16, BF16 = torch.float16, torch.bfloat16


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def offsets(ns):
    return i32(np.concatenate([[0], np.cumsum(ns)]))


def exact(q, k, v, causal=True, window=0, scale=None):
    """One request on the GPU in 64 bits: (out, lse, bound of out, bound of lse)."""
    n, n_q, d = q.shape
    m, n_kv = k.shape[:2]
    u = U[q.dtype]
    scale = d ** 0.5 if scale is None else scale
    i = torch.arange(n, device=DEV)[:, None] + m - n
    j = torch.arange(m, device=DEV)[None]
    ok = j <= i if causal else torch.ones(n, m, dtype=torch.bool, device=DEV)
    if window:
        ok = ok & (j > i - window)
    kk = k.double().repeat_interleave(n_q // n_kv, 1)
    vv = v.double().repeat_interleave(n_q // n_kv, 1)
    s = torch.einsum("nhd,mhd->hnm", q.double(), kk) / scale
    S = torch.einsum("nhd,mhd->hnm", q.double().abs(), kk.abs()) / scale
    s = s.masked_fill(~ok, -torch.inf)
    S = S.masked_fill(~ok, 0.0)
    S = S.amax(-1).T if m else torch.zeros(n, n_q, dtype=torch.float64, device=DEV)
    lse = torch.logsumexp(s, -1).T if m else torch.full((n, n_q), -torch.inf, dtype=torch.float64, device=DEV)
    p = torch.exp(s - torch.where(lse.T == -torch.inf, 0.0, lse.T)[..., None])
    vz = torch.where(ok.any(0)[:, None, None], vv, 0.0) if m else vv  # keys nobody sees do not count
    out = torch.einsum("hnm,mhd->nhd", p, vz)
    A = torch.einsum("hnm,mhd->nhd", p, vz.abs())
    e = 2.0 ** -16 * S + 2.0 ** -14
    top = vz.abs().amax() if m else 0.0
    return out, lse, u * out.abs() + (u + 2 * e)[..., None] * A + 2.0 ** -20 * top, e + 2.0 ** -22 * lse.abs()


def check(got, lse, want, what=""):
    out_x, lse_x, tol, tol_l = want
    got = got.double()
    assert torch.isfinite(got).all(), what
    off = (got - out_x).abs() - tol
    assert (off <= 0).all(), (what, off.max().item(), (got - out_x).abs().max().item())
    empty = lse_x == -torch.inf
    assert ((lse == -torch.inf) == empty).all(), what
    assert (got[empty] == 0).all(), what
    off = ((lse.double() - lse_x).abs() - tol_l)[~empty]
    assert (off <= 0).all(), (what, off.max().item())


# --------------------------------------------------------------------- map --


@pytest.mark.parametrize("batch,page,most,spare,cut,narrow", [
    (1, 64, 1, 0, 0, 0), (3, 16, 100, 5, 0, 0), (300, 64, 1, 2, 0, 0), (48, 16, 900, 0, 0, 0), (7, 1, 30, 3, 0, 0),
    (40, 100, 700, -3, 0, 0), (25, 8, 50, 4, -40, 0), (25, 8, 50, 4, 37, 0), (30, 32, 300, 1, 0, 3), (4096, 16, 3, 0, 0, 0),
    (2, 16, 40000, 9, 0, 0), (5, 16, 0, 4, 12, 0)])
def test_map_vs_oracle(batch, page, most, spare, cut, narrow):
    """cut < 0: fewer tokens than the requests bring; > 0: padding.  narrow:
    table columns missing for the longest; spare < 0: pages missing."""
    from kvr_b200 import kernels as K
    rng = np.random.default_rng(batch + page)
    new = rng.integers(0, most + 1, batch)
    ctx = rng.integers(0, 4 * page + 1, batch) * rng.integers(0, 2, batch)
    had, now = -(-ctx // page), -(-(ctx + new) // page)
    need = int((now - had).sum())
    ids = rng.permutation(int(now.sum()) + abs(spare) + 8)
    width = max(int(now.max()) - narrow, 1)
    table = np.full((batch, width), -1, np.int32)
    at = 0
    for b in range(batch):
        table[b, :had[b]] = ids[at:at + had[b]][:width]
        at += had[b]
    n_free = max(need + spare, 0)
    free = ids[at:at + n_free]
    n_tokens = max(int(new.sum()) + cut, 0)
    want = R.page_map(ctx, new, table, free, n_free, page, n_tokens)
    tab = torch.from_numpy(table).to(DEV)
    fr = i32(np.concatenate([free, [-5]]))  # the list's capacity is larger than what is free
    for _ in range(2):  # repeating a call repeats its result
        st = K.paged_map(i32(ctx), i32(new), tab, fr, i32([n_free]), page, n_tokens, n_q=8, n_kv=2)
        got = {"cu_q": st.cu_q, "kv_len": st.kv_len, "positions": st.positions, "slots": st.slots, "table": tab,
               "info": st.info}
        for name, x in got.items():
            assert np.array_equal(x.cpu().numpy(), want[name]), name
        assert st.n_free.item() == want["n_free"]


# ------------------------------------------------------------------- write --


def tables(n):
    inv = 500000.0 ** (-torch.arange(0, 128, 2, device=DEV).float() / 128)
    a = torch.arange(n, device=DEV).float()[:, None] * inv
    return torch.cat([a.cos()] * 2, 1), torch.cat([a.sin()] * 2, 1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,n_q,n_kv,page,form", [
    (1, 32, 8, 64, "fused"), (5, 8, 8, 16, "plain"), (333, 6, 2, 24, "fused"), (1000, 32, 8, 7, "pair"), (64, 1, 1, 16, "plain"),
    (2500, 64, 8, 16, "fused"), (9, 32, 8, 16, "no q"), (9, 32, 8, 16, "no rope")])
def test_write_vs_exact(n, n_q, n_kv, page, form, dtype):
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(n)
    qkv = torch.randn(n, n_q + 2 * n_kv, 128, device=DEV, generator=g).to(dtype)
    q, k, v = qkv.split([n_q, n_kv, n_kv], 1)
    if form == "plain":
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    n_pages = -(-n // page) + 3
    if form == "pair":  # K and V interleaved in one pool, pages padded
        pool = torch.randn(n_pages, 2, page + 1, n_kv, 128, device=DEV, generator=g).to(dtype)
        kp, vp = pool[:, 0, :page], pool[:, 1, :page]
    else:
        kp = torch.randn(n_pages, page, n_kv, 128, device=DEV, generator=g).to(dtype)
        vp = torch.randn(n_pages, page, n_kv, 128, device=DEV, generator=g).to(dtype)
    cos, sin = tables(700)
    cos[:, 64:] *= 1.25  # halves that differ
    slots = torch.randperm(n_pages * page, device=DEV, generator=g)[:n].contiguous()
    pos = torch.randint(0, 700, (n,), device=DEV, generator=g, dtype=torch.int32)
    dead = torch.zeros(n, dtype=torch.bool, device=DEV)
    if n > 4:
        slots[1], slots[2] = -1, n_pages * page  # padding, outside the pool
        if form != "no rope":
            pos[3], pos[4] = 700, -1             # outside the tables
        dead[1:3] = True
        dead[3:5] = form != "no rope"
    k0, v0 = kp.clone(), vp.clone()
    rope = form != "no rope"
    out = K.paged_write(None if form == "no q" else q, k, v, kp, vp, slots, pos if rope else None, cos if rope else None,
                        sin if rope else None)
    c, s = (cos[pos.clamp(0, 699)].double(), sin[pos.clamp(0, 699)].double()) if rope else (torch.ones(n, 128, device=DEV).double(),
                                                                                             torch.zeros(n, 128, device=DEV).double())
    live = ~dead

    def turned(x):
        x = x.double()
        y = torch.cat([-x[..., 64:], x[..., :64]], -1)
        return x * c[:, None] + y * s[:, None], U[dtype], 2.0 ** -22 * (x.abs() + y.abs()) + HALF_STEP[dtype]

    if form == "no q":
        assert out is None
    else:
        want, u, fl = turned(q)
        assert ((out.double() - want).abs() <= u * want.abs() + fl)[live].all()
        assert (out[dead] == 0).all()
    want, u, fl = turned(k)
    at = (slots[live] // page, slots[live] % page)
    assert ((kp[at].double() - want[live]).abs() <= (u * want.abs() + fl)[live]).all()
    assert torch.equal(vp[at], v[live])
    # nothing else in the pool changed
    k0[at], v0[at] = kp[at], vp[at]
    assert torch.equal(k0, kp) and torch.equal(v0, vp)


# --------------------------------------------------------------- attention --


def make_pages(g, kv, n_kv, page, dtype, spread=1.0, poison=False, spare=5):
    need = [-(-m // page) for m in kv]
    n_pages = sum(need) + spare
    perm = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    table = torch.full((len(kv), max(max(need), 1) + 1), -1, dtype=torch.int32, device=DEV)
    kp = spread * torch.randn(n_pages, page, n_kv, 128, device=DEV, generator=g)
    kp, vp = kp.to(dtype), torch.randn(n_pages, page, n_kv, 128, device=DEV, generator=g).to(dtype)
    used = torch.zeros(n_pages, page, dtype=torch.bool, device=DEV)
    at, rows = 0, []
    for b, m in enumerate(kv):
        pages = perm[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = pages
        j = torch.arange(m, device=DEV)
        rows.append((pages.long()[j // page], j % page))
        used[rows[-1]] = True
    if poison:  # rows of the pool that no request owns
        bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device=DEV, dtype=dtype)
        kp[~used] = bad[torch.randint(0, 3, (int((~used).sum()), n_kv, 128), device=DEV, generator=g)]
        vp[~used] = bad[torch.randint(0, 3, (int((~used).sum()), n_kv, 128), device=DEV, generator=g)]
        table[table < 0] = perm[-1]  # and table entries past the end point into them
    return kp, vp, table, rows


def run_paged(new, ctx, n_q, n_kv, page, dtype, window=0, spread=1.0, poison=False, scale=None, causal=True, seed=0, pad=0):
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(seed)
    kv = [n + c for n, c in zip(new, ctx)]
    kp, vp, table, rows = make_pages(g, kv, n_kv, page, dtype, spread, poison)
    n = sum(new)
    q = torch.randn(n + pad, n_q, 128, device=DEV, generator=g).to(dtype)
    if pad and poison:
        q[n:] = float("nan")
    plan = K.attn_plan(offsets(new), n + pad, n_q, n_kv, kv_len=i32(kv), window=window, causal=causal)
    out, lse = K.paged_attn(q, kp, vp, table, plan, scale=scale, return_lse=True)
    K.attn_status()
    assert (out[n:] == 0).all() and (lse[n:] == -torch.inf).all()
    at = 0
    for b, m in enumerate(new):
        want = exact(q[at:at + m], kp[rows[b]], vp[rows[b]], causal, window, scale)
        check(out[at:at + m], lse[at:at + m], want, (b, m, kv[b]))
        at += m
    return out, lse


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,ctx,n_q,n_kv,page,window", [
    ([1], [0], 32, 8, 64, 0),                       # the first token
    ([1], [4095], 32, 8, 64, 0),
    ([1] * 5, [0, 127, 128, 129, 1000], 8, 2, 16, 0),
    ([1, 1, 1], [2000, 3, 700], 8, 8, 32, 0),       # one query head per KV head
    ([2, 1, 4, 3], [300, 0, 511, 90], 64, 8, 64, 0),
    ([64], [448], 32, 8, 64, 0),
    ([65, 1, 200], [63, 700, 0], 32, 8, 16, 0),
    ([129, 31], [5, 129], 6, 2, 8, 0),              # g = 3: rows that do not fill a tile
    ([40, 1], [700, 30], 28, 4, 128, 0),            # g = 7
    ([300], [10], 8, 8, 24, 0),                     # pages that end inside a key tile
    ([10, 3], [200, 50], 128, 1, 16, 0),            # 128 heads on one
    ([30, 1], [900, 900], 32, 8, 256, 0),           # pages larger than a key tile
    ([1, 1, 1], [1500, 255, 256], 32, 8, 16, 256),  # windows
    ([77, 1, 300], [1000, 2047, 100], 32, 8, 64, 100),
    ([200], [500], 8, 2, 32, 1),                    # a window of the token itself
    ([7, 0, 5, 0], [33, 64, 0, 0], 8, 2, 16, 0),    # idle requests
    ([520], [1600], 32, 8, 64, 0),
])
def test_paged_attn_vs_exact(new, ctx, n_q, n_kv, page, window, dtype):
    run_paged(new, ctx, n_q, n_kv, page, dtype, window)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,ctx,window", [([1, 40, 1], [300, 77, 1023], 0), ([1, 130, 9], [77, 500, 1], 64)])
def test_paged_attn_ignores_what_requests_do_not_own(new, ctx, window, dtype):
    """NaN and infinities in unused rows and pages, in table entries past the
    end and in padding queries change nothing."""
    run_paged(new, ctx, 8, 2, 16, dtype, window, poison=True, pad=37)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n_q,n_kv,new", [
    (8, 8, [15, 16, 17, 300, 8, 9]), (16, 2, [2, 3, 150, 1]), (32, 2, [1, 2, 100, 1]), (34, 2, [1, 90, 1]),
    (48, 16, [5, 6, 200, 4, 1])])
def test_paged_attn_items_of_about_16_rows(n_q, n_kv, new, dtype):
    """Items with up to 16 rows (tokens x heads per KV head) take a narrower
    product: sizes on both sides of it, after one another and cut in pieces."""
    for seed, base in enumerate((0, 130, 9000)):
        ctx = [base + 77 * i for i in range(len(new))]
        run_paged(new, ctx, n_q, n_kv, 16, dtype, spread=3.0 if seed else 1.0, poison=True, seed=seed, pad=3)


@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_paged_attn_flat_and_peaked(spread):
    """All scores equal, and scores of several hundred."""
    run_paged([1, 100], [2047, 900], 8, 2, 64, F16, spread=spread)
    run_paged([1, 100], [2047, 900], 8, 2, 64, BF16, spread=spread)


def test_paged_attn_scale_and_full():
    run_paged([33, 1], [100, 400], 8, 2, 16, BF16, scale=3.0)
    run_paged([33, 150, 1], [100, 0, 400], 8, 2, 16, F16, causal=False)


@pytest.mark.parametrize("new,ctx,n_q,n_kv,window", [
    ([512], [8000], 32, 8, 0),                     # fewer items than SMs, long ones: every CTA takes an equal range
    ([300, 40], [5000, 9000], 8, 2, 0),            # ... of items of two requests
    ([100, 700], [3000, 2500], 16, 1, 2000),
    ([64, 3, 65], [12000, 11000, 100], 6, 2, 0)])
def test_paged_attn_few_long_items(new, ctx, n_q, n_kv, window):
    run_paged(new, ctx, n_q, n_kv, 64, BF16, window=window, seed=4)
    run_paged(new, ctx, n_q, n_kv, 16, F16, window=window, seed=5)


def test_paged_attn_many_requests_long_and_short():
    """More work than CTAs, lengths from 1 to 6000 in one call."""
    rng = np.random.default_rng(5)
    ctx = [int(x) for x in np.exp(rng.uniform(0, np.log(6000), 60))]
    new = [1 if i % 3 else int(rng.integers(1, 150)) for i in range(60)]
    run_paged(new, ctx, 32, 8, 16, BF16, seed=1)


def test_paged_attn_more_queries_than_keys():
    """Queries before the first key see nothing: zeros and -inf."""
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(3)
    kv, new = [3, 0, 200, 1], [9, 4, 450, 1]
    kp, vp, table, rows = make_pages(g, kv, 2, 16, F16, poison=True)
    q = torch.randn(sum(new), 8, 128, device=DEV, generator=g).half()
    for window in (0, 2):
        plan = K.attn_plan(offsets(new), sum(new), 8, 2, kv_len=i32(kv), window=window)
        out, lse = K.paged_attn(q, kp, vp, table, plan, return_lse=True)
        at = 0
        for b, n in enumerate(new):
            check(out[at:at + n], lse[at:at + n], exact(q[at:at + n], kp[rows[b]], vp[rows[b]], window=window), (b, window))
            at += n


def test_paged_attn_missing_pages_read_as_zeros():
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(4)
    kp, vp, table, rows = make_pages(g, [700], 2, 16, BF16)
    q = torch.randn(5, 8, 128, device=DEV, generator=g).bfloat16()
    plan = K.attn_plan(i32([0, 5]), 5, 8, 2, kv_len=i32([700]))
    table[0, 3], table[0, 20], table[0, 43] = -1, kp.shape[0], 1 << 30
    out, lse = K.paged_attn(q, kp, vp, table[:, :40], plan, return_lse=True)  # a table that is too narrow as well
    k, v = kp[rows[0]].clone(), vp[rows[0]].clone()
    for x in (k, v):
        x[48:64], x[320:336], x[640:] = 0, 0, 0
    check(out, lse, exact(q, k, v), "missing")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,n_q,n_kv,window", [
    ([1], 32, 8, 0), ([64], 32, 8, 0), ([65, 1, 63, 128, 257], 32, 8, 0), ([1000, 1, 500], 8, 8, 0), ([333], 6, 2, 0),
    ([129, 130], 28, 4, 0), ([90], 128, 1, 0), ([700, 33], 64, 8, 100), ([500, 5], 8, 2, 128), ([2049], 32, 8, 0),
    ([1] * 50, 8, 2, 0), ([0, 5, 0, 0, 300, 0], 8, 2, 0)])
def test_prompt_attn_vs_exact(lens, n_q, n_kv, window, dtype):
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(len(lens))
    n = sum(lens)
    qkv = torch.randn(n, n_q + 2 * n_kv, 128, device=DEV, generator=g).to(dtype)
    q, k, v = qkv.split([n_q, n_kv, n_kv], 1)  # strided views
    plan = K.attn_plan(offsets(lens), n, n_q, n_kv, window=window)
    out, lse = K.prompt_attn(q, k, v, plan, return_lse=True)
    K.attn_status()
    same = K.prompt_attn(q.contiguous(), k.contiguous(), v.contiguous(), plan)
    assert torch.equal(out, same)
    at = 0
    for b, m in enumerate(lens):
        r = slice(at, at + m)
        check(out[r], lse[r], exact(q[r], k[r], v[r], window=window), (b, m))
        at += m


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_attn_other_keys(causal):
    """Keys of other lengths than the queries; a neighbour's NaN stays there."""
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(9)
    ql, kl = [40, 7, 300, 5], [100, 3, 129, 0]
    q = torch.randn(sum(ql), 8, 128, device=DEV, generator=g).half()
    k = torch.randn(sum(kl) + 9, 2, 128, device=DEV, generator=g).half()
    v = torch.randn(sum(kl) + 9, 2, 128, device=DEV, generator=g).half()
    k[sum(kl):], v[sum(kl):] = float("nan"), float("inf")
    k[100:103], v[100:103] = float("nan"), float("nan")  # request 1's keys
    plan = K.attn_plan(offsets(ql), sum(ql), 8, 2, cu_k=offsets(kl), causal=causal)
    out, lse = K.prompt_attn(q, k, v, plan, return_lse=True)
    for b in (0, 2, 3):
        r, s = slice(sum(ql[:b]), sum(ql[:b + 1])), slice(sum(kl[:b]), sum(kl[:b + 1]))
        check(out[r], lse[r], exact(q[r], k[s], v[s], causal=causal), b)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes and 2^31 elements, pages at its far end."""
    from kvr_b200 import kernels as K
    n_kv, page = 8, 64
    n_pages = (1 << 31) // (page * n_kv * 128) + 40
    kp = torch.zeros(n_pages, page, n_kv, 128, dtype=F16, device=DEV)
    vp = torch.zeros(n_pages, page, n_kv, 128, dtype=F16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    n = 200
    q, k, v = (torch.randn(n, h, 128, device=DEV, generator=g).half() for h in (32, n_kv, n_kv))
    table = torch.arange(n_pages - 1, n_pages - 5, -1, dtype=torch.int32, device=DEV)[None].contiguous()
    j = torch.arange(n, device=DEV)
    slots = table[0].long()[j // page] * page + j % page
    assert K.paged_write(None, k, v, kp, vp, slots) is None
    plan = K.attn_plan(i32([0, n]), n, 32, n_kv, kv_len=i32([n]))
    out, lse = K.paged_attn(q, kp, vp, table, plan, return_lse=True)
    check(out, lse, exact(q, k, v), "far")


def test_interleaved_pool_and_strided_table():
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(6)
    pool = torch.randn(20, 2, 17, 2, 128, device=DEV, generator=g).bfloat16()
    kp, vp = pool[:, 0, :16], pool[:, 1, :16]
    wide = torch.full((2, 30), -1, dtype=torch.int32, device=DEV)
    wide[:, :9] = torch.randperm(20, device=DEV, generator=g)[:18].view(2, 9).int()
    table = wide[:, :9]
    q = torch.randn(30, 10, 128, device=DEV, generator=g).bfloat16()[:, 2:10]
    kv, new = [140, 77], [20, 10]
    plan = K.attn_plan(offsets(new), 30, 8, 2, kv_len=i32(kv))
    out, lse = K.paged_attn(q, kp, vp, table, plan, return_lse=True)
    for b, r in enumerate([slice(0, 20), slice(20, 30)]):
        k, v = (x[table[b].long()].reshape(-1, 2, 128)[:kv[b]] for x in (kp, vp))
        check(out[r], lse[r], exact(q[r], k, v), b)


def test_other_stream_and_graph():
    """A step on a side stream, captured once and replayed on new inputs and lengths."""
    from kvr_b200 import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(7)
    cos, sin = tables(512)
    n = 40
    qkv = torch.randn(n, 12, 128, device=DEV, generator=g).half()
    new = i32([20, 1, 0])
    cache = PagedKVCache(1, 8, 2, 24, page=16, max_requests=3, max_len=256, dtype=F16)
    eager = PagedKVCache(1, 8, 2, 24, page=16, max_requests=3, max_len=256, dtype=F16)

    def step(c, x, lens):
        q, k, v = x.split([8, 2, 2], 1)
        c.begin(lens, n)
        out, lse = c.attend(0, c.write(0, q, k, v, cos, sin), return_lse=True)
        c.commit()
        return out, lse

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x, lens = torch.zeros_like(qkv), torch.zeros_like(new)
        step(cache, x, lens)  # allocates the stream's workspace; appends nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, lse = step(cache, x, lens)
        for it in range(4):
            x.copy_(torch.randn(n, 12, 128, device=DEV, generator=g).half())
            lens.copy_(i32([[20, 1, 0], [5, 17, 3], [1, 1, 1], [0, 30, 2]][it]))
            graph.replay()
            a, b = step(eager, x.clone(), lens.clone())
            assert torch.equal(a, out) and torch.equal(b, lse), it
            assert torch.equal(cache.ctx_len, eager.ctx_len) and torch.equal(cache.n_free, eager.n_free)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("kind", ["decode", "prompt"])
def test_repeated_calls_give_the_same_bits(kind):
    """Copies that land in another order must not show: 60 calls, the inputs out of cache before each."""
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(12)
    flush = torch.empty(160 << 20, dtype=torch.uint8, device=DEV)
    if kind == "decode":
        kv, new = [3000 + 37 * b for b in range(24)], [1] * 24
        kp, vp, table, _ = make_pages(g, kv, 8, 16, BF16)
        q = torch.randn(24, 32, 128, device=DEV, generator=g).bfloat16()
        plan = K.attn_plan(offsets(new), 24, 32, 8, kv_len=i32(kv))
        call = lambda: K.paged_attn(q, kp, vp, table, plan)  # noqa: E731
    else:
        lens = [1500, 700, 1, 350]
        q, k, v = torch.randn(sum(lens), 48, 128, device=DEV, generator=g).half().split([32, 8, 8], 1)
        plan = K.attn_plan(offsets(lens), sum(lens), 32, 8)
        call = lambda: K.prompt_attn(q, k, v, plan)  # noqa: E731
    first = call()
    for _ in range(60):
        flush.zero_()
        assert torch.equal(call(), first)
    K.attn_status()


def test_capture_on_a_stream_without_a_workspace():
    """torch's own capture stream: the graph uses the device's capture workspace."""
    from kvr_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(21)
    q, k, v = torch.randn(700, 12, 128, device=DEV, generator=g).half().split([8, 2, 2], 1)
    plan = K.attn_plan(i32([0, 700]), 700, 8, 2)
    want = K.prompt_attn(q, k, v, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.prompt_attn(q, k, v, plan)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_output_over_the_queries_is_refused():
    from kvr_b200 import _native as N
    from kvr_b200 import kernels as K
    q = torch.randn(6, 8, 128, device=DEV).half()
    kv = torch.randn(6, 2, 128, device=DEV).half()
    plan = K.attn_plan(i32([0, 6]), 6, 8, 2)
    ws, wb, s = K._attn_workspace(q.device)
    with pytest.raises(N.KvrError, match="must not be q"):
        N.call("kvr_prompt_attn", N.ptr(q), N.ptr(kv), N.ptr(kv), 1, 6, 6, 1, 8, 2, 128, 1024, 256, 256, N.ptr(plan.buf),
               plan.nbytes, 0.0, N.ptr(q), None, ws, wb, s)


def test_plan_of_another_call_is_reported():
    from kvr_b200 import _native as N
    from kvr_b200 import kernels as K
    q = torch.randn(6, 8, 128, device=DEV).half()
    kv = torch.randn(6, 2, 128, device=DEV).half()
    plan = K.attn_plan(i32([0, 6]), 6, 8, 2)
    with pytest.raises(ValueError, match="plan"):
        K.prompt_attn(q[:5], kv[:5], kv[:5], plan)
    with pytest.raises(ValueError, match="plan"):
        K.paged_attn(q, kv[None], kv[None], torch.zeros(1, 1, dtype=torch.int32, device=DEV), plan)
    other = K.attn_plan(i32([0, 3, 6]), 6, 8, 2)
    plan.buf[:64].copy_(other.buf[:64])  # what a caller of the C ABI could pass by mistake
    K.prompt_attn(q, kv, kv, plan)
    with pytest.raises(N.KvrError, match="plan"):
        K.attn_status()
    K.attn_status()  # the word is cleared


def test_offsets_that_make_no_sense_do_no_harm():
    """Lengths and offsets are device data that no host check sees: falling
    offsets and negative lengths give some output, no fault."""
    from kvr_b200 import kernels as K
    q = torch.randn(64, 8, 128, device=DEV).half()
    kv = torch.randn(4, 16, 2, 128, device=DEV).half()
    table = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    for cu in ([0, 90, 10, -5, 64], [64, 0, 64, 0, 64], [5, 5, 5, 5, 5]):
        plan = K.attn_plan(i32(cu), 64, 8, 2, kv_len=i32([30, -7, 1 << 30, 5]), window=700)
        out = K.paged_attn(q, kv, kv, table, plan)
        plan = K.attn_plan(i32(cu), 64, 8, 2, cu_k=i32([0, 40, 20, -3, 70]))
        K.prompt_attn(q, kv.view(-1, 2, 128), kv.view(-1, 2, 128), plan, out=out)
    torch.cuda.synchronize()


def test_cache_serves_requests_like_whole_prompts():
    """Two layers, three requests: prompts in chunks mixed with decode steps give
    what prompt attention over each whole sequence gives; released pages are
    taken again."""
    from kvr_b200 import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(8)
    cos, sin = tables(1024)
    n_q, n_kv = 8, 2
    total = [300, 150, 37]
    cache = PagedKVCache(2, n_q, n_kv, 40, page=16, max_requests=4, max_len=512, dtype=BF16)
    steps = [[100, 150, 0, 0], [100, 0, 36, 0], [99, 0, 1, 0], [1, 0, 0, 0]]
    x = {(b, l): torch.randn(total[b], n_q + 2 * n_kv, 128, device=DEV, generator=g).bfloat16()
         for b in range(3) for l in range(2)}
    got = {key: [] for key in x}
    for rnd in range(2):
        done = [0, 0, 0]
        for new in steps:
            cache.begin(new, sum(new))
            cache.check()
            for layer in range(2):
                rows = torch.cat([x[b, layer][done[b]:done[b] + new[b]] for b in range(3)])
                q, k, v = rows.split([n_q, n_kv, n_kv], 1)
                out = cache.attend(layer, cache.write(layer, q, k, v, cos, sin))
                at = 0
                for b in range(3):
                    got[b, layer].append(out[at:at + new[b]])
                    at += new[b]
            cache.commit()
            done = [d + n for d, n in zip(done, new)]
        assert cache.ctx_len.tolist() == total + [0]
        if rnd == 0:
            left = cache.n_free.item()
            cache.release([0, 2])
            assert cache.n_free.item() == left + 19 + 3
            cache.release([1])
            assert cache.n_free.item() == 40
            got = {key: [] for key in x}
    for (b, layer), rows in got.items():
        q, k, v = x[b, layer].split([n_q, n_kv, n_kv], 1)

        def turned(y):
            y = y.float()
            return (y * cos[:len(y), None] + torch.cat([-y[..., 64:], y[..., :64]], -1) * sin[:len(y), None]).bfloat16()

        out, _, tol, _ = exact(turned(q), turned(k), v)
        # a rotation rounded the other way moves q or k by 2 u: scores by 4 u S, and so the weights
        assert ((torch.cat(rows).double() - out).abs() <= tol + 0.05).all()
    with pytest.raises(RuntimeError, match="does not fit"):
        cache.begin([0, 0, 0, 400], 400)
        cache.check()
