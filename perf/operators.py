"""Measured cases of the paged-cache serving operators.

Four operators that a server of many requests calls in this order:

* map     block tables and slot maps from request lengths (kernels.paged_map):
          pages for the new tokens of every request, the position and the cache
          slot of each new token, and the attention plan of the step;
* write   RoPE of the new q and k and the scatter of k and v into their pages
          (kernels.paged_write);
* paged   attention of each request's new tokens (one, or a chunk) over its
          pages (kernels.paged_attn);
* prompt  causal attention over whole packed prompts with grouped heads
          (kernels.prompt_attn).

``run`` computes them in elementary torch operations in 32 bits, or, where
``own`` is true, with the calls of this package.  A case is a dict of plain
values; lists of lengths are texts ("17,1,300").  head_dim is 128 throughout.
"""
import math
import os
import sys

import torch

own = False

D = 128
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _kernels():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rina-1bit-kv_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from kvr_b200 import kernels
    return kernels


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(ns):
    return ",".join(str(n) for n in ns)


# ------------------------------------------------------------------- cases --


def listed():
    ragged = [1, 700, 33, 64, 257, 1, 128, 1000, 5, 411, 63, 65, 2, 900, 129, 337]  # 4096 tokens
    mixed_new = [701] + [1] * 20 + [17, 64, 3]
    mixed_ctx = [1500] + [37 + 193 * i for i in range(20)] + [0, 4000, 129]
    prompts_new = [(37 * i * i + 211 * i) % 1999 + 1 for i in range(48)]
    return [
        # a decode step of the batched serving shape: 32 sequences near 16384 tokens, one new token each
        {"name": "map decode 32", "op": "map", "ctx": _text([16383 - 61 * i for i in range(32)]), "new": _text([1] * 32),
         "page": 64, "spare": 3, "n_q": 32, "n_kv": 8},
        # admission of 48 prompts of very different lengths, a third of them after a prefix that is already cached
        {"name": "map prompts 48", "op": "map", "ctx": _text([(97 * i) % 1500 if i % 3 == 0 else 0 for i in range(48)]),
         "new": _text(prompts_new), "page": 16, "spare": 100, "n_q": 32, "n_kv": 8},
        # one generated token of one sequence: latency
        {"name": "write 1", "op": "write", "tokens": 1, "pad": 0, "page": 64, "n_q": 32, "n_kv": 8, "dtype": "bf16"},
        # an odd number of tokens with padding at the end, 64 query heads on 8 KV heads
        {"name": "write 2047 f16", "op": "write", "tokens": 2047, "pad": 41, "page": 16, "n_q": 64, "n_kv": 8,
         "dtype": "f16"},
        # a whole 16384-token prompt written at once
        {"name": "write 16384", "op": "write", "tokens": 16384, "pad": 0, "page": 64, "n_q": 32, "n_kv": 8,
         "dtype": "bf16"},
        # one token of one sequence over 4096 cached tokens: latency
        {"name": "paged decode 1x4096", "op": "paged", "ctx": "4095", "new": "1", "page": 64, "n_q": 32, "n_kv": 8,
         "dtype": "f16", "window": 0, "lse": False},
        # the batched decode shape, 32 sequences of 16384 tokens: bandwidth
        {"name": "paged decode 32x16384", "op": "paged", "ctx": _text([16383] * 32), "new": _text([1] * 32), "page": 64,
         "n_q": 32, "n_kv": 8, "dtype": "bf16", "window": 0, "lse": False},
        # a chunk of 512 prompt tokens after 32256 cached ones
        {"name": "paged chunk 512 at 32256", "op": "paged", "ctx": "32256", "new": "512", "page": 64, "n_q": 32, "n_kv": 8,
         "dtype": "bf16", "window": 0, "lse": False},
        # decode rows, a chunk, a first chunk and ragged pages in one call, a sliding window, log-sum-exps for a merge
        {"name": "paged mixed 24 window", "op": "paged", "ctx": _text(mixed_ctx), "new": _text(mixed_new), "page": 16,
         "n_q": 32, "n_kv": 8, "dtype": "f16", "window": 1024, "lse": True},
        # 16 packed prompts of odd lengths, the shortest of one token
        {"name": "prompt ragged 4096", "op": "prompt", "lens": _text(ragged), "n_q": 32, "n_kv": 8, "dtype": "f16",
         "window": 0, "lse": True},
        # two prompts with a window of 1024 and 8 query heads per KV head
        {"name": "prompt window 2x4097", "op": "prompt", "lens": "4097,4095", "n_q": 64, "n_kv": 8, "dtype": "bf16",
         "window": 1024, "lse": False},
        # one long prompt: the tensor cores' rate
        {"name": "prompt 16384", "op": "prompt", "lens": "16384", "n_q": 32, "n_kv": 8, "dtype": "bf16", "window": 0,
         "lse": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _split(rng, total, parts):
    """`total` tokens in `parts` pieces of uneven sizes, one token at least in each."""
    parts = max(1, min(parts, total))
    cuts = sorted(rng.sample(range(1, total), parts - 1)) if parts > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    op = rng.choice(["map", "write", "paged", "paged", "paged", "prompt", "prompt"])
    n_q, n_kv = rng.choice([(32, 8), (64, 8), (8, 2), (8, 8), (6, 2), (28, 4)])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    window = rng.choice([0, 0, 256, 512, 1024])
    if op == "map":
        if rng.random() < 0.5:  # decode: one new token each, some requests idle
            b = _log(rng, 1, 512)
            new = [0 if rng.random() < 0.1 else 1 for _ in range(b)]
            new[rng.randrange(b)] = 1
            ctx = [_log(rng, 1, 16384) for _ in range(b)]
        else:
            new = _split(rng, _log(rng, 2, 65536), _log(rng, 1, 64))
            ctx = [0 if rng.random() < 0.6 else _log(rng, 1, 4096) for _ in new]
        return {"op": "map", "ctx": _text(ctx), "new": _text(new), "page": page, "spare": rng.randrange(200), "n_q": n_q,
                "n_kv": n_kv}
    if op == "write":
        tokens = _log(rng, 1, 12288)
        return {"op": "write", "tokens": tokens, "pad": rng.randrange(1 + tokens // 8), "page": page, "n_q": n_q,
                "n_kv": n_kv, "dtype": dtype}
    if op == "paged":
        if rng.random() < 0.5:  # decode, with a few tokens each where they are drafted
            b, longest = _log(rng, 1, 32), _log(rng, 16, 12000)
            ctx = [rng.randrange(longest // 3, longest) for _ in range(b)]
            most = rng.choice([1, 1, 4])
            new = [rng.randint(1, most) for _ in range(b)]
        else:  # chunks, some requests of the step decoding beside them
            first = _log(rng, 2, 1024)
            ctx = [_log(rng, 1, 16384 if first <= 512 else 6000)]
            new = [first]
            for _ in range(rng.choice([0, 0, 1, 3])):
                ctx.append(rng.randrange(0, 3000))
                new.append(rng.choice([1, 1, 1 + rng.randrange(first)]))
            if n_q > 32:
                n_q = 32
        return {"op": "paged", "ctx": _text(ctx), "new": _text(new), "page": page, "n_q": n_q, "n_kv": n_kv, "dtype": dtype,
                "window": window, "lse": rng.random() < 0.3}
    total = _log(rng, 1, 8192 if n_q > 32 else 12288)
    return {"op": "prompt", "lens": _text(_split(rng, total, _log(rng, 1, 16))), "n_q": n_q, "n_kv": n_kv, "dtype": dtype,
            "window": window, "lse": rng.random() < 0.3}


# -------------------------------------------------------------------- work --


def _pairs(q_len, kv_len, window):
    """(query, key) pairs that a causal request has, its queries being its last tokens."""
    first = kv_len - q_len + 1  # keys that the first query sees
    if window <= 0 or window >= kv_len:
        return q_len * first + q_len * (q_len - 1) // 2
    short = max(0, min(q_len, window - first))  # queries that see fewer keys than the window
    return short * first + short * (short - 1) // 2 + (q_len - short) * window


def _span(q_len, kv_len, window):
    """Keys of a request that any of its queries sees."""
    return kv_len if window <= 0 else min(kv_len, q_len - 1 + window)


def work(case):
    n_q, n_kv = case["n_q"], case["n_kv"]
    if case["op"] == "map":
        ctx, new, p = _ints(case["ctx"]), _ints(case["new"]), case["page"]
        fresh = sum(-(-(c + n) // p) - -(-c // p) for c, n in zip(ctx, new))
        touched = sum(-(-(c + n) // p) - c // p for c, n in zip(ctx, new) if n)
        # lengths in, kv lengths and offsets out; position (4) and slot (8) of a token; a page id from the free list to the table
        return {"bytes": 16 * len(ctx) + 12 * sum(new) + 8 * fresh + 4 * (touched - fresh), "flops": 4 * sum(new)}
    if case["op"] == "write":
        t = case["tokens"]
        real = t - case["pad"]
        # q in and out, k and v in and out, half rows of two tables, position and slot
        return {"bytes": t * (n_q * D * 4 + 12) + real * (n_kv * D * 8 + D * 4), "flops": 3 * real * (n_q + n_kv) * D}
    if case["op"] == "paged":
        new = _ints(case["new"])
        kv = [c + n for c, n in zip(_ints(case["ctx"]), new)]
    else:
        new = kv = _ints(case["lens"])
    pairs = sum(_pairs(n, k, case["window"]) for n, k in zip(new, kv))
    span = sum(_span(n, k, case["window"]) for n, k in zip(new, kv))
    io = sum(new) * n_q * (D * 4 + (4 if case["lse"] else 0))
    table = 4 * sum(-(-k // case["page"]) for k in kv) if case["op"] == "paged" else 0
    return {"bytes": io + span * n_kv * D * 4 + table, "flops": 4 * D * n_q * pairs}


# ------------------------------------------------------------------ inputs --


def _offsets(ns):
    out = [0]
    for n in ns:
        out.append(out[-1] + n)
    return out


def _key_scale(g, n_kv):
    """Keys differ in scale from channel to channel, and a few channels are much larger."""
    s = torch.exp(0.5 * torch.randn(n_kv, D, device="cuda", generator=g))
    s.scatter_(1, torch.randint(0, D, (n_kv, 4), device="cuda", generator=g), 5.0)
    return s


def _pages(g, ctx, new, page):
    """A pool in which every request's pages lie anywhere: (table (B, width), pages in the pool)."""
    need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    width, total = max(max(need), 1), sum(need) + 7
    perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    j = torch.arange(width, device="cuda")
    start = torch.tensor(_offsets(need)[:-1], device="cuda")
    have = torch.tensor(need, device="cuda")
    at = (start[:, None] + j).clamp(max=total - 1)
    return torch.where(j < have[:, None], perm[at], torch.full_like(perm[at], -1)), total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_q, n_kv = case["n_q"], case["n_kv"]
    s = {"case": dict(case)}
    i32 = dict(dtype=torch.int32, device="cuda")
    if case["op"] == "map":
        ctx, new, p = _ints(case["ctx"]), _ints(case["new"]), case["page"]
        had, now = [-(-c // p) for c in ctx], [-(-(c + n) // p) for c, n in zip(ctx, new)]
        fresh = sum(now) - sum(had)
        pool = torch.randperm(sum(now) + case["spare"], device="cuda", generator=g).to(torch.int32)
        width = max(now) + 2
        j = torch.arange(width, device="cuda")
        at = torch.tensor(_offsets(had)[:-1], device="cuda")[:, None] + j
        held = pool[at.clamp(max=pool.numel() - 1)]
        s["table"] = torch.where(j < torch.tensor(had, device="cuda")[:, None], held, torch.full_like(held, -1))
        s["free"] = pool[sum(had):].clone()
        s["n_free"] = torch.tensor([fresh + case["spare"]], **i32)
        s["ctx"], s["new"], s["tokens"] = torch.tensor(ctx, **i32), torch.tensor(new, **i32), sum(new)
        return s
    dt = DT[case["dtype"]]
    if case["op"] == "write":
        t, p = case["tokens"], case["page"]
        qkv = torch.randn(t, n_q + 2 * n_kv, D, device="cuda", generator=g)
        qkv[:, n_q:n_q + n_kv] *= _key_scale(g, n_kv)
        # one projection's output: q, k and v are strided views of it
        s["q"], s["k"], s["v"] = qkv.to(dt).split([n_q, n_kv, n_kv], dim=1)
        n_pages = -(-t // p) + 5
        s["kp"] = torch.randn(n_pages, p, n_kv, D, device="cuda", generator=g).to(dt)
        s["vp"] = torch.randn(n_pages, p, n_kv, D, device="cuda", generator=g).to(dt)
        order = torch.randperm(n_pages, device="cuda", generator=g)
        i = torch.arange(t, device="cuda")
        s["slots"] = order[i // p] * p + i % p
        s["slots"][t - case["pad"]:] = -1
        s["pos"] = (i + int(torch.randint(0, 8192, (1,), device="cuda", generator=g))).to(torch.int32)
        inv = 500000.0 ** (-torch.arange(0, D, 2, device="cuda").float() / D)
        a = torch.arange(32768, device="cuda").float()[:, None] * inv
        s["cos"], s["sin"] = torch.cat([a.cos()] * 2, 1), torch.cat([a.sin()] * 2, 1)
        return s
    if case["op"] == "paged":
        ctx, new, p = _ints(case["ctx"]), _ints(case["new"]), case["page"]
        kv = [c + n for c, n in zip(ctx, new)]
        s["table"], n_pages = _pages(g, ctx, new, p)
        s["q"] = torch.randn(sum(new), n_q, D, device="cuda", generator=g).to(dt)
        s["kp"] = (torch.randn(n_pages, p, n_kv, D, device="cuda", generator=g) * _key_scale(g, n_kv)).to(dt)
        s["vp"] = torch.randn(n_pages, p, n_kv, D, device="cuda", generator=g).to(dt)
        s["kv_len"], s["max_q"], s["max_k"] = torch.tensor(kv, **i32), max(new), max(kv)
    else:
        new = _ints(case["lens"])
        qkv = torch.randn(sum(new), n_q + 2 * n_kv, D, device="cuda", generator=g)
        qkv[:, n_q:n_q + n_kv] *= _key_scale(g, n_kv)
        s["q"], s["k"], s["v"] = qkv.to(dt).split([n_q, n_kv, n_kv], dim=1)
    s["cu"] = torch.tensor(_offsets(new), **i32)
    if own:  # a step's plan is made once and serves every layer (paged_map makes it with the block tables)
        s["plan"] = _kernels().attn_plan(s["cu"], sum(new), n_q, n_kv, kv_len=s.get("kv_len"), window=case["window"])
    return s


# --------------------------------------------------------------------- run --


def _map_plain(s):
    p, table, new, ctx, tokens = s["case"]["page"], s["table"], s["new"], s["ctx"], s["tokens"]
    b = torch.arange(new.numel(), device="cuda")
    cu = torch.cat([new.new_zeros(1), new.cumsum(0).to(torch.int32)])
    kv = ctx + new
    had, now = (ctx + p - 1) // p, (kv + p - 1) // p
    fresh = now - had
    start = fresh.cumsum(0) - fresh
    j = torch.arange(table.shape[1], device="cuda")
    k = start[:, None] + j - had[:, None]
    mine = (j >= had[:, None]) & (j < now[:, None])
    table = torch.where(mine, s["free"][torch.where(mine, s["n_free"] - 1 - k, 0)], table)
    who = b.repeat_interleave(new, output_size=tokens)
    pos = torch.arange(tokens, device="cuda", dtype=torch.int32) - cu[who] + ctx[who]
    slots = table[who, pos // p].long() * p + pos % p
    return {"cu": cu, "kv_len": kv, "table": table, "pos": pos, "slots": slots,
            "n_free": (s["n_free"] - fresh.sum()).to(torch.int32)}


def _write_plain(s):
    real = s["slots"] >= 0
    at = s["slots"][real]
    c, sn = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]

    def rope(x):
        x = x.float()
        return x * c + torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1) * sn

    q = torch.where(real[:, None, None], rope(s["q"]), 0.0).to(s["q"].dtype)
    s["kp"].view(-1, *s["kp"].shape[2:])[at] = rope(s["k"])[real].to(s["k"].dtype)
    s["vp"].view(-1, *s["vp"].shape[2:])[at] = s["v"][real]
    return {"q": q, "k": s["kp"], "v": s["vp"]}


def _softmax_out(scores, seen, v):
    """(softmax(scores where seen) v, log-sum-exp), zeros and -inf where a row sees nothing."""
    scores = torch.where(seen, scores, -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    return torch.where(l > 0, p @ v / l, 0.0), (torch.log(l) + m)[..., 0]


def _seen(q_pos, k_pos, window):
    ok = k_pos <= q_pos
    return ok & (k_pos > q_pos - window) if window > 0 else ok


def _paged_plain(s):
    case, q, cu, kv = s["case"], s["q"], s["cu"], s["kv_len"]
    n_kv, p, t = case["n_kv"], case["page"], q.shape[0]
    gq = case["n_q"] // n_kv
    b = kv.numel()
    new = cu[1:] - cu[:-1]
    i = torch.arange(s["max_q"], device="cuda")
    j = torch.arange(s["max_k"], device="cuda")
    rows = (cu[:-1, None] + i).clamp(max=t - 1)  # (B, max_q) token of each padded query
    q_pos = torch.where(i < new[:, None], kv[:, None] - new[:, None] + i, -1)
    at = s["table"].clamp(min=0).long()[:, j // p] * p + j % p  # (B, max_k) cache slot of each padded key
    seen = _seen(q_pos[:, :, None], j, case["window"])[:, :, None].expand(-1, -1, gq, -1).reshape(b, -1, s["max_k"])
    who = torch.arange(b, device="cuda").repeat_interleave(new, output_size=t)
    back = torch.arange(t, device="cuda") - cu[who]
    out = torch.empty(q.shape, dtype=torch.float32, device="cuda")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    kp, vp = s["kp"].view(-1, n_kv, D), s["vp"].view(-1, n_kv, D)
    for h in range(n_kv):  # head by head: the padded scores of all heads would not fit
        heads = slice(h * gq, (h + 1) * gq)
        qh = q[:, heads][rows].float().view(b, -1, D)
        o, e = _softmax_out(qh @ kp[:, h][at].float().transpose(1, 2) / math.sqrt(D), seen, vp[:, h][at].float())
        out[:, heads] = o.view(b, -1, gq, D)[who, back]
        lse[:, heads] = e.view(b, -1, gq)[who, back]
    return (out.to(q.dtype), lse) if case["lse"] else (out.to(q.dtype),)


def _prompt_plain(s):
    case, q, cu = s["case"], s["q"], s["cu"]
    n_kv, t = case["n_kv"], q.shape[0]
    gq = case["n_q"] // n_kv
    i = torch.arange(t, device="cuda")
    who = torch.searchsorted(cu[1:], i, right=True)
    seen = (who[:, None] == who) & _seen(i[:, None], i, case["window"])
    out = torch.empty(q.shape, dtype=torch.float32, device="cuda")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    for h in range(n_kv):
        heads = slice(h * gq, (h + 1) * gq)
        qh = q[:, heads].float().transpose(0, 1)  # (gq, T, D)
        o, e = _softmax_out(qh @ s["k"][:, h].float().t() / math.sqrt(D), seen, s["v"][:, h].float())
        out[:, heads] = o.transpose(0, 1)
        lse[:, heads] = e.t()
    return (out.to(q.dtype), lse) if case["lse"] else (out.to(q.dtype),)


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"map": _map_plain, "write": _write_plain, "paged": _paged_plain, "prompt": _prompt_plain}[case["op"]](s)
    K = _kernels()
    if case["op"] == "map":
        st = K.paged_map(s["ctx"], s["new"], s["table"], s["free"], s["n_free"], case["page"], s["tokens"],
                         n_q=case["n_q"], n_kv=case["n_kv"])
        return {"cu": st.cu_q, "kv_len": st.kv_len, "table": s["table"], "pos": st.positions, "slots": st.slots,
                "n_free": st.n_free}
    if case["op"] == "write":
        q = K.paged_write(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["slots"], s["pos"], s["cos"], s["sin"])
        return {"q": q, "k": s["kp"], "v": s["vp"]}
    if case["op"] == "paged":
        out = K.paged_attn(s["q"], s["kp"], s["vp"], s["table"], s["plan"], return_lse=case["lse"])
    else:
        out = K.prompt_attn(s["q"], s["k"], s["v"], s["plan"], return_lse=case["lse"])
    return tuple(out) if case["lse"] else (out,)


# ------------------------------------------------------------------- exact --


def _rows_exact(q, k, v, first, window):
    """Queries q (n, g, D) at positions first, first + 1, ... over keys 0 .. of k, v (m, D), in 64 bits."""
    outs, lses = [], []
    for a in range(0, q.shape[0], 512):
        c = q[a:a + 512].double()
        i = first + a + torch.arange(c.shape[0], device="cuda")
        lo = max(0, first + a - window + 1) if window > 0 else 0
        hi = min(k.shape[0], first + a + c.shape[0])
        j = torch.arange(lo, hi, device="cuda")
        hidden = j[None] > i[:, None]
        if window > 0:
            hidden |= j[None] <= i[:, None] - window
        z = torch.einsum("ngd,md->ngm", c, k[lo:hi].double()) / math.sqrt(D)
        z.masked_fill_(hidden[:, None], -math.inf)
        lse = torch.logsumexp(z, -1)
        outs.append(torch.einsum("ngm,md->ngd", torch.exp(z - lse[..., None]), v[lo:hi].double()))
        lses.append(lse)
    return torch.cat(outs), torch.cat(lses)


def exact(case, seed):
    if case["op"] == "map":
        return None  # whole numbers: they have to be equal
    s = prepare(case, seed)
    n_q, n_kv = case["n_q"], case["n_kv"]
    if case["op"] == "write":
        live = (s["slots"] >= 0).nonzero()[:, 0]
        turn = torch.complex(s["cos"][s["pos"], :D // 2].double(), s["sin"][s["pos"], :D // 2].double())[:, None]

        def rotated(x):
            y = torch.complex(x[..., :D // 2].double(), x[..., D // 2:].double()) * turn
            return torch.cat([y.real, y.imag], -1)

        q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        q[live] = rotated(s["q"])[live]
        k, v = s["kp"].double(), s["vp"].double()
        k.view(-1, n_kv, D).index_copy_(0, s["slots"][live], rotated(s["k"])[live])
        v.view(-1, n_kv, D).index_copy_(0, s["slots"][live], s["v"].double()[live])
        return {"q": q, "k": k, "v": v}
    g = n_q // n_kv
    if case["op"] == "paged":
        new = _ints(case["new"])
        kv = [c + n for c, n in zip(_ints(case["ctx"]), new)]
    else:
        new = kv = _ints(case["lens"])
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        if case["op"] == "paged":
            pages = s["table"][b, :-(-m // case["page"])].long()
            k, v = (s[x][pages].reshape(-1, n_kv, D)[:m] for x in ("kp", "vp"))
        else:
            k, v = s["k"][at:at + n], s["v"][at:at + n]
        for h in range(n_kv):
            heads = slice(h * g, (h + 1) * g)
            out[at:at + n, heads], lse[at:at + n, heads] = _rows_exact(s["q"][at:at + n, heads], k[:, h], v[:, h], m - n,
                                                                       case["window"])
        at += n
    return (out, lse) if case["lse"] else (out,)
