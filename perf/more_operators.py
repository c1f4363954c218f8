"""Measured cases of the operators of a batched decode step beyond the attention.

Three operators that a server of many requests calls for every generated token:

* moe      a sparse MLP of a few tokens: router, choice of experts, their gated
           products and the weighted sum (kernels.moe_layer);
* select   beam search's choice of the best continuations over the beams and the
           vocabulary of each request (kernels.beam_select);
* reorder  the cache rows of each request's beams become copies of their parents':
           block tables and counts of shared pages, pages given back, and copies of
           last pages that are not full (kernels.paged_reorder).

``run`` computes them in elementary torch operations, or, where ``own`` is
true, with the calls of this package.  A case is a dict of plain values; lists of
lengths are texts ("17,1,300").
"""
import math
import os
import sys

import torch

own = False

D = 128
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


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
    return [
        # one token through a small sparse MLP: latency
        {"name": "moe 1 of 16 experts", "op": "moe", "tokens": 1, "hidden": 1024, "inter": 512, "experts": 16, "top_k": 2,
         "norm": True, "dtype": "f16"},
        # one generated token of one sequence, many small experts: the weights of eight of them are the work
        {"name": "moe 1 of 128 experts", "op": "moe", "tokens": 1, "hidden": 2048, "inter": 768, "experts": 128, "top_k": 8,
         "norm": True, "dtype": "bf16"},
        # seven sequences, sizes that fill no tile, weights that are not normalised
        {"name": "moe 7 odd sizes", "op": "moe", "tokens": 7, "hidden": 1544, "inter": 1000, "experts": 60, "top_k": 5,
         "norm": False, "dtype": "f16"},
        # a batched decode step with few large experts
        {"name": "moe 32 of 8 large", "op": "moe", "tokens": 32, "hidden": 4096, "inter": 14336, "experts": 8, "top_k": 2,
         "norm": True, "dtype": "bf16"},
        # 16 requests of 8 beams each: nearly every expert has tokens
        {"name": "moe 128 of 128 experts", "op": "moe", "tokens": 128, "hidden": 4096, "inter": 1408, "experts": 128,
         "top_k": 8, "norm": True, "dtype": "bf16"},
        # one request of 4 beams: latency
        {"name": "select 1x4", "op": "select", "batch": 1, "beams": 4, "vocab": 32000, "pad": 0, "eos": 1, "allowed": 0,
         "first": False, "dtype": "f32"},
        # an odd vocabulary in padded rows, two ends of sequence
        {"name": "select 6x5 odd", "op": "select", "batch": 6, "beams": 5, "vocab": 50257, "pad": 47, "eos": 2, "allowed": 0,
         "first": False, "dtype": "bf16"},
        # decoding held to a grammar: all but a few tokens are masked, the first step (one beam of each request counts)
        {"name": "select 24x8 masked", "op": "select", "batch": 24, "beams": 8, "vocab": 128256, "pad": 0, "eos": 1,
         "allowed": 11, "first": True, "dtype": "f16"},
        # the vocabulary of the benchmarked model for 64 requests of 8 beams: bandwidth
        {"name": "select 64x8", "op": "select", "batch": 64, "beams": 8, "vocab": 128256, "pad": 0, "eos": 1, "allowed": 0,
         "first": False, "dtype": "f32"},
        # a prompt of 1000 tokens becomes four beams, in a cache of 32 layers: latency
        {"name": "reorder fork 1x4", "op": "reorder", "kind": "fork", "ctx": "1000", "made": 0, "beams": 4, "page": 64,
         "layers": 32, "n_kv": 8, "dtype": "bf16"},
        # long sequences in small pages: the tables are the work
        {"name": "reorder 8x8 long", "op": "reorder", "kind": "beams",
         "ctx": _text([32000 - 1777 * i for i in range(8)]), "made": 300, "beams": 8, "page": 16, "layers": 2, "n_kv": 2,
         "dtype": "f16"},
        # 16 requests of 4 beams, some of which have ended, in a cache of 32 layers: the copies are the work
        {"name": "reorder 16x4", "op": "reorder", "kind": "ended", "ctx": _text([290 + 37 * i for i in range(16)]),
         "made": 150, "beams": 4, "page": 64, "layers": 32, "n_kv": 8, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["moe", "moe", "select", "reorder"])
    if op == "moe":
        while True:
            experts = rng.choice([4, 8, 16, 60, 64, 128, 160])
            case = {"op": "moe", "tokens": _log(rng, 1, 128), "hidden": 8 * _log(rng, 64, 512), "inter": 8 * _log(rng, 16, 1792),
                    "experts": experts, "top_k": rng.randint(1, min(8, experts)), "norm": rng.random() < 0.7,
                    "dtype": rng.choice(["f16", "bf16"])}
            if experts * case["hidden"] * case["inter"] <= 128 * 4096 * 1408:
                return case
    if op == "select":
        while True:
            vocab = rng.choice([32000, 32001, 50257, 128256, 151936, _log(rng, 300, 200000)])
            case = {"op": "select", "batch": _log(rng, 1, 64), "beams": _log(rng, 1, 16), "vocab": vocab,
                    "pad": rng.choice([0, 0, 1, 64]), "eos": rng.choice([0, 1, 1, 2]),
                    "allowed": rng.choice([0, 0, 0, _log(rng, 1, 200)]), "first": rng.random() < 0.2,
                    "dtype": rng.choice(["f32", "f16", "bf16"])}
            if case["batch"] * case["beams"] * vocab <= 512 * 128256:
                return case
    while True:
        kind = rng.choice(["beams", "beams", "fork", "ended"])
        case = {"op": "reorder", "kind": kind, "ctx": _text([_log(rng, 1, 16000) for _ in range(_log(rng, 1, 32))]),
                "made": 0 if kind == "fork" else _log(rng, 1, 400), "beams": _log(rng, 2, 16), "page": rng.choice([16, 32, 64, 128]),
                "layers": _log(rng, 1, 32), "n_kv": rng.choice([1, 2, 4, 8]), "dtype": rng.choice(["f16", "bf16"])}
        last = _reorder_pages(case) * case["page"] * case["layers"] * case["n_kv"] * D * 4
        if last <= 3 << 30:  # bytes of the pool
            return case


def _reorder_pages(case):
    """Pages that a reorder case's pool has."""
    p, k = case["page"], case["beams"]
    return sum(c // p + k * (-(-(c + case["made"]) // p) - c // p + 1) for c in _ints(case["ctx"])) + 5


# -------------------------------------------------------------------- work --


def work(case):
    size = DT[case["dtype"]].itemsize
    if case["op"] == "moe":
        t, h, i, e, k = (case[x] for x in ("tokens", "hidden", "inter", "experts", "top_k"))
        used = min(e * (1.0 - (1.0 - k / e) ** t), t * k)  # experts that any token goes to, if it chooses evenly
        return {"bytes": size * (used * 3 * h * i + e * h + 2 * t * h) + 8 * t * k, "flops": 2 * t * (e * h + k * 3 * h * i)}
    if case["op"] == "select":
        rows, n = case["batch"] * case["beams"], _candidates(case)
        return {"bytes": rows * (case["vocab"] * size + 16) + 12 * case["batch"] * n, "flops": 3 * rows * case["vocab"]}
    p, k, made = case["page"], case["beams"], case["made"]
    copied = entries = 0
    for c in _ints(case["ctx"]):
        n = c + made
        if case["kind"] == "fork":
            copied += (k - 1) * (n % p)
            entries += k * -(-n // p)
        else:  # of k beams with a parent drawn evenly each, those that are not their parent's first child
            kept = k * (1.0 - (1.0 - 1.0 / k) ** k)
            copied += (k - kept) * (n % p) * (0.75 if case["kind"] == "ended" else 1.0)
            entries += 2 * k * -(-n // p)
    token = case["layers"] * case["n_kv"] * D * 2 * size
    return {"bytes": 2 * copied * token + 4 * entries + 16 * k * len(_ints(case["ctx"])), "flops": entries}


def _candidates(case):
    return case["beams"] * (1 + case["eos"])


# ------------------------------------------------------------------ inputs --


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]
    s = {"case": dict(case)}
    i32 = dict(dtype=torch.int32, device="cuda")

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "moe":
        t, h, i, e = (case[x] for x in ("tokens", "hidden", "inter", "experts"))
        # normalised rows, a few channels much larger than the others
        x = randn(t, h)
        x[:, torch.randint(0, h, (4,), device="cuda", generator=g)] *= 6.0
        s["x"] = x.to(dt)
        s["router"] = (randn(e, h) * (1.2 / math.sqrt(h))).to(dt)
        s["gate_up"] = torch.empty(e, 2 * i, h, dtype=dt, device="cuda").normal_(0.0, 1.0 / math.sqrt(h), generator=g)
        s["down"] = torch.empty(e, h, i, dtype=dt, device="cuda").normal_(0.0, 1.0 / math.sqrt(i), generator=g)
        return s
    if case["op"] == "select":
        b, k, v = case["batch"], case["beams"], case["vocab"]
        rows = randn(b * k, v + case["pad"]) * (1.5 + 1.5 * torch.rand(b * k, 1, device="cuda", generator=g))
        # a model is sure of a few tokens
        likely = torch.randint(0, v, (b * k, 6), device="cuda", generator=g)
        rows.scatter_add_(1, likely, 8.0 * torch.rand(b * k, 6, device="cuda", generator=g))
        if case["allowed"]:
            keep = torch.randint(0, v, (b * k, case["allowed"]), device="cuda", generator=g)
            rows = torch.full_like(rows, -math.inf).scatter_(1, keep, rows.gather(1, keep))
        s["logits"] = rows.to(dt)[:, :v]
        s["scores"] = (-12.0 * torch.rand(b, k, device="cuda", generator=g)).sort(dim=1, descending=True)[0]
        if case["first"]:
            s["scores"] = torch.full_like(s["scores"], -math.inf)
            s["scores"][:, 0] = 0.0
        s["eos"] = tuple(range(2, 2 + case["eos"]))
        return s
    ctx, k, p, made = _ints(case["ctx"]), case["beams"], case["page"], case["made"]
    b, n_pages = len(ctx), _reorder_pages(case)
    perm = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    lens = torch.tensor([c + made for c in ctx], device="cuda")
    cols = -(-(max(ctx) + made) // p) + 3
    j = torch.arange(cols, device="cuda")
    own_from = torch.tensor([c // p for c in ctx], device="cuda")[:, None, None]  # first page that beams do not all share
    held = ((lens + p - 1) // p)[:, None, None]
    beam = torch.arange(k, device="cuda")[None, :, None]
    # whose page a beam has: the prompt's, its pair's while the two had one past, at last its own
    whose = torch.where(j < own_from, 0, torch.where((j < held - 1) & (j < own_from + 3), beam // 2 * 2, beam))
    if case["kind"] == "fork":
        whose = whose.clamp(max=0)
    live = (j < held) & ((beam == 0) | (case["kind"] != "fork"))
    first = live & (whose == beam)  # one number for each page that there is
    number = (first.reshape(-1).cumsum(0) - 1).view(b, k, cols)
    table = torch.where(live, perm[number.gather(1, whose.expand(b, k, cols)).clamp(min=0)], -1).view(b * k, cols)
    taken = first.sum()
    # the rows of a request lie anywhere in the table
    order = torch.randperm(b * k, device="cuda", generator=g)
    s["table"] = torch.full((b * k, cols), -1, **i32)
    s["table"][order] = table.to(torch.int32)
    s["rows"] = order.to(torch.int32).view(b, k)
    s["ctx"] = torch.zeros(b * k, **i32)
    s["ctx"][order] = (lens[:, None] * live[:, :, 0]).reshape(-1).to(torch.int32)
    s["shared"] = (torch.bincount(table[table >= 0].long(), minlength=n_pages) - 1).clamp(min=0).to(torch.int32)
    s["n_free"] = (n_pages - taken).to(torch.int32).view(1)
    s["free"] = torch.cat([perm[taken:], perm[:taken]])  # behind the free pages the list's entries mean nothing
    s["parents"] = torch.randint(0, k, (b, k), generator=g, **i32)
    if case["kind"] == "fork":
        s["parents"].zero_()
    if case["kind"] == "ended":
        s["parents"][torch.rand(b, device="cuda", generator=g) < 0.25] = -1
    shape = (case["layers"], n_pages, p, case["n_kv"], D)
    s["k"] = torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g)
    s["v"] = torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g)
    return s


# --------------------------------------------------------------------- run --


def _moe_plain(s):
    case, x = s["case"], s["x"].float()
    t, k, e = case["tokens"], case["top_k"], case["experts"]
    # in 64 bits: the last chosen and the first left out lie close together
    logits = s["x"].double() @ s["router"].double().t()
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    ids = logits.sort(dim=1, descending=True, stable=True)[1][:, :k]
    w = p.gather(1, ids)
    if case["norm"]:
        w = w / w.sum(1, keepdim=True)
    w = w.float()

    def gated(rows, gate_up):
        gate, up = (rows @ gate_up.float().transpose(1, 2)).chunk(2, -1)
        return gate / (1.0 + torch.exp(-gate)) * up

    if t * k <= e:  # the chosen experts' weights, once for each choice
        at = ids.reshape(-1)
        rows = x.repeat_interleave(k, 0)[:, None]
        y = gated(rows, s["gate_up"][at]) @ s["down"][at].float().transpose(1, 2)
        y = (y.view(t, k, -1) * w[..., None]).sum(1)
    else:  # every expert over all tokens
        dense = torch.zeros(t, e, device="cuda").scatter_(1, ids, w)
        y = gated(x.expand(e, -1, -1), s["gate_up"]) * dense.t()[..., None]
        y = (y @ s["down"].float().transpose(1, 2)).sum(0)
    return {"y": y.to(s["x"].dtype), "ids": ids.to(torch.int32), "weights": w}


def _select_plain(s):
    case, cum = s["case"], s["scores"].double()
    b, k, n = case["batch"], case["beams"], _candidates(case)
    lg = s["logits"].double()
    m = lg.amax(1, keepdim=True)
    lse = torch.log(torch.exp(lg - m).sum(1, keepdim=True)) + m
    n_row = min(n, case["vocab"])
    # of each beam the best n, the lowest tokens first where they are equal
    best, token = s["logits"].sort(dim=1, descending=True, stable=True)
    best, token = best[:, :n_row].double(), token[:, :n_row]
    score = (cum.view(-1, 1) + (best - lse)).view(b, -1)
    beam = torch.arange(k, device="cuda").repeat_interleave(n_row).expand(b, -1)
    token = token.reshape(b, -1)
    score, at = torch.where(score.isfinite(), score, -math.inf).sort(dim=1, descending=True, stable=True)
    score, at = score[:, :n], at[:, :n]
    real = score > -math.inf
    score = torch.nn.functional.pad(score, (0, n - score.shape[1]), value=-math.inf).float()
    beam, token = (torch.nn.functional.pad(torch.where(real, x.gather(1, at), -1), (0, n - at.shape[1]), value=-1).to(torch.int32)
                   for x in (beam, token))
    # the first that do not end a sequence go on
    ended = (token[..., None] == torch.tensor(s["eos"], dtype=torch.int32, device="cuda")).any(-1)
    on = ((token < 0) | ended).to(torch.int32).sort(dim=1, stable=True)
    stop, first = on[0][:, :k] > 0, on[1][:, :k]
    return {"scores": score, "beams": beam, "tokens": token,
            "next_scores": torch.where(stop, -math.inf, score.gather(1, first)),
            "next_beams": torch.where(stop, -1, beam.gather(1, first)), "next_tokens": torch.where(stop, -1, token.gather(1, first))}


def _reorder_plain(s):
    case, table, rows = s["case"], s["table"], s["rows"].reshape(-1).long()
    p, k, shared, free = case["page"], case["beams"], s["shared"], s["free"]
    n, n_pages, cols = rows.numel(), shared.numel(), table.shape[1]
    parent = s["parents"].reshape(-1).long()
    live = parent >= 0
    parent = torch.arange(n, device="cuda") // k * k + parent.clamp(min=0)
    j = torch.arange(cols, device="cuda")
    had = s["ctx"][rows]
    old = torch.where(j < ((had + p - 1) // p)[:, None], table[rows], -1)
    new = torch.where(live[:, None], old[parent], -1)
    now = torch.where(live, had[parent], 0)
    # holders of each page beyond its first; one place more for entries without a page
    count = torch.cat([shared, shared.new_zeros(1)])
    one = torch.ones_like(old)
    count.index_add_(0, torch.where(old < 0, n_pages, old).view(-1), -one.view(-1))
    count.index_add_(0, torch.where(new < 0, n_pages, new).view(-1), one.view(-1))
    # pages that nothing holds any more go to the end of the list, in the order of rows and columns
    at = torch.where(old < 0, n_pages, old).view(-1).long()
    place = torch.arange(at.numel(), device="cuda")
    first = torch.full((n_pages + 1,), at.numel(), device="cuda").scatter_reduce_(0, at, place, "amin")
    gone = (at < n_pages) & (count[at] < 0) & (first[at] == place)
    to = torch.where(gone, s["n_free"] + gone.cumsum(0) - 1, n_pages)
    free = torch.cat([free, free.new_zeros(1)]).index_put_((to,), at.to(torch.int32))[:n_pages]
    n_free = s["n_free"] + gone.sum()
    count = count[:n_pages].clamp(min=0)
    # a last page that is not full has one row: the parent's first child keeps it, the others get copies
    last = ((now - 1) // p).clamp(min=0).long()
    page = new.gather(1, last[:, None])[:, 0].long()
    part = live & (now % p > 0) & (page >= 0)
    same = (parent[:, None] == parent) & part[:, None] & part
    rank = (same & (torch.arange(n, device="cuda") < torch.arange(n, device="cuda")[:, None])).sum(1)
    outside = count[page.clamp(min=0)] + 1 > same.sum(1)
    copy = part & ((rank > 0) | outside)
    nth = copy.cumsum(0) - 1
    have = nth < n_free
    fresh = free[(n_free - 1 - nth).clamp(min=0)]
    count.index_add_(0, page[copy], -torch.ones_like(count[:1]).expand(int(copy.sum())))
    new.scatter_(1, last[:, None], torch.where(copy, torch.where(have, fresh, -1), new.gather(1, last[:, None])[:, 0])[:, None])
    moved = copy & have
    src, dst, upto = page[moved], fresh[moved].long(), (now % p)[moved]
    mine = (torch.arange(p, device="cuda") < upto[:, None])[None, :, :, None, None]
    s["k"][:, dst] = torch.where(mine, s["k"][:, src], s["k"][:, dst])
    s["v"][:, dst] = torch.where(mine, s["v"][:, src], s["v"][:, dst])
    now = torch.where(copy & ~have, last.to(torch.int32) * p, now)
    wide = torch.maximum((had + p - 1) // p, (now + p - 1) // p)[:, None]
    table[rows] = torch.where(j < wide, new, table[rows])
    s["ctx"][rows] = now
    s["shared"].copy_(count)
    s["free"].copy_(free)
    s["info"] = torch.stack([(copy & ~have).sum(), moved.sum(), gone.sum(), gone.sum() * 0]).to(torch.int32)
    s["n_free"].copy_((n_free - copy.sum()).clamp(min=0))
    return _reorder_out(s)


def _reorder_out(s):
    return {x: s[x] for x in ("table", "ctx", "shared", "free", "n_free", "info", "k", "v")}


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"moe": _moe_plain, "select": _select_plain, "reorder": _reorder_plain}[case["op"]](s)
    K = _kernels()
    if case["op"] == "moe":
        y, ids, weights = K.moe_layer(s["x"], s["router"], s["gate_up"], s["down"], case["top_k"], norm_topk=case["norm"],
                                      return_routing=True)
        return {"y": y, "ids": ids, "weights": weights}
    if case["op"] == "select":
        st = K.beam_select(s["logits"], s["scores"], eos=s["eos"])
        return {x: getattr(st, x) for x in ("scores", "beams", "tokens", "next_scores", "next_beams", "next_tokens")}
    s["info"] = K.paged_reorder(s["table"], s["ctx"], s["shared"], s["free"], s["n_free"], s["rows"], s["parents"], s["k"], s["v"])
    return _reorder_out(s)


# ------------------------------------------------------------------- exact --


def exact(case, seed):
    if case["op"] == "reorder":
        return None  # whole numbers and copies: they have to be equal
    s = prepare(case, seed)
    if case["op"] == "moe":
        x, h = s["x"].double(), s["x"].shape[1]
        z = torch.einsum("th,eh->te", x, s["router"].double())
        lse = torch.logsumexp(z, 1)
        chosen = [sorted(range(case["experts"]), key=lambda e: (-row[e], e))[:case["top_k"]] for row in z.tolist()]
        ids = torch.tensor(chosen, device="cuda")
        w = torch.exp(z.gather(1, ids) - (torch.logsumexp(z.gather(1, ids), 1) if case["norm"] else lse)[:, None])
        y = torch.zeros(case["tokens"], h, dtype=torch.float64, device="cuda")
        for e in sorted({e for c in chosen for e in c}):
            t, n = (ids == e).nonzero(as_tuple=True)
            gate, up = s["gate_up"][e].double().view(2, -1, h)
            a = x[t] @ gate.t()
            y.index_add_(0, t, w[t, n, None] * ((a * torch.sigmoid(a) * (x[t] @ up.t())) @ s["down"][e].double().t()))
        return {"y": y, "ids": None, "weights": w}
    b, k, v, n = case["batch"], case["beams"], case["vocab"], _candidates(case)
    scores, nexts = [], []
    for i in range(b):
        z = torch.log_softmax(s["logits"][i * k:(i + 1) * k].double(), 1) + s["scores"][i].double()[:, None]
        z = torch.where(z.isfinite(), z, -math.inf)
        best = torch.topk(z.view(-1), min(n, k * v))[0]
        scores.append(torch.cat([best, best.new_full((n - best.numel(),), -math.inf)]))
        z[:, [e for e in s["eos"] if e < v]] = -math.inf
        # a sequence that goes on is among the n best of all
        best = torch.topk(z.view(-1), min(k, k * v))[0]
        nexts.append(torch.cat([best, best.new_full((k - best.numel(),), -math.inf)]))
    return {"scores": torch.stack(scores), "beams": None, "tokens": None, "next_scores": torch.stack(nexts), "next_beams": None,
            "next_tokens": None}
