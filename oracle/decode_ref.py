"""CPU specification of the operators of a decode step beyond the attention, in
numpy and 64 bits: beam search's choice of continuations, the reordering of paged
rows, and a sparse MLP.  No reference counterpart (the reference decodes one
sequence of a dense model greedily)."""
import numpy as np


def beam_select(logits, cum, n, eos=()):
    """logits (B, K, V), cum (B, K) -> dict of scores, beams, tokens (B, n), next_* (B, K)."""
    B, K, V = logits.shape
    out = {x: np.full((B, n), -np.inf if x == "scores" else -1) for x in ("scores", "beams", "tokens")}
    out.update({x: np.full((B, K), -np.inf if x == "next_scores" else -1) for x in ("next_scores", "next_beams", "next_tokens")})
    for b in range(B):
        found = []
        for k in range(K):
            x = np.asarray(logits[b, k], dtype=np.float64)
            m = x.max()  # a NaN stays one
            with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
                score = float(cum[b, k]) + (x - (m + np.log(np.exp(x - m).sum())))
                there = np.isfinite(score.astype(np.float32))  # (what is returned is fp32)
            found += [(-score[t], k, t) for t in np.nonzero(there)[0]]
        found.sort()
        on = 0
        for i, (s, k, t) in enumerate(found[:n]):
            out["scores"][b, i], out["beams"][b, i], out["tokens"][b, i] = -s, k, t
            if t not in eos and on < K:
                out["next_scores"][b, on], out["next_beams"][b, on], out["next_tokens"][b, on] = -s, k, t
                on += 1
    return out


def reorder(table, ctx, shared, free, n_free, rows, parents, page):
    """Block tables after rows[g][i] has become rows[g][parents[g][i]] -> dict of
    table, ctx, shared, free, n_free, info and copies [(from page, to page, tokens)]."""
    table, ctx, shared, free = (np.array(x, copy=True) for x in (table, ctx, shared, free))
    held = lambda c: -(-c // page)  # noqa: E731
    before = {r: (list(table[r, :held(ctx[r])]), int(ctx[r])) for g in rows for r in g}
    places = [(g, i) for g in range(len(rows)) for i in range(len(rows[g]))]
    now = {}
    for g, i in places:
        p = parents[g][i]
        now[g, i] = (list(before[rows[g][p]][0]), before[rows[g][p]][1]) if 0 <= p < len(rows[g]) else ([], 0)
    holders = shared.astype(np.int64)
    for g, i in places:
        for p in before[rows[g][i]][0]:
            holders[p] -= p >= 0
    for g, i in places:
        for p in now[g, i][0]:
            holders[p] += p >= 0
    gone = []
    for g, i in places:
        for p in before[rows[g][i]][0]:
            if p >= 0 and holders[p] < 0 and p not in gone:
                gone.append(p)
    for p in gone:
        free[n_free] = p
        n_free += 1
        holders[p] = 0
    # a last page that is not full stays with the first place that gets it, if no row outside of the call has it
    want, copies, missing = [], [], 0
    gets = {}
    for place in places:
        pages, c = now[place]
        if c % page and pages[-1] >= 0:
            gets.setdefault(pages[-1], []).append(place)
    for place in places:
        pages, c = now[place]
        if c % page and pages[-1] >= 0:
            same = gets[pages[-1]]
            if place != same[0] or holders[pages[-1]] + 1 > len(same):
                want.append(place)
    for g, i in want:
        pages, c = now[g, i]
        holders[pages[-1]] -= 1
        if n_free:
            n_free -= 1
            copies.append((pages[-1], free[n_free], c % page))
            pages[-1] = free[n_free]
        else:
            missing += 1
            pages[-1] = -1
            now[g, i] = (pages, c // page * page)
    for g, i in places:
        r = rows[g][i]
        pages, c = now[g, i]
        wide = max(len(before[r][0]), len(pages))
        table[r, :wide] = pages + [-1] * (wide - len(pages))
        ctx[r] = c
    return {"table": table, "ctx": ctx, "shared": holders.astype(np.int32), "free": free, "n_free": n_free,
            "info": np.array([missing, len(copies), len(gone), 0], np.int32), "copies": copies}


def moe(x, router, gate_up, down, top_k, norm=True, scale=1.0):
    """x (T, H), router (E, H), gate_up (E, 2 I, H), down (E, H, I) in float64 ->
    (y (T, H), ids (T, k), weights (T, k), by_h, by_sums, by_one): what errors of y
    scale with: sum of |w d h| (a relative error of h), of |w d| times the change of h
    by one unit of the absolute products of its gate and up sums, and of |w d|."""
    z = x @ router.T
    ids = np.argsort(-z, axis=1, kind="stable")[:, :top_k]
    e = np.exp(z - z.max(1, keepdims=True))
    w = np.take_along_axis(e, ids, 1)
    w = scale * w / (w.sum(1, keepdims=True) if norm else e.sum(1, keepdims=True))
    inter = gate_up.shape[1] // 2
    y, by_h, by_sums, by_one = (np.zeros((x.shape[0], down.shape[1])) for _ in range(4))
    for t in range(x.shape[0]):
        for n, ex in enumerate(ids[t]):
            gu, ab = gate_up[ex] @ x[t], np.abs(gate_up[ex]) @ np.abs(x[t])
            g, u = gu[:inter], gu[inter:]
            silu = g / (1 + np.exp(-g))
            d = np.abs(w[t, n]) * np.abs(down[ex])
            y[t] += w[t, n] * (down[ex] @ (silu * u))
            by_h[t] += d @ np.abs(silu * u)
            by_sums[t] += d @ (1.1 * ab[:inter] * np.abs(u) + np.abs(silu) * ab[inter:])  # |silu'| < 1.1
            by_one[t] += d.sum(1)
    return y, ids, w, by_h, by_sums, by_one
