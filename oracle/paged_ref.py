"""CPU specification of the paged-cache serving operators, in numpy and 64
bits: block tables and slot maps, RoPE + page write, and attention of packed
queries over their requests' keys.  No reference counterpart (the reference
serves one sequence); the attention is the softmax of modules/kvr_window.py:43-69
over a request's visible keys."""
import numpy as np


def page_map(ctx_len, new_len, table, free_pages, n_free, page, n_tokens):
    """-> dict of cu_q, kv_len, positions, slots, table, n_free, info."""
    ctx = [max(int(c), 0) for c in ctx_len]
    table = np.array(table, dtype=np.int32, copy=True)
    width = table.shape[1]
    cu, kv, pos, slots = [0], [], [], []
    taken = beyond = cut = over = 0
    for b, c in enumerate(ctx):
        want = max(int(new_len[b]), 0)
        n = min(want, n_tokens - cu[-1])
        cut += n < want
        cu.append(cu[-1] + n)
        stored = c + n  # keys the request has after the step: those up to its first token without a page
        if -(-(c + n) // page) > width:
            over += 1
            stored = min(stored, max(c, width * page))
        for j in range(-(-c // page), -(-(c + n) // page)):
            if j >= width:  # no page is taken for what has no table entry
                beyond += 1
                continue
            table[b, j] = free_pages[n_free - 1 - taken] if taken < n_free else -1
            if taken >= n_free:
                stored = min(stored, j * page)
            taken += 1
        kv.append(stored)
        for p in range(c, c + n):
            pg = table[b, p // page] if p // page < width else -1
            pos.append(p)
            slots.append(int(pg) * page + p % page if pg >= 0 else -1)
    pos += [0] * (n_tokens - len(pos))
    slots += [-1] * (n_tokens - len(slots))
    i32 = lambda x: np.array(x, dtype=np.int32)  # noqa: E731
    return {"cu_q": i32(cu), "kv_len": i32(kv), "positions": i32(pos), "slots": np.array(slots, dtype=np.int64),
            "table": table, "n_free": max(n_free - taken, 0), "info": i32([max(taken + beyond - n_free, 0), cut, over, 0])}


def rope(x, cos, sin):
    """x (..., heads, d), cos/sin (..., d): rotate_half convention."""
    h = x.shape[-1] // 2
    rot = np.concatenate([-x[..., h:], x[..., :h]], -1)
    return x * cos[..., None, :] + rot * sin[..., None, :]


def attention(q, keys, values, q_len, kv_len, causal=True, window=0, scale=None):
    """One request: q (q_len, n_q, d), keys/values (kv_len, n_kv, d) float64 ->
    (out (q_len, n_q, d), lse (q_len, n_q), spread (q_len, n_q, d)) with
    spread = sum_j p_j |v_j|, what an error of the weights scales with."""
    n_q, d = q.shape[1:]
    g = n_q // keys.shape[1] if kv_len else 1
    scale = np.sqrt(d) if scale is None else scale
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full(q.shape[:2], -np.inf)
    for i in range(q_len):
        end = min(kv_len, kv_len - q_len + i + 1) if causal else kv_len
        begin = max(0, kv_len - q_len + i + 1 - window) if window > 0 else 0
        if end <= begin:
            continue
        for h in range(n_q):
            s = keys[begin:end, h // g] @ q[i, h] / scale
            m = s.max()
            p = np.exp(s - m)
            lse[i, h] = m + np.log(p.sum())
            p /= p.sum()
            out[i, h] = p @ values[begin:end, h // g]
            spread[i, h] = p @ np.abs(values[begin:end, h // g])
    return out, lse, spread
