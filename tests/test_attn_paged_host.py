"""CPU checks of the paged-cache operators: the oracle against plain torch, the
argument checks of the C entry points (they refuse before any CUDA call, so no
GPU is needed) and of the Python calls."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import paged_ref as R


def test_oracle_map_by_hand():
    # pages of 4; request 0 holds 5 tokens (2 pages) and gets 4 (1 fresh page), request 1 is new, request 2 idle
    t = np.full((3, 4), -1, np.int32)
    t[0, :2] = [7, 3]
    t[2, 0] = 9
    m = R.page_map([5, 0, 2], [4, 6, 0], t, np.arange(20, 30), 10, 4, 12)
    assert m["cu_q"].tolist() == [0, 4, 10, 10] and m["kv_len"].tolist() == [9, 6, 2]
    assert m["table"][0].tolist() == [7, 3, 29, -1] and m["table"][1].tolist() == [28, 27, -1, -1]
    assert m["positions"].tolist() == [5, 6, 7, 8, 0, 1, 2, 3, 4, 5, 0, 0]
    assert m["slots"].tolist() == [13, 14, 15, 116, 112, 113, 114, 115, 108, 109, -1, -1]
    assert m["n_free"] == 7 and m["info"].tolist() == [0, 0, 0, 0]


def test_oracle_map_that_does_not_fit():
    m = R.page_map([0, 0], [9, 3], np.full((2, 2), -1, np.int32), [5, 6], 2, 4, 10)
    assert m["table"].tolist() == [[6, 5], [-1, -1]]
    assert m["slots"].tolist() == [24, 25, 26, 27, 20, 21, 22, 23, -1, -1]
    assert m["n_free"] == 0 and m["info"].tolist() == [2, 1, 1, 0]


@pytest.mark.parametrize("q_len,kv_len,window", [(5, 5, 0), (3, 11, 0), (3, 11, 2), (6, 4, 0), (2, 0, 0)])
def test_oracle_attention_vs_torch(q_len, kv_len, window):
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((q_len, 4, 128)), rng.standard_normal((kv_len, 2, 128)), rng.standard_normal((kv_len, 2, 128))
    out, lse, spread = R.attention(q, k, v, q_len, kv_len, window=window)
    i, j = np.arange(q_len)[:, None] + kv_len - q_len, np.arange(kv_len)[None]
    ok = (j <= i) & ((j > i - window) if window else True)
    for h in range(4):
        s = np.where(ok, q[:, h] @ k[:, h // 2].T / np.sqrt(128), -np.inf)
        for r in range(q_len):
            if not ok[r].any():
                assert (out[r, h] == 0).all() and lse[r, h] == -np.inf
                continue
            t = torch.from_numpy(s[r])
            assert abs(torch.logsumexp(t, 0).item() - lse[r, h]) < 1e-12
            assert np.abs(torch.softmax(t, 0).numpy() @ v[:, h // 2] - out[r, h]).max() < 1e-12
            assert (spread[r, h] >= np.abs(out[r, h]) - 1e-12).all()


# ---------------------------------------------------------------- refusals --

BUF = ctypes.create_string_buffer(1 << 16)
PTR = (ctypes.addressof(BUF) + 255) // 256 * 256  # never dereferenced: every call below is refused first


def _refused(name, args, code, match):
    from kvr_b200 import _native as N
    with pytest.raises(N.KvrError, match=match) as e:
        N.call(name, *args)
    assert e.value.code == code


def _plan_args(**kw):
    a = dict(cu=PTR, kv=PTR, cu_k=None, batch=2, n=16, n_q=8, n_kv=2, causal=1, window=0, plan=PTR, nbytes=1 << 15)
    a.update(kw)
    return [a["cu"], a["kv"], a["cu_k"], a["batch"], a["n"], a["n_q"], a["n_kv"], a["causal"], a["window"], a["plan"],
            a["nbytes"], None]


@pytest.mark.parametrize("kw,code,match", [
    (dict(cu=None), 1, "null"), (dict(cu_k=PTR), 1, "not both"), (dict(batch=0), 1, "batch"), (dict(batch=4097), 1, "batch"),
    (dict(n=-1), 1, "token"), (dict(n=(1 << 24) + 1), 1, "token"), (dict(n_q=7), 1, "multiple"), (dict(n_kv=0), 1, "multiple"),
    (dict(n_q=258), 3, "128 query heads"), (dict(window=-1), 1, "window"), (dict(window=5, causal=0), 1, "causal"),
    (dict(plan=PTR + 4), 1, "16-byte"), (dict(nbytes=64), 1, "bytes"),
])
def test_plan_refusals(kw, code, match):
    _refused("kvr_attn_plan", _plan_args(**kw), code, match)


def _map_args(**kw):
    a = dict(ctx=PTR, new=PTR, batch=2, n=16, page=16, table=PTR, stride=4, width=4, free=PTR, cap=9, n_free=PTR,
             pos=PTR, slots=PTR, out=PTR + 64, plan=None)
    a.update(kw)
    return [a["ctx"], a["new"], a["batch"], a["n"], a["page"], a["table"], a["stride"], a["width"], a["free"], a["cap"],
            a["n_free"], PTR, PTR, a["pos"], a["slots"], a["out"], PTR, 8, 2, 0, a["plan"], 0, None]


@pytest.mark.parametrize("kw,match", [
    (dict(ctx=None), "null"), (dict(slots=None), "null"), (dict(free=None), "free"), (dict(batch=5000), "batch"),
    (dict(page=0), "page"), (dict(width=0), "table"), (dict(stride=3), "table"), (dict(out=PTR), "n_free_out"),
    (dict(plan=PTR), "bytes"),
])
def test_map_refusals(kw, match):
    _refused("kvr_paged_map", _map_args(**kw), 1, match)


def _write_args(**kw):
    a = dict(q=PTR, k=PTR, dt=1, n=3, n_q=8, n_kv=2, d=128, qs=1024, ks=256, vs=256, cos=PTR, sin=PTR, rs=128, pos=PTR,
             slots=PTR, q_out=PTR, page=16, ps=4096, ts=256)
    a.update(kw)
    return [a["q"], a["k"], PTR, a["dt"], a["n"], a["n_q"], a["n_kv"], a["d"], a["qs"], a["ks"], a["vs"], a["cos"], a["sin"],
            a["rs"], 100, a["pos"], a["slots"], a["q_out"], PTR, PTR, 4, a["page"], a["ps"], a["ts"], None]


@pytest.mark.parametrize("kw,code,match", [
    (dict(k=None), 1, "null"), (dict(slots=None), 1, "null"), (dict(q=None), 1, "together"), (dict(sin=None), 1, "RoPE"),
    (dict(pos=None), 1, "RoPE"), (dict(d=64), 3, "head_dim"), (dict(dt=0), 3, "fp16 or bf16"), (dict(qs=1000), 1, "contiguous"),
    (dict(ks=260), 1, "16-byte"), (dict(rs=130), 1, "16-byte"), (dict(k=PTR + 2), 1, "aligned"), (dict(page=0), 1, "pool"),
    (dict(n=-2), 1, "shape"),
])
def test_write_refusals(kw, code, match):
    _refused("kvr_paged_write", _write_args(**kw), code, match)


def _attn_args(**kw):
    a = dict(q=PTR, dt=2, n=16, batch=2, n_q=8, n_kv=2, d=128, qs=1024, kp=PTR, np=4, page=16, ps=4096, ts=256, table=PTR,
             stride=4, width=4, plan=PTR, nbytes=1 << 15, scale=0.0, out=PTR, ws=PTR, wb=1 << 40)
    a.update(kw)
    return [a["q"], a["dt"], a["n"], a["batch"], a["n_q"], a["n_kv"], a["d"], a["qs"], a["kp"], PTR, a["np"], a["page"],
            a["ps"], a["ts"], a["table"], a["stride"], a["width"], a["plan"], a["nbytes"], a["scale"], a["out"], None,
            a["ws"], a["wb"], None]


@pytest.mark.parametrize("kw,code,match", [
    (dict(q=None), 1, "null"), (dict(plan=None), 1, "null"), (dict(out=None), 1, "null"), (dict(d=64), 3, "head_dim"),
    (dict(dt=0), 3, "fp16 or bf16"), (dict(n_q=9), 1, "multiple"), (dict(n_q=512, qs=1 << 16), 3, "128 query heads"),
    (dict(batch=0), 1, "batch"), (dict(qs=1020), 1, "16-byte"), (dict(qs=8), 1, "contiguous"), (dict(q=PTR + 2), 1, "aligned"),
    (dict(nbytes=16), 1, "plan"), (dict(ws=PTR + 16), 1, "workspace"), (dict(wb=16), 1, "workspace"),
    (dict(scale=float("nan")), 1, "scale"), (dict(table=None), 1, "table"), (dict(np=0), 1, "pool"), (dict(page=20), 3, "multiple of 8"),
    (dict(page=4), 3, "multiple of 8"), (dict(ts=100), 1, "16-byte"), (dict(ps=4097), 1, "16-byte"),
])
def test_paged_attn_refusals(kw, code, match):
    _refused("kvr_paged_attn", _attn_args(**kw), code, match)


def _prompt_args(**kw):
    a = dict(q=PTR, dt=1, n=16, nk=16, batch=2, n_q=8, n_kv=2, d=128, qs=1024, ks=256, vs=256)
    a.update(kw)
    return [a["q"], PTR, PTR, a["dt"], a["n"], a["nk"], a["batch"], a["n_q"], a["n_kv"], a["d"], a["qs"], a["ks"], a["vs"],
            PTR, 1 << 15, 0.0, PTR, None, PTR, 1 << 40, None]


@pytest.mark.parametrize("kw,code,match", [
    (dict(q=None), 1, "null"), (dict(nk=0), 1, "key count"), (dict(ks=100), 1, "contiguous"), (dict(vs=260), 1, "16-byte"),
    (dict(d=256), 3, "head_dim"), (dict(dt=0), 3, "fp16 or bf16"),
])
def test_prompt_attn_refusals(kw, code, match):
    _refused("kvr_prompt_attn", _prompt_args(**kw), code, match)


def test_output_over_the_queries_is_refused():
    from kvr_b200 import kernels as K
    q = torch.zeros(4, 8, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="not q itself"):
        K._attn_out(q, q, False)


def test_nothing_to_do_is_no_error():
    from kvr_b200 import _native as N
    N.call("kvr_paged_write", *_write_args(n=0))
    N.call("kvr_paged_attn", *_attn_args(n=0))
    N.call("kvr_prompt_attn", *_prompt_args(n=0))


def test_python_calls_refuse():
    from kvr_b200 import PagedKVCache
    from kvr_b200 import kernels as K
    pool = torch.zeros(2, 16, 2, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        K.attn_plan(torch.zeros(3, dtype=torch.int32), 4, 8, 2)
    with pytest.raises(TypeError, match="int32"):
        K.attn_plan(torch.zeros(3, dtype=torch.int64), 4, 8, 2)
    with pytest.raises(ValueError, match="entries"):
        K.attn_plan(torch.zeros(3, dtype=torch.int32), 4, 8, 2, kv_len=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(TypeError, match="dtype"):
        K.paged_write(None, torch.zeros(3, 2, 128), torch.zeros(3, 2, 128), pool, pool, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="one shape"):
        K.paged_write(None, pool[0], pool[0], pool, pool[:1], torch.zeros(16, dtype=torch.int64))
    with pytest.raises(ValueError, match="page must"):
        PagedKVCache(1, 8, 2, 4, page=12, device="cpu")
    with pytest.raises(RuntimeError, match="begin"):
        PagedKVCache(1, 8, 2, 4, page=16, device="cpu").commit()


def test_release_returns_pages():
    """Host logic of PagedKVCache.release (torch only, runs on the CPU)."""
    from kvr_b200 import PagedKVCache
    c = PagedKVCache(1, 8, 2, 10, page=16, max_requests=3, max_len=64, device="cpu")
    assert c.free_pages.tolist() == [9, 8, 7, 6, 5, 4, 3, 2, 1, 0]
    c.block_table[0, :2] = torch.tensor([0, 1], dtype=torch.int32)
    c.block_table[1, :3] = torch.tensor([2, 3, 4], dtype=torch.int32)
    c.ctx_len[:] = torch.tensor([17, 48, 0], dtype=torch.int32)
    c.n_free.fill_(5)
    c.release([1])
    assert c.n_free.item() == 8 and c.free_pages[:8].tolist() == [9, 8, 7, 6, 5, 2, 3, 4]
    assert c.ctx_len.tolist() == [17, 0, 0] and (c.block_table[1] == -1).all()
    c.release([0, 2])
    assert c.n_free.item() == 10 and sorted(c.free_pages.tolist()) == list(range(10))
