"""Torch-facing wrappers of the native kernels (one per C-ABI entry point).

All tensors must live on a CUDA device; outputs are allocated here with torch
(the C ABI itself never allocates).  Shapes follow the reference
(modules/kvr_retrieval.py, modules/kvr_window.py) unless noted.
"""
from __future__ import annotations

import collections
import contextlib
import ctypes as C
import math
import threading

import torch

from . import _native as N
from ._native import call, dtype_code, ptr, stream

D = 128


def _c(t):
    return t if t.is_contiguous() else t.contiguous()


# ------------------------------------------------------------------ int4w --


def absmax_scales(x: torch.Tensor, clamp_min: float = 1e-8) -> torch.Tensor:
    """calibrate()'s k_scales (kvr_retrieval.py:99): (n, ...) -> (...) fp32."""
    x = _c(x)
    n = x.shape[0]
    out = torch.empty(x.shape[1:], dtype=torch.float32, device=x.device)
    call("kvr_absmax_scales", ptr(x), dtype_code(x), n, out.numel(), clamp_min, ptr(out), stream())
    return out


def int4w_encode_k(k: torch.Tensor, k_scales: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """(n, n_kv, d) -> packed (n, n_kv, d/2) uint8 (kvr_retrieval.py:190-193)."""
    n, n_kv, d = k.shape
    if k.stride(2) != 1 or k.stride(1) != d:
        k = k.contiguous()
    ks = _c(k_scales.float())
    if out is None:
        out = torch.empty(n, n_kv, d // 2, dtype=torch.uint8, device=k.device)
    call("kvr_int4w_encode_k", ptr(k), dtype_code(k), n, n_kv, d, k.stride(0), ptr(ks), ptr(out), stream())
    return out


def int4w_encode_vres(v, v_pred, vr_scales, out=None):
    """(n, n_kv, d) -> packed (n, n_kv, d/4) uint8 (kvr_retrieval.py:196-203)."""
    v = _c(v)
    n, n_kv, d = v.shape
    vp = _c(v_pred.float())
    vr = _c(vr_scales.float().reshape(-1))
    if out is None:
        out = torch.empty(n, n_kv, d // 4, dtype=torch.uint8, device=v.device)
    call("kvr_int4w_encode_vres", ptr(v), dtype_code(v), ptr(vp), n, n_kv, d, ptr(vr), ptr(out), stream())
    return out


def compute_scores(q_avg, k_packed, k_scales, cos_tbl, sin_tbl, n_stored=None):
    """Drop-in for the reference native kernel (kvr_cuda.cu:53-77)."""
    n_kv, d = k_packed.shape[1], k_packed.shape[2] * 2
    n = k_packed.shape[0] if n_stored is None else n_stored
    q = _c(q_avg.float())
    out = torch.empty(n, n_kv, dtype=torch.float32, device=q.device)
    call("kvr_compute_scores", ptr(q), ptr(_c(k_packed)), ptr(_c(k_scales.float())), ptr(_c(cos_tbl.float())),
         ptr(_c(sin_tbl.float())), n_kv, d, n, ptr(out), stream())
    return out


def _rope_args(cos, sin):
    if cos.stride(-1) != 1 or sin.stride(-1) != 1 or cos.stride(0) != sin.stride(0):
        cos, sin = cos.contiguous(), sin.contiguous()
    return cos, sin, cos.stride(0)


def int4w_token_scores(q_post, k_packed, k_scales, cos, sin, n_stored, halves_equal=False, out=None):
    """compute_all_scores (kvr_retrieval.py:265-289) -> HEAD-MAJOR (n_kv, n_stored)."""
    n_kv = k_packed.shape[1]
    q = _c(q_post.float())
    cos, sin, rs = _rope_args(cos.float(), sin.float())
    if out is None:
        out = torch.empty(n_kv, n_stored, dtype=torch.float32, device=q.device)
    call("kvr_int4w_token_scores", ptr(q), q.shape[0], ptr(_c(k_packed)), ptr(_c(k_scales.float())), ptr(cos),
         ptr(sin), rs, int(halves_equal), n_kv, D, n_stored, ptr(out), out.stride(0), stream())
    return out


def int4w_token_topk(q_post, k_packed, k_scales, cos, sin, n_stored, k, halves_equal=False, ex_start=0, ex_end=0):
    """Token branch of retrieve_topk in one call (scores + exclusion + top-k,
    kvr_retrieval.py:265-289, 389-392) -> idx (k, n_kv) int64."""
    n_kv = k_packed.shape[1]
    q = _c(q_post.float())
    cos, sin, rs = _rope_args(cos.float(), sin.float())
    idx = torch.empty(k, n_kv, dtype=torch.int64, device=q.device)
    ws = N.workspace("int4w_topk", call("kvr_int4w_token_topk_workspace_bytes", n_kv, n_stored, k), q.device)
    call("kvr_int4w_token_topk", ptr(q), q.shape[0], ptr(_c(k_packed)), ptr(_c(k_scales.float())), ptr(cos),
         ptr(sin), rs, int(halves_equal), n_kv, D, n_stored, k, ex_start, ex_end, ptr(idx), ptr(ws), ws.numel(),
         stream())
    return idx


def int4w_chunk_scores(q_post, k_packed, k_scales, cos, sin, n_stored, chunk, halves_equal=False):
    """compute_chunk_scores (kvr_retrieval.py:291-315) -> HEAD-MAJOR (n_kv, n_stored // chunk)."""
    n_kv = k_packed.shape[1]
    q = _c(q_post.float())
    cos, sin, rs = _rope_args(cos.float(), sin.float())
    nc = n_stored // chunk
    out = torch.empty(n_kv, nc, dtype=torch.float32, device=q.device)
    call("kvr_int4w_chunk_scores", ptr(q), q.shape[0], ptr(_c(k_packed)), ptr(_c(k_scales.float())), ptr(cos),
         ptr(sin), rs, int(halves_equal), n_kv, D, n_stored, chunk, ptr(out), out.stride(0), stream())
    return out


def topk_rows(scores: torch.Tensor, k: int, ex_start: int = 0, ex_end: int = 0, transpose_out: bool = False):
    """Per-row top-k of (rows, n) fp32, (score desc, index asc); entries in
    [ex_start, ex_end) and NaN count as -inf.  Returns (idx int64, vals fp32)
    shaped (rows, k), or (k, rows) when transpose_out."""
    assert scores.dim() == 2 and scores.stride(1) == 1 and scores.dtype == torch.float32
    rows, n = scores.shape
    shape = (k, rows) if transpose_out else (rows, k)
    idx = torch.empty(shape, dtype=torch.int64, device=scores.device)
    vals = torch.empty(shape, dtype=torch.float32, device=scores.device)
    ors, oes = (1, rows) if transpose_out else (k, 1)
    call("kvr_topk_rows", ptr(scores), rows, n, scores.stride(0), k, ex_start, ex_end, ptr(idx), ptr(vals), ors, oes,
         stream())
    return idx, vals


def int4w_gather(k_packed, k_scales, top, cos, sin, k_mean=None, want_x=True, count=None, ret_k=None):
    """-> (ret_k (k, n_kv, d) fp32 post-RoPE, x (n_kv, k, n_kv*d) fp32 = deq
    K_pre - K_mean, or None when want_x is False).  count: optional device
    int32 row count (rows past it are left untouched)."""
    k, n_kv = top.shape
    cos, sin, rs = _rope_args(cos.float(), sin.float())
    if ret_k is None:
        ret_k = torch.empty(k, n_kv, D, dtype=torch.float32, device=top.device)
    x = torch.empty(n_kv, k, n_kv * D, dtype=torch.float32, device=top.device) if want_x else None
    km = _c(k_mean.float().reshape(-1)) if want_x else None
    call("kvr_int4w_gather", ptr(_c(k_packed)), ptr(_c(k_scales.float())), ptr(_c(top)), k, n_kv, D, ptr(cos),
         ptr(sin), rs, ptr(km), ptr(ret_k), ptr(x), ptr(count), stream())
    return ret_k, x


def int4w_vpredict_prepare(W, k_mean, v_mean, k_scales, n_kv):
    """Once per calibration: (w3, unscale fp32 (n_kv*d), bias fp32 (n_kv*d))
    for int4w_vpredict; w3 holds the fp16 hi/lo parts of W' = W diag(step) in
    the kernel's tensor-core operand layout (n_kv*2*d*n_kv*d halves)."""
    dev = W.device
    KD = n_kv * D
    w3 = torch.empty(n_kv, 2, D, KD, dtype=torch.float16, device=dev)
    unscale = torch.empty(KD, dtype=torch.float32, device=dev)
    bias = torch.empty(KD, dtype=torch.float32, device=dev)
    call("kvr_int4w_vpredict_prepare", ptr(_c(W.float())), ptr(_c(k_mean.float().reshape(-1))),
         ptr(_c(v_mean.float().reshape(-1))), ptr(_c(k_scales.float().reshape(-1))), n_kv, D, ptr(w3),
         ptr(unscale), ptr(bias), stream())
    return w3, unscale, bias


def int4w_vpredict(k_packed, top, prep, vr_packed, vr_scales, count=None, out=None):
    """ret_v (k, n_kv, d) fp16 = W-predicted V + int2 residual of the tokens
    top (k, n_kv) int64 (kvr_retrieval.py:394-402), on the tensor cores."""
    k, n_kv = top.shape
    w3, unscale, bias = prep
    if out is None:
        out = torch.empty(k, n_kv, D, dtype=torch.float16, device=top.device)
    call("kvr_int4w_vpredict", ptr(_c(k_packed)), ptr(_c(top)), ptr(count), k, n_kv, D, ptr(w3), ptr(unscale),
         ptr(bias), ptr(_c(vr_packed)), ptr(_c(vr_scales.float().reshape(-1))), ptr(out), stream())
    return out


def int4w_vpredict_status():
    """Raises if a bounded device-side wait of the V-predict kernel gave up
    since the last check (synchronises the current stream)."""
    call("kvr_int4w_vpredict_status", stream())


def int4w_attractor_select(q, n_kv, k_packed, k_scales, cos, sin, centroids, labels, n_labelled, top_a=48,
                           ex_start=0, ex_end=0):
    """Attractor branch selection (kvr_retrieval.py:332-367) on the device:
    labels int32 (>= n_labelled) -> (top (top_a*16, n_kv) int64, count (1,)
    int32 device tensor)."""
    q = _c(q.float())
    n_q = q.shape[0]
    cos, sin, rs = _rope_args(cos.float(), sin.float())
    rows = top_a * 16
    top = torch.empty(rows, n_kv, dtype=torch.int64, device=q.device)
    count = torch.empty(1, dtype=torch.int32, device=q.device)
    ws = N.workspace("attractor", call("kvr_int4w_attractor_workspace_bytes", n_labelled, top_a), q.device)
    call("kvr_int4w_attractor_select", ptr(q), n_q, n_kv, ptr(_c(k_packed)), ptr(_c(k_scales.float())), ptr(cos),
         ptr(sin), rs, ptr(_c(centroids.float())), centroids.shape[0], ptr(_c(labels)), n_labelled, top_a, ex_start,
         ex_end, ptr(top), ptr(count), ptr(ws), ws.numel(), stream())
    return top, count


def int4w_assign_basins(k_packed, k_scales, t0, t1, centroids, labels):
    """labels[t0:t1] (int32, in place) = nearest basin of each token's head-0 K."""
    call("kvr_int4w_assign_basins", ptr(_c(k_packed)), ptr(_c(k_scales.float())), k_packed.shape[1], t0, t1,
         ptr(_c(centroids.float())), centroids.shape[0], ptr(labels), stream())


# ----------------------------------------------------------------- window --


def window_write(k, v, ring_k, ring_v, pos: int):
    """Ring write of n tokens at slots (pos + i) % cap (kvr_window.py:19-41)."""
    k, v = _c(k), _c(v)
    if v.dtype != k.dtype:
        v = v.to(k.dtype)
    n = k.shape[0]
    n_kv, d = ring_k.shape[1], ring_k.shape[2]
    call("kvr_window_write", ptr(k), ptr(v), dtype_code(k), n, n_kv, d, ptr(ring_k), ptr(ring_v), ring_k.shape[0],
         pos, stream())


def decode_store_update(q, k, v, cos, sin, pos, ring_k, ring_v, slot, tail_k=None, tail_v=None, tail_row=0,
                        write_kv=True, q_out=None):
    """One decode step's RoPE + window write (+ eviction of the slot's old row
    into the sd1 tail) in one launch.  q (n_q, d), k/v (n_kv, d) of the model
    dtype -> q_out = RoPE(q) (same dtype)."""
    q, k, v = _c(q), _c(k), _c(v)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must share a dtype")
    cos, sin, rs = _rope_args(cos, sin)
    if q_out is None:
        q_out = torch.empty_like(q)
    call("kvr_decode_store_update", ptr(q), ptr(k), ptr(v), dtype_code(q), q.shape[0], k.shape[0], D, ptr(cos),
         ptr(sin), rs, pos, ptr(q_out), ptr(ring_k), ptr(ring_v), ring_k.shape[0], slot, ptr(tail_k), ptr(tail_v),
         tail_row, int(write_kv), stream())
    return q_out


# -------------------------------------------------------------- attention --


def _seg_rows(k, v, d):
    if k.stride(-1) != 1 or k.stride(-2) != d:
        k = k.contiguous()
    if v.stride(-1) != 1 or v.stride(-2) != d or v.stride(0) != k.stride(0):
        v = v.contiguous()
        if v.stride(0) != k.stride(0):
            k = k.contiguous()
    return k, v


def decode_attn(q, segments, scale=None, out_dtype=None, n_kv=None, n1_count=None, out=None):
    """Exact attention of q (n_q, d) over up to two K/V segments
    [(k0, v0), (k1, v1)], each (n_i, n_kv, d) with contiguous rows.
    n1_count: optional device int32 holding how many rows of the second
    segment are valid (kvr_decode_attn_counted)."""
    q = _c(q)
    n_q, d = q.shape
    if n_kv is None:
        n_kv = segments[0][0].shape[1]
    segs = [_seg_rows(k, v, d) if k.shape[0] else None for k, v in segments]
    if n1_count is None:
        segs = [sg for sg in segs if sg is not None]
    while len(segs) < 2:
        segs.append(None)
    if segs[1] is None:
        n1_count = None
    out_dtype = out_dtype or q.dtype
    if out is None:
        out = torch.empty(n_q, d, dtype=out_dtype, device=q.device)
    n_tot = sum(sg[0].shape[0] for sg in segs if sg is not None)
    ws = N.workspace("attn", call("kvr_decode_attn_workspace_bytes", n_q, n_kv, d, n_tot), q.device)
    args = []
    for sg in segs:
        if sg is not None:
            k, v = sg
            args.append([ptr(k), ptr(v), dtype_code(k), dtype_code(v), k.shape[0], k.stride(0)])
        else:
            args.append([None, None, 0, 0, 0, 0])
    if n1_count is not None:
        call("kvr_decode_attn_counted", ptr(q), dtype_code(q), n_q, n_kv, d, *args[0], *args[1], ptr(n1_count),
             float(scale or 0.0), ptr(out), dtype_code(out), ptr(ws), ws.numel(), stream())
    else:
        call("kvr_decode_attn", ptr(q), dtype_code(q), n_q, n_kv, d, *args[0], *args[1], float(scale or 0.0),
             ptr(out), dtype_code(out), ptr(ws), ws.numel(), stream())
    return out


def lse_merge(partials: torch.Tensor, out_dtype=torch.float32):
    """partials (P, n_q, d+2) [m, l, o] -> (n_q, d)."""
    p = _c(partials.float())
    P_, n_q, dd = p.shape
    out = torch.empty(n_q, dd - 2, dtype=out_dtype, device=p.device)
    call("kvr_lse_merge", ptr(p), P_, n_q, dd - 2, ptr(out), dtype_code(out), stream())
    return out


def merge_candidates(scores, idx, k_sel, tile_base=0, n_local=0, global_out=True):
    """scores fp32 / idx int32 (N, B, H, k_local) gathered candidates ->
    (global_sel (B, H, k_sel) int32 or None, local_sel (B, H, k_sel) int32)."""
    N_, B, H, kl = scores.shape
    sc, ix = _c(scores.float()), _c(idx.to(torch.int32))
    lsel = torch.empty(B, H, k_sel, dtype=torch.int32, device=sc.device)
    gsel = torch.empty_like(lsel) if global_out else None
    call("kvr_merge_candidates", ptr(sc), ptr(ix), N_, B * H, kl, k_sel, tile_base, n_local, ptr(gsel), ptr(lsel),
         stream())
    return gsel, lsel


# -------------------------------------------------------------------- sd1 --


def transform(x: torch.Tensor, kind: str = "hadamard", inverse: bool = False) -> torch.Tensor:
    """Orthonormal Hadamard / DCT along the last axis (d = 128), fp32."""
    x = _c(x.float())
    y = torch.empty_like(x)
    call("kvr_transform", ptr(x), ptr(y), x.numel() // D, N.TRANSFORMS[kind], int(inverse), stream())
    return y


class Sd1Store:
    """Device buffers of one layer's 1-bit store for `batch` sequences x n_kv heads.

    kbits/vbits (B, n_kv, nt_cap, tile, 4) uint32 (stored as int32 tensors),
    kscale/vscale (B, n_kv, nt_cap, 128) fp16.  `n_tiles` full tiles are valid."""

    def __init__(self, batch, n_kv, nt_cap, tile=64, kind="hadamard", device="cuda"):
        if tile not in (32, 64, 128):
            raise ValueError("tile must be 32, 64 or 128")
        self.batch, self.n_kv, self.nt_cap, self.tile, self.kind = batch, n_kv, nt_cap, tile, kind
        self.kbits = torch.zeros(batch, n_kv, nt_cap, tile, 4, dtype=torch.int32, device=device)
        self.vbits = torch.zeros_like(self.kbits)
        self.kscale = torch.zeros(batch, n_kv, nt_cap, D, dtype=torch.float16, device=device)
        self.vscale = torch.zeros_like(self.kscale)
        self.n_tiles = 0

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.kbits, self.vbits, self.kscale, self.vscale))

    def grow(self, nt_cap):
        if nt_cap <= self.nt_cap:
            return
        def ext(t):
            z = torch.zeros(*t.shape[:2], nt_cap - self.nt_cap, *t.shape[3:], dtype=t.dtype, device=t.device)
            return torch.cat([t, z], 2)
        self.kbits, self.vbits = ext(self.kbits), ext(self.vbits)
        self.kscale, self.vscale = ext(self.kscale), ext(self.vscale)
        self.nt_cap = nt_cap


def sd1_encode(store: Sd1Store, k, v, n_tiles=None, tile0=None, cos=None, sin=None, pos0=0):
    """Encode full tiles of k, v ((B, n, n_kv, d) or (n, n_kv, d)) into the store
    starting at tile `tile0` (default: store.n_tiles, then advances n_tiles)."""
    if k.dim() == 3:
        k, v = k.unsqueeze(0), v.unsqueeze(0)
    B, n, n_kv, d = k.shape
    if v.dtype != k.dtype:
        v = v.to(k.dtype)
    if k.stride(-1) != 1 or k.stride(-2) != d:
        k = k.contiguous()
    if v.stride() != k.stride():
        k, v = k.contiguous(), v.contiguous()
    nt = n // store.tile if n_tiles is None else n_tiles
    t0 = store.n_tiles if tile0 is None else tile0
    if cos is not None:
        cos, sin, rs = _rope_args(cos.float(), sin.float())
    else:
        rs = 0
    call("kvr_sd1_encode", ptr(k), ptr(v), dtype_code(k), B, n_kv, nt, store.tile, k.stride(0), k.stride(1),
         ptr(cos), ptr(sin), rs, pos0, N.TRANSFORMS[store.kind], ptr(store.kbits), ptr(store.kscale),
         ptr(store.vbits), ptr(store.vscale), store.nt_cap, t0, stream())
    if tile0 is None:
        store.n_tiles = t0 + nt
    return nt


def sd1_tile_scores(store: Sd1Store, q):
    """q (B, n_q, d) -> (B, n_kv, n_tiles) fp32 selection scores."""
    q = _c(q if q.dim() == 3 else q.unsqueeze(0))
    B, n_q, _ = q.shape
    out = torch.empty(B, store.n_kv, max(store.n_tiles, 0), dtype=torch.float32, device=q.device)
    call("kvr_sd1_tile_scores", ptr(q), dtype_code(q), B, n_q, store.n_kv, ptr(store.kbits), ptr(store.kscale),
         store.nt_cap, store.n_tiles, store.tile, N.TRANSFORMS[store.kind], ptr(out), stream())
    return out


def sd1_select(store: Sd1Store, q, k_sel, ex_t0=0, ex_t1=0, tile_base=0, n_tiles=None):
    """-> (sel (B, n_kv, k_sel) int32, sel_scores fp32, qprime (B, n_q, d) fp32)."""
    q = _c(q if q.dim() == 3 else q.unsqueeze(0))
    B, n_q, _ = q.shape
    nt = store.n_tiles if n_tiles is None else n_tiles
    sel = torch.empty(B, store.n_kv, k_sel, dtype=torch.int32, device=q.device)
    sc = torch.empty(B, store.n_kv, k_sel, dtype=torch.float32, device=q.device)
    qp = torch.empty(B, n_q, D, dtype=torch.float32, device=q.device)
    ws = N.workspace("sd1_select", call("kvr_sd1_select_workspace_bytes", B, store.n_kv, nt), q.device)
    call("kvr_sd1_select", ptr(q), dtype_code(q), B, n_q, store.n_kv, ptr(store.kbits), ptr(store.kscale),
         store.nt_cap, nt, store.tile, N.TRANSFORMS[store.kind], k_sel, ex_t0, ex_t1, tile_base, ptr(sel), ptr(sc),
         ptr(qp), ptr(ws), ws.numel(), stream())
    return sel, sc, qp


def _win_args(win_k, win_v, n_win):
    if win_k is None or n_win == 0:
        return None, None, 1, 0
    return ptr(win_k), ptr(win_v), win_k.shape[-3], n_win


def sd1_attend(store: Sd1Store, q, qprime, sel, win_k=None, win_v=None, n_win=0, tail_k=None, tail_v=None,
               n_tail=0, scale=None, out_dtype=None, partial=False):
    """Attention over window (B, cap, n_kv, d) fp16 + tail (B, t, n_kv, d) fp16 +
    selected tiles.  Returns out (B, n_q, d) or partial rows (B, n_q, d+2)."""
    q = _c(q if q.dim() == 3 else q.unsqueeze(0))
    B, n_q, _ = q.shape
    k_sel = sel.shape[-1]
    out_dtype = out_dtype or q.dtype
    if partial:
        part = torch.empty(B, n_q, D + 2, dtype=torch.float32, device=q.device)
        out = None
    else:
        out = torch.empty(B, n_q, D, dtype=out_dtype, device=q.device)
        part = None
    wk, wv, wcap, nw = _win_args(win_k, win_v, n_win)
    tk, tv = (ptr(tail_k), ptr(tail_v)) if n_tail else (None, None)
    ws = N.workspace("sd1_attend", call("kvr_sd1_attend_workspace_bytes", B, n_q, store.n_kv, store.tile, k_sel, nw,
                                        n_tail), q.device)
    call("kvr_sd1_attend", ptr(q), dtype_code(q), ptr(qprime), B, n_q, store.n_kv, wk, wv, wcap, nw, tk, tv, n_tail,
         ptr(store.kbits), ptr(store.kscale), ptr(store.vbits), ptr(store.vscale), store.nt_cap, store.tile,
         N.TRANSFORMS[store.kind], ptr(_c(sel)), k_sel, float(scale or 0.0), ptr(out),
         dtype_code(out) if out is not None else 0, ptr(part), ptr(ws), ws.numel(), stream())
    return part if partial else out


_STEP_WS: dict = {}


@contextlib.contextmanager
def sd1_step_path(path):
    """Within the block, kvr_sd1_decode_step runs the one-kernel cluster path
    where shapes allow ("cluster", the default; "cluster8": 8-CTA clusters
    only) or always the selection + attention kernels ("split").
    Process-wide; restores the previous value."""
    fn = N.lib().kvr_set_sd1_step_path  # returns the previous value, not a status
    prev = fn({"cluster": 0, "split": 1, "cluster8": 2}[path])
    try:
        yield
    finally:
        fn(prev)


def sd1_decode_step(store: Sd1Store, q, k_sel, win_k=None, win_v=None, n_win=0, tail_k=None, tail_v=None,
                    n_tail=0, ex_t0=0, ex_t1=0, scale=None, out=None, sel_out=None, ws=None):
    """Tile selection + attention in one call: one cluster kernel for few rows,
    else the selection and attention kernels.  Returns out (B, n_q, d)."""
    q = _c(q if q.dim() == 3 else q.unsqueeze(0))
    B, n_q, _ = q.shape
    if out is None:
        out = torch.empty(B, n_q, D, dtype=q.dtype, device=q.device)
    wk, wv, wcap, nw = _win_args(win_k, win_v, n_win)
    tk, tv = (ptr(tail_k), ptr(tail_v)) if n_tail else (None, None)
    if ws is None:
        key = (B, n_q, store.n_kv, store.n_tiles, store.tile, k_sel, nw, n_tail)
        need = _STEP_WS.get(key)
        if need is None:
            need = _STEP_WS[key] = call("kvr_sd1_workspace_bytes", *key)
            if len(_STEP_WS) > 4096:
                _STEP_WS.clear()
        ws = N.workspace("sd1_step", need, q.device)
    call("kvr_sd1_decode_step", ptr(q), dtype_code(q), B, n_q, store.n_kv, wk, wv, wcap, nw, tk, tv, n_tail,
         ptr(store.kbits), ptr(store.kscale), ptr(store.vbits), ptr(store.vscale), store.nt_cap, store.n_tiles,
         store.tile, N.TRANSFORMS[store.kind], k_sel, ex_t0, ex_t1, float(scale or 0.0), ptr(out), dtype_code(out),
         ptr(sel_out), ptr(ws), ws.numel(), stream())
    return out


def sd1_decode_step_update(store: Sd1Store, q, k, v, cos, sin, pos, k_sel, win_k, win_v, n_win, slot,
                           tail_k=None, tail_v=None, n_tail=0, evict=False, ex_t0=0, ex_t1=0, scale=None,
                           out=None, q_out=None, sel_out=None, ws=None):
    """The layer's store update fused with its decode step (batch 1).

    q (n_q, d), k and v (n_kv, d): the new token's pre-RoPE rows, one dtype.
    The rotated K / V land in window slot `slot` (one of the n_win rows
    attended, n_win counting the new row); with `evict` the slot's old row
    first moves to tail row n_tail - 1.  Returns (out (1, n_q, d) of q's
    dtype, q_out = RoPE(q))."""
    q, k, v = _c(q), _c(k), _c(v)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must share a dtype")
    n_q, n_kv = q.shape[0], k.shape[0]
    cos, sin, rs = _rope_args(cos, sin)
    if out is None:
        out = torch.empty(1, n_q, D, dtype=q.dtype, device=q.device)
    if q_out is None:
        q_out = torch.empty_like(q)
    if ws is None:
        key = (1, n_q, n_kv, store.n_tiles, store.tile, k_sel, n_win, n_tail)
        need = _STEP_WS.get(key)
        if need is None:
            need = _STEP_WS[key] = call("kvr_sd1_workspace_bytes", *key)
            if len(_STEP_WS) > 4096:
                _STEP_WS.clear()
        ws = N.workspace("sd1_step", need, q.device)
    call("kvr_sd1_decode_step_update", ptr(q), ptr(k), ptr(v), dtype_code(q), n_q, n_kv, ptr(cos), ptr(sin), rs,
         pos, ptr(q_out), ptr(win_k), ptr(win_v), win_k.shape[-3], n_win, slot, ptr(tail_k), ptr(tail_v), n_tail,
         int(evict), ptr(store.kbits), ptr(store.kscale), ptr(store.vbits), ptr(store.vscale), store.nt_cap,
         store.n_tiles, store.tile, N.TRANSFORMS[store.kind], k_sel, ex_t0, ex_t1, float(scale or 0.0), ptr(out),
         dtype_code(out), ptr(sel_out), ptr(ws), ws.numel(), stream())
    return out, q_out


def sd1_decode_tiles(store: Sd1Store, sel):
    """sel (B, n_kv, k) int64 -> (K (B, k*t, n_kv, d) fp32, V fp16)."""
    sel = _c(sel.long())
    B, n_kv, k = sel.shape
    ok = torch.empty(B, k * store.tile, n_kv, D, dtype=torch.float32, device=sel.device)
    ov = torch.empty(B, k * store.tile, n_kv, D, dtype=torch.float16, device=sel.device)
    call("kvr_sd1_decode_tiles", ptr(store.kbits), ptr(store.kscale), ptr(store.vbits), ptr(store.vscale),
         store.nt_cap, B, n_kv, store.tile, N.TRANSFORMS[store.kind], ptr(sel), k, ptr(ok), ptr(ov), stream())
    return ok, ov


def sd1_prefill_scores(store: Sd1Store, q):
    """Tensor-core tile scores for a block of prefill queries (batch-1 store):
    q (nq, n_q, d) -> (nq, n_kv, n_tiles) fp32."""
    if store.batch != 1:
        raise ValueError("prefill scoring takes a batch-1 store")
    q = _c(q)
    nq, n_q, _ = q.shape
    out = torch.empty(nq, store.n_kv, store.n_tiles, dtype=torch.float32, device=q.device)
    ws = N.workspace("sd1_prefill", call("kvr_sd1_prefill_workspace_bytes", nq, store.n_kv), q.device)
    call("kvr_sd1_prefill_scores", ptr(q), dtype_code(q), nq, n_q, store.n_kv, ptr(store.kbits), ptr(store.kscale),
         store.nt_cap, store.n_tiles, store.tile, N.TRANSFORMS[store.kind], ptr(out), ptr(ws), ws.numel(), stream())
    return out


# ----------------------------------------------------- paged exact cache --


def _tokens(x, name):
    """(n, heads, 128) with contiguous heads and 16-byte aligned rows, and its
    token stride in elements; views that are not laid out so are copied."""
    shape = x.shape
    if len(shape) != 3 or shape[2] != D:
        raise ValueError(f"{name} must be (tokens, heads, {D}), got {tuple(shape)}")
    n, heads, _ = shape
    st, sh, sd = x.stride()
    if not (sd == 1 and (heads == 1 or sh == D) and x.data_ptr() % 16 == 0
            and (n <= 1 or (st >= heads * D and st % 8 == 0))):
        x = x.clone(memory_format=torch.contiguous_format)
        st = heads * D
    return x, st if n > 1 else heads * D


def _pool(k_pages, v_pages):
    """(n_pages, page, n_kv, 128) pools, e.g. views of one (n_pages, 2, page,
    n_kv, 128) tensor; never copied, since they are the caller's cache."""
    shape, strides = k_pages.shape, k_pages.stride()
    if len(shape) != 4 or shape[3] != D:
        raise ValueError(f"k_pages must be (pages, page, heads, {D}), got {tuple(shape)}")
    if strides[3] != 1 or (shape[2] > 1 and strides[2] != D):
        raise ValueError("k_pages: a token's heads must be contiguous")
    if v_pages.shape != shape or v_pages.dtype != k_pages.dtype or v_pages.stride() != strides:
        raise ValueError("k_pages and v_pages must have one shape, type and layout")
    return shape[0], shape[1], strides[0], strides[1]


_INT32 = torch.int32


def _i32(x, name, numel=None):
    """Checks an int32 vector; returns its number of entries."""
    n = x.numel()
    if x.dtype is not _INT32 or x.dim() != 1 or not x.is_contiguous():
        raise TypeError(f"{name} must be a contiguous int32 vector")
    if numel is not None and n != numel:
        raise ValueError(f"{name} must have {numel} entries, got {n}")
    return n


def _on_gpu(*tensors):
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("kvr_b200 operators need CUDA tensors (this build has no CPU path)")


def _on_current_gpu(*tensors):
    """What a call reads and writes lies where its stream is."""
    here = torch.cuda.current_device()
    for t in tensors:
        if t.get_device() != here:
            raise ValueError(f"kvr_b200 operators need CUDA tensors on the current device (cuda:{here}; this build has no CPU "
                             f"path), got one on {t.device}")


def _table(block_table, batch):
    """Checks a block table with a row for each of `batch` requests; returns its
    width and row stride."""
    if block_table.dtype is not _INT32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise TypeError("block_table must be an int32 matrix with contiguous rows")
    rows, width = block_table.shape
    if rows < batch:
        raise ValueError(f"block_table has {rows} rows for {batch} requests")
    stride = block_table.stride(0)
    if rows == 1:  # no second row that the stride leads to
        stride = max(stride, width)
    elif stride < width:
        raise ValueError("block_table: rows must not share memory (an expanded table has to be copied)")
    return width, stride


_PLAN_BYTES: dict = {}


class AttnPlan:
    """The work list of an attention call (kvr_attn_plan), on the device, and
    the shapes it was built for."""

    def __init__(self, n_tokens, batch, n_q, n_kv, paged, device, own_keys=False):
        self.n_tokens, self.batch, self.n_q, self.n_kv, self.paged = n_tokens, batch, n_q, n_kv, paged
        self.own_keys = own_keys  # packed keys that are the queries' own tokens
        key = (n_tokens, batch, n_q, n_kv)
        nbytes = _PLAN_BYTES.get(key)
        if nbytes is None:
            if len(_PLAN_BYTES) > 4096:
                _PLAN_BYTES.clear()
            nbytes = _PLAN_BYTES[key] = max(call("kvr_attn_plan_bytes", *key), 16)
        self.nbytes = nbytes
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)

    def _match(self, n_tokens, n_q, paged):
        if (self.n_tokens, self.n_q, self.paged) != (n_tokens, n_q, paged):
            raise ValueError(f"the plan is for {self.n_tokens} tokens of {self.n_q} heads"
                             f"{' over pages' if self.paged else ''}, not {n_tokens} of {n_q}"
                             f"{' over pages' if paged else ''}")


def attn_plan(cu_q, n_tokens, n_q, n_kv, kv_len=None, cu_k=None, causal=True, window=0):
    """Plan of the attention of packed queries: those of request b are
    [cu_q[b], cu_q[b+1]) of n_tokens and are the last tokens of kv_len[b] keys
    in pages (paged_attn), or of the packed keys [cu_k[b], cu_k[b+1])
    (prompt_attn; cu_k None: the queries' own tokens).  window > 0: a query
    sees the last `window` keys up to itself.  All lengths int32 on the device;
    one plan serves every layer."""
    _i32(cu_q, "cu_q")
    batch = cu_q.numel() - 1
    if batch < 1:
        raise ValueError("cu_q must have at least two entries")
    if kv_len is not None:
        _i32(kv_len, "kv_len", batch)
    if cu_k is not None:
        _i32(cu_k, "cu_k", batch + 1)
    plan = AttnPlan(n_tokens, batch, n_q, n_kv, kv_len is not None, cu_q.device, kv_len is None and cu_k is None)
    call("kvr_attn_plan", ptr(cu_q), ptr(kv_len), ptr(cu_k), batch, n_tokens, n_q, n_kv, int(causal), window,
         ptr(plan.buf), plan.nbytes, stream())
    return plan


class PagedStep:
    """What paged_map makes of a step's lengths (int32 on the device unless
    noted): cu_q (B + 1), kv_len (B) = ctx_len + new_len, or the keys that have a
    page where pages are missing or the table row ends, positions (T), slots (T) int64, n_free
    (1) left, info (4) = [pages missing, requests cut, requests longer than
    their table row, 0], and the attention plan (None without n_q)."""

    __slots__ = ("cu_q", "kv_len", "positions", "slots", "n_free", "info", "plan", "n_tokens")


def paged_map(ctx_len, new_len, block_table, free_pages, n_free, page, n_tokens, n_q=0, n_kv=0, window=0):
    """Block tables, slot maps and the attention plan of a step in one launch:
    request b has ctx_len[b] tokens cached and gets new_len[b]; pages come off
    the end of free_pages[:n_free] and are entered into block_table (B, width)
    in place.  n_tokens: the step's packed length (>= the sum of new_len; the
    rest is padding).  ctx_len, new_len and n_free are left as they are."""
    batch = _i32(ctx_len, "ctx_len")
    _i32(new_len, "new_len", batch)
    n_pages = _i32(free_pages, "free_pages")
    _i32(n_free, "n_free", 1)
    width, stride = _table(block_table, batch)
    _on_gpu(ctx_len, new_len, free_pages, n_free, block_table)
    dev = ctx_len.device
    buf = torch.empty(2 * batch + 6 + n_tokens, dtype=_INT32, device=dev)
    st = PagedStep()
    st.cu_q, st.kv_len, st.n_free, st.info, st.positions = torch.split_with_sizes(buf, (batch + 1, batch, 1, 4, n_tokens))
    st.slots = torch.empty(n_tokens, dtype=torch.int64, device=dev)
    st.n_tokens = n_tokens
    st.plan = AttnPlan(n_tokens, batch, n_q, n_kv, True, dev) if n_q else None
    at = buf.data_ptr()
    plan = st.plan
    call("kvr_paged_map", ctx_len.data_ptr(), new_len.data_ptr(), batch, n_tokens, page, block_table.data_ptr(),
         stride, width, free_pages.data_ptr(), n_pages, n_free.data_ptr(), at,
         at + 4 * (batch + 1), at + 4 * (2 * batch + 6), st.slots.data_ptr(), at + 4 * (2 * batch + 1),
         at + 4 * (2 * batch + 2), n_q, n_kv, window, plan.buf.data_ptr() if plan else None,
         plan.nbytes if plan else 0, stream())
    return st


def paged_write(q, k, v, k_pages, v_pages, slots, positions=None, cos=None, sin=None, q_out=None):
    """RoPE of q (T, n_q, d) and k (T, n_kv, d) at `positions` (cos None: no
    rotation) and the write of k and v into cache slots `slots` (T) int64 of
    the pools (n_pages, page, n_kv, d).  Returns the rotated q (None if q is);
    rows of tokens with slot -1 are 0."""
    n_pages, page, ps, ts = _pool(k_pages, v_pages)
    dt = k_pages.dtype
    k, ks = _tokens(k, "k")
    v, vs = _tokens(v, "v")
    n_tokens, n_kv, _ = shape = k.shape
    if k.dtype is not dt or v.dtype is not dt or (q is not None and q.dtype is not dt):
        raise TypeError("q, k, v and the pools must share a dtype")
    if v.shape != shape or n_kv != k_pages.shape[2] or (q is not None and q.shape[0] != n_tokens):
        raise ValueError("q, k, v and the pools do not fit together")
    if slots.dtype is not torch.int64 or slots.numel() != n_tokens or not slots.is_contiguous():
        raise TypeError("slots must be a contiguous int64 vector, one per token")
    _on_gpu(k, v, k_pages, v_pages, slots)
    qp = qo = cp = sp = pp = None
    qs = n_q = rs = max_pos = 0
    if q is not None:
        q, qs = _tokens(q, "q")
        n_q = q.shape[1]
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif q_out.shape != q.shape or q_out.dtype is not dt or not q_out.is_contiguous():
            raise ValueError("q_out must be contiguous and of q's shape and dtype")
        _on_gpu(q, q_out)
        qp, qo = q.data_ptr(), q_out.data_ptr()
    if cos is not None or sin is not None:
        if cos is None or sin is None or positions is None:
            raise ValueError("RoPE needs both tables and positions")
        _i32(positions, "positions", n_tokens)
        if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
            raise TypeError("the RoPE tables must be fp32")
        max_pos, width = table = cos.shape
        if sin.shape != table or width != D:
            raise ValueError(f"the RoPE tables must be (max_pos, {D})")
        cos, sin, rs = _rope_args(cos, sin)
        _on_gpu(positions, cos, sin)
        cp, sp, pp = cos.data_ptr(), sin.data_ptr(), positions.data_ptr()
    call("kvr_paged_write", qp, k.data_ptr(), v.data_ptr(), dtype_code(k), n_tokens, n_q, n_kv, D, qs, ks, vs, cp, sp, rs,
         max_pos, pp, slots.data_ptr(), qo, k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page, ps, ts, stream())
    return q_out


_ATTN_WS: dict = {}
_ATTN_MAKE = threading.Lock()
# An attention call enqueues two kernels, the second of which reads what the first left in the workspace; the GIL is
# released meanwhile.  A host thread that shares the stream must not come in between: a lock per workspace address.
_ATTN_LOCKS: collections.defaultdict = collections.defaultdict(threading.Lock)


def _attn_workspace(device):
    """(address, bytes) of the attention workspace, and the current stream.
    Calls on one stream do not overlap, so each stream has its own; its size
    does not depend on the call.  Calls in a graph capture take another one, the
    stream's second or, on a stream without (torch's own capture stream), the
    device's (the default stream's second): a graph may be replayed on another
    stream, beside calls on the one it was captured on.  A stream's first call
    outside of a capture allocates both: what a capture allocates is zeroed at
    each replay and belongs to the graph."""
    s = stream()
    capturing = torch.cuda.is_current_stream_capturing()
    ws = _ATTN_WS.get((s, capturing, device))
    if ws is None:
        if capturing:
            ws = _ATTN_WS.get((0, True, device))
            if ws is None:
                raise RuntimeError("the first attention call on a device must be made outside of a graph capture")
        else:
            with _ATTN_MAKE:
                nbytes = call("kvr_attn_workspace_bytes")
                for key in ((0, True, device), (s, True, device), (s, False, device)):
                    if key not in _ATTN_WS:
                        _ATTN_WS[key] = (N.workspace(f"attn_work_{key[0]}_{key[1]}", nbytes, device), nbytes)
                torch.cuda.current_stream(device).synchronize()  # zeroed before a graph on any stream uses them
            ws = _ATTN_WS[s, False, device]
    return ws[0].data_ptr(), ws[1], s


def _attn_out(q, out, return_lse):
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif (out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous()
          or (out.data_ptr() == q.data_ptr() and q.numel())):  # (tensors without elements have one address)
        raise ValueError("out must be contiguous, of q's shape and dtype, and not q itself")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    return out, lse


def paged_attn(q, k_pages, v_pages, block_table, plan, scale=None, out=None, return_lse=False):
    """Attention of a step's query tokens q (T, n_q, d) over their requests'
    pages; `plan` from paged_map or attn_plan(kv_len=...).  Returns out of q's
    shape and dtype, or (out, lse (T, n_q) fp32)."""
    n_pages, page, ps, ts = _pool(k_pages, v_pages)
    q, qs = _tokens(q, "q")
    n_tokens, n_q, _ = q.shape
    plan._match(n_tokens, n_q, True)
    if q.dtype is not k_pages.dtype:
        raise TypeError("q and the pools must share a dtype")
    if k_pages.shape[2] != plan.n_kv:
        raise ValueError(f"the plan is for {plan.n_kv} KV heads, the pool has {k_pages.shape[2]}")
    width, stride = _table(block_table, plan.batch)
    out, lse = _attn_out(q, out, return_lse)
    _on_gpu(q, k_pages, v_pages, block_table, out)
    ws, ws_bytes, s = _attn_workspace(q.device)
    with _ATTN_LOCKS[ws]:
        call("kvr_paged_attn", q.data_ptr(), dtype_code(q), n_tokens, plan.batch, n_q, plan.n_kv, D, qs, k_pages.data_ptr(),
             v_pages.data_ptr(), n_pages, page, ps, ts, block_table.data_ptr(), stride, width, plan.buf.data_ptr(), plan.nbytes,
             float(scale or 0.0), out.data_ptr(), lse.data_ptr() if return_lse else None, ws, ws_bytes, s)
    return (out, lse) if return_lse else out


def prompt_attn(q, k, v, plan, scale=None, out=None, return_lse=False):
    """Attention over whole packed prompts: q (T, n_q, d), k and v (T_k, n_kv,
    d), possibly strided views of one projection; `plan` from attn_plan (made
    without cu_k: k and v are of q's tokens; with it, keys that its offsets name
    past T_k read as zeros).  Returns out of q's shape and dtype, or (out, lse (T, n_q) fp32)."""
    q, qs = _tokens(q, "q")
    k, ks = _tokens(k, "k")
    v, vs = _tokens(v, "v")
    n_tokens, n_q, _ = q.shape
    plan._match(n_tokens, n_q, False)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must share a dtype")
    if k.shape != v.shape or k.shape[1] != plan.n_kv:
        raise ValueError("k and v must be (tokens, n_kv, d) with the plan's n_kv")
    if plan.own_keys and k.shape[0] != n_tokens:
        raise ValueError(f"the plan has no cu_k: the keys must be the {n_tokens} tokens of q, got {k.shape[0]}")
    if k.shape[0] == 0:  # no request has keys: a row that none of them sees stands for the address
        k, v, ks, vs = q.new_zeros(1, plan.n_kv, D), q.new_zeros(1, plan.n_kv, D), plan.n_kv * D, plan.n_kv * D
    out, lse = _attn_out(q, out, return_lse)
    ws, ws_bytes, s = _attn_workspace(q.device)
    with _ATTN_LOCKS[ws]:
        call("kvr_prompt_attn", ptr(q), ptr(k), ptr(v), dtype_code(q), n_tokens, k.shape[0], plan.batch, n_q, plan.n_kv, D,
             qs, ks, vs, ptr(plan.buf), plan.nbytes, float(scale or 0.0), ptr(out), ptr(lse), ws, ws_bytes, s)
    return (out, lse) if return_lse else out


def attn_status(device=None):
    """Raises if an attention call on the current stream, or one in a graph replayed
    on it, gave up or met a plan of other shapes (synchronises the stream).  It
    reads and clears the stream's workspace and those that captures on the
    device use."""
    device = torch.device("cuda" if device is None else device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    _attn_workspace(device)
    s, first = stream(), None
    for (of, capture, dev), ws in list(_ATTN_WS.items()):
        if dev == device and (capture or of == s):
            try:
                call("kvr_workspace_status", ws[0].data_ptr(), s)
            except N.KvrError as e:
                first = first or e
    if first:
        raise first


# ----------------------------------------------------------- beam search --


class BeamStep:
    """What beam_select chose: the n best continuations of each request in order,
    scores (B, n) fp32, beams and tokens (B, n) int32, and the first K of them that
    do not end a sequence, next_scores, next_beams, next_tokens (B, K).  Places
    without a continuation hold -inf, -1, -1.  All lie in one buffer with the call's
    workspace (at most 128 KB a request): clone what is to be kept for long."""

    __slots__ = ("scores", "beams", "tokens", "next_scores", "next_beams", "next_tokens")


BEAM_MAX_BEAMS, BEAM_MAX_N, BEAM_MAX_EOS = 32, 128, 8
_BEAM_WS: dict = {}
_EOS: dict = {}


def beam_select(logits, scores, n=None, eos=()):
    """Beam search's choice: logits (B * K, V), or (B, K, V), of K beams of B
    requests (rows may be strided or expanded) and the beams' scores (B, K) fp32.  A
    continuation's score is its beam's plus the log-softmax of its logit; those that
    are not finite in fp32 (masked by -inf, of a beam of score -inf) are none.  n: how many
    are listed of each request (K * (1 + len(eos)) where not given: enough for K to
    go on).  eos: token ids (host integers) that end a sequence."""
    if logits.dim() == 3:
        logits = logits.flatten(0, 1)
    if scores.dim() != 2 or logits.dim() != 2 or logits.shape[0] != scores.numel():
        raise ValueError(f"logits must be (B * K, V) and scores (B, K), got {tuple(logits.shape)} and {tuple(scores.shape)}")
    if scores.dtype is not torch.float32:
        raise TypeError("scores must be fp32")
    batch, beams = scores.shape
    vocab = logits.shape[1]
    if n is None:
        n = beams * (1 + len(eos))
    if beams < 1 or vocab < 1 or n < beams:
        raise ValueError(f"{beams} beams, {vocab} tokens and {n} continuations: each request needs one at least, and n >= K")
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    scores = _c(scores)
    _on_current_gpu(logits, scores)
    code, dev = dtype_code(logits), logits.device
    eos = tuple(map(int, eos))  # (by value: the arrays below are kept by it)
    ends = _EOS.get(eos)
    if ends is None:
        if len(_EOS) > 256:
            _EOS.clear()
        if not all(0 <= t < 1 << 31 for t in eos):
            raise ValueError(f"eos must be token ids, got {eos}")
        ends = _EOS[eos] = (C.c_int32 * max(len(eos), 1))(*eos)
    key = (batch, beams, vocab, code, n)
    need = _BEAM_WS.get(key)
    if need is None:
        if len(_BEAM_WS) > 4096:
            _BEAM_WS.clear()
        need = _BEAM_WS[key] = call("kvr_beam_select_workspace_bytes", *key)
    # outputs and workspace in one allocation, in this order: scores, next_scores, beams, tokens, next_beams, next_tokens
    m, k = batch * n, batch * beams
    at = (3 * (m + k) + 3) // 4 * 4
    buf = torch.empty(at + need // 4, dtype=_INT32, device=dev)
    st = BeamStep()
    f, listed, kept = buf.view(torch.float32), (n, 1), (beams, 1)
    st.scores, st.next_scores = f.as_strided((batch, n), listed, 0), f.as_strided((batch, beams), kept, m)
    st.beams, st.tokens = buf.as_strided((batch, n), listed, m + k), buf.as_strided((batch, n), listed, 2 * m + k)
    st.next_beams = buf.as_strided((batch, beams), kept, 3 * m + k)
    st.next_tokens = buf.as_strided((batch, beams), kept, 3 * m + 2 * k)
    p = buf.data_ptr()
    call("kvr_beam_select", logits.data_ptr(), code, logits.stride(0), batch, beams, vocab, scores.data_ptr(), n, ends,
         len(eos), p, p + 4 * (m + k), p + 4 * (2 * m + k), p + 4 * m, p + 4 * (3 * m + k), p + 4 * (3 * m + 2 * k),
         p + 4 * at, need, stream())
    return st


REORDER_MAX_BEAMS, REORDER_MAX_ROWS, REORDER_MAX_TABLE = 32, 4096, 1 << 16
REORDER_MAX_ENTRIES = (1 << 30) - 1  # of the call's rows, columns by 32
_REORDER_WS: dict = {}


def paged_reorder(block_table, ctx_len, shared, free_pages, n_free, rows, parents, k_pages, v_pages):
    """Rows of a paged cache become copies of their parents', in place: row rows[g,
    i] of block_table and ctx_len gets what row rows[g, parents[g, i]] had (a parent
    of -1: nothing, the row is emptied).  rows and parents (G, K) int32 on the
    device; no row may be named twice.  shared (n_pages) int32 counts the holders of
    each page beyond the first; free_pages[:n_free] is the list of free ones, with
    room for all.  Full pages are shared; a last page that is not full is copied for
    every row that it falls to but the call's first (for that too, where a row outside of the
    call holds it), in the pools k_pages and v_pages ([layers,] n_pages, page,
    n_kv, d).  Returns info (4) int32 = [pages missing, copied, given back, 0]; a row that finds no page keeps
    its full pages."""
    shape, strides = k_pages.shape, k_pages.stride()
    layers, ls = 1, 0
    if len(shape) == 5:
        layers, ls, shape, strides = shape[0], strides[0], shape[1:], strides[1:]
    if len(shape) != 4 or shape[3] != D or layers < 1:
        raise ValueError(f"k_pages must be ([layers,] pages, page, heads, {D}), got {tuple(k_pages.shape)}")
    if strides[3] != 1 or (shape[2] > 1 and strides[2] != D):
        raise ValueError("k_pages: a token's heads must be contiguous")
    if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.stride() != k_pages.stride():
        raise ValueError("k_pages and v_pages must have one shape, type and layout")
    n_pages, page, n_kv, _ = shape
    ps, ts = strides[0], strides[1]
    _i32(shared, "shared", n_pages)
    cap = _i32(free_pages, "free_pages")
    _i32(n_free, "n_free", 1)
    n_rows = _i32(ctx_len, "ctx_len")
    width, stride = _table(block_table, n_rows)
    if rows.dtype is not _INT32 or parents.dtype is not _INT32 or rows.dim() != 2 or rows.shape != parents.shape:
        raise TypeError("rows and parents must be int32 matrices of one shape (groups, beams)")
    groups, beams = rows.shape
    if beams < 1:
        raise ValueError("a group needs at least one row")
    rows, parents = _c(rows), _c(parents)
    _on_current_gpu(block_table, ctx_len, shared, free_pages, n_free, rows, parents, k_pages, v_pages)
    dev = rows.device
    key = (groups, beams, width)
    need = _REORDER_WS.get(key)
    if need is None:
        if len(_REORDER_WS) > 4096:
            _REORDER_WS.clear()
        need = _REORDER_WS[key] = max(call("kvr_paged_reorder_workspace_bytes", *key), 16)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    info = torch.empty(4, dtype=_INT32, device=dev)
    call("kvr_paged_reorder", block_table.data_ptr(), stride, n_rows, width, ctx_len.data_ptr(), page, shared.data_ptr(),
         n_pages, free_pages.data_ptr(), cap, n_free.data_ptr(), rows.data_ptr(), parents.data_ptr(), groups, beams,
         k_pages.data_ptr(), v_pages.data_ptr(), dtype_code(k_pages), layers, n_kv, D, ls, ps, ts, info.data_ptr(),
         ws.data_ptr(), need, stream())
    return info


# ------------------------------------------------------------ sparse MLP --

MOE_MAX_TOKENS, MOE_MAX_EXPERTS, MOE_MAX_TOP_K = 128, 512, 16
MOE_MAX_HIDDEN, MOE_MAX_INTER = 1 << 16, 1 << 20
_MOE_WS: dict = {}
_MOE_STATUS: dict = {}
_MOE_LOCK = threading.Lock()


def _experts(w, name, shape):
    """(E, rows, columns) with contiguous columns; its strides of experts and rows."""
    if w.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(w.shape)}")
    es, rs, cs = w.stride()
    if cs != 1:
        raise ValueError(f"{name}: rows must be contiguous")
    return (es if shape[0] > 1 else shape[1] * rs), rs


def moe_status_word(device):
    """A word of the caller's own for moe_layer's `status`: what its calls set, no
    other caller's moe_status reads and clears.  Zeroed when this returns."""
    device = torch.device(device)
    word = torch.zeros(256, dtype=torch.uint8, device=device)
    if device.type == "cuda":
        torch.cuda.current_stream(device).synchronize()  # before a call on any stream uses it
    return word


def _moe_status(device):
    ws = _MOE_STATUS.get(device)
    if ws is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first moe_layer call on a device must be made outside of a graph capture")
        with _MOE_LOCK:
            ws = _MOE_STATUS.get(device)
            if ws is None:
                ws = torch.zeros(256, dtype=torch.uint8, device=device)
                torch.cuda.current_stream(device).synchronize()  # zeroed before a call on any stream uses it
                _MOE_STATUS[device] = ws
    return ws


def moe_layer(x, router, gate_up, down, top_k, norm_topk=True, scale=1.0, out=None, return_routing=False, status=None):
    """A sparse MLP of at most MOE_MAX_TOKENS tokens: x (T, H), router (E, H),
    gate_up (E, 2 I, H) with the gate's rows first, down (E, H, I), all fp16 or all
    bf16.  Each token goes to the top_k experts of the largest softmax(x router^T),
    with those as weights (norm_topk: divided by their sum), times scale; an expert is
    down(silu(gate x) * up x).  Returns y (T, H), or (y, ids (T, k) int32, weights (T, k) fp32).
    status: a word of moe_status_word (None: the device's, which moe_status() reads)."""
    if x.dim() != 2 or router.dim() != 2 or gate_up.dim() != 3:
        raise ValueError("x must be (T, H), router (E, H), gate_up (E, 2 I, H), down (E, H, I)")
    n_tokens, hidden = x.shape
    experts, inter = gate_up.shape[0], gate_up.shape[1] // 2
    if router.shape != (experts, hidden):
        raise ValueError(f"router must be {(experts, hidden)}, got {tuple(router.shape)}")
    ge, gr = _experts(gate_up, "gate_up", (experts, 2 * inter, hidden))
    de, dr = _experts(down, "down", (experts, hidden, inter))
    dt = x.dtype
    if router.dtype is not dt or gate_up.dtype is not dt or down.dtype is not dt:
        raise TypeError("x, router and the experts must share a dtype")
    xs, rs = x.stride(0), router.stride(0)
    if x.stride(1) != 1 or (n_tokens > 1 and (xs < hidden or xs % 8)) or x.data_ptr() % 16:
        x, xs = x.clone(memory_format=torch.contiguous_format), hidden
    if n_tokens <= 1:
        xs = hidden
    if router.stride(1) != 1 or (experts > 1 and (rs < hidden or rs % 8)):
        raise ValueError("router: rows must be contiguous and 16-byte aligned")
    if experts == 1:
        rs = hidden
    if out is None:
        out = torch.empty(n_tokens, hidden, dtype=dt, device=x.device)
    elif out.shape != (n_tokens, hidden) or out.dtype is not dt or not out.is_contiguous():
        raise ValueError("out must be contiguous and of x's shape and dtype")
    _on_current_gpu(x, router, gate_up, down, out)
    dev = x.device
    if status is None:
        status = _moe_status(dev)
    elif status.dtype is not torch.uint8 or status.numel() < 4 or status.device != dev:
        raise ValueError("status must be a word of moe_status_word on x's device")
    key = (n_tokens, hidden, inter, experts, top_k)
    need = _MOE_WS.get(key)
    if need is None:
        if len(_MOE_WS) > 4096:
            _MOE_WS.clear()
        need = _MOE_WS[key] = call("kvr_moe_workspace_bytes", *key)
    # workspace (256-byte aligned, as allocations are), then ids and weights, which have their own memory if they are returned
    picks, at = n_tokens * top_k, (need + 3) // 4
    if return_routing:
        buf = torch.empty(at, dtype=_INT32, device=dev)
        ids = torch.empty(n_tokens, top_k, dtype=_INT32, device=dev)
        weights = torch.empty(n_tokens, top_k, dtype=torch.float32, device=dev)
        p, pi, pw = buf.data_ptr(), ids.data_ptr(), weights.data_ptr()
    else:
        buf = torch.empty(at + 2 * picks, dtype=_INT32, device=dev)
        p = buf.data_ptr()
        pi, pw = p + 4 * at, p + 4 * (at + picks)
    call("kvr_moe_layer", x.data_ptr(), dtype_code(x), n_tokens, hidden, xs, router.data_ptr(), rs, gate_up.data_ptr(), ge, gr,
         down.data_ptr(), de, dr, experts, inter, top_k, int(norm_topk), scale, out.data_ptr(), pi, pw, p, need,
         status.data_ptr(), stream())
    return (out, ids, weights) if return_routing else out


def moe_status(device=None, status=None):
    """Raises if a moe_layer call on the device gave up a wait, or, with a word of
    moe_status_word, one that was given it (synchronises the current stream)."""
    if status is None:
        device = torch.device("cuda" if device is None else device)
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        status = _moe_status(device)
    call("kvr_workspace_status", status.data_ptr(), stream())


def kmeans(x, k=128, iters=10):
    """Deterministic Lloyd k-means on the device: x (n, 128) -> (labels (n,)
    int32, centroids (k, 128) fp32)."""
    x = _c(x.float())
    n = x.shape[0]
    c = torch.empty(k, D, dtype=torch.float32, device=x.device)
    lab = torch.empty(n, dtype=torch.int32, device=x.device)
    ws = N.workspace("kmeans", call("kvr_kmeans_workspace_bytes", n, k), x.device)
    call("kvr_kmeans", ptr(x), n, D, k, iters, ptr(c), ptr(lab), ptr(ws), ws.numel(), stream())
    return lab, c


def workspace_status(ws: torch.Tensor):
    call("kvr_workspace_status", ptr(ws), stream())


def default_scale(d=D):
    return math.sqrt(d)
