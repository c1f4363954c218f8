"""PagedKVCache — the exact K/V of many requests of different lengths in pages.

No reference counterpart (the reference keeps one sequence's window,
modules/kvr_window.py).  A step appends the new tokens of every request (whole
prompts, chunks of prompts, single tokens, in any mix), packed in request
order:

    step = cache.begin(new_len, n_tokens)       # pages, slots, attention plan: one launch
    for layer in range(cache.n_layers):
        q = cache.write(layer, q, k, v, cos, sin)   # RoPE + write into the pages
        out = cache.attend(layer, q)                # every request's tokens over its pages
    cache.commit()                              # the new tokens count as cached

Nothing reads a length on the host, so a step of fixed n_tokens can be captured
in a CUDA graph.
"""
import torch

from . import kernels as K


class PagedKVCache:
    def __init__(self, n_layers, n_q, n_kv, n_pages, page=64, max_requests=32, max_len=32768, window=0,
                 dtype=torch.bfloat16, device="cuda"):
        if page < 8 or page % 8:
            raise ValueError("page must be a multiple of 8")
        self.n_layers, self.n_q, self.n_kv, self.page, self.window = n_layers, n_q, n_kv, page, window
        self.n_pages, self.max_requests = n_pages, max_requests
        self.k = torch.zeros(n_layers, n_pages, page, n_kv, K.D, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_requests, -(-max_len // page)), -1, **i32)
        self.ctx_len = torch.zeros(max_requests, **i32)
        # the last page of the list is taken first; one entry behind it takes what `release` masks out
        self._free = torch.arange(n_pages - 1, -2, -1, **i32)
        self.free_pages = self._free[:n_pages]
        self.n_free = torch.full((1,), n_pages, **i32)
        self.step = None

    def begin(self, new_len, n_tokens):
        """Starts a step that appends new_len[b] tokens to request b (int32 on
        the device, or a list), n_tokens in all (more: padding at the end)."""
        if not torch.is_tensor(new_len):
            new_len = torch.tensor(list(new_len), dtype=torch.int32, device=self.ctx_len.device)
        self.step = K.paged_map(self.ctx_len, new_len, self.block_table, self.free_pages, self.n_free, self.page,
                                n_tokens, n_q=self.n_q, n_kv=self.n_kv, window=self.window)
        return self.step

    def _open(self):
        if self.step is None:
            raise RuntimeError("Call begin() first")
        return self.step

    def write(self, layer, q, k, v, cos=None, sin=None):
        """RoPE of the step's q (T, n_q, d) and k (T, n_kv, d) at their
        positions (cos None: none) and the write of k and v into the layer's
        pages; returns the rotated q."""
        st = self._open()
        return K.paged_write(q, k, v, self.k[layer], self.v[layer], st.slots, st.positions, cos, sin)

    def attend(self, layer, q, scale=None, out=None, return_lse=False):
        """Attention of the step's q over each request's pages, the step's own
        tokens included (write first)."""
        st = self._open()
        return K.paged_attn(q, self.k[layer], self.v[layer], self.block_table, st.plan, scale=scale, out=out,
                            return_lse=return_lse)

    def commit(self):
        """Ends the step: its tokens count as cached, its pages as taken."""
        st = self._open()
        self.ctx_len.copy_(st.kv_len)
        self.n_free.copy_(st.n_free)
        self.step = None

    def check(self):
        """Raises if the open step ran out of pages, tokens or table width
        (synchronises)."""
        missing, cut, over, _ = self._open().info.tolist()
        if missing or cut or over:
            raise RuntimeError(f"step does not fit: {missing} pages missing, {cut} requests cut at n_tokens, "
                               f"{over} longer than max_len")

    def release(self, requests):
        """Gives the pages of `requests` (a list of rows) back to the free list
        and empties the rows; between steps only."""
        if self.step is not None:
            raise RuntimeError("commit() the open step first")
        rows = torch.tensor(list(requests), dtype=torch.int64, device=self.ctx_len.device)
        held = (self.ctx_len[rows] + self.page - 1) // self.page
        j = torch.arange(self.block_table.shape[1], device=rows.device)
        pages = self.block_table[rows]
        mine = (j < held[:, None]) & (pages >= 0)
        at = torch.where(mine, self.n_free + mine.view(-1).cumsum(0).view_as(mine) - 1, self.n_pages)
        self._free.index_put_((at,), pages)
        self.n_free += mine.sum().to(torch.int32)
        self.block_table[rows] = -1
        self.ctx_len[rows] = 0

    def __repr__(self):
        return (f"PagedKVCache(layers={self.n_layers}, heads={self.n_q}/{self.n_kv}, pages={self.n_pages}x{self.page}, "
                f"requests={self.max_requests})")
