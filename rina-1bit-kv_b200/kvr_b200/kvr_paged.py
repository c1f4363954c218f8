"""PagedKVCache — the exact K/V of many requests of different lengths in pages —
and PagedGenerator, which serves them on a HF decoder model.

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
in a CUDA graph.  Between steps ``cache.reorder(rows, parents)`` makes rows the
continuations of others (beams of one request, samples of one prompt): they share
full pages.
"""
import contextlib

import torch

from . import kernels as K


class PagedKVCache:
    """Up to max_requests requests of at most max_len tokens each, on n_pages
    pages of `page` tokens a layer.  Positions stay below max_len, so RoPE tables
    of max_len rows do; a step that would pass it is one that does not fit
    (`check`): its tokens past max_len do not count as cached."""

    def __init__(self, n_layers, n_q, n_kv, n_pages, page=64, max_requests=32, max_len=32768, window=0,
                 dtype=torch.bfloat16, device="cuda"):
        if page < 8 or page % 8:
            raise ValueError("page must be a multiple of 8")
        self.n_layers, self.n_q, self.n_kv, self.page, self.window = n_layers, n_q, n_kv, page, window
        self.n_pages, self.max_requests, self.max_len = n_pages, max_requests, max_len
        self.k = torch.zeros(n_layers, n_pages, page, n_kv, K.D, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_requests, -(-max_len // page)), -1, **i32)
        self.ctx_len = torch.zeros(max_requests, **i32)
        # the last page of the list is taken first; one entry behind it takes what `release` masks out
        self._free = torch.arange(n_pages - 1, -2, -1, **i32)
        self.free_pages = self._free[:n_pages]
        self.n_free = torch.full((1,), n_pages, **i32)
        self.shared = torch.zeros(n_pages, **i32)  # rows that hold a page, beyond the first
        self._sharing = False
        # whether rows can come to share pages, by `reorder` or by kernels.paged_reorder on these tensors
        self._countable = (self.ctx_len.is_cuda and dtype in (torch.float16, torch.bfloat16) and n_layers > 0
                           and max_requests <= K.REORDER_MAX_TABLE)
        self.lost = torch.zeros(4, **i32)  # what committed steps had no room for, as their info counts it
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
        """Ends the step: its tokens (those that found a page and lie below
        max_len) count as cached, its pages as taken."""
        st = self._open()
        self.lost += self._info(st)
        torch.clamp(st.kv_len, max=self.max_len, out=self.ctx_len)
        self.n_free.copy_(st.n_free)
        self.step = None

    def _info(self, st):
        """A step's info with the requests past max_len in its place of requests too long."""
        if self.block_table.shape[1] * self.page == self.max_len:
            return st.info
        past = (st.kv_len > self.max_len).sum(0, keepdim=True, dtype=torch.int32)  # the table's rows are whole pages
        return torch.cat([st.info[:2], torch.maximum(st.info[2:3], past), st.info[3:]])

    def check(self):
        """Raises if the open step ran out of pages, tokens or table width, or,
        between steps, if any step did that was committed since the last such
        check (what a loop of captured steps can ask now and then).
        Synchronises."""
        info = self.lost if self.step is None else self._info(self.step)
        missing, cut, over, _ = info.tolist()
        if missing or cut or over:
            if self.step is None:
                self.lost.zero_()
            raise RuntimeError(f"{'committed steps did' if self.step is None else 'step does'} not fit: {missing} pages missing, "
                               f"{cut} requests cut at n_tokens, {over} longer than max_len")

    def reorder(self, rows, parents):
        """Between steps: rows rows[g][i] become the continuations of rows
        rows[g][parents[g][i]] of their group (a parent of -1: the row is emptied).
        Lists, checked here, or int32 tensors (groups, beams) on the device, which
        must not name a row twice.  Returns kernels.paged_reorder's info; a row that
        finds no page for its copy of a last page that is not full keeps the full
        ones, and `check` says so."""
        if self.step is not None:
            raise RuntimeError("commit() the open step first")
        dev = self.ctx_len.device
        if not torch.is_tensor(rows):
            rows = [[int(b) for b in g] for g in rows]
            flat = [b for g in rows for b in g]
            if len({len(g) for g in rows}) > 1 or not flat:
                raise ValueError("groups must have one number of rows, one at least")
            if len(set(flat)) < len(flat):
                raise ValueError("a row is named twice")
            if not all(0 <= b < self.max_requests for b in flat):
                raise ValueError(f"rows must be in [0, {self.max_requests}), got {rows}")
            rows = torch.tensor(rows, dtype=torch.int32, device=dev)
        if not torch.is_tensor(parents):
            parents = [[int(p) for p in g] for g in parents]
            if any(not -1 <= p < rows.shape[1] for g in parents for p in g):
                raise ValueError(f"parents must be places of the group, or -1, got {parents}")
            parents = torch.tensor(parents, dtype=torch.int32, device=dev)
        info = K.paged_reorder(self.block_table, self.ctx_len, self.shared, self.free_pages, self.n_free, rows, parents,
                               self.k, self.v)
        self._sharing = True
        self.lost[:1] += info[:1]
        return info

    def release(self, requests):
        """Gives the pages of `requests` (a list of rows; one named twice counts
        once) back to the free list and empties the rows; between steps only."""
        if self.step is not None:
            raise RuntimeError("commit() the open step first")
        rows = list(dict.fromkeys(int(b) for b in requests))
        if not all(0 <= b < self.max_requests for b in rows):
            raise ValueError(f"rows must be in [0, {self.max_requests}), got {rows}")
        if rows and (self._sharing or self._countable):  # pages that other rows hold too stay theirs
            columns = -(-self.block_table.shape[1] // 32) * 32
            most = min(K.REORDER_MAX_ROWS, max(K.REORDER_MAX_ENTRIES // columns, 1))
            dev = self.ctx_len.device
            with torch.cuda.device(dev) if dev.type == "cuda" else contextlib.nullcontext():
                for i in range(0, len(rows), most):
                    some = rows[i:i + most]
                    self.reorder([[b] for b in some], [[-1]] * len(some))
            self.block_table[torch.tensor(rows, device=self.ctx_len.device)] = -1  # (steps that were given up leave entries behind)
            return
        rows = torch.tensor(rows, dtype=torch.int64, device=self.ctx_len.device)
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


_MODELS = ("llama", "mistral", "qwen2", "qwen3", "qwen3_moe")  # whose decoder layer `PagedGenerator._layers` is
_ROPE = ("default", "linear", "llama3", "yarn")        # one table for sequences of every length
_PARTS = {"q_proj", "k_proj", "v_proj", "o_proj", "q_norm", "k_norm", "rotary_emb"}


def _model_window(model, max_len):
    """The model's sliding window (0: none, or none within max_len); raises
    NotImplementedError for models with parts that PagedGenerator does not apply."""
    cfg = model.config
    if cfg.model_type not in _MODELS:
        raise NotImplementedError(f"PagedGenerator serves {', '.join(_MODELS)} models, not {cfg.model_type}")
    rope = getattr(cfg, "rope_parameters", None) or getattr(cfg, "rope_scaling", None) or {}
    kind = rope.get("rope_type", rope.get("type", "default"))
    if kind not in _ROPE:
        raise NotImplementedError(f"RoPE of type {kind} (its angles may depend on a sequence's length)")
    for layer in model.model.layers:
        if _sparse(layer.mlp) and cfg.hidden_act != "silu":
            raise NotImplementedError(f"experts with {cfg.hidden_act}")
        more = {n for n, _ in layer.self_attn.named_children()} - _PARTS
        if more:
            raise NotImplementedError(f"attention with {', '.join(sorted(more))}")
        if abs(getattr(layer.self_attn, "scaling", K.D ** -0.5) - K.D ** -0.5) > 1e-6:
            raise NotImplementedError("attention scores scaled by other than 1 / sqrt(head_dim)")
    window = (getattr(cfg, "sliding_window", None) or 0) if getattr(cfg, "use_sliding_window", True) else 0
    if not 0 < window < max_len:
        return 0
    kinds = set(getattr(cfg, "layer_types", None) or ["sliding_attention"])
    if kinds == {"full_attention"}:
        return 0
    if kinds != {"sliding_attention"}:
        raise NotImplementedError("layers with and without a window (a step has one attention plan)")
    return window


def _sparse(mlp):
    """Whether a decoder layer's MLP is a router and experts that kernels.moe_layer
    computes; raises NotImplementedError for one that has other parts."""
    if not hasattr(mlp, "experts"):
        return False
    more = {n for n, _ in mlp.named_children()} - {"gate", "experts"}
    if more:
        raise NotImplementedError(f"a sparse MLP with {', '.join(sorted(more))}")
    gate, experts = mlp.gate, mlp.experts
    names = {n for n, _ in experts.named_parameters()} | {f"gate.{n}" for n, _ in gate.named_parameters()}
    if names != {"gate_up_proj", "down_proj", "gate.weight"} or not hasattr(gate, "top_k"):
        raise NotImplementedError(f"a sparse MLP of {', '.join(sorted(names))}")
    e, h = gate.weight.shape
    if (experts.gate_up_proj.shape[::2] != (e, h) or experts.down_proj.shape[:2] != (e, h)
            or getattr(experts, "is_transposed", False) or not getattr(experts, "has_gate", True)):
        raise NotImplementedError("experts whose weights are laid out otherwise")
    return True


def _readable(w, dtype):
    """Whether kernels.moe_layer takes these weights: their type, 16-byte aligned rows that share no memory."""
    if w.dtype is not dtype or w.data_ptr() % 16:
        return False
    if w.is_contiguous():  # (rows of a multiple of 8)
        return True
    st = w.stride()
    return st[-1] == 1 and not any(s % 8 for s in st[:-1]) and all(s >= n * t for s, n, t in zip(st, w.shape[1:], st[1:]))


class PagedGenerator:
    """Many requests on one HF decoder model (Llama, Mistral, Qwen2 or Qwen3, dense or
    with sparse MLPs, of head_dim 128, fp16 or bf16) with an exact paged cache.

        gen = PagedGenerator(model, n_pages=4096, max_requests=32)
        rows = gen.add([prompt_a, prompt_b])          # prompts in chunks of `chunk` tokens
        tokens = gen.generate(rows, max_new_tokens=64)
        gen.drop(rows)                                # their pages are free again

    ``beam_search`` continues prompts by beams, which share the pages of what they
    have in common.  A step takes any mix of chunks and single tokens (``step``); ``score``
    gives the logits of whole packed prompts without a cache.  window: a query
    sees the last `window` tokens only (0: as many as the model's own sliding
    window, or all); a model's own window bounds it."""

    _status = None  # of sparse MLPs: the word that a call sets whose wait gave up

    def __init__(self, model, n_pages, page=64, max_requests=32, max_len=None, window=0, chunk=2048):
        from .kvr_hook import rope_tables

        cfg = model.config
        self.model, self.device, self.chunk = model, model.device, chunk
        self.n_q, self.n_kv = cfg.num_attention_heads, cfg.num_key_value_heads
        d = getattr(cfg, "head_dim", None) or cfg.hidden_size // self.n_q
        if d != K.D:
            raise ValueError(f"head_dim must be {K.D}, the model has {d}")
        if model.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"the cache holds fp16 or bf16, the model is {model.dtype}")
        max_len = max_len or cfg.max_position_embeddings
        window = min((w for w in (window, _model_window(model, max_len)) if w > 0), default=0)
        self.cache = PagedKVCache(cfg.num_hidden_layers, self.n_q, self.n_kv, n_pages, page, max_requests, max_len, window,
                                  dtype=model.dtype, device=self.device)
        self.cos_tbl, self.sin_tbl = rope_tables(model, max_len, self.device)
        if any(_sparse(layer.mlp) for layer in model.model.layers):
            self._status = K.moe_status_word(self.device)
        self.last = {}  # row -> logits (vocab,) fp32 after its last token

    def _layers(self, h, attend):
        """The decoder layers over packed rows h (T, hidden); attend(layer index, q, k, v) -> (T, n_q, d)."""
        for li, layer in enumerate(self.model.model.layers):
            at = layer.self_attn
            x = layer.input_layernorm(h)
            q, k, v = (p(x).view(x.shape[0], -1, K.D) for p in (at.q_proj, at.k_proj, at.v_proj))
            if hasattr(at, "q_norm"):  # over the channels of each head
                q, k = at.q_norm(q), at.k_norm(k)
            h = h + at.o_proj(attend(li, q, k, v).reshape(x.shape[0], -1))
            h = h + self._mlp(layer.mlp, layer.post_attention_layernorm(h), self._status)
        return self.model.model.norm(h)

    def _check_sparse(self, n_tokens):
        """Raises if a sparse MLP of a pass of n_tokens gave up a wait: its logits, and what it wrote into the cache, then mean
        nothing.  Synchronises, if there was such a call."""
        if self._status is not None and n_tokens <= K.MOE_MAX_TOKENS:
            K.moe_status(status=self._status)

    @staticmethod
    def _mlp(mlp, x, status=None):
        """A layer's MLP over packed rows: a sparse one of a few tokens in one call,
        of more, or of a shape or type that the call does not take, by the model's own module."""
        if not hasattr(mlp, "experts"):
            return mlp(x)
        gate, experts = mlp.gate, mlp.experts
        n, hidden, inter = experts.down_proj.shape
        if (x.shape[0] <= K.MOE_MAX_TOKENS and n <= K.MOE_MAX_EXPERTS and gate.top_k <= K.MOE_MAX_TOP_K
                and hidden % 8 == 0 and inter % 8 == 0 and hidden <= K.MOE_MAX_HIDDEN and inter <= K.MOE_MAX_INTER
                and x.dtype in (torch.float16, torch.bfloat16)
                and all(_readable(w, x.dtype) for w in (gate.weight, experts.gate_up_proj, experts.down_proj))):
            return K.moe_layer(x, gate.weight, experts.gate_up_proj, experts.down_proj, gate.top_k,
                               norm_topk=bool(getattr(gate, "norm_topk_prob", True)), status=status)
        y = mlp(x[None])
        return (y[0] if isinstance(y, tuple) else y)[0]

    @torch.no_grad()
    def step(self, new):
        """One pass: new maps rows to the token ids they get (a chunk or one).
        Returns {row: logits (vocab,) fp32 after its last new token}."""
        rows = sorted(new)
        if rows and not 0 <= rows[0] <= rows[-1] < self.cache.max_requests:
            raise ValueError(f"rows must be in [0, {self.cache.max_requests}), got {rows}")
        lens = [len(new.get(b, ())) for b in range(self.cache.max_requests)]
        if not rows or min(lens[b] for b in rows) < 1:
            raise ValueError("every row of a step needs at least one token")
        ids = torch.tensor([t for b in rows for t in new[b]], device=self.device)
        st = self.cache.begin(lens, ids.numel())
        try:
            self.cache.check()
            h = self._layers(self.model.model.embed_tokens(ids), lambda li, q, k, v: self.cache.attend(
                li, self.cache.write(li, q, k, v, self.cos_tbl, self.sin_tbl)))
            ends = st.cu_q[1:].long()[torch.tensor(rows, device=self.device)] - 1
            logits = self.model.lm_head(h[ends]).float()
            self._check_sparse(ids.numel())
        except BaseException:
            self.cache.step = None  # nothing counts as cached: the step can be tried again, or its rows dropped
            raise
        self.cache.commit()
        out = {b: logits[i] for i, b in enumerate(rows)}
        self.last.update(out)
        return out

    @torch.no_grad()
    def add(self, prompts):
        """Takes prompts (lists of token ids) into free rows, `chunk` tokens a
        step and prompt; returns the rows.  All of them or, where a step fails,
        none: what was taken is given back."""
        left = [list(p) for p in prompts]
        if not all(left):
            raise ValueError("every prompt needs at least one token")
        free = [b for b in range(self.cache.max_requests) if b not in self.last]
        if len(free) < len(left):
            raise RuntimeError(f"{len(left)} prompts for {len(free)} free rows")
        rows = free[:len(left)]
        try:
            while any(left):
                self.step({b: left[i][:self.chunk] for i, b in enumerate(rows) if left[i]})
                left = [p[self.chunk:] for p in left]
        except BaseException:
            self.drop(rows)
            raise
        return rows

    @torch.no_grad()
    def generate(self, rows, max_new_tokens):
        """Greedy decoding of all rows together; returns {row: new token ids}."""
        if len(set(rows)) < len(rows):
            raise ValueError("a row is named twice")
        out = {b: [] for b in rows}
        for _ in range(max_new_tokens):
            for b in rows:
                out[b].append(int(self.last[b].argmax()))
            self.step({b: out[b][-1:] for b in rows})
        return out

    @torch.no_grad()
    def beam_search(self, prompts, n_beams, max_new_tokens, eos=(), length_penalty=1.0):
        """Continues each prompt by beam search over n_beams beams; returns for each
        prompt its best continuations, at most n_beams, best first, as (tokens, score):
        score is the sum of the tokens' log-probabilities over their number to the
        power of length_penalty.  eos: a token id, or several, that end a sequence.  A
        prompt is done when it has n_beams ended sequences that its beams, at their
        present length, do not beat.  It takes n_beams free rows a prompt, and gives
        them back.  At most 32 beams, 8 ends, n_beams * (1 + ends) of 128, and 4096 rows in all."""
        eos = (eos,) if isinstance(eos, int) else tuple(dict.fromkeys(int(t) for t in eos))
        prompts = [list(p) for p in prompts]
        if n_beams < 1 or max_new_tokens < 1:
            raise ValueError("n_beams and max_new_tokens must be 1 at least")
        # what the selection and the reordering take, before prompts are computed for nothing
        if n_beams > K.BEAM_MAX_BEAMS or len(eos) > K.BEAM_MAX_EOS or n_beams * (1 + len(eos)) > K.BEAM_MAX_N:
            raise ValueError(f"at most {K.BEAM_MAX_BEAMS} beams, {K.BEAM_MAX_EOS} ends of sequence and n_beams * (1 + ends) of "
                             f"{K.BEAM_MAX_N}, got {n_beams} beams and {len(eos)} ends")
        if not all(0 <= t < 1 << 31 for t in eos):
            raise ValueError(f"eos must be token ids, got {eos}")
        if n_beams * len(prompts) > K.REORDER_MAX_ROWS or self.cache.max_requests > K.REORDER_MAX_TABLE:
            raise ValueError(f"at most {K.REORDER_MAX_ROWS} rows at a time, of a cache of at most {K.REORDER_MAX_TABLE}")
        free = [b for b in range(self.cache.max_requests) if b not in self.last]
        if len(free) < n_beams * len(prompts):
            raise RuntimeError(f"{len(prompts)} prompts of {n_beams} beams for {len(free)} free rows")
        if not prompts:
            return []
        first = self.add(prompts)
        rest = iter(b for b in free if b not in first)
        rows = [[b] + [next(rest) for _ in range(n_beams - 1)] for b in first]
        try:
            return self._beams(rows, max_new_tokens, eos, length_penalty)
        finally:
            self.drop([b for g in rows for b in g])

    def _reorder(self, rows, parents):
        self.cache.reorder(rows, parents)
        self.cache.check()  # a beam without a page for its copy would go on from a shorter text

    def _beams(self, rows, max_new_tokens, eos, length_penalty):
        n, k = len(rows), len(rows[0])
        logits = torch.stack([self.last[g[0]] for g in rows])[:, None].expand(n, k, -1)  # all beams see the prompt's
        scores = torch.full((n, k), -float("inf"), device=self.device)
        scores[:, 0] = 0.0
        self._reorder(rows, [[0] * k] * n)
        seqs = [[[] for _ in range(k)] for _ in range(n)]
        ended = [[] for _ in range(n)]  # (score, tokens)
        live = set(range(n))
        for t in range(1, max_new_tokens + 1):
            st = K.beam_select(logits, scores, eos=eos)
            cand = [x.tolist() for x in (st.scores, st.beams, st.tokens)]
            nexts = [x.tolist() for x in (st.next_scores, st.next_beams, st.next_tokens)]
            for g in list(live):
                for s, b, tok in list(zip(cand[0][g], cand[1][g], cand[2][g]))[:k]:
                    if b >= 0 and tok in eos:
                        ended[g].append((s / t ** length_penalty, seqs[g][b] + [tok]))
                ended[g] = sorted(ended[g], key=lambda e: -e[0])[:k]
                seqs[g] = [seqs[g][b] + [tok] if b >= 0 else [] for b, tok in zip(nexts[1][g], nexts[2][g])]
                best = max(nexts[0][g])
                if best == -float("inf") or (len(ended[g]) == k and ended[g][-1][0] >= best / t ** length_penalty):
                    live.discard(g)
                    if len(ended[g]) == k:
                        nexts[0][g] = [-float("inf")] * k
            if not live or t == max_new_tokens:
                break
            scores = st.next_scores
            self._reorder(rows, [nexts[1][g] if g in live else [-1] * k for g in range(n)])
            out = self.step({rows[g][i]: [nexts[2][g][i]] for g in sorted(live) for i in range(k) if nexts[1][g][i] >= 0})
            empty = next(iter(out.values()))  # (of beams that there are not: their scores are -inf)
            logits = torch.stack([out.get(b, empty) for g in rows for b in g])
            if len(live) < n:
                scores = scores.clone()
                scores[[g for g in range(n) if g not in live]] = -float("inf")
        for g in range(n):  # beams that have not ended, as they are
            ended[g] += [(s / max(len(q), 1) ** length_penalty, q) for s, q in zip(nexts[0][g], seqs[g]) if s > -float("inf")]
            ended[g] = sorted(ended[g], key=lambda e: -e[0])[:k]
        return [[(q, s) for s, q in e] for e in ended]

    def drop(self, rows):
        """Ends requests: their pages and rows are free again."""
        self.cache.release(rows)
        for b in rows:
            self.last.pop(b, None)

    @torch.no_grad()
    def score(self, prompts):
        """Logits (T, vocab) fp32 of each whole prompt, packed into one pass and
        kept nowhere."""
        lens = [len(p) for p in prompts]
        if not lens or min(lens) < 1:
            raise ValueError("every prompt needs at least one token")
        if max(lens) > self.cos_tbl.shape[0]:
            raise ValueError(f"a prompt of {max(lens)} tokens is longer than max_len = {self.cos_tbl.shape[0]}")
        cu = torch.tensor([0] + lens, device=self.device).cumsum(0).to(torch.int32)
        n = sum(lens)
        plan = K.attn_plan(cu, n, self.n_q, self.n_kv, window=self.cache.window)
        pos = torch.cat([torch.arange(m, device=self.device) for m in lens])
        c, s = self.cos_tbl[pos][:, None], self.sin_tbl[pos][:, None]

        def rope(x):
            y = x.float()
            return (y * c + torch.cat([-y[..., K.D // 2:], y[..., :K.D // 2]], -1) * s).to(x.dtype)

        h = self._layers(self.model.model.embed_tokens(torch.tensor([t for p in prompts for t in p], device=self.device)),
                         lambda li, q, k, v: K.prompt_attn(rope(q), rope(k), v, plan))
        logits = self.model.lm_head(h).float()
        self._check_sparse(n)
        return list(logits.split(lens))
