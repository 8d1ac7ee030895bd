"""Serving a compressed LLaMA / Qwen3 model from a paged key/value cache.

`DecodeEngine` feeds a prompt token by token into one dense cache slot per
sequence. `PagedEngine` runs prompts as a whole, keeps every sequence's keys and
values in pages of one pool, lets sequences fork (sharing their common pages),
end and be packed together, and scores tokens:

  per layer   add_rmsnorm (the embedding gather at layer 0) -> q,k,v in one fused SLR launch -> paged_append ->
              paged_prompt_attention / paged_decode_attention -> o_proj ->
              add_rmsnorm -> gate,up -> silu·up -> down_proj
  then        the final add_rmsnorm, the LM head (a plain library GEMM) and,
              for scores, token_logprobs

The reference's generation recomputes the prefix each step
(ssalaad/inference/generate.py:1-26) and keeps no cache. Pages are given out on
the host's count of each sequence's length. A step copies its sequences,
positions and lengths from host memory and so waits for the device's earlier
work; one that needs a new page also reads the free ones' numbers, and a fork
whether it was served.
"""

from __future__ import annotations

import functools

import torch
from torch import nn

from . import _lib
from .decode import _group, _Layer
from .logprobs import TokenLogprobs, token_logprobs
from .paged import (compact_pages, fork_pages, free_pages, paged_append, paged_decode_attention,
                    paged_prompt_attention)


def _on_device(method):
    """The method with the engine's device as torch's current one, without gradients."""
    @functools.wraps(method)
    def call(self, *args, **kw):
        with torch.cuda.device(self.device), torch.no_grad():
            return method(self, *args, **kw)
    return call


class PagedEngine:
    """A model with a pool of `pages` pages of `page` positions for up to
    `max_seqs` sequences. With a window, every layer's attention sees the last
    `window` positions and the first `sinks`."""

    def __init__(self, model: nn.Module, *, max_seqs: int, pages: int, page: int = 64,
                 max_context: int | None = None, window: int = 0, sinks: int = 0) -> None:
        cfg = model.config
        if cfg.model_type not in ("llama", "qwen3"):
            raise ValueError(f"Unsupported model type: {cfg.model_type}")
        if getattr(cfg, "hidden_act", "silu") != "silu":
            raise ValueError(f"unsupported activation {cfg.hidden_act}; the paged step uses silu")
        if any(t != "full_attention" for t in (getattr(cfg, "layer_types", None) or [])):
            raise NotImplementedError("per-layer attention types are not supported by the paged step")
        rot = model.model.rotary_emb
        if getattr(rot, "rope_type", "default") == "dynamic":
            raise NotImplementedError("dynamic rotary scaling is not supported by the paged step")
        if max_seqs < 1 or pages < 1:
            raise ValueError("max_seqs and pages must be positive")
        embed = model.model.embed_tokens.weight
        if not embed.is_cuda:
            raise ValueError("the paged engine runs on a ROCm GPU; move the model to 'cuda' first")
        self.lib = _lib.load()
        self.device, self.dtype = embed.device, embed.dtype
        self.heads, self.kv_heads = cfg.num_attention_heads, cfg.num_key_value_heads
        self.head_dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // self.heads
        if self.head_dim not in (64, 128, 256):
            raise NotImplementedError(f"head_dim {self.head_dim}: the paged attention runs 64, 128 or 256")
        self.eps = float(cfg.rms_norm_eps)
        self.embed, self.norm, self.lm_head = embed, model.model.norm.weight, model.lm_head
        self.window, self.sinks, self.page = window, sinks, page
        self.max_context = max_context or cfg.max_position_embeddings
        self.layers: list[_Layer] = []
        for layer in model.model.layers:
            at, mlp = layer.self_attn, layer.mlp
            L = _Layer()
            L.in_norm = layer.input_layernorm.weight
            L.post_norm = layer.post_attention_layernorm.weight
            L.q_norm = at.q_norm.weight if hasattr(at, "q_norm") else None
            L.k_norm = at.k_norm.weight if hasattr(at, "k_norm") else None
            L.qkv = _group(at.q_proj, at.k_proj, at.v_proj)
            L.o = at.o_proj
            L.gu = _group(mlp.gate_proj, mlp.up_proj)
            L.down = mlp.down_proj
            self.layers.append(L)
        dev = self.device
        shape = (len(self.layers), pages, self.kv_heads, page, self.head_dim)
        self.k_pool = torch.zeros(shape, dtype=self.dtype, device=dev)
        self.v_pool = torch.zeros_like(self.k_pool)
        cols = -(-self.max_context // page)
        self.table = torch.full((max_seqs, cols), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(max_seqs, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        # each sequence's length and pages; a call that fails leaves the lengths, and
        # the pages it reserved to the sequence
        self._host_lengths = [0] * max_seqs
        self._host_pages = [0] * max_seqs
        with torch.no_grad():
            pos = torch.arange(self.max_context, device=dev)[None]
            cos, sin = rot(torch.zeros(1, dtype=torch.float32, device=dev), position_ids=pos)
        half = self.head_dim // 2
        self.cos = cos[0, :, :half].float().contiguous()
        self.sin = sin[0, :, :half].float().contiguous()

    # ------------------------------------------------------------------ pages
    def _ints(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def _names(self, seqs) -> list[int]:
        seqs = [int(s) for s in seqs]
        if not seqs or len(set(seqs)) != len(seqs) or not all(
                0 <= s < len(self._host_lengths) for s in seqs):
            raise ValueError(f"sequences must be distinct and lie in [0, {len(self._host_lengths)})")
        return seqs

    def _reserve(self, seqs: list[int], counts: list[int]) -> None:
        """Pages for `counts` more positions of each sequence."""
        rows, cols = [], []
        for s, n in zip(seqs, counts):
            last = self._host_lengths[s] + n
            if last > self.max_context:
                raise ValueError(f"sequence {s} would pass {self.max_context} positions")
            new = range(self._host_pages[s], -(-last // self.page))
            rows += [s] * len(new)
            cols += new
        if not rows:
            return
        free = (self.refs == 0).nonzero()[: len(rows), 0]
        if free.numel() < len(rows):
            raise RuntimeError(f"{len(rows)} pages needed, {free.numel()} are free")
        at = (torch.tensor(rows, device=self.device), torch.tensor(cols, device=self.device))
        self.table[at] = free.int()
        self.refs[free] = 1
        for s in rows:
            self._host_pages[s] += 1

    @_on_device
    def fork(self, src, dst) -> None:
        """Let the ended sequences dst go on as src do."""
        src, dst = [int(s) for s in src], self._names(dst)
        if len(src) != len(dst):
            raise ValueError(f"{len(src)} sequences to fork into {len(dst)}")
        if not all(0 <= s < len(self._host_lengths) for s in src):
            raise ValueError(f"sequences must lie in [0, {len(self._host_lengths)})")
        if any(self._host_lengths[d] for d in dst):
            raise ValueError("a sequence can be forked into one that has ended only")
        held = [d for d in dst if self._host_pages[d]]  # by a call that failed
        if held:
            self.free(held)
        out = fork_pages(self.table, self.lengths, self.refs, self.k_pool, self.v_pool,
                         self._ints(src), self._ints(dst))
        if not bool(out[3].all()):
            raise RuntimeError("no page is free for a fork")
        self.table, self.lengths, self.refs = out[:3]
        for s, d in zip(src, dst):
            self._host_lengths[d] = self._host_lengths[s]
            self._host_pages[d] = -(-self._host_lengths[s] // self.page)

    @_on_device
    def free(self, seqs) -> None:
        """End sequences."""
        seqs = self._names(seqs)
        self.table, self.lengths, self.refs = free_pages(self.table, self.lengths, self.refs,
                                                         self._ints(seqs))
        for s in seqs:
            self._host_lengths[s] = self._host_pages[s] = 0

    @_on_device
    def compact(self) -> torch.Tensor:
        """Move the pages in use to the lowest numbers; their count (0-d int32)."""
        self.table, self.refs, live = compact_pages(self.table, self.refs, self.k_pool, self.v_pool)
        return live

    # ------------------------------------------------------------------ model
    def _tokens(self, tokens) -> torch.Tensor:
        """Token ids, 1-D int64 on the device; those given on the host are checked."""
        t = torch.as_tensor(tokens, dtype=torch.int64).reshape(-1)
        if not t.is_cuda and t.numel() and (int(t.min()) < 0 or int(t.max()) >= self.embed.shape[0]):
            raise ValueError(f"token ids must lie in [0, {self.embed.shape[0]})")
        return t.to(self.device)

    def _embed_rmsnorm(self, tokens, w):
        h = torch.empty(tokens.numel(), self.embed.shape[1], dtype=self.dtype, device=self.device)
        out = torch.empty_like(h)
        rc = self.lib.ssl_embed_rmsnorm(
            self.embed.data_ptr(), self.embed.stride(0), self.embed.shape[0], tokens.data_ptr(),
            h.data_ptr(), h.stride(0), w.data_ptr(), out.data_ptr(), out.stride(0), h.shape[0],
            h.shape[1], self.eps, _lib.dtype_code(self.dtype), _lib.stream_ptr(self.device))
        _lib.check(rc, "ssl_embed_rmsnorm")
        return h, out

    def _add_rmsnorm(self, h, delta, w):
        out = torch.empty_like(h)
        rc = self.lib.ssl_add_rmsnorm(
            h.data_ptr(), h.stride(0), _lib.ptr(delta), delta.stride(0) if delta is not None else 0,
            w.data_ptr(), out.data_ptr(), out.stride(0), h.shape[0], h.shape[1], self.eps,
            _lib.dtype_code(self.dtype), _lib.stream_ptr(self.device))
        _lib.check(rc, "ssl_add_rmsnorm")
        return out

    def _silu_mul(self, g, u):
        out = torch.empty_like(g)
        rc = self.lib.ssl_silu_mul(
            g.data_ptr(), g.stride(0), u.data_ptr(), u.stride(0), out.data_ptr(), out.stride(0),
            g.shape[0], g.shape[1], _lib.dtype_code(self.dtype), _lib.stream_ptr(self.device))
        _lib.check(rc, "ssl_silu_mul")
        return out

    def _logits(self, tokens: torch.Tensor, seqs: list[int], counts: list[int],
                rows: torch.Tensor | None = None) -> torch.Tensor:
        """Append new tokens, counts[i] of seqs[i]: their logits, or those of `rows`
        of them. The sequences grow when all has been issued."""
        at = self._ints(seqs).long()
        ends = [self._host_lengths[s] + n for s, n in zip(seqs, counts)]
        lengths = self._ints(ends)
        x = self._forward(tokens, seqs, counts, at, lengths, max(ends))
        logits = self.lm_head(x if rows is None else x[rows])
        self.lengths[at] = lengths
        for s, n in zip(seqs, ends):
            self._host_lengths[s] = n
        return logits

    def _forward(self, tokens: torch.Tensor, seqs: list[int], counts: list[int],
                 at: torch.Tensor, lengths: torch.Tensor, longest: int) -> torch.Tensor:
        """The final hidden states of new tokens, counts[i] of seqs[i] (`at` on the
        device), which come to `lengths` by them."""
        starts = [self._host_lengths[s] for s in seqs]
        self._reserve(seqs, counts)
        owners = self._ints([s for s, n in zip(seqs, counts) for _ in range(n)])
        positions = self._ints([a + j for a, n in zip(starts, counts) for j in range(n)])
        table = self.table[at]
        cu = None
        if max(counts) > 1:
            edges = [0]
            for n in counts:
                edges.append(edges[-1] + n)
            cu = self._ints(edges)
        n, H, KH, hd = tokens.numel(), self.heads, self.kv_heads, self.head_dim
        for i, L in enumerate(self.layers):
            if i == 0:
                h, x = self._embed_rmsnorm(tokens, L.in_norm)
            else:
                x = self._add_rmsnorm(h, delta, L.in_norm)
            q, k, v = L.qkv(x)
            q = paged_append(q.view(n, H, hd), k.view(n, KH, hd), v.view(n, KH, hd), self.cos,
                             self.sin, self.k_pool[i], self.v_pool[i], self.table, owners,
                             positions, q_norm=L.q_norm, k_norm=L.k_norm, eps=self.eps)
            if cu is None:
                a = paged_decode_attention(q, self.k_pool[i], self.v_pool[i], table, lengths,
                                           window=self.window, sinks=self.sinks, max_length=longest)
            else:
                a = paged_prompt_attention(q, self.k_pool[i], self.v_pool[i], table, lengths, cu,
                                           window=self.window, sinks=self.sinks,
                                           max_tokens=max(counts), max_length=longest)
            x = self._add_rmsnorm(h, L.o(a.view(n, H * hd)), L.post_norm)
            delta = L.down(self._silu_mul(*L.gu(x)))
        return self._add_rmsnorm(h, delta, self.norm)

    @_on_device
    def feed(self, seqs, tokens, *, all_logits: bool = False):
        """Append tokens to sequences: tokens[i], a 1-D int64 tensor or a list, to
        seqs[i]. Returns the logits after each sequence's last token [n, vocab],
        or with all_logits those after every token [tokens, vocab]. Ids on the host
        are checked; one on the device that no embedding has counts as a zero row."""
        seqs = self._names(seqs)
        parts = [self._tokens(t) for t in tokens]
        counts = [t.numel() for t in parts]
        if len(parts) != len(seqs) or min(counts, default=0) < 1:
            raise ValueError("every sequence takes one or more tokens")
        last = None if all_logits else torch.tensor(counts, device=self.device).cumsum(0) - 1
        return self._logits(torch.cat(parts), seqs, counts, last)

    @_on_device
    def step(self, seqs, tokens: torch.Tensor) -> torch.Tensor:
        """One token a sequence (tokens [n] int64): the logits [n, vocab]."""
        seqs = self._names(seqs)
        if tokens.shape != (len(seqs),):
            raise ValueError(f"a step takes {len(seqs)} tokens, one a sequence")
        return self._logits(self._tokens(tokens), seqs, [1] * len(seqs))

    @_on_device
    def score(self, seq: int, tokens, *, top: int = 0) -> TokenLogprobs:
        """Feed `tokens` to an ended sequence and score each after the first under
        the ones before it."""
        tokens = self._tokens(tokens)
        if self._host_lengths[self._names([seq])[0]]:
            raise ValueError("scores are of a sequence's first tokens; free it before")
        logits = self.feed([seq], [tokens], all_logits=True)
        return token_logprobs(logits[:-1], tokens[1:], top=top)
