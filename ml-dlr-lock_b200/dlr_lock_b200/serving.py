"""Decoding with a locked model on a paged key-value cache.

``PagedCache`` holds the keys and values of many requests in pages, for all layers, with its bookkeeping on the device;
``PagedDecoder`` runs a locked decoder (``build_locked_model``, ``locked_model_from_config``) on it: prompts are admitted,
then every request takes one token per step, at its own length.  The reference decodes through the host framework's
``generate`` and its cache of one length for the whole batch; projections, embedding and the attention within a prompt are
still the host framework's here.

A step reads nothing back from the device and can be captured in a CUDA graph (``PagedDecoder.capture``), with pages taken
from the free ones inside the graph.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from . import attention
from .model import RotaryTables, _fusable, attention_fusable, head_norms


class PagedCache:
    """Keys and values of up to ``requests`` requests of up to ``max_tokens`` tokens, in ``pages`` pages of ``page_size``
    tokens that they share (by default enough for all of them at their longest)."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, requests: int, max_tokens: int, *, pages: Optional[int] = None,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if min(layers, kv_heads, head_dim, requests, max_tokens) < 1:
            raise ValueError("PagedCache: layers, kv_heads, head_dim, requests and max_tokens are at least 1")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"PagedCache holds bfloat16 or float16, not {dtype}")
        attention._page_size("PagedCache", page_size)
        columns = -(-max_tokens // page_size)
        pages = requests * columns if pages is None else pages
        if pages < 1 or pages * page_size > 0x7fffffff or requests > attention.MAX_REQUESTS:
            raise ValueError(f"PagedCache: {pages} pages of {page_size} for {requests} requests")
        self.page_size, self.max_tokens = page_size, columns * page_size
        ints = dict(dtype=torch.int32, device=device)
        with torch.inference_mode(False):        # (a cache made in inference mode may be written to outside of it)
            # (what no token was written to is never read: the memory is not cleared)
            self.values = torch.empty(layers, 2, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
            self.block_table = torch.full((requests, columns), -1, **ints)
            self.lengths = torch.zeros(requests, **ints)
            self.free_pages = torch.arange(pages - 1, -1, -1, **ints)
            self.n_free = torch.full((1,), pages, **ints)

    @property
    def requests(self) -> int:
        return self.lengths.shape[0]

    def layer(self, i: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """The key and value caches of a layer."""
        return self.values[i, 0], self.values[i, 1]

    def plan(self, new_tokens: torch.Tensor, width: int = 1, finished: Optional[torch.Tensor] = None) -> attention.PagedPlan:
        """``paged_plan`` on this cache, in place."""
        return attention.paged_plan(self.lengths, new_tokens, self.block_table, self.free_pages, self.n_free, self.page_size,
                                    width=width, finished=finished, in_place=True)

    def release(self, finished: torch.Tensor) -> None:
        """Give the pages of the requests marked in ``finished`` (requests, bool) back."""
        self.plan(torch.zeros_like(self.lengths), finished=finished)


class PagedDecoder:
    """A locked decoder on a ``PagedCache``.

    ``admit`` takes prompts, ``step`` one token per request; both return the logits of the last token of every request
    that has one.  A request that could not be given its tokens (no free pages, or ``max_tokens`` reached) keeps its length
    (``cache.lengths``; none, where a new prompt was to replace it), and its row of logits is NaN, as is that of a request
    without a token.
    """

    def __init__(self, model, requests: int, max_tokens: int, *, pages: Optional[int] = None, page_size: int = 64):
        layers = model.model.layers
        attn = layers[0].self_attn
        like = attn.q_proj.weight
        if not like.is_cuda or like.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("PagedDecoder runs bfloat16 or float16 models on a GPU (there is no CPU path)")
        for i, layer in enumerate(layers):
            if not _fusable(layer) or not attention_fusable(layer.self_attn):
                raise ValueError(f"PagedDecoder: layer {i} is not a locked layer with full attention and a rotation")
        if not RotaryTables.fixed(model):
            raise ValueError("PagedDecoder: the rotary embedding changes with the length")
        if attn.head_dim not in (64, 96, 128, 256):
            raise ValueError(f"PagedDecoder: heads of {attn.head_dim}: 64, 96, 128 and 256 are supported")
        self.model = model
        kv_heads = attn.k_proj.out_features // attn.head_dim
        self.cache = PagedCache(len(layers), kv_heads, attn.head_dim, requests, max_tokens, pages=pages, page_size=page_size,
                                dtype=like.dtype, device=like.device)
        self._tables = RotaryTables(model, self.cache.max_tokens).on(like.device)
        self._one = torch.ones(requests, dtype=torch.int32, device=like.device)

    def _layers(self, h, plan, attend):
        """h (rows, d) through the layers; attend(layer's attention module, q, k, v, key cache, value cache) -> (rows, heads, dim)."""
        cos, sin = self._tables
        for i, layer in enumerate(self.model.model.layers):
            attn = layer.self_attn
            x = layer.input_layernorm(h)
            q, k, v = (proj(x).unflatten(-1, (-1, attn.head_dim)) for proj in (attn.q_proj, attn.k_proj, attn.v_proj))
            q_weight, k_weight, eps = head_norms(attn)
            out = attend(attn, q, k, v, (q_weight, k_weight, cos, sin, plan.positions, plan.slots, *self.cache.layer(i)), eps)
            h = layer.mlp.dlrnet(h + attn.o_proj(out.flatten(1)))
        return h

    def _flags(self, what, name, flags):
        if flags.shape != (self.cache.requests,):
            raise ValueError(f"{what}: {name} must have shape {(self.cache.requests,)}, not {tuple(flags.shape)}")
        return flags.bool()

    def _embed(self, ids, plan):
        """Embeddings of the rows that have a token; what stands in the others' ids is not looked up."""
        return self.model.model.embed_tokens(ids.flatten().masked_fill(plan.slots < 0, 0))

    def _logits(self, h, has_token):
        logits = self.model.lm_head(self.model.model.norm(h))
        return logits.masked_fill(~has_token[:, None], float("nan"))

    @torch.no_grad()
    def admit(self, ids: torch.Tensor, counts: torch.Tensor, finished: Optional[torch.Tensor] = None) -> torch.Tensor:
        """New prompts: ``ids`` (requests, width), of which the first ``counts`` (requests, int32) of each row count; the
        others may be anything.  A request with a prompt loses what it held; one with a count of 0 keeps it, unless
        ``finished`` (requests, bool) gives its pages back.  Returns logits (requests, vocabulary)."""
        cache = self.cache
        if ids.dim() != 2 or ids.shape[0] != cache.requests or ids.shape[1] < 1:
            raise ValueError(f"admit: expected ids ({cache.requests}, width), got {tuple(ids.shape)}")
        if counts.dtype != torch.int32 or counts.shape != (cache.requests,):
            raise ValueError(f"admit: counts must be int32 of shape {(cache.requests,)}")
        width = ids.shape[1]
        again = counts > 0 if finished is None else (counts > 0) | self._flags("admit", "finished", finished)
        plan = cache.plan(counts, width, again)

        def attend(attn, q, k, v, where, eps):
            q, k = attention.qk_norm_rope_append(q, k, v, *where, eps=eps, return_keys=True)
            # rows behind a prompt's end come after all of its tokens: causal attention never looks there
            q, k, v = (t.view(cache.requests, width, -1, attn.head_dim).transpose(1, 2) for t in (q, k, v))
            out = F.scaled_dot_product_attention(q, k, v, is_causal=True, scale=attn.scaling, enable_gqa=True)
            return out.transpose(1, 2).flatten(0, 1)

        h = self._layers(self._embed(ids, plan), plan, attend)
        first = torch.arange(cache.requests, device=ids.device) * width
        last = first + (counts.long().clamp(1, width) - 1)
        return self._logits(h[last], (counts > 0) & (plan.slots[first] >= 0))

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, active: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token of every request, ``tokens`` (requests), or of those marked in ``active`` (requests, bool; the others'
        may be anything); returns logits (requests, vocabulary)."""
        cache = self.cache
        if tokens.shape != (cache.requests,):
            raise ValueError(f"step: expected tokens ({cache.requests},), got {tuple(tokens.shape)}")
        plan = cache.plan(self._one if active is None else self._flags("step", "active", active).to(torch.int32))

        def attend(attn, q, k, v, where, eps):
            q = attention.qk_norm_rope_append(q, k, v, *where, eps=eps)
            return attention.paged_attention(q, where[-2], where[-1], cache.block_table, cache.lengths, scale=attn.scaling)

        h = self._layers(self._embed(tokens, plan), plan, attend)
        return self._logits(h, plan.slots >= 0)

    def capture(self):
        """One step of all requests as a CUDA graph: (graph, tokens, logits).  Put the tokens in, replay, read the logits.
        The cache is left as it was.  Like all graphs that run the nets, those of one process are not replayed at the same
        time: the nets' workspaces belong to the stream of the capture."""
        cache = self.cache
        tokens = torch.zeros(cache.requests, dtype=torch.long, device=cache.lengths.device)
        state = [t.clone() for t in (cache.lengths, cache.n_free, cache.block_table, cache.free_pages)]

        def restore():
            for t, was in zip((cache.lengths, cache.n_free, cache.block_table, cache.free_pages), state):
                t.copy_(was)

        with torch.cuda.device(tokens.device):
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                # (a first pass on this stream makes the workspaces; its tokens go to free pages or to a place that the first
                # replay writes again)
                self.step(tokens)
                restore()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                logits = self.step(tokens)
        graph.decoder = self                 # (a replay reads its cache and its tables)
        return graph, tokens, logits
