"""TitanMAC without neural memory: the model-level plumbing around the attention path.

``forward`` mirrors titans_core/models/titanmac.py:554-686 for
``use_neural_memory=False``: token + learned position embeddings, the persistent
tokens prepended to every sequence (:608-619), the block stack (:629-640), final
norm, tied LM head over all rows and the slice that drops the persistent rows
(:652-662), optional shifted cross-entropy (:674-684).  Parameter names match the
reference (``embed_tokens``, ``embed_positions``, ``persistent_tokens``,
``layers.N...``, ``norm``, ``lm_head``), so its checkpoints load.  In 16-bit types a
forward, a decode step, a generation and the two halves of a training step
(``forward(ids, labels=...)["loss"].backward()``) are one library call each
(``_stack``, ``_train``); fp32, hooks, active dropout, frozen or shared parameters and
the like go through the modules one by one, where with grad mode on the attention
cores have their own backward kernels and norms and GELU are PyTorch's.

``prefill`` / ``decode_step`` / ``generate`` are new: the reference has no KV cache,
its generation helper re-runs the whole forward for every new token
(examples/train_math.py:146-161).  Here a prompt is run once, every layer's last
``w+1`` keys/values go into a ring cache, the persistent keys/values (which do not
depend on the prompt) are kept once per layer, and each new token attends to one ring
per layer.  A decode step returns the logits the reference's
re-forward would return for its last row.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Union

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import _native, _stack, _train
from ..blocks.titan_block import RMSNorm, TitanBlock
from ..paged_cache import PagedCache, draft_tree
from ..logprobs import TokenLogprobs, token_logprobs


def _in_table(embedding: nn.Module, ids: torch.Tensor):
    """``(ids that can be looked up, which of them are not the ones given)``."""
    rows = getattr(embedding, "num_embeddings", None)  # (another kind of embedding: whatever is not negative)
    known = ids.clamp(0, None if rows is None else rows - 1)
    return known, known != ids


class TitanMAC(nn.Module):
    def __init__(self, config):
        super().__init__()
        self.config = config
        config.validate()
        if getattr(config, "use_neural_memory", False):
            raise NotImplementedError("the neural-memory variants (MAC/MAG/MAL) are not part of this package")
        self.embed_tokens = nn.Embedding(config.vocab_size, config.d_model)
        self.embed_positions = nn.Embedding(config.max_seq_len, config.d_model)
        if config.n_persistent > 0:
            self.persistent_tokens = nn.Parameter(torch.zeros(config.n_persistent, config.d_model))
        else:
            self.register_parameter("persistent_tokens", None)
        self.layers = nn.ModuleList([TitanBlock(config) for _ in range(config.n_layers)])
        self.norm = RMSNorm(config.d_model, eps=config.norm_eps)
        self.lm_head = nn.Linear(config.d_model, config.vocab_size, bias=False)
        if config.tie_weights:
            self.lm_head.weight = self.embed_tokens.weight
        self._init_weights()

    def _init_weights(self) -> None:
        # titanmac.py:140-158: only embeddings, persistent tokens and an untied head are re-initialised
        nn.init.normal_(self.embed_tokens.weight, mean=0.0, std=0.02)
        nn.init.normal_(self.embed_positions.weight, mean=0.0, std=0.02)
        if self.persistent_tokens is not None:
            nn.init.normal_(self.persistent_tokens, mean=0.0, std=0.02)
        if not self.config.tie_weights:
            nn.init.normal_(self.lm_head.weight, mean=0.0, std=0.02)

    # ------------------------------------------------------------------ forward --
    def _embed(self, input_ids: torch.Tensor, first_position: int = 0) -> torch.Tensor:
        B, T = input_ids.shape
        positions = torch.arange(first_position, first_position + T, device=input_ids.device)
        x = self.embed_tokens(input_ids) + self.embed_positions(positions)[None]
        if self.persistent_tokens is not None and first_position == 0:
            x = torch.cat([self.persistent_tokens[None].expand(B, -1, -1), x], dim=1)
        return x

    def _embeds(self) -> bool:
        """Whether the one-call paths embed as this model does (a subclass may do it otherwise)."""
        return not _stack.overrides(self, TitanMAC, "_embed", "_forward_modules")

    def forward(self, input_ids: torch.Tensor, labels: Optional[torch.Tensor] = None,
                attention_mask: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """``{"logits": [B, T, V]}`` and, with ``labels``, ``"loss"``, whose backward reads the logits: until then change a copy
        of them, not themselves.

        An id or label outside the vocabulary is met on the device: in 16-bit types its sequence's logits, or the loss and
        the gradients, are NaN, and ``_native.poll_status`` (which synchronises) raises; otherwise PyTorch's own device-side
        check ends the process's CUDA context.  ``decode_step`` likewise, for its positions too; with paged caches ``prefill``
        and ``decode_step`` meet them on the device in every type."""
        Np = self.config.n_persistent
        rows = logits = held = None  # logits of every row, persistent rows first; of the sequence rows; what holds both
        if torch.is_grad_enabled() and any(p.requires_grad for p in self.parameters()):
            found = _train.stack_forward(self, input_ids) if self._embeds() else None  # one autograd node
            if found is not None:
                logits, held = found
                rows, held.rows = held.rows, None
        else:
            table = _stack.table_of(self) if self._embeds() else None
            if table is not None:  # the whole forward as one call (tmw_stack_forward)
                rows = _stack.forward(table, input_ids)
        if rows is None:
            rows = self._forward_modules(input_ids)
        loss = None
        if labels is not None:
            found = _train.shifted_cross_entropy(rows, labels, Np, logits, held)
            if found is not None:
                logits, loss = found
        if logits is None:
            logits = rows[:, Np:, :] if Np > 0 else rows
        out = {"logits": logits}
        if labels is not None:
            if loss is None:
                shift_logits = logits[..., :-1, :].contiguous()
                shift_labels = labels[..., 1:].contiguous()
                loss = F.cross_entropy(shift_logits.reshape(-1, self.config.vocab_size), shift_labels.reshape(-1),
                                       reduction="mean", ignore_index=-100)
            out["loss"] = loss
        return out

    def token_logprobs(self, input_ids: torch.Tensor, labels: Optional[torch.Tensor] = None, n_top: int = 0) -> TokenLogprobs:
        """What the model says of every next token: entry ``[b, t]`` is the log-probability of ``labels[b, t + 1]`` (default: the
        ids themselves; -100: none) behind the tokens ``0 .. t``, with the entropy and the ``n_top`` most likely ids there.  The
        last column has no next token: its log-probability is 0, its alternatives are what comes next.  ``forward``'s loss is minus
        the mean of the counted entries; gradients flow as they do there."""
        labels = input_ids if labels is None else labels
        targets = torch.full_like(labels, -100)
        targets[:, :-1] = labels[:, 1:]
        return token_logprobs(self.forward(input_ids)["logits"], targets, n_top)

    def _forward_modules(self, input_ids: torch.Tensor) -> torch.Tensor:
        """Logits of every row, persistent rows first, module by module."""
        x = self._embed(input_ids)
        # Same wiring as TitanBlock.forward, with every residual add folded into the RMSNorm that follows it
        # (one kernel): the MLP output of a layer is added by the next layer's first norm, or by the final norm.
        pending = None
        for layer in self.layers:
            if pending is None:
                h = layer.norm_attn(x)
            else:
                x, h = layer.norm_attn.add_forward(x, pending, inplace=True)
            a = layer.attention(h, attn_mask=None)
            x, h = layer.norm_mlp.add_forward(x, a, inplace=True)
            pending = layer.mlp(h)
        h = self.norm(x) if pending is None else self.norm.add_forward(x, pending, inplace=True)[1]
        return _native.project(self.lm_head, h)

    # --------------------------------------------------------------- generation --
    def _need_windowed(self) -> None:
        if getattr(self.config, "use_block_sparse", False):
            raise NotImplementedError(
                "the ring-cache generation path (prefill / decode_step / generate) is built for WindowedAttention; "
                "build the config with use_block_sparse=False (forward() works with either attention class)")

    def _need_caches(self, caches) -> None:
        if len(caches) != len(self.layers):
            raise ValueError(f"one cache for each of the {len(self.layers)} layers expected, got {len(caches)}")

    def new_caches(self, batch: int, device, dtype) -> List[_native.RingCache]:
        self._need_windowed()
        c = self.config
        geometry = (batch, c.n_heads, c.d_head, c.window_size, c.n_persistent)
        if dtype not in _native._DTYPES or c.window_size < 0:
            return [_native.RingCache(*geometry, dtype, device)]  # (raises)
        storage = torch.zeros((len(self.layers), _native.RingCache.elements(*geometry)), dtype=dtype, device=device)
        return [_native.RingCache(*geometry, dtype, device, storage=storage[i]) for i in range(len(self.layers))]

    def new_paged_caches(self, page_table: torch.Tensor, pages: int, page_size: int, dtype,
                         page_dtype: Optional[torch.dtype] = None) -> List[PagedCache]:
        """Caches for ``prefill`` and ``decode_step`` whose sequences live in pages: ``page_table [B, columns]`` (int32, on the
        device, shared by the layers), a pool of ``pages`` pages of ``page_size`` tokens per layer.  ``prefill`` fills every
        sequence's pages with the whole prompt it is given, all prompts of one length; ``decode_step`` takes positions of -1 for
        rows without a sequence (their logits mean nothing).  ``page_dtype`` int8 or float8_e4m3fn: keys and values, the persistent
        ones too, in 8 bits with a scale for every token and head.

        An id outside the vocabulary, a position of ``decode_step`` outside the model's or the pages' table: that row's logits are
        NaN, what it adds to its pages is too (steps that see it are NaN again), the other rows are as they would be, and
        ``_native.poll_status`` raises.  ``prefill`` raises a ValueError for a prompt longer than the model's positions; what of
        it has no place in the pages is left out and reported."""
        self._need_windowed()
        c = self.config
        return [PagedCache(page_table, pages, page_size, c.n_heads, c.d_head, c.window_size, c.n_persistent, dtype, page_dtype=page_dtype)
                for _ in self.layers]

    @torch.no_grad()
    def prefill(self, input_ids: torch.Tensor, caches: Optional[List[Union[_native.RingCache, PagedCache]]] = None):
        """Run the prompt ``[B, T]`` once; returns (logits of the last prompt token ``[B, V]``, caches)."""
        self._need_windowed()
        B, T = input_ids.shape
        Np = self.config.n_persistent
        table = _stack.table_of(self) if self._embeds() else None
        if table is not None:  # the prompt as one call (tmw_stack_forward)
            if caches is None:
                caches = self.new_caches(B, input_ids.device, table.dtype)
            logits = _stack.forward(table, input_ids, caches)
            if logits is not None:
                return logits, caches
        bad = wrong = None  # sequences with an id outside the vocabulary
        if caches is not None and any(isinstance(cache, PagedCache) for cache in caches) and self._embeds():
            if T > getattr(self.embed_positions, "num_embeddings", T):
                raise ValueError(f"a prompt of {T} tokens exceeds max_seq_len (the position-embedding table)")
            input_ids, bad = _in_table(self.embed_tokens, input_ids)
            bad = bad.any(dim=1)
            wrong = bad.to(torch.int32)
        x = self._embed(input_ids)
        if caches is None:  # (the keys' type is that of the embedded rows, not of one table)
            caches = self.new_caches(B, x.device, x.dtype)
        pending = None
        for layer, cache in zip(self.layers, caches):
            attn = layer.attention
            if pending is None:
                h = layer.norm_attn(x)
            else:
                x, h = layer.norm_attn.add_forward(x, pending, inplace=True)
            L = h.shape[1]
            attn._check_lengths(L)
            attn._check_supported(h, None)
            qkv = _native.project(attn.qkv_proj, h)
            q, k, v = attn.split_qkv(qkv)
            o = torch.empty((B, L, attn.n_heads, attn.d_head), dtype=qkv.dtype, device=qkv.device)
            _native.prefill(q, k, v, attn.window_size, attn.num_persistent, out=o.permute(0, 2, 1, 3), algo=attn.algo)
            # hand the keys/values over: the persistent rows are the same for every sequence
            if Np > 0:
                cache.set_persistent(k[0, :, :Np], v[0, :, :Np])
            cache.fill(k[:, :, Np:], v[:, :, Np:], t0=0)
            if wrong is not None and isinstance(cache, PagedCache):  # (one layer's keys are enough: the step's others see its NaN)
                nan = torch.full(k.shape[-1:], float("nan"), dtype=k.dtype, device=k.device).expand(B, k.shape[1], T, -1)
                cache.append(nan, nan, wrong - 1)  # over the wrong sequences' tokens; -1: the others are not there
                cache.append(nan[:, :, :1], nan[:, :, :1], -1 - wrong)  # (-2 stores nothing: it reports)
                wrong = None
            x, h = layer.norm_mlp.add_forward(x, _native.project(attn.out_proj, o.view(B, L, -1)), inplace=True)
            pending = layer.mlp(h)
        last = self.norm(x[:, -1]) if pending is None else self.norm.add_forward(x[:, -1], pending[:, -1])[1]
        logits = self.lm_head(last)
        return logits if bad is None else logits.masked_fill(bad[:, None], float("nan")), caches

    @torch.no_grad()
    def decode_step(self, token_ids: torch.Tensor, pos: torch.Tensor,
                    caches: List[Union[_native.RingCache, PagedCache]]) -> torch.Tensor:
        """One new token per sequence.  ``token_ids [B]``, ``pos [B] int32`` = its index in the sequence
        (the prompt occupied 0..T-1).  Returns logits ``[B, V]``; ``pos`` is not modified."""
        self._need_windowed()
        table = _stack.table_of(self)
        if table is not None:  # the whole step as one call (tmw_decode_step)
            logits = _stack.decode_step(table, token_ids, pos, caches)
            if logits is not None:
                return logits
        c = self.config
        B = token_ids.shape[0]
        at, seen = pos.long(), None
        if any(isinstance(cache, PagedCache) for cache in caches):
            token_ids, unknown = _in_table(self.embed_tokens, token_ids)
            at, outside = _in_table(self.embed_positions, at)
            bad = (unknown | outside) & (pos != -1)  # (-1: a row without a sequence)
            seen = pos.masked_fill(bad, -2)  # where no sequence is: the attention's output is NaN, and it reports
        x = self.embed_tokens(token_ids) + self.embed_positions(at)
        if seen is not None:
            x = x.masked_fill(bad[:, None], float("nan"))
        pending = None
        for layer, cache in zip(self.layers, caches):
            attn = layer.attention
            if pending is None:
                h = layer.norm_attn(x)
            else:
                x, h = layer.norm_attn.add_forward(x, pending, inplace=True)
            qkv = attn.qkv_proj(h).view(B, 3, c.n_heads, c.d_head)
            at_pages = (seen,) if isinstance(cache, PagedCache) else ()
            o = cache.decode(qkv[:, 0], qkv[:, 1], qkv[:, 2], pos, None, *at_pages)
            x, h = layer.norm_mlp.add_forward(x, attn.out_proj(o.view(B, -1)), inplace=True)
            pending = layer.mlp(h)
        h = self.norm(x) if pending is None else self.norm.add_forward(x, pending, inplace=True)[1]
        return self.lm_head(h)

    @torch.no_grad()
    def decode_tree(self, token_ids: torch.Tensor, parents: torch.Tensor, start: torch.Tensor, caches: List[PagedCache],
                    counts: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One step of drafted tokens, a tree of them per sequence: ``token_ids``, ``parents [B, nodes]`` (at most 64; a node's parent is an
        earlier node, -1 where it follows the cached tokens), ``start [B] int32`` = how many tokens are cached (-1: no sequence in this row),
        ``counts [B] int32`` nodes of each (None: all).  Returns logits ``[B, nodes, V]``: at node ``i`` what ``decode_step`` would return
        for its token behind the cached ones and its ancestors.  The nodes' keys and values are tokens ``start ..`` of the pages, where
        ``keep_drafts`` leaves those of an accepted path; the next step, or tree, writes over the others.  Ids and positions outside
        their tables: as for ``new_paged_caches``, node by node, but a tree that does not end within its pages has NaN at every node; rows
        from ``counts`` on mean nothing."""
        self._need_windowed()
        if not all(isinstance(cache, PagedCache) for cache in caches):
            raise TypeError("decode_tree works with paged caches (new_paged_caches)")
        self._need_caches(caches)
        if parents.shape != token_ids.shape:
            raise ValueError(f"token_ids and parents must be [batch, nodes] alike, got {list(token_ids.shape)} and {list(parents.shape)}")
        B, N = token_ids.shape
        tree = draft_tree(parents, start, self.config.window_size)
        if token_ids.numel() == 0:
            return self.lm_head.weight.new_empty(B, N, self.config.vocab_size)
        ids, unknown = _in_table(self.embed_tokens, token_ids)
        at, outside = _in_table(self.embed_positions, tree.positions.long())
        there = (start >= 0)[:, None].expand(B, N)
        if counts is not None:
            there = there & (torch.arange(N, device=start.device) < counts[:, None])
        bad = (unknown | outside) & there
        x = (self.embed_tokens(ids) + self.embed_positions(at)).masked_fill(bad[..., None], float("nan"))
        pending, reported = None, False
        for layer, cache in zip(self.layers, caches):
            attn = layer.attention
            if pending is None:
                h = layer.norm_attn(x)
            else:
                x, h = layer.norm_attn.add_forward(x, pending, inplace=True)
            q, k, v = attn.split_qkv(_native.project(attn.qkv_proj, h))
            o = cache.decode_tree(q, k, v, start, tree, counts)
            if not reported:  # (a start of -2 stores nothing: it reports)
                cache.append(k[:, :, :1], v[:, :, :1], -1 - bad.any(dim=1).to(torch.int32))
                reported = True
            o = o.permute(0, 2, 1, 3).reshape(B, N, -1)
            x, h = layer.norm_mlp.add_forward(x, _native.project(attn.out_proj, o), inplace=True)
            pending = layer.mlp(h)
        h = self.norm(x) if pending is None else self.norm.add_forward(x, pending, inplace=True)[1]
        return _native.project(self.lm_head, h)

    @torch.no_grad()
    def keep_drafts(self, caches: List[PagedCache], start: torch.Tensor, kept: torch.Tensor, counts: torch.Tensor) -> None:
        """The accepted path of ``decode_tree``'s nodes: nodes ``kept[b, : counts[b]]`` (int32, rising) become tokens ``start[b] ..`` of every
        layer's pages; the sequence then has ``start + counts`` tokens."""
        self._need_caches(caches)
        for cache in caches:
            cache.keep(start, kept, counts)

    @torch.no_grad()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int, use_cuda_graph: bool = True) -> torch.Tensor:
        """Greedy continuation of ``input_ids [B, T]``; returns ``[B, T + max_new_tokens]``.

        On the whole-model path all steps are issued by one library call.  Otherwise a step is launch-bound (a dozen small
        kernels per layer), so it is captured once in a CUDA graph and replayed (``use_cuda_graph``); token ids and
        positions live in static device buffers.
        """
        B, T = input_ids.shape
        if T + max_new_tokens > self.config.max_seq_len:
            raise ValueError("prompt + new tokens exceed max_seq_len (the position-embedding table)")
        logits, caches = self.prefill(input_ids)
        table = None if _stack.overrides(self, TitanMAC, "decode_step") else _stack.table_of(self)
        if table is not None:  # every choice and step from one call (tmw_generate)
            tokens = _stack.generate(table, input_ids, logits, caches, max_new_tokens)
            if tokens is not None:
                return tokens
        tok = logits.argmax(dim=-1)
        pos = torch.full((B,), T, dtype=torch.int32, device=input_ids.device)
        out = [input_ids, tok[:, None]]
        step = self.decode_step
        graph = None
        if use_cuda_graph and max_new_tokens > 2:
            static_tok, static_pos = tok.clone(), pos.clone()
            side = torch.cuda.Stream(input_ids.device)
            side.wait_stream(torch.cuda.current_stream(input_ids.device))
            with torch.cuda.stream(side):  # one eager step on the capture stream warms up cuBLAS workspaces
                static_logits = step(static_tok, static_pos, caches)
                static_tok.copy_(static_logits.argmax(dim=-1))
                static_pos += 1
            torch.cuda.current_stream(input_ids.device).wait_stream(side)
            out.append(static_tok.clone()[:, None])
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                static_logits = step(static_tok, static_pos, caches)
                static_tok.copy_(static_logits.argmax(dim=-1))
                static_pos += 1
            for _ in range(max_new_tokens - 2):
                graph.replay()
                out.append(static_tok.clone()[:, None])
        else:
            for _ in range(max_new_tokens - 1):
                logits = step(tok, pos, caches)
                tok = logits.argmax(dim=-1)
                pos = pos + 1
                out.append(tok[:, None])
        return torch.cat(out, dim=1)[:, : T + max_new_tokens]
