"""Llama-shaped models served over a paged key/value cache: prompts in chunks, single tokens and drafted tokens of many
requests in one step.

The reference's generation loop pushes the whole token buffer of one batch through the model for every new token
(Merak/inference/text_generation_inference.py:199-203).  ``LlamaDecoder`` keeps one cache row per sequence and takes one
token at a time; here requests come and go, bring any number of tokens each, and share a pool of pages.

A step of ``PagedLlamaDecoder``: ``ops.paged_plan`` hands out pages, positions and slots from the lengths, and per block
the QKV product, ``ops.qk_norm_rope_append`` (rotary embedding, optional norms of the query and key heads, keys and
values to their pages), ``ops.attn_paged``, and the block's other products.  Everything that depends on lengths lives on
the device.  ``verify`` runs the drafts of every request through one such step and keeps what ``ops.verify_draft``
accepts.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from .. import ops
from .llama_decode import LlamaBlockWeights, hf_weights, rope_tables


class PagedLlamaDecoder:
    """``slots`` requests over ``n_pages`` pages of ``page_size`` tokens per layer.

    ``append(tokens, new_lens)`` adds ``new_lens[r]`` tokens to request r (host numbers; the tokens of all requests one
    after the other) and returns the final-norm output of every new token.  A request that finds no page, or whose length
    would pass ``max_len``, is refused: ``self.granted[r]`` is False, its rows are meaningless and its state is as before.
    ``release([r, ...])`` gives requests' pages back.  ``q_norms`` / ``k_norms``: norm weights [head_dim] of each block's
    query and key heads, for models that have them."""

    def __init__(self, embed: torch.Tensor, blocks: List[LlamaBlockWeights], final_norm: torch.Tensor,
                 lm_head: torch.Tensor, n_q_heads: int, n_kv_heads: int, head_dim: int = 128, eps: float = 1e-5,
                 rope_theta: float = 10000.0, rope_scaling: Optional[dict] = None, max_len: int = 4096, slots: int = 8,
                 page_size: int = 64, n_pages: Optional[int] = None, q_norms: Optional[Sequence[torch.Tensor]] = None,
                 k_norms: Optional[Sequence[torch.Tensor]] = None):
        dev, dt = lm_head.device, lm_head.dtype
        self.embed, self.blocks, self.final_norm, self.lm_head = embed, blocks, final_norm, lm_head
        self.n_q, self.n_kv, self.head_dim, self.eps = n_q_heads, n_kv_heads, head_dim, eps
        self.max_len, self.slots, self.page_size = max_len, slots, page_size
        # what the operators of a step would refuse only after pages have been handed out
        if dt not in (torch.bfloat16, torch.float16) or head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128 and the weights bf16 or f16, got {head_dim} and {dt}")
        if n_kv_heads < 1 or n_q_heads < 1 or n_q_heads % n_kv_heads:
            raise ValueError(f"{n_q_heads} query heads for {n_kv_heads} key heads")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two of at least 16, got {page_size}")
        if max_len < 1 or not 1 <= slots <= 4096 or (n_pages is not None and n_pages < 1):
            raise ValueError(f"max_len {max_len}, slots {slots} (1 .. 4096), n_pages {n_pages}")
        self.q_norms = list(q_norms) if q_norms is not None else [None] * len(blocks)
        self.k_norms = list(k_norms) if k_norms is not None else [None] * len(blocks)
        if len(self.q_norms) != len(blocks) or len(self.k_norms) != len(blocks):
            raise ValueError("q_norms and k_norms need one entry per block")
        for i, (w, *norms) in enumerate(zip(blocks, self.q_norms, self.k_norms)):
            if w.qkv.shape[0] != (n_q_heads + 2 * n_kv_heads) * head_dim or w.o.shape[1] != n_q_heads * head_dim:
                raise ValueError(f"block {i}: weights {tuple(w.qkv.shape)} and {tuple(w.o.shape)} for {n_q_heads}+2*"
                                 f"{n_kv_heads} heads of {head_dim}")
            if any(n is not None and (n.shape != (head_dim,) or n.dtype != dt) for n in norms):
                raise ValueError(f"block {i}: head norms must be {dt} [{head_dim}]")
        per_request = -(-max_len // page_size)
        n_pages = slots * per_request if n_pages is None else n_pages
        cache = lambda: torch.zeros((n_pages, n_kv_heads, page_size, head_dim), dtype=dt, device=dev)
        self.k_cache = [cache() for _ in blocks]
        self.v_cache = [cache() for _ in blocks]
        self.cos, self.sin = rope_tables(head_dim, max_len, rope_theta, rope_scaling, dtype=torch.float32, device=dev)
        self.lens = torch.zeros((slots,), dtype=torch.int64, device=dev)
        self.held = torch.zeros((slots,), dtype=torch.int32, device=dev)
        self.block_tables = torch.full((slots, per_request), -1, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.free_count = torch.tensor([n_pages], dtype=torch.int32, device=dev)
        self.granted = torch.ones((slots,), dtype=torch.bool, device=dev)
        self.attn_ws = ops.attn_paged_workspace(dev)
        self._dev = dev

    @classmethod
    def from_hf(cls, model, **kw):
        """From a ``transformers`` causal model of Llama's arithmetic (``hf_weights`` refuses others), with norms of the query
        and key heads where its attention has them; ``kw``: the sizes of the cache."""
        embed, blocks, norm, head, n_q, n_kv, head_dim, eps, theta, scaling, q_norms, k_norms = hf_weights(
            model, kw.get("max_len", 4096), head_norms=True)
        kw.setdefault("q_norms", q_norms)
        kw.setdefault("k_norms", k_norms)
        return cls(embed, blocks, norm, head, n_q, n_kv, head_dim, eps, theta, scaling, **kw)

    def release(self, finished: Sequence[int]) -> None:
        """The pages of these requests go back to the pool; their lengths become 0."""
        mask = torch.zeros((self.slots,), dtype=torch.bool)
        mask[list(finished)] = True
        mask = mask.to(self._dev)
        ops.paged_release(mask, self.held, self.block_tables, self.free_pages, self.free_count)
        self.lens.masked_fill_(mask, 0)

    def _run(self, tokens: torch.Tensor, new_lens: Sequence[int], takes: Optional[torch.Tensor] = None):
        """-> (hidden of the new tokens, plan, new_lens on the device).  ``takes`` bool [slots] on the device: False: the
        slot's tokens are computed for nothing (the plan refuses them).  Nothing of the decoder changes but table entries
        behind the pages held and cache slots behind the lengths: a step that raises half way has not happened, and
        ``_keep`` makes it count."""
        new_lens = [int(n) for n in new_lens]
        T = sum(new_lens)
        if len(new_lens) != self.slots or min(new_lens) < 0 or tokens.shape != (T,):
            raise ValueError(f"append: {tuple(tokens.shape)} tokens for new_lens {new_lens} of {self.slots} requests")
        new = torch.tensor(new_lens, dtype=torch.int64).to(self._dev)
        lens = self.lens
        if self.max_len % self.page_size:     # the last page has room behind max_len, but the rotary tables end there
            lens = torch.where(lens + new > self.max_len, -1, lens)      # a length that the plan refuses
        if takes is not None:
            lens = torch.where(takes, lens, -1)
        plan = ops.paged_plan(lens, new, self.held, self.block_tables, self.free_pages, self.free_count,
                              self.page_size, T)
        x = ops.embedding_gather(tokens, self.embed, 0, self.embed.shape[0])
        if T == 0:
            return x, plan, new
        residual, most = None, max(new_lens)
        for i, w in enumerate(self.blocks):
            h, residual = ops.rmsnorm(x, w.input_norm, self.eps, residual, want_residual=True)
            qkv = ops.linear_fwd(h, w.qkv, None)[0]
            q = ops.qk_norm_rope_append(qkv, self.cos, self.sin, plan.positions, plan.slots, self.k_cache[i],
                                        self.v_cache[i], self.n_q, self.q_norms[i], self.k_norms[i], self.eps)
            a = ops.attn_paged(q, self.k_cache[i], self.v_cache[i], self.block_tables, plan.cu, plan.kv_lens, max_new=most,
                               workspace=self.attn_ws)
            o = ops.linear_fwd(a.view(T, -1), w.o, None)[0]
            h, residual = ops.rmsnorm(o, w.post_norm, self.eps, residual, want_residual=True)
            act = ops.linear_fwd(h, w.gate_up, None, ops.EPI_SWIGLU, want_pre=False)[1]
            x = ops.linear_fwd(act, w.down, None)[0]
        return ops.rmsnorm(x, self.final_norm, self.eps, residual), plan, new

    def _keep(self, plan: ops.PagedPlan, new: torch.Tensor) -> None:
        """The pages of a step that has run, and ``new[r]`` of its tokens, stay."""
        self.held, self.free_count, self.granted = plan.held, plan.free_count, plan.granted
        self.lens = torch.where(plan.granted, self.lens + new, self.lens)

    def append(self, tokens: torch.Tensor, new_lens: Sequence[int]) -> torch.Tensor:
        """``tokens`` int64 [sum(new_lens)] -> hidden [sum(new_lens), H] after the final norm."""
        hidden, plan, new = self._run(tokens, new_lens)
        self._keep(plan, new)
        return hidden

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return ops.linear_fwd(hidden, self.lm_head, None)[0]

    def step(self, tokens: torch.Tensor, new_lens: Sequence[int]) -> torch.Tensor:
        """Greedy next token of every request that brought tokens (int64 [slots], -1 for the others and for refused
        ones): what the reference picks at :223-227 from the last position."""
        hidden = self.append(tokens, new_lens)
        last = torch.tensor(new_lens).cumsum(0) - 1
        who = [r for r, n in enumerate(new_lens) if n]
        out = torch.full((self.slots,), -1, dtype=torch.int64, device=self._dev)
        if who:
            rows = hidden[last[who].to(self._dev)]
            out[torch.tensor(who).to(self._dev)] = ops.argmax_rows(self.logits(rows))
        return torch.where(self.granted, out, -1)

    def verify(self, last_tokens: torch.Tensor, draft_tokens: torch.Tensor, uniforms: torch.Tensor,
               draft_probs: Optional[torch.Tensor] = None, temperature: float = 1.0, top_k: int = 0, top_p: float = 0.0,
               draft_lens: Optional[Sequence[int]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """One step of speculative decoding: ``last_tokens`` int64 [slots] (not yet in the cache) and ``draft_tokens``
        int64 [slots, K] go through the model together, the sampling tail's filter and softmax give the target's
        probabilities, and ``ops.verify_draft`` decides.  -> (tokens [slots, K + 1], accepted [slots]); the cache keeps
        ``last_tokens`` and the accepted drafts, the last of ``tokens`` is the next call's ``last_tokens``.
        ``draft_probs`` fp32 [slots, K, V], or None for drafts without probabilities of their own; ``uniforms`` fp32
        [slots, K + 1].

        ``draft_lens`` (host numbers) says how many drafts each request has, 0 .. K, or -1 for a slot that is left out;
        a request near ``max_len`` or a full pool can ask for fewer.  None: K drafts for every slot that holds tokens;
        empty slots (never used, or released) are left out, though their rows are computed.  Slots that are left out and
        refused requests (``self.granted[r]`` False) have only -1 and 0 accepted, and stay as they are."""
        R, K = draft_tokens.shape
        if R != self.slots or last_tokens.shape != (R,):
            raise ValueError(f"verify: {tuple(last_tokens.shape)} tokens and {tuple(draft_tokens.shape)} drafts for "
                             f"{self.slots} requests")
        tokens = torch.cat([last_tokens[:, None], draft_tokens], 1).reshape(-1)
        if draft_lens is None:
            takes, limits, rows = self.lens > 0, None, None
            hidden, plan, _ = self._run(tokens, [K + 1] * R, takes)
        else:
            draft_lens = [int(n) for n in draft_lens]
            if len(draft_lens) != R or min(draft_lens) < -1 or max(draft_lens) > K:
                raise ValueError(f"verify: draft_lens {draft_lens} for {R} requests of {K} drafts")
            limits = torch.tensor(draft_lens, dtype=torch.int64).to(self._dev)
            takes = limits >= 0
            rows = torch.tensor([r * (K + 1) + i for r, n in enumerate(draft_lens) for i in range(n + 1)],
                                dtype=torch.int64).to(self._dev)
            hidden, plan, _ = self._run(tokens[rows], [n + 1 for n in draft_lens])
        if hidden.shape[0] == 0:
            self._keep(plan, torch.zeros_like(self.lens))
            return torch.full_like(tokens, -1).view(R, K + 1), torch.zeros_like(self.lens)
        z = ops.sample_top_k_top_p(self.logits(hidden), temperature, top_k, top_p, None, want_filtered=True)[1]
        probs = torch.softmax(z, -1)
        if rows is not None and rows.shape[0] < R * (K + 1):      # rows of drafts that are not there: no weight
            probs = torch.zeros((R * (K + 1), probs.shape[1]), dtype=probs.dtype, device=self._dev).index_copy_(0, rows, probs)
        tokens, accepted = ops.verify_draft(draft_tokens, probs.view(R, K + 1, -1), draft_probs, uniforms, limits)
        served = plan.granted & takes
        # rejected drafts leave the cache by the length alone: their slots are written again by the next tokens
        self._keep(plan, torch.where(served, 1 + accepted, 0))
        self.granted = plan.granted | ~takes
        return torch.where(served[:, None], tokens, -1), torch.where(served, accepted, 0)
