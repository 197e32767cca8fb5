"""A prefix run through the model once, continued by many sequences.

Scoring several continuations of one context, or generating from one prompt,
needs the context's keys and values only once. :class:`SharedPrefix` keeps each
block's packed Wqkv output of the prefix and then runs only the new tokens:

    shared = SharedPrefix(model, prefix_ids)
    hidden = shared.score([[5, 17], [9]])   # all tokens of both, packed
    logits = shared.logits(hidden)

    shared.begin(count=2, slots=32)         # two sequences, empty so far
    logits = shared.logits(shared.step(torch.tensor([5, 9])))

Runs without gradients, in the model's own precision (autocast included).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from ..ops.attention import flash_attention_qkv
from ..ops.prefix_attention import (
    prefix_attention_decode,
    prefix_attention_qkv,
    sequence_starts,
)
from .mpt import MPTCausalLM


class SharedPrefix:
    """``prefix_ids``: the P >= 1 tokens that all sequences begin with."""

    @torch.no_grad()
    def __init__(self, model, prefix_ids):
        if not isinstance(model, MPTCausalLM):
            raise TypeError("SharedPrefix: wants an MPTCausalLM itself, got "
                            f"{type(model).__name__} (a wrapper that gathers "
                            "parameters in its forward cannot be passed by)")
        self.model = model
        trunk = model.transformer
        self.device = trunk.wte.weight.device
        ids = torch.as_tensor(prefix_ids, dtype=torch.long).to(self.device)
        if ids.dim() != 1 or ids.numel() == 0:
            raise ValueError("SharedPrefix: prefix_ids must be a row of one "
                             "token or more")
        self.length = ids.numel()
        self._qkv: list[torch.Tensor] = []

        def keep(qkv, n_heads, slopes, impl):
            self._qkv.append(qkv[0])
            return flash_attention_qkv(qkv, n_heads, slopes, causal=True, impl=impl)

        hidden = trunk(ids[None], [keep] * len(trunk.blocks))
        #: final hidden state of the prefix's last token, [1, d_model]
        self.last_hidden = hidden[0, -1:]
        self._cache: list[torch.Tensor] = []
        self._held: torch.Tensor | None = None
        self._steps = self._slots = 0

    @torch.no_grad()
    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return F.linear(hidden, self.model.transformer.wte.weight)

    @torch.no_grad()
    def score(self, sequences) -> torch.Tensor:
        """Final hidden states [T, d_model] of all tokens of all sequences
        (lists of token ids; empty ones are allowed), packed in order."""
        flat = [t for s in sequences for t in s]
        starts = sequence_starts([len(s) for s in sequences], self.device)
        if not flat:
            return self.last_hidden[:0]
        ids = torch.tensor([flat], dtype=torch.long, device=self.device)

        def over(prefix):
            def attend(qkv, n_heads, slopes, impl):
                return prefix_attention_qkv(
                    qkv[0], prefix, n_heads, slopes, starts, impl=impl)[None]
            return attend

        return self.model.transformer(ids, [over(p) for p in self._qkv])[0]

    @torch.no_grad()
    def begin(self, count: int, slots: int) -> None:
        """Start ``count`` sequences with room for ``slots`` own tokens each.
        Sequences that were stepped before are gone."""
        if count < 1 or slots < 1:
            raise ValueError("SharedPrefix.begin: count and slots must be >= 1")
        self._cache = []
        for block, qkv in zip(self.model.transformer.blocks, self._qkv):
            h = block.attn.n_heads
            self._cache.append(qkv.new_empty(
                (count, slots, 2, h, qkv.shape[1] // (3 * h))))
        self._held = torch.zeros(count, dtype=torch.int32, device=self.device)
        self._steps, self._slots = 0, slots

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One more token for each sequence ([count] ids); returns their final
        hidden states [count, d_model]."""
        if self._held is None:
            raise RuntimeError("SharedPrefix.step: call begin() first")
        if tokens.shape != self._held.shape:
            raise ValueError(f"SharedPrefix.step: {self._held.numel()} tokens "
                             f"are wanted, got {tuple(tokens.shape)}")
        if self._steps >= self._slots:
            raise IndexError(f"SharedPrefix.step: all {self._slots} slots are filled")
        ids = tokens.to(self.device).view(1, -1)

        def over(prefix, cache):
            def attend(qkv, n_heads, slopes, impl):
                return prefix_attention_decode(
                    qkv[0], prefix, n_heads, slopes, cache, self._held, impl=impl)[None]
            return attend

        hidden = self.model.transformer(
            ids, [over(p, c) for p, c in zip(self._qkv, self._cache)])[0]
        self._held += 1
        self._steps += 1
        return hidden
