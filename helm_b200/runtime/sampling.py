"""Sampling of the next token in the decode loops.

HELM's PipelineRuntime decodes greedily (helm/runtime/pipeline_runtime.py:300-338:
argmax, eos / pad handling); greedy stays the default here.  With SamplingParams
the loops draw the token on the device instead (helm_sample_tokens): temperature,
top-k, top-p and min-p, from uniforms that a seeded generator on the host gives,
so the same seed gives the same tokens eagerly and from a replayed graph.  Vocabularies
of up to 262144 tokens.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence, Union

import torch

from .. import _capi

_PerRow = Union[float, Sequence[float]]


@dataclass(frozen=True)
class SamplingParams:
    """Per row (a sequence) or for all rows (a number).  temperature 0: the row
    is greedy; top_k 0, top_p 1 and min_p 0: that filter is off."""
    temperature: _PerRow = 1.0
    top_k: Union[int, Sequence[int]] = 0
    top_p: _PerRow = 1.0
    min_p: _PerRow = 0.0
    seed: int = 0


def _rows(name: str, value, batch: int, lo: float, hi: float) -> list:
    rows = list(value) if isinstance(value, (list, tuple)) else [value] * batch
    if len(rows) != batch:
        raise ValueError(f"{name}: {len(rows)} values for a batch of {batch}")
    for x in rows:
        if not lo <= x <= hi:
            raise ValueError(f"{name} = {x} is outside [{lo}, {hi}]")
    return rows


class TokenSampler:
    """Draws one token per row and call.  The uniforms of the next ROWS steps lie
    in a device table, and the step that is next is a device counter, so a captured
    call draws anew at every replay; tick() on the host, before each step, refills
    the table when it is used up."""

    ROWS = 1024

    def __init__(self, params: SamplingParams, batch: int, device: torch.device):
        temp = _rows("temperature", params.temperature, batch, 0.0, float("inf"))
        top_k = _rows("top_k", params.top_k, batch, 0, 2 ** 31 - 1)
        top_p = _rows("top_p", params.top_p, batch, 0.0, 1.0)
        min_p = _rows("min_p", params.min_p, batch, 0.0, 1.0)

        def on(rows, off, dtype):
            if all(x == off for x in rows):
                return None  # the filter is off everywhere
            return torch.tensor(rows, dtype=dtype, device=device)

        self.temperature = on(temp, 1.0, torch.float32)
        self.top_k = on(top_k, 0, torch.int32)
        self.top_p = on(top_p, 1.0, torch.float32)
        self.min_p = on(min_p, 0.0, torch.float32)
        self._gen = torch.Generator().manual_seed(params.seed)
        self._table = torch.empty(self.ROWS, batch, device=device)
        self._next = torch.zeros(1, dtype=torch.long, device=device)
        self._u = torch.empty(1, batch, device=device)
        self._used = self.ROWS
        self.ids = torch.empty(batch, 1, dtype=torch.long, device=device)
        self.logprobs = torch.empty(batch, device=device)

    def tick(self) -> None:
        """Host side of a step: to be called before the step is run or replayed."""
        if self._used == self.ROWS:
            self._table.copy_(torch.rand(self.ROWS, self._table.shape[1], generator=self._gen))
            self._next.zero_()
            self._used = 0
        self._used += 1

    def __call__(self, logits: torch.Tensor) -> torch.Tensor:
        """ids [B, 1] drawn from logits [B, V]; self.logprobs [B] is their log
        softmax(logits / T).  A row without a finite logit gives token 0."""
        torch.index_select(self._table, 0, self._next, out=self._u)
        _capi.sample_tokens(logits, self._u.view(-1), temperature=self.temperature,
                            top_k=self.top_k, top_p=self.top_p, min_p=self.min_p,
                            out=self.ids.view(-1), logprobs=self.logprobs)
        self._next.add_(1)
        return self.ids.clamp_(min=0)
