"""What the rules on the next token keep for every sequence on the device, and what a step hands the kernels."""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

from ..ops import kernels


@dataclass
class StepRules:
    """The rules of one step's rows: ``slots`` int32 [B], and of what the sampler's rules need ``penalties`` float32 [B, 3], the list of biases with
    ``bias_range`` int32 [B, 2]."""
    memory: "RuleMemory"
    slots: torch.Tensor
    penalties: Optional[torch.Tensor] = None
    bias_range: Optional[torch.Tensor] = None
    bias_ids: Optional[torch.Tensor] = None
    bias_values: Optional[torch.Tensor] = None
    grammar: Optional[object] = None

    def apply(self, logits: torch.Tensor) -> torch.Tensor:
        """The logits under the rules, in place."""
        m = self.memory
        masks = None if self.grammar is None else self.grammar.on(logits.device)[1]
        return kernels.adjust_logits(logits, self.slots, None if self.penalties is None else m.history, self.penalties, self.bias_range, self.bias_ids,
                                     self.bias_values, masks, out=logits, states=None if masks is None else m.states)

    def note(self, chosen: torch.Tensor) -> None:
        """The chosen tokens (int32 [B], on the device) into what the sequences have seen, and their automata one state on."""
        m = self.memory
        if self.penalties is not None or self.grammar is not None:
            kernels.note_tokens(None if self.penalties is None else m.history, self.slots, chosen, states=None if self.grammar is None else m.states,
                                transitions=None if self.grammar is None else self.grammar.on(chosen.device)[0])


class RuleMemory:
    """Seen tokens (``history`` int16 [slots, vocab]) and automaton states (int32 [slots]) of the sequence slots and, behind them, of the idle slot."""

    def __init__(self, slots: int, vocab: int, device):
        self.slots, self.vocab, self.device = slots, vocab, torch.device(device)
        self.states = torch.full((slots + 1,), -1, dtype=torch.int32, device=self.device)
        self._history: Optional[torch.Tensor] = None

    @property
    def history(self) -> torch.Tensor:
        if self._history is None:
            self._history = torch.zeros(self.slots + 1, self.vocab, dtype=torch.int16, device=self.device)
        return self._history

    def _ids(self, values) -> torch.Tensor:
        return torch.tensor(list(values), dtype=torch.int32).to(self.device, non_blocking=True)

    def begin(self, params, slots: Sequence[int], prompts: Sequence[Sequence[int]], further: Sequence[Sequence[int]] = ()) -> None:
        """Sequences of ``prompts`` start in ``slots``; those of ``further[i]`` have the prompt of ``slots[i]``."""
        everyone = list(slots) + [s for more in further for s in more]
        if params.penalized:
            h = self.history
            h[slots] = 0
            kernels.note_tokens(h, self._ids(s for s, p in zip(slots, prompts) for _ in p), self._ids(t for p in prompts for t in p), prompt=True)
            for s, more in zip(slots, further):
                if more:
                    h[list(more)] = h[s:s + 1].clone()
        self.states[everyone] = -1 if params.grammar is None else params.grammar.start

    def snapshot(self, slots: List[int]):
        """What the rows of these slots hold (for running a step on trial)."""
        return list(slots), self.states.clone(), None if self._history is None else self._history[slots].clone()

    def restore(self, kept) -> None:
        slots, states, history = kept
        self.states.copy_(states)
        if history is not None:
            self._history[slots] = history

    def rules(self, params, slots: torch.Tensor) -> StepRules:
        """The rules of ``params`` for the rows whose slots are ``slots`` (int32 [B], on the device)."""
        B = slots.shape[0]
        r = StepRules(self, slots, grammar=params.grammar)
        if params.penalized:
            r.penalties = torch.tensor([params.penalties] * B, dtype=torch.float32).to(self.device, non_blocking=True)
        if params.logit_bias:
            r.bias_range = torch.tensor([[0, len(params.logit_bias)]] * B, dtype=torch.int32).to(self.device, non_blocking=True)
            r.bias_ids = self._ids(i for i, _ in params.logit_bias)
            r.bias_values = torch.tensor([v for _, v in params.logit_bias], dtype=torch.float32).to(self.device, non_blocking=True)
        return r
