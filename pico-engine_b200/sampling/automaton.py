"""What a sequence may go on with, told by a token automaton: a grammar, a schema, a list of allowed words, compiled to states and transitions."""
from __future__ import annotations

from typing import Dict, Optional, Tuple

import torch


def pack_mask(allowed: torch.Tensor) -> torch.Tensor:
    """Truth values [S, V] as int32 [S, ceil(V / 32)]: bit v % 32 of word v / 32 (``kernels.adjust_logits``)."""
    S, V = allowed.shape
    words = -(-V // 32)
    bits = torch.zeros(S, words * 32, dtype=torch.int64, device=allowed.device)
    bits[:, :V] = allowed
    packed = (bits.view(S, words, 32) << torch.arange(32, device=allowed.device)).sum(dim=2)
    return torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)


class TokenAutomaton:
    """``transitions`` int [S, V]: the state that token v leads to from state s, -1 where the state does not allow it; a sequence starts in
    state ``start``.  Every state has to allow a token (a sequence in one that allows none could not go on); where a sequence may end, that is a stop
    token.  One object serves any number of requests; the engine keeps its tables on the device as long as it lives."""

    def __init__(self, transitions, start: int = 0):
        t = torch.as_tensor(transitions)
        if t.dim() != 2 or t.numel() == 0 or t.is_floating_point() or t.dtype == torch.bool:
            raise ValueError("transitions must be whole numbers [states, vocabulary]")
        if int(t.min()) < -1 or int(t.max()) >= t.shape[0]:
            raise ValueError(f"transitions lead to states -1 (not allowed) to {t.shape[0] - 1}, not to {int(t.min())} .. {int(t.max())}")
        if not 0 <= start < t.shape[0]:
            raise ValueError(f"the start must be one of the {t.shape[0]} states, not {start}")
        stuck = (t < 0).all(dim=1)
        if bool(stuck.any()):
            raise ValueError(f"state {int(stuck.nonzero()[0])} allows no token")
        self.transitions, self.start = t.to(torch.int32, copy=True).contiguous(), int(start)      # (its own: the caller may use the array again)
        self._on: Dict[torch.device, Tuple[torch.Tensor, torch.Tensor]] = {}

    @property
    def vocab(self) -> int:
        return self.transitions.shape[1]

    def on(self, device) -> Tuple[torch.Tensor, torch.Tensor]:
        """(transitions, masks) on ``device``."""
        device = torch.device(device)
        if device not in self._on:
            t = self.transitions.to(device)
            self._on[device] = (t, pack_mask(t >= 0))
        return self._on[device]

    def walk(self, tokens, state: Optional[int] = None) -> int:
        """The state after ``tokens`` (-1: one of them was not allowed)."""
        s = self.start if state is None else state
        for t in tokens:
            s = int(self.transitions[s, t]) if s >= 0 else -1
        return s
