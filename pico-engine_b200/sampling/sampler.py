"""Choosing next tokens from logits on the device."""
from __future__ import annotations

import math
import operator
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from ..ops import kernels
from .automaton import TokenAutomaton

FLOAT32_TINY, FLOAT32_MAX = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max       # what the kernels take


@dataclass(frozen=True)
class SamplingParams:
    """Names, defaults and meanings of pico-engine's sampler (src/pico_engine/sampler.py:8-27,
    src/pico_engine/__main__.py:25-28): ``temperature <= 0`` is greedy; ``top_k`` 0 is off and
    keeps ties with the k-th largest; ``top_p`` keeps the smallest set of most likely tokens
    whose mass reaches it (1.0 is off).  ``seed`` names the stream of draws, which the project
    leaves to torch's global generator.

    Rules on what may be chosen, which the project does not have, change the logits before all that: ``repetition_penalty`` divides the
    positive and multiplies the negative ones of tokens in the prompt or the output; ``presence_penalty`` and ``frequency_penalty`` (times
    the number of times) are taken off those of tokens in the output; ``logit_bias`` ((token, value), ..) is added; ``grammar`` allows what its
    state for the sequence allows (where biases of -inf leave none of that, the choice is no longer the grammar's)."""
    temperature: float = 0.7
    top_k: int = 0
    top_p: float = 0.9
    seed: int = 0
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Tuple[Tuple[int, float], ...] = ()
    grammar: Optional[TokenAutomaton] = None

    def __post_init__(self):
        if not FLOAT32_TINY <= self.repetition_penalty <= FLOAT32_MAX:
            raise ValueError("repetition_penalty must be positive")
        if not (abs(self.presence_penalty) <= FLOAT32_MAX and abs(self.frequency_penalty) <= FLOAT32_MAX):
            raise ValueError("presence_penalty and frequency_penalty must be numbers")
        bias = self.logit_bias.items() if isinstance(self.logit_bias, dict) else self.logit_bias
        try:
            bias = tuple((operator.index(t), float(v)) for t, v in bias)
        except TypeError:
            raise ValueError("logit_bias must be pairs of a token and a number") from None
        if any(t < 0 or not (abs(v) <= FLOAT32_MAX or v == -math.inf) for t, v in bias) or len({t for t, _ in bias}) != len(bias):
            raise ValueError("logit_bias names tokens, each once, with a number (or -inf) each")
        object.__setattr__(self, "logit_bias", bias)
        if self.grammar is not None and not isinstance(self.grammar, TokenAutomaton):
            raise ValueError("grammar must be a TokenAutomaton")
        if self.top_k < 0:
            raise ValueError("top_k must be non-negative")
        if not 0.0 < self.top_p <= 1.0:
            raise ValueError("top_p must lie in (0, 1]")

    @property
    def greedy(self) -> bool:
        return self.temperature <= 0

    @property
    def penalties(self) -> Tuple[float, float, float]:
        return (self.repetition_penalty, self.presence_penalty, self.frequency_penalty)

    @property
    def penalized(self) -> bool:
        return self.penalties != (1.0, 0.0, 0.0)

    @property
    def ruled(self) -> bool:
        """Whether any rule changes the logits."""
        return self.penalized or bool(self.logit_bias) or self.grammar is not None

    def check_vocab(self, vocab: int) -> None:
        """Refuse rules on tokens that the model does not have."""
        if any(t >= vocab for t, _ in self.logit_bias):
            raise ValueError(f"logit_bias names token {max(t for t, _ in self.logit_bias)}, the vocabulary has {vocab}")
        if self.grammar is not None and self.grammar.vocab != vocab:
            raise ValueError(f"the grammar is for a vocabulary of {self.grammar.vocab}, the model's has {vocab}")


class Sampler:
    def __init__(self, params: SamplingParams):
        self.params = params

    def kind(self, vocab: int) -> tuple:
        """What fixes the kernels that a choice launches: (greedy, a cut by rank, a cut by mass).  Samplers of
        one kind differ in numbers only (temperature, k, p, seed), which a captured launch reads at run time."""
        p = self.params
        return (True, False, False) if p.greedy else (False, 0 < p.top_k < vocab, p.top_p < 1.0)

    BIAS_ROOM = 64       # a captured launch has room for a multiple of so many biases (the next power of two times it)

    def rule_kind(self) -> tuple:
        """The same for its rules: (penalties, room for so many biases, the grammar)."""
        p, room = self.params, 0
        if p.logit_bias:
            room = self.BIAS_ROOM
            while room < len(p.logit_bias):
                room *= 2
        return (p.penalized, room, p.grammar)

    def choose(self, logits: torch.Tensor, request: torch.Tensor, step: torch.Tensor,
               out: torch.Tensor | None = None, settings: torch.Tensor | None = None, rules=None) -> torch.Tensor:
        """int32 [B] next tokens for float32 logits [B, V].  Row b draws with the uniform of
        (seed, request[b], step[b]); greedy choice ignores both.  ``settings``: int32 [6] on the device
        (``kernels.sample_settings_words``) from which the kernels take temperature, top-k, top-p and seed
        instead of from this sampler's parameters, which then only say which kind of choice it is.  ``rules`` (``StepRules``): change the
        logits (in place) before the choice, and learn what was chosen."""
        p = self.params
        if rules is not None:
            rules.apply(logits)
        if p.greedy:
            chosen = kernels.argmax(logits, out)
        else:
            chosen = kernels.sample(logits, p.temperature, p.top_k, p.top_p, p.seed, request, step, out, settings)
        if rules is not None:
            rules.note(chosen)
        return chosen
