"""Sampling: greedy, temperature, top-k and top-p, under rules on what may be chosen (penalties, biases, a token automaton)."""
from .automaton import TokenAutomaton
from .rules import RuleMemory, StepRules
from .sampler import Sampler, SamplingParams

__all__ = ["RuleMemory", "Sampler", "SamplingParams", "StepRules", "TokenAutomaton"]
