"""Token automata (CPU): the tables are the automaton's own."""
import numpy as np
import pytest
import torch

from pico_engine.sampling import TokenAutomaton


@pytest.mark.parametrize("make", [
    lambda rows: np.array(rows, dtype=np.int32), lambda rows: torch.tensor(rows, dtype=torch.int32), lambda rows: torch.tensor(rows), lambda rows: np.array(rows, dtype=np.int64),
])
def test_an_array_that_is_used_again_changes_no_automaton(make):
    rows = [[1, -1, 0], [-1, 0, -1]]
    array = make(rows)
    first = TokenAutomaton(array)
    array[0], array[1] = 7, -1                                            # (states that there are not)
    assert first.transitions.tolist() == rows and first.walk([0, 1, 2]) == 0 and first.walk([1]) == -1
    transitions, masks = first.on("cpu")
    assert transitions.tolist() == rows and masks.tolist() == [[0b101], [0b010]]
    array[:] = 0
    assert first.transitions.tolist() == rows and first.on("cpu")[0].tolist() == rows
