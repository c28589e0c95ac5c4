"""The cache's page tables on the device, brought up to date by the pages that a step takes."""
from __future__ import annotations

from typing import Dict, List, Sequence, Tuple

import numpy as np
import torch

from ..cache import Cache, pages_for


class ResidentTables:
    """A page table row for every sequence slot in every group of the cache.  A step of one token a row sends four numbers a row and the pages that
    are not there yet, and ``kernels.step_tables`` lays the step out; without them the host writes and sends rows x pages of the longest sequence, every step.
    Rows are known by the sequence that holds the slot (``Cache.births``), so a slot that is closed and opened again starts anew."""

    def __init__(self, cache: Cache, max_context: int):
        self.cache, self.width = cache, pages_for(max_context)
        self.tables = [torch.full((cache.max_seqs + 1, self.width), -1, dtype=torch.int32, device=cache.device) for _ in cache.groups]
        for t in self.tables:
            t[cache.idle_slot, 0] = cache.idle_page
        self.known: List[Dict[int, Tuple[int, int]]] = [{} for _ in cache.groups]       # slot -> (birth, entries on the device)

    @staticmethod
    def takes(cache: Cache) -> bool:
        """Whether tables only ever grow: a group with a window takes entries back, which the rows on the device do not learn."""
        return len(cache.groups) > 0 and all(g.need.window is None for g in cache.groups)

    def fresh(self, group: int, slots: Sequence[int]):
        """(entries on the device of each row, the pages behind them in the rows' order, what the device knows when they are there: for ``learn``) of a step of
        one token a row whose pages have been reserved.  A row's entries go as far as the step's token: what the sequence holds beyond it (reserved ahead) is
        sent when its positions reach there."""
        cache, table, known = self.cache, self.cache.groups[group].table, self.known[group]
        held, pages, learned = np.empty(len(slots), dtype=np.int32), [], {}
        for b, s in enumerate(slots):
            if s == cache.idle_slot:
                held[b] = 1
                continue
            birth, n = known.get(s, (0, 0))
            row = table[s]
            if birth != cache.births[s]:
                n = 0
            held[b] = n
            need = pages_for(cache.lengths[s] + 1)
            if n < need:
                pages.extend(row[n:need])
                learned[s] = (cache.births[s], need)
        return held, pages, learned

    def learn(self, group: int, learned: Dict[int, Tuple[int, int]]) -> None:
        """The step that ``fresh`` described has been launched: its pages need not be sent again.  (One that failed before is described anew.)"""
        self.known[group].update(learned)
