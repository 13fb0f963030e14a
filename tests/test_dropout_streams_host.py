"""Which calls of dropout draw masks that have nothing to do with each other."""

from __future__ import annotations

from itertools import combinations

import torch

from _philox import keep


def test_calls_of_a_step_need_offsets_of_their_own():
    """Two calls a step under one seed: with the step alone as their offset, what the first
    drops the second drops too; with two offsets a step no two calls share their drops."""
    rows, cols, p, q = 64, 512, 0.05, 0.1
    one, two = ~keep(rows, cols, p, 7, 3)[0], ~keep(rows, cols, q, 7, 3)[0]
    assert (two | ~one).all()
    masks = []
    for step in range(4):
        masks.append((p, ~keep(rows, cols, p, 7, 2 * step)[0]))
        masks.append((q, ~keep(rows, cols, q, 7, 2 * step + 1)[0]))
    n = rows * cols
    for (a, x), (b, y) in combinations(masks, 2):
        both = float((x & y).double().mean())
        assert abs(both - a * b) < 6 * (a * b * (1 - a * b) / n) ** 0.5
