"""What the nodes of a tree of drafted tokens see and where they sit. TEST INFRASTRUCTURE ONLY.

The tree's L nodes are the last L of a sequence's S_b keys. A node sees every key before the tree, itself and
its ancestors; with a window, keys at positions > its own - window, where a node's position is the number of
keys before the tree plus its depth (ancestors are never cut: a window holds at least L keys). A parent of -1 is
the last key before the tree; any other value outside [0, l) makes node l absent, and its descendants with it:
they see nothing and nothing sees them. This operator has no counterpart in the reference.
"""

from __future__ import annotations

import numpy as np


def path(parents, l: int):
    """Node l and its ancestors, or None for an absent node."""
    out = []
    j = l
    while j >= 0:
        out.append(j)
        p = int(parents[j])
        if p < -1 or p >= j:
            return None
        j = p
    return out


def depths(parents) -> list:
    """The depth of every node, -1 for an absent one."""
    ps = [path(parents, l) for l in range(len(parents))]
    return [-1 if p is None else len(p) - 1 for p in ps]


def words(parents) -> np.ndarray:
    """uint32 [L, ceil(L / 32)]: bit j % 32 of word j / 32 of row l set if node j is on l's path."""
    L = len(parents)
    out = np.zeros((L, (L + 31) // 32), np.uint32)
    for l in range(L):
        for j in path(parents, l) or []:
            out[l, j // 32] |= np.uint32(1 << (j % 32))
    return out


def visible(parents, S_b: int, S: int, window: int = 0) -> np.ndarray:
    """bool [L, S]: the keys each node sees in a cache of S rows whose first S_b are the sequence's."""
    L = len(parents)
    out = np.zeros((L, S), bool)
    first = S_b - L
    for l in range(L):
        p = path(parents, l)
        if p is None:
            continue
        lo = max(0, first + len(p) - 1 - window + 1) if window > 0 else 0
        out[l, lo:max(first, 0)] = True
        for j in p:
            if first + j >= 0:
                out[l, first + j] = True
    return out
