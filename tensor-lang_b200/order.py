"""Execution order of a lowered program's steps, for passes that recompute a
value instead of reading the stored one: the two are the same only where the
step that stored it ran in the same pass over the same body, and nothing has
written one of its operands since.
"""
from __future__ import annotations

from typing import Iterable, List, Tuple


def ordered(P) -> List[Tuple[object, list, object]]:
    """(body, owning list, step) for every step in execution order; the body is
    the loop that repeats the step, None at the top level."""
    from .engine import _Loop

    out: List[Tuple[object, list, object]] = []

    def walk(body, lst):
        for s in lst:
            if isinstance(s, _Loop):
                for sub in (s.pre, s.bw, s.post, s.rebind):
                    walk(s, sub)
            else:
                out.append((body, lst, s))
    for lst in (P.phase_pre, P.phase_bw, P.phase_post):
        walk(None, lst)
    return out


def buffers(P, names: Iterable[str]) -> set:
    """The names of the buffers that these tensors live in (a rebound value
    lives in its target's)."""
    return {P.alias.get(n, n) for n in names}


def writes_any(P, steps, names) -> bool:
    """Whether one of the steps writes the buffer of one of these tensors."""
    held = buffers(P, names)
    return any(held & buffers(P, s.writes) for s in steps)
