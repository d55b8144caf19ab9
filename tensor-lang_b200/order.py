"""Execution order of a lowered program's steps, for passes that recompute a
value instead of reading the stored one, or that meet a stored value with a
recomputed one: the two are the same only where the step that stored it ran in
the same pass over the same body, and nothing has written one of its operands
since.
"""
from __future__ import annotations

from typing import Iterable, List, Tuple

from .steps import LibCall


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


# argument slots: what tl_linear_ce and tl_linear_ce_backward begin with, and
# where each has its operands and the rows' log sums
_HEAD, _OPERANDS, _FWD_LSE, _BWD_LSE = slice(0, 13), (5, 7, 9), 15, 13


def refresh_log_sums(P) -> int:
    """tl_linear_ce_backward multiplies the logits again, from what x, W and the
    bias are by then, and subtracts the log sums that tl_linear_ce kept: its
    probabilities sum to 1 only where both saw the same operands.  Where they may
    have changed in between (the forward outside of the loop that updates W, an
    update between the two, another loss of the same name), the log sums are
    computed again just before the backward, as the VJP of the current values.
    Returns for how many backwards."""
    made = 0
    while _refresh_once(P):  # a new call's log sums may be what a later backward finds
        made += 1
    return made


def _refresh_once(P) -> bool:
    flat = ordered(P)
    steps = [s for _, _, s in flat]
    for k, (body, lst, b) in enumerate(flat):
        if not isinstance(b, LibCall) or b.fname != "tl_linear_ce_backward":
            continue
        lse = b.args[_BWD_LSE]
        operands = [b.args[i][1] for i in _OPERANDS]
        at = next((i for i in reversed(range(k)) if writes_any(P, [steps[i]], [lse[1]])), None)
        if at is not None and flat[at][0] is body and isinstance(steps[at], LibCall) and \
                steps[at].fname == "tl_linear_ce" and steps[at].args[_FWD_LSE] == lse and \
                all(steps[at].args[i] == b.args[i] for i in range(11)) and \
                not writes_any(P, steps[at:k], operands):
            continue
        scratch = b.args[-2:]
        again = LibCall(f"log_sums:{lse[1]}", "tl_linear_ce",
                        list(b.args[_HEAD]) + [("null",), ("null",), lse] + list(scratch),
                        operands + [b.args[10][1]], [lse[1], scratch[0][1]])
        lst.insert(lst.index(b), again)
        return True
    return False
