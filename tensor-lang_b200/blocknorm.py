"""Block-boundary fusion: a peephole pass over a lowered program.

``y = residual_norm(x, u, w, gate)`` followed by ``n = scaled_norm(y, w2)`` is
the end of one block and the start of the next.  Lowered one by one, y is
written by the first kernel and read again by the second, and in the backward
the gradient of y passes through memory between their VJPs.  This pass makes
each pair one call: tl_residual_norm writes y and n from one read of x and u,
and tl_residual_norm_backward takes the gradient of n beside the gradient y has
from its other readers.  The second norm then works on y as the first kernel
holds it, the same float32 value, so forward results do not change.

Forward: nothing between the two steps writes y, the second weight or anything
the first step writes or reads, or touches n.  Backward: the second norm's VJP
is the last to write y's gradient, the first's VJP its only reader after that,
and no one else keeps it; the weight gradient of the second norm is not
touched between them.  The fused call recomputes y from x, u, the weight and
the gate, where the second norm's own VJP reads the stored y: the forward step
that stored it runs in the same loop body as both VJPs (or all of them outside
of loops), and no step between it and them writes y or one of its operands'
buffers.
"""
from __future__ import annotations

from .epilogue import _flat
from .order import ordered, writes_any
from .steps import LibCall

# argument slots of tl_residual_norm and of tl_residual_norm_backward
_DT, _KIND, _ROWS, _COLS, _X, _LDX, _U, _LDU, _WPOST, _GATE, _MODE, _LDG, _ALPHA, _WPRE, _EPS = range(15)
_Y, _LDY, _N, _LDN = range(15, 19)
_DY, _LDDY, _DN, _LDDN, _DX, _LDDX, _DU, _LDDU, _DGATE, _LDDG, _DWPOST, _DWPRE, _ACC = range(15, 28)
_SAME = (_DT, _KIND, _ROWS, _COLS, _EPS)
NULL = ("null",)
ACC_DX, ACC_DW_PRE = 1, 16


def fuse_block_norms(P) -> int:
    """Apply both rewrites wherever they match; returns how many were made."""
    aliased = set(P.alias) | set(P.alias.values())
    pinned = None if P.fetch is None else set(P.fetch) | set(P.initial) | {s["tensor"] for s in P.saves}
    total = 0
    while _forward_once(P, aliased):
        total += 1
    while pinned is not None and _backward_once(P, aliased, pinned):
        total += 1
    return total


def _touched(steps, name) -> bool:
    return any(name in s.reads or name in s.writes for s in steps)


def _forward_once(P, aliased) -> bool:
    flat = _flat(P)
    steps = [s for _, s in flat]
    for i, first in enumerate(steps):
        if not _is(first, "tl_residual_norm") or first.args[_N] != NULL or first.args[_U] == NULL:
            continue
        y = first.args[_Y][1]
        for j in range(i + 1, len(steps)):
            second = steps[j]
            if flat[j][0] is not flat[i][0]:  # another phase or loop
                break
            if not _is(second, "tl_residual_norm") or second.args[_X] != ("ptr", y):
                continue
            b = second.args
            if b[_U] != NULL or b[_Y] != NULL or b[_ALPHA][1] != 1.0 or \
                    any(b[k] != first.args[k] for k in _SAME):
                continue
            n, between = b[_N][1], steps[i + 1:j]
            weights = [b[_WPRE][1]] if b[_WPRE] != NULL else []
            if n in aliased or y in aliased or n == y or _touched(between, n) or \
                    writes_any(P, between, [y] + weights) or n in first.reads:
                continue
            fused = LibCall(f"{first.label}+{second.label}", first.fname,
                            _with(first.args, {_WPRE: b[_WPRE], _N: b[_N], _LDN: b[_LDN]}),
                            list(first.reads) + weights, list(first.writes) + [n])
            lst = flat[i][0]
            lst[lst.index(first)] = fused
            lst.remove(second)
            return True
    return False


def _backward_once(P, aliased, pinned) -> bool:
    flat = ordered(P)
    steps = [s for _, _, s in flat]
    for i, inner in enumerate(steps):  # the VJP of n = scaled_norm(y)
        if not _is(inner, "tl_residual_norm_backward") or inner.args[_U] != NULL or \
                inner.args[_DX] == NULL or inner.args[_DY] != NULL:
            continue
        a = inner.args
        gy = a[_DX][1]
        if gy in pinned or gy in aliased:
            continue
        j = next((k for k in range(i + 1, len(steps)) if gy in steps[k].reads or gy in steps[k].writes), None)
        if j is None or flat[j][1] is not flat[i][1]:
            continue
        outer = steps[j]  # the VJP of y = residual_norm(x, u)
        b = outer.args
        if not _is(outer, "tl_residual_norm_backward") or b[_DY] != ("ptr", gy) or b[_DN] != NULL or \
                any(b[k] != a[k] for k in _SAME) or gy in outer.writes or \
                _touched(steps[j + 1:], gy) or \
                any(gy in s.reads for s, f in zip(steps[:i], flat) if f[1] is not flat[i][1]):
            continue  # (the last: a step before the backward reads the last iteration's)
        y = a[_X][1]
        # y is what the outer VJP recomputes: the last step to write it had the same
        # operands, in the same body, and they are what they were
        at = next((k for k in reversed(range(i)) if writes_any(P, [steps[k]], [y])), None)
        if at is None or flat[at][0] is not flat[i][0]:
            continue
        made = steps[at]
        if not _is(made, "tl_residual_norm") or made.args[_Y] != ("ptr", y) or \
                made.args[_ROWS:_WPRE] != b[_ROWS:_WPRE] or \
                writes_any(P, steps[at:j], made.reads):
            continue
        dn, w, dw = a[_DN][1], a[_WPRE], a[_DWPRE]
        between, operands = steps[i + 1:j], [dn] + ([w[1]] if w != NULL else [])
        if writes_any(P, between, [y] + operands):
            continue
        if dw != NULL and (_touched(between, dw[1]) or dw[1] in outer.reads or dw[1] in outer.writes):
            continue
        others = a[_ACC][1] & ACC_DX  # y's gradient from its other readers
        acc = b[_ACC][1] | (a[_ACC][1] & ACC_DW_PRE)
        fused = LibCall(f"{inner.label}+{outer.label}", outer.fname,
                        _with(b, {_WPRE: w, _DN: a[_DN], _LDDN: a[_LDDN], _DWPRE: dw,
                                  _DY: b[_DY] if others else NULL, _ACC: ("int", acc)}),
                        [r for r in outer.reads if others or r != gy] + operands +
                        ([dw[1]] if dw != NULL and a[_ACC][1] & ACC_DW_PRE else []),
                        list(outer.writes) + ([dw[1]] if dw != NULL else []))
        lst = flat[j][1]
        lst[lst.index(outer)] = fused
        lst.remove(inner)
        return True
    return False


def _is(s, fname) -> bool:
    return isinstance(s, LibCall) and s.fname == fname


def _with(args, changes) -> list:
    args = list(args)
    for k, v in changes.items():
        args[k] = v
    return args
