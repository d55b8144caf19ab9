"""Programs of the language-model operators whose forward, backward and updates
stand in different places, against the float64 oracle.

Tolerance rel 1e-4 of the value and of the tensor's largest, the suite's for
training.
"""
import numpy as np
import pytest

from conftest import assert_close, load_backend
from oracle import OracleProgram
from test_lm_programs_cpu import BW, C, CE_BW, L, N, S, Y, _loop, _sgd, _sgd2, head, loss, norms

pytestmark = pytest.mark.gpu
tl = load_backend()


def agree(ast, feeds, fetch, **kw):
    env = {"s": {"shape": ()}}
    P = tl.Program(ast, env, feeds=feeds, fetch=list(fetch), **kw)
    got = P.run()
    shapes = {k: {"shape": v} for k, v in P.shapes.items()}
    P.free()
    ref = OracleProgram(ast, shapes, dtype=np.float64, feeds=feeds).run()
    for k in fetch:
        assert_close(got[k], ref[k], 1e-4, k)


def norm_feeds(seed=0):
    rng = np.random.default_rng(seed)
    f = lambda *s, a=1.0, b=0.0: (rng.standard_normal(s) * a + b).astype(np.float32)  # noqa: E731
    return {"x": f(4, 6), "u": f(4, 6), "w": f(6, b=1.0), "wn": f(6, b=1.0)}


@pytest.mark.parametrize("inside", [(N, S, BW), (S, BW), (BW,)])
@pytest.mark.parametrize("graphs", [True, False])
def test_norms_of_a_forward_outside_the_loop(inside, graphs):
    outside = [n for n in (Y, N, S) if n not in inside]
    agree(norms(*outside, _loop(*inside, *_sgd("w", "wn"))), norm_feeds(), ("s", "w", "wn"), use_graphs=graphs)


def head_feeds(rows=(4, 4), seed=1):
    rng = np.random.default_rng(seed)
    d = {"W": rng.standard_normal((5, 7)).astype(np.float32), "b": rng.standard_normal(7).astype(np.float32)}
    for i, r in enumerate(rows):
        d[f"x{i}"] = rng.standard_normal((r, 5)).astype(np.float32)
        d[f"t{i}"] = rng.integers(0, 7, r).astype(np.float32)
        if r > 3:
            d[f"t{i}"][2] = -100
    return d


def ce_agree(ast, feeds, fetch, **kw):
    env = {"ce": {"shape": ()}}
    P = tl.Program(ast, env, feeds=feeds, fetch=list(fetch), **kw)
    got = P.run()
    shapes = {k: {"shape": v} for k, v in P.shapes.items()}
    P.free()
    ref = OracleProgram(ast, shapes, dtype=np.float64, feeds=feeds).run()
    for k in fetch:
        assert_close(got[k], ref[k], 1e-4, k)


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("rows", [(4, 4), (40, 40)])
def test_a_head_whose_forward_is_outside_the_loop(graphs, rows):
    ce_agree(head(loss(), _loop(CE_BW, *_sgd2("W")), rows=rows), head_feeds(rows), ("ce", "W"), use_graphs=graphs)


def test_a_head_updated_before_a_top_level_backward():
    step = [L("W_new", C("mult", "W", "lr")), {"type": "rebind", "name": "W", "expr": {"type": "name", "name": "W_new"}}]
    ce_agree(head(loss(), _loop(*step), CE_BW), head_feeds(), ("ce", "W", "W_grad"))


@pytest.mark.parametrize("rows", [(200, 4), (4, 200)])
def test_a_longer_batch_under_the_same_loss_name(rows):
    """A loss of one batch before the loop, of another in it (the gradient is
    taken of both, as the names say)."""
    ce_agree(head(loss(0), _loop(loss(1), CE_BW, *_sgd2("W")), rows=rows), head_feeds(rows), ("ce", "W"))


def test_a_norm_under_the_name_of_what_it_norms():
    agree(norms(Y, L("y", {"type": "scaled_norm", "args": ["y", "wn"]})), norm_feeds(), ("y",))
