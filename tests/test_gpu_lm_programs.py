"""Programs of the language-model operators whose forward, backward and updates
stand in different places, against the float64 oracle.

Tolerance rel 1e-4 of the value and of the tensor's largest, the suite's for
training.
"""
import numpy as np
import pytest

from conftest import assert_close, load_backend
from oracle import OracleProgram
from test_lm_programs_cpu import BW, N, S, Y, _loop, _sgd, norms

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
