"""The language-model operators together, as a program uses them: a training
loop over a block boundary, the head and both losses (programs.lm_head_train)
against the float64 oracle, as a captured graph and kernel by kernel.

Tolerance rel 1e-4 of the value and of the tensor's largest, the suite's for
training: the products run under the GEMM's BF16X3 scheme.
"""
import ctypes

import numpy as np
import pytest

from conftest import assert_close, load_backend
from lm_util import Dev, rt
from oracle import OracleProgram, lm_ops

pytestmark = pytest.mark.gpu
tl = load_backend()

FETCH = ["loss", "ce", "kd", "Wb", "bb", "wp", "g", "wn", "Wv", "bv"]


def both(cfg, gate="channel", fetch=FETCH, **kw):
    ast = tl.programs.lm_head_train(**cfg, gate=gate, **kw)
    sizes = {k: cfg[k] for k in "BDVK"}
    feeds = tl.programs.lm_head_inputs(**sizes, gate=gate)
    P = tl.Program(ast, None, feeds=feeds, fetch=fetch)
    got = P.run()
    env = {k: {"shape": v} for k, v in P.shapes.items()}
    P.free()
    ref = OracleProgram(ast, env, dtype=np.float64, feeds=feeds).run()
    return got, ref


@pytest.mark.parametrize("norm,gate", [("rms", "channel"), ("layer", "full"), ("rms", "token")])
def test_training_loop_matches_the_oracle(norm, gate):
    got, ref = both(dict(B=256, D=128, V=1000, K=8, epochs=4), gate, norm=norm)
    for k in FETCH:
        assert_close(got[k], ref[k], 1e-4, k)


def test_odd_sizes_and_every_tensor():
    """Sizes that are no multiple of anything; everything kept (nothing fused away)."""
    got, ref = both(dict(B=37, D=61, V=131, K=5, epochs=2), fetch=None)
    for k in FETCH + ["y", "n", "y_grad", "n_grad", "z_grad", "u_grad"]:
        assert_close(got[k], ref[k], 1e-4, k)


def test_fused_and_unfused_programs_agree():
    cfg = dict(B=64, D=96, V=300, K=4)
    ast = tl.programs.lm_head_train(**cfg, epochs=3)
    feeds = tl.programs.lm_head_inputs(**cfg)
    out = []
    for kw in ({}, {"use_graphs": False}, {"fuse_ops": False}):
        P = tl.Program(ast, None, feeds=feeds, fetch=FETCH, **kw)
        out.append(P.run())
        P.free()
    for k in FETCH:
        np.testing.assert_array_equal(out[0][k], out[1][k], err_msg=f"{k}: graph and eager differ")
        assert_close(out[2][k], out[0][k].astype(np.float64), 1e-5, k)


def test_weighted_losses_and_repeated_operands():
    """A loss times a constant reaches the kernels as their upstream gradient; an
    operand used twice in one call gets both gradients."""
    L, F, C = tl.programs._let, tl.programs._fill, tl.programs._call
    B, D, V = 48, 40, 90
    rng = np.random.default_rng(0)
    feeds = {"x": rng.standard_normal((B, D)).astype(np.float32),
             "w": (1 + 0.1 * rng.standard_normal(D)).astype(np.float32),
             "W": (rng.standard_normal((D, V)) * 0.2).astype(np.float32),
             "b": np.zeros(V, np.float32), "t": rng.integers(0, V, B).astype(np.float32)}
    ast = [L("x", F((B, D)), (B, D), grad=True), L("w", F((D,)), (D,), grad=True),
           L("W", F((D, V)), (D, V), grad=True), L("b", F((V,)), (V,), grad=True), L("t", F((B,)), (B,)),
           L("c", tl.programs._lit([0.25], (1,)), (1,)),
           L("y", {"type": "residual_norm", "args": ["x", "x", "w", "w"], "norm": "layer", "alpha": 0.5}),
           L("n", {"type": "scaled_norm", "args": ["y", "w"], "norm": "layer"}),
           L("ce", dict(C("linear_cross_entropy", "n", "W", "b", "t"), divisor=100.0)),
           L("loss", C("mult", "ce", "c"), ()),
           {"type": "backward", "loss_tensor": "loss"}]
    env = {"loss": {"shape": ()}}
    P = tl.Program(ast, env, feeds=feeds, fetch=["loss", "x_grad", "w_grad", "W_grad", "b_grad"])
    got = P.run()
    P.free()
    x, w, W = (feeds[k].astype(np.float64) for k in ("x", "w", "W"))
    y, n = lm_ops.residual_norm(x, x, w, w, "channel", 0.5, w, "layer")
    r = lm_ops.linear_ce(n, W, feeds["t"].astype(int), divisor=100.0, upstream=0.25)
    g = lm_ops.residual_norm_vjp(x, None, r["dx"], x, w, w, "channel", 0.5, w, "layer")
    assert_close(got["loss"], np.asarray(r["loss"] * 0.25), 1e-5, "loss")
    for k, want in (("x", g["dx"] + g["du"]), ("w", g["dw_post"] + g["dgate"] + g["dw_pre"]),
                    ("W", r["dw"]), ("b", r["dbias"])):
        assert_close(got[f"{k}_grad"], want, 1e-5, k)


def test_other_streams_and_concurrent_graphs():
    """Two graphs of one call on two streams, each with its own scratch, replayed
    side by side; and the same call on a stream that is not the library's."""
    rng = np.random.default_rng(1)
    rows, classes, width = 300, 2000, 96
    x = rng.standard_normal((rows, width)).astype(np.float32)
    w = (rng.standard_normal((width, classes)) * 0.1).astype(np.float32)
    t = rng.integers(0, classes, rows).astype(np.int64)
    L = rt.lib()
    with Dev() as D:
        px, pw, pt = D.put(x, "f32"), D.put(w, "f32"), D.put(t)
        nb = L.tl_linear_ce_scratch_bytes(0, 0, rows, classes, width, 1)
        runs = []
        for _ in range(2):
            st = ctypes.c_void_p()
            rt.check(L.tl_stream_create(ctypes.byref(st)))
            o = {"loss": D.new(1), "lse": D.new(rows), "dx": D.new(x.size), "dw": D.new(w.size)}
            runs.append((st, o, D.zeros(nb)))
        D.dev.sync()

        def issue(st, o, scratch):
            a = (0, 0, rows, classes, width, px, width, pw, classes, None, pt, 2, 0.0)
            rt.check(L.tl_linear_ce(*a, o["loss"], None, o["lse"], scratch, nb, st))
            rt.check(L.tl_linear_ce_backward(*a, o["lse"], None, o["dx"], width, o["dw"], classes, None, 0,
                                             scratch, nb, st))
        graphs = []
        for r in runs:
            issue(*r)  # eager once, then captured
            rt.check(L.tl_graph_begin(r[0]))
            issue(*r)
            g = ctypes.c_void_p()
            rt.check(L.tl_graph_end(r[0], ctypes.byref(g)))
            graphs.append(g)
        for _ in range(5):
            for g, r in zip(graphs, runs):
                rt.check(L.tl_graph_launch(g, r[0]))
        for r in runs:
            rt.check(L.tl_stream_sync(r[0]))
        got = [{k: D.get(p, (n,)) for (k, p), n in zip(r[1].items(), (1, rows, x.size, w.size))} for r in runs]
        for g in graphs:
            rt.check(L.tl_graph_destroy(g))
        for r in runs:
            rt.check(L.tl_stream_destroy(r[0]))
    ref = lm_ops.linear_ce(x.astype(np.float64), w.astype(np.float64), t)
    for o in got:
        for k in o:
            np.testing.assert_array_equal(o[k], got[0][k])
            assert_close(o[k], np.asarray(ref[k]).ravel(), 1e-5, k)
