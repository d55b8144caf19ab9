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
from lm_util import BF16_STEP, Dev, bf16_bits, close, rounded, rt
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


def _captured(D, calls):
    """Each (issue, stream) eagerly once, then as a graph; five replays side by side."""
    L, graphs = rt.lib(), []
    for issue, st in calls:
        issue()
        rt.check(L.tl_graph_begin(st))
        issue()
        g = ctypes.c_void_p()
        rt.check(L.tl_graph_end(st, ctypes.byref(g)))
        graphs.append(g)
    for _ in range(5):
        for g, (_, st) in zip(graphs, calls):
            rt.check(L.tl_graph_launch(g, st))
    for g, (_, st) in zip(graphs, calls):
        rt.check(L.tl_stream_sync(st))
        rt.check(L.tl_graph_destroy(g))


@pytest.mark.parametrize("rows", [5, 130])  # the one-launch form, and the three kernels
def test_concurrent_graphs_of_distillation_and_norms(rows):
    rng = np.random.default_rng(2)
    classes, top, cols = 5000, 12, 200
    z = rng.standard_normal((rows, classes)).astype(np.float32)
    t = rng.standard_normal((rows, top)).astype(np.float32)
    i = rng.integers(0, classes, (rows, top))
    i[0] = -1
    x, u, dy = (rng.standard_normal((rows, cols)).astype(np.float32) for _ in range(3))
    w = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)
    L = rt.lib()
    with Dev() as D:
        pz, pt, pi = D.put(z), D.put(t), D.put(i)
        px, pu, pdy, pw = D.put(x), D.put(u), D.put(dy), D.put(w)
        nd, nn = L.tl_distill_topk_scratch_bytes(rows), L.tl_residual_norm_scratch_bytes(rows, cols)
        outs, calls = [], []
        for _ in range(2):
            st = ctypes.c_void_p()
            rt.check(L.tl_stream_create(ctypes.byref(st)))
            o = {"loss": D.new(1), "dz": D.new(z.size), "n": D.new(x.size), "dx": D.new(x.size),
                 "du": D.new(x.size), "dw": D.new(cols)}
            sd, sn = D.zeros(nd), D.zeros(nn)

            def issue(st=st, o=o, sd=sd, sn=sn):
                rt.check(L.tl_distill_topk(0, rows, classes, top, pz, classes, pt, top, pi, top, 2, 2.0, 0.0,
                                           None, o["loss"], None, None, o["dz"], classes, 0, sd, nd, st))
                a = (0, 1, rows, cols, px, cols, pu, cols, pw, pw, rt.GATE_CHANNEL, 0, 0.5, pw, 1e-5)
                rt.check(L.tl_residual_norm(*a, None, cols, o["n"], cols, st))
                rt.check(L.tl_residual_norm_backward(*a, None, cols, pdy, cols, o["dx"], cols, o["du"], cols,
                                                     None, 0, o["dw"], None, 0, sn, nn, st))
            outs.append(o)
            calls.append((issue, st))
        D.dev.sync()
        _captured(D, calls)
        got = [{k: D.get(o[k], (n,)) for k, n in (("loss", 1), ("dz", z.size), ("n", x.size), ("dx", x.size),
                                                  ("du", x.size), ("dw", cols))} for o in outs]
        for _, st in calls:
            rt.check(L.tl_stream_destroy(st))
    d = lm_ops.distill_topk(z.astype(np.float64), t.astype(np.float64), i, 2.0)
    x, u, dy, w = (a.astype(np.float64) for a in (x, u, dy, w))
    _, n = lm_ops.residual_norm(x, u, w, w, "channel", 0.5, w, "rms")
    g = lm_ops.residual_norm_vjp(x, None, dy, u, w, w, "channel", 0.5, w, "rms")
    want = {"loss": np.array([d["loss"]]), "dz": d["dz"], "n": n, "dx": g["dx"], "du": g["du"],
            "dw": g["dw_post"]}
    for o in got:
        for k in o:
            np.testing.assert_array_equal(o[k], got[0][k])
            assert_close(o[k], np.asarray(want[k]).ravel(), 1e-5, k)


def test_offsets_past_32_bits():
    """Three rows 1.1e9 elements apart in every matrix: the last begins past 2^31
    elements and 2^32 bytes."""
    ld, n, cols = 1_100_000_000, 3, 40
    rng = np.random.default_rng(3)
    L = rt.lib()
    with Dev() as D:
        def far(a=None):
            p = D.raw((2 * ld + cols) * 2)
            for r in range(n):
                row = np.zeros(cols) if a is None else a[r]
                D.bytes_to(p + r * ld * 2, bf16_bits(row))
            return p

        def back(p):
            return np.stack([D.get(p + r * ld * 2, (cols,), "bf16") for r in range(n)])

        def near(a):
            return D.put(a, "bf16")
        m = [rounded(rng.standard_normal((n, cols)), "bf16") for _ in range(4)]
        x, u, dy, dn = m
        px, pu, po, pq = far(x), far(u), far(), far()
        # a norm and its gradients, the gate a matrix of the same stride
        pg = near(m[2])
        a = (1, 1, n, cols, px, ld, pu, ld, None, pg, rt.GATE_FULL, cols, 1.0, None, 1e-5)
        rt.check(L.tl_residual_norm(*a, po, ld, pq, ld, D.stream))
        y, nrm = lm_ops.residual_norm(x, u, None, m[2], "full", 1.0, None, "rms")
        close(back(po), y, "bf16", "y")
        close(back(pq), nrm, "bf16", "n")
        nb = L.tl_residual_norm_scratch_bytes(n, cols)
        pn = near(dn)
        rt.check(L.tl_residual_norm_backward(*a, None, cols, pn, cols, po, ld, pq, ld, None, cols, None, None,
                                             0, D.zeros(nb), nb, D.stream))
        g = lm_ops.residual_norm_vjp(x, None, dn, u, None, m[2], "full", 1.0, None, "rms")
        close(back(po), g["dx"], "bf16", "dx")
        close(back(pq), g["du"], "bf16", "du")
        # distillation: logits and gradient
        t, i = rounded(rng.standard_normal((n, 4)), "bf16"), rng.integers(0, cols, (n, 4))
        nb = L.tl_distill_topk_scratch_bytes(n)
        rt.check(L.tl_distill_topk(1, n, cols, 4, px, ld, near(t), 4, D.put(i), 4, 2, 1.0, 0.0, None, None,
                                   None, None, po, ld, 0, D.zeros(nb), nb, D.stream))
        close(back(po), lm_ops.distill_topk(x, t, i)["dz"], "bf16", "dz")
        # the head: three tokens, three classes; x and W (stored by class) both far apart
        tgt = np.array([0, 2, -100])
        nb = L.tl_linear_ce_scratch_bytes(1, 1, n, n, cols, 1)
        s, lse, loss = D.zeros(nb), D.new(n), D.new(1)
        b = (1, 1, n, n, cols, px, ld, pu, ld, None, D.put(tgt), 2, 0.0)
        rt.check(L.tl_linear_ce(*b, loss, None, lse, s, nb, D.stream))
        rt.check(L.tl_linear_ce_backward(*b, lse, None, po, ld, pq, ld, None, 0, s, nb, D.stream))
        r = lm_ops.linear_ce(x, u.T, tgt)
        close(D.get(loss, (1,)), [r["loss"]], "f32", "loss", scale=10.0)
        # g is bf16: half a step of each element more
        for p, want, size in ((po, r["dx"], np.abs(r["g"]) @ np.abs(u)),
                              (pq, r["dw"].T, np.abs(r["g"]).T @ np.abs(x))):
            close(back(p), want, "bf16", "gradient", rel=1e-5, scale=(BF16_STEP / 1e-5) * size)
