"""tl_linear_ce and its gradients against the definition in float64.

Tolerances, with S = |x| |W| (the magnitudes a logit sums): a product's terms
are exact (bf16) or miss less than 3 * 2^-24 of themselves (float32 as three
bf16 terms, six products); the tensor core's accumulator drops up to 2^-23 of
the running sum at each of the additions of full-size terms in a chunk of K
(1024 / 16 = 64 bf16, 256 / 16 = 16 float32), and chunks add in float32:
  e = 1.2e-5 (bf16) or 4e-6 (float32) of the magnitudes summed, for logits and
  for the gradients' products.
A logit off by d changes p by the factor 1 + d, lse by at most d; exp, log and
the sums of exponentials add 4e-6.  g is held as bf16 for bf16 operands (half a
step of each element, p - 1 at the target included), as three terms for float32.  Outputs in bf16 add half a step of their own.
"""
import numpy as np
import pytest

from conftest import REPO  # noqa: F401
from lm_util import BF16_STEP, CODE, Dev, rounded, rt
from oracle import lm_ops

pytestmark = pytest.mark.gpu

IDX = {"f32": (rt.IDX_F32, np.float32), "i32": (rt.IDX_I32, np.int32), "i64": (rt.IDX_I64, np.int64)}
GRADS = ("dx", "dw", "dbias")


def inputs(rows, classes, width, dtype, bias=True, seed=0, ignored=True):
    rng = np.random.default_rng(seed + 101 * rows + classes + width)
    x = rounded(rng.standard_normal((rows, width)), dtype)
    w = rounded(rng.standard_normal((width, classes)) * 1.5 / np.sqrt(width), dtype)
    b = rounded(rng.standard_normal(classes) * 0.5, "f32") if bias else None
    t = rng.integers(0, classes, rows)
    if ignored and rows > 4:
        t[rng.integers(0, rows, max(1, rows // 20))] = -100
    return x, w, b, t


def run(x, w, b, t, dtype, trans=0, idx="i64", divisor=0.0, up=None, pad=0, lead=0, want=GRADS, start=None,
        calls=1, fwd=("loss", "row_loss", "lse")):
    rows, width = x.shape
    classes = w.shape[1]
    code, ity = IDX[idx]
    with Dev() as D:
        L = rt.lib()
        px, ldx = D.rows(x, dtype, width + pad, lead)
        wm = w.T if trans else w
        pw, ldw = D.rows(wm, dtype, wm.shape[1] + pad, lead)
        pb = D.put(b, "f32")
        pt = D.put(t.astype(ity))
        nb = L.tl_linear_ce_scratch_bytes(CODE[dtype], trans, rows, classes, width, 1)
        scratch = D.zeros(nb)
        o = {k: D.new(1 if k == "loss" else rows) for k in set(fwd) | {"lse"}}
        out = {}
        base = (CODE[dtype], trans, rows, classes, width, px, ldx, pw, ldw, pb, pt, code, divisor)
        pu = None if up is None else D.put(np.float32([up]))
        start = start or {}
        acc = sum({"dx": rt.ACC_DX, "dw": rt.ACC_DW, "dbias": rt.ACC_DBIAS}[k] for k in start)
        g = {}
        if "dx" in want:
            g["dx"] = D.rows(start.get("dx", np.full(x.shape, 7.0)), dtype, ldx, lead)[0]
        if "dw" in want:
            s = start.get("dw", np.full(w.shape, 7.0))
            g["dw"] = D.rows(s.T if trans else s, dtype, ldw, lead)[0]
        if "dbias" in want and b is not None:
            g["dbias"] = D.put(start.get("dbias", np.full(classes, 7.0)), "f32")
        for _ in range(calls):
            rt.check(L.tl_linear_ce(*base, o.get("loss"), o.get("row_loss"), o["lse"], scratch, nb, D.stream),
                     "forward")
            if g:
                rt.check(L.tl_linear_ce_backward(*base, o["lse"], pu, g.get("dx"), ldx, g.get("dw"), ldw,
                                                 g.get("dbias"), acc, scratch, nb, D.stream), "backward")
        for k, p in o.items():
            out[k] = D.get(p, (1,) if k == "loss" else (rows,))
        if "dx" in g:
            out["dx"], rest = D.get_rows(g["dx"], rows, width, ldx, dtype, lead)
            assert np.all(rest == 7.0), "dx: written between rows"
        if "dw" in g:
            m, rest = D.get_rows(g["dw"], *wm.shape, ldw, dtype, lead)
            out["dw"] = m.T if trans else m
            assert np.all(rest == 7.0), "dw: written between rows"
        if "dbias" in g:
            out["dbias"] = D.get(g["dbias"], (classes,))
        code = np.zeros(1, np.int32)
        rt.check(L.tl_device_error(code.ctypes.data_as(__import__("ctypes").POINTER(rt.c_int)), 1))
        assert code[0] == 0, "a bounded wait gave up"
    return out


def within(got, ref, tol, name):
    got = np.asarray(got, np.float64)
    assert got.shape == ref.shape, name
    fin = np.isfinite(ref)
    np.testing.assert_array_equal(got[~fin], ref[~fin], err_msg=name)
    tol = np.broadcast_to(tol, ref.shape)
    bad = fin & ~(np.abs(got - ref) <= tol)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - ref) / tol, -1)), ref.shape)
        raise AssertionError(f"{name}: {int(bad.sum())} of {ref.size} off; worst at {i}: got {got[i]!r}, "
                             f"want {ref[i]!r}, allowed {tol[i]:.3g}")


def compare(out, x, w, b, t, dtype, divisor=0.0, up=1.0, start=None):
    ref = lm_ops.linear_ce(x, w, t, b, divisor, up)
    e, half = (1.2e-5, BF16_STEP) if dtype == "bf16" else (4e-6, 0.0)
    ax, aw = np.abs(x), np.abs(w)
    size = ax @ aw + (0.0 if b is None else np.where(np.isfinite(b), np.abs(b), 0.0))
    ez = e * size.max(axis=1) + 4e-6          # of a logit, and so of lse
    lse = np.where(np.isfinite(ref["lse"]), np.abs(ref["lse"]), 0.0)
    ez = ez + 2.0 ** -23 * lse                # lse is stored in float32
    if "lse" in out:
        within(out["lse"], ref["lse"], ez, "lse")
    if "row_loss" in out:
        within(out["row_loss"], ref["row_loss"], 2 * ez + 2.0 ** -23 * lse, "row_loss")
    if "loss" in out:
        within(out["loss"], np.array([ref["loss"]]), 2 * ez.mean() + 1e-6 * np.abs(lse).mean() + 1e-6, "loss")
    g = np.abs(ref["g"])
    ok = (t >= 0) & (t < w.shape[1])
    div = divisor if divisor > 0 else max(1, int(ok.sum()))
    p = g.copy()
    r = np.nonzero(ok)[0]
    p[r, t[r]] = np.abs(ref["g"][r, t[r]] + up / div)
    eg = p * (2 * ez + 4e-6)[:, None]                          # g before it is rounded
    eg8 = eg + half * g
    start = start or {}

    def grad(name, err, size):
        want = ref[name] + start.get(name, 0.0)
        tol = err + e * size + 2e-6 * (np.abs(ref[name]) + np.abs(start.get(name, 0.0)))
        if dtype == "bf16" and name != "dbias":
            tol = tol + half * (np.abs(want) + tol)
        within(out[name], want, tol + 1e-30, name)

    if "dx" in out:
        grad("dx", eg8 @ aw.T, g @ aw.T)
    if "dw" in out:
        grad("dw", ax.T @ eg8, ax.T @ g)
    if "dbias" in out:
        grad("dbias", eg.sum(axis=0), g.sum(axis=0))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("rows,classes,width", [
    (1, 1, 1), (1, 2, 3), (3, 17, 5), (5, 300, 64), (130, 257, 65), (257, 1000, 72), (300, 515, 200),
    (64, 20011, 100), (520, 3001, 1000), (1, 16384, 256), (1025, 2048, 1288), (2000, 40, 333)])
def test_sizes(dtype, trans, rows, classes, width):
    a = inputs(rows, classes, width, dtype)
    compare(run(*a, dtype, trans), *a, dtype)


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("rows", [1, 2, 4, 7, 8, 11, 16, 17])
def test_few_rows_of_float32(rows, pad, trans):
    """Up to 16 rows the float32 units read W as it is; odd leading dimensions,
    sizes that cut every block, gradients that are added to."""
    x, w, b, t = a = inputs(rows, 2111, 780, "f32", seed=11, ignored=False)
    if rows > 2:
        t[1] = -100
    rng = np.random.default_rng(rows)
    start = {"dx": rounded(rng.standard_normal(x.shape) * 0.01, "f32"),
             "dw": rounded(rng.standard_normal(w.shape) * 0.01, "f32"),
             "dbias": rounded(rng.standard_normal(b.shape) * 0.01, "f32")}
    compare(run(*a, "f32", trans, pad=pad, calls=1, start=start), *a, "f32", start=start)
    compare(run(*a, "f32", trans, pad=pad, calls=2, divisor=3.0, up=0.5), *a, "f32", 3.0, 0.5)
    compare(run(x, w, None, t, "f32", trans), x, w, None, t, "f32")
    if rows > 2:
        clean, bad = x.copy(), x.copy()
        clean[1], bad[1] = 0.0, np.nan
        out = run(bad, w, b, t, "f32", trans)
        out.pop("lse")
        compare(out, clean, w, b, t, "f32")


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("rows,classes,width", [(2, 100003, 3), (3, 2, 5003), (16, 40000, 513), (5, 1, 1)])
def test_few_rows_of_long_and_short_axes(rows, classes, width, trans):
    a = inputs(rows, classes, width, "f32", seed=12, ignored=False)
    compare(run(*a, "f32", trans), *a, "f32")
    p, q = run(*a, "f32", trans), run(*a, "f32", trans)
    for k in p:
        np.testing.assert_array_equal(p[k], q[k])


def test_few_rows_with_masked_classes():
    x, w, b, t = inputs(8, 300, 64, "f32", seed=13, ignored=False)
    b[100:200] = -np.inf
    b[250:] = np.finfo(np.float32).min
    t[:] = np.arange(8)
    t[3] = 150                              # a masked target: loss +inf
    with np.errstate(invalid="ignore"):
        out, ref = run(x, w, b, t, "f32"), lm_ops.linear_ce(x, w, t, b)
    assert np.isposinf(out["row_loss"][3]) and np.isposinf(out["loss"][0])
    good = np.arange(8) != 3
    within(out["row_loss"][good], ref["row_loss"][good], 1e-3, "row_loss")
    compare({k: out[k] for k in ("lse", "dx", "dw", "dbias")}, x, w, b, t, "f32")
    out = run(x, w, np.full(300, -np.inf), t, "f32")
    assert np.isneginf(out["lse"]).all() and np.isposinf(out["loss"][0])
    assert np.isfinite(out["dx"]).all() and np.isfinite(out["dw"]).all()
    out = run(x, w, None, np.full(8, -100), "f32")
    assert out["loss"][0] == 0 and not out["row_loss"].any() and not out["dx"].any() and not out["dw"].any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,lead", [(8, 0), (3, 0), (0, 1), (5, 3)])
@pytest.mark.parametrize("trans", [0, 1])
def test_strides_and_offsets(dtype, pad, lead, trans):
    a = inputs(70, 392, 136, dtype, seed=1)
    compare(run(*a, dtype, trans, pad=pad, lead=lead), *a, dtype)


@pytest.mark.parametrize("idx", ["f32", "i32", "i64"])
@pytest.mark.parametrize("divisor,up", [(0.0, None), (0.0, 0.25), (512.0, 2.0)])
def test_targets_and_scales(idx, divisor, up):
    a = inputs(90, 700, 96, "bf16", seed=2)
    a[3][:3] = [700, -1, 2 ** 24 + 1]      # out of range; the last also as a float
    compare(run(*a, "bf16", 1, idx=idx, divisor=divisor, up=up), *a, "bf16", divisor, up or 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_parts_and_accumulate(dtype):
    a = inputs(150, 600, 100, dtype, seed=3)
    x, w, b, t = a
    for want in (("dx",), ("dw",), ("dbias",), ()):
        compare(run(*a, dtype, want=want), *a, dtype)
    out = run(*a, dtype, want=(), fwd=("loss",))
    compare({"loss": out["loss"]}, *a, dtype)
    rng = np.random.default_rng(5)
    for trans in (0, 1):
        start = {"dx": rounded(rng.standard_normal(x.shape) * 0.01, dtype),
                 "dw": rounded(rng.standard_normal(w.shape) * 0.01, dtype),
                 "dbias": rounded(rng.standard_normal(b.shape) * 0.01, "f32")}
        compare(run(*a, dtype, trans, start=start), *a, dtype, start=start)
    compare(run(*a, dtype, calls=3), *a, dtype)


def test_masked_classes_and_rows_without_target():
    """bias -inf and the type's lowest value mask classes; a row may lose every
    class, its target, or all rows their targets."""
    x, w, b, t = inputs(40, 300, 64, "f32", seed=4, ignored=False)
    b[100:200] = -np.inf
    b[250:] = np.finfo(np.float32).min
    t[:] = np.arange(40)
    t[3] = 150                              # a masked target: loss +inf
    with np.errstate(invalid="ignore"):
        out, ref = run(x, w, b, t, "f32"), lm_ops.linear_ce(x, w, t, b)
    assert np.isposinf(out["row_loss"][3]) and np.isposinf(out["loss"][0])
    good = np.arange(40) != 3
    within(out["row_loss"][good], ref["row_loss"][good], 1e-3, "row_loss")
    compare({k: out[k] for k in ("lse", "dx", "dw", "dbias")}, x, w, b, t, "f32")
    everything = np.full(300, -np.inf)
    out = run(x, w, everything, t, "f32")
    assert np.isneginf(out["lse"]).all() and np.isposinf(out["loss"][0])
    assert np.isfinite(out["dx"]).all() and np.isfinite(out["dw"]).all()
    none = np.full(40, -100)
    out = run(x, w, None, none, "f32")
    assert out["loss"][0] == 0 and not out["row_loss"].any() and not out["dx"].any() and not out["dw"].any()


def test_nan_rows_stay_their_own():
    x, w, b, t = inputs(20, 500, 64, "bf16", seed=6, ignored=False)
    x[7, 3] = np.nan
    out = run(x, w, b, t, "bf16", divisor=20.0)
    keep = np.arange(20) != 7
    ref = lm_ops.linear_ce(x[keep], w, t[keep], b, 20.0)
    assert np.isnan(out["row_loss"][7]) and np.isnan(out["dx"][7]).all()
    within(out["row_loss"][keep], ref["row_loss"], 1e-3, "row_loss")
    assert np.isfinite(out["dx"][keep]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,trans", [(20, 0), (300, 1)])
def test_padded_rows_may_hold_anything(dtype, rows, trans):
    """Rows without a target hold NaN and infinities: nothing of them reaches
    the loss or the gradients."""
    x, w, b, t = inputs(rows, 500, 72, dtype, seed=9)
    t[[2, rows - 1]], t[5:9] = -100, 500
    clean = x.copy()
    pad = (t < 0) | (t >= 500)
    clean[pad] = 0.0
    x[pad] = np.nan
    x[2] = np.inf
    out = run(x, w, b, t, dtype, trans)
    out.pop("lse")
    assert not out["row_loss"][pad].any() and not out["dx"][pad].any()
    compare(out, clean, w, b, t, dtype)


def test_pieces_of_the_vocabulary():
    """A width whose weights' terms make the vocabulary two pieces, in both
    directions (512 MB of terms: 10752 classes of 8192 floats)."""
    a = inputs(5, 11800, 8192, "f32", seed=7)
    compare(run(*a, "f32", 1), *a, "f32")


def test_many_rows():
    """More rows than 2^16, the last tile cut.  dW sums 274 chunks of K (256 rows
    each) in float32: 274 * 2^-24 = 1.7e-5 of the magnitudes, beside a chunk's own."""
    x, w, b, t = a = inputs(70001, 130, 24, "f32", seed=10)
    out = run(*a, "f32")
    dw = out.pop("dw")
    compare(out, *a, "f32")
    ref = lm_ops.linear_ce(x, w, t, b)
    ez = 4e-6 * (np.abs(x) @ np.abs(w) + np.abs(b)).max() + 4e-6 + 2.0 ** -23 * np.abs(ref["lse"]).max()
    g = np.abs(ref["g"])
    r = np.nonzero(t >= 0)[0]
    p = g.copy()
    p[r, t[r]] = np.abs(ref["g"][r, t[r]] + 1.0 / len(r))
    ax = np.abs(x).T
    within(dw, ref["dw"], ax @ (p * (2 * ez + 4e-6)) + (4e-6 + 1.7e-5) * (ax @ g) + 2e-6 * np.abs(ref["dw"]), "dw")


def test_two_runs_agree():
    a = inputs(700, 2500, 520, "bf16", seed=8)
    p, q = run(*a, "bf16", 1), run(*a, "bf16", 1)
    for k in p:
        np.testing.assert_array_equal(p[k], q[k])


def test_no_rows():
    with Dev() as D:
        L = rt.lib()
        nb = L.tl_linear_ce_scratch_bytes(0, 0, 0, 12, 8, 1)
        s, w, loss = D.zeros(nb), D.new(96), D.new(1)
        dw, db = D.new(8 * 13, fill=7.0), D.new(12)
        rt.check(L.tl_linear_ce(0, 0, 0, 12, 8, None, 8, w, 12, None, None, 2, 0.0, loss, None, None, s, nb,
                                D.stream))
        rt.check(L.tl_linear_ce_backward(0, 0, 0, 12, 8, None, 8, w, 12, None, None, 2, 0.0, None, None,
                                         None, 8, dw, 13, db, 0, s, nb, D.stream))
        assert D.get(loss, (1,))[0] == 0
        m, rest = D.get_rows(dw, 8, 12, 13, "f32")
        assert not m.any() and np.all(rest == 7.0) and not D.get(db, (12,)).any()


# -- more than one piece of the vocabulary ------------------------------------
# 512 MB of scratch for the terms of W, for g and for the forward's partials cut
# the vocabulary (make_plan in linear_ce.cu); each test says where its cut is.

@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("rows", [17, 140])
def test_pieces_of_float32_weights(rows, trans):
    """10752 classes of 3 x 8192 terms a piece, both directions: the running
    join, gradients added to, a last piece shorter than the first, for tiles of
    one CTA and of two."""
    x, w, b, t = a = inputs(rows, 11800, 8192, "f32", seed=20)
    t[:3] = [10751, 10752, 11799]  # the classes around the cut, and the last
    rng = np.random.default_rng(rows)
    start = {"dx": rounded(rng.standard_normal(x.shape) * 0.01, "f32"),
             "dw": rounded(rng.standard_normal(w.shape) * 0.01, "f32"),
             "dbias": rounded(rng.standard_normal(b.shape) * 0.01, "f32")} if rows == 17 else None
    compare(run(*a, "f32", trans, start=start), *a, "f32", start=start)


@pytest.mark.parametrize("trans", [0, 1])
def test_pieces_of_copied_bf16_weights(trans):
    """Rows that TMA cannot address are copied: 32768 classes of 8192 a piece."""
    rng = np.random.default_rng(21)
    rows, classes, width = 20, 33000, 8192
    x = rounded(rng.standard_normal((rows, width)), "bf16")
    w = np.tile(rounded(rng.standard_normal((width, 997)) * 1.5 / np.sqrt(width), "bf16"), (1, 34))[:, :classes]
    b = rounded(rng.standard_normal(classes) * 0.5, "f32")  # tells equal columns apart
    t = rng.integers(0, classes, rows)
    t[:4] = [32767, 32768, classes - 1, -100]
    compare(run(x, w, b, t, "bf16", trans, pad=3), x, w, b, t, "bf16")


def repeated(rows, classes, width, dtype, seed, distinct=509):
    """A batch whose rows repeat `distinct` ones (the definition is computed for
    those): (x, w, b, t of them, which row is which)."""
    x, w, b, t = inputs(distinct, classes, width, dtype, seed=seed)
    t[:3] = [0, classes - 1, -100]
    return x, w, b, t, np.arange(rows) % distinct


@pytest.mark.parametrize("trans", [0, 1])
def test_pieces_of_many_rows(trans):
    """1024 classes of g for 2^18 rows a piece, and 1024 tiles of rows in 128 bands.

    dW adds 256 chunks of K (1024 rows each) in float32, 256 * 2^-24 = 1.6e-5 of
    the magnitudes beside a chunk's own; dbias adds 8192 groups of 32 rows in eight
    chains, 1024 * 2^-24 = 6.2e-5 beside a group's."""
    rows = 1 << 18
    x, w, b, t, which = repeated(rows, 1100, 40, "bf16", 22)
    n = np.bincount(which, minlength=len(t)).astype(np.float64)
    ok = t >= 0
    div = float(n[ok].sum())
    out = run(x[which], w, b, t[which], "bf16", trans)
    for k in ("lse", "row_loss", "dx"):  # equal rows, equal results
        np.testing.assert_array_equal(out[k], out[k][which], err_msg=k)
    compare({k: out[k][:len(t)] for k in ("lse", "row_loss", "dx")}, x, w, b, t, "bf16", divisor=div)
    ref = lm_ops.linear_ce(x, w, t, b, divisor=div)
    e = 1.2e-5
    size = (np.abs(x) @ np.abs(w) + np.abs(b)).max(axis=1)
    ez = e * size + 4e-6 + 2.0 ** -23 * np.abs(ref["lse"])
    within(out["loss"], np.array([(ref["row_loss"] * n).sum()]) / div,
           2 * ez.max() + 1e-6 * np.abs(ref["lse"]).mean() + 1e-6, "loss")
    g = np.abs(ref["g"]) * n[:, None]
    p = g.copy()
    r = np.nonzero(ok)[0]
    p[r, t[r]] = np.abs(ref["g"][r, t[r]] + 1.0 / div) * n[r]
    eg = p * (2 * ez + 4e-6)[:, None]
    ax = np.abs(x).T
    want = x.T @ (ref["g"] * n[:, None])
    tol = ax @ (eg + BF16_STEP * g) + (e + 1.6e-5) * (ax @ g) + 2e-6 * np.abs(want)
    within(out["dw"], want, tol + BF16_STEP * (np.abs(want) + tol), "dw")
    within(out["dbias"], (ref["g"] * n[:, None]).sum(axis=0), eg.sum(axis=0) + (e + 6.2e-5) * g.sum(axis=0), "dbias")


def test_pieces_of_a_forward_of_many_rows():
    """8192 classes of partials for 2^20 rows a piece; the second has eight classes.
    The mean of 2^20 losses is taken in float64."""
    rows = 1 << 20
    x, w, b, t, which = repeated(rows, 8200, 16, "bf16", 23)
    t[3:5] = [8191, 8192]
    n = np.bincount(which, minlength=len(t)).astype(np.float64)
    out = run(x[which], w, b, t[which], "bf16", 1, want=())
    for k in ("lse", "row_loss"):
        np.testing.assert_array_equal(out[k], out[k][which], err_msg=k)
    loss = out.pop("loss")
    compare({k: out[k][:len(t)] for k in ("lse", "row_loss")}, x, w, b, t, "bf16")
    ref = lm_ops.linear_ce(x, w, t, b)
    tol = 2 * (1.2e-5 * (np.abs(x) @ np.abs(w) + np.abs(b)).max() + 4e-6) + 3e-7 * np.abs(ref["lse"]).max()
    within(loss, np.array([(ref["row_loss"] * n).sum() / n[t >= 0].sum()]), tol, "loss")


# -- masks, for every kind of tile and type ------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("rows", [8, 40, 300])
def test_masked_classes_in_whole_blocks(rows, trans, dtype):
    """Whole blocks of 128 classes of bias -inf (their maximum is -inf), others of
    the type's lowest value; a masked target; every class masked; no targets.  A
    class of the lowest value is one of -inf beside ordinary ones."""
    low = float(np.finfo(np.float32).min)
    x, w, b, t = inputs(rows, 1000, 72, dtype, seed=24, ignored=False)
    b[100:520], b[900:] = -np.inf, -np.inf
    t[:] = np.arange(rows) % 100
    t[1], t[2] = 899, 520
    masked = b.copy()
    masked[640:800] = -np.inf
    b[640:800] = low
    compare(run(x, w, b, t, dtype, trans), x, w, masked, t, dtype)
    t[3], t[4] = 300, 700  # masked targets: their losses are +inf and lowest's own
    with np.errstate(invalid="ignore"):
        out, ref = run(x, w, b, t, dtype, trans), lm_ops.linear_ce(x, w, t, masked)
    assert np.isposinf(out["row_loss"][3]) and out["row_loss"][4] > 1e38 and np.isposinf(out["loss"][0])
    good = (np.arange(rows) != 3) & (np.arange(rows) != 4)
    ez = (1.2e-5 if dtype == "bf16" else 4e-6) * (np.abs(x) @ np.abs(w) + 3.0).max() + 1e-5
    within(out["row_loss"][good], ref["row_loss"][good], 2 * ez, "row_loss")
    compare({k: out[k] for k in ("lse", "dx", "dw", "dbias")}, x, w, masked, t, dtype)
    out = run(x, w, np.full(1000, -np.inf), t, dtype, trans)
    assert np.isneginf(out["lse"]).all() and np.isposinf(out["loss"][0])
    # nothing left: g = -onehot / rows
    g = np.zeros((rows, 1000))
    g[np.arange(rows), t] = -1.0 / rows
    step = 2 * BF16_STEP if dtype == "bf16" else 0.0
    for k, want, mag in (("dx", g @ w.T, np.abs(g) @ np.abs(w).T), ("dw", x.T @ g, np.abs(x).T @ np.abs(g)),
                         ("dbias", g.sum(axis=0), np.abs(g).sum(axis=0))):
        within(out[k], want, (1.3e-5 + step) * mag + step * np.abs(want), k)
    out = run(x, w, b, np.full(rows, -100), dtype, trans)
    assert out["loss"][0] == 0 and not out["row_loss"].any()
    assert not out["dx"].any() and not out["dw"].any() and not out["dbias"].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nan_rows_stay_their_own_in_tiles_of_two_ctas(dtype):
    x, w, b, t = inputs(300, 500, 64, dtype, seed=25, ignored=False)
    x[7, 3], x[200, 0] = np.nan, np.nan
    out = run(x, w, b, t, dtype, divisor=300.0)
    keep = np.ones(300, bool)
    keep[[7, 200]] = False
    assert np.isnan(out["row_loss"][~keep]).all() and np.isnan(out["dx"][~keep]).all()
    compare({k: out[k][keep] for k in ("lse", "row_loss", "dx")}, x[keep], w, b, t[keep], dtype, divisor=300.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_more_than_one_band_of_row_tiles(dtype):
    """Tiles go in bands of 2048 rows: two whole ones and a cut one."""
    a = inputs(4700, 1300, 200, dtype, seed=26)
    compare(run(*a, dtype, 1), *a, dtype)
    compare(run(*a, dtype, 0, pad=8), *a, dtype)
