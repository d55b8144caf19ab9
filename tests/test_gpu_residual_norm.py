"""tl_residual_norm and its gradients against the definition in float64.

Tolerances: a row's sums are trees of at most 16 elements a thread, then 5 + 4
shuffle levels (relative error below 25 * 2^-24 = 1.5e-6 of the magnitudes), and
each output takes a handful of float32 operations after them: rel 1e-5 of the
value plus 1e-5 of the tensor's largest (the suite's tolerance for norms).
A gradient through a norm is a difference, r (g - hat mean(g hat)): with one or
two columns the terms cancel almost wholly, and so does u - mean where u is near
its mean; each gradient is held to 2e-5 of the magnitudes of its terms (two
norms deep, 1e-5 each).  Sums over rows add at most 60 terms in a chain here (rows / blocks + blocks / 8
+ 8): 60 * 2^-24 = 3.6e-6 of the sum of magnitudes besides.
bf16 adds its half step.
"""
import numpy as np
import pytest

from conftest import REPO  # noqa: F401  (puts the repository on sys.path)
from lm_util import CODE, Dev, close, rounded, rt
from oracle import lm_ops

pytestmark = pytest.mark.gpu

KIND = {"layer": rt.NORM_LAYER, "rms": rt.NORM_RMS}
GATE = {"none": 0, "channel": 1, "token": 2, "full": 3}


def inputs(rows, cols, gate_mode, dtype, seed=0, u=True, w_post=True, w_pre=True):
    rng = np.random.default_rng(seed + 7919 * rows + cols)
    f = lambda *s, a=1.0, b=0.0: rounded(rng.standard_normal(s) * a + b, dtype)  # noqa: E731
    d = {"x": f(rows, cols, a=2.0), "u": f(rows, cols, a=0.7, b=0.2) if u else None,
         "w_post": f(cols, a=0.2, b=1.0) if u and w_post else None,
         "w_pre": f(cols, a=0.2, b=1.0) if w_pre else None, "gate": None,
         "gate_mode": gate_mode, "alpha": 0.75}
    shape = {"channel": (cols,), "token": (rows,), "full": (rows, cols)}.get(gate_mode)
    if shape and u:
        d["gate"] = f(*shape, a=0.5)
    d["dy"], d["dn"] = f(rows, cols), f(rows, cols)
    return d


def run(d, dtype, kind, eps=1e-5, train=True, want=("y", "n"), pad=0, lead=0, dy=True, dn=True,
        acc=0, seed_out=None, in_place=False):
    """The two calls on fresh device arrays; outputs by name.  `pad` elements
    between rows and `lead` before the first; seed_out: what accumulated
    outputs start from."""
    rows, cols = d["x"].shape
    out = {}
    with Dev() as D:
        L = rt.lib()
        mat = lambda a: (None, cols) if a is None else D.rows(a, dtype, cols + pad, lead)  # noqa: E731
        vec = lambda a: D.put(a, dtype)  # noqa: E731
        x, ldx = mat(d["x"])
        u, ldu = mat(d["u"])
        full = d["gate_mode"] == "full" and d["gate"] is not None
        gate, ldg = mat(d["gate"]) if full else (vec(d["gate"]), cols)
        wa, wb = vec(d["w_post"]), vec(d["w_pre"])
        base = (CODE[dtype], KIND[kind], rows, cols, x, ldx, u, ldu, wa, gate, GATE[d["gate_mode"]],
                ldg, d["alpha"], wb, eps)
        ld = cols + pad

        def fresh(name, shape):
            start = np.full(shape, 7.0) if seed_out is None or name not in seed_out else seed_out[name]
            return D.rows(start, dtype, ld, lead)[0] if len(shape) == 2 else D.put(start, dtype)

        y = fresh("y", (rows, cols)) if "y" in want else None
        n = fresh("n", (rows, cols)) if "n" in want else None
        rt.check(L.tl_residual_norm(*base, y, ld, n, ld, D.stream), "forward")
        for name, p in (("y", y), ("n", n)):
            if p:
                out[name], rest = D.get_rows(p, rows, cols, ld, dtype, lead)
                assert np.all(rest == 7.0), f"{name}: written between rows"
        if not train:
            return out
        pdy, pdn = (mat(d["dy"])[0] if dy else None), (mat(d["dn"])[0] if dn else None)
        g = {"dx": pdy if in_place else fresh("dx", (rows, cols)), "dw_pre": fresh("dw_pre", (cols,))}
        if d["u"] is not None:
            g["du"] = pdn if in_place else fresh("du", (rows, cols))
            g["dw_post"] = fresh("dw_post", (cols,))
            if d["gate"] is not None:
                g["dgate"] = fresh("dgate", d["gate"].shape)
        nb = L.tl_residual_norm_scratch_bytes(rows, cols)
        rt.check(L.tl_residual_norm_backward(*base, pdy, ld, pdn, ld, g["dx"], ld, g.get("du"), ld,
                                             g.get("dgate"), ld, g.get("dw_post"), g["dw_pre"], acc,
                                             D.zeros(nb), nb, D.stream), "backward")
        for name, p in g.items():
            if name in ("dx", "du") or (name == "dgate" and full):
                out[name], rest = D.get_rows(p, rows, cols, ld, dtype, lead)
                assert np.all(rest == 7.0), f"{name}: written between rows"
            else:
                out[name] = D.get(p, d["gate"].shape if name == "dgate" else (cols,), dtype)
    return out


def compare(out, d, dtype, kind, eps=1e-5, dy=True, dn=True, add=None):
    f = {k: d[k] for k in ("u", "w_post", "gate", "gate_mode", "alpha", "w_pre")}
    y, n = lm_ops.residual_norm(d["x"], kind=kind, eps=eps, **f)
    ref = lm_ops.residual_norm_vjp(d["x"], d["dy"] if dy else None, d["dn"] if dn else None,
                                   kind=kind, eps=eps, **f)
    ref.update(y=y, n=n)
    for k, got in out.items():
        want = ref[k]
        scale = ref[k + "_abs"] if k + "_abs" in ref else None
        if add and k in add:  # the sum is rounded, and so is what it started from
            scale = (np.abs(want).max() if scale is None else scale) + np.abs(add[k])
            want = want + add[k]
        close(got, want, dtype, k, rel=2e-5 if k + "_abs" in ref else 1e-5, scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [
    (1, 1), (3, 2), (5, 7), (1, 64), (37, 33), (9, 127), (300, 256), (17, 260), (64, 1000),
    (701, 1021), (1, 4096), (33, 2048), (310, 4096), (2, 8192), (7, 8191), (3, 8200), (2, 20000)])
def test_sizes(dtype, rows, cols):
    """One element to rows longer than the register kernels hold; a training
    pass with every gradient, both norms."""
    for kind, mode in (("rms", "channel"), ("layer", "full")):
        d = inputs(rows, cols, mode, dtype)
        compare(run(d, dtype, kind), d, dtype, kind)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("mode", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("cols", [96, 515, 9001])
def test_gates(dtype, kind, mode, cols):
    d = inputs(41, cols, mode, dtype, seed=1)
    compare(run(d, dtype, kind), d, dtype, kind)


@pytest.mark.parametrize("cols", [512, 333, 8500])
def test_parts_left_out(cols):
    """No block, no weights, one output, one incoming gradient."""
    d = inputs(20, cols, "none", "f32", u=False)
    compare(run(d, "f32", "rms"), d, "f32", "rms")
    d = inputs(20, cols, "channel", "f32", w_post=False, w_pre=False)
    compare(run(d, "f32", "layer"), d, "f32", "layer")
    d = inputs(20, cols, "token", "f32", seed=3)
    for want in (("y",), ("n",)):
        compare(run(d, "f32", "rms", train=False, want=want), d, "f32", "rms")
    compare(run(d, "f32", "rms", dy=False), d, "f32", "rms", dy=False)
    compare(run(d, "f32", "rms", dn=False), d, "f32", "rms", dn=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,lead", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_strides_and_offsets(dtype, pad, lead):
    """Rows apart, rows that start at no 16-byte boundary; nothing between
    rows is written."""
    for cols in (256, 251):
        d = inputs(13, cols, "full", dtype, seed=5)
        compare(run(d, dtype, "layer", pad=pad, lead=lead), d, dtype, "layer")


@pytest.mark.parametrize("cols", [264, 129, 8300])
def test_accumulate_and_in_place(cols):
    for mode in ("channel", "token", "full"):
        d = inputs(23, cols, mode, "f32", seed=9)
        rng = np.random.default_rng(4)
        shape = {"dx": (23, cols), "du": (23, cols), "dw_post": (cols,), "dw_pre": (cols,),
                 "dgate": d["gate"].shape}
        start = {k: rounded(rng.standard_normal(s), "f32") for k, s in shape.items()}
        compare(run(d, "f32", "rms", acc=31, seed_out=start), d, "f32", "rms", add=start)
        compare(run(d, "f32", "rms", in_place=True), d, "f32", "rms")


def test_constant_and_non_finite_rows():
    """A row without variance (layer norm of a constant) is 0, not NaN; a row
    with a NaN or infinity touches no other row."""
    d = inputs(6, 320, "channel", "f32", seed=2)
    d["u"][1] = 3.0
    d["x"][1] = 0.0
    compare(run(d, "f32", "layer", train=False), d, "f32", "layer")
    d["u"][2, 5] = np.nan
    d["x"][4, 7] = np.inf
    with np.errstate(invalid="ignore"):
        out = run(d, "f32", "layer")
        ref = lm_ops.residual_norm(d["x"], kind="layer", u=d["u"], w_post=d["w_post"],
                                   gate=d["gate"], gate_mode="channel", alpha=0.75, w_pre=d["w_pre"])
    good = [0, 1, 3, 5]
    close(out["n"][good], ref[1][good], "f32", "n")
    for k in ("dx", "du"):
        assert np.isfinite(out[k][good]).all()
        assert np.isnan(out[k][2]).any() and np.isnan(out[k][4]).any()


def test_no_rows():
    with Dev() as D:
        L = rt.lib()
        nb = L.tl_residual_norm_scratch_bytes(0, 40)
        dw = D.new(40)
        x = D.new(40)
        rt.check(L.tl_residual_norm(0, 1, 0, 40, x, 40, None, 40, None, None, 0, 40, 1.0, None, 1e-5,
                                    x, 40, None, 40, D.stream))
        rt.check(L.tl_residual_norm_backward(0, 1, 0, 40, x, 40, None, 40, None, None, 0, 40, 1.0,
                                             None, 1e-5, None, 40, x, 40, None, 40, None, 40, None, 40,
                                             None, dw, 0, D.zeros(nb), nb, D.stream))
        np.testing.assert_array_equal(D.get(dw, (40,)), 0.0)


@pytest.mark.parametrize("mode", [rt.GATE_CHANNEL, rt.GATE_TOKEN, rt.GATE_FULL])
def test_no_rows_and_no_arrays_of_rows(mode):
    """Arrays without rows are null; the weights' gradients are zero, whatever the
    weights hold."""
    with Dev() as D:
        L = rt.lib()
        nb = L.tl_residual_norm_scratch_bytes(0, 40)
        o = [D.new(40) for _ in range(3)]
        w = D.put(np.full(40, np.inf), "f32")
        dgate = o[2] if mode == rt.GATE_CHANNEL else None
        args = (0, 1, 0, 40, None, 40, None, 40, w, None, mode, 40, 1.0, w, 1e-5)
        rt.check(L.tl_residual_norm(*args, None, 40, None, 40, D.stream))
        rt.check(L.tl_residual_norm_backward(*args, None, 40, None, 40, None, 40, None, 40, dgate, 40,
                                             o[0], o[1], 0, D.zeros(nb), nb, D.stream))
        for p in o[:2] + ([dgate] if dgate else []):
            np.testing.assert_array_equal(D.get(p, (40,)), 0.0)


def test_many_rows_two_runs_agree():
    """More rows than blocks hold at once; the same call twice gives the same bits."""
    d = inputs(5000, 136, "channel", "bf16", seed=6)
    a, b = run(d, "bf16", "rms"), run(d, "bf16", "rms")
    for k in a:
        np.testing.assert_array_equal(a[k], b[k])
    compare(a, d, "bf16", "rms")
