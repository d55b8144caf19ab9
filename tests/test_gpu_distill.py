"""tl_distill_topk against the definition in float64.

Tolerances (float32): lse is m + log(s) with s a sum of positive terms, each
within 2^-22 + |x| 2^-24 (x the exponent, below 40 here): 3e-6 relative, so 3e-6
absolute in lse, which is of order 10; row losses are sums of magnitude
tau^2 (log s + |z - m|) < tau^2 (|lse| + 2 |z|): rel 1e-5 of that; dz is cf (p - q), p within 5e-6 and q
within 2e-6 of themselves: rel 1e-5 of the row's p + q.  bf16 adds its half step
to dz.
"""
import numpy as np
import pytest

from conftest import REPO  # noqa: F401
from lm_util import CODE, Dev, close, rounded, rt
from oracle import lm_ops

pytestmark = pytest.mark.gpu

IDX = {"f32": (rt.IDX_F32, np.float32), "i32": (rt.IDX_I32, np.int32), "i64": (rt.IDX_I64, np.int64)}


def inputs(rows, classes, top, dtype, seed=0, ragged=False, spread=2.0):
    rng = np.random.default_rng(seed + 31 * rows + classes + top)
    z = rounded(rng.standard_normal((rows, classes)) * spread, dtype)
    t = rounded(rng.standard_normal((rows, top)) * 2 + 8, dtype)
    i = rng.integers(0, classes, (rows, top))
    if ragged:
        i[np.arange(top)[None, :] >= rng.integers(0, top + 1, rows)[:, None]] = -1
    return z, t, i


def run(z, t, i, dtype, idx="i64", tau=1.0, divisor=0.0, up=None, want=("loss", "row_loss", "lse", "dz"),
        pad=0, lead=0, start=None, in_place=False, calls=1):
    rows, classes = z.shape
    top = t.shape[1]
    code, ity = IDX[idx]
    with Dev() as D:
        L = rt.lib()
        pz, ldz = D.rows(z, dtype, classes + pad, lead)
        pt, ldt = D.rows(t, dtype, top + pad)
        ii = np.full((rows, top + 2), 0, ity)
        ii[:, :top] = i
        pi = D.put(ii)
        nb = L.tl_distill_topk_scratch_bytes(rows)
        o = {k: D.new(n) for k, n in (("loss", 1), ("row_loss", rows), ("lse", rows)) if k in want}
        ld = classes + pad
        acc = 0
        if in_place:
            o["dz"] = pz
        elif "dz" in want:
            o["dz"] = D.rows(np.full(z.shape, 7.0) if start is None else start, dtype, ld, lead)[0]
            acc = 0 if start is None else 1
        pu = None if up is None else D.put(np.float32([up]))
        scratch = D.zeros(nb)
        for _ in range(calls):
            rt.check(L.tl_distill_topk(CODE[dtype], rows, classes, top, pz, ldz, pt, ldt, pi, top + 2, code,
                                       tau, divisor, pu, o.get("loss"), o.get("row_loss"), o.get("lse"),
                                       o.get("dz"), ld, acc, scratch, nb, D.stream), "distill")
        got = {k: D.get(p, (1,) if k == "loss" else (rows,)) for k, p in o.items() if k != "dz"}
        if "dz" in o:
            got["dz"], rest = D.get_rows(o["dz"], rows, classes, ld, dtype, lead)
            assert np.all(rest == 7.0), "written between rows"
    return got


def compare(got, z, t, i, dtype, tau=1.0, divisor=0.0, up=1.0, start=None):
    ref = lm_ops.distill_topk(z, t, i, tau, divisor, up)
    size = tau * tau * (np.abs(ref["lse"]) + 2 * np.abs(z / tau).max(axis=1) + 10)
    if "lse" in got:
        close(got["lse"], ref["lse"], "f32", "lse", scale=1.0)
    if "row_loss" in got:
        close(got["row_loss"], ref["row_loss"], "f32", "row_loss", scale=size)
    if "loss" in got:
        close(got["loss"], [ref["loss"]], "f32", "loss", scale=size.mean())
    if "dz" in got:
        want = ref["dz"]
        scale = np.abs(ref["dz"]).max(axis=1, keepdims=True) + (0 if start is None else np.abs(start))
        close(got["dz"], want if start is None else want + start, dtype, "dz", scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,classes,top", [
    (1, 1, 1), (2, 2, 1), (3, 5, 9), (1, 31, 4), (7, 33, 3), (40, 500, 16), (5, 1000, 100),
    (2, 4097, 8), (3, 8192, 64), (2, 16391, 37), (9, 32000, 16), (3, 50021, 33), (2, 131072, 64),
    (600, 300, 5), (1, 120000, 1024)])
def test_sizes(dtype, rows, classes, top):
    """One class to clusters of eight; lists longer than the vocabulary, with
    the same class several times."""
    z, t, i = inputs(rows, classes, top, dtype)
    compare(run(z, t, i, dtype), z, t, i, dtype)


@pytest.mark.parametrize("idx", ["f32", "i32", "i64"])
@pytest.mark.parametrize("tau,divisor,up", [(1.0, 0.0, None), (2.0, 0.0, 0.5), (0.7, 64.0, 3.0)])
def test_index_types_and_scales(idx, tau, divisor, up):
    z, t, i = inputs(50, 777, 12, "f32", ragged=True, seed=3)
    compare(run(z, t, i, "f32", idx=idx, tau=tau, divisor=divisor, up=up), z, t, i, "f32", tau, divisor,
            1.0 if up is None else up)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,lead", [(0, 1), (1, 0), (8, 0), (3, 5)])
@pytest.mark.parametrize("classes", [203, 20011])
def test_strides_and_offsets(dtype, pad, lead, classes):
    z, t, i = inputs(6, classes, 7, dtype, seed=4)
    compare(run(z, t, i, dtype, pad=pad, lead=lead), z, t, i, dtype)


def test_parts_in_place_accumulate_and_repeated_calls():
    z, t, i = inputs(33, 2500, 20, "f32", ragged=True, seed=5)
    compare(run(z, t, i, "f32", want=("loss",)), z, t, i, "f32")
    compare(run(z, t, i, "f32", want=("row_loss", "lse")), z, t, i, "f32")
    compare(run(z, t, i, "f32", want=("dz",)), z, t, i, "f32")
    compare(run(z, t, i, "f32", in_place=True), z, t, i, "f32")
    start = rounded(np.random.default_rng(1).standard_normal(z.shape) * 0.01, "f32")
    compare(run(z, t, i, "f32", start=start), z, t, i, "f32", start=start)
    compare(run(z, t, i, "f32", calls=3), z, t, i, "f32")  # the scratch is ready again


def test_masks_and_empty_lists():
    """-inf logits, -inf teacher logits, classes out of range, rows without a
    list, all rows without one."""
    z, t, i = inputs(8, 700, 6, "f32", seed=6)
    z[0, 100:] = -np.inf
    i[0] = np.arange(6)              # a masked row, the list inside the support
    z[1, i[1, 0]] = -np.inf          # a listed class without probability: loss +inf
    t[2, 1:] = -np.inf               # one entry counts
    t[3] = -np.inf                   # none does
    i[4] = [700, -1, 10 ** 6, -100, 701, -2 ** 31]
    z[5] = np.finfo(np.float32).min  # the type's lowest value everywhere: uniform
    z[6] = -np.inf                   # nothing left
    got = run(z, t, i, "f32")
    with np.errstate(invalid="ignore"):
        ref = lm_ops.distill_topk(z, t, i)
    assert np.isposinf(ref["row_loss"][[1, 6]]).all() and np.isposinf(got["row_loss"][[1, 6]]).all()
    assert np.isposinf(got["loss"][0])
    assert got["row_loss"][3] == 0 and got["row_loss"][4] == 0
    assert not got["dz"][3].any() and not got["dz"][4].any()
    assert np.isneginf(got["lse"][6])
    ok = [0, 2, 3, 4, 5, 7]
    close(got["row_loss"][ok], ref["row_loss"][ok], "f32", "row_loss", scale=20.0)
    close(got["dz"], ref["dz"], "f32", "dz", scale=np.abs(ref["dz"]).max(axis=1, keepdims=True) + 1e-30)
    none = run(z, t, np.full_like(i, -1), "f32")
    assert none["loss"][0] == 0 and not none["row_loss"].any() and not none["dz"].any()


def test_nan_stays_in_its_row():
    z, t, i = inputs(4, 3000, 5, "f32", seed=7)
    z[1, 2999] = np.nan
    t[2, 0] = np.nan
    got = run(z, t, i, "f32")
    ref = lm_ops.distill_topk(z[[0, 3]], t[[0, 3]], i[[0, 3]], divisor=4.0)
    close(got["dz"][[0, 3]], ref["dz"], "f32", "dz")
    assert np.isnan(got["row_loss"][[1, 2]]).all() and np.isnan(got["dz"][1]).all()


def test_float_indices_that_name_no_class():
    z, t, _ = inputs(2, 64, 4, "f32", seed=8)
    i = np.array([[1.0, 2.5, np.nan, -1.0], [63.0, 64.0, 3.0, np.inf]])
    ints = np.array([[1, -1, -1, -1], [63, -1, 3, -1]])
    got = run(z, t, i, "f32", idx="f32")
    compare(got, z, t, ints, "f32")


def test_two_runs_agree():
    z, t, i = inputs(700, 5003, 50, "bf16", seed=9)
    a, b = run(z, t, i, "bf16"), run(z, t, i, "bf16")
    for k in a:
        np.testing.assert_array_equal(a[k], b[k])


def test_no_rows():
    with Dev() as D:
        L = rt.lib()
        nb = L.tl_distill_topk_scratch_bytes(0)
        loss = D.new(1)
        rt.check(L.tl_distill_topk(0, 0, 10, 2, None, 10, None, 2, None, 2, 2, 1.0, 0.0, None, loss, None,
                                   None, None, 10, 0, D.zeros(nb), nb, D.stream))
        assert D.get(loss, (1,))[0] == 0


# -- every cell to its own size ------------------------------------------------
# dz = cf (p - q).  p = 2^((z - m) k2) / s: z - m, k2 and the product round (three
# times 2^-24 of an exponent below 30 here), 2^x and the inverse add 2^-21: below 1e-5
# of p.  q the same way.  So a class that no list names is held to 1e-5 of its own
# p, however large the row's listed ones are.

def cells(got, z, t, i, dtype, tau=1.0, divisor=0.0, up=1.0, start=None):
    ref = lm_ops.distill_topk(z, t, i, tau, divisor, up)
    ok = (i >= 0) & (i < z.shape[1]) & ~np.isneginf(t)
    some = ok.any(axis=1)
    cf = np.where(some, tau * up / (divisor if divisor > 0 else max(1, int(some.sum()))), 0.0)[:, None]
    size = np.zeros(z.shape)  # cf (p + q)
    for r in np.nonzero(some)[0]:
        q = np.exp((t[r, ok[r]] - t[r, ok[r]].max()) / tau)
        np.add.at(size[r], i[r, ok[r]].astype(int), 2 * np.abs(cf[r]) * q / q.sum())
    size += np.abs(ref["dz"])  # p - q + 2 q
    want = ref["dz"] if start is None else ref["dz"] + start
    tol = 1e-5 * size + (0.0 if start is None else 2.0 ** -23 * (np.abs(start) + np.abs(want)))
    if dtype == "bf16":
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
    bad = ~(np.abs(got["dz"].astype(np.float64) - want) <= tol)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, np.abs(got["dz"] - want) / (tol + 1e-300), -1)), want.shape)
        raise AssertionError(f"dz: {int(bad.sum())} of {want.size} off; worst at {at}: got {got['dz'][at]!r}, "
                             f"want {want[at]!r}, allowed {tol[at]:.3g}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,classes,top", [
    (1, 1, 1), (3, 5, 9), (7, 33, 3), (40, 500, 16), (2, 4097, 8), (3, 8192, 64), (2, 16391, 37), (9, 32000, 16),
    (3, 50021, 33), (40, 50021, 37), (2, 131072, 64), (300, 16391, 20)])
def test_every_cell(dtype, rows, classes, top):
    z, t, i = inputs(rows, classes, top, dtype, seed=20, ragged=rows > 2)
    cells(run(z, t, i, dtype, want=("dz",)), z, t, i, dtype)
    cells(run(z, t, i, dtype, tau=2.0, divisor=7.0, up=0.5), z, t, i, dtype, 2.0, 7.0, 0.5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,lead", [(0, 1), (1, 0), (3, 5)])
@pytest.mark.parametrize("rows,classes", [(5, 20011), (30, 20011)])
def test_every_cell_of_odd_rows(dtype, pad, lead, rows, classes):
    z, t, i = inputs(rows, classes, 7, dtype, seed=21)
    cells(run(z, t, i, dtype, pad=pad, lead=lead), z, t, i, dtype)
    start = rounded(np.random.default_rng(2).standard_normal(z.shape) * 1e-5, dtype)
    cells(run(z, t, i, dtype, pad=pad, lead=lead, start=start), z, t, i, dtype, start=start)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [6, 60])
def test_every_cell_of_masked_rows(dtype, rows):
    """-inf in whole segments of a cluster, the type's lowest value beside ordinary
    logits and alone, listed classes without probability, NaN in another row."""
    low = float(rounded([-3.3e38], dtype)[0])
    z, t, i = inputs(rows, 20000, 6, dtype, seed=22)
    z[0, 3000:] = -np.inf
    z[1, :17000] = -np.inf
    z[2, 100:] = low
    z[3] = low
    z[4, i[4, 0]] = -np.inf
    t[0, 2:] = -np.inf
    z[5, 19999] = np.nan
    got = run(z, t, i, dtype, divisor=float(rows))
    keep = np.arange(rows) != 5
    assert np.isnan(got["dz"][5]).all()
    cells({"dz": got["dz"][keep]}, z[keep], t[keep], i[keep], dtype, divisor=float(rows))


@pytest.mark.parametrize("dtype,classes", [("f32", 393216), ("bf16", 786432), ("f32", 393001), ("bf16", 786001)])
@pytest.mark.parametrize("rows", [2, 20])
def test_the_longest_rows_and_lists(dtype, classes, rows):
    """Rows of 1536 KB (segments of 192 KB) beside lists of 1024."""
    z, t, i = inputs(rows, classes, 1024, dtype, seed=23)
    got = run(z, t, i, dtype)
    cells(got, z, t, i, dtype)
    compare({k: got[k] for k in ("loss", "row_loss", "lse")}, z, t, i, dtype)
