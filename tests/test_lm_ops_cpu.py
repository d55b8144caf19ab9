"""The language-model operators without a GPU: what their entry points refuse
(before anything is launched), and the definitions' gradients against
differences."""
import numpy as np
import pytest

from conftest import REPO, load_backend  # noqa: F401

tl = load_backend()
from tensor_lang_b200 import runtime as rt  # noqa: E402
from oracle import lm_ops  # noqa: E402

P = 1 << 20          # a 16-byte aligned address that nothing dereferences
BAD, UNSUP = rt.TL_ERR_INVALID_ARG, rt.TL_ERR_UNSUPPORTED


def refused(fn, good, order, cases):
    """Each case changes some of the good arguments and names the status."""
    for change, status in cases:
        a = dict(good, **change)
        assert getattr(rt.load_library(), fn)(*[a[k] for k in order]) == status, (fn, change)


NORM = ["dtype", "kind", "rows", "cols", "x", "ldx", "u", "ldu", "w_post", "gate", "gate_mode",
        "ldg", "alpha", "w_pre", "eps"]
NORM_GOOD = {"dtype": 0, "kind": 1, "rows": 4, "cols": 8, "x": P, "ldx": 8, "u": P, "ldu": 8,
             "w_post": P, "gate": P, "gate_mode": 3, "ldg": 8, "alpha": 1.0, "w_pre": P, "eps": 1e-5,
             "stream": None}
NORM_BAD = [({"dtype": 2}, BAD), ({"dtype": -1}, BAD), ({"kind": 2}, BAD), ({"rows": -1}, BAD),
            ({"cols": 0}, BAD), ({"cols": -8}, BAD), ({"rows": 1 << 40}, BAD), ({"x": None}, BAD),
            ({"ldx": 7}, BAD), ({"ldu": 7}, BAD), ({"ldg": 7}, BAD), ({"gate": None}, BAD),
            ({"gate_mode": 4}, BAD), ({"gate_mode": -1}, BAD), ({"eps": -1.0}, BAD),
            ({"eps": float("nan")}, BAD), ({"alpha": float("nan")}, BAD)]


def test_residual_norm_refuses():
    good = dict(NORM_GOOD, y=2 * P, ldy=8, n=3 * P, ldn=8)
    refused("tl_residual_norm", good, NORM + ["y", "ldy", "n", "ldn", "stream"], NORM_BAD + [
        ({"y": None, "n": None}, BAD), ({"ldy": 7}, BAD), ({"ldn": 7}, BAD), ({"n": 2 * P}, BAD)])


def test_residual_norm_backward_refuses():
    nb = rt.load_library().tl_residual_norm_scratch_bytes(4, 8)
    assert nb > 0
    good = dict(NORM_GOOD, dy=P, lddy=8, dn=P, lddn=8, dx=2 * P, lddx=8, du=3 * P, lddu=8, dgate=4 * P,
                lddg=8, dw_post=5 * P, dw_pre=6 * P, acc=0, scratch=7 * P, nb=nb)
    order = NORM + ["dy", "lddy", "dn", "lddn", "dx", "lddx", "du", "lddu", "dgate", "lddg", "dw_post",
                    "dw_pre", "acc", "scratch", "nb", "stream"]
    refused("tl_residual_norm_backward", good, order, NORM_BAD + [
        ({"lddy": 7}, BAD), ({"lddn": 7}, BAD), ({"lddx": 7}, BAD), ({"lddu": 7}, BAD), ({"lddg": 7}, BAD),
        ({"u": None}, BAD), ({"gate_mode": 0}, BAD), ({"dgate": P}, BAD), ({"acc": 32}, BAD),
        ({"acc": -1}, BAD), ({"scratch": None}, BAD), ({"scratch": 7 * P + 4}, BAD), ({"nb": nb - 1}, BAD),
        ({"dx": None, "du": None, "dgate": None, "dw_post": None, "dw_pre": None}, BAD)])


def test_residual_norm_backward_refuses_one_tensor_for_two_gradients():
    nb = rt.load_library().tl_residual_norm_scratch_bytes(4, 8)
    good = dict(NORM_GOOD, dy=P, lddy=8, dn=P, lddn=8, dx=2 * P, lddx=8, du=3 * P, lddu=8, dgate=4 * P,
                lddg=8, dw_post=5 * P, dw_pre=6 * P, acc=0, scratch=7 * P, nb=nb)
    order = NORM + ["dy", "lddy", "dn", "lddn", "dx", "lddx", "du", "lddu", "dgate", "lddg", "dw_post",
                    "dw_pre", "acc", "scratch", "nb", "stream"]
    refused("tl_residual_norm_backward", good, order, [({"du": 2 * P}, BAD), ({"dw_pre": 5 * P}, BAD)])


def test_distill_refuses():
    nb = rt.load_library().tl_distill_topk_scratch_bytes(4)
    good = {"dtype": 0, "rows": 4, "classes": 100, "top": 8, "z": P, "ldz": 100, "teacher": 2 * P, "ldt": 8,
            "index": 3 * P, "ldi": 8, "it": 2, "tau": 1.0, "div": 0.0, "up": None, "loss": 4 * P,
            "row_loss": None, "lse": None, "dz": 5 * P, "lddz": 100, "acc": 0, "scratch": 6 * P, "nb": nb,
            "stream": None}
    refused("tl_distill_topk", good, list(good), [
        ({"dtype": 2}, BAD), ({"it": 3}, BAD), ({"it": -1}, BAD), ({"rows": -1}, BAD), ({"classes": 0}, BAD),
        ({"top": 0}, BAD), ({"top": -3}, BAD), ({"top": 1025, "ldt": 2000, "ldi": 2000}, UNSUP),
        ({"classes": 400000, "ldz": 400000, "lddz": 400000}, UNSUP), ({"z": None}, BAD),
        ({"teacher": None}, BAD), ({"index": None}, BAD), ({"ldz": 99}, BAD), ({"ldt": 7}, BAD),
        ({"ldi": 7}, BAD), ({"lddz": 99}, BAD), ({"tau": 0.0}, BAD), ({"tau": -1.0}, BAD),
        ({"tau": float("nan")}, BAD), ({"tau": float("inf")}, BAD), ({"div": -1.0}, BAD),
        ({"div": float("nan")}, BAD), ({"dz": P, "acc": 1}, BAD), ({"dz": P, "lddz": 101}, BAD),
        ({"loss": None, "dz": None}, BAD), ({"scratch": None}, BAD), ({"scratch": 6 * P + 8}, BAD),
        ({"nb": nb - 1}, BAD), ({"rows": 1 << 30}, UNSUP)])


def test_distill_refuses_temperatures_whose_square_or_inverse_overflows():
    nb = rt.load_library().tl_distill_topk_scratch_bytes(4)
    good = {"dtype": 0, "rows": 4, "classes": 100, "top": 8, "z": P, "ldz": 100, "teacher": 2 * P, "ldt": 8,
            "index": 3 * P, "ldi": 8, "it": 2, "tau": 1.0, "div": 0.0, "up": None, "loss": 4 * P,
            "row_loss": None, "lse": None, "dz": 5 * P, "lddz": 100, "acc": 0, "scratch": 6 * P, "nb": nb,
            "stream": None}
    refused("tl_distill_topk", good, list(good), [({"tau": t}, BAD) for t in (1e-40, 1e-19, 1e19, 3e38)])
    g = tl.KernelGenerator()
    for t in (1e-40, 1e30):
        with pytest.raises(ValueError):
            g.distill_topk("distill_topk", "l", "z", "v", "i", (4, 8), (4, 3), (4, 3), temperature=t)


def _difference(f, a, at, h=1e-5):
    up, dn = a.copy(), a.copy()
    up[at] += h
    dn[at] -= h
    return (f(up) - f(dn)) / (2 * h)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("mode", ["none", "channel", "token", "full"])
def test_residual_norm_gradients_against_differences(kind, mode):
    rng = np.random.default_rng(0)
    r, c = 3, 5
    v = {"x": rng.standard_normal((r, c)), "u": rng.standard_normal((r, c)),
         "w_post": rng.standard_normal(c), "w_pre": rng.standard_normal(c)}
    shape = {"channel": (c,), "token": (r,), "full": (r, c)}.get(mode)
    if shape:
        v["gate"] = rng.standard_normal(shape)
    dy, dn = rng.standard_normal((2, r, c))

    def total(**kw):
        y, n = lm_ops.residual_norm(gate_mode=mode, alpha=0.6, kind=kind, **kw)
        return (y * dy).sum() + (n * dn).sum()

    g = lm_ops.residual_norm_vjp(dy=dy, dn=dn, gate_mode=mode, alpha=0.6, kind=kind, **v)
    for k, a in v.items():
        for at in np.ndindex(*a.shape):
            d = _difference(lambda b: total(**dict(v, **{k: b})), a, at)
            assert abs(g["d" + k][at] - d) < 1e-7 * (1 + abs(d)), (k, at)


def test_distill_gradient_against_differences():
    rng = np.random.default_rng(1)
    z, t = rng.standard_normal((3, 7)), rng.standard_normal((3, 4))
    i = np.array([[0, 3, 3, 6], [1, -1, 2, 7], [-1, -1, -1, -1]])
    g = lm_ops.distill_topk(z, t, i, 1.7)["dz"]
    for at in np.ndindex(*z.shape):
        d = _difference(lambda b: lm_ops.distill_topk(b, t, i, 1.7)["loss"], z, at)
        assert abs(g[at] - d) < 1e-8, at


def test_linear_ce_gradients_against_differences():
    rng = np.random.default_rng(2)
    x, w, b = rng.standard_normal((4, 3)), rng.standard_normal((3, 6)), rng.standard_normal(6)
    t = np.array([0, 5, -100, 6])
    ref = lm_ops.linear_ce(x, w, t, b)
    for name, a, f in (("dx", x, lambda v: lm_ops.linear_ce(v, w, t, b)["loss"]),
                       ("dw", w, lambda v: lm_ops.linear_ce(x, v, t, b)["loss"]),
                       ("dbias", b, lambda v: lm_ops.linear_ce(x, w, t, v)["loss"])):
        for at in np.ndindex(*a.shape):
            assert abs(ref[name][at] - _difference(f, a, at)) < 1e-8, (name, at)


CE = ["dtype", "trans", "rows", "classes", "width", "x", "ldx", "w", "ldw", "bias", "target", "it", "div"]
CE_GOOD = {"dtype": 1, "trans": 0, "rows": 4, "classes": 100, "width": 16, "x": P, "ldx": 16, "w": 2 * P,
           "ldw": 100, "bias": None, "target": 3 * P, "it": 2, "div": 0.0, "scratch": 16 * P, "stream": None}
CE_BAD = [({"dtype": 2}, BAD), ({"trans": 2}, BAD), ({"trans": 1, "ldw": 15}, BAD), ({"rows": -1}, BAD),
          ({"classes": 0}, BAD), ({"width": 0}, BAD), ({"rows": 1 << 31}, UNSUP), ({"x": None}, BAD),
          ({"w": None}, BAD), ({"target": None}, BAD), ({"ldx": 15}, BAD), ({"ldw": 99}, BAD),
          ({"it": 3}, BAD), ({"div": -1.0}, BAD), ({"div": float("nan")}, BAD), ({"scratch": None}, BAD),
          ({"scratch": 16 * P + 8}, BAD)]


def test_linear_ce_refuses():
    nb = rt.load_library().tl_linear_ce_scratch_bytes(1, 0, 4, 100, 16, 0)
    good = dict(CE_GOOD, loss=4 * P, row_loss=None, lse=None, nb=nb)
    refused("tl_linear_ce", good, CE + ["loss", "row_loss", "lse", "scratch", "nb", "stream"], CE_BAD + [
        ({"loss": None}, BAD), ({"nb": nb - 1}, BAD)])


def test_linear_ce_backward_refuses():
    L = rt.load_library()
    nb = L.tl_linear_ce_scratch_bytes(1, 0, 4, 100, 16, 1)
    assert nb >= L.tl_linear_ce_scratch_bytes(1, 0, 4, 100, 16, 0)
    good = dict(CE_GOOD, lse=5 * P, up=None, dx=6 * P, lddx=16, dw=7 * P, lddw=100, dbias=8 * P, acc=0, nb=nb)
    order = CE + ["lse", "up", "dx", "lddx", "dw", "lddw", "dbias", "acc", "scratch", "nb", "stream"]
    refused("tl_linear_ce_backward", good, order, CE_BAD + [
        ({"lse": None}, BAD), ({"dx": None, "dw": None, "dbias": None}, BAD), ({"lddx": 15}, BAD),
        ({"lddw": 99}, BAD), ({"acc": 8}, BAD), ({"dx": P}, BAD), ({"dw": 2 * P}, BAD), ({"dw": P}, BAD),
        ({"dx": 7 * P}, BAD), ({"nb": nb - 1}, BAD)])


# -- lowering ----------------------------------------------------------------

def _steps(P):
    P._fuse_all()
    return [s for s in P._all_steps() if hasattr(s, "fname")]


def test_program_lowers_to_one_call_per_block_boundary():
    """With a fetch list the two norms are one call in each direction."""
    P = tl.Program(tl.programs.lm_head_train(B=64, D=32, V=100, K=4), None, fetch=["loss", "Wv"])
    names = [s.fname for s in _steps(P)]
    assert names.count("tl_residual_norm") == 1 and names.count("tl_residual_norm_backward") == 1
    assert names.count("tl_linear_ce") == 1 and names.count("tl_linear_ce_backward") == 1
    assert names.count("tl_distill_topk") == 2
    b = next(s for s in P._all_steps() if getattr(s, "fname", "") == "tl_residual_norm_backward")
    # y's gradient comes from n alone, so the fused call has no dy
    assert b.args[15] == ("null",) and b.args[17] == ("ptr", "n_grad") and b.args[25][0] == "ptr"
    # a kept gradient of y keeps the two calls apart
    P = tl.Program(tl.programs.lm_head_train(B=64, D=32, V=100, K=4), None, fetch=["loss", "y_grad"])
    names = [s.fname for s in _steps(P)]
    assert names.count("tl_residual_norm") == 1 and names.count("tl_residual_norm_backward") == 2
    P = tl.Program(tl.programs.lm_head_train(B=64, D=32, V=100, K=4), None, fuse_ops=False)
    names = [s.fname for s in _steps(P)]
    assert names.count("tl_residual_norm") == 2 and names.count("tl_residual_norm_backward") == 2


def test_second_gradient_of_one_operand_gets_its_own_tensor():
    """residual_norm(x, x, ...): one call may not write a gradient twice."""
    L = tl.programs._let
    ast = [L("x", tl.programs._fill((4, 8)), (4, 8), grad=True), L("w", tl.programs._fill((8,)), (8,)),
           L("y", {"type": "residual_norm", "args": ["x", "x", "w"]}),
           L("s", {"type": "sum", "tensor": "y", "axis": None}), {"type": "backward", "loss_tensor": "s"}]
    P = tl.Program(ast, None, fetch=["x_grad"])
    b = next(s for s in _steps(P) if s.fname == "tl_residual_norm_backward")
    dx, du = b.args[19], b.args[21]
    assert dx == ("ptr", "x_grad") and du[0] == "ptr" and du != dx


def test_generator_refuses_shapes():
    g = tl.KernelGenerator()
    for f, a in [(g.linear_cross_entropy, ("x", "w", "b", "t", (4, 8), (9, 5), (4,))),
                 (g.linear_cross_entropy, ("x", "w", "b", "t", (4, 8), (8, 5), (4, 5))),
                 (g.distill_topk, ("z", "v", "i", (4, 8), (4, 3), (4, 2))),
                 (g.distill_topk, ("z", "v", "i", (4, 8), (3, 2), (3, 2))),
                 (g.residual_norm, ("x", "u", "w", None, (4, 8), (4, 7), (8,), None)),
                 (g.residual_norm, ("x", "u", "w", "g", (4, 8), (4, 8), (8,), (4,))),
                 (g.scaled_norm, ("x", "w", (4, 8), (4,)))]:
        with pytest.raises(NotImplementedError):
            f(f.__name__, "out", *a)
    with pytest.raises(ValueError):
        g.scaled_norm("scaled_norm", "n", "x", "w", (4, 8), (8,), norm="batch")
    with pytest.raises(ValueError):
        g.distill_topk("distill_topk", "l", "z", "v", "i", (4, 8), (4, 3), (4, 3), temperature=0.0)
    with pytest.raises(ValueError):
        g.linear_cross_entropy("linear_cross_entropy", "l", "x", "w", "b", "t", (4, 8), (8, 5), (4,),
                               divisor=-1.0)
    with pytest.raises(ValueError):
        g.distill_topk("linear", "l", "z", "v", "i", (4, 8), (4, 3), (4, 3))


def test_sharded_batches_name_their_divisor():
    from tensor_lang_b200 import dp
    ast = tl.programs.lm_head_train(B=64, D=32, V=100, K=4)
    derived = dp.batch_derived(ast, ("x", "t", "top", "topi"))
    assert {"n", "z"} <= derived and "ce" not in derived and "Wv_new" not in derived
    with pytest.raises(NotImplementedError):
        dp.check_loss_divisors(ast, derived)
    for node in ast[-1]["body"]:
        if node["type"] == "let" and node["expr"]["type"] in ("linear_cross_entropy", "distill_topk"):
            node["expr"]["divisor"] = 64
    dp.check_loss_divisors(ast, derived)


def test_residual_norm_refuses_outputs_over_other_rows_of_an_operand():
    """In place is row on row: another leading dimension would write rows not read yet."""
    good = dict(NORM_GOOD, x=P, u=5 * P, y=2 * P, ldy=9, n=3 * P, ldn=9)
    refused("tl_residual_norm", good, NORM + ["y", "ldy", "n", "ldn", "stream"], [
        ({"y": P}, BAD), ({"y": 5 * P}, BAD), ({"n": P}, BAD), ({"n": 5 * P}, BAD)])


def test_residual_norm_backward_refuses_outputs_over_what_it_still_reads():
    nb = rt.load_library().tl_residual_norm_scratch_bytes(4, 8)
    good = dict(NORM_GOOD, x=8 * P, u=9 * P, w_post=10 * P, gate=11 * P, w_pre=12 * P, dy=13 * P, lddy=8,
                dn=14 * P, lddn=8, dx=2 * P, lddx=8, du=3 * P, lddu=8, dgate=4 * P, lddg=8, dw_post=5 * P,
                dw_pre=6 * P, acc=0, scratch=7 * P, nb=nb)
    order = NORM + ["dy", "lddy", "dn", "lddn", "dx", "lddx", "du", "lddu", "dgate", "lddg", "dw_post",
                    "dw_pre", "acc", "scratch", "nb", "stream"]
    channel = {"gate_mode": 1}
    refused("tl_residual_norm_backward", good, order, [
        ({"dx": 13 * P, "lddx": 9}, BAD), ({"du": 14 * P, "lddu": 9}, BAD), ({"dx": 11 * P}, BAD),
        ({"du": 11 * P}, BAD), ({"dgate": 2 * P}, BAD), ({"dgate": 3 * P}, BAD), ({"dgate": 5 * P}, BAD),
        ({"dgate": 6 * P}, BAD), (dict(channel, dw_post=11 * P), BAD), (dict(channel, dw_post=10 * P), BAD),
        (dict(channel, dgate=10 * P), BAD)])
