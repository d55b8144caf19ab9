"""What the planner may do with the language-model operators of a program, by
the steps that it lowers to: where a backward recomputes a value of the forward,
the two have to be the same value."""
import pytest

from conftest import load_backend

tl = load_backend()
L, F, C = tl.programs._let, tl.programs._fill, tl.programs._call
BW = {"type": "backward", "loss_tensor": "s"}
Y = L("y", {"type": "residual_norm", "args": ["x", "u", "w"]})
N = L("n", {"type": "scaled_norm", "args": ["y", "wn"]})
S = L("s", {"type": "sum", "tensor": "n", "axis": None})


def _sgd(*params):
    out = []
    for p in params:
        out += [L(f"{p}_step", C("mult", f"{p}_grad", "lr")), L(f"{p}_new", C("minus", p, f"{p}_step"))]
    return out + [{"type": "rebind", "name": p, "expr": {"type": "name", "name": f"{p}_new"}} for p in params]


def _loop(*body, n=3):
    return {"type": "for", "loop_var": "i", "iterations": n, "body": list(body)}


def norms(*nodes):
    """A program over x, u [4, 6] and the weights w, wn, whose gradients it takes."""
    return [L("x", F((4, 6)), (4, 6)), L("u", F((4, 6)), (4, 6)), L("w", F((6,)), (6,), grad=True),
            L("wn", F((6,)), (6,), grad=True), L("lr", tl.programs._lit([0.1], (1,)), (1,))] + list(nodes)


def calls(ast, fetch=("s", "w", "wn")):
    P = tl.Program(ast, None, fetch=list(fetch))
    P._fuse_all()
    return P, [s for s in P._all_steps() if hasattr(s, "fname")]


def count(ast, fname, **kw):
    return sum(s.fname == fname for s in calls(ast, **kw)[1])


BWD = "tl_residual_norm_backward"


@pytest.mark.parametrize("inside", [(N, S, BW), (S, BW), (BW,)])
def test_norms_of_a_forward_outside_the_loop_keep_their_own_backward(inside):
    """y was made before the loop that updates its weight: recomputed in the loop
    it would follow the weight, which the stored y does not."""
    outside = [n for n in (Y, N, S) if n not in inside]
    ast = norms(*outside, _loop(*inside, *_sgd("w", "wn")))
    P, steps = calls(ast)
    assert P.alias.get("w_new") == "w"  # the update writes the weight's buffer
    assert sum(s.fname == BWD for s in steps) == 2


def test_norms_apart_where_a_loop_updates_the_weight_before_a_top_level_backward():
    step = [L("w_step", C("mult", "w", "lr")), L("w_new", C("minus", "w", "w_step")),
            {"type": "rebind", "name": "w", "expr": {"type": "name", "name": "w_new"}}]
    P, steps = calls(norms(Y, N, S, _loop(*step), BW), fetch=("s", "w_grad", "wn_grad"))
    assert P.alias.get("w_new") == "w"
    assert sum(s.fname == BWD for s in steps) == 2


def test_norms_of_one_body_are_one_backward():
    assert count(norms(_loop(Y, N, S, BW, *_sgd("w", "wn"))), BWD) == 1
    assert count(norms(Y, N, S, BW), BWD, fetch=("s", "w_grad", "wn_grad")) == 1
    # a loop between that leaves the operands alone
    other = _loop(L("q", C("mult", "lr", "lr")))
    assert count(norms(Y, N, S, other, BW), BWD, fetch=("s", "w_grad", "wn_grad")) == 1


def head(*nodes, rows=(4, 4)):
    """A program over two batches x0, t0 and x1, t1 and the head W, b."""
    out = []
    for i, r in enumerate(rows):
        out += [L(f"x{i}", F((r, 5)), (r, 5)), L(f"t{i}", F((r,)), (r,))]
    return out + [L("W", F((5, 7)), (5, 7), grad=True), L("b", F((7,)), (7,), grad=True),
                  L("lr", tl.programs._lit([0.1], (1, 1)), (1, 1))] + list(nodes)


def loss(batch=0, name="ce"):
    return L(name, C("linear_cross_entropy", f"x{batch}", "W", "b", f"t{batch}"))


@pytest.mark.parametrize("rows", [(12, 4), (4, 12)])
@pytest.mark.parametrize("loop", [False, True])
def test_two_losses_of_one_name_have_room_for_their_rows(rows, loop):
    """Each call writes the log sums of its own rows into the loss's tensor."""
    ast = head(loss(0), _loop(loss(1)) if loop else loss(1), rows=rows)
    P, steps = calls(ast, fetch=("ce",))
    for s in steps:
        if s.fname == "tl_linear_ce":
            assert P.shapes[s.args[15][1]][0] >= s.args[2][1]


CE_BW = {"type": "backward", "loss_tensor": "ce"}


def sums_before_backward(ast, fetch=("ce", "W", "b")):
    """For each backward of the head: whether the step just before it in its list
    computes the log sums it subtracts."""
    P = tl.Program(ast, None, fetch=list(fetch), fuse_ops=False)
    out = []
    for lst in [P.phase_bw] + [lp.bw for lp in P.loops]:
        for s, before in zip(lst, [None] + lst[:-1]):
            if getattr(s, "fname", "") == "tl_linear_ce_backward":
                out.append(getattr(before, "fname", "") == "tl_linear_ce" and before.args[13] == ("null",)
                           and before.args[15] == s.args[13] and before.args[:11] == s.args[:11])
    return out


def _sgd2(*params):
    """_sgd with a rate that matrices take."""
    out = []
    for p in params:
        out += [L(f"{p}_step", C("mult", "lr", f"{p}_grad")), L(f"{p}_new", C("minus", p, f"{p}_step"))]
    return out + [{"type": "rebind", "name": p, "expr": {"type": "name", "name": f"{p}_new"}} for p in params]


def test_log_sums_follow_the_operands_where_the_forward_is_outside_the_loop():
    assert sums_before_backward(head(loss(), _loop(CE_BW, *_sgd2("W")))) == [True]


def test_log_sums_follow_an_update_before_a_top_level_backward():
    step = [L("W_new", C("mult", "W", "lr")), {"type": "rebind", "name": "W", "expr": {"type": "name", "name": "W_new"}}]
    assert sums_before_backward(head(loss(), _loop(*step), CE_BW), fetch=("W_grad",)) == [True]


def test_log_sums_of_another_loss_of_the_same_name():
    """Both losses' backwards run; the second loss's log sums are what is kept."""
    assert sorted(sums_before_backward(head(loss(0), loss(1), CE_BW), fetch=("W_grad",))) == [False, True]


def test_log_sums_are_computed_once_where_nothing_changes():
    assert sums_before_backward(head(_loop(loss(), CE_BW, *_sgd2("W")))) == [False]
    assert sums_before_backward(head(loss(), CE_BW), fetch=("W_grad",)) == [False]
    other = _loop(L("q", C("mult", "lr", "lr")))
    assert sums_before_backward(head(loss(), other, CE_BW), fetch=("W_grad",)) == [False]


def test_log_sums_computed_again_are_not_taken_for_the_forwards():
    """Two backwards of two losses of one name: the first one's second call leaves
    the first loss's log sums, which the second backward must not meet."""
    got = sums_before_backward(head(loss(0), loss(1), CE_BW, CE_BW), fetch=("W_grad",))
    assert got == [False, True, True, True]


def test_a_norm_under_the_name_of_what_it_norms_stays_a_call_of_its_own():
    """One call may not write y and n to one tensor (tl_residual_norm refuses it)."""
    again = L("y", {"type": "scaled_norm", "args": ["y", "wn"]})
    got = [s for s in calls(norms(Y, again), fetch=("y",))[1] if s.fname == "tl_residual_norm"]
    assert len(got) == 2 and all(s.args[15] != s.args[17] for s in got)


def test_a_gradient_that_the_next_iteration_reads_is_kept():
    """q reads the gradient of y that the iteration before left."""
    q = L("q", {"type": "sum", "tensor": "y_grad", "axis": None})
    ast = norms(_loop(q, Y, N, S, BW, *_sgd("w", "wn")))
    P = tl.Program(ast, {"y_grad": {"shape": (4, 6)}}, fetch=["q", "w"])
    P._fuse_all()
    assert any("y_grad" in s.writes for s in P._all_steps())
    assert sum(getattr(s, "fname", "") == BWD for s in P._all_steps()) == 2


@pytest.mark.parametrize("bias", [(1,), (6,), (8,), (1, 7)])
def test_a_bias_of_another_length_is_refused(bias):
    """The kernels read a bias for every class."""
    ast = [L("b2", F(bias), bias) if n.get("name") == "b" else n for n in head()]
    with pytest.raises(NotImplementedError):
        tl.Program(ast + [L("ce", C("linear_cross_entropy", "x0", "W", "b2", "t0"))], None, fetch=["ce"])


@pytest.mark.parametrize("node", [
    L("y", {"type": "residual_norm", "args": ["x", "u", "w"]}, (3, 6)),
    L("n", {"type": "scaled_norm", "args": ["x", "wn"]}, (4, 5)),
    L("n", {"type": "scaled_norm", "args": ["x", "wn"]}, (24,)),
    L("l", {"type": "distill_topk", "args": ["x", "u", "u"]}, (4,)),
    L("l", C("linear_cross_entropy", "x", "W", "b", "t"), (4,))])
def test_a_result_declared_in_another_shape_is_refused(node):
    ast = norms(L("W", F((6, 7)), (6, 7)), L("b", F((7,)), (7,)), L("t", F((4,)), (4,)), node)
    with pytest.raises(NotImplementedError):
        tl.Program(ast, None, fetch=[node["name"]])


def test_one_name_for_results_of_two_shapes_is_refused():
    """The name's buffer has the first one's size."""
    ast = norms(Y, L("x2", F((9, 6)), (9, 6)), L("y", {"type": "scaled_norm", "args": ["x2", "wn"]}))
    with pytest.raises(NotImplementedError):
        tl.Program(ast, None, fetch=["y"])
    tl.Program(head(L("l", C("linear_cross_entropy", "x0", "W", "b", "t0"), (1,))), None, fetch=["l"])
