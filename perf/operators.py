"""Language-model head and block-boundary operators: cases, plain forms, exact values.

Three operators, each with its gradient:

* ``linear_ce``      cross entropy of a linear layer over a large vocabulary,
                     without keeping the logits;
* ``distill_topk``   distillation from a teacher's top logits (KL divergence);
* ``residual_norm``  the norm after a block, its gate, the scaled residual and
                     the norm before the next block.

``own`` selects what ``run`` does: the plain form in elementary torch
operations, or the calls of this repository's C interface.
"""
import ctypes
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_CODE = {"f32": 0, "bf16": 1}          # TL_F32, TL_BF16
_I64 = 2                               # TL_IDX_I64
_KIND = {"layer": 0, "rms": 1}         # TL_NORM_LAYER, TL_NORM_RMS
_GATE = {"none": 0, "channel": 1, "token": 2, "full": 3}
_EPS = 1e-5


# --------------------------------------------------------------------- cases

def _lce(name, rows, vocab, width, dtype, layout, bias, train):
    c = {"op": "linear_ce", "rows": rows, "vocab": vocab, "width": width, "dtype": dtype,
         "layout": layout, "bias": bias, "train": train}
    return dict(c, name=name) if name else c


def _kd(name, rows, vocab, top, dtype, ragged, temperature):
    c = {"op": "distill_topk", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype,
         "ragged": ragged, "temperature": temperature}
    return dict(c, name=name) if name else c


def _rn(name, rows, width, dtype, kind, gate, train):
    c = {"op": "residual_norm", "rows": rows, "width": width, "dtype": dtype, "kind": kind,
         "gate": gate, "train": train}
    return dict(c, name=name) if name else c


def listed():
    return [
        # scoring one token while serving: the weights are read once, nothing else counts
        _lce("ce score 1", 1, 32768, 4096, "bf16", "vd", False, False),
        # perplexity of a few short prompts, weights stored as linear() takes them
        _lce("ce score 96", 96, 65536, 2048, "bf16", "dv", False, False),
        # a small fine-tuning step in float32 with a bias, as linear() + cross_entropy would run it
        _lce("ce train f32", 2048, 32000, 1024, "f32", "dv", True, True),
        # odd sizes: a vocabulary that is no multiple of anything, rows that are padding
        _lce("ce train odd", 1537, 50021, 1000, "bf16", "dv", True, True),
        # the largest: a whole training batch, tied embedding weights
        _lce("ce train large", 8192, 131072, 4096, "bf16", "vd", False, True),
        # distillation of a handful of answers: latency
        _kd("distill 8", 8, 32000, 16, "f32", False, 1.0),
        # odd vocabulary, lists of different lengths, a temperature
        _kd("distill odd", 1537, 50021, 37, "f32", True, 2.0),
        # the largest: a training batch against cached teacher logits
        _kd("distill large", 8192, 131072, 64, "bf16", False, 1.0),
        # one token while serving
        _rn("norm 1", 1, 4096, "bf16", "rms", "channel", False),
        # a prefill's worth of tokens, no backward
        _rn("norm 4096", 4096, 8192, "bf16", "rms", "none", False),
        # odd sizes, layer norm, a gate per element, float32
        _rn("norm train odd", 3001, 1021, "f32", "layer", "full", True),
        # the largest: a training batch with a learned gate per channel
        _rn("norm train large", 65536, 4096, "bf16", "rms", "channel", True),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear_ce", "distill_topk", "residual_norm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "linear_ce":
        width = _spread(rng, 64, 4096)
        if rng.random() < 0.6:
            width = max(64, width // 8 * 8)
        return _lce(None, _spread(rng, 1, 8192), _spread(rng, 500, 131072), width, dtype,
                    rng.choice(["vd", "dv"]), rng.random() < 0.3, rng.random() < 0.7)
    if op == "distill_topk":
        return _kd(None, _spread(rng, 1, 8192), _spread(rng, 500, 131072), _spread(rng, 1, 400),
                   dtype, rng.random() < 0.5, rng.choice([1.0, 2.0, 0.7]))
    width = _spread(rng, 64, 8192)
    return _rn(None, min(_spread(rng, 1, 65536), 65536 * 4096 // width), width, dtype,
               rng.choice(["layer", "rms"]), rng.choice(["none", "channel", "token", "full"]),
               rng.random() < 0.7)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    t = case["rows"]
    if case["op"] == "linear_ce":
        v, d = case["vocab"], case["width"]
        b = (4 * v if case["bias"] else 0) + 8 * t + 8 * t + 4
        n = e * (t * d + v * d)
        if case["train"]:  # gradients of the input and the weights (and the bias)
            return {"bytes": 2 * n + 2 * b, "flops": 6 * t * v * d}
        return {"bytes": n + b, "flops": 2 * t * v * d}
    if case["op"] == "distill_topk":
        v, k = case["vocab"], case["top"]
        return {"bytes": 2 * e * t * v + (8 + e) * t * k + 8 * t, "flops": 8 * t * v}
    d = case["width"]
    g = {"none": 0, "channel": d, "token": t, "full": t * d}[case["gate"]]
    fwd = 4 * t * d + 2 * d + g
    if not case["train"]:
        return {"bytes": e * fwd, "flops": 12 * t * d}
    # forward, then the two gradients and the inputs again, and all gradients out
    bwd = 4 * t * d + 2 * d + g + 2 * t * d + 2 * d + g
    return {"bytes": e * (fwd + bwd), "flops": 40 * t * d}


# -------------------------------------------------------------------- inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    t = case["rows"]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=dev) * scale + shift).to(dtype)

    def ids(n, *shape):
        return torch.randint(0, n, shape, generator=gen, device=dev)

    s = {"case": dict(case), "up": torch.full((1,), 0.5, device=dev)}
    if case["op"] == "linear_ce":
        v, d = case["vocab"], case["width"]
        shape = (v, d) if case["layout"] == "vd" else (d, v)
        s["x"] = normal(t, d)
        s["w"] = normal(*shape, scale=1.5 / math.sqrt(d))
        s["bias"] = normal(v, scale=0.5, dtype=torch.float32) if case["bias"] else None
        target = ids(v, t)
        if t > 16:  # padding: rows without a target
            target[ids(t, max(1, t // 40))] = -100
        s["target"] = target
    elif case["op"] == "distill_topk":
        v, k = case["vocab"], case["top"]
        s["z"] = normal(t, v, scale=2.0)
        s["teacher"] = normal(t, k, scale=2.0, shift=8.0).sort(dim=1, descending=True).values.contiguous()
        s["index"] = ids(v, t, k)
        if case["ragged"]:  # lists end early; some rows have none
            length = ids(k + 1, t)
            s["index"][torch.arange(k, device=dev)[None, :] >= length[:, None]] = -1
    else:
        d = case["width"]
        gate = {"none": None, "channel": (d,), "token": (t,), "full": (t, d)}[case["gate"]]
        s["x"], s["u"] = normal(t, d, scale=2.0), normal(t, d, scale=0.7, shift=0.1)
        s["w_post"], s["w_pre"] = normal(d, scale=0.2, shift=1.0), normal(d, scale=0.2, shift=1.0)
        s["gate"] = normal(*gate, scale=0.5) if gate else None
        s["alpha"] = 0.75
        if case["train"]:
            s["dy"], s["dn"] = normal(t, d), normal(t, d)
    return s


# --------------------------------------------------------------- plain forms

def _plain_linear_ce(s):
    c = s["case"]
    x, w, target = s["x"].float(), s["w"].float(), s["target"]
    z = x @ (w.t() if c["layout"] == "vd" else w)
    if s["bias"] is not None:
        z += s["bias"]
    keep = (target >= 0) & (target < c["vocab"])
    rows = torch.arange(c["rows"], device=z.device)
    at = torch.where(keep, target, torch.zeros_like(target))
    m = z.amax(dim=1, keepdim=True)
    chosen = z[rows, at]
    p = torch.exp(z.sub_(m))
    total = p.sum(dim=1, keepdim=True)
    lse = (m + torch.log(total))[:, 0]
    row_loss = torch.where(keep, lse - chosen, torch.zeros_like(lse))
    count = keep.sum().clamp(min=1)
    out = {"loss": (row_loss.sum() / count).reshape(1), "row_loss": row_loss, "lse": lse}
    if not c["train"]:
        return out
    g = p.div_(total)
    g[rows, at] -= 1.0
    g *= (keep.float() * (s["up"] / count))[:, None]
    out["dx"] = (g @ (w if c["layout"] == "vd" else w.t())).to(s["x"].dtype)
    out["dw"] = (g.t() @ x if c["layout"] == "vd" else x.t() @ g).to(s["w"].dtype)
    if s["bias"] is not None:
        out["dbias"] = g.sum(dim=0)
    return out


def _plain_distill_topk(s):
    tau = s["case"]["temperature"]
    z, index = s["z"].float() / tau, s["index"]
    keep = (index >= 0) & (index < s["case"]["vocab"])
    at = torch.where(keep, index, torch.zeros_like(index))
    some = keep.any(dim=1)
    t = torch.where(keep, s["teacher"].float() / tau, float("-inf"))
    tm = torch.where(some, t.amax(dim=1), 0.0)[:, None]
    te = torch.exp(t - tm)
    ts = torch.where(some, te.sum(dim=1), 1.0)[:, None]
    q = te / ts
    m = z.amax(dim=1, keepdim=True)
    chosen = torch.gather(z, 1, at)
    p = torch.exp(z.sub_(m))
    total = p.sum(dim=1, keepdim=True)
    lse = m + torch.log(total)
    log_q = torch.where(q > 0, t - tm - torch.log(ts), 0.0)
    row_loss = tau * tau * torch.where(q > 0, q * (log_q - (chosen - lse)), 0.0).sum(dim=1)
    count = some.sum().clamp(min=1)
    dz = p.div_(total).scatter_add_(1, at, -q)
    dz *= (some.float() * (s["up"] * tau / count))[:, None]
    return {"loss": (row_loss.sum() / count).reshape(1), "row_loss": row_loss, "lse": lse[:, 0],
            "dz": dz.to(s["z"].dtype)}


def _normed(v, kind):
    """(normalised v, 1 / scale) along the last axis, in float32."""
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    r = torch.rsqrt((v * v).mean(dim=1, keepdim=True) + _EPS)
    return v * r, r


def _normed_grad(g, hat, r, kind):
    """Gradient of the norm's input, from that of its normalised output."""
    if kind == "layer":
        g = g - g.mean(dim=1, keepdim=True)
    return r * (g - hat * (g * hat).mean(dim=1, keepdim=True))


def _plain_residual_norm(s):
    c = s["case"]
    x, u, wa, wb = s["x"].float(), s["u"].float(), s["w_post"].float(), s["w_pre"].float()
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    if c["gate"] == "token":
        gate = gate[:, None]
    hat_u, ru = _normed(u, c["kind"])
    post = hat_u * wa
    y = s["alpha"] * x + gate * post
    hat_y, ry = _normed(y, c["kind"])
    dt = s["x"].dtype
    out = {"y": y.to(dt), "n": (hat_y * wb).to(dt)}
    if not c["train"]:
        return out
    dn = s["dn"].float()
    dy = s["dy"].float() + _normed_grad(dn * wb, hat_y, ry, c["kind"])
    dpost = dy * gate
    out["dx"] = (s["alpha"] * dy).to(dt)
    out["du"] = _normed_grad(dpost * wa, hat_u, ru, c["kind"]).to(dt)
    out["dw_post"] = (dpost * hat_u).sum(dim=0).to(dt)
    out["dw_pre"] = (dn * hat_y).sum(dim=0).to(dt)
    if c["gate"] == "channel":
        out["dgate"] = (dy * post).sum(dim=0).to(dt)
    elif c["gate"] == "token":
        out["dgate"] = (dy * post).sum(dim=1).to(dt)
    elif c["gate"] == "full":
        out["dgate"] = (dy * post).to(dt)
    return out


# ------------------------------------------------- the framework's own calls

_backend = None


def _lib():
    """(library, status check) of this repository's package, loaded on first use."""
    global _backend
    if _backend is None:
        name = "tensor_lang_b200"
        tl = sys.modules.get(name)
        if tl is None:
            root = Path(__file__).resolve().parent.parent / "tensor-lang_b200"
            spec = importlib.util.spec_from_file_location(name, root / "__init__.py",
                                                          submodule_search_locations=[str(root)])
            tl = importlib.util.module_from_spec(spec)
            sys.modules[name] = tl
            spec.loader.exec_module(tl)
        tl.Device.get(torch.cuda.current_device())
        _backend = (tl.load_library(), tl.runtime.check)
    return _backend


def _stream():
    """The stream torch works on; 1 is the handle of the legacy default stream."""
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream or 1)


def _p(t):
    return None if t is None else t.data_ptr()


def _buffers(s, make):
    """Output buffers and scratch, kept beside the inputs as a training program keeps them."""
    if "own" not in s:
        s["own"] = make()
    return s["own"]


def _like(*ts):
    return [None if t is None else torch.empty_like(t) for t in ts]


def _own_linear_ce(s):
    L, check = _lib()
    c = s["case"]
    t, v, d = c["rows"], c["vocab"], c["width"]
    code, vd = _CODE[c["dtype"]], 1 if c["layout"] == "vd" else 0
    x, w, bias, target = s["x"], s["w"], s["bias"], s["target"]

    def make():
        n = L.tl_linear_ce_scratch_bytes(code, vd, t, v, d, 1 if c["train"] else 0)
        o = {k: torch.empty(m, device=x.device) for k, m in (("loss", 1), ("row_loss", t), ("lse", t))}
        if c["train"]:
            o["dx"], o["dw"], o["dbias"] = _like(x, w, bias)
        return {k: b for k, b in o.items() if b is not None}, torch.zeros(n, dtype=torch.uint8, device=x.device)

    o, scratch = _buffers(s, make)
    st = _stream()
    check(L.tl_linear_ce(code, vd, t, v, d, _p(x), d, _p(w), w.shape[1], _p(bias), _p(target), _I64, 0.0,
                         _p(o["loss"]), _p(o["row_loss"]), _p(o["lse"]), _p(scratch), scratch.numel(), st))
    if c["train"]:
        check(L.tl_linear_ce_backward(code, vd, t, v, d, _p(x), d, _p(w), w.shape[1], _p(bias), _p(target), _I64,
                                      0.0, _p(o["lse"]), _p(s["up"]), _p(o["dx"]), d, _p(o["dw"]), w.shape[1],
                                      _p(o.get("dbias")), 0, _p(scratch), scratch.numel(), st))
    return o


def _own_distill_topk(s):
    L, check = _lib()
    c = s["case"]
    t, v, k, code = c["rows"], c["vocab"], c["top"], _CODE[c["dtype"]]
    z = s["z"]

    def make():
        n = L.tl_distill_topk_scratch_bytes(t)
        o = {q: torch.empty(m, device=z.device) for q, m in (("loss", 1), ("row_loss", t), ("lse", t))}
        o["dz"] = torch.empty_like(z)
        return o, torch.zeros(n, dtype=torch.uint8, device=z.device)

    o, scratch = _buffers(s, make)
    # the loss and its gradient from one read of the logits
    check(L.tl_distill_topk(code, t, v, k, _p(z), v, _p(s["teacher"]), k, _p(s["index"]), k, _I64,
                            c["temperature"], 0.0, _p(s["up"]), _p(o["loss"]), _p(o["row_loss"]), _p(o["lse"]),
                            _p(o["dz"]), v, 0, _p(scratch), scratch.numel(), _stream()))
    return o


def _own_residual_norm(s):
    L, check = _lib()
    c = s["case"]
    t, d, code, kind, mode = c["rows"], c["width"], _CODE[c["dtype"]], _KIND[c["kind"]], _GATE[c["gate"]]
    x, u, wa, wb, gate = s["x"], s["u"], s["w_post"], s["w_pre"], s["gate"]

    def make():
        o = dict(zip(("y", "n"), _like(x, x)))
        n = 0
        if c["train"]:
            o.update(zip(("dx", "du", "dgate", "dw_post", "dw_pre"), _like(x, u, gate, wa, wb)))
            n = L.tl_residual_norm_scratch_bytes(t, d)
        return {k: b for k, b in o.items() if b is not None}, torch.zeros(n, dtype=torch.uint8, device=x.device)

    o, scratch = _buffers(s, make)
    st = _stream()
    check(L.tl_residual_norm(code, kind, t, d, _p(x), d, _p(u), d, _p(wa), _p(gate), mode, d, s["alpha"], _p(wb),
                             _EPS, _p(o["y"]), d, _p(o["n"]), d, st))
    if c["train"]:
        check(L.tl_residual_norm_backward(code, kind, t, d, _p(x), d, _p(u), d, _p(wa), _p(gate), mode, d,
                                          s["alpha"], _p(wb), _EPS, _p(s["dy"]), d, _p(s["dn"]), d,
                                          _p(o["dx"]), d, _p(o["du"]), d, _p(o.get("dgate")), d,
                                          _p(o["dw_post"]), _p(o["dw_pre"]), 0, _p(scratch), scratch.numel(), st))
    return o


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear_ce": _own_linear_ce, "distill_topk": _own_distill_topk,
                "residual_norm": _own_residual_norm}[op](state)
    return {"linear_ce": _plain_linear_ce, "distill_topk": _plain_distill_topk,
            "residual_norm": _plain_residual_norm}[op](state)


# ------------------------------------------------------- exact values (float64)

def _exact_linear_ce(s, c):
    w = s["w"].double()
    w = w if c["layout"] == "vd" else w.t()          # [vocab, width]
    x = s["x"].double()
    z = torch.matmul(x, w.t())
    if s["bias"] is not None:
        z = z + s["bias"].double()
    lse = torch.logsumexp(z, dim=1)
    counted = torch.nonzero((s["target"] >= 0) & (s["target"] < c["vocab"]))[:, 0]
    hit = s["target"][counted]
    row_loss = torch.zeros_like(lse)
    row_loss[counted] = lse[counted] - z[counted, hit]
    n = max(1, int(counted.numel()))
    out = {"loss": row_loss.sum().reshape(1) / n, "row_loss": row_loss, "lse": lse}
    if not c["train"]:
        return out
    z.sub_(lse[:, None]).exp_()                      # softmax
    used = torch.zeros_like(lse)
    used[counted] = 1.0
    z[counted, hit] -= 1.0
    z *= (used * s["up"].double() / n)[:, None]
    out["dx"] = torch.matmul(z, w)
    out["dw"] = torch.matmul(z.t(), x) if c["layout"] == "vd" else torch.matmul(x.t(), z)
    if s["bias"] is not None:
        out["dbias"] = z.sum(0)
    return out


def _exact_distill_topk(s, c):
    tau = c["temperature"]
    logp = torch.log_softmax(s["z"].double() / tau, dim=1)
    lse = torch.logsumexp(s["z"].double() / tau, dim=1)
    ok = (s["index"] >= 0) & (s["index"] < c["vocab"])
    logq = (s["teacher"].double() / tau).masked_fill(~ok, -1e300)
    logq = torch.log_softmax(logq, dim=1)
    q = torch.where(ok, logq.exp(), 0.0)
    at = s["index"].clamp(0, c["vocab"] - 1)
    row_loss = tau ** 2 * torch.where(ok, q * (logq - logp.gather(1, at)), 0.0).sum(1)
    used = ok.any(1)
    n = max(1, int(used.sum()))
    dz = logp.exp_()
    dz.scatter_add_(1, at, -q)
    dz *= (used.double() * tau * s["up"].double() / n)[:, None]
    return {"loss": row_loss.sum().reshape(1) / n, "row_loss": row_loss, "lse": lse, "dz": dz}


def _exact_residual_norm(s, c):
    """The gradients by the chain rule on the definition, through torch's autograd in float64."""
    names = ["x", "u", "w_post", "w_pre"] + ([] if s["gate"] is None else ["gate"])
    v = {k: s[k].double().requires_grad_(c["train"]) for k in names}

    def norm(a):
        if c["kind"] == "layer":
            a = a - a.mean(1, keepdim=True)
        return a / torch.sqrt(a.pow(2).mean(1, keepdim=True) + _EPS)

    branch = norm(v["u"]) * v["w_post"]
    if s["gate"] is not None:
        branch = branch * (v["gate"][:, None] if c["gate"] == "token" else v["gate"])
    y = s["alpha"] * v["x"] + branch
    n = norm(y) * v["w_pre"]
    out = {"y": y.detach(), "n": n.detach()}
    if c["train"]:
        grads = torch.autograd.grad([y, n], [v[k] for k in names], [s["dy"].double(), s["dn"].double()])
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear_ce": _exact_linear_ce, "distill_topk": _exact_distill_topk,
            "residual_norm": _exact_residual_norm}[case["op"]](s, case)
