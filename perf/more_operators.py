"""A float recurrent layer's operators and the choice of the next token, in plain form and through the framework: what is
timed and compared.

Three operators, each in the forms a user calls: the gated linear recurrence h[t] = a[t] h[t-1] + (1 - a[t]) x[t] with
sigmoid gates (a prompt, a training step with every gradient, one new token a stream), the layer norm with the residual's
addition (a prompt, a training step), and sampling from logits with temperature, top-k, top-p and min-p by given random
numbers.

Sizes are those of this repository's configurations (d_model 256 / 768 / 1024, d_inner 512 / 1536 / 2048, vocabularies of
4096 and 32768, up to 256 streams, prompts of 256 to 2048 tokens), long sequences, and odd sizes between and around them.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
CELLS = 8 * 2048 * 1536    # positions x channels of the largest listed recurrence
NORM_CELLS = 16384 * 768   # and of the largest listed norm
LOGITS = 256 * 32768       # and of the largest listed choice


def _rec(form, dtype, batch, length, width, convex=True, gate=True, bias=True, carry=False, ragged=False):
    return {"op": "recurrence", "form": form, "dtype": dtype, "batch": batch, "length": length, "width": width,
            "convex": convex, "gate": gate, "bias": bias, "carry": carry, "ragged": ragged}


def _norm(form, dtype, rows, width, residual="none", bias=True):
    return {"op": "norm", "form": form, "dtype": dtype, "rows": rows, "width": width, "residual": residual, "bias": bias}


def _sample(dtype, rows, vocab, requests="mixed", spread=2.5, banned=False):
    return {"op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "requests": requests, "spread": spread,
            "banned": banned}


def listed():
    return [
        # a full decode batch, one token a stream: the states are read and written once
        dict(_rec("step", "bfloat16", 256, 1, 2048), name="recurrence_step_256x2048"),
        # one prompt alone, as a server admits it, continuing from a state: few channels, a serial axis
        dict(_rec("prompt", "bfloat16", 1, 2048, 1536, carry=True), name="recurrence_prompt_1x2048x1536"),
        # prompts of unequal lengths admitted together
        dict(_rec("prompt", "float16", 6, 777, 2048, carry=True, ragged=True), name="recurrence_prompt_ragged_6x777"),
        # a training step of the d_model 768 layer
        dict(_rec("train", "bfloat16", 8, 2048, 1536), name="recurrence_train_8x2048x1536"),
        # one long document, no output gate: the work lies along the sequence
        dict(_rec("train", "bfloat16", 1, 32768, 512, gate=False), name="recurrence_train_1x32768x512"),
        # a small fp32 training step with odd sizes and inputs that are not weighed by the gate
        dict(_rec("train", "float32", 2, 257, 509, convex=False, gate=False, bias=False, carry=True),
             name="recurrence_train_2x257x509"),
        # the norm of four streams' tokens: latency is all that counts
        dict(_norm("prompt", "float32", 4, 512), name="norm_4x512"),
        # residual + norm of a decode batch, the residual stream kept in fp32
        dict(_norm("prompt", "bfloat16", 256, 1024, residual="float32"), name="norm_256x1024"),
        # a training step's norm
        dict(_norm("train", "bfloat16", 16384, 768, residual="same"), name="norm_train_16384x768"),
        # the next tokens of four streams that all sample with every filter
        dict(_sample("float32", 4, 32768, requests="filtered"), name="sample_4x32768"),
        # a full decode batch, each request with settings of its own (greedy ones among them)
        dict(_sample("float32", 256, 32768), name="sample_256x32768"),
        # an odd vocabulary in 16 bits (many equal logits), a part of it banned
        dict(_sample("bfloat16", 64, 50021, requests="nucleus", banned=True), name="sample_64x50021"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "recurrence", "norm", "norm", "sample", "sample"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    yes = lambda p=0.5: rng.random() < p  # noqa: E731
    if op == "sample":
        vocab = _spread(rng, 64, 131072)
        rows = max(1, min(_spread(rng, 1, 256), LOGITS // vocab))
        return _sample(dtype if yes() else "float32", rows, vocab, requests=rng.choice(["mixed", "filtered", "nucleus", "plain"]),
                       spread=rng.choice([0.5, 2.5, 2.5, 5.0]), banned=yes(0.3))
    width = _spread(rng, 64, 4096)
    if yes(0.6):
        width = max(64, width // 64 * 64)
    if op == "norm":
        form = rng.choice(["prompt", "train"])
        rows = max(1, min(_spread(rng, 1, 32768), NORM_CELLS // width))
        return _norm(form, dtype, rows, width, residual=rng.choice(["none", "same", "float32"]), bias=yes(0.8))
    form = rng.choice(["step", "prompt", "prompt", "train", "train"])
    batch = _spread(rng, 1, 256) if form == "step" else _spread(rng, 1, 32)
    length = 1 if form == "step" else _spread(rng, 1, 32768)
    length = max(1, min(length, CELLS // (batch * width)))
    return _rec(form, dtype, batch, length, width, convex=yes(0.7), gate=yes(), bias=yes(0.7), carry=yes(),
                ragged=form != "step" and yes(0.3))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _settings(case, g, dev):
    """Each row's temperature, k, p and min_p, as the requests of a server have them: [rows] tensors."""
    m, kind = case["rows"], case["requests"]
    rand = lambda: torch.rand(m, generator=g, device=dev)  # noqa: E731
    t = 0.5 + rand()
    off_k, off_p = torch.zeros(m, device=dev, dtype=torch.int32), torch.ones(m, device=dev)
    k = torch.exp(rand() * math.log(min(1000, case["vocab"]))).int().clamp(min=1)
    p, min_p = 0.5 + 0.49 * rand(), 0.2 * rand()
    if kind == "plain":
        return t, off_k, off_p, torch.zeros_like(t)
    if kind == "nucleus":
        return t, off_k, p, torch.zeros_like(t)
    if kind == "filtered":
        return t, k, p, 0.1 * min_p
    some = lambda: rand() < 0.5  # noqa: E731
    return (torch.where(rand() < 0.15, torch.zeros_like(t), t), torch.where(some(), k, off_k),
            torch.where(some(), p, off_p), torch.where(some(), min_p, torch.zeros_like(t)))


def _lengths(g, batch, length, dev):
    """Right-padded batches: any length from 0 on, the first sequence full."""
    n = torch.randint(0, length + 1, (batch,), generator=g, device=dev, dtype=torch.int32)
    n[0] = length
    return n


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, generator=g, device=dev)  # noqa: E731
    train = case.get("form") == "train"
    leaf = lambda t: t.requires_grad_(True) if train else t  # noqa: E731
    s = {"case": case}
    if case["op"] == "sample":
        m, v = case["rows"], case["vocab"]
        logits = case["spread"] * randn(m, v)
        # a model is sure of some of its tokens: a few dozen stand out
        logits = torch.where(rand(m, v) < 48 / v, 4 + 10 * rand(m, v), logits)
        if case["banned"]:
            logits.masked_fill_(rand(m, v) < 0.2, float("-inf"))
            logits[:, 0] = 0.0
        s["logits"] = logits.to(dt)
        s["u"] = rand(m)
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = _settings(case, g, dev)
        return s
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        s["x"] = leaf((randn(n, d) + 0.5 * randn(n, 1)).to(dt))
        s["weight"] = leaf(1 + 0.1 * randn(d))
        s["bias"] = leaf(0.1 * randn(d)) if case["bias"] else None
        s["residual"] = None
        if case["residual"] != "none":
            s["residual"] = leaf((3 * randn(n, d)).to(dt if case["residual"] == "same" else torch.float32))
        if train:
            s["dy"] = randn(n, d).to(dt)
            s["dsum"] = None if s["residual"] is None else randn(n, d).to(s["residual"].dtype)
        return s
    b, n, d = case["batch"], case["length"], case["width"]
    # the gates' biases give the channels memories of 2 to 1000 positions
    bias = torch.log(torch.exp(math.log(2) + rand(d) * math.log(500)) - 1)
    lead = (b,) if case["form"] == "step" else (b, n)
    s["bias"] = leaf(bias) if case["bias"] else None
    gate = randn(*lead, d) if case["bias"] else randn(*lead, d) + bias
    s["lengths"] = _lengths(g, b, n, dev) if case["ragged"] else None
    if train:
        s["x"], s["f"] = leaf(randn(b, n, d).to(dt)), leaf(gate.to(dt))
        s["z"] = leaf(randn(b, n, d).to(dt)) if case["gate"] else None
    else:
        # columns of one projection's rows: [x | f | z]
        wide = torch.cat([randn(*lead, d), gate] + ([randn(*lead, d)] if case["gate"] else []), -1).to(dt)
        s["x"], s["f"] = wide[..., :d], wide[..., d:2 * d]
        s["z"] = wide[..., 2 * d:] if case["gate"] else None
    if case["form"] == "step":
        s["h"] = randn(b, d)
        return s
    s["h0"] = leaf(randn(b, d)) if case["carry"] else None
    if train:
        s["dy"] = randn(b, n, d).to(dt)
        s["dh"] = randn(b, d) if case["carry"] else None
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _f(t):
    return None if t is None else t.detach().float()


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dim 1 with h[-1] = 0: each pass doubles the span that a position has summed."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], torch.addcmul(b[:, span:], a[:, span:], b[:, :-span])], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _gates(s):
    """a and the weight of the input: 1 - a, taken from the other side so that it keeps its digits where a is near 1."""
    f = _f(s["f"])
    if s["bias"] is not None:
        f = f + _f(s["bias"])
    a, rest = 1 / (1 + torch.exp(-f)), 1 / (1 + torch.exp(f))
    return a, rest, rest if s["case"]["convex"] else torch.ones_like(a)


def _inside(s):
    """[batch, length, 1]: which positions lie before the sequence's end (None: all)."""
    if s["lengths"] is None:
        return None
    return (torch.arange(s["case"]["length"], device=s["lengths"].device) < s["lengths"].unsqueeze(1)).unsqueeze(2)


def _recurrence_plain(s):
    c, dt = s["case"], s["x"].dtype
    x, z = _f(s["x"]), _f(s["z"])
    a, rest, weight = _gates(s)
    inside = _inside(s)
    if inside is not None:
        a, weight = torch.where(inside, a, 1), torch.where(inside, weight, 0)
    b = weight * x
    first = b[:, :1] if s["h0"] is None else b[:, :1] + a[:, :1] * _f(s["h0"]).unsqueeze(1)
    h = _recurrence(a, torch.cat([first, b[:, 1:]], 1))
    sig = None if z is None else 1 / (1 + torch.exp(-z))
    y = h if z is None else h * z * sig
    if inside is not None:
        y = torch.where(inside, y, 0)
    answer = {"y": y.to(dt), "h": h[:, -1].clone()}
    if c["form"] != "train":
        return answer
    dy = _f(s["dy"])
    if inside is not None:
        dy = torch.where(inside, dy, 0)
    q = dy.clone() if z is None else dy * z * sig
    if s["dh"] is not None:
        q[:, -1] += s["dh"]
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _recurrence(later.flip(1), q.flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]) if s["h0"] is None else _f(s["h0"]).unsqueeze(1), h[:, :-1]], 1)
    df = g * (before - x if c["convex"] else before) * a * rest
    if inside is not None:
        df = torch.where(inside, df, 0)
    grads = {"x": (weight * g).to(dt), "f": df.to(dt)}
    if z is not None:
        grads["z"] = (dy * h * sig * (1 + z * (1 - sig))).to(dt)
    if s["bias"] is not None:
        grads["bias"] = df.sum((0, 1))
    if s["h0"] is not None:
        grads["h0"] = a[:, 0] * g[:, 0]
    return dict(answer, grads=grads)


def _recurrence_step_plain(s):
    a, _, weight = _gates(s)
    h = a * s["h"] + weight * _f(s["x"])
    s["h"].copy_(h)
    if s["z"] is not None:
        z = _f(s["z"])
        h = h * z / (1 + torch.exp(-z))
    return {"y": h.to(s["x"].dtype), "h": s["h"]}


EPS = 1e-5


def _norm_plain(s):
    c, dt = s["case"], s["x"].dtype
    x, w, bias, r = (_f(s[k]) for k in ("x", "weight", "bias", "residual"))
    answer = {}
    if r is not None:
        answer["sum"] = (x + r).to(s["residual"].dtype)  # the residual stream as it is kept, and as it is normed
        x = answer["sum"].float()
    x = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    xhat = x * rstd
    y = xhat * w if bias is None else xhat * w + bias
    answer["y"] = y.to(dt)
    if c["form"] != "train":
        return answer
    dy = _f(s["dy"])
    wdy = w * dy
    dx = rstd * (wdy - wdy.mean(1, keepdim=True) - xhat * (wdy * xhat).mean(1, keepdim=True))
    grads = {"weight": (dy * xhat).sum(0)}
    if bias is not None:
        grads["bias"] = dy.sum(0)
    if r is not None:
        dx = dx + _f(s["dsum"])
        grads["residual"] = dx.to(s["residual"].dtype)
    grads["x"] = dx.to(dt)
    return dict(answer, grads=grads)


def _sample_plain(s):
    logits = s["logits"].double()  # the borders between tokens are sharp: 64 bits
    u, t, p, min_p = (s[k].double().unsqueeze(1) for k in ("u", "temperature", "top_p", "min_p"))
    k = s["top_k"].long().unsqueeze(1)
    v = logits.shape[1]
    most, best = logits.max(1, keepdim=True)
    weight = torch.exp((logits - most) / torch.where(t > 0, t, 1))
    # sorted downwards, equal logits by their index
    _, order = torch.sort(logits, dim=1, descending=True, stable=True)
    sorted_weight = weight.gather(1, order)
    rank = torch.arange(v, device=logits.device).unsqueeze(0)
    keep = rank < torch.where(k > 0, k, v)
    mass = torch.where(keep, sorted_weight, 0)
    before = torch.cumsum(mass, 1) - mass
    keep &= (before < p * mass.sum(1, keepdim=True)) | (rank == 0) | (p >= 1)
    keep &= sorted_weight >= min_p
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    upto = torch.cumsum(torch.where(kept, weight, 0), 1)
    token = (upto <= u * upto[:, -1:]).sum(1, keepdim=True)
    # the first index of the maximum where the temperature is 0
    first = (logits == most).long().argmax(1, keepdim=True)
    prob = torch.where(t > 0, weight.gather(1, token) / upto[:, -1:], 1)
    return {"token": torch.where(t > 0, token, first).squeeze(1), "prob": prob.squeeze(1).float()}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _grads(s, names, outputs, givens):
    """The gradients of every leaf, by name."""
    names = [k for k in names if s.get(k) is not None]
    got = torch.autograd.grad(outputs, [s[k] for k in names], givens)
    return dict(zip(names, got))


def _recurrence_own(s):
    from mamba_integer_b200 import selective

    c = s["case"]
    if c["form"] == "step":
        y = selective.gated_recurrence_step(s["h"], s["x"], s["f"], z=s["z"], gate_bias=s["bias"], convex=c["convex"])
        return {"y": y, "h": s["h"]}
    y, h = selective.gated_recurrence(s["x"], s["f"], z=s["z"], gate_bias=s["bias"], convex=c["convex"], h0=s["h0"],
                                      lengths=s["lengths"], return_state=True)
    if c["form"] != "train":
        return {"y": y, "h": h}
    outs, givens = ([y], [s["dy"]]) if s["dh"] is None else ([y, h], [s["dy"], s["dh"]])
    return {"y": y, "h": h, "grads": _grads(s, ("x", "f", "z", "bias", "h0"), outs, givens)}


def _norm_own(s):
    from mamba_integer_b200 import selective

    y, total = selective.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, residual=s["residual"])
    answer = {"y": y} if total is None else {"y": y, "sum": total}
    if s["case"]["form"] != "train":
        return answer
    outs, givens = ([y], [s["dy"]]) if total is None else ([y, total], [s["dy"], s["dsum"]])
    return dict(answer, grads=_grads(s, ("x", "weight", "bias", "residual"), outs, givens))


def _sample_own(s):
    from mamba_integer_b200 import kernels

    token, prob = kernels.sample_rows(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                      top_p=s["top_p"], min_p=s["min_p"], return_prob=True)
    return {"token": token, "prob": prob}


def run(state):
    op, form = state["case"]["op"], state["case"].get("form")
    if own:
        return {"recurrence": _recurrence_own, "norm": _norm_own, "sample": _sample_own}[op](state)
    if op == "recurrence":
        return _recurrence_step_plain(state) if form == "step" else _recurrence_plain(state)
    return _norm_plain(state) if op == "norm" else _sample_plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = DTYPES[case["dtype"]].itemsize
    if case["op"] == "sample":  # the logits, four settings and a random number a row in; a token and its share out
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * e + case["rows"] * 32, "flops": 4 * cells}
    if case["op"] == "norm":
        cells, d = case["rows"] * case["width"], case["width"]
        r = {"none": 0, "same": e, "float32": 4}[case["residual"]]
        params = 4 * d * (1 + case["bias"])
        if case["form"] == "prompt":  # x, the residual in; y, the sum out
            return {"bytes": cells * (2 * e + 2 * r) + params, "flops": 8 * cells}
        # and dy, the sum's gradient in; the gradients out
        return {"bytes": cells * (4 * e + 4 * r) + 2 * params, "flops": 22 * cells}
    b, n, d = case["batch"], case["length"], case["width"]
    cells, wide = b * n * d, 2 + case["gate"]
    bias, state = 4 * d * case["bias"], 4 * b * d * (2 if case["carry"] or case["form"] == "step" else 1)
    moved, flops = cells * (wide + 1) * e + bias + state, cells * (8 + 5 * case["gate"])
    if case["form"] == "train":  # dy in; dx, df, dz and the parameters' gradients out
        moved += cells * (wide + 1) * e + bias + (8 * b * d if case["carry"] else 0)
        flops += cells * (14 + 8 * case["gate"])
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _d(t):
    return None if t is None else t.detach().double()


def _recurrence_exact(s):
    """Position by position; the gradients by the chain rule, backwards."""
    c = s["case"]
    step, train = c["form"] == "step", c["form"] == "train"
    x, f, z, bias = (_d(s[k]) for k in ("x", "f", "z", "bias"))
    if step:
        x, f, z = (None if t is None else t.unsqueeze(1) for t in (x, f, z))
    f = f if bias is None else f + bias
    b, n, d = x.shape
    a, weight = torch.sigmoid(f), torch.sigmoid(-f) if c["convex"] else torch.ones_like(f)
    live = torch.ones(b, n, 1, dtype=torch.bool, device=x.device)
    if s["lengths"] is not None:
        live = (torch.arange(n, device=x.device)[None] < s["lengths"][:, None])[..., None]
    keep, add = torch.where(live, a, 1.0), torch.where(live, weight * x, 0.0)
    start = s["h"] if step else s["h0"]
    h = torch.zeros(b, d, dtype=torch.float64, device=x.device) if start is None else _d(start)
    states = torch.empty(b, n + 1, d, dtype=torch.float64, device=x.device)
    states[:, 0] = h
    for t in range(n):
        torch.addcmul(add[:, t], keep[:, t], states[:, t], out=states[:, t + 1])
    gate = torch.ones_like(x) if z is None else z * torch.sigmoid(z)
    y = torch.where(live, states[:, 1:] * gate, 0.0)
    answer = {"y": y[:, 0] if step else y, "h": states[:, n].clone()}
    if not train:
        return answer
    dy = torch.where(live, _d(s["dy"]), 0.0)
    g = dy * gate
    flow = torch.zeros(b, d, dtype=torch.float64, device=x.device) if s["dh"] is None else _d(s["dh"])
    for t in reversed(range(n)):
        g[:, t] += flow
        flow = keep[:, t] * g[:, t]
    through = torch.where(live, g, 0.0)
    slope = torch.sigmoid(f) * torch.sigmoid(-f)
    df = through * slope * (states[:, :n] - x if c["convex"] else states[:, :n])
    grads = {"x": through * weight, "f": df}
    if z is not None:
        sig = torch.sigmoid(z)
        grads["z"] = dy * states[:, 1:] * (sig + z * sig * (1 - sig))
    if bias is not None:
        grads["bias"] = df.sum((0, 1))
    if s["h0"] is not None:
        grads["h0"] = flow
    return dict(answer, grads=grads)


def _norm_exact(s):
    train = s["case"]["form"] == "train"
    x, w, bias, r = (_d(s[k]) for k in ("x", "weight", "bias", "residual"))
    answer = {}
    if r is not None:
        answer["sum"] = x + r
        # the operator norms the sum as it is kept: its rounding is part of the definition
        x = (s["x"].detach().float() + s["residual"].detach().float()).to(s["residual"].dtype).double()
    leaves = [t.clone().requires_grad_(train) for t in (x, w) + (() if bias is None else (bias,))]
    x = leaves[0]
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + EPS) * leaves[1]
    if bias is not None:
        y = y + leaves[2]
    answer["y"] = y.detach()
    if not train:
        return answer
    got = torch.autograd.grad(y, leaves, _d(s["dy"]))
    grads = {"weight": got[1]}
    if bias is not None:
        grads["bias"] = got[2]
    grads["x"] = got[0]
    if r is not None:
        grads["x"] = grads["residual"] = got[0] + _d(s["dsum"])
    return dict(answer, grads=grads)


def _sample_exact(s):
    """Row by row over the tokens that are left after each filter."""
    rows = s["logits"].double().cpu().numpy()
    u, t, p, min_p = (s[k].double().cpu().tolist() for k in ("u", "temperature", "top_p", "min_p"))
    ks = s["top_k"].cpu().tolist()
    tokens, probs = [], []
    for row, u_, t_, p_, m_, k_ in zip(rows, u, t, p, min_p, ks):
        best = int(np.argmax(row))
        if not t_ > 0:
            tokens.append(best)
            probs.append(1.0)
            continue
        left = np.lexsort((np.arange(row.size), -row))  # downwards, equal ones by index
        left = left[np.isfinite(row[left])]
        if 0 < k_ < left.size:
            left = left[:k_]
        mass = np.exp((row[left] - row[best]) / t_)
        if p_ < 1:
            count = int(np.searchsorted(np.cumsum(mass), p_ * mass.sum(), side="left")) + 1
            left, mass = left[:count], mass[:count]
        ok = mass >= m_
        left, mass = left[ok], mass[ok]
        by_index = np.argsort(left)
        left, mass = left[by_index], mass[by_index]
        upto = np.cumsum(mass)
        at = min(np.searchsorted(upto, u_ * upto[-1], side="right"), left.size - 1)
        tokens.append(int(left[at]))
        probs.append(float(mass[at] / upto[-1]))
    dev = s["logits"].device
    return {"token": torch.tensor(tokens, device=dev), "prob": torch.tensor(probs, dtype=torch.float64, device=dev)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"recurrence": _recurrence_exact, "norm": _norm_exact, "sample": _sample_exact}[case["op"]](s)
