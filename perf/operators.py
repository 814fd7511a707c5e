"""The float Mamba layer's operators, in plain form and through the framework: what is timed and compared.

Three operators, each in the forms a user calls: the selective scan with exponential decays, the short causal
convolution, and the RMS norm with the residual's addition (with a floating or an int8 output).  Forms: a prompt
("prompt"), a training step with every gradient ("train"), one new token a stream ("step"), and for the norm an int8
output for the ternary projections ("quant").

Sizes are those of this repository's configurations (d_model 256 / 768 / 1024, d_inner 512 / 1536 / 2048, 16 states, up to
256 streams, prompts of 256 to 2048 tokens) and odd ones between and around them.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LARGEST = 8 * 2048 * 1536  # positions x channels of the largest listed case


def _case(op, form, dtype, batch, length, width, **more):
    c = {"op": op, "form": form, "dtype": dtype, "batch": batch, "length": length, "width": width}
    c.update(more)
    return c


def _scan(form, dtype, batch, length, width, states=16, gate=True, skip=True, softplus=True, carry=False, ragged=False):
    return _case("scan", form, dtype, batch, length, width, states=states, gate=gate, skip=skip, softplus=softplus,
                 carry=carry, ragged=ragged)


def _conv(form, dtype, batch, length, width, taps=4, silu=True, bias=True, carry=False, ragged=False):
    return _case("conv", form, dtype, batch, length, width, taps=taps, silu=silu, bias=bias, carry=carry, ragged=ragged)


def _norm(form, dtype, rows, width, residual="same"):
    return _case("norm", form, dtype, 1, rows, width, residual=residual)


def listed():
    return [
        # the layer's three operators for the tokens of four streams: latency is all that counts
        dict(_scan("step", "float32", 4, 1, 512), name="scan_step_4x512"),
        # a full decode batch: the states are read and written once
        dict(_scan("step", "bfloat16", 256, 1, 2048), name="scan_step_256x2048"),
        # one prompt alone, as a server admits it: few channels, a long serial axis
        dict(_scan("prompt", "bfloat16", 1, 2048, 1536, carry=True), name="scan_prompt_1x2048x1536"),
        # prompts of unequal lengths admitted together, continuing from given states
        dict(_scan("prompt", "float16", 6, 777, 2048, carry=True, ragged=True), name="scan_prompt_ragged_6x777"),
        # a training step of the d_model 768 layer
        dict(_scan("train", "bfloat16", 8, 2048, 1536), name="scan_train_8x2048x1536"),
        # a small fp32 training step with odd sizes (no gate, 24 states)
        dict(_scan("train", "float32", 2, 257, 509, states=24, gate=False, carry=True), name="scan_train_2x257x509"),
        # the convolution of a decode batch
        dict(_conv("step", "bfloat16", 256, 1, 2048), name="conv_step_256x2048"),
        # and of a training step
        dict(_conv("train", "bfloat16", 8, 2048, 1536), name="conv_train_8x2048x1536"),
        # prompts of unequal lengths with their windows
        dict(_conv("prompt", "float16", 6, 777, 2048, carry=True, ragged=True), name="conv_prompt_ragged_6x777"),
        # residual + norm + int8 rows in front of a projection, decode batch
        dict(_norm("quant", "bfloat16", 256, 1024, residual="float32"), name="norm_quant_256x1024"),
        # the same over a prefill batch
        dict(_norm("quant", "bfloat16", 32768, 768), name="norm_quant_32768x768"),
        # a training step's norm
        dict(_norm("train", "bfloat16", 16384, 768), name="norm_train_16384x768"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "conv", "conv", "norm", "norm"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    width = _spread(rng, 64, 4096)
    if rng.random() < 0.6:
        width = max(64, width // 64 * 64)
    yes = lambda p=0.5: rng.random() < p  # noqa: E731
    if op == "norm":
        form = rng.choice(["prompt", "train", "quant"])
        rows = min(_spread(rng, 1, 32768), LARGEST // width)
        return _norm(form, dtype, rows, width, residual=rng.choice(["none", "same", "float32"]))
    form = rng.choice(["step", "prompt", "prompt", "train", "train"])
    batch = _spread(rng, 1, 256) if form == "step" else _spread(rng, 1, 32)
    length = 1 if form == "step" else _spread(rng, 1, 4096)
    if op == "conv":
        length = max(1, min(length, LARGEST // (batch * width)))
        return _conv(form, dtype, batch, length, width, taps=rng.choice([4, 4, 4, 3, 2]), silu=yes(0.8), bias=yes(0.8),
                     carry=yes(), ragged=form != "step" and yes(0.3))
    states = rng.choice([16, 16, 16, 8, 32, 64, rng.randint(1, 64)])
    # no more state updates than the largest listed case
    length = max(1, min(length, LARGEST // 2 * 16 // (batch * width * max(states, 16))))
    return _scan(form, dtype, batch, length, width, states=states, gate=yes(0.7), skip=yes(0.7), softplus=yes(0.8),
                 carry=yes(), ragged=form != "step" and yes(0.3))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(g, batch, length, dev):
    """Right-padded batches: any length from 0 on, the first sequence full."""
    n = torch.randint(0, length + 1, (batch,), generator=g, device=dev, dtype=torch.int32)
    n[0] = length
    return n


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    b, n, d = case["batch"], case["length"], case["width"]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, generator=g, device=dev)  # noqa: E731
    train = case["form"] == "train"
    leaf = lambda t: t.requires_grad_(True) if train else t  # noqa: E731
    s = {"case": case}
    if case["op"] == "norm":
        s["x"] = leaf(randn(n, d).to(dt))
        s["weight"] = leaf(1 + 0.1 * randn(d))
        s["residual"] = None
        if case["residual"] != "none":
            s["residual"] = leaf((3 * randn(n, d)).to(dt if case["residual"] == "same" else torch.float32))
        if train:
            s["dy"] = randn(n, d).to(dt)
            s["dsum"] = None if s["residual"] is None else randn(n, d).to(s["residual"].dtype)
        return s
    if case["op"] == "conv":
        taps = case["taps"]
        s["w"] = leaf((rand(d, taps) - 0.5))
        s["bias"] = leaf(rand(d) - 0.5) if case["bias"] else None
        s["lengths"] = _lengths(g, b, n, dev) if case["ragged"] else None
        if case["form"] == "step":
            # the x half of the input projection's rows
            s["x"] = randn(b, 2 * d).to(dt)[:, :d]
            s["win"] = randn(b, taps - 1, d).to(dt)
            return s
        # the x half of the input projection's rows; a training step's leaf stands alone
        s["x"] = leaf(randn(b, n, d).to(dt)) if train else randn(b, n, 2 * d).to(dt)[:, :, :d]
        s["win"] = leaf(randn(b, taps - 1, d).to(dt)) if case["carry"] else None
        if train:
            s["dy"] = randn(b, n, d).to(dt)
            s["dwin"] = randn(b, taps - 1, d).to(dt) if case["carry"] else None
        return s
    k = case["states"]
    # decays of the usual initialisation: A = -(1 .. N) varied a little, dt between 1e-3 and 1e-1
    s["A"] = leaf(-(torch.arange(1, k + 1, device=dev).float().expand(d, k) * torch.exp(0.2 * randn(d, k))).contiguous())
    dt0 = torch.exp(rand(d) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    s["D"] = leaf(1 + 0.1 * randn(d)) if case["skip"] else None
    s["lengths"] = _lengths(g, b, n, dev) if case["ragged"] else None
    lead = (b,) if case["form"] == "step" else (b, n)
    s["u"] = leaf(randn(*lead, d).to(dt))
    if case["softplus"]:
        s["bias"] = leaf(dt0 + torch.log(-torch.expm1(-dt0)))
        s["delta"] = leaf(randn(*lead, d).to(dt))
    else:
        s["bias"] = None
        s["delta"] = leaf((dt0 * torch.exp(0.5 * randn(*lead, d))).to(dt))
    if train:
        s["B"], s["C"] = leaf(randn(*lead, k).to(dt)), leaf(randn(*lead, k).to(dt))
        s["z"] = leaf(randn(*lead, d).to(dt)) if case["gate"] else None
    else:
        # columns of the projections' rows: [dt | B | C] and [x | z]
        pad = 48
        rows = randn(*lead, pad + 2 * k).to(dt)
        s["B"], s["C"] = rows[..., pad:pad + k], rows[..., pad + k:]
        s["z"] = randn(*lead, 2 * d).to(dt)[..., d:] if case["gate"] else None
    if case["form"] == "step":
        s["h"] = randn(b, d, k)
        return s
    s["h0"] = leaf(randn(b, d, k)) if case["carry"] else None
    if train:
        s["dy"] = randn(b, n, d).to(dt)
        s["dh"] = randn(b, d, k) if case["carry"] else None
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


def _step_sizes(s):
    raw = _f(s["delta"])
    if s["bias"] is not None:
        raw = raw + _f(s["bias"])
    if not s["case"]["softplus"]:
        return raw, raw
    return raw, torch.clamp(raw, min=0) + torch.log1p(torch.exp(-torch.abs(raw)))


def _inside(s):
    """[batch, length, 1]: which positions lie before the sequence's end (None: all)."""
    if s["lengths"] is None:
        return None
    return (torch.arange(s["case"]["length"], device=s["lengths"].device) < s["lengths"].unsqueeze(1)).unsqueeze(2)


def _scan_plain(s):
    c, dt_ = s["case"], s["u"].dtype
    train = c["form"] == "train"
    u, A, B, C, D, z = (_f(s[k]) for k in ("u", "A", "B", "C", "D", "z"))
    raw, dt = _step_sizes(s)
    inside = _inside(s)
    if inside is not None:
        dt = torch.where(inside, dt, 0)
    a = torch.exp(dt.unsqueeze(3) * A)
    b = (dt * u).unsqueeze(3) * B.unsqueeze(2)
    first = a[:, :1] * _f(s["h0"]).unsqueeze(1) if s["h0"] is not None else torch.zeros_like(b[:, :1])
    h = _recurrence(a, torch.cat([b[:, :1] + first, b[:, 1:]], 1))
    del b
    y = torch.einsum("btdn,btn->btd", h, C) if not train else (h * C.unsqueeze(2)).sum(3)
    if D is not None:
        y = y + D * u
    sig = None if z is None else 1 / (1 + torch.exp(-z))
    out = y if z is None else y * z * sig
    if inside is not None:
        out = torch.where(inside, out, 0)
    answer = {"y": out.to(dt_), "h": h[:, -1].clone()}
    if not train:
        return answer
    dy = _f(s["dy"])
    if inside is not None:
        dy = torch.where(inside, dy, 0)
    ds = dy if z is None else dy * z * sig
    q = ds.unsqueeze(3) * C.unsqueeze(2)
    if s["dh"] is not None:
        q[:, -1] += s["dh"]
    # the adjoint of h runs backwards, with the decays one position on
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _recurrence(later.flip(1), q.flip(1)).flip(1)
    del q, later
    before = torch.cat([torch.zeros_like(h[:, :1]) if s["h0"] is None else _f(s["h0"]).unsqueeze(1), h[:, :-1]], 1)
    dC = (ds.unsqueeze(3) * h).sum(2)
    dB = (g * (dt * u).unsqueeze(3)).sum(2)
    along = (g * B.unsqueeze(2)).sum(3)
    du = dt * along if D is None else dt * along + D * ds
    w = g * a * before
    ddt = u * along + (w * A).sum(3)
    dA = (w * dt.unsqueeze(3)).sum((0, 1))
    draw_ = ddt / (1 + torch.exp(-raw)) if c["softplus"] else ddt
    if inside is not None:
        draw_ = torch.where(inside, draw_, 0)
    grads = {"u": du.to(dt_), "delta": draw_.to(dt_), "A": dA, "B": dB.to(dt_), "C": dC.to(dt_)}
    if D is not None:
        grads["D"] = (ds * u).sum((0, 1))
    if z is not None:
        grads["z"] = (dy * y * sig * (1 + z * (1 - sig))).to(dt_)
    if s["bias"] is not None:
        grads["bias"] = draw_.sum((0, 1))
    if s["h0"] is not None:
        grads["h0"] = a[:, 0] * g[:, 0]
    return dict(answer, grads=grads)


def _scan_step_plain(s):
    u, A, B, C, D, z = (_f(s[k]) for k in ("u", "A", "B", "C", "D", "z"))
    _, dt = _step_sizes(s)
    h = torch.exp(dt.unsqueeze(2) * A) * s["h"] + (dt * u).unsqueeze(2) * B.unsqueeze(1)
    s["h"].copy_(h)
    y = (h * C.unsqueeze(1)).sum(2)
    if D is not None:
        y = y + D * u
    if z is not None:
        y = y * z / (1 + torch.exp(-z))
    return {"y": y.to(s["u"].dtype), "h": s["h"]}


def _padded(x, win, taps):
    front = torch.zeros_like(x[:, :1]).expand(-1, taps - 1, -1) if win is None else win
    return torch.cat([front, x], 1)


def _conv_plain(s):
    c, dt_ = s["case"], s["x"].dtype
    taps, n = c["taps"], c["length"]
    x, w, bias, win = (_f(s[k]) for k in ("x", "w", "bias", "win"))
    inside = _inside(s)
    row = _padded(x, win, taps)
    pieces = row.unfold(1, taps, 1)  # [batch, length, width, taps]
    pre = (pieces * w).sum(3)
    if bias is not None:
        pre = pre + bias
    sig = 1 / (1 + torch.exp(-pre)) if c["silu"] else None
    y = pre * sig if c["silu"] else pre
    if inside is not None:
        y = torch.where(inside, y, 0)
    last = torch.full((c["batch"],), n, device=x.device) if s["lengths"] is None else s["lengths"].long()
    at = (last.unsqueeze(1) + torch.arange(taps - 1, device=x.device)).unsqueeze(2).expand(-1, -1, x.shape[2])
    answer = {"y": y.to(dt_), "win": row.gather(1, at).to(dt_)}
    if c["form"] != "train":
        return answer
    dy = _f(s["dy"])
    if inside is not None:
        dy = torch.where(inside, dy, 0)
    dp = dy * sig * (1 + pre * (1 - sig)) if c["silu"] else dy
    # what each place of `row` gets: from the taps that read it, and from the window that leaves
    edge = torch.zeros_like(dp[:, :1]).expand(-1, taps - 1, -1)
    drow = (torch.cat([edge, dp, edge], 1).unfold(1, taps, 1) * w.flip(1)).sum(3)
    if s["dwin"] is not None:
        drow = drow.scatter_add(1, at, _f(s["dwin"]))
    grads = {"x": drow[:, taps - 1:].to(dt_), "w": (dp.unsqueeze(3) * pieces).sum((0, 1))}
    if bias is not None:
        grads["bias"] = dp.sum((0, 1))
    if win is not None:
        grads["win"] = drow[:, :taps - 1].to(dt_)
    return dict(answer, grads=grads)


def _conv_step_plain(s):
    x, w, bias, win = (_f(s[k]) for k in ("x", "w", "bias", "win"))
    row = torch.cat([win, x.unsqueeze(1)], 1)
    y = (row * w.t()).sum(1)
    if bias is not None:
        y = y + bias
    if s["case"]["silu"]:
        y = y / (1 + torch.exp(-y))
    s["win"].copy_(row[:, 1:])
    return {"y": y.to(s["x"].dtype), "win": s["win"]}


EPS = 1e-6


def _norm_plain(s):
    c, dt_ = s["case"], s["x"].dtype
    x, w, r = (_f(s[k]) for k in ("x", "weight", "residual"))
    answer = {}
    if r is not None:
        answer["sum"] = (x + r).to(s["residual"].dtype)  # the residual stream as it is kept, and as it is normed
        x = answer["sum"].float()
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    y = x * rstd * w
    if c["form"] == "quant":
        most = torch.clamp(y.abs().amax(1, keepdim=True), min=1e-8)
        q = torch.round(y / most * 127)
        return dict(answer, values=(q * (most / 127)).to(torch.bfloat16), scale=(most / 127).squeeze(1))
    answer["y"] = y.to(dt_)
    if c["form"] != "train":
        return answer
    dy = _f(s["dy"])
    xhat = x * rstd
    wdy = w * dy
    dx = rstd * (wdy - xhat * (wdy * xhat).mean(1, keepdim=True))
    grads = {"weight": (dy * xhat).sum(0)}
    if r is not None:
        dx = dx + _f(s["dsum"])
        grads["residual"] = dx.to(s["residual"].dtype)
    grads["x"] = dx.to(dt_)
    return dict(answer, grads=grads)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _grads(s, names, outputs, givens):
    """The gradients of every leaf, by name."""
    names = [k for k in names if s.get(k) is not None]
    got = torch.autograd.grad(outputs, [s[k] for k in names], givens)
    return dict(zip(names, got))


def _scan_own(s):
    from mamba_integer_b200 import selective

    c = s["case"]
    if c["form"] == "step":
        y = selective.selective_scan_step(s["h"], s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                          delta_bias=s["bias"], delta_softplus=c["softplus"])
        return {"y": y, "h": s["h"]}
    y, h = selective.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                    delta_bias=s["bias"], delta_softplus=c["softplus"], h0=s["h0"],
                                    lengths=s["lengths"], return_state=True)
    if c["form"] != "train":
        return {"y": y, "h": h}
    outs, givens = ([y], [s["dy"]]) if s["dh"] is None else ([y, h], [s["dy"], s["dh"]])
    grads = _grads(s, ("u", "delta", "A", "B", "C", "D", "z", "bias", "h0"), outs, givens)
    return {"y": y, "h": h, "grads": grads}


def _conv_own(s):
    from mamba_integer_b200 import selective

    c = s["case"]
    if c["form"] == "step":
        y = selective.causal_conv1d_step(s["x"], s["w"], s["win"], bias=s["bias"], silu=c["silu"])
        return {"y": y, "win": s["win"]}
    y, win = selective.causal_conv1d(s["x"], s["w"], bias=s["bias"], silu=c["silu"], win=s["win"],
                                     lengths=s["lengths"], return_window=True)
    if c["form"] != "train":
        return {"y": y, "win": win}
    outs, givens = ([y], [s["dy"]]) if s["dwin"] is None else ([y, win], [s["dy"], s["dwin"]])
    return {"y": y, "win": win, "grads": _grads(s, ("x", "w", "bias", "win"), outs, givens)}


def _norm_own(s):
    from mamba_integer_b200 import selective

    c = s["case"]
    if c["form"] == "quant":
        q, scale, total = selective.rms_norm_quant(s["x"], s["weight"], eps=EPS, residual=s["residual"])
        values = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        torch.mul(q, scale.unsqueeze(1), out=values)
        answer = {"values": values, "scale": scale}
        return answer if total is None else dict(answer, sum=total)
    y, total = selective.rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"])
    answer = {"y": y} if total is None else {"y": y, "sum": total}
    if c["form"] != "train":
        return answer
    outs, givens = ([y], [s["dy"]]) if total is None else ([y, total], [s["dy"], s["dsum"]])
    return dict(answer, grads=_grads(s, ("x", "weight", "residual"), outs, givens))


def run(state):
    op, form = state["case"]["op"], state["case"]["form"]
    if own:
        return {"scan": _scan_own, "conv": _conv_own, "norm": _norm_own}[op](state)
    if op == "norm":
        return _norm_plain(state)
    if op == "conv":
        return _conv_step_plain(state) if form == "step" else _conv_plain(state)
    return _scan_step_plain(state) if form == "step" else _scan_plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = DTYPES[case["dtype"]].itemsize
    b, n, d = case["batch"], case["length"], case["width"]
    cells, form = b * n * d, case["form"]
    if case["op"] == "norm":
        r = {"none": 0, "same": e, "float32": 4}[case["residual"]]
        if form == "quant":  # x and the residual in; the sum, 8 bits a value and a scale a row out
            return {"bytes": cells * (e + 2 * r + 1) + 4 * n, "flops": 8 * cells}
        read = cells * (e + 2 * r + e)
        if form == "train":  # and dy, the sum's gradient in; the gradients out
            read += cells * (2 * e + 2 * r) + 4 * d
        return {"bytes": read, "flops": (6 if form == "prompt" else 16) * cells}
    if case["op"] == "conv":
        k = case["taps"]
        edge = b * (k - 1) * d * e
        moved = 2 * cells * e + 4 * d * (k + 1) + edge * (2 if case["carry"] or form == "step" else 1)
        if form == "train":
            moved += 2 * cells * e + 4 * d * (k + 1) + (2 * edge if case["carry"] else 0)
        return {"bytes": moved, "flops": cells * (2 * k + 6) * (3 if form == "train" else 1)}
    k = case["states"]
    wide = 3 + case["gate"]  # u, delta, y and z
    moved = cells * wide * e + 2 * b * n * k * e + 4 * d * (k + 2) + 4 * b * d * k * (2 if case["carry"] or form == "step" else 1)
    flops = cells * (7 * k + 16)  # a state: the decay's product and exp, the input's product, two multiply-adds
    if form == "train":  # dy in; du, ddelta, dz, dB, dC and the parameters' gradients out
        moved += cells * wide * e + 2 * b * n * k * e + 4 * d * (k + 2) + (8 * b * d * k if case["carry"] else 0)
        flops += cells * (24 * k + 32)
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, position by position
# ---------------------------------------------------------------------------
def _d(t):
    return None if t is None else t.detach().double()


def _silu64(v):
    """x sigmoid(x) and its derivative."""
    sig = torch.sigmoid(v)
    return v * sig, sig + v * sig * (1 - sig)


def _scan_exact(s):
    c = s["case"]
    u, A, B, C, D, z, raw = (_d(s[k]) for k in ("u", "A", "B", "C", "D", "z", "delta"))
    step = c["form"] == "step"
    if step:
        u, B, C, raw = (t.unsqueeze(1) for t in (u, B, C, raw))
        z = None if z is None else z.unsqueeze(1)
    if s["bias"] is not None:
        raw = raw + _d(s["bias"])
    dt = torch.logaddexp(raw, torch.zeros_like(raw)) if c["softplus"] else raw
    batch, n, d = u.shape
    k = A.shape[1]
    live = torch.ones(batch, n, device=u.device, dtype=torch.bool)
    if s["lengths"] is not None:
        live = torch.arange(n, device=u.device)[None] < s["lengths"][:, None]
    start = s["h"] if step else s["h0"]
    h = torch.zeros(batch, d, k, dtype=torch.float64, device=u.device) if start is None else _d(start)
    train = c["form"] == "train"
    kept, y = [], torch.zeros_like(u)
    for t in range(n):
        kept.append(h if train else None)
        new = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[..., None] * B[:, t, None, :]
        h = torch.where(live[:, t, None, None], new, h)
        y[:, t] = torch.matmul(h, C[:, t, :, None])[..., 0] + (0 if D is None else D * u[:, t])
    gate, slope = (1, 0) if z is None else _silu64(z)
    out = torch.where(live[..., None], y * gate, 0)
    answer = {"y": out[:, 0] if step else out, "h": h}
    if not train:
        return answer
    dy = torch.where(live[..., None], _d(s["dy"]), 0)
    ds = dy * gate
    g = torch.zeros_like(h) if s["dh"] is None else _d(s["dh"])
    du, ddt = torch.zeros_like(u), torch.zeros_like(u)
    dA, dB, dC = torch.zeros_like(A), torch.zeros_like(B), torch.zeros_like(C)
    for t in reversed(range(n)):
        now = live[:, t, None, None]
        a = torch.exp(dt[:, t, :, None] * A)
        new = a * kept[t] + (dt[:, t] * u[:, t])[..., None] * B[:, t, None, :]
        g = g + torch.where(now, ds[:, t, :, None] * C[:, t, None, :], 0)
        gl = torch.where(now, g, 0)
        dC[:, t] = torch.matmul(ds[:, t, None, :], torch.where(now, new, 0))[:, 0]
        dB[:, t] = torch.matmul((dt[:, t] * u[:, t])[:, None, :], gl)[:, 0]
        s1 = torch.matmul(gl, B[:, t, :, None])[..., 0]
        w = gl * a * kept[t]
        du[:, t] = dt[:, t] * s1
        ddt[:, t] = u[:, t] * s1 + (w * A).sum(2)
        dA += (w * dt[:, t, :, None]).sum(0)
        g = torch.where(now, a * g, g)
    draw_ = ddt * torch.sigmoid(raw) if c["softplus"] else ddt
    grads = {"u": du if D is None else du + D * ds, "delta": draw_, "A": dA, "B": dB, "C": dC}
    if D is not None:
        grads["D"] = (ds * u).sum((0, 1))
    if z is not None:
        grads["z"] = dy * y * slope
    if s["bias"] is not None:
        grads["bias"] = draw_.sum((0, 1))
    if s["h0"] is not None:
        grads["h0"] = g
    return dict(answer, grads=grads)


def _conv_exact(s):
    c = s["case"]
    step, train = c["form"] == "step", c["form"] == "train"
    x, w, bias, win = (_d(s[k]) for k in ("x", "w", "bias", "win"))
    x = x.unsqueeze(1) if step else x
    batch, n, d = x.shape
    k = c["taps"]
    ends = [n] * batch if step or s["lengths"] is None else s["lengths"].tolist()
    w, x = w.clone().requires_grad_(train), x.clone().requires_grad_(train)
    bias = None if bias is None else bias.clone().requires_grad_(train)
    win = None if win is None else win.clone().requires_grad_(train)
    front = torch.zeros(batch, k - 1, d, dtype=torch.float64, device=x.device) if win is None else win
    rows = torch.cat([front, x], 1)
    pre = torch.nn.functional.conv1d(rows.transpose(1, 2), w.unsqueeze(1), bias, groups=d).transpose(1, 2)
    y = pre * torch.sigmoid(pre) if c["silu"] else pre
    live = torch.arange(n, device=x.device)[None] < torch.tensor(ends, device=x.device)[:, None]
    y = y * live[..., None]
    left = torch.stack([rows[i, e:e + k - 1] for i, e in enumerate(ends)])
    answer = {"y": (y[:, 0] if step else y).detach(), "win": left.detach()}
    if not train:
        return answer
    total = (y * _d(s["dy"])).sum()
    if s["dwin"] is not None:
        total = total + (left * _d(s["dwin"])).sum()
    names = [("x", x), ("w", w), ("bias", bias), ("win", win)]
    names = [(name, t) for name, t in names if t is not None]
    return dict(answer, grads=dict(zip([a for a, _ in names], torch.autograd.grad(total, [t for _, t in names]))))


def _norm_exact(s):
    c = s["case"]
    train = c["form"] == "train"
    x, w, r = (_d(s[k]) for k in ("x", "weight", "residual"))
    answer = {}
    if r is not None:
        answer["sum"] = x + r
        # the operator norms the sum as it is kept: its rounding is part of the definition
        x = (s["x"].detach().float() + s["residual"].detach().float()).to(s["residual"].dtype).double()
    x, w = x.clone().requires_grad_(train), w.clone().requires_grad_(train)
    y = x / torch.sqrt(x.square().mean(1, keepdim=True) + EPS) * w
    if c["form"] == "quant":
        scale = y.abs().amax(1).clamp(min=1e-8) / 127
        return dict(answer, values=torch.round(y / scale[:, None]) * scale[:, None], scale=scale)
    answer["y"] = y.detach()
    if not train:
        return answer
    dx, dw = torch.autograd.grad(y, [x, w], _d(s["dy"]))
    grads = {"weight": dw, "x": dx}
    if r is not None:
        grads["x"] = grads["residual"] = dx + _d(s["dsum"])
    return dict(answer, grads=grads)


def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _scan_exact, "conv": _conv_exact, "norm": _norm_exact}[case["op"]](s)
