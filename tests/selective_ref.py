"""The float Mamba operators position by position in 64 bits, with hand-written gradients, and what their terms add up
to without their signs: a sum's rounding error is at most the roundings on the way of a term, times half a step, times
that."""
import torch


def silu(v):
    s = torch.sigmoid(v)
    return v * s, s * (1 + v * (1 - s))


def live(batch, n, lengths):
    if lengths is None:
        return torch.ones(batch, n, dtype=torch.bool)
    return torch.arange(n)[None] < lengths.cpu().long()[:, None]


def scan(a, mag=False):
    """a: dict of u, delta, A, B, C, D, z, bias, softplus, h0, lengths, dy, dh (missing or None: not there), any type.
    Returns y, h and the gradients in 64 bits on the CPU; mag: the sums of the terms' magnitudes in their place."""
    v = {k: (None if t is None else t.detach().cpu().double() if isinstance(t, torch.Tensor) and t.is_floating_point()
             else t) for k, t in a.items()}
    ab = torch.abs if mag else (lambda t: t)
    get = lambda k: v.get(k)  # noqa: E731
    batch, n, d = v["u"].shape
    on = live(batch, n, a.get("lengths"))
    wipe = lambda t: None if t is None else torch.where(on[..., None], t, 0)  # noqa: E731
    u, B, C, z = (wipe(get(k)) for k in ("u", "B", "C", "z"))
    raw = wipe(v["delta"])
    if get("bias") is not None:
        raw = raw + v["bias"]
    dt = torch.nn.functional.softplus(raw, threshold=700) if get("softplus") else raw
    dt = wipe(dt)
    slope = torch.sigmoid(raw) if get("softplus") else torch.ones_like(raw)
    gate, dgate = (torch.ones_like(u), torch.zeros_like(u)) if z is None else silu(z)
    if mag and z is not None:
        # silu'(z) = s + s z (1 - s) crosses zero at z = -1.28, where its two terms cancel: each is rounded, so the error
        # goes by s + s |z| (1 - s) and not by what is left of them
        sg = torch.sigmoid(z)
        dgate = sg + sg * z.abs() * (1 - sg)
    A = v["A"]
    decay = torch.exp(dt[..., None] * A)
    u, B, C, gate, dgate, dt_, A_ = (ab(t) for t in (u, B, C, gate, dgate, dt, A))
    D = torch.zeros(d, dtype=torch.float64) if get("D") is None else ab(v["D"])
    h = torch.zeros(batch, d, A.shape[1], dtype=torch.float64) if get("h0") is None else ab(v["h0"])
    hs, s = [h], torch.zeros_like(u)
    for t in range(n):
        h = decay[:, t] * h + (dt_[:, t] * u[:, t])[..., None] * B[:, t, None]
        hs.append(h)
        s[:, t] = (h * C[:, t, None]).sum(2) + D * u[:, t]
    out = {"y": wipe(s * gate), "h": h}
    if get("dy") is None and get("dh") is None:
        return out
    dy = torch.zeros_like(u) if get("dy") is None else ab(wipe(v["dy"]))
    ds = dy * gate
    g = torch.zeros_like(h) if get("dh") is None else ab(v["dh"])
    du, ddt = torch.zeros_like(u), torch.zeros_like(u)
    dB, dC, dA = torch.zeros_like(B), torch.zeros_like(C), torch.zeros_like(A)
    for t in reversed(range(n)):
        g = g + ds[:, t, :, None] * C[:, t, None]
        dC[:, t] = (ds[:, t, :, None] * hs[t + 1]).sum(1)
        dB[:, t] = (g * (dt_[:, t] * u[:, t])[..., None]).sum(1)
        s1 = (g * B[:, t, None]).sum(2)
        w = g * decay[:, t] * hs[t]
        du[:, t] = dt_[:, t] * s1 + D * ds[:, t]
        ddt[:, t] = u[:, t] * s1 + (w * A_).sum(2)
        dA += (w * dt_[:, t, :, None]).sum(0)
        g = g * decay[:, t]
    ddelta = wipe(ddt * slope)
    out.update(du=wipe(du), ddelta=ddelta, dA=dA, dB=wipe(dB), dC=wipe(dC), dD=(ds * u).sum((0, 1)),
               dz=wipe(dy * s * dgate), dbias=ddelta.sum((0, 1)), dh0=g)
    return out


def conv(a, mag=False):
    """a: dict of x, w, bias, silu, win, lengths, dy, dwin."""
    v = {k: (None if t is None else t.detach().cpu().double() if isinstance(t, torch.Tensor) and t.is_floating_point()
             else t) for k, t in a.items()}
    ab = torch.abs if mag else (lambda t: t)
    x, w = v["x"], v["w"]
    batch, n, d = x.shape
    k = w.shape[1]
    on = live(batch, n, a.get("lengths"))
    x = torch.where(on[..., None], x, 0)
    ends = on.sum(1)
    win = torch.zeros(batch, k - 1, d, dtype=torch.float64) if v.get("win") is None else v["win"]
    rows = torch.cat([win, x], 1)
    pre = sum(rows[:, i:i + n] * w[:, i] for i in range(k))
    if v.get("bias") is not None:
        pre = pre + v["bias"]
    f, df = silu(pre) if v.get("silu") else (pre, torch.ones_like(pre))
    out = {"y": torch.where(on[..., None], f, 0),
           "win": torch.stack([rows[i, e:e + k - 1] for i, e in enumerate(ends.tolist())])}
    if mag:
        premag = sum(rows[:, i:i + n].abs() * w[:, i].abs() for i in range(k))
        if v.get("bias") is not None:
            premag = premag + v["bias"].abs()
        out["y"] = torch.where(on[..., None], premag, 0)  # |silu'| < 1.1: the sum's error passes through
        out["win"] = out["win"].abs()
    if v.get("dy") is None and v.get("dwin") is None:
        return out
    dy = torch.zeros_like(x) if v.get("dy") is None else torch.where(on[..., None], v["dy"], 0)
    dc = dy * df
    if mag:  # the derivative's own error: |silu''| <= 1/2 times the sum's, on top of its value's
        dc = dy.abs() * (df.abs() + out["y"] + 1) if v.get("silu") else dy.abs()
    drows = torch.zeros_like(rows)
    for i in range(k):
        drows[:, i:i + n] += dc * ab(w[:, i])
    if v.get("dwin") is not None:
        for b, e in enumerate(ends.tolist()):
            drows[b, e:e + k - 1] += ab(v["dwin"][b])
    dw = torch.stack([(dc * ab(rows[:, i:i + n])).sum((0, 1)) for i in range(k)], 1)
    out.update(dx=drows[:, k - 1:], dwin=drows[:, :k - 1], dw=dw, dbias=dc.sum((0, 1)))
    return out


def norm(s, w, eps, dy=None, dsum=None):
    """s: the sum as it is kept.  Returns y and, with dy, ds and dw."""
    s, w = s.detach().cpu().double(), w.detach().cpu().double()
    rstd = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    out = {"y": s * rstd * w, "rstd": rstd}
    if dy is not None:
        dy = dy.detach().cpu().double()
        xh, g = s * rstd, w * dy
        m = (g * xh).mean(1, keepdim=True)
        out["ds"] = rstd * (g - xh * m) + (0 if dsum is None else dsum.detach().cpu().double())
        out["ds_mag"] = rstd * (g.abs() + xh.abs() * (g * xh).abs().mean(1, keepdim=True)) + (
            0 if dsum is None else dsum.detach().cpu().double().abs())
        out["dw"] = (dy * xh).sum(0)
        out["dw_mag"] = (dy * xh).abs().sum(0)
    return out


def check(got, want, mag, units, name):
    """|got - want| <= units half steps of fp32 of the terms' magnitudes, and half a step of the result's own type
    (at least half its smallest subnormal)."""
    got, dtype = got.detach().cpu(), got.dtype
    want, mag = want.expand(got.shape), mag.expand(got.shape)
    tol = units * 2.0 ** -24 * mag + 1e-37
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + 2.0 ** (-25 if dtype == torch.float16 else -134)
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((off / tol)[bad].max()), got[bad][:4], want[bad][:4])
