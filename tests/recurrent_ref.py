"""The gated recurrence, the layer norm and the choice of a token in 64 bits, and how far fp32 arithmetic may be off.

Errors are counted in units of 2^-24, half a step of fp32, and carried through the formulas term by term: next to a value
stands the sum of its terms' magnitudes (M) and the error that these have met (E).  A product's error is each factor's
error times the other's magnitude, a rounding adds one unit of the magnitude, and a few more units than there are
roundings are granted where the order of the sums is the kernel's own (folds of stretches instead of single positions).
"""
import numpy as np
import torch

U = 2.0 ** -24


def d64(t):
    return None if t is None else t.detach().cpu().double()


def live(batch, n, lengths):
    if lengths is None:
        return torch.ones(batch, n, 1, dtype=torch.bool)
    return (torch.arange(n)[None] < lengths.cpu().long()[:, None])[..., None]


def _sig(v):
    """sigmoid, its complement, and both's relative errors in units: 2^x to 2 ulp (4), 1 + e, the reciprocal (2), the product
    (8 in all); the argument's rounding, the one of its product with log2(e) and the constant's are 3 |v| of the power,
    which the smaller of the two has in full and the larger at most e^-|v| 3 |v| <= 1.2 of."""
    s, n = torch.sigmoid(v), torch.sigmoid(-v)
    small, large = 9 + 3 * v.abs(), torch.full_like(v, 10.0)
    return s, n, torch.where(v < 0, small, large), torch.where(v < 0, large, small)


def recurrence(a):
    """a: dict of x, f, z, bias, h0, lengths, convex, dy, dh (missing or None: not there), any type.  Returns
    {name: (value, error)} in 64 bits on the CPU, the error in fp32 units before the result's own rounding."""
    x, f, z, bias, h0, dy, dh = (d64(a.get(k)) for k in ("x", "f", "z", "bias", "h0", "dy", "dh"))
    b, n, d = x.shape
    on = live(b, n, a.get("lengths"))
    wipe = lambda t: None if t is None else torch.where(on, t, 0.0)  # noqa: E731
    x, f, z, dy = wipe(x), wipe(f), wipe(z), wipe(dy)
    f = f if bias is None else f + bias
    up, down, r_up, r_down = _sig(f)
    c, rc = (down, r_down) if a.get("convex", True) else (torch.ones_like(up), torch.zeros_like(up))
    keep, add, madd = torch.where(on, up, 1.0), wipe(c * x), wipe(c * x.abs())
    e_keep, e_add = wipe(r_up + 3), wipe((rc + 3) * c * x.abs())
    h = torch.zeros(b, d, dtype=torch.float64) if h0 is None else h0
    H, M, E = [h], [h.abs()], [torch.zeros_like(h)]
    for t in range(n):
        k = keep[:, t]
        m = k * M[-1] + madd[:, t]
        E.append(k * E[-1] + e_keep[:, t] * k * M[-1] + e_add[:, t] + torch.where(on[:, t], m, 0.0))
        H.append(k * H[-1] + add[:, t])
        M.append(m)
    H, M, E = (torch.stack(v, 1) for v in (H, M, E))
    now, mnow, enow = H[:, 1:], M[:, 1:], E[:, 1:]
    if z is None:
        gate, e_gate = torch.ones_like(x), torch.zeros_like(x)
        slope = torch.zeros_like(x)
    else:
        s, s_n, r_s, r_n = _sig(z)
        gate, e_gate, slope = z * s, (r_s + 1) * z.abs() * s, s + z * s * s_n
    out = {"y": (wipe(now * gate), wipe(enow * gate.abs() + mnow * (e_gate + gate.abs()))), "h": (H[:, n], E[:, n])}
    if dy is None and dh is None:
        return out
    dy = torch.zeros_like(x) if dy is None else dy
    ds, e_ds = dy * gate, dy.abs() * (e_gate + gate.abs())
    flow = torch.zeros(b, d, dtype=torch.float64) if dh is None else dh
    MG, EG = flow.abs(), torch.zeros_like(flow)
    g, mg, eg = (torch.zeros_like(x) for _ in range(3))
    for t in reversed(range(n)):
        g[:, t], mg[:, t] = ds[:, t] + flow, ds[:, t].abs() + MG
        eg[:, t] = e_ds[:, t] + EG + mg[:, t]
        k = keep[:, t]
        flow, MG, EG = k * g[:, t], k * mg[:, t], k * eg[:, t] + e_keep[:, t] * k * mg[:, t]
    before, mb, eb = H[:, :n], M[:, :n], E[:, :n]
    away, m_away = (before - x, mb + x.abs()) if a.get("convex", True) else (before, mb)
    bend = up * down
    df = wipe(g * bend * away)
    m_df = wipe(mg * bend * m_away)
    e_df = wipe(bend * (eg * m_away + mg * (eb + m_away)) + (r_up + r_down + 4) * mg * bend * m_away)
    out.update(dx=(wipe(c * g), wipe(c * (eg + (rc + 1) * mg))), df=(df, e_df), dh0=(flow, EG),
               dbias=(df.sum((0, 1)), e_df.sum((0, 1)) + (b * n) * m_df.sum((0, 1))))
    if z is not None:
        m_slope = s + z.abs() * s * s_n
        e_slope = (2 * r_s + r_n + 4) * m_slope
        out["dz"] = (wipe(dy * now * slope), wipe(dy.abs() * (enow * m_slope + mnow * (e_slope + 2 * m_slope))))
    return out


def norm(s, w, bias, eps, dy=None, dsum=None):
    """s: the sum as it is kept, [rows, width].  {name: (value, error)}.  A row's sums: at most 32 terms in a thread, then
    over 5 steps of a warp and at most 16 warps: 64 units of the terms' magnitudes."""
    s, w, bias, dy, dsum = (d64(t) for t in (s, w, bias, dy, dsum))
    K = 64
    mean = s.mean(1, keepdim=True)
    e_mean = (K + 1) * s.abs().mean(1, keepdim=True)
    xc = s - mean
    e_xc = e_mean + xc.abs()
    var = (xc * xc).mean(1, keepdim=True) + eps
    e_var = (2 * xc.abs() * e_xc).mean(1, keepdim=True) + (K + 3) * var
    # errors of second order matter where a row is nearly constant: (e_xc U)^2 in units of U
    e_var = e_var + (e_xc * e_xc).mean(1, keepdim=True) * U
    rstd = 1 / torch.sqrt(var)
    r_rstd = 0.5 * e_var / var + 4
    xh = xc * rstd
    e_xh = rstd * e_xc + xh.abs() * (r_rstd + 1)
    y = xh * w
    e_y = w.abs() * (e_xh + xh.abs())
    if bias is not None:
        e_y = e_y + y.abs() + bias.abs()
        y = y + bias
    out = {"y": (y, e_y)}
    if dy is None:
        return out
    g, n = w * dy, s.shape[0]
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    e1 = (K + 2) * g.abs().mean(1, keepdim=True)
    e2 = (g.abs() * e_xh).mean(1, keepdim=True) + (K + 3) * (g * xh).abs().mean(1, keepdim=True)
    mag = g.abs() + m1.abs() + (xh * m2).abs()
    ds = rstd * (g - m1 - xh * m2)
    e_ds = rstd * (e1 + xh.abs() * e2 + e_xh * m2.abs() + (4 + r_rstd) * mag)
    if dsum is not None:
        ds, e_ds = ds + dsum, e_ds + ds.abs() + dsum.abs()
    out["ds"] = (ds, e_ds)
    out["dw"] = ((dy * xh).sum(0), (dy.abs() * e_xh).sum(0) + (n + 2) * (dy * xh).abs().sum(0))
    out["dbias"] = (dy.sum(0), (n + 2) * dy.abs().sum(0))
    return out


def check(got, want, name):
    """|got - want| within the error's units and half a step of the result's own type (half its smallest subnormal)."""
    want, err = want
    got, dtype = got.detach().cpu(), got.dtype
    assert got.shape == want.shape, (name, got.shape, want.shape)
    tol = U * err * (1 + 2.0 ** -10) + 1e-37  # errors of errors
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + 2.0 ** (-25 if dtype == torch.float16 else -134)
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((off / tol)[bad].max()), got[bad][:4], want[bad][:4])


# ---------------------------------------------------------------------------
# the choice of a token
# ---------------------------------------------------------------------------
def sample(logits, u, temperature, top_k, top_p, min_p):
    """One row, 1-D logits: (token, its share of the kept mass, how near the closest border lay).  Borders are compared
    relative to the mass: a choice that changes where a sum moves by less than this distance is within rounding."""
    row = logits.detach().cpu().double().numpy()
    best = int(np.argmax(np.where(np.isnan(row), np.inf, row)))
    if np.isnan(row).any():
        best = int(np.argmax(np.isnan(row)))
    if not temperature > 0 or not np.isfinite(row[best]):
        return best, 1.0, 1.0
    left = np.lexsort((np.arange(row.size), -row))
    left = left[np.isfinite(row[left])]
    if 0 < top_k < left.size:
        left = left[:top_k]
    mass = np.exp((row[left] - row[best]) / temperature)
    near = 1.0
    whole = (mass == 1).all()  # equal tokens: their sums, and a number of 24 bits times those, are exact on both sides
    if top_p < 1:  # a NaN keeps all
        total = mass.sum()
        before = np.cumsum(mass) - mass
        ok = before < top_p * total
        ok[0] = True
        near = min(near, np.abs(before[1:] / total - top_p).min(initial=1.0))
        left, mass = left[ok], mass[ok]
    floor = min(max(min_p, 0.0), 1.0) if min_p == min_p else 0.0
    if floor > 0:
        near = min(near, np.abs(mass[mass < 1] / floor - 1).min(initial=1.0))  # that of the maximum is exact
        ok = mass >= floor
        left, mass = left[ok], mass[ok]
    order = np.argsort(left)
    left, mass = left[order], mass[order]
    upto = np.cumsum(mass)
    target = (min(max(u, 0.0), 1.0) if u == u else 0.0) * upto[-1]
    at = min(int(np.searchsorted(upto, target, side="right")), left.size - 1)
    near = min(near, np.abs(upto[:-1] / upto[-1] - target / upto[-1]).min(initial=1.0))
    return int(left[at]), float(mass[at] / upto[-1]), 1.0 if whole else float(near)
