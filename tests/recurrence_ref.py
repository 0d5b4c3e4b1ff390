"""The gated linear recurrence in 64 bits, with a bound of what fp32 arithmetic may be off, element by element.

u = 2^-24.  A gate's exponent -log2(e) f is off by |f| log2(e) 2u (constant and product), so its exponential is off by
2u |f| + 2u (exp2, one ulp), relatively; 1 + e adds u and the reciprocal 2u: sigmoid(f) and 1 - sigmoid(f) are off by at most
g(f) = (2 |f| + 6) u.  Errors of h run through the recurrence like h itself: E_t = a E_{t-1} + g |a h_{t-1}| + (g + u) |b z| + u |h_t|.
A split of the sequence multiplies gates first and adds partial sums later; every term of the sum still carries the errors of its
own gates, and a few more additions, hence the factor 2 at the end."""
import numpy as np

U = 2.0 ** -24


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-x))


def _g(f):
    return (2.0 * np.abs(np.where(np.isfinite(f), f, 0.0)) + 6.0) * U


def _turned(x, lens, reverse):
    """Every row in the order of its recurrence (padding stays behind)."""
    if not reverse:
        return x.copy()
    y = x.copy()
    for b, n in enumerate(lens):
        y[b, :n] = x[b, :n][::-1]
    return y


def forward(z, f, o, lens, state, reverse):
    """float64 arrays [B, T, H]; lens int array; state [B, H].  Returns a dict with y, final and their bounds (and what the backward
    pass needs, in the order of the recurrence)."""
    B, T, H = z.shape
    with np.errstate(invalid="ignore", over="ignore"):
        return _forward(*(_turned(x, lens, reverse) if x is not None else None for x in (z, f, o)), lens, state, reverse)


def _forward(z, f, o, lens, state, reverse):
    B, T, H = z.shape
    live = np.arange(T)[None, :] < lens[:, None]
    a, b, g = sigmoid(f), sigmoid(-f), _g(f)
    h, e = state.astype(np.float64).copy(), np.zeros((B, H))
    hs, es, before, ebefore = (np.zeros((B, T, H)) for _ in range(4))
    for t in range(T):
        on = live[:, t, None]
        before[:, t], ebefore[:, t] = h, e
        new = a[:, t] * h + b[:, t] * z[:, t]
        enew = a[:, t] * e + g[:, t] * np.abs(a[:, t] * h) + (g[:, t] + U) * np.abs(b[:, t] * z[:, t]) + U * np.abs(new)
        h, e = np.where(on, new, h), np.where(on, enew, e)
        hs[:, t], es[:, t] = h, e
    so = None if o is None else sigmoid(o)
    y = hs if o is None else hs * so
    ey = es if o is None else es * so + np.abs(y) * (_g(o) + U)
    y, ey = np.where(live[..., None], y, 0.0), np.where(live[..., None], ey, 0.0)
    return {"y": _turned(y, lens, reverse), "ey": 2 * _turned(ey, lens, reverse), "final": h, "efinal": 2 * e, "z": z, "a": a, "b": b, "g": g, "o": o, "so": so,
            "h": hs, "eh": es, "before": before, "ebefore": ebefore, "live": live}


def backward(x, dy, dfinal, lens, reverse):
    dy = _turned(dy, lens, reverse)
    B, T, H = dy.shape
    d, e = dfinal.astype(np.float64).copy(), np.zeros((B, H))
    out = {k: np.zeros((B, T, H)) for k in ("dz", "df", "do", "edz", "edf", "edo")}
    for t in range(T - 1, -1, -1):
        on = x["live"][:, t, None]
        a, b, g, z = x["a"][:, t], x["b"][:, t], x["g"][:, t], x["z"][:, t]
        if x["o"] is None:
            here, egate = dy[:, t], 0.0
        else:
            so, go = x["so"][:, t], _g(x["o"][:, t])
            here = dy[:, t] * so
            egate = np.abs(here) * (go + U)
            out["do"][:, t] = np.where(on, here * x["h"][:, t] * (1 - so), 0.0)
            out["edo"][:, t] = np.where(on, np.abs(here * (1 - so)) * x["eh"][:, t] + np.abs(out["do"][:, t]) * (2 * go + 4 * U), 0.0)
        cur = d + here
        ecur = e + egate + U * np.abs(cur)
        w = x["before"][:, t] - z
        out["dz"][:, t] = np.where(on, b * cur, 0.0)
        out["edz"][:, t] = np.where(on, b * ecur + np.abs(b * cur) * (g + U), 0.0)
        out["df"][:, t] = np.where(on, cur * w * a * b, 0.0)
        out["edf"][:, t] = np.where(on, a * b * (ecur * np.abs(w) + np.abs(cur) * (x["ebefore"][:, t] + U * np.abs(w))) + np.abs(out["df"][:, t]) * (2 * g + 4 * U), 0.0)
        d = np.where(on, a * cur, d)
        e = np.where(on, a * ecur + np.abs(a * cur) * (g + U), e)
    got = {k: _turned(v, lens, reverse) for k, v in out.items()}
    got.update({k: 2 * got[k] for k in ("edz", "edf", "edo")})
    got["dstate"], got["edstate"] = d, 2 * e
    return got
