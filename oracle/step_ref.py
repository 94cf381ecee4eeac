"""Float64 oracle of the transformer-block functions: RMSNormalization, the
residual step and 8-bit copies (NumPy, straight from the definitions).

Every function returns its results as (value, terms) pairs where a tolerance
needs it: `terms` is the sum of the magnitudes of what was added up, the scale
that a float32 evaluation's error is relative to."""
import numpy as np

GROUP = 32
F64 = np.float64


# ---------------------------------------------------------------- 8-bit copies
def e4m3_values():
    """The value of each of the 256 codes (nan for 0x7f and 0xff)."""
    code = np.arange(256)
    e, m = (code >> 3) & 15, code & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return np.where(code & 128, -v, v)


def _round_e4m3(z):
    _, p = np.frexp(z)
    ulp = np.ldexp(1.0, np.maximum(np.where(z == 0, -5, p), -5) - 4)
    return np.rint(z / ulp) * ulp


def act8(x, form):
    """(code values [rows, cols] as float64, exponent codes [rows, groups])."""
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    v = np.zeros((rows, groups * GROUP))
    v[:, :cols] = x
    v = v.reshape(rows, groups, GROUP)
    finite = np.isfinite(v).all(2)
    v = np.where(finite[:, :, None], v, 0.0)
    m, e = np.frexp(np.abs(v).max(2))
    k = e - 7 + (m >= 127.5 / 128) if form == "int8" else e - 9 + (m > 448 / 512)
    k = np.maximum(np.where(m == 0, -120, k), -120)
    z = np.ldexp(v, -k[:, :, None])
    q = np.rint(z) if form == "int8" else _round_e4m3(z)
    code = np.where(finite, k + 127, 255)
    return q.reshape(rows, -1)[:, :cols], code.astype(np.uint8)


def act8_value(q, code):
    s = np.where(code == 255, np.nan, np.ldexp(1.0, code.astype(int) - 127))
    return q * np.repeat(s, GROUP, 1)[:, :q.shape[1]]


# ------------------------------------------------------------------ the norms
def moments(v, norm):
    mean = v.mean(1, keepdims=True) if norm == "layer" else np.zeros((v.shape[0], 1))
    return mean, ((v - mean) ** 2).mean(1, keepdims=True)


def norm_fwd(v, gamma, beta, norm, eps):
    mean, var = moments(v, norm)
    rho = 1 / np.sqrt(var + eps)
    g = np.ones(v.shape[1]) if gamma is None else gamma
    b = np.zeros(v.shape[1]) if beta is None else beta
    y = (v - mean) * rho * g + b
    terms = (np.abs(v) + np.abs(mean)) * rho * np.abs(g) + np.abs(b)
    return y, terms, mean, var


def norm_bwd(v, dy, gamma, mean, var, norm, eps, dy_terms=None):
    """(dv, terms), (dgamma, terms), (dbeta, terms) for given moments; dy_terms:
    the terms dy itself was summed from, where it is a computed value."""
    dyt = np.abs(dy) if dy_terms is None else dy_terms
    rho = 1 / np.sqrt(var + eps)
    vh = (v - mean) * rho
    vht = (np.abs(v) + np.abs(mean)) * rho
    g = np.ones(v.shape[1]) if gamma is None else gamma
    G, Gt = dy * g, dyt * np.abs(g)
    dv = G - vh * (G * vh).mean(1, keepdims=True)
    t = Gt + vht * (Gt * vht).mean(1, keepdims=True)
    if norm == "layer":
        dv = dv - G.mean(1, keepdims=True)
        t = t + Gt.mean(1, keepdims=True)
    return (rho * dv, rho * t), ((dy * vh).sum(0), (dyt * vht).sum(0)), (dy.sum(0), dyt.sum(0))


def gate_rows(gate, rows):
    """The gate with a row per token."""
    if gate is None:
        return np.ones((1, 1))
    return gate if gate.shape[0] == rows else np.repeat(gate, rows // gate.shape[0], 0)


def step_fwd(x, res, gate, gp, bp, gn, bn, norm, post, pre, rs, bs, eps):
    """dict of (value, terms): h, y; and the moments mean_post, ..., var_pre."""
    out = {}
    u, ut = x, np.abs(x)
    if post:
        u, ut, out["mean_post"], out["var_post"] = norm_fwd(x, gp, bp, norm, eps)
    g = gate_rows(gate, x.shape[0])
    h, ht = bs * g * u, np.abs(bs * g) * ut
    if res is not None:
        h, ht = h + rs * res, ht + np.abs(rs * res)
    out["h"] = (h, ht)
    if pre:
        mean, var = moments(h, norm)
        rho = 1 / np.sqrt(var + eps)
        g2 = np.ones(x.shape[1]) if gn is None else gn
        b2 = np.zeros(x.shape[1]) if bn is None else bn
        out["y"] = ((h - mean) * rho * g2 + b2,
                    (ht + ht.mean(1, keepdims=True)) * rho * np.abs(g2) + np.abs(b2))
        out["mean_pre"], out["var_pre"] = mean, var
        out["pre_terms"] = (ht ** 2).mean(1, keepdims=True)
    return out


def step_bwd(x, h, dh, dy, stats, gate, gate_full, gp, bp, gn, norm, post, pre, has_res, rs, bs, eps):
    """dict of (value, terms) of every gradient that exists.  stats: the kept
    moments (mean_post, var_post, mean_pre, var_pre) as columns."""
    out = {}
    rows, cols = (dh if dh is not None else dy).shape
    t, tt = (np.zeros((rows, cols)),) * 2 if dh is None else (dh, np.abs(dh))
    if pre:
        d, out["dgamma_pre"], out["dbeta_pre"] = norm_bwd(h, dy, gn, stats[2], stats[3], norm, eps)
        t, tt = t + d[0], tt + d[1]
    if has_res:
        out["dres"] = rs * t, abs(rs) * tt
    w, wt = bs * t, abs(bs) * tt
    if gate is not None:
        if post:
            rho = 1 / np.sqrt(stats[1] + eps)
            g1 = np.ones(cols) if gp is None else gp
            b1 = np.zeros(cols) if bp is None else bp
            u = (x - stats[0]) * rho * g1 + b1
            ut = (np.abs(x) + np.abs(stats[0])) * rho * np.abs(g1) + np.abs(b1)
        else:
            u, ut = x, np.abs(x)
        if gate_full:
            out["dgate"] = w * u, wt * ut
        else:
            n = gate.shape[0]
            out["dgate"] = ((w * u).reshape(n, rows // n, cols).sum(1),
                            (wt * ut).reshape(n, rows // n, cols).sum(1))
        g = gate_rows(gate, rows)
        w, wt = w * g, wt * np.abs(g)
    if post:
        out["dx"], out["dgamma_post"], out["dbeta_post"] = norm_bwd(x, w, gp, stats[0], stats[1],
                                                                    norm, eps, wt)
    else:
        out["dx"] = w, wt
    return out
