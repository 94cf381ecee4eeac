"""Sums over very long rows and over very many rows of equal and nearly equal
values: every addition of such values onto a running float32 sum is rounded the
same way, so that a long chain is off by far more than its terms are (8192 times
0.1 by 1085 u, 2^18 times by 41460 u).

Unit: u = 2^-24, half a step of float32.  A row sum of the kernels for long rows: a
vector of at most 8 elements in float32 (8 u), the vectors in double, rounded once
(1), 6 levels of a wave and 8 waves (14), the division by the columns, as a product
with a rounded reciprocal (2): 25 u of the sum of the magnitudes, at any length.  A
column sum: at most 256 rows one after another, partial sums in double, rounded once,
7 + 7 levels: 271 u, with the roundings of its terms: 280."""
import numpy as np
import pytest
import torch

from _step import DTYPES, f64
from _util import load_package

K = load_package()
pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROW, COLUMN = 25 * U, 280 * U
LONG = (1 << 22) + 5


SPREAD = pytest.mark.parametrize("spread", [0.0, 1e-3])


def near(n, gen, spread, rows=1, level=0.1):
    return level * (1 + spread * torch.randn(rows, n, generator=gen))


def check(got, want, tol, name):
    err = np.abs(f64(got).reshape(np.shape(want)) - want)
    assert (err <= tol).all(), (name, (err / tol).max())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("which", ["post", "pre"])
@SPREAD
def test_row_statistics(spread, which, dtype):
    x = near(LONG, torch.Generator().manual_seed(1), spread).to(DTYPES[dtype]).cuda()
    xv = f64(x)
    kw = dict(post=which == "post", pre=which == "pre")
    i = 1 if which == "post" else 3
    ms = (xv * xv).mean()
    f = K.resnorm_forward(x, None, 1, norm="rms", **kw)
    check(f.stats[i], [ms], ROW * ms, "mean square")

    f = K.resnorm_forward(x, None, 1, norm="layer", **kw)
    mean, var = xv.mean(), xv.var()
    off = ROW * np.abs(xv).mean()
    check(f.stats[i - 1], [mean], off, "mean")
    # about the mean it has: larger by the square of what that is off; a difference
    # rounded once (2 u of its square)
    check(f.stats[i], [var], (ROW + 2 * U) * (var + off ** 2) + off ** 2, "variance")


@pytest.mark.parametrize("kept", [None, "int8"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("which", ["post", "pre"])
@SPREAD
def test_row_sums_of_the_backward(spread, which, norm, kept):
    """dx = rho (G - mean G - v^ mean(G v^)) of nearly equal G: what is left is small."""
    gen = torch.Generator().manual_seed(2)
    x = (1 + 0.5 * torch.rand(1, LONG, generator=gen)).cuda()
    dy = near(LONG, gen, spread).cuda()
    xk = x if kept is None else K.act8_pack(x, 1, kept)
    xv = f64(x if kept is None else K.act8_unpack(xk, 1, torch.float32))
    mean = torch.full((1,), 0.25 if norm == "layer" else 0.0, device="cuda")
    var = torch.ones(1, device="cuda")
    stats = (mean if norm == "layer" else None, var)
    none = (None, None)
    if which == "post":
        g = K.resnorm_backward(xk, None, dy, None, stats + none, 1, norm=norm, pre=False, has_res=False)
    else:
        g = K.resnorm_backward(None, xk, None, dy, none + stats, 1, norm=norm, post=False, has_res=False)
    rho = 1 / np.sqrt(1 + float(np.float32(1e-5)))
    vh, G = (xv - f64(mean)) * rho, f64(dy)
    s1, s2 = G.mean() if norm == "layer" else 0.0, (G * vh).mean()
    want = rho * (G - s1 - vh * s2)
    # v^ by 4.5 u of itself in both places; a product, two sums and a product after
    # them: 4 u of the magnitudes
    off = rho * (ROW * s1 + np.abs(vh) * (ROW + 4.5 * U) * np.abs(G * vh).mean() + 4.5 * U * np.abs(vh * s2)
                 + 4 * U * (np.abs(G) + s1 + np.abs(vh * s2))) + 2.5 * U * np.abs(want)
    check(g.dx, want, off, "dx")


@pytest.mark.parametrize("cols", [1, 3, 7])
@pytest.mark.parametrize("which", ["post", "pre"])
@SPREAD
def test_column_sums_of_many_short_rows(spread, which, cols):
    rows = (1 << 21) + 3
    gen = torch.Generator().manual_seed(3)
    dt = torch.float32 if cols < 4 else torch.bfloat16      # rows of less than a vector
    x, dy = (near(cols, gen, spread, rows, level).to(dt).cuda() for level in (1.0, 0.1))
    mean, var = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    none = (None, None)
    if which == "post":
        g = K.resnorm_backward(x, None, dy, None, (mean, var) + none, rows, norm="layer", pre=False,
                               has_res=False)
        dg, db = g.dgamma_post, g.dbeta_post
    else:
        g = K.resnorm_backward(None, x, None, dy, none + (mean, var), rows, norm="layer", post=False,
                               has_res=False)
        dg, db = g.dgamma_pre, g.dbeta_pre
    rho = 1 / np.sqrt(1 + float(np.float32(1e-5)))
    for got, terms, name in ((dg, f64(dy) * f64(x) * rho, "dgamma"), (db, f64(dy), "dbeta")):
        check(got, terms.sum(0), COLUMN * np.abs(terms).sum(0), name)


@pytest.mark.parametrize("cols", [3, 16])
@SPREAD
def test_a_gate_row_per_token(spread, cols):
    """Every token leaves a partial sum of its own for the fold: dgamma through the gate."""
    rows = 1 << 20
    gen = torch.Generator().manual_seed(4)
    x, dh, gate = (near(cols, gen, spread, rows, level).cuda() for level in (1.0, 0.1, 0.5))
    x, dh = x.bfloat16(), dh.bfloat16()
    var = torch.ones(rows, device="cuda")
    gamma = (1 + 0.2 * torch.randn(cols, generator=gen)).cuda()
    g = K.resnorm_backward(x, None, dh, None, (None, var, None, None), rows, gate=gate, gamma_post=gamma,
                           norm="rms", pre=False, has_res=False)
    rho = 1 / np.sqrt(1 + float(np.float32(1e-5)))
    each = f64(dh) * f64(x) * rho
    terms = each * f64(gate)
    # a partial sum of one row: 3.5 u of v^, 1 of its product with dh; the gate 1; the fold 15
    check(g.dgamma_post, terms.sum(0), 24 * U * np.abs(terms).sum(0), "dgamma")
    want = each * f64(gamma)
    check(g.dgate, want, 24 * U * np.abs(want), "dgate")


def test_more_runs_of_rows_than_a_grid_has_blocks():
    rows = 65536 * 256 + 3
    dy = torch.full((rows, 1), 0.1, dtype=torch.bfloat16, device="cuda")
    x = torch.full((rows, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    dy[-3:] = 64.0
    mean, var = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    g = K.resnorm_backward(x, x, None, dy, (mean, var, mean, var), rows, norm="layer", post=False)
    rho = 1 / np.sqrt(1 + float(np.float32(1e-5)))
    want = dy.double().sum().item()
    check(g.dbeta_pre, [want], COLUMN * want, "dbeta")
    check(g.dgamma_pre, [want * 2 * rho], COLUMN * want * 2 * rho, "dgamma")
    # one column: G - mean G - v^ mean(G v^) is -v^ G v^, of 0.1, 2 and 64
    vh = 2 * rho
    for part, G in ((g.dx[:-3], 0.1), (g.dx[-3:], 64.0)):
        G = float(torch.tensor(G).bfloat16())
        d = -rho * vh * G * vh
        # 4.5 u of v^ twice, 2.5 u of rho, three products, the sums before them
        tol = torch.finfo(torch.bfloat16).eps / 2 * abs(d) + 16 * U * (abs(d) + 2 * abs(G))
        assert (part.double() - d).abs().max().item() <= tol
