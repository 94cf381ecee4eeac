"""LayerNormalization of the transformer-block functions on rows far from zero:
what is normalized is centred before it is scaled.

Unit: u = 2^-24, half a step of float32.  1 / sqrt(var + eps) is off by 0.5 u
(the sum, under the root) + u + u, a difference, a product or a fma by u each.
v^ = (v - mean) / std of given statistics is therefore off by 2.5 + 1 + 1 = 4.5 u of
itself, whatever the mean: an element at the mean gives exactly zero.  Evaluated
as v / std - mean / std it would be off by u of mean / std instead."""
import numpy as np
import pytest
import torch

from _step import DTYPES, f64
from _util import load_package

K = load_package()
pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def bound(want, dtype, n):
    """n roundings to float32, one to dtype (float16: half its least step at least)."""
    return np.abs(want) * (n * U + torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def check(got, want, tol, name):
    bad = np.abs(f64(got) - want) > tol
    assert not bad.any(), (name, int(bad.sum()), np.abs(f64(got) - want)[bad].max())


def whole_rows(rows, cols, mean, gen):
    """Whole numbers about `mean` with exactly that mean, many of them equal to it.
    Sums of them (below 2^24) and of their squares about the mean are exact in float32
    in any order; so is a division by `cols`, a power of two."""
    a = torch.randint(-8, 9, (rows, cols // 2), generator=gen)
    d = torch.cat([a, -a], 1)[:, torch.randperm(cols, generator=gen)]
    return d.double().numpy(), (d + mean).double()


# whole and ragged (tensors one element off a vector), a gate per element, every width
@pytest.mark.parametrize("form", ["whole", "ragged", "gate"])
@pytest.mark.parametrize("dtype,mean", [("f16", 1000), ("bf16", 120), ("f32", 1000)])
@pytest.mark.parametrize("cols", [64, 256, 1024, 4096, 8192, 16384])
def test_forward_at_the_mean(cols, dtype, mean, form):
    rows, dt = 5, DTYPES[dtype]
    gen = torch.Generator().manual_seed(cols)
    d, x = whole_rows(rows, cols, mean, gen)
    gamma = (1 + 0.2 * torch.randn(cols, generator=gen)).float()
    flat = torch.zeros(rows * cols + 8, dtype=dt, device="cuda")
    off = 1 if form == "ragged" else 0
    xd = flat[off:off + rows * cols].view(rows, cols)
    xd.copy_(x.to(dt))
    assert np.array_equal(f64(xd), x.numpy())       # held exactly
    gate = torch.ones(rows, cols, dtype=dt, device="cuda") if form == "gate" else None
    var = (d * d).mean(1, keepdims=True)
    eps = float(np.float32(1e-5))
    want = d / np.sqrt(var + eps) * f64(gamma)
    for which in ("post", "pre"):
        f = K.resnorm_forward(xd, None, rows, gate=gate, norm="layer", post=which == "post",
                              pre=which == "pre", **{"gamma_" + which: gamma.cuda()})
        i = 1 if which == "post" else 3
        assert np.array_equal(f64(f.stats[i - 1]), np.full(rows, float(mean)))
        assert np.array_equal(f64(f.stats[i]), var[:, 0])
        # 4.5 of v^ and one of gamma
        check(f.h if which == "post" else f.y, want, bound(want, dt, 6), which)


def kept_forms(x, dtype):
    for kept in (None, "int8", "e4m3"):
        k = x if kept is None else K.act8_pack(x, x.shape[0], kept)
        yield kept, k, f64(x if kept is None else K.act8_unpack(k, x.shape[0], torch.float32))


# one row: dgamma is one product.  Three: sums of three.
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("cols", [72, 1000, 1031, 4096, 6144, 8192, 10240, 16384, 20000])
def test_parameter_gradients_of_rows_far_from_zero(cols, dtype, rows):
    """From given statistics: rows 300 standard deviations from zero."""
    dt = DTYPES[dtype]
    gen = torch.Generator().manual_seed(rows + cols)
    x = (300 + torch.randn(rows, cols, generator=gen)).to(dt).cuda()
    dy = torch.randn(rows, cols, generator=gen).to(dt).cuda()
    mean = f64(x).mean(1)
    mean32 = torch.tensor(mean, dtype=torch.float32, device="cuda")
    var32 = torch.ones(rows, dtype=torch.float32, device="cuda")
    gamma = (1 + 0.2 * torch.randn(cols, generator=gen)).cuda()
    rho = 1 / np.sqrt(1 + float(np.float32(1e-5)))
    for kept, k, xv in kept_forms(x, dt):
        terms = f64(dy) * (xv - f64(mean32)[:, None]) * rho
        want = terms.sum(0)
        # 4.5 of v^, one of the product, one per addition of a row's, in the block and
        # where the blocks' sums are added up (zeros add nothing)
        tol = (6 + 2 * rows) * U * np.abs(terms).sum(0)
        post = K.resnorm_backward(k, None, dy, None, (mean32, var32, None, None), rows, gamma_post=gamma,
                                  norm="layer", pre=False, has_res=False)
        check(post.dgamma_post, want, tol, ("post", kept))
        pre = K.resnorm_backward(None, k, None, dy, (None, None, mean32, var32), rows, gamma_pre=gamma,
                                 norm="layer", post=False, has_res=False)
        check(pre.dgamma_pre, want, tol, ("pre", kept))
        if kept:
            one = K.ln_backward_act8(k, dy, gamma, mean32, var32, rows)
            check(one[1], want, tol, ("layer", kept))
