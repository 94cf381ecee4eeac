"""What the transformer-block functions refuse, without a GPU: the C-ABI's
argument checks (pointers that are never followed) and the Python wrappers';
and the oracle's own gradients against differences."""
import itertools

import numpy as np
import pytest
import torch

from _util import load_package
from oracle import step_ref as S

K = load_package()
L = K.lib()
EINVAL, EWORKSPACE, ERANGE, EALIAS = -1, -2, -3, -4
BASE = 0x7F0000000000


class Places:
    """Distinct fake addresses, 64 MiB apart."""

    def __init__(self):
        self.n = itertools.count(1)

    def __call__(self):
        return BASE + next(self.n) * (1 << 26)


def fwd_args(**over):
    p = Places()
    a = dict(x=p(), res=p(), gate=None, gate_kind=0, gate_rows=0, gp=p(), bp=None, gn=p(), bn=None,
             h=p(), y=p(), mp=None, vp=p(), mn=None, vn=p(), x8=None, x8s=None, h8=None, h8s=None, f=0,
             rows=8, cols=64, rs=1.0, bs=1.0, eps=1e-5, norm=0, post=1, pre=1, dtype=1, stream=None)
    a.update(over)
    return list(a.values())


def bwd_args(**over):
    p = Places()
    a = dict(x=p(), xs=None, h=p(), hs=None, f=0, dh=p(), dy=p(), gate=None, gate_kind=0, gate_rows=0,
             gp=p(), bp=None, gn=p(), mp=None, vp=p(), mn=None, vn=p(), dx=p(), dres=p(), dgate=None,
             dgp=p(), dbp=None, dgn=p(), dbn=None, accum=0, rows=8, cols=64, rs=1.0, bs=1.0, eps=1e-5,
             norm=0, post=1, pre=1, dtype=1, ws=p(), wsn=1 << 25, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(dtype=3), EINVAL), (dict(norm=2), EINVAL), (dict(post=0, pre=0, gp=None, gn=None), EINVAL),
    (dict(x=None), EINVAL), (dict(h=None), EINVAL), (dict(y=None), EINVAL), (dict(vp=None), EINVAL),
    (dict(vn=None), EINVAL), (dict(norm=1), EINVAL),                       # no means
    (dict(bp=BASE), EINVAL), (dict(bn=BASE), EINVAL),                      # RMS has no beta
    (dict(post=0), EINVAL),                                                # gamma_post without post
    (dict(pre=0), EINVAL),
    (dict(gate=BASE), EINVAL), (dict(gate_kind=1, gate_rows=1), EINVAL),
    (dict(gate=BASE, gate_kind=1, gate_rows=3), EINVAL), (dict(gate=BASE, gate_kind=1), EINVAL),
    (dict(gate=BASE, gate_kind=4, gate_rows=1), EINVAL),
    (dict(x8=BASE, f=1), EINVAL), (dict(x8=BASE, x8s=BASE + 65536, f=0), EINVAL),
    (dict(h8=BASE, h8s=BASE + 65536, f=3), EINVAL),
    (dict(rows=-1), EINVAL), (dict(cols=-1), EINVAL), (dict(cols=1 << 27), ERANGE),
    (dict(rows=1 << 40, cols=1 << 20), ERANGE),
    (dict(post=1, pre=0, gn=None, h8=BASE, h8s=BASE + 65536, f=1), EINVAL),
    (dict(rows=0), 0), (dict(cols=0), 0),
])
def test_forward_refusals(over, code):
    assert L.nblahip_resnorm_fwd(*fwd_args(**over)) == code


def test_forward_overlaps():
    a = fwd_args()
    x, res, gp, h, y, vp = a[0], a[1], a[5], a[9], a[10], a[12]
    n = 8 * 64 * 2
    for over in (dict(h=x + 2), dict(h=x - n + 2), dict(y=res + n - 2), dict(y=h), dict(y=h + 2),
                 dict(h=gp), dict(y=gp + 60 * 4), dict(vp=x), dict(vn=vp + 4), dict(h=vp - 2),
                 dict(x8=x, x8s=BASE, f=1), dict(x8=h + n - 1, x8s=BASE, f=1),
                 dict(x8=BASE, x8s=BASE + 511, f=2), dict(h8=y, h8s=BASE, f=2),
                 dict(gate=gp, gate_kind=1, gate_rows=2, y=gp + 64 * 4 + 4, gn=None)):
        assert L.nblahip_resnorm_fwd(*fwd_args(**over)) == EALIAS, over


@pytest.mark.parametrize("over,code", [
    (dict(dtype=-1), EINVAL), (dict(norm=-1), EINVAL), (dict(x=None), EINVAL), (dict(h=None), EINVAL),
    (dict(dy=None), EINVAL), (dict(pre=0, gn=None, dgn=None, dh=None), EINVAL), (dict(vp=None), EINVAL),
    (dict(vn=None), EINVAL), (dict(norm=1), EINVAL), (dict(bp=BASE), EINVAL), (dict(dbp=BASE), EINVAL),
    (dict(dbn=BASE), EINVAL), (dict(post=0), EINVAL), (dict(pre=0), EINVAL), (dict(dgate=BASE), EINVAL),
    (dict(f=1), EINVAL), (dict(f=5, xs=BASE, hs=BASE + 4096), EINVAL),
    (dict(gate=BASE, gate_kind=1, gate_rows=5), EINVAL), (dict(gate=BASE, gate_kind=2, gate_rows=0,
                                                               dgate=BASE + 2), EALIAS),
    (dict(ws=None), EWORKSPACE), (dict(wsn=16), EWORKSPACE), (dict(ws=BASE + 128), EWORKSPACE),
    (dict(rows=-3), EINVAL), (dict(cols=1 << 27), ERANGE), (dict(cols=0), 0),
])
def test_backward_refusals(over, code):
    assert L.nblahip_resnorm_bwd(*bwd_args(**over)) == code


def test_backward_overlaps():
    a = bwd_args()
    x, h, dh, dy, gp, vp, dx, dres, ws = a[0], a[2], a[5], a[6], a[10], a[14], a[17], a[18], a[34]
    for over in (dict(dx=dh + 2), dict(dx=x - 2), dict(dres=dy + 4), dict(dres=dx), dict(dgp=gp),
                 dict(dgp=vp), dict(dx=ws), dict(dgn=dx + 1000), dict(dres=h + 8),
                 dict(f=1, xs=BASE, hs=BASE + 4096, dx=x), dict(f=2, xs=BASE, hs=BASE + 4096, dres=h)):
        assert L.nblahip_resnorm_bwd(*bwd_args(**over)) == EALIAS, over


def test_rms_and_layer_refusals():
    p = Places()
    x, g, y, ms, dy, dx, dg, ws, sc, mean = (p() for _ in range(10))
    rms = L.nblahip_rms_fwd
    assert rms(None, g, y, ms, 4, 64, 1e-5, 1, None) == EINVAL
    assert rms(x, g, None, ms, 4, 64, 1e-5, 1, None) == EINVAL
    assert rms(x, g, y, None, 4, 64, 1e-5, 1, None) == EINVAL
    assert rms(x, g, y, ms, 4, 64, 1e-5, 7, None) == EINVAL
    assert rms(x, g, x + 2, ms, 4, 64, 1e-5, 1, None) == EALIAS
    assert rms(x, g, y, ms, 0, 64, 1e-5, 1, None) == 0
    b = lambda **k: L.nblahip_rms_bwd(*{**dict(x=x, s=None, f=0, dy=dy, g=g, ms=ms, dx=dx, dg=dg, a=0,
                                               b=0, r=4, c=64, e=1e-5, d=1, ws=ws, n=1 << 20,
                                               st=None), **k}.values())
    assert b(x=None) == EINVAL and b(dy=None) == EINVAL and b(ms=None) == EINVAL
    assert b(f=1) == EINVAL and b(f=3, s=sc) == EINVAL and b(d=5) == EINVAL
    assert b(ws=None) == EWORKSPACE and b(n=8) == EWORKSPACE and b(dx=dy + 2) == EALIAS
    l = lambda **k: L.nblahip_ln_bwd_act8(*{**dict(x=x, s=sc, f=1, dy=dy, g=g, m=mean, v=ms, dx=dx,
                                                   dg=dg, db=None, a=0, b=0, c=0, r=4, n=64, e=1e-5,
                                                   d=1, ws=ws, wn=1 << 20, st=None), **k}.values())
    assert l(f=0) == EINVAL and l(s=None) == EINVAL and l(m=None) == EINVAL and l(wn=0) == EWORKSPACE


def test_act8_refusals():
    p = Places()
    x, q, s = p(), p(), p()
    for f in (L.nblahip_act8_pack, L.nblahip_act8_unpack):
        a = (x, q, s) if f is L.nblahip_act8_pack else (q, s, x)
        assert f(*a, 4, 64, 0, 1, None) == EINVAL and f(*a, 4, 64, 1, 3, None) == EINVAL
        assert f(None, *a[1:], 4, 64, 1, 1, None) == EINVAL and f(*a[:2], None, 4, 64, 1, 1, None) == EINVAL
        assert f(*a, -1, 64, 1, 1, None) == EINVAL and f(*a, 4, 1 << 27, 1, 1, None) == ERANGE
        assert f(*a, 0, 64, 1, 1, None) == 0
    assert L.nblahip_act8_pack(x, x + 100, s, 4, 64, 1, 1, None) == EALIAS
    assert L.nblahip_act8_pack(x, q, q + 255, 4, 64, 1, 1, None) == EALIAS
    assert L.nblahip_act8_unpack(q, s, s - 2, 4, 64, 1, 1, None) == EALIAS
    assert [L.nblahip_act8_scales_per_row(c) for c in (-1, 0, 1, 32, 33, 4096)] == [0, 0, 1, 1, 2, 128]


def test_other_functions_refuse_bfloat16():
    p = Places()
    a = [p() for _ in range(6)]
    assert L.nblahip_ln_fwd(*a, 4, 64, 1e-5, 2, None) == EINVAL
    assert L.nblahip_ln_bwd_workspace_bytes(4, 64, 2) == 0
    assert L.nblahip_gn_fwd(*a, 2, 4, 16, 2, 1e-5, 2, None) == EINVAL
    assert L.nblahip_bn_fwd_infer(*a, 4, 4, 4, 1e-5, 2, None) == EINVAL


def test_workspace_sizes():
    w = L.nblahip_resnorm_bwd_workspace_bytes
    assert w(0, 64, 0, 0, 0, 1, 1, 1) == 0 and w(64, 64, 0, 0, 0, 1, 1, 9) == 0
    assert w(64, 64, 1, 5, 0, 1, 1, 1) == 0
    for rows, cols in ((1, 1), (16384, 4096), (7, 100000)):
        for g, n in ((0, 0), (1, 1), (2, 0)):
            b = w(rows, cols, g, n, 1, 1, 1, 2)
            assert b % 256 == 0 and 0 < b < 64 * rows * cols + (1 << 20)


def test_workspace_holds_a_partial_sum_per_gate_row():
    # one column, a gate row per row: a partial row (8 floats) per gate row
    n = (1 << 30) + 4096
    assert L.nblahip_resnorm_bwd_workspace_bytes(n, 1, 1, n, 0, 0, 1, 1) >= n * 32 * 2 + n * 16


def test_wrappers_refuse():
    x = torch.zeros(4, 64)
    with pytest.raises(TypeError, match="GPU"):
        K.rms_forward(x, None, 4)
    with pytest.raises(TypeError, match="GPU"):
        K.resnorm_forward(x, None, 4)
    with pytest.raises(TypeError, match="GPU"):
        K.act8_pack(x, 4)
    with pytest.raises(ValueError, match="rows"):
        K.rms_forward(x, None, 3)
    with pytest.raises(TypeError, match="dtype"):
        K.rms_forward(x.double(), None, 4)
    with pytest.raises(KeyError):
        K.act8_pack(x, 4, "int4")
    with pytest.raises(TypeError, match="Act8"):
        K.ln_backward_act8(x, x, None, None, None, 4)
    with pytest.raises(TypeError, match="codes"):
        K.rms_backward(K.Act8(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)),
                       x, None, None, 4)
    with pytest.raises(ValueError, match="scales"):
        K.rms_backward(K.Act8(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8)),
                       x, None, None, 4)
    with pytest.raises(ValueError, match="dh or dy"):
        K.resnorm_backward(x, x, None, None, (None,) * 4, 4)


# ------------------------------------------------- the oracle against itself
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("gate", [None, "rows", "full"])
def test_oracle_gradients_match_differences(gate, post, pre, norm):
    rng = np.random.default_rng(0)
    rows, cols, rs, bs, eps = 6, 10, 0.8, 0.5, 1e-3
    n = rng.standard_normal
    v = dict(x=n((rows, cols)), res=n((rows, cols)))
    if gate:
        v["gate"] = n((2 if gate == "rows" else rows, cols))
    for k, on in (("post", post), ("pre", pre)):
        if on:
            v["gamma_" + k] = 1 + 0.1 * n(cols)
            if norm == "layer":
                v["beta_" + k] = 0.1 * n(cols)
    dh, dy = n((rows, cols)), n((rows, cols)) if pre else None

    def loss(d):
        f = S.step_fwd(d["x"], d["res"], d.get("gate"), d.get("gamma_post"), d.get("beta_post"),
                       d.get("gamma_pre"), d.get("beta_pre"), norm, post, pre, rs, bs, eps)
        return (f["h"][0] * dh).sum() + ((f["y"][0] * dy).sum() if pre else 0.0), f

    _, f = loss(v)
    zero = np.zeros((rows, 1))
    stats = [f.get(k, zero) for k in ("mean_post", "var_post", "mean_pre", "var_pre")]
    g = S.step_bwd(v["x"], f["h"][0], dh, dy, stats, v.get("gate"), gate == "full", v.get("gamma_post"),
                   v.get("beta_post"), v.get("gamma_pre"), norm, post, pre, True, rs, bs, eps)
    for name, t in v.items():
        want = g["d" + name][0]
        step = 1e-6
        for i in itertools.islice(np.ndindex(t.shape), 0, None, 7):
            old = t[i]
            t[i] = old + step
            up, _ = loss(v)
            t[i] = old - step
            down, _ = loss(v)
            t[i] = old
            # central differences: error step^2 * third derivative (about 1e-11
            # here) + 2^-53 * |loss| / step (about 1e-8)
            assert abs((up - down) / (2 * step) - want[i]) < 1e-6 * (1 + abs(want[i])), (name, i)


def test_oracle_codes_are_nearest():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((20, 70)) * np.exp(rng.standard_normal((20, 70)))
    vals = S.e4m3_values()
    vals = vals[np.isfinite(vals)]
    for form, grid in (("int8", np.arange(-127, 128.0)), ("e4m3", vals)):
        q, code = S.act8(x, form)
        z = x / np.repeat(np.ldexp(1.0, code.astype(int) - 127), 32, 1)[:, :70]
        best = np.abs(z[:, :, None] - grid).min(2)
        assert np.array_equal(np.abs(z - q), best) and np.isin(q, grid).all()
        top = np.abs(z).max()
        assert top < 127.5 if form == "int8" else top <= 448
