"""RMSNormalization and ResidualNormalization through the Function classes, as a
graph runs them, against the float64 oracle (tolerances: _step.py)."""
import numpy as np
import pytest
import torch

from _step import depth
from _util import load_package
from oracle import step_ref as S

load_package()
from nnabla_ext_cuda_amd import binding as B  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(autouse=True)
def _init():
    B.init()


def stored(a, half):
    """The values that an array holds after Variable.set_data / set_grad, which
    take float32 and round that to half."""
    a = np.float32(a)
    return np.float64(np.float16(a)) if half else np.float64(a)


def put(v, a, half=False):
    v.set_data(a, half=half)
    return stored(a, half)


def close(got, ref, shape, name, half, column_sum=False):
    value, terms = ref
    t = torch.float16 if half else torch.float32
    bound = torch.finfo(t).eps / 2 * np.abs(value) + depth(*shape, column_sum) * 2.0 ** -24 * terms
    if half:
        bound = bound + 2.0 ** -25
    err = np.abs(np.float64(got).reshape(value.shape) - value)
    assert (err <= bound).all(), (name, float((err - bound).max()))


@pytest.mark.parametrize("tc", ["float", "half"])
@pytest.mark.parametrize("checkpoint", ["", "int8", "e4m3"])
@pytest.mark.parametrize("shape,batch_axis", [((6, 40), (0,)), ((3, 5, 96), (0, 1)), ((4, 3, 8, 9), (0, 1)),
                                              ((2, 33, 1030), (1, 0))])
def test_rms_normalization(shape, batch_axis, checkpoint, tc):
    half = tc == "half"
    rng = np.random.default_rng(0)
    nb = len(batch_axis)
    rows, cols = int(np.prod(shape[:nb])), int(np.prod(shape[nb:]))
    f = B.RMSNormalization(B.context(type_config=tc), batch_axis=batch_axis, eps=EPS, checkpoint=checkpoint)
    x, g, y = B.Variable(shape), B.Variable(shape[nb:]), B.Variable(shape)
    xv = put(x, rng.standard_normal(shape) * 2, half).reshape(rows, cols)
    gv = put(g, 1 + 0.1 * rng.standard_normal(shape[nb:]), half).reshape(-1)
    f.setup([x, g], [y])
    f.forward([x, g], [y])
    yr, yt, mean, var = S.norm_fwd(xv, gv, None, "rms", EPS)
    close(y.d, (yr, yt), (rows, cols), "y", half)
    dy = rng.standard_normal(shape)
    y.set_grad(dy, half=half)
    dyv = stored(dy, half).reshape(rows, cols)
    kept = S.act8_value(*S.act8(xv, checkpoint)) if checkpoint else xv
    if checkpoint:
        x.set_data(np.zeros(shape))        # the backward reads the copy
    f.backward([x, g], [y])
    dx, dg, _ = S.norm_bwd(kept, dyv, gv, mean, var, "rms", EPS)
    # the mean squares are float32 values the oracle has in 64 bits: inside depth
    close(x.g, dx, (rows, cols), "dx", half)
    close(g.g, dg, (rows, cols), "dgamma", half, column_sum=True)
    assert g.stored_dtype(1) == ("half" if half else "float")
    before = x.g
    f.backward([x, g], [y], propagate_down=[True, False], accum=[True, False])
    close(x.g, (before.reshape(rows, cols) + dx[0], dx[1] + np.abs(dx[0])), (rows, cols), "accumulated", half)


@pytest.mark.parametrize("tc", ["float", "half"])
@pytest.mark.parametrize("checkpoint", ["", "e4m3"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("post,pre,residual,gate", [(True, True, True, None), (True, True, True, (72,)),
                                                    (True, False, False, (2, 72)), (False, True, True, "x"),
                                                    (False, True, True, None)])
def test_residual_normalization(post, pre, residual, gate, norm, checkpoint, tc):
    half, shape, rows, cols = tc == "half", (2, 11, 72), 22, 72
    rng = np.random.default_rng(1)
    layer = norm == "layer"
    f = B.ResidualNormalization(B.context(type_config=tc), batch_axis=(0, 1), norm=norm, post=post, pre=pre,
                                residual=residual, gate=gate is not None, res_scale=0.75, branch_scale=0.5,
                                eps=EPS, checkpoint=checkpoint)
    names, ins, val = [], [], {}

    def add(name, a, s=shape):
        v = B.Variable(s)
        names.append(name)
        ins.append(v)
        val[name] = put(v, a, half)
    n = rng.standard_normal
    add("x", n(shape) * 2 + 0.5)
    if residual:
        add("res", n(shape) * 3)
    if gate is not None:
        s = shape if gate == "x" else gate
        add("gate", n(s), s)
    for k, on in (("post", post), ("pre", pre)):
        if on and layer:
            add("beta_" + k, 0.2 * n(72), (72,))
        if on:
            add("gamma_" + k, 1 + 0.1 * n(72), (72,))
    outs = [B.Variable(shape) for _ in range(2 if pre else 1)]
    f.setup(ins, outs)
    f.forward(ins, outs)
    full = gate == "x"
    m = {k: v.reshape(rows, cols) if k in ("x", "res") else v.reshape(-1, cols) if k == "gate" else v
         for k, v in val.items()}
    ref = S.step_fwd(m["x"], m.get("res"), m.get("gate"), m.get("gamma_post"), m.get("beta_post"),
                     m.get("gamma_pre"), m.get("beta_pre"), norm, post, pre, 0.75, 0.5, EPS)
    close(outs[0].d, ref["h"], (rows, cols), "h", half)
    if pre:
        close(outs[1].d, ref["y"], (rows, cols), "y", half)
    dh = n(shape)
    outs[0].set_grad(dh, half=half)
    dy = None
    if pre:
        dy = n(shape)
        outs[1].set_grad(dy, half=half)
    xk, hk = m["x"], np.float64(outs[0].d).reshape(rows, cols)
    if checkpoint:
        xk, hk = (S.act8_value(*S.act8(t, checkpoint)) for t in (xk, hk))
    zero = np.zeros((rows, 1))
    stats = [ref.get(k, zero) for k in ("mean_post", "var_post", "mean_pre", "var_pre")]
    want = S.step_bwd(xk, hk, stored(dh, half).reshape(rows, cols),
                      None if dy is None else stored(dy, half).reshape(rows, cols),
                      stats, m.get("gate"), full, m.get("gamma_post"), m.get("beta_post"),
                      m.get("gamma_pre"), norm, post, pre, residual, 0.75, 0.5, EPS)
    f.backward(ins, outs)
    # the statistics kept are those of h before its rounding, in float32; the
    # oracle's are the same in 64 bits
    for name, v in zip(names, ins):
        close(v.g, want["d" + name], (rows, cols), "d" + name, half,
              column_sum=name not in ("x", "res") and not (name == "gate" and full))
    # one input at a time, added onto what is there
    first = [v.g.copy() for v in ins]
    for i in range(len(ins)):
        pd = [k == i for k in range(len(ins))]
        f.backward(ins, outs, propagate_down=pd, accum=pd)
        for k, v in enumerate(ins):
            twice = np.float64(first[k]) * (2 if k <= i else 1)
            step = 2.0 ** -11 if half else 2.0 ** -22
            assert (np.abs(v.g - twice) <= step * np.abs(twice) * 2 + 2.0 ** -24).all(), names[k]


@pytest.mark.parametrize("checkpoint", ["", "int8"])
def test_no_rows(checkpoint):
    f = B.RMSNormalization(B.context(), checkpoint=checkpoint)
    x, g, y = B.Variable((0, 40)), B.Variable((40,)), B.Variable((0, 40))
    put(g, np.ones(40))
    f.setup([x, g], [y])
    f.forward([x, g], [y])
    f.backward([x, g], [y], [True, True], [False, False])
    assert (np.asarray(g.g) == 0).all()
    r = B.ResidualNormalization(B.context(), no_scale=True, checkpoint=checkpoint)
    res, h, z = B.Variable((0, 40)), B.Variable((0, 40)), B.Variable((0, 40))
    r.setup([x, res], [h, z])
    r.forward([x, res], [h, z])
    r.backward([x, res], [h, z], [True, True], [False, False])


def test_the_same_variable_as_block_output_and_residual():
    shape = (9, 64)
    rng = np.random.default_rng(2)
    f = B.ResidualNormalization(B.context(), norm="rms", no_scale=True)
    x, h, y = (B.Variable(shape) for _ in range(3))
    xv = put(x, rng.standard_normal(shape))
    f.setup([x, x], [h, y])
    f.forward([x, x], [h, y])
    dh, dy = (np.float64(np.float32(rng.standard_normal(shape))) for _ in range(2))
    h.set_grad(dh)
    y.set_grad(dy)
    f.backward([x, x], [h, y], accum=[False, True])
    ref = S.step_fwd(xv, xv, None, None, None, None, None, "rms", True, True, 1, 1, EPS)
    zero = np.zeros((9, 1))
    stats = [zero, ref["var_post"], zero, ref["var_pre"]]
    g = S.step_bwd(xv, np.float64(h.d), dh, dy, stats, None, False, None, None, None, "rms", True, True,
                   True, 1, 1, EPS)
    close(x.g, (g["dx"][0] + g["dres"][0], g["dx"][1] + g["dres"][1]), shape, "dx + dres", False)
