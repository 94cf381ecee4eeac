"""Random residual steps - sizes, types, norms, gates, 8-bit copies, missing
gradients, accumulation, tensors at any element - against the float64 oracle."""
import random

import pytest
import torch

from _step import Step, close, f64
from _util import load_package

K = load_package()
pytestmark = pytest.mark.gpu


def at_element(t, off):
    """The same values at `off` elements past an allocation's start."""
    if t is None:
        return None
    flat = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)
    v = flat[off:off + t.numel()].view(t.shape)
    v.copy_(t)
    return v


@pytest.mark.parametrize("seed", range(120))
def test_random_step(seed):
    rng = random.Random(seed)
    dtype = rng.choice(["f32", "f16", "bf16"])
    cols = int(round(2 ** rng.uniform(0, 14.2)))
    if rng.random() < 0.5:
        cols = max(8, cols // 8 * 8)
    rows = max(1, min(int(round(2 ** rng.uniform(0, 12))), 400000 // cols))
    samples = 1
    gate = rng.choice(["none", "channel", "sample", "full"])
    if gate == "sample":
        samples = rng.randint(1, min(rows, 9))
        rows = rows // samples * samples
    post, pre = rng.choice([(True, True), (True, False), (False, True)])
    st = Step(rows, cols, dtype, rng.choice(["rms", "layer"]), post, pre, rng.random() < 0.8, gate, samples,
              rs=rng.choice([1.0, 0.7]), bs=rng.choice([1.0, 0.4]), eps=rng.choice([1e-5, 1e-3]), seed=seed,
              affine=rng.random() < 0.85)
    if rng.random() < 0.3:
        off = rng.randint(1, 8)
        for name in ("x", "res", "dh", "dy"):
            setattr(st, name, at_element(getattr(st, name), off))
        if st.full:
            st.gate = at_element(st.gate, off)
        if st.gn is not None:
            st.gn = at_element(st.gn, rng.randint(0, 3))
    kept = rng.choice([None, None, "int8", "e4m3"])
    f = K.resnorm_forward(st.x, st.res, rows, checkpoint=kept, **st.args())
    st.check_fwd(f)
    x, h = (f.x8, f.h8) if kept else (st.x, f.h)
    xv, hv = (None if t is None else f64(K.act8_unpack(t, rows, torch.float32) if kept else t)
              for t in (x, h))
    if kept:
        for t, c in ((st.x, f.x8), (f.h, f.h8)):
            if c is not None:
                want = K.act8_pack(t, rows, kept)
                assert torch.equal(c.scales, want.scales)
                assert torch.equal(c.codes.view(torch.uint8), want.codes.view(torch.uint8))
    ref = st.oracle_bwd(xv, hv, f.stats)
    g = K.resnorm_backward(x, h, st.dh, st.dy, f.stats, rows, has_res=st.res is not None, **st.args())
    st.check_grads(g, ref)
    # some gradients only, added onto old ones
    need = [rng.random() < 0.6 for _ in range(7)]
    accum = [rng.random() < 0.5 for _ in range(7)]
    old = [None if t is None else torch.randn_like(t) for t in g]
    part = K.resnorm_backward(x, h, st.dh, st.dy, f.stats, rows, has_res=st.res is not None, need=need,
                              accum=accum, out=K.ResNormGrads(*[None if t is None else t.clone() for t in old]),
                              **st.args())
    for i, name in enumerate(part._fields):
        assert (part[i] is None) == (g[i] is None or not need[i]), name
        if part[i] is None:
            continue
        value, terms = ref[name]
        if accum[i]:
            o = f64(old[i]).reshape(value.shape)
            value, terms = value + o, terms + abs(o)
        close(part[i], value, terms, rows, cols, name, column_sum=name.startswith(("dgamma", "dbeta")) or
              (name == "dgate" and not st.full))
