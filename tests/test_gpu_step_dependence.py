"""What RMSNormalization and ResidualNormalization declare not to read after the
forward may be gone: it holds NaN here, and the gradients have the same bits."""
import itertools

import numpy as np
import pytest

from _util import load_package

load_package()
from nnabla_ext_cuda_amd import binding as B  # noqa: E402

pytestmark = pytest.mark.gpu
SHAPE, P = (2, 9, 72), (72,)


@pytest.fixture(autouse=True)
def _init():
    B.init()


def gradients(make, shapes, n_out, half, gone):
    rng = np.random.default_rng(5)
    f = make()
    ins, outs = [B.Variable(s) for s in shapes], [B.Variable(SHAPE) for _ in range(n_out)]
    for v, s in zip(ins, shapes):
        v.set_data(rng.standard_normal(s) + 0.5, half=half)
    f.setup(ins, outs)
    f.forward(ins, outs)
    for v in outs:
        v.set_grad(rng.standard_normal(SHAPE), half=half)
    if gone:
        freed = 0
        for j, (v, s) in enumerate(zip(ins, shapes)):
            if not any(f.grad_depends_input_data(i, j) for i in range(len(ins))):
                v.set_data(np.full(s, np.nan), half=half)
                freed += 1
        for o, v in enumerate(outs):
            if not any(f.grad_depends_output_data(i, o) for i in range(len(ins))):
                v.set_data(np.full(SHAPE, np.nan), half=half)
                freed += 1
        assert freed
    f.backward(ins, outs)
    return [v.g for v in ins]


def check(make, shapes, n_out, half):
    kept = gradients(make, shapes, n_out, half, False)
    for a, b in zip(kept, gradients(make, shapes, n_out, half, True)):
        assert np.isfinite(a).all() and np.array_equal(a, b)


@pytest.mark.parametrize("tc", ["float", "half"])
@pytest.mark.parametrize("checkpoint", ["", "int8", "e4m3"])
def test_rms(checkpoint, tc):
    check(lambda: B.RMSNormalization(B.context(type_config=tc), batch_axis=(0, 1), checkpoint=checkpoint),
          [SHAPE, P], 1, tc == "half")


@pytest.mark.parametrize("tc", ["float", "half"])
@pytest.mark.parametrize("checkpoint", ["", "int8"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True)])
def test_residual(post, pre, norm, checkpoint, tc):
    for residual, gate in itertools.product((False, True), (None, P, SHAPE)):
        shapes = [SHAPE] + [SHAPE] * residual + ([] if gate is None else [gate])
        for on in (post, pre):
            shapes += [P] * (on * (2 if norm == "layer" else 1))
        check(lambda: B.ResidualNormalization(
            B.context(type_config=tc), batch_axis=(0, 1), norm=norm, post=post, pre=pre, residual=residual,
            gate=gate is not None, checkpoint=checkpoint), shapes, 1 + pre, tc == "half")
