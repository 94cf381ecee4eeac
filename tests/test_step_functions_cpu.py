"""RMSNormalization and ResidualNormalization functions without a device: the
registry, and the arguments that setup refuses before it looks for a device."""
import pytest

from _util import load_package

load_package()
from nnabla_ext_cuda_amd import binding as B  # noqa: E402


@pytest.fixture(autouse=True)
def _init():
    B.init()


def V(*shape):
    return B.Variable(shape)


def test_registered_for_float_and_half():
    for tc in ("float", "half"):
        assert B.RMSNormalization(B.context(type_config=tc)).name == "RMSNormalizationHip"
        assert B.ResidualNormalization(B.context(type_config=tc)).name == "ResidualNormalizationHip"
    cpu = {"backends": "cpu:float", "array_class": "CpuArray", "device_id": "0"}
    for make in (B.RMSNormalization, B.ResidualNormalization):
        with pytest.raises(B.NblaError, match="No implementation"):
            make(cpu)


def test_checkpoint_names():
    for make in (B.RMSNormalization, B.ResidualNormalization):
        with pytest.raises(B.NblaError, match="checkpoint"):
            make(B.context(), checkpoint="fp8")


@pytest.mark.parametrize("kw,inputs,outputs,text", [
    (dict(), [(4, 8)], [(4, 8)], "expects 2 inputs"),
    (dict(no_scale=True), [(4, 8), (8,)], [(4, 8)], "expects 1 inputs"),
    (dict(), [(4, 8), (8,)], [(4, 8), (4, 8)], "1 output"),
    (dict(), [(4, 8), (4,)], [(4, 8)], "8 elements"),
    (dict(batch_axis=()), [(4, 8), (8,)], [(4, 8)], "must not be empty"),
    (dict(batch_axis=(2,)), [(4, 8), (8,)], [(4, 8)], "out of range"),
    (dict(batch_axis=(1,)), [(4, 8), (4,)], [(4, 8)], "leading axes"),
    (dict(batch_axis=(0, 0)), [(4, 8), (8,)], [(4, 8)], "leading axes"),
])
def test_rms_refusals(kw, inputs, outputs, text):
    f = B.RMSNormalization(B.context(), **kw)
    with pytest.raises(B.NblaError, match=text):
        f.setup([V(*s) for s in inputs], [V(*s) for s in outputs])


X, P = (4, 8), (8,)


@pytest.mark.parametrize("kw,inputs,n_out,text", [
    (dict(norm="batch"), [X, X, P, P], 2, "norm must be"),
    (dict(post=False, pre=False), [X, X], 1, "post, pre or both"),
    (dict(), [X, X, P], 2, "expects 4 inputs"),
    (dict(norm="layer"), [X, X, P, P], 2, "expects 6 inputs"),
    (dict(gate=True), [X, X, P, P], 2, "expects 5 inputs"),
    (dict(), [X, X, P, P], 1, "2 output"),
    (dict(pre=False), [X, X, P], 2, "1 output"),
    (dict(), [X, (8, 4), P, P], 2, "shape of x"),
    (dict(), [X, X, (4,), P], 2, "8 elements"),
    (dict(gate=True), [X, X, (3, 8), P, P], 2, "gate must have"),
    (dict(gate=True), [X, X, (7,), P, P], 2, "gate must have"),
    (dict(batch_axis=(1,)), [X, X, (4,), (4,)], 2, "leading axes"),
])
def test_residual_refusals(kw, inputs, n_out, text):
    f = B.ResidualNormalization(B.context(), **kw)
    with pytest.raises(B.NblaError, match=text):
        f.setup([V(*s) for s in inputs], [V(*X) for _ in range(n_out)])
