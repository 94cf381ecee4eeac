"""Which data the gradients of RMSNormalization and ResidualNormalization read, as a
graph asks before it frees data between the forward and the backward (no device)."""
import itertools

import pytest

from _util import load_package

load_package()
from nnabla_ext_cuda_amd import binding as B  # noqa: E402


@pytest.fixture(autouse=True)
def _init():
    B.init()


@pytest.mark.parametrize("tc", ["float", "half"])
@pytest.mark.parametrize("checkpoint", ["", "int8", "e4m3"])
def test_rms(checkpoint, tc):
    f = B.RMSNormalization(B.context(type_config=tc), checkpoint=checkpoint)
    for i in range(2):
        assert f.grad_depends_input_data(i, 0) == (checkpoint == "")
        assert f.grad_depends_input_data(i, 1)
        assert not f.grad_depends_output_data(i, 0)


@pytest.mark.parametrize("tc", ["float", "half"])
@pytest.mark.parametrize("checkpoint", ["", "int8", "e4m3"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True)])
def test_residual(post, pre, norm, checkpoint, tc):
    layer = norm == "layer"
    for residual, gate, no_scale, no_bias in itertools.product((False, True), repeat=4):
        names = ["x"] + ["res"] * residual + ["gate"] * gate
        for k, on in (("post", post), ("pre", pre)):
            names += ["beta_" + k] * (on and layer and not no_bias) + ["gamma_" + k] * (on and not no_scale)
        f = B.ResidualNormalization(B.context(type_config=tc), norm=norm, post=post, pre=pre,
                                    residual=residual, gate=gate, no_scale=no_scale, no_bias=no_bias,
                                    checkpoint=checkpoint)
        read = {"x": (post or gate) and checkpoint == "", "res": False, "gate": True, "gamma_post": True,
                "gamma_pre": True, "beta_post": gate, "beta_pre": False}
        for i in range(len(names)):
            for j, name in enumerate(names):
                assert f.grad_depends_input_data(i, j) == read[name], (name, names)
            assert f.grad_depends_output_data(i, 0) == (pre and checkpoint == "")
            if pre:
                assert not f.grad_depends_output_data(i, 1)
