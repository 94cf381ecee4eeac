"""8-bit copies of activations: codes and scales equal the oracle's exactly (the
scale is a power of two, so the one rounding is fixed by the definition), and
the values read back are code * scale rounded once."""
import numpy as np
import pytest
import torch

from _step import DTYPES, f64
from _util import load_package
from oracle import step_ref as S

K = load_package()
pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 31), (1, 32), (3, 33), (5, 100), (7, 1000), (64, 128), (129, 2560), (1000, 8),
          (2, 40001), (300, 4096)]


def codes_as_values(a):
    if a.codes.dtype == torch.int8:
        return f64(a.codes)
    return S.e4m3_values()[a.codes.view(torch.uint8).cpu().numpy()]


def make(rows, cols, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed + rows + cols)
    x = torch.randn(rows, cols, generator=gen)
    x = x * torch.where(torch.rand(cols, generator=gen) < 0.05, 30.0, 1.0)
    return x.to(DTYPES[dtype]).cuda()


def check_pack(x, outer, form):
    a = K.act8_pack(x, outer, form)
    xv = f64(x).reshape(outer, -1)
    q, code = S.act8(xv, form)
    assert np.array_equal(a.scales.cpu().numpy(), code)
    assert np.array_equal(codes_as_values(a).reshape(xv.shape), q)
    for out in DTYPES.values():
        got = K.act8_unpack(a, outer, out)
        assert got.shape == x.shape and got.dtype == out
        want = torch.from_numpy(S.act8_value(q, code).reshape(x.shape)).to(torch.float32).to(out)
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(), want.nan_to_num())
    return a


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_pack_and_unpack(shape, dtype, form):
    check_pack(make(*shape, dtype), shape[0], form)


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_every_half_and_every_rounding_border(form, dtype):
    """All 65536 bit patterns of a 16-bit float (non-finite among them), each in
    a group of its own with a fixed largest magnitude, and float values next to
    every border between two codes."""
    if dtype == "f32":
        grid = np.arange(-127, 127) + 0.5 if form == "int8" else np.sort(S.e4m3_values()[
            np.isfinite(S.e4m3_values())])
        mids = grid if form == "int8" else (grid[1:] + grid[:-1]) / 2
        top = 127.0 if form == "int8" else 448.0
        vals = np.concatenate([mids, np.nextafter(mids.astype(np.float32), np.float32(np.inf)),
                               np.nextafter(mids.astype(np.float32), np.float32(-np.inf))])
        x = np.zeros((len(vals), 32), np.float32)
        x[:, 0], x[:, 5] = top, vals
        x = torch.from_numpy(x).cuda()
    else:
        bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
        x = torch.zeros(65536, 32, dtype=torch.int16)
        x[:, 7] = bits
        x[:, 3] = torch.tensor([1.75], dtype=DTYPES[dtype]).view(torch.int16)
        x = x.view(DTYPES[dtype]).cuda()
    check_pack(x, x.shape[0], form)


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_scale_borders_and_extremes(form):
    """Largest magnitudes at which the scale steps, zeros, subnormals, the
    largest float."""
    tops = []
    for e in (-149, -130, -127, -126, -120, -113, -60, -1, 0, 1, 60, 127):
        for m in (1.0, 1.75, 1.7500001, 1.9921874, 1.9921875, 1.9999999):
            t = np.float32(np.ldexp(m, e))
            if np.isfinite(t):
                tops += [t, -t]
    tops += [0.0, -0.0, np.finfo(np.float32).max, np.inf, -np.inf, np.nan]
    x = np.zeros((len(tops), 40), np.float32)
    x[:, 2], x[:, 20], x[:, 35] = tops, np.array(tops, np.float32) / 3, 1.0
    check_pack(torch.from_numpy(x).cuda(), len(tops), form)


def test_views_at_any_element_offset():
    for off in range(1, 9):
        flat = make(1, 64 * 72 + 16, "f16", seed=off)[0]
        x = flat[off:off + 64 * 72].view(64, 72)
        assert x.is_contiguous()
        check_pack(x, 64, "int8")


def test_only_the_copy_is_written():
    x = make(5, 100, "f16")
    codes = torch.full((5 * 100 + 64,), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((5 * 4 + 64,), 77, dtype=torch.uint8, device="cuda")
    K.check(K.lib().nblahip_act8_pack(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), 5, 100, 1, 1,
                                      torch.cuda.current_stream().cuda_stream))
    assert (codes[500:] == 77).all() and (scales[20:] == 77).all()
    out = torch.full((500 + 64,), 7.0, device="cuda", dtype=torch.float32)
    a = K.Act8(codes[:500].view(5, 100), scales[:20].view(5, 4))
    K.act8_unpack(a, 5, torch.float32, out=out[:500].view(5, 100))
    assert (out[500:] == 7).all()
