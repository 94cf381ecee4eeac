"""Steps on tensors whose element offsets pass 32 bits (and byte offsets 33), and
on many rows of a column: every row is one of few, so a row's answer is that of
a small call."""
import pytest
import torch

from _util import load_package

K = load_package()
pytestmark = pytest.mark.gpu

COPIES = (1 << 16) + 1


def repeated(t, n):
    return t.repeat(n, 1)


def same(big, small, n):
    """Every run of small's rows in big equals small, bit for bit."""
    big, small = big.view(n, *small.shape), small.contiguous()
    if big.dtype == torch.float8_e4m3fn:
        big, small = big.view(torch.uint8), small.view(torch.uint8)
    step = max(1, (1 << 26) // max(1, small.numel()))
    return all(bool((big[i:i + step] == small).all()) for i in range(0, n, step))


@pytest.mark.parametrize("cols", [2048, 2050])
def test_offsets_past_32_bits(cols):
    gen = torch.Generator(device="cuda").manual_seed(1)

    def rnd(*s):
        return torch.randn(*s, device="cuda", generator=gen)
    rows = 33
    x, res, dh, dy = (rnd(rows, cols).bfloat16() for _ in range(4))
    gp, gn = rnd(cols), rnd(cols)
    args = dict(gamma_post=gp, gamma_pre=gn, res_scale=0.5)
    small = K.resnorm_forward(x, res, rows, checkpoint="int8", **args)
    n = COPIES
    big_x = repeated(x, n)
    assert big_x.numel() > 1 << 32
    big = K.resnorm_forward(big_x, repeated(res, n), rows * n, checkpoint="int8", **args)
    for a, b in ((big.h, small.h), (big.y, small.y), (big.x8.codes, small.x8.codes),
                 (big.h8.codes, small.h8.codes), (big.x8.scales, small.x8.scales),
                 (big.h8.scales, small.h8.scales)):
        assert same(a, b, n)
    for a, b in zip(big.stats, small.stats):
        assert a is None and b is None or same(a, b, n)
    need = (True, True) + (False,) * 5
    for kept in (False, True):
        k = (lambda f, t: (f.x8, f.h8)) if kept else (lambda f, t: (t, f.h))
        want = K.resnorm_backward(*k(small, x), dh, dy, small.stats, rows, need=need, **args)
        got = K.resnorm_backward(*k(big, big_x), repeated(dh, n), repeated(dy, n), big.stats, rows * n,
                                 need=need, **args)
        assert same(got.dx, want.dx, n) and same(got.dres, want.dres, n)
    packed = K.act8_pack(big_x, rows * n)
    assert same(packed.codes, small.x8.codes, n) and same(packed.scales, small.x8.scales, n)
    assert same(K.act8_unpack(packed, rows * n, torch.bfloat16),
                K.act8_unpack(small.x8, rows, torch.bfloat16), n)


def test_long_rows_past_32_bits():
    gen = torch.Generator(device="cuda").manual_seed(2)
    rows, cols, n = 3, 40000, 36000
    x, dy = (torch.randn(rows, cols, device="cuda", generator=gen).half() for _ in range(2))
    y, ms = K.rms_forward(x, None, rows)
    big = repeated(x, n)
    assert big.numel() > 1 << 32
    by, bms = K.rms_forward(big, None, rows * n)
    assert same(by, y, n) and same(bms, ms, n)
    dx, _ = K.rms_backward(x, dy, None, ms, rows, need=(True, False))
    bdx, _ = K.rms_backward(big, repeated(dy, n), None, bms, rows * n, need=(True, False))
    assert same(bdx, dx, n)
