"""The MX4 oracle against closed forms and another computation of the same values (CPU only)."""

import pytest
import torch

from oracle import mx4


def test_hand_written_blocks():
    y = torch.zeros(1, 64)
    y[0, 0], y[0, 1], y[0, 2], y[0, 3] = 6.5, -0.25, 0.75, 5.0  # block 0: scale 1
    y[0, 32], y[0, 33] = 7.0, -14.0                             # block 1: 14 / 2 = 7 is too much for 2, so 4
    code, s = mx4.encode(y)
    assert s.tolist() == [[127, 129]]
    # 6.5 -> 6; -0.25 is half way to the odd code 1 -> -0; 0.75 -> 1 (even code 2); 5 -> 4 (even code 6)
    assert code[0, :4].tolist() == [7, 8, 2, 6]
    # 1.75 -> 2 (code 4, the even one), -3.5 -> -4 (code 6 and the sign)
    assert code[0, 32].item() == 4 and code[0, 33].item() == 14
    v = mx4.decode(mx4.pack(code), s)
    assert v[0, :4].tolist() == [6.0, 0.0, 1.0, 4.0]


@pytest.mark.parametrize("mag", [1e-30, 2.0 ** -66, 1e-3, 1.0, 1e4, 2.0 ** 34])
def test_no_value_is_off_by_more_than_half_a_step(mag):
    g = torch.Generator().manual_seed(3)
    y = torch.randn(40, 256, generator=g, dtype=torch.float64) * mag
    code, s = mx4.encode(y)
    v = mx4.decode(mx4.pack(code), s)
    f = torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s.long() - 127).repeat_interleave(32, -1)
    fine = (s != mx4.NAN).repeat_interleave(32, -1)
    m = (y / f).abs()
    half = torch.where(m < 2, 0.25, torch.where(m < 4, 0.5, 1.0)) * f
    assert ((v - y).abs()[fine] <= half[fine]).all()
    assert torch.isnan(v[~fine]).all()


def test_limits_of_the_scale():
    y = torch.zeros(6, 32, dtype=torch.float64)
    y[0, 5] = 7 * 2.0 ** 32 * (1 - 2.0 ** -20)
    y[1, 5] = 7 * 2.0 ** 32
    y[2, 5] = float("inf")
    y[3, 5] = float("nan")
    y[4, 5] = 1e-40
    assert mx4.scale_bytes(y)[:, 0].tolist() == [159, 255, 255, 255, 63, 63]


def test_pack_order():
    codes = torch.arange(64, dtype=torch.uint8).view(2, 32) % 16
    p = mx4.pack(codes)
    assert p.shape == (2, 16) and p[0, 1].item() == 2 | 3 << 4
    one = torch.full((2, 1), 127, dtype=torch.uint8)
    assert torch.equal(mx4.decode(p, one).abs(), mx4.LEVELS[codes.long() & 7])


def test_attend_against_a_plain_softmax():
    g = torch.Generator().manual_seed(4)
    q = torch.randn(3, 5, 48, generator=g)
    x, r = torch.randn(20, 32, generator=g), torch.randn(20, 16, generator=g)
    o, lse, w = mx4.attend(q, x, r, [20, 0, 7], 0.3)
    s = (q[2].double() @ torch.cat((x, r), -1)[:7].double().t()) * 0.3
    torch.testing.assert_close(o[2], torch.softmax(s, -1) @ x[:7].double())
    torch.testing.assert_close(lse[2], s.exp().sum(-1).log())
    assert (o[1] == 0).all() and (lse[1] == float("-inf")).all()
    assert (w >= o.abs() - 1e-12).all()
