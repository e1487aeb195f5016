"""Rotary positions on the GPU against angles reduced in exact arithmetic and pairs turned in float64.

Tolerance: sine and cosine are formed in FP32 from an angle of at most an eighth of a
turn (three roundings of the angle, the series' own, the scale): off by at most 2^-22 each, times the scale. With the
products' and the sum's roundings a result is off by at most 2^-21 scale (|a| + |b|),
then rounded once, by half a step of its type (for fp16 2^-25 below its normal range).
"""

import math
from fractions import Fraction

import pytest
import torch

from mla_kv_quant_amd import rotary

pytestmark = pytest.mark.gpu
DEV = "cuda"
PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def expected(x, positions, rope):
    """float64 results and their tolerance for ``x [T, H, dim]`` (CPU)."""
    n = rope.dim // 2
    turn = [[float((Fraction(p) * Fraction(f) / (2 * PI)) % 1) for f in rope.inv_freq] for p in positions.tolist()]
    w = torch.tensor(turn, dtype=torch.float64).view(len(positions), 1, n) * (2 * math.pi)
    x = x.double()
    a, b = (x[..., 0::2], x[..., 1::2]) if rope.interleaved else (x[..., :n], x[..., n:])
    u, v = rope.scale * (a * w.cos() - b * w.sin()), rope.scale * (b * w.cos() + a * w.sin())
    off = 2.0 ** -21 * abs(rope.scale) * (a.abs() + b.abs())
    join = (lambda p, q: torch.stack((p, q), -1).flatten(-2)) if rope.interleaved else (lambda p, q: torch.cat((p, q), -1))
    return join(u, v), join(off, off)


def check(got, x, positions, rope):
    want, off = expected(x.cpu().view(x.shape[0], -1, rope.dim), positions.cpu(), rope)
    got = got.cpu().double().reshape(want.shape)
    tol = off + torch.finfo(x.dtype).eps / 2 * want.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    bad = (got - want).abs() > tol
    assert not bad.any(), (bad.sum().item(), ((got - want).abs() / (tol + 1e-300)).max().item())


def inputs(T, H, dim, dtype, seed=0, far=200000):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(T, H, dim, generator=g).to(dtype).to(DEV)
    k = torch.randn(T, dim, generator=g).to(dtype).to(DEV)
    return torch.randint(0, far, (T,), generator=g).to(DEV), q, k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dim", [2, 6, 32, 64, 80, 128, 512])
def test_values(dim, interleaved, dtype):
    rope = rotary.Rotary(dim, interleaved=interleaved, scale=1.25, inv_freq=rotary.frequencies(dim)[0], device=DEV)
    p, q, k = inputs(37, 5, dim, dtype, dim)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    assert rotary.apply_rotary(rope, p, q, k, qo, ko) == (qo, ko)
    check(qo, q, p, rope)
    check(ko, k, p, rope)


@pytest.mark.parametrize("T,H", [(1, 1), (1, 16), (3, 128), (257, 40), (2049, 16), (33000, 1)])
def test_shapes(T, H):
    rope = rotary.Rotary(64, scaling={"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096,
                                      "mscale": 1.0, "mscale_all_dim": 0.707}, device=DEV)
    p, q, k = inputs(T, H, 64, torch.bfloat16, T)
    x, y = q.clone(), k.clone()
    rotary.apply_rotary(rope, p, q, k)  # in place
    some = torch.tensor(sorted({0, T - 1, T // 2, T // 3}))
    check(q[some], x[some], p[some], rope)
    check(k[some], y[some], p[some], rope)
    full = torch.empty_like(x)
    rotary.apply_rotary(rope, p, x, q_out=full)
    assert torch.equal(full, q)


@pytest.mark.parametrize("interleaved", [True, False])
def test_slices_and_strides(interleaved):
    """Parts of heads of wider tensors, misaligned rows, transposed heads, several key heads; the rest stays as it is."""
    rope = rotary.Rotary(32, interleaved=interleaved, device=DEV)
    p, _, _ = inputs(50, 4, 32, torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    for width, start in ((96, 64), (97, 65), (33, 1), (40, 4)):
        q = torch.randn(50, 4, width, generator=g).to(torch.bfloat16).to(DEV)
        k = torch.randn(2, 50, width, generator=g).to(torch.bfloat16).to(DEV).transpose(0, 1)
        qo, ko = torch.full((50, 4, 70), 3.0, dtype=torch.bfloat16, device=DEV), torch.empty_like(k)
        rotary.apply_rotary(rope, p, q[..., start:start + 32], k[..., :32], qo[..., 38:], ko[..., :32])
        check(qo[..., 38:], q[..., start:start + 32], p, rope)
        check(ko[..., :32], k[..., :32], p, rope)
        assert (qo[..., :38] == 3).all()
        x = q.clone()
        rotary.apply_rotary(rope, p, x[..., start:start + 32])
        assert torch.equal(x[..., start:start + 32], qo[..., 38:])
        x[..., start:start + 32] = q[..., start:start + 32]
        assert torch.equal(x, q)


def test_positions_of_any_size_and_sign():
    rope = rotary.Rotary(64, device=DEV)
    p = torch.tensor([0, 1, -1, 131071, -131071, 2 ** 31 - 1, 2 ** 31, -2 ** 40, 2 ** 52 + 1], device=DEV)
    q = torch.randn(9, 3, 64, generator=torch.Generator().manual_seed(3)).to(DEV)
    out = torch.empty_like(q)
    rotary.apply_rotary(rope, p, q, q_out=out)
    # a frequency is held to 2^-65 of a turn, as here: 2^52 positions keep 2^-13 of one; up to 2^40 nothing shows
    check(out[:8], q[:8], p[:8], rope)
    back = torch.empty_like(q)
    rotary.apply_rotary(rope, -p, out, q_out=back)
    assert ((back - q).abs() <= 2.0 ** -18 * q.abs().amax()).all()
    i32 = torch.empty_like(q)
    rotary.apply_rotary(rope, p[:6].to(torch.int32), q[:6], q_out=i32[:6])
    assert torch.equal(i32[:6], out[:6])


def test_broadcast_inputs_and_nothing_to_do():
    rope = rotary.Rotary(32, device=DEV)
    p, q, k = inputs(9, 4, 32, torch.float32)
    one = q[:, :1].expand(9, 4, 32)
    out = torch.empty(9, 4, 32, device=DEV)
    rotary.apply_rotary(rope, p, one, q_out=out)
    check(out, one, p, rope)
    with pytest.raises(ValueError, match="repeat"):
        rotary.apply_rotary(rope, p, one)
    rotary.apply_rotary(rope, p[:0], q[:0], k[:0])
    rotary.apply_rotary(rope, p, q[:, :0])


def test_values_that_are_not_finite_stay_in_their_pairs():
    rope = rotary.Rotary(64, interleaved=False, device=DEV)
    p, q, _ = inputs(5, 2, 64, torch.bfloat16)
    out, bad = torch.empty_like(q), torch.empty_like(q)
    rotary.apply_rotary(rope, p, q, q_out=out)
    x = q.clone()
    x[2, 1, 7] = float("nan")
    x[3, 0, 40] = float("inf")
    rotary.apply_rotary(rope, p, x, q_out=bad)
    same = torch.ones_like(x, dtype=torch.bool)
    same[2, 1, [7, 39]] = False
    same[3, 0, [8, 40]] = False
    assert torch.equal(bad[same], out[same])
    assert not torch.isfinite(bad[~same]).any()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("H,Hk", [(0, 1), (0, 5), (1, 40), (3, 7), (16, 16), (7, 3), (128, 2)])
def test_heads_of_both_tensors(H, Hk, interleaved):
    rope = rotary.Rotary(64, interleaved=interleaved, device=DEV)
    g = torch.Generator().manual_seed(H + Hk)
    p = torch.randint(0, 100000, (37,), generator=g).to(DEV)
    q, k = (torch.randn(37, n, 64, generator=g).to(torch.bfloat16).to(DEV) for n in (H, Hk))
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    rotary.apply_rotary(rope, p, q, k, qo, ko)
    if H:
        check(qo, q, p, rope)
    check(ko, k, p, rope)


@pytest.mark.parametrize("T,H,dim,dtype", [(70001, 2, 32, torch.bfloat16), (20000, 17, 64, torch.float32), (9001, 5, 6, torch.float16)])
def test_many_tokens_as_few(T, H, dim, dtype):
    p, q, k = inputs(T, H, dim, dtype, seed=5)
    rope = rotary.Rotary(dim, interleaved=T % 2 == 0, device=DEV)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    rotary.apply_rotary(rope, p, q, k, qo, ko)
    some = torch.cat([torch.arange(3), torch.randint(0, T, (20,)), torch.arange(T - 3, T)]).to(DEV)
    check(qo[some], q[some], p[some], rope)
    check(ko[some], k[some], p[some], rope)
    for i in range(0, T, 1501):
        s = slice(i, i + 1501)
        a, b = rotary.apply_rotary(rope, p[s], q[s], k[s], torch.empty_like(q[s]), torch.empty_like(k[s]))
        assert torch.equal(a, qo[s]) and torch.equal(b, ko[s])
