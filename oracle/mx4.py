"""MX4 rows and the attention over them, from their definition (CPU, float64).

Values are looked up and compared with midpoints one by one; nothing is shared
with the kernels' bit arithmetic.
"""

from __future__ import annotations

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
LOW, HIGH, NAN = 63, 159, 255
BLOCK = 32


def scale_bytes(y: torch.Tensor) -> torch.Tensor:
    """Scale bytes ``[n, D / 32]`` of rows ``y``: the least power of two, from 2^-64
    on, under which the block's largest magnitude is below 7; 255 above 2^32 and
    for blocks that are not finite."""
    v = y.double().abs().unflatten(-1, (-1, BLOCK))
    big = v.amax(-1)
    out = torch.full(big.shape, NAN, dtype=torch.int64)
    for s in range(HIGH, LOW - 1, -1):
        out = torch.where(big < 7.0 * 2.0 ** (s - 127), torch.full_like(out, s), out)
    return torch.where(torch.isfinite(v).all(-1), out, torch.full_like(out, NAN)).to(torch.uint8)


def encode(y: torch.Tensor):
    """(codes u8 ``[n, D]`` one a byte, scale bytes) of rows ``y``: nearest level, ties to the even code."""
    s = scale_bytes(y)
    f = torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s.long() - 127)
    f = torch.where(s == NAN, torch.ones_like(f), f).repeat_interleave(BLOCK, -1)
    w = y.double() / f
    w = torch.where((s == NAN).repeat_interleave(BLOCK, -1), torch.zeros_like(w), w)
    m = w.abs()
    code = torch.zeros(y.shape, dtype=torch.int64)
    for c in range(7):
        mid = (LEVELS[c] + LEVELS[c + 1]) / 2
        code += ((m > mid) | ((m == mid) & (c % 2 == 1))).long()
    return (code + 8 * torch.signbit(w).long()).to(torch.uint8), s


def pack(codes: torch.Tensor) -> torch.Tensor:
    """One code a byte -> two: element 2 j low, 2 j + 1 high."""
    c = codes.unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4)


def decode(packed: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """Stored values in float64 of packed codes and scale bytes."""
    c = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).long()
    v = torch.where(c >= 8, -LEVELS[c & 7], LEVELS[c & 7])
    f = torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s.long() - 127)
    return v * torch.where(s == NAN, torch.full_like(f, float("nan")), f).repeat_interleave(BLOCK, -1)


def attend(q, x, rope, visible, sm_scale):
    """(output, LSE, sum of softmax * |x|) in float64 of queries ``q [n, H, D + R]`` over rows
    ``x [L, D]``, ``rope [L, R]``, query i seeing the first ``visible[i]`` of them."""
    n, H, _ = q.shape
    L, D = x.shape
    o = torch.zeros(n, H, D, dtype=torch.float64)
    w = torch.zeros_like(o)
    lse = torch.full((n, H), float("-inf"), dtype=torch.float64)
    for i in range(n):
        m = min(int(visible[i]), L)
        if m <= 0:
            continue
        k = torch.cat((x[:m].double(), rope[:m].double()), -1)
        s = (q[i].double() @ k.t()) * sm_scale
        lse[i] = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[i][:, None])
        o[i], w[i] = p @ x[:m].double(), p @ x[:m].double().abs()
    return o, lse, w
