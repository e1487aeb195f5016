"""Attention over expanded keys and values on the GPU against float64.

Tolerance: a weight is rounded to bf16 (2^-8 of itself) and the output divided by the
sum of the rounded ones, so that it is off by at most 2^-8 sum w |v - o| / (1 - 2^-8), which is at most that
times the weighted deviation of v (Cauchy); scores are FP32 sums of exact products, off
by at most ds = (DK + 2) 2^-23 sm_scale sum |q k|, exponentials and sums by 2^-20 more: (2 ds + 2^-20) of
sum w |v|; the output is rounded once, 2^-8 of itself. The LSE has the scores' error and 2^-20 of its size.
"""

import math

import pytest
import torch

from mla_kv_quant_amd import expanded, kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


class Batch:
    def __init__(self, dn, H, qlens, klens, seed=0, q_std=2.0, v_std=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dn, self.dr, self.H, self.qlens, self.klens = dn, dn // 2, H, qlens, klens
        T, N = sum(qlens), sum(klens)
        self.q = (torch.randn(T, H, dn + self.dr, generator=g) * q_std).to(BF)
        self.kv = torch.randn(N, H, 2 * dn, generator=g)
        self.kv[..., dn:] *= v_std
        self.kv = self.kv.to(BF)
        self.pe = torch.randn(N, self.dr, generator=g).to(BF)
        self.sm = (dn + self.dr) ** -0.5

    def offsets(self, lens):
        at = [0]
        for n in lens:
            at.append(at[-1] + n)
        return torch.tensor(at, dtype=torch.int32, device=DEV)

    def run(self, causal=True, lse=None, o=None, max_q_len=None, **kw):
        if o is None:
            o = torch.full((self.q.shape[0], self.H, self.dn), 7.0, dtype=BF, device=DEV)
        expanded.expanded_attend_fwd(self.q.to(DEV), self.kv.to(DEV), self.pe.to(DEV), o, self.offsets(self.qlens),
                                     self.offsets(self.klens), max(self.qlens, default=0) if max_q_len is None else max_q_len,
                                     self.sm, causal=causal, lse=lse, **kw)
        return o

    def check(self, o, causal=True, lse=None, rows=None):
        o, dn = o.double().cpu(), self.dn
        t = k0 = 0
        for m, n in zip(self.qlens, self.klens):
            sel = torch.arange(m) if rows is None or m <= rows else torch.unique(torch.linspace(0, m - 1, rows).long())
            q = self.q[t:t + m][sel].double().transpose(0, 1)  # [H, r, dk]
            k = torch.cat((self.kv[k0:k0 + n, :, :dn], self.pe[k0:k0 + n, None].expand(n, self.H, self.dr)), -1)
            k, v = k.double().transpose(0, 1), self.kv[k0:k0 + n, :, dn:].double().transpose(0, 1)
            s = q @ k.transpose(1, 2) * self.sm
            ds = (dn + self.dr + 2) * 2.0 ** -23 * self.sm * (q.abs() @ k.abs().transpose(1, 2))
            see = torch.ones(len(sel), n, dtype=torch.bool)
            if causal:
                see = torch.arange(n) <= n - m + sel[:, None]
            s = s.masked_fill(~see, float("-inf"))
            ds = ds.masked_fill(~see, 0).amax(-1, keepdim=True) if n else torch.zeros(self.H, len(sel), 1).double()
            top = torch.logsumexp(s, -1, keepdim=True) if n else torch.full_like(ds, float("-inf"))
            w = torch.where(torch.isfinite(top), torch.exp(s - top), 0.0)
            want, w1 = w @ v, w @ v.abs()
            dev = (w @ v.square() - want.square()).clamp(min=0).sqrt()
            tol = 2.0 ** -8 * 1.01 * dev + (2 * ds + 2.0 ** -20) * w1 + 2.0 ** -8 * want.abs()
            got = o[t:t + m][sel].transpose(0, 1)
            bad = ~((got - want).abs() <= tol)
            assert not bad.any(), (m, n, bad.sum().item(), ((got - want).abs() / (tol + 1e-300)).max().item())
            if lse is not None:
                gl, wl = lse[t:t + m].double().cpu()[sel].t()[..., None], top
                seen = torch.isfinite(wl)
                assert torch.equal(seen, torch.isfinite(gl)) and (gl[~seen] == float("-inf")).all()
                assert ((gl - wl).abs() <= ds + 2.0 ** -20 * (1 + wl.abs()))[seen].all()
            t += m
            k0 += n


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dn", [128, 64])
@pytest.mark.parametrize("H", [1, 3, 16])
@pytest.mark.parametrize("qlens,klens", [
    ([1], [1]), ([1], [64]), ([1], [65]), ([31], [31]), ([33], [97]), ([128], [128]), ([129], [200]), ([257], [257]),
    ([1, 1, 1], [5, 700, 64]), ([3, 0, 70, 1], [10, 4, 70, 333]), ([40, 300], [500, 301]), ([5, 8], [3, 0]),
])
def test_attention(dn, H, qlens, klens, causal):
    b = Batch(dn, H, qlens, klens, seed=sum(qlens) + H)
    lse = torch.full((sum(qlens), H), 5.0, device=DEV)
    o = b.run(causal, lse)
    b.check(o, causal, lse)
    assert torch.equal(o, b.run(causal))  # the same without the LSE, and again


@pytest.mark.parametrize("dn,H,qlens,klens", [
    (128, 2, [700, 2000], [700, 2500]), (64, 2, [1500, 5], [4000, 5000]), (128, 128, [5], [300]), (128, 1, [2], [20000]),
    (64, 40, [1] * 6, [900] * 6), (64, 8, [1100] * 3, [1100] * 3),
    (128, 128, [260, 1, 300, 257], [400, 70, 300, 600]), (64, 128, [260, 1, 300, 257], [400, 70, 300, 600]),
    (128, 40, [1500, 3, 700, 64], [1500, 2000, 701, 65]), (64, 40, [1500, 3, 700, 64], [1500, 2000, 701, 65]),
])
def test_long_and_many(dn, H, qlens, klens):
    b = Batch(dn, H, qlens, klens, seed=7)
    lse = torch.empty(sum(qlens), H, device=DEV)
    b.check(b.run(True, lse), True, lse, rows=24)


@pytest.mark.parametrize("B", [65, 200])
def test_many_requests(B):
    g = torch.Generator().manual_seed(B)
    qlens = torch.randint(0, 9, (B,), generator=g).tolist()
    klens = [q + k for q, k in zip(qlens, torch.randint(0, 90, (B,), generator=g).tolist())]
    b = Batch(64, 2, qlens, klens, seed=B)
    b.check(b.run())


@pytest.mark.parametrize("dn", [128, 64])
@pytest.mark.parametrize("H,m", [(2, 200), (128, 1030)])
def test_scores_that_grow_and_fall(dn, H, m):
    """Scores far above and below what a row saw first, and logits of thousands."""
    for sign in (1.0, -1.0):
        b = Batch(dn, H, [m], [m + 400], seed=3)
        k = torch.linspace(0, 30, m + 400)[:, None] * sign
        b.kv[:, 0, :dn] = (k * torch.sign(b.q[100, 0, :dn].float())).to(BF)
        lse = torch.empty(m, H, device=DEV)
        b.check(b.run(True, lse), True, lse, rows=None if H == 2 else 40)


@pytest.mark.parametrize("dn", [128, 64])
@pytest.mark.parametrize("m,n,H", [(40, 1500, 1), (300, 340, 2), (520, 560, 128)])
def test_what_a_query_does_not_see_does_not_reach_it(dn, m, n, H):
    b = Batch(dn, H, [m, 8], [n, 8], seed=11)
    clean = b.run()
    b.check(clean, rows=50)
    for row, what in ((n - 1, float("nan")), (n - m // 2, float("inf")), (n - m + 1, float("-inf"))):
        c = Batch(dn, H, [m, 8], [n, 8], seed=11)
        c.kv[row] = what
        c.pe[row] = what
        o = c.run()
        first = row - (n - m)  # the first query that sees the row
        assert torch.equal(o[:first], clean[:first]) and torch.equal(o[m:], clean[m:])
        assert not torch.isfinite(o[first:m]).any()
        # the value alone: every feature of it, no other
        c = Batch(dn, H, [m, 8], [n, 8], seed=11)
        c.kv[row, H - 1, dn + 5] = what
        o = c.run()
        assert torch.equal(o[:first], clean[:first]) and torch.equal(o[m:], clean[m:])
        ok = torch.ones(H, dn, dtype=torch.bool)
        ok[H - 1, 5] = False
        assert torch.equal(o[:, ok], clean[:, ok]) and not torch.isfinite(o[first:m, H - 1, 5]).any()
        if what == what:
            assert (o[first:m, H - 1, 5] == what).all()


def test_strides_and_what_is_left_as_it_was():
    b = Batch(64, 3, [70, 20], [100, 20], seed=5)
    want = b.run()
    q = torch.zeros(3, 90, 120, dtype=BF, device=DEV).transpose(0, 1)
    q[..., 16:112] = b.q.to(DEV)
    kv = torch.zeros(120, 3, 160, dtype=BF, device=DEV)
    kv[..., 8:136] = b.kv.to(DEV)
    rows = torch.zeros(120, 288, dtype=BF, device=DEV)
    rows[:, 256:] = b.pe.to(DEV)
    o = torch.full((95, 3, 80), 3.0, dtype=BF, device=DEV)
    qo, ko = b.offsets([70, 20]), b.offsets([100, 20])
    expanded.expanded_attend_fwd(q[..., 16:112], kv[..., 8:136], rows[:, 256:], o[..., 8:72], qo, ko, 70, b.sm)
    assert torch.equal(o[:90, :, 8:72], want)
    assert (o[90:] == 3).all() and (o[..., :8] == 3).all() and (o[..., 72:] == 3).all()
    # a shorter maximum leaves the later queries out; the others still end at the last key
    o = torch.full((90, 3, 64), 3.0, dtype=BF, device=DEV)
    expanded.expanded_attend_fwd(b.q.to(DEV), b.kv.to(DEV), b.pe.to(DEV), o, qo, ko, 33, b.sm)
    assert torch.equal(o[:33], want[:33]) and (o[33:70] == 3).all() and torch.equal(o[70:], want[70:])


def test_queries_before_the_first_key_that_are_cut_off_from_the_last():
    """Of more queries than keys only the first ones, which see nothing."""
    b = Batch(64, 2, [300, 5], [10, 5], seed=6)
    lse = torch.full((305, 2), 5.0, device=DEV)
    o = b.run(lse=lse, max_q_len=33)
    assert (o[:33] == 0).all() and (lse[:33] == float("-inf")).all() and (o[33:300] == 7).all() and (lse[33:300] == 5).all()
    b.check(b.run())


def test_prefix_in_parts_joined_by_lse():
    """A prefix without the causal rule and the chunk with it, joined by their LSEs, are the whole."""
    m, p, H, dn = 50, 300, 4, 128
    b = Batch(dn, H, [m], [p + m], seed=21)
    lse = torch.empty(m, H, device=DEV)
    b.check(b.run(True, lse), True, lse)
    parts = []
    for lo, hi, causal in ((0, p, False), (p, p + m, True)):
        o, l = torch.empty(m, H, dn, dtype=BF, device=DEV), torch.empty(m, H, device=DEV)
        expanded.expanded_attend_fwd(b.q.to(DEV), b.kv[lo:hi].to(DEV), b.pe[lo:hi].to(DEV), o, b.offsets([m]),
                                     b.offsets([hi - lo]), m, b.sm, causal=causal, lse=l)
        parts.append((o.double(), l.double()))
    both = torch.logaddexp(parts[0][1], parts[1][1])
    assert ((both - lse.double()).abs() <= 2.0 ** -18 * (1 + both.abs())).all()
    o = sum(o * torch.exp(l - both)[..., None] for o, l in parts)
    b.check(o)  # (each part rounded once more, by less than the weights' allowance)


def test_workspace_and_side_stream():
    b = Batch(128, 4, [8], [4000], seed=2)
    n = kernels.expanded_attend_workspace_bytes(8, 4000, 1, 4, 128, 8, DEV)
    assert n > 0 and kernels.expanded_attend_workspace_bytes(4096, 4096, 1, 16, 128, 4096, DEV) == 0
    want = b.run()
    b.check(want)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(b.run(workspace=ws), want)
    with pytest.raises(ValueError, match="workspace"):
        b.run(workspace=ws[:n - 16])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = b.run()
    side.synchronize()
    assert torch.equal(o, want)


@pytest.mark.parametrize("dn,H,qlens,klens", [
    (128, 1, [20], [13000]), (64, 1, [3, 140], [17000, 200]),  # more parts than a row has lanes
    (128, 8, [60, 282, 0, 100, 5], [60, 7000, 300, 101, 2]),  # parts by the longest request's length
    (128, 2, [5, 130, 2], [6, 131, 3]), (64, 4, [1, 1], [1, 30]), (128, 1, [0, 0, 4], [4000, 0, 0]),  # room, not used
    (128, 128, [400], [400]), (64, 100, [150, 180], [150, 900]),  # two blocks a CU, the second in reverse
    (128, 128, [129, 1, 300, 128], [129, 800, 300, 500]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_parts_and_orders_of_row_blocks(dn, H, qlens, klens, causal):
    b = Batch(dn, H, qlens, klens, seed=len(qlens) + H)
    T = sum(qlens)
    n = kernels.expanded_attend_workspace_bytes(T, sum(klens), len(qlens), H, dn, max(qlens), DEV)
    ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device=DEV)
    lse = torch.full((T, H), 5.0, device=DEV)
    o = b.run(causal, lse, workspace=ws)
    b.check(o, causal, lse, rows=40)
    ws.fill_(127)
    assert torch.equal(b.run(causal, workspace=ws), o)


@pytest.mark.parametrize("dn,H,qlens,klens", [(128, 2, [300, 40], [500, 3000]), (64, 3, [70, 129], [90, 129]), (128, 1, [8], [6000])])
@pytest.mark.parametrize("causal", [True, False])
def test_outputs_that_overflow_or_hold_the_largest_values(dn, H, qlens, klens, causal):
    """Outputs that are not finite are as the formula has them, those beside them are not touched."""
    b = Batch(dn, H, qlens, klens, seed=17)
    big = torch.finfo(BF).max
    clean = b.run(causal)
    b.kv[:, 0, dn + 1] = big  # every value of a column: sums of outputs pass the range, the outputs do not
    b.kv[:, 0, dn + 2] = big
    o = b.run(causal)
    ok = torch.ones(H, dn, dtype=torch.bool)
    ok[0, 1:3] = False
    assert torch.equal(o[:, ok], clean[:, ok])
    seen = torch.cat([torch.arange(m) + n - m >= 0 for m, n in zip(qlens, klens)]) if causal else slice(None)
    assert (o[seen, 0, 1].float() >= big * (1 - 2.0 ** -7)).all()
    b.q[3] = float("nan")
    lse = torch.zeros(sum(qlens), H, device=DEV)
    o2 = b.run(causal, lse)
    rest = torch.arange(sum(qlens)) != 3
    assert torch.equal(o2[rest], o[rest]) and torch.isnan(o2[3]).all() and torch.isfinite(lse[rest]).all()
