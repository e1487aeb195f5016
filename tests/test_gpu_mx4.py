"""The MX4 cache on the GPU against the float64 oracle (oracle/mx4.py).

Tolerances, from the arithmetic of the kernels:

* rows without a rotation and stored rows: none, the bytes are exact;
* rotated rows: an FP32 sum of D exact products is off by at most D 2^-24 of the
  sum of their magnitudes (``err``); a stored value is then a level whose
  distance from the exact value is at most the nearest level's plus 2 err;
* rows rotated back: that error plus half a bf16 step (2^-8 of the value);
* attention: each probability is rounded to bf16 (2^-8 of itself), scores are
  FP32 sums (``ds`` = (D + R) 2^-23 sum |q k| sm_scale, the query's split off by at
  most 2^-21 of its largest element more), and the output is rounded once:
  |do| <= (2^-8 + 2 ds + 2^-16) sum softmax |x| + 2^-8 |o|. The LSE has the scores' error and
  2^-20 for the FP32 sum, its logarithm and the final product with ln 2.
"""

import math

import numpy as np
import pytest
import torch

from mla_kv_quant_amd import MX4MLAPool, kernels, mx4, synth
from oracle import mx4 as oracle
from tests.helpers import alloc_slots

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dims(D):
    return D, D // 8


def fill(pool, slots, x, pe):
    """Write fp32 rows into layer 0 with the oracle's codec."""
    code, s = oracle.encode(x)
    at = torch.as_tensor(slots)
    pool.c_codes[0][at.to(DEV)] = oracle.pack(code).to(DEV)
    pool.c_scales[0][at.to(DEV)] = s.to(DEV)
    pool.rope_buf[0][at.to(DEV)] = pe.to(DEV)


class Batch:
    """A cache with requests of the given lengths and query counts, and its oracle results."""

    def __init__(self, D, H, lens, qlens, page, seed=0, spread=1.0, q_std=None, grow=0.0):
        D, R = dims(D)
        self.D, self.R, self.H, self.page, self.lens, self.qlens = D, R, H, page, lens, qlens
        self.slots, pages, num = alloc_slots(lens, page, seed)
        self.pool = MX4MLAPool(num - 1, 1, D, R, device=DEV)
        # what nobody sees: NaN blocks and infinite rope rows
        self.pool.c_scales[0].fill_(255)
        self.pool.c_codes[0].random_(0, 256)
        self.pool.rope_buf[0].fill_(float("inf"))
        g = torch.Generator().manual_seed(seed + 5)
        self.sm = 1 / math.sqrt(1.5 * D / 4)
        self.T = sum(qlens)
        std = q_std if q_std is not None else 2.0 / (self.sm * math.sqrt(D + R) * spread)
        self.q = (torch.randn(self.T, H, D + R, generator=g) * std).to(torch.bfloat16)
        self.x, self.pe = [], []
        for b, n in enumerate(lens):
            x = torch.randn(n, D, generator=g) * spread
            if grow:  # later rows lie more and more along the first query
                x += torch.linspace(0, grow, n)[:, None] * self.q[0, 0, :D].float()
            pe = torch.randn(n, R, generator=g).to(torch.bfloat16)
            if n:
                fill(self.pool, self.slots[b], x, pe)
            code, s = oracle.encode(x)
            self.x.append(oracle.decode(oracle.pack(code), s))
            self.pe.append(pe)
        self.qo = torch.tensor(np.concatenate(([0], np.cumsum(qlens))), dtype=torch.int32, device=DEV)
        self.kv_indptr = torch.tensor(np.concatenate(([0], np.cumsum([len(p) for p in pages]))), dtype=torch.int32,
                                      device=DEV)
        self.kv_indices = torch.tensor(np.concatenate([p for p in pages] + [np.zeros(0)]), dtype=torch.int32, device=DEV)
        self.kv_lens = torch.tensor(lens, dtype=torch.int64, device=DEV)

    def run(self, q=None, o=None, lse=None, decode=False, **kw):
        q = self.q.to(DEV) if q is None else q
        o = torch.full((self.T, self.H, self.D), 7.0, dtype=torch.bfloat16, device=DEV) if o is None else o
        mx4.attend_fwd(q, o, self.pool, 0, self.kv_indptr, self.kv_indices, self.kv_lens, self.sm,
                       qo_indptr=None if decode else self.qo, max_q_len=max(self.qlens), page_size=self.page, lse=lse,
                       **kw)
        return o

    def check(self, o, lse=None, requests=None):
        o = o.double().cpu()
        t = 0
        for b, (n, m) in enumerate(zip(self.lens, self.qlens)):
            if requests is not None and b not in requests:
                t += m
                continue
            q = self.q[t:t + m]
            vis = [n - m + i + 1 for i in range(m)]
            want, wl, w = oracle.attend(q, self.x[b], self.pe[b], vis, self.sm)
            if n:
                k = torch.cat((self.x[b], self.pe[b].double()), -1).abs()
                big = q[..., :self.D].double().abs().amax(-1, keepdim=True)
                ds = self.sm * ((self.D + self.R) * 2.0 ** -23 * (q.double().abs() @ k.t()).amax(-1)
                                + (2.0 ** -21 * big * self.x[b].abs().sum(-1).amax())[..., 0])
            else:
                ds = torch.zeros(m, self.H, dtype=torch.float64)
            tol = (2.0 ** -8 + 2 * ds[..., None] + 2.0 ** -16) * w + 2.0 ** -8 * want.abs()
            bad = (o[t:t + m] - want).abs() > tol
            assert not bad.any(), (b, n, m, bad.sum().item(), ((o[t:t + m] - want).abs() / (tol + 1e-300)).max().item())
            if lse is not None:
                got = lse[t:t + m].double().cpu()
                seen = torch.isfinite(wl)
                assert torch.equal(seen, torch.isfinite(got)) and (got[~seen] == float("-inf")).all()
                off = (got - wl).abs()[seen]
                assert (off <= (ds + 2.0 ** -20 * (1 + wl.abs()))[seen]).all(), off.max().item()
            t += m


# ---- rows ------------------------------------------------------------------------
@pytest.mark.parametrize("D", [512, 256])
@pytest.mark.parametrize("n", [1, 3, 64, 257])
def test_plain_rows_are_exact(D, n):
    D, R = dims(D)
    pool = MX4MLAPool(600, 2, D, R, device=DEV, start_layer=3)
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, D, generator=g) * torch.exp2(torch.rand(n, D // 32, generator=g) * 90 - 60).repeat_interleave(32, 1)
    x[0, :32] = 0
    x = x.to(torch.bfloat16)
    pe = torch.randn(n, R, generator=g).to(torch.bfloat16)
    loc = torch.randperm(600, generator=g)[:n] + 1
    mx4.write_rows(pool, 4, loc.to(DEV), x.to(DEV), pe.to(DEV))
    code, s = oracle.encode(x.float())
    assert torch.equal(pool.c_codes[1][loc.to(DEV)].cpu(), oracle.pack(code))
    assert torch.equal(pool.c_scales[1][loc.to(DEV)].cpu(), s)
    assert torch.equal(pool.rope_buf[1][loc.to(DEV)].cpu(), pe)
    other = torch.ones(601, dtype=torch.bool)
    other[loc] = False
    assert (pool.c_codes[1][other.to(DEV)] == 0).all() and (pool.rope_buf[1][other.to(DEV)] == 0).all()
    assert (pool.c_codes[0] == 0).all()
    back = mx4.read_rows(pool, 4, loc.to(DEV)).cpu()
    assert torch.equal(back[:, :D].double(), oracle.decode(oracle.pack(code), s)) and torch.equal(back[:, D:], pe)


@pytest.mark.parametrize("D", [512, 256])
@pytest.mark.parametrize("n", [1, 15, 17, 100, 1000, 9000])
def test_rotated_rows(D, n):
    D, R = dims(D)
    rot = synth.make_rotation(D, 3)
    pool = MX4MLAPool(n + 20, 1, D, R, device=DEV, rotations=[rot])
    x = synth.make_latent(n, D, 5, seed=n, factor=8.0)
    pe = synth.make_normal((n, R), n + 1)
    loc = torch.randperm(n + 20, generator=torch.Generator().manual_seed(n))[:n] + 1
    mx4.write_rows(pool, 0, loc.to(DEV), x.to(DEV), pe.to(DEV))
    r = rot.to(torch.bfloat16).double()
    y = x.double() @ r
    err = D * 2.0 ** -24 * (x.double().abs() @ r.abs())
    s = pool.c_scales[0][loc.to(DEV)].cpu()
    v = oracle.decode(pool.c_codes[0][loc.to(DEV)].cpu(), s)
    # scales: those of the exact rows, moved by the error at most
    eb = err.unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(-2)
    lo = oracle.scale_bytes(torch.sign(y) * (y.abs() - eb).clamp(min=0))
    hi = oracle.scale_bytes(y + torch.sign(y) * eb)
    assert ((s >= lo) & (s <= hi)).all()
    f = torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s.long() - 127).repeat_interleave(32, -1)
    near = torch.full_like(y, float("inf"))
    for level in oracle.LEVELS:
        near = torch.minimum(near, (y.abs() - level * f).abs())
    assert ((v - y).abs() <= near + 2 * err).all()
    assert torch.equal(pool.rope_buf[0][loc.to(DEV)].cpu(), pe)
    # as stored, and rotated back
    assert torch.equal(mx4.read_rows(pool, 0, loc.to(DEV), unrotate=False).cpu()[:, :D].double(), v)
    back = mx4.read_rows(pool, 0, loc.to(DEV)).cpu()
    want = v @ r.t()
    tol = 2.0 ** -8 * want.abs() + 1.01 * D * 2.0 ** -24 * (v.abs() @ r.abs().t())
    assert ((back[:, :D].double() - want).abs() <= tol).all() and torch.equal(back[:, D:], pe)


def test_rotated_rows_do_not_depend_on_the_launch_size():
    D, R, n = 512, 64, 9000
    rot = synth.make_rotation(D, 3)
    x, pe = synth.make_latent(n, D, 5, seed=1).to(DEV), synth.make_normal((n, R), 2).to(DEV)
    a = MX4MLAPool(n, 1, D, R, device=DEV, rotations=[rot])
    b = MX4MLAPool(n, 1, D, R, device=DEV, rotations=[rot])
    loc = torch.arange(1, n + 1, device=DEV)
    mx4.write_rows(a, 0, loc, x, pe)
    for i in range(0, n, 1500):
        mx4.write_rows(b, 0, loc[i:i + 1500], x[i:i + 1500], pe[i:i + 1500])
    assert torch.equal(a.c_codes[0], b.c_codes[0]) and torch.equal(a.c_scales[0], b.c_scales[0])


@pytest.mark.parametrize("rotated", [False, True])
def test_rows_that_are_not_finite(rotated):
    D, R = 512, 64
    pool = MX4MLAPool(16, 1, D, R, device=DEV, rotations=[synth.make_rotation(D, 1)] if rotated else None)
    x = torch.randn(6, D, generator=torch.Generator().manual_seed(1))
    x[0, 7], x[1, 40], x[2, 100], x[3, 500], x[4] = float("nan"), float("inf"), -float("inf"), 3e38, 0
    x = x.to(torch.bfloat16)
    loc = torch.arange(1, 7, device=DEV)
    mx4.write_rows(pool, 0, loc, x.to(DEV), torch.zeros(6, R, dtype=torch.bfloat16, device=DEV))
    s = pool.c_scales[0][loc].cpu()
    v = mx4.read_rows(pool, 0, loc, unrotate=False)[:, :D].float().cpu()
    if rotated:
        assert (s[:4] == 255).all() and torch.isnan(v[:4]).all()
        assert torch.isnan(mx4.read_rows(pool, 0, loc)[:4, :D]).all()
    else:
        assert torch.equal(s, oracle.scale_bytes(x.float()))
        assert [(s[i] == 255).nonzero().tolist() for i in range(4)] == [[[0]], [[1]], [[3]], [[15]]]
    assert (v[4] == 0).all() and torch.isfinite(v[5]).all()


@pytest.mark.parametrize("rotated", [False, True])
@pytest.mark.parametrize("D", [512, 256])
def test_strided_inputs_and_slots_outside_the_cache(rotated, D):
    D, R = dims(D)
    rot = [synth.make_rotation(D, 1)] if rotated else None
    n = 40
    x = synth.make_latent(n, D, 3, 1).to(DEV)
    pe = synth.make_normal((n, R), 2).to(DEV)
    loc = torch.arange(1, n + 1, device=DEV)
    want = MX4MLAPool(n, 1, D, R, device=DEV, rotations=rot)
    mx4.write_rows(want, 0, loc, x, pe)
    pool = MX4MLAPool(n, 1, D, R, device=DEV, rotations=rot)
    wide = torch.zeros(n, D + R + 8, dtype=torch.bfloat16, device=DEV)
    wide[:, :D] = x
    pe_t = pe.t().contiguous().t()  # columns apart
    bad = loc.clone()
    bad[3], bad[5], bad[7] = -1, n + 1, 1 << 40
    mx4.write_rows(pool, 0, bad, wide[:, :D], pe_t)
    keep = torch.ones(n + 1, dtype=torch.bool, device=DEV)
    keep[[4, 6, 8]] = False
    for a, b in ((pool.c_codes, want.c_codes), (pool.c_scales, want.c_scales), (pool.rope_buf, want.rope_buf)):
        assert torch.equal(a[0][keep], b[0][keep]) and (a[0][~keep] == 0).all()
    out = torch.full((n + 2, D + R + 16), 3.0, dtype=torch.bfloat16, device=DEV)
    mx4.read_rows(want, 0, bad, out=out)
    assert torch.isnan(out[[3, 5, 7], :D + R]).all()
    assert (out[n:] == 3).all() and (out[:, D + R:] == 3).all()
    ok = [i for i in range(n) if i not in (3, 5, 7)]
    assert torch.equal(out[ok, :D + R], mx4.read_rows(want, 0, loc)[ok])


@pytest.mark.parametrize("D", [512, 256])
def test_rows_back_do_not_depend_on_the_launch_size(D):
    """Many rows and few take different kernels: the same sums, row by row, wherever the rows lie and go."""
    D, R = dims(D)
    n = 20001 if D == 256 else 9001
    pool = MX4MLAPool(n + 7, 1, D, R, device=DEV, rotations=[synth.make_rotation(D, 6)])
    g = torch.Generator().manual_seed(5)
    loc = (torch.randperm(n + 7, generator=g)[:n] + 1).to(DEV)
    mx4.write_rows(pool, 0, loc, synth.make_latent(n, D, 5, seed=8).to(DEV), synth.make_normal((n, R), 9).to(DEV))
    at = loc.clone()
    at[[0, 63, 64, 5000, n - 1]] = torch.tensor([-1, n + 8, 1 << 40, -(1 << 50), n + 8], device=DEV)
    at[100] = at[101] = at[7000]  # (a slot more than once)
    out = torch.full((n + 3, D + R + 24), 5.0, dtype=torch.bfloat16, device=DEV)
    mx4.read_rows(pool, 0, at, out=out)
    few = torch.cat([mx4.read_rows(pool, 0, at[i:i + 900]) for i in range(0, n, 900)])
    dead = torch.zeros(n, dtype=torch.bool, device=DEV)
    dead[[0, 63, 64, 5000, n - 1]] = True
    assert torch.equal(out[:n][~dead, :D + R], few[~dead])
    assert torch.isnan(out[:n][dead, :D + R]).all() and torch.isnan(few[dead]).all()
    assert (out[n:] == 5).all() and (out[:, D + R:] == 5).all()
    assert torch.isfinite(few[~dead]).all()


def test_a_rotation_with_values_far_apart():
    """Rows of R_eff whose values span more than the split's exact range: off by 2^-21 of the largest for each product."""
    D, R, n = 512, 64, 300
    rot = synth.make_rotation(D, 2).float()
    rot[3] *= torch.exp2(torch.linspace(0, -40, D))
    rot[7], rot[9] = 0, 1e-30
    pool = MX4MLAPool(n, 1, D, R, device=DEV)
    loc = torch.arange(1, n + 1, device=DEV)
    mx4.write_rows(pool, 0, loc, synth.make_latent(n, D, 5, seed=8).to(DEV), synth.make_normal((n, R), 9).to(DEV))
    v = mx4.read_rows(pool, 0, loc)[:, :D].double().cpu()
    pool.rotations = [rot.to(DEV, torch.bfloat16)]
    back = mx4.read_rows(pool, 0, loc)[:, :D].double().cpu()
    r = rot.to(torch.bfloat16).double()
    want = v @ r.t()
    tol = 2.0 ** -8 * want.abs() + 1.01 * D * 2.0 ** -24 * (v.abs() @ r.abs().t()) \
        + 2.0 ** -21 * v.abs().sum(-1, keepdim=True) * r.abs().amax(-1)
    assert ((back - want).abs() <= tol).all() and (back[:, 7] == 0).all()


def test_rows_back_captured_and_on_another_stream():
    D, R, n = 512, 64, 5000
    pool = MX4MLAPool(n, 1, D, R, device=DEV, rotations=[synth.make_rotation(D, 6)])
    loc = torch.arange(1, n + 1, device=DEV)
    pe = synth.make_normal((n, R), 9).to(DEV)
    out = torch.empty(n, D + R, dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    x = synth.make_latent(n, D, 5, seed=0).to(DEV)

    def step():
        mx4.write_rows(pool, 0, loc, x, pe)
        mx4.read_rows(pool, 0, loc, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        x.copy_(synth.make_latent(n, D, 5, seed=i + 1))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        assert torch.equal(got, out) and got.abs().max() > 0


def test_no_rows():
    pool = MX4MLAPool(16, 1, device=DEV)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    mx4.write_rows(pool, 0, none, torch.zeros(0, 512, dtype=torch.bfloat16, device=DEV),
                   torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV))
    assert mx4.read_rows(pool, 0, none).shape == (0, 576)
    q = torch.zeros(0, 16, 576, dtype=torch.bfloat16, device=DEV)
    i32 = torch.zeros(1, dtype=torch.int32, device=DEV)
    mx4.attend_fwd(q, q[..., :512].contiguous(), pool, 0, i32, i32, none, 0.1)


# ---- attention -----------------------------------------------------------------------
@pytest.mark.parametrize("D", [512, 256])
@pytest.mark.parametrize("H", [1, 8, 16, 17, 32, 40, 128])
@pytest.mark.parametrize("page", [1, 64])
def test_decode(D, H, page):
    b = Batch(D, H, [1, 63, 0, 64, 65, 300, 1025], [1] * 7, page, seed=H)
    lse = torch.empty(b.T, H, device=DEV)
    o = b.run(lse=lse, decode=True)
    b.check(o, lse)
    assert torch.equal(o, b.run())  # the same batch by query offsets, bit for bit


@pytest.mark.parametrize("D", [512, 256])
@pytest.mark.parametrize("H,qlens", [(16, [3, 1, 4, 2, 0, 4]), (40, [2, 9, 1, 0, 5, 3]), (5, [7, 1, 20, 2, 9, 33])])
@pytest.mark.parametrize("page", [16, 128])
def test_a_few_queries(D, H, qlens, page):
    # the third request has fewer positions than queries: its first see nothing
    b = Batch(D, H, [3, 500, 2, 64, 10, 700], qlens, page, seed=3)
    lse = torch.empty(b.T, H, device=DEV)
    b.check(b.run(lse=lse), lse)


@pytest.mark.parametrize("D,H,lens,qlens", [
    (512, 16, [130, 900, 257], [130, 200, 1]),
    (256, 40, [200, 513], [199, 77]),
    (256, 3, [1000], [1000]),
])
def test_prefill(D, H, lens, qlens):
    b = Batch(D, H, lens, qlens, 32, seed=9)
    lse = torch.empty(b.T, H, device=DEV)
    b.check(b.run(lse=lse), lse)


@pytest.mark.parametrize("D,H", [(512, 16), (256, 40)])
def test_many_row_blocks(D, H):
    # more row blocks than are shared out: a block each
    n = 8200 if H == 16 else 3300
    b = Batch(D, H, [n, 70], [n - 50, 66], 64, seed=2)
    o = b.run()
    rows = [0, 1, 63, 64, 1000, n - 51]
    want, _, w = oracle.attend(b.q[rows], b.x[0], b.pe[0], [51 + i for i in rows], b.sm)
    tol = (2.0 ** -8 + 2.0 ** -10) * w + 2.0 ** -8 * want.abs()  # (scores off by far less than 2^-11)
    assert ((o[rows].double().cpu() - want).abs() <= tol).all()
    b.check(o, requests=[1])


def test_many_requests():
    # more requests than a block's sums hold
    lens = [(37 * i) % 130 for i in range(1100)]
    b = Batch(256, 4, lens, [1] * 1100, 16, seed=4)
    o = b.run(decode=True)
    b.check(o, requests=range(0, 1100, 7))
    few = Batch(256, 4, lens[:1000], [1] * 1000, 16, seed=4)
    few.check(few.run(decode=True), requests=range(0, 1000, 11))


@pytest.mark.parametrize("H", [16, 30, 64])
def test_scores_that_outgrow_the_reference(H):
    """Row references have to move by far more than the slack, at tiles of every wave."""
    b = Batch(512, H, [1500, 200], [1, 1], 64, seed=6, q_std=1.0, grow=6.0)
    lse = torch.empty(b.T, H, device=DEV)
    b.check(b.run(lse=lse), lse)
    assert lse.max().item() > 60


@pytest.mark.parametrize("H,qlens", [(16, [1] * 1100), (40, [1 + i % 3 for i in range(1100)])])
def test_many_requests_of_the_large_width(H, qlens):
    lens = [(41 * i) % 200 for i in range(1100)]
    b = Batch(512, H, lens, qlens, 32, seed=4)
    b.check(b.run(), requests=range(0, 1100, 37))


def test_a_few_requests_with_queries_among_many_without():
    """Blocks whose part of the work holds no tile, and what an earlier call left in the workspace."""
    before = Batch(512, 40, [5000, 3, 2600, 70] * 9, [1, 30, 2, 9] * 9, 64, seed=6)
    lens, qlens = [60 + 7 * i for i in range(302)], [20] + [0] * 300 + [3]
    b = Batch(512, 40, lens, qlens, 64, seed=5)
    ws = torch.empty(kernels.mx4_attend_workspace_bytes(512, DEV), dtype=torch.uint8, device=DEV)
    before.run(workspace=ws)
    lse = torch.empty(b.T, 40, device=DEV)
    o = b.run(workspace=ws, lse=lse)
    b.check(o, lse, requests=[0, 301])
    assert torch.equal(o, b.run(workspace=torch.zeros_like(ws)))


@pytest.mark.parametrize("n", [1, 2, 3, 8, 64, 256, 300])
@pytest.mark.parametrize("D,H", [(512, 16), (256, 40)])
def test_requests_of_one_length(D, H, n):
    """Pairs that fill whole blocks, blocks that fill whole pairs, and neither."""
    for tiles in (1, 4, 5):
        b = Batch(D, H, [64 * tiles - 3] * n, [1] * n, 64, seed=n + tiles)
        some = range(0, n, max(1, n // 16))
        b.check(b.run(decode=True), requests=some)


@pytest.mark.parametrize("H,longest", [(16, 2), (40, 1), (4, 7)])
def test_queries_past_the_longest_are_left_out(H, longest):
    b = Batch(512, H, [200, 90, 300], [5, 1, 9], 64, seed=3)
    o = torch.full((b.T, H, 512), 7.0, dtype=torch.bfloat16, device=DEV)
    mx4.attend_fwd(b.q.to(DEV), o, b.pool, 0, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm, qo_indptr=b.qo,
                   max_q_len=longest, page_size=64)
    o = o.cpu()
    t = 0
    for i, (n, m) in enumerate(zip(b.lens, b.qlens)):
        k = min(m, longest)  # these see what they see beside the ones left out
        want, _, w = oracle.attend(b.q[t:t + k], b.x[i], b.pe[i], [n - m + j + 1 for j in range(k)], b.sm)
        tol = (2.0 ** -8 + 2.0 ** -10) * w + 2.0 ** -8 * want.abs()  # (scores off by far less than 2^-11)
        assert ((o[t:t + k].double() - want).abs() <= tol).all()
        assert (o[t + k:t + m] == 7).all()
        t += m


@pytest.mark.parametrize("H", [16, 48])
def test_scores_far_below_any_mask(H):
    """Equal rows under a query that scores each at -7e11: their mean is the row itself, exactly."""
    b = Batch(512, H, [300, 64], [1, 1], 64, seed=3)
    for i, s in enumerate(b.slots):
        x = torch.full((len(s), 512), 1.0 + i)
        x[:, 1::2] = 3.0
        fill(b.pool, s, x, torch.zeros(len(s), 64, dtype=torch.bfloat16))
    q = torch.full((2, H, 576), -float(1 << 20), dtype=torch.bfloat16, device=DEV)
    o, lse = torch.empty(2, H, 512, dtype=torch.bfloat16, device=DEV), torch.empty(2, H, device=DEV)
    mx4.attend_fwd(q, o, b.pool, 0, b.kv_indptr, b.kv_indices, b.kv_lens, 640.0, page_size=64, lse=lse)
    for i in range(2):
        assert (o[i, :, 0::2] == 1.0 + i).all() and (o[i, :, 1::2] == 3.0).all()
        score = -640.0 * (1 << 20) * 256 * (4.0 + i)
        assert torch.isfinite(lse[i]).all() and ((lse[i].double().cpu() / score - 1).abs() < 2.0 ** -20).all()


def test_latents_of_small_and_large_magnitude():
    for spread in (1e-4, 3e3):
        b = Batch(512, 16, [400, 100], [1, 2], 16, seed=8, spread=spread)
        b.check(b.run())


def test_long_context_beside_short_ones():
    b = Batch(256, 16, [70001, 5, 3000], [1, 1, 1], 64, seed=12)
    lse = torch.empty(b.T, 16, device=DEV)
    b.check(b.run(lse=lse), lse)


def test_rows_that_are_not_finite_stay_where_they_are():
    b = Batch(512, 16, [200, 200, 200], [1, 1, 1], 64, seed=1)
    q = b.q.clone()
    q[0, 3, 17] = float("nan")
    q[1, 5, 530] = float("inf")
    o = b.run(q=q.to(DEV)).float().cpu()
    assert torch.isnan(o[0, 3]).all() and torch.isnan(o[1, 5]).all()
    o[0, 3], o[1, 5] = 0, 0
    assert torch.isfinite(o).all()
    # a NaN row that is seen makes its request NaN, and no other
    b.pool.c_scales[0][int(b.slots[1][150])] = 255
    o = b.run().float().cpu()
    assert torch.isnan(o[1]).all() and torch.isfinite(o[0]).all() and torch.isfinite(o[2]).all()


def test_strides_and_rows_behind_the_last_sequence():
    b = Batch(512, 16, [100, 300], [2, 3], 32, seed=7)
    q = torch.zeros(b.T + 4, 20, b.D + b.R + 16, dtype=torch.bfloat16, device=DEV)
    q[:b.T, 2:18, 8:8 + b.D + b.R] = b.q.to(DEV)
    o = torch.full((b.T + 4, 18, b.D + 8), 5.0, dtype=torch.bfloat16, device=DEV)
    mx4.attend_fwd(q[:, 2:18, 8:8 + b.D + b.R], o[:, 1:17, 4:4 + b.D], b.pool, 0, b.kv_indptr, b.kv_indices, b.kv_lens,
                   b.sm, qo_indptr=b.qo, max_q_len=3, page_size=32)
    b.check(o[:b.T, 1:17, 4:4 + b.D])
    assert (o[b.T:] == 5).all() and (o[:, 0] == 5).all() and (o[:, 17] == 5).all()
    assert (o[..., :4] == 5).all() and (o[..., 4 + b.D:] == 5).all()


def test_bad_pages_read_inside_the_cache():
    b = Batch(256, 16, [300, 300], [1, 1], 64, seed=7)
    bad = b.kv_indices.clone()
    bad[0], bad[1], bad[2] = 1 << 30, -5, 0x7fffffff
    o = torch.zeros(2, 16, 256, dtype=torch.bfloat16, device=DEV)
    mx4.attend_fwd(b.q.to(DEV), o, b.pool, 0, b.kv_indptr, bad, b.kv_lens, b.sm, page_size=64)
    b.check(o, requests=[1])
    # a list that ends early cuts the length
    short = b.kv_indptr.clone()
    lens = b.kv_lens.clone()
    lens[1] = 1 << 40
    mx4.attend_fwd(b.q.to(DEV), o, b.pool, 0, short, b.kv_indices[:-1], lens, b.sm, page_size=64)
    want, _, w = oracle.attend(b.q[1:], b.x[1][:256], b.pe[1][:256], [256], b.sm)
    assert ((o[1:].double().cpu() - want).abs() <= (2.0 ** -8 + 2.0 ** -10) * w + 2.0 ** -8 * want.abs()).all()


def test_same_call_repeats_bit_for_bit_and_layout_does_not_matter():
    a = Batch(512, 16, [700, 40, 2000], [1, 1, 1], 64, seed=11)
    first = a.run()
    mx4.attend_workspace(a.pool).fill_(255)
    assert torch.equal(first, a.run())
    ws = torch.zeros(kernels.mx4_attend_workspace_bytes(512, DEV), dtype=torch.uint8, device=DEV)
    assert torch.equal(first, a.run(workspace=ws))


def test_captured_step_is_replayed():
    """Write and attend captured together; every replay against the eager result, with eager work between."""
    D, R, H, n = 512, 64, 16, 3
    rot = synth.make_rotation(D, 5)
    lens = [129, 700, 64]
    b = Batch(D, H, lens, [1] * n, 64, seed=13)
    b.pool.rotations = [rot.to(DEV, torch.bfloat16)]
    loc = torch.tensor([int(s[-1]) for s in b.slots], device=DEV)
    x, pe = torch.zeros(n, D, dtype=torch.bfloat16, device=DEV), torch.zeros(n, R, dtype=torch.bfloat16, device=DEV)
    q = b.q.to(DEV)
    o = torch.zeros(n, H, D, dtype=torch.bfloat16, device=DEV)

    def step():
        mx4.write_rows(b.pool, 0, loc, x, pe)
        mx4.attend_fwd(q, o, b.pool, 0, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm, page_size=64)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(synth.make_latent(n, D, 5, seed=i))
        pe.copy_(synth.make_normal((n, R), i))
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone()
        o.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, o)
        assert got.abs().max() > 0


def test_another_stream():
    b = Batch(512, 16, [500, 900], [1, 1], 64, seed=14)
    want = b.run()
    q = b.q.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = b.run(q=q)
    side.synchronize()
    assert torch.equal(got, want)


def test_prefill_then_decode_as_a_server_does():
    """Prefill in two chunks, each written and then attended over, then decode steps, on a rotated layer."""
    D, R, H, page = 512, 64, 16, 64
    rot = synth.make_rotation(D, 21)
    slots, pages, num = alloc_slots([330, 210], page, 5)
    pool = MX4MLAPool(num - 1, 1, D, R, device=DEV, rotations=[rot])
    sm = 1 / math.sqrt(192)
    xs = [synth.make_latent(len(s), D, 5, seed=40 + i, factor=8.0) for i, s in enumerate(slots)]
    pes = [synth.make_normal((len(s), R), 50 + i) for i, s in enumerate(slots)]
    kv_indptr = torch.tensor([0, len(pages[0]), len(pages[0]) + len(pages[1])], dtype=torch.int32, device=DEV)
    kv_indices = torch.tensor(np.concatenate(pages), dtype=torch.int32, device=DEV)
    done = [0, 0]
    for step, m in enumerate([(128, 200), (200, 8), (1, 1), (1, 1)]):
        loc = np.concatenate([slots[i][done[i]:done[i] + m[i]] for i in range(2)])
        x = torch.cat([xs[i][done[i]:done[i] + m[i]] for i in range(2)])
        pe = torch.cat([pes[i][done[i]:done[i] + m[i]] for i in range(2)])
        mx4.write_rows(pool, 0, torch.from_numpy(loc).to(DEV), x.to(DEV), pe.to(DEV))
        done = [done[i] + m[i] for i in range(2)]
        T = sum(m)
        q = synth.make_normal((T, H, D + R), 60 + step, std=0.5)
        o = torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV)
        mx4.attend_fwd(q.to(DEV), o, pool, 0, kv_indptr, kv_indices, torch.tensor(done, device=DEV), sm,
                       qo_indptr=torch.tensor([0, m[0], T], dtype=torch.int32, device=DEV), max_q_len=max(m),
                       page_size=page)
        t = 0
        for i in range(2):
            at = torch.from_numpy(slots[i][:done[i]]).to(DEV)
            v = oracle.decode(pool.c_codes[0][at].cpu(), pool.c_scales[0][at].cpu())
            want, _, w = oracle.attend(q[t:t + m[i]], v, pes[i][:done[i]], [done[i] - m[i] + j + 1 for j in range(m[i])], sm)
            off = (o[t:t + m[i]].double().cpu() - want).abs()
            assert (off <= (2.0 ** -8 + 2.0 ** -10) * w + 2.0 ** -8 * want.abs()).all()
            t += m[i]


# ---- a layer's rotation, as it is when a row is written ---------------------------------
def written_codes(rot, x, pe, loc):
    """Cached rows of a pool that has never had another rotation."""
    pool = MX4MLAPool(loc.numel() + 8, 1, x.shape[1], pe.shape[1], device=DEV, rotations=[rot])
    mx4.write_rows(pool, 0, loc, x, pe)
    return pool.c_codes[0], pool.c_scales[0]


@pytest.mark.parametrize("D", [512, 256])
def test_rows_take_the_rotation_as_it_is(D):
    D, R = dims(D)
    n = 70
    loc = torch.arange(1, n + 1, device=DEV)
    x, pe = synth.make_latent(n, D, 5, seed=1).to(DEV), synth.make_normal((n, R), 2).to(DEV)
    rots = [synth.make_rotation(D, s).to(DEV, torch.bfloat16) for s in range(4)]
    want = [written_codes(r.clone(), x, pe, loc) for r in rots]
    pool = MX4MLAPool(n + 8, 1, D, R, device=DEV, rotations=[rots[0].clone()])

    def check(i):
        assert torch.equal(pool.c_codes[0], want[i][0]) and torch.equal(pool.c_scales[0], want[i][1])

    mx4.write_rows(pool, 0, loc, x, pe)
    check(0)
    pool.rotations[0].copy_(rots[1])  # in place
    mx4.write_rows(pool, 0, loc, x, pe)
    check(1)
    pool.rotations[0] = rots[2].clone()  # another tensor
    mx4.write_rows(pool, 0, loc, x, pe)
    check(2)
    # a first write (after a change) on one stream, the next at once on another
    side = torch.cuda.Stream()
    pool.rotations[0].copy_(rots[3])
    torch.cuda.synchronize()
    mx4.write_rows(pool, 0, loc[:1], x[:1], pe[:1])
    with torch.cuda.stream(side):
        mx4.write_rows(pool, 0, loc, x, pe)
    torch.cuda.synchronize()
    check(3)


@pytest.mark.parametrize("warm", [False, True])
def test_captured_writes_and_a_rotation_that_changes(warm):
    """A write whose layer has not been laid out yet when it is captured, and one whose has."""
    D, R, n = 256, 32, 30
    loc = torch.arange(1, n + 1, device=DEV)
    x, pe = synth.make_latent(n, D, 5, seed=1).to(DEV), synth.make_normal((n, R), 2).to(DEV)
    rots = [synth.make_rotation(D, s).to(DEV, torch.bfloat16) for s in range(2)]
    want = [written_codes(r.clone(), x, pe, loc) for r in rots]
    pool = MX4MLAPool(n + 8, 1, D, R, device=DEV, rotations=[rots[0].clone()])
    mx4.write_rows(MX4MLAPool(n, 1, D, R, device=DEV, rotations=[rots[1]]), 0, loc, x, pe)
    if warm:
        mx4.write_rows(pool, 0, loc, x, pe)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mx4.write_rows(pool, 0, loc, x, pe)
    for i in (0, 0, 1, 1, 0):
        pool.rotations[0].copy_(rots[i])
        if warm:  # (captured calls follow with the next call outside a capture)
            mx4.write_rows(pool, 0, loc, x, pe)
        pool.c_codes[0].zero_()
        pool.c_scales[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool.c_codes[0], want[i][0]) and torch.equal(pool.c_scales[0], want[i][1])
        mx4.write_rows(pool, 0, loc, x, pe)
        assert torch.equal(pool.c_codes[0], want[i][0])


@pytest.mark.parametrize("D", [512, 256])
@pytest.mark.parametrize("n", [5, 9000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_one_value_of_a_rotated_block_that_is_not_finite(D, n, bad):
    """Any column of a block, each in blocks of its own: R_eff is not finite there, the rest of the row is."""
    D, R = dims(D)
    rot = synth.make_rotation(D, 4)
    loc = torch.arange(1, n + 1, device=DEV)
    x, pe = synth.make_latent(n, D, 5, seed=1).to(DEV), synth.make_normal((n, R), 2).to(DEV)
    x[x == 0] = 1.0  # (so that the products with infinities are infinities)
    clean_codes, clean_scales = written_codes(rot.to(DEV), x, pe, loc)
    for first in range(0, 32, 8):  # columns first .. first + 7 of the blocks 0 .. 7
        at = [32 * i + first + i for i in range(8)]
        r = rot.clone()
        r[0, at] = bad
        codes, scales = written_codes(r.to(DEV), x, pe, loc)
        assert (scales[loc][:, :8] == 255).all(), first
        assert torch.equal(scales[loc][:, 8:], clean_scales[loc][:, 8:])
        assert torch.equal(codes[loc][:, 128:], clean_codes[loc][:, 128:])


# ---- the attention's workspace: calls that overlap do not meet in it -----------------------
def test_streams_and_captures_have_workspaces_of_their_own():
    pool = MX4MLAPool(64, 1, 256, 32, device=DEV)
    size = kernels.mx4_attend_workspace_bytes(256, DEV)
    here = mx4.attend_workspace(pool)
    assert here.numel() == size and mx4.attend_workspace(pool) is here
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        there = mx4.attend_workspace(pool)
        assert there.data_ptr() != here.data_ptr() and mx4.attend_workspace(pool) is there
    captured, graphs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):  # (a stream that has one already)
            ws = mx4.attend_workspace(pool)
            ws[:8].zero_()
            captured.append(ws.data_ptr())
        graphs.append(graph)
        del ws
    assert len({here.data_ptr(), there.data_ptr(), *captured}) == 4
    assert mx4.attend_workspace(pool) is here
    with torch.cuda.stream(side):
        assert mx4.attend_workspace(pool) is there


def two_batches():
    """A prefill and a decode batch over one pool, whose pairs are cut into many parts."""
    a = Batch(512, 40, [3000, 2500, 700], [300, 200, 90], 64, seed=21)
    b = Batch(512, 16, [9000, 4000], [1, 1], 64, seed=22)
    for name in ("c_codes", "c_scales", "rope_buf"):  # one pool: b's slots behind a's
        rows = getattr(a.pool, name)[0].shape[0]
        both = torch.cat((getattr(a.pool, name)[0], getattr(b.pool, name)[0]))
        getattr(a.pool, name)[0] = both
    b.kv_indices = b.kv_indices + rows // 64
    assert rows % 64 == 0
    b.pool = a.pool
    return a, b


def test_calls_on_two_streams_overlap():
    a, b = two_batches()
    want_a, want_b = a.run(), b.run()
    qa, qb = a.q.to(DEV), b.q.to(DEV)
    out_a = [torch.empty_like(want_a) for _ in range(12)]
    out_b = [torch.empty_like(want_b) for _ in range(60)]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(streams[0]):
            a.run(q=qa, o=out_a[i])
        with torch.cuda.stream(streams[1]):
            for o in out_b[5 * i:5 * i + 5]:
                b.run(q=qb, o=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want_a) for o in out_a) and all(torch.equal(o, want_b) for o in out_b)


def test_graphs_replayed_side_by_side():
    a, b = two_batches()
    want_a, want_b = a.run(), b.run()
    qa, qb = a.q.to(DEV), b.q.to(DEV)
    outs = [torch.empty_like(want_a), torch.empty_like(want_b), torch.empty_like(want_b)]
    graphs, streams = [], [torch.cuda.Stream() for _ in outs]
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(4):
                a.run(q=qa, o=outs[0]) if i == 0 else b.run(q=qb, o=outs[1])
        graphs.append(graph)
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            b.run(q=qb, o=outs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want_a) and torch.equal(outs[1], want_b) and torch.equal(outs[2], want_b)


# ---- launches of more threads or blocks than one dimension of a grid holds -----------------
def test_rows_of_more_than_2_32_threads():
    """59.7 million rows of 72 threads each, without a rotation: read, and written (nearly all outside the cache)."""
    D, R, n = 512, 64, (1 << 32) // 72 + 1000
    pool = MX4MLAPool(99, 1, D, R, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(100, D, device=DEV, generator=g).bfloat16()
    pe = torch.randn(100, R, device=DEV, generator=g).bfloat16()
    mx4.write_rows(pool, 0, torch.arange(100, device=DEV), x, pe)
    table = mx4.read_rows(pool, 0, torch.arange(100, device=DEV))
    big = torch.empty(n, D + R, dtype=torch.bfloat16, device=DEV)  # 69 GB
    try:
        slots = torch.randint(0, 100, (n,), device=DEV, generator=g)
        mx4.read_rows(pool, 0, slots, out=big)
        for at in (0, 1 << 25, n - 100000):
            assert torch.equal(big[at:at + 100000], table[slots[at:at + 100000]]), at
        slots.fill_(-1)
        at = torch.cat((torch.arange(50, device=DEV), torch.arange(n - 50, n, device=DEV)))
        slots[at] = torch.arange(100, device=DEV)
        big[at, :D] = x.flip(0)
        mx4.write_rows(pool, 0, slots, big[:, :D], pe[:1].expand(n, R))
        code, s = oracle.encode(x.flip(0).float().cpu())
        assert torch.equal(pool.c_codes[0].cpu(), oracle.pack(code)) and torch.equal(pool.c_scales[0].cpu(), s)
        assert torch.equal(pool.rope_buf[0], pe[:1].expand(100, R))
    finally:
        del big
        torch.cuda.empty_cache()


@pytest.mark.parametrize("D", [512, 256])
def test_attention_of_2_24_blocks(D):
    """2048 requests with a stated longest chunk of 4096 queries of 128 heads: the bits that the true length gives."""
    n = 2048
    b = Batch(D, 128, [2 + (7 * i) % 90 for i in range(n)], [2] * n, 16, seed=4)
    q = b.q.to(DEV)
    outs = []
    for longest in (2, 8192):
        o = torch.full((b.T, 128, D), 7.0, dtype=torch.bfloat16, device=DEV)
        mx4.attend_fwd(q, o, b.pool, 0, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm, qo_indptr=b.qo, max_q_len=longest,
                       page_size=16)
        outs.append(o)
    assert torch.equal(outs[0], outs[1])
    b.check(outs[1], requests=[0, 5, 1024, n - 1])


@pytest.mark.parametrize("D", [512, 256])
@pytest.mark.parametrize("H,qlens", [(16, [1, 1, 1, 1]), (5, [3, 1, 4, 4]), (40, [1, 2, 60, 3])])
@pytest.mark.parametrize("page", [1, 64])
def test_weights_add_up_to_one(D, H, qlens, page):
    """Requests of equal rows, whatever each position's score (the rope parts differ): the row itself, exactly.

    Weights that add up to 1 + e give the row times 1 + e; FP32 sums and the division leave
    |e| < 2^-16, which no bf16 value of one or two significant bits (a level times a power of
    two) is changed by in rounding. The first request's first queries see one position and two.
    """
    b = Batch(D, H, [qlens[0], 2, 700, 9001], qlens, page, seed=17)
    g = torch.Generator().manual_seed(3)
    rows = []
    for i, s in enumerate(b.slots):
        x = torch.randn(1, D, generator=g).expand(len(s), D)
        fill(b.pool, s, x, b.pe[i])
        code, sc = oracle.encode(x[:1])
        rows.append(oracle.decode(oracle.pack(code), sc)[0])
    lse = torch.empty(b.T, H, device=DEV)
    o = b.run(lse=lse).double().cpu()
    t = 0
    for row, m, n in zip(rows, qlens, b.lens):
        seen = [j for j in range(m) if n - m + j >= 0]
        assert (o[[t + j for j in seen]] == row).all(), (n, m)
        t += m
    assert lse.std() > 0.1


@pytest.mark.parametrize("B", [3, 1100])
def test_offsets_far_outside_read_and_write_nothing_there(B):
    """Offsets whose differences do not fit 32 bits: such a request has no queries, or no positions; others are as they were."""
    b = Batch(256, 16, [100] * B, [1] * B, 16, seed=7)
    want = b.run()
    room = torch.full((2 * B + 64, 16, 256), 7.0, dtype=torch.bfloat16, device=DEV)
    low = -(1 << 31)
    for at, value in ((2, low), (2, low + 1), (B, low), (1, (1 << 31) - 1)):
        for which in ("qo_indptr", "kv_indptr"):
            room.fill_(7.0)
            off = {"qo_indptr": b.qo.clone(), "kv_indptr": b.kv_indptr.clone()}
            off[which][at] = value
            mx4.attend_fwd(b.q.to(DEV), room[:B], b.pool, 0, off["kv_indptr"], b.kv_indices, b.kv_lens, b.sm,
                           qo_indptr=off["qo_indptr"], max_q_len=1, page_size=16)
            assert (room[B:] == 7).all()
            same = [i for i in range(1, B) if i not in (at - 1, at)]  # (a start cut to 0 is row 0's)
            assert torch.equal(room[same], want[same]), (at, value, which)


# ---- pages, caches and batches at their edges ----------------------------------------------
@pytest.mark.parametrize("D,H", [(512, 16), (256, 40)])
@pytest.mark.parametrize("page", [2, 8, 256])
def test_other_page_sizes(D, H, page):
    b = Batch(D, H, [1, 130, 77, 600], [1, 2, 3, 1], page, seed=page)
    b.check(b.run())


@pytest.mark.parametrize("lens", [[0], [0, 0, 0], [1]])
@pytest.mark.parametrize("H", [3, 40])
def test_batches_that_see_next_to_nothing(lens, H):
    b = Batch(512, H, lens, [2] * len(lens), 64, seed=1)
    lse = torch.empty(b.T, H, device=DEV)
    b.check(b.run(lse=lse), lse)


@pytest.mark.parametrize("D", [512, 256])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("left", [1, 5, 15])
def test_a_cache_that_ends_inside_its_last_page(D, page, left):
    """The last page's slots past the cache's end are neither read nor needed."""
    n = 3 * page + left
    b = Batch(D, 16, [n, 100], [1, 2], page, seed=left)
    num = (b.pool.c_codes[0].shape[0] // page + 4) * page + left  # the first request's pages become the last ones
    pool = MX4MLAPool(num - 1, 1, D, D // 8, device=DEV)
    first = num // page - 3
    where = torch.arange(first * page, first * page + n)
    assert where[-1] == num - 1
    for name in ("c_codes", "c_scales", "rope_buf"):
        old, new = getattr(b.pool, name)[0], getattr(pool, name)[0]
        new[: old.shape[0]] = old
        new[where.to(DEV)] = old[torch.as_tensor(b.slots[0]).to(DEV)]
    b.kv_indices[:4] = torch.arange(first, first + 4, device=DEV)
    b.pool = pool
    b.check(b.run())


@pytest.mark.parametrize("D", [512, 256])
def test_rows_far_into_a_large_cache(D):
    """Slots whose codes lie past 4 GB (and rope rows past 2 GB): written, read both ways and attended over."""
    D, R = dims(D)
    num = (1 << 33) // D + 4096  # D / 2 bytes a row: 4.3 GB of codes and more
    rot = synth.make_rotation(D, 3)
    n, page = 1000, 64
    start = num // page * page - 16 * page
    loc = torch.arange(start, start + n, device=DEV)
    x, pe = synth.make_latent(n, D, 5, seed=1).to(DEV), synth.make_normal((n, R), 2).to(DEV)
    big, small = (MX4MLAPool(k - 1, 1, D, R, device=DEV, rotations=[rot]) for k in (num, 16 * page))
    here = loc - start
    try:
        for rotated in (True, False):
            if not rotated:
                big.rotations[0] = small.rotations[0] = None
            mx4.write_rows(big, 0, loc, x, pe)
            mx4.write_rows(small, 0, here, x, pe)
            assert torch.equal(big.c_codes[0][loc], small.c_codes[0][here])
            assert torch.equal(mx4.read_rows(big, 0, loc), mx4.read_rows(small, 0, here))
        q = synth.make_normal((2, 16, D + R), 5, std=0.3).to(DEV)
        for p in (page, 1):
            outs = []
            for pool, at in ((big, loc), (small, here)):
                o = torch.empty(2, 16, D, dtype=torch.bfloat16, device=DEV)
                idx = (at[::p] // p).to(torch.int32)
                ptr = torch.tensor([0, idx.numel() // 2, idx.numel()], dtype=torch.int32, device=DEV)
                lens = torch.tensor([500 // p * p, n - 500 // p * p - 7], device=DEV)
                mx4.attend_fwd(q, o, pool, 0, ptr, idx, lens, 0.1, page_size=p)
                outs.append(o)
            assert torch.equal(*outs) and outs[0].abs().max() > 0
    finally:
        del big
        torch.cuda.empty_cache()
