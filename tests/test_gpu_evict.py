"""Accumulated attention weights and eviction on the GPU.

Weights against float64, tolerance from the arithmetic: a score is an FP32 sum of
D + R exact products, off by at most ds = (D + R) 2^-24 sm_scale sum |q k|; scale, difference and exponential add
2^-22 of the exponent's size and 2^-22; so a weight is off by (ds + 2^-22 |s - lse| + 2^-22) of itself, and the
FP32 sum over n rows by n 2^-24 more. Eviction is exact: the chosen positions, their slots and weights.
"""

import math

import numpy as np
import pytest
import torch

from mla_kv_quant_amd import evict, kernels, mx4
from tests.helpers import alloc_slots
from tests.test_gpu_mx4 import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def lse_of(b, i, q, n, m):
    """float64 scores [m, H, n] of request i's queries (-inf: not seen) and their LSE."""
    k = torch.cat((b.x[i], b.pe[i].double()), -1)
    s = q.double() @ k.t() * b.sm
    s = s.masked_fill(torch.arange(n) > n - m + torch.arange(m)[:, None, None], float("-inf"))
    return s, torch.logsumexp(s, -1) if n else torch.full(s.shape[:2], float("-inf"), dtype=torch.float64), k


def check_weights(b, reqs=None, add=False, decode=False, cols=None):
    T, B = b.T, len(b.lens)
    lse = torch.zeros(T, b.H, dtype=torch.float32)
    t, want, tol = 0, [], []
    for i, (n, m) in enumerate(zip(b.lens, b.qlens)):
        s, l, k = lse_of(b, i, b.q[t:t + m], n, m)
        lse[t:t + m] = l.float()
        diff = s - lse[t:t + m].double()[..., None]
        w = torch.where(torch.isfinite(s), torch.exp(diff), 0.0)
        ds = (b.D + b.R) * 2.0 ** -24 * b.sm * (b.q[t:t + m].double().abs() @ k.abs().t())
        off = ds + 2.0 ** -22 * torch.where(torch.isfinite(s), diff, 0.0).abs() + 2.0 ** -22 + m * b.H * 2.0 ** -24
        want.append(w.sum((0, 1)))
        tol.append((w * off).sum((0, 1)))
        t += m
    cols = max(b.lens) + 3 if cols is None else cols
    acc = torch.rand(B + 2, cols, generator=torch.Generator().manual_seed(1))
    got = acc.to(DEV)
    evict.accumulate_weights(b.q.to(DEV), lse.to(DEV), b.pool, 0, got, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm,
                             qo_indptr=None if decode else b.qo, max_q_len=max(b.qlens), page_size=b.page,
                             req_pool_indices=None if reqs is None else torch.tensor(reqs, device=DEV), add=add)
    got = got.cpu().double()
    left = torch.ones_like(acc, dtype=torch.bool)
    for i, n in enumerate(b.lens):
        r = i if reqs is None else reqs[i]
        if not 0 <= r < B + 2:
            continue
        n = min(n, cols)
        left[r, :n] = False
        base = acc[r, :n].double() if add else 0.0
        want_i = want[i][:n] + base
        bad = (got[r, :n] - want_i).abs() > tol[i][:n] + (2.0 ** -24 * want_i.abs() if add else 0) + 1e-30
        assert not bad.any(), (i, n, bad.sum().item())
    assert torch.equal(got[left].float(), acc[left])
    return got


@pytest.mark.parametrize("D", [512, 256])
@pytest.mark.parametrize("H,lens,qlens,page", [
    (1, [1], [1], 1), (16, [1, 64, 65, 500], [1, 1, 1, 1], 64), (16, [17, 300, 128], [2, 4, 1], 16),
    (3, [200, 33], [9, 5], 2), (20, [129, 1000], [3, 3], 64), (40, [300, 150, 700], [5, 2, 32], 32),
    (128, [260, 90], [1, 3], 8), (16, [700], [300], 64), (16, [3, 0, 40], [5, 0, 40], 1),
])
def test_weights(D, H, lens, qlens, page):
    b = Batch(D, H, lens, qlens, page, seed=len(lens) + H)
    check_weights(b)
    check_weights(b, reqs=[len(lens) + 1 - i for i in range(len(lens))], add=True)


@pytest.mark.parametrize("D,H", [(512, 16), (256, 40)])
def test_weights_of_many_requests_with_many_rows(D, H):
    # more than a wave's lanes of them, short and long, with few and many rows: shares of blocks
    lens = [1 + (37 * i) % 150 for i in range(70)] + [2500, 900, 64, 1]
    qlens = [min(n, 1 + i % 7) for i, n in enumerate(lens)]
    b = Batch(D, H, lens, qlens, 16, seed=12)
    check_weights(b)


@pytest.mark.parametrize("D,H,m", [(512, 16, 1), (512, 16, 3), (512, 16, 9), (256, 40, 1), (256, 40, 33)])
def test_weights_of_rows_and_sums_between_others(D, H, m):
    lens, qlens = [300, 700], [m, max(1, m - 1)]
    b = Batch(D, H, lens, qlens, 32, seed=13)
    lse = torch.full((b.T, H), 3.0, device=DEV)
    apart = torch.zeros(2 * b.T, H + 3, b.D + b.R + 16, dtype=torch.bfloat16, device=DEV)
    apart[::2, 1:1 + H, 8:8 + b.D + b.R] = b.q.to(DEV)
    wide = torch.full((2, 1024), 7.0, device=DEV)
    outs = []
    for q, acc in ((b.q.to(DEV), torch.empty(2, 701, device=DEV)),
                   (apart[::2, 1:1 + H, 8:8 + b.D + b.R], wide[:, 5:706])):
        evict.accumulate_weights(q, lse, b.pool, 0, acc, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm,
                                 qo_indptr=b.qo, max_q_len=m, page_size=32, add=False)
        outs.append([acc[0, :300], acc[1, :700]])
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert outs[0][0].min() > 0
    wide[0, 5:305], wide[1, 5:705] = 7.0, 7.0
    assert (wide == 7.0).all()


@pytest.mark.parametrize("D,H,lens,qlens", [
    (512, 128, [170, 51, 90], [51, 20, 1]), (512, 128, [60] * 9, [57, 1, 0, 60, 2, 3, 30, 9, 5]), (512, 16, [1275], [60]),
    (256, 40, [300], [64]), (256, 48, [65, 64, 1, 700], [2, 64, 1, 9]), (256, 20, [900], [5]),
])
def test_weights_of_many_rows_over_few_positions(D, H, lens, qlens):
    b = Batch(D, H, lens, qlens, 16, seed=14)
    check_weights(b)
    check_weights(b, add=True, reqs=[-1] + list(range(1, len(lens))), cols=120)


def test_workspace_of_weights():
    b = Batch(512, 64, [200, 333], [40, 9], 16, seed=15)
    args = (b.pool.c_codes[0], b.pool.c_scales[0], b.pool.rope_buf[0], b.qo, b.kv_indptr, b.kv_indices, b.kv_lens, 40)
    n = kernels.accumulate_weights_workspace_bytes(b.T, 2, 64, 512, b.kv_indices.shape[0], 16, 40, DEV)
    assert n > 0 and kernels.accumulate_weights_workspace_bytes(b.T, 2, 64, 512, 1 << 20, 16, 40, DEV) == 0
    assert kernels.accumulate_weights_workspace_bytes(2, 2, 64, 512, 40, 16, 1, DEV) == 0
    lse = torch.full((b.T, 64), 2.0, device=DEV)
    outs = []
    for fill in (0, 127, 255):
        ws = torch.full((n,), fill, dtype=torch.uint8, device=DEV)
        acc = torch.zeros(2, 333, device=DEV)
        kernels.mx4_accumulate_weights(b.q.to(DEV), lse, *args, acc, b.sm, 16, workspace=ws)
        outs.append(acc)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and outs[0][0, :200].min() > 0
    with pytest.raises(ValueError, match="workspace"):
        kernels.mx4_accumulate_weights(b.q.to(DEV), lse, *args, acc, b.sm, 16, workspace=ws[:n - 16])


def test_weights_of_a_decode_step_and_the_attention_calls_lse():
    b = Batch(512, 16, [100, 3000, 1], [1, 1, 1], 64, seed=9)
    check_weights(b, decode=True)
    lse = torch.empty(3, 16, device=DEV)
    b.run(lse=lse, decode=True)
    acc = torch.zeros(3, 3000, device=DEV)
    for _ in range(2):
        evict.accumulate_weights(b.q.to(DEV), lse, b.pool, 0, acc, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm,
                                 page_size=64)
    # a row's weights add up to one: 16 heads, twice (the attention's scores are off by some 2^-18 of a score)
    assert ((acc.sum(1) - 32).abs() <= 32 * 2.0 ** -14).all()


def test_rows_and_columns_that_are_not_there():
    b = Batch(256, 8, [150, 90, 200], [1, 2, 1], 32, seed=4)
    check_weights(b, reqs=[-1, 4, 9])
    check_weights(b, cols=128)


def test_a_nan_row_is_seen_where_it_is_seen():
    D, H = 512, 16
    for qlens, rows in (([4, 4], 64), ([5, 5], 80)):
        b = Batch(D, H, [200, 70], qlens, 64, seed=6)
        acc = torch.zeros(2, 200, device=DEV)
        lse = torch.zeros(sum(qlens), H, device=DEV)

        def run():
            evict.accumulate_weights(b.q.to(DEV), lse, b.pool, 0, acc, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm,
                                     qo_indptr=b.qo, max_q_len=max(qlens), page_size=64, add=False)
            return acc.clone()

        clean = run()
        assert torch.isfinite(clean).all()
        b.pool.c_scales[0][int(b.slots[0][50]), 3] = 255
        bad = run()
        assert torch.isnan(bad[0, 50]) and torch.isfinite(bad).sum() == bad.numel() - 1
        same = torch.isfinite(bad)
        assert torch.equal(bad[same], clean[same])
        lse[1, 2] = float("-inf")  # a row that saw nothing
        lse[0] = float("inf")
        assert torch.isfinite(run()[:, :50]).all()


def test_weights_do_not_depend_on_the_batch():
    b = Batch(512, 16, [900, 333, 64], [3, 1, 4], 16, seed=8)
    lse = torch.zeros(b.T, 16, device=DEV)
    acc = torch.zeros(3, 900, device=DEV)
    args = dict(max_q_len=4, page_size=16, add=False)
    evict.accumulate_weights(b.q.to(DEV), lse, b.pool, 0, acc, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm,
                             qo_indptr=b.qo, **args)
    one = torch.zeros(1, 900, device=DEV)
    p = b.kv_indptr.tolist()
    evict.accumulate_weights(b.q[:3].to(DEV), lse[:3], b.pool, 0, one, b.kv_indptr[:2], b.kv_indices[:p[1]],
                             b.kv_lens[:1], b.sm, qo_indptr=b.qo[:2], **args)
    assert torch.equal(one[0], acc[0])


# ---- eviction ------------------------------------------------------------------------
def expected(w, slots, budget, sink, recent):
    """(positions that stay, the others) of one request."""
    n = len(slots)
    if n <= budget:
        return np.arange(n), np.zeros(0, dtype=np.int64)
    mid = np.arange(sink, n - recent)
    v = w[mid].astype(np.float64)
    order = mid[np.lexsort((mid, np.where(np.isnan(v), -np.inf, -v), ~np.isnan(v)))]
    stay = np.concatenate([np.arange(sink), order[:budget - sink - recent], np.arange(n - recent, n)])
    keep = np.zeros(n, dtype=bool)
    keep[stay] = True
    return np.nonzero(keep)[0], np.nonzero(~keep)[0]


def run_evict(lens, budget, sink, recent, page, w=None, seed=0, reqs=None, in_place=False, cols=None, max_kv_len=None,
              freed_size=None):
    B = len(lens)
    slots, pages, _ = alloc_slots(lens, page, seed)
    cols = max(max(lens), 1) + 5 if cols is None else cols
    g = np.random.default_rng(seed)
    rows = B + 2
    acc = g.lognormal(0, 3, (rows, cols)).astype(np.float32) if w is None else w
    reqs = list(range(B)) if reqs is None else reqs
    indptr = torch.tensor(np.concatenate(([0], np.cumsum([len(p) for p in pages]))), dtype=torch.int32, device=DEV)
    indices = torch.tensor(np.concatenate([*pages, np.zeros(0)]), dtype=torch.int32, device=DEV)
    total = int(indices.numel() * page) + 2 if freed_size is None else freed_size
    freed = torch.full((total,), -7, dtype=torch.int32, device=DEV)
    kept = torch.full((B, budget), -7, dtype=torch.int32, device=DEV)
    a = torch.from_numpy(acc).to(DEV)
    out = a if in_place else torch.full_like(a, -3.0)
    k, kl, f = evict.evict(a, indptr, indices, torch.tensor(lens, device=DEV), budget, sink, recent, page_size=page,
                           req_pool_indices=torch.tensor(reqs, device=DEV), acc_out=None if in_place else out,
                           kept=kept, freed=freed, max_kv_len=max_kv_len)
    assert k is kept and f is freed
    if not in_place:
        assert torch.equal(a.cpu().view(torch.int32), torch.from_numpy(acc).view(torch.int32))
    want_out = acc.copy() if in_place else np.full_like(acc, -3.0)
    want_freed, gone = np.full(total, -7, dtype=np.int32), []
    for b, n in enumerate(lens):
        n = min(n, cols, n if max_kv_len is None else max_kv_len)
        there = 0 <= reqs[b] < rows
        stay, rest = expected(acc[reqs[b]] if there else np.zeros(cols, np.float32), slots[b][:n], budget, sink, recent)
        want = np.full(budget, -7)
        want[:len(stay)] = slots[b][stay]
        assert int(kl[b]) == len(stay) and np.array_equal(k[b].cpu().numpy(), want), (b, n)
        gone.append(slots[b][rest])
        if there:
            want_out[reqs[b], :n] = 0
            want_out[reqs[b], :len(stay)] = acc[reqs[b]][stay]
    gone = np.concatenate(gone)[:total]
    want_freed[:len(gone)] = gone
    assert np.array_equal(f.cpu().numpy(), want_freed)
    assert np.array_equal(out.cpu().numpy().view(np.int32), want_out.view(np.int32))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget,sink,recent,page", [
    ([1], 1, 0, 0, 1), ([2], 1, 0, 0, 1), ([2], 1, 1, 0, 1), ([2], 1, 0, 1, 1), ([0, 5, 0], 3, 1, 1, 2),
    ([100, 64, 65, 7], 64, 4, 16, 16), ([1000], 999, 4, 16, 64), ([1000, 3000, 500], 20, 4, 16, 64),
    ([1025, 16384], 700, 0, 700, 1), ([16385, 20], 300, 4, 16, 32), ([40000, 16384, 33000, 0], 9000, 16, 64, 64),
    ([140000], 131, 4, 127, 64), ([32768], 16000, 0, 16000, 1), ([50000], 20000, 18000, 1, 1),
])
def test_evict(lens, budget, sink, recent, page, in_place):
    run_evict(lens, budget, sink, recent, page, seed=len(lens) + budget, in_place=in_place)


@pytest.mark.parametrize("n,budget", [(900, 300), (20000, 7001)])
def test_equal_weights_go_to_the_earlier_position(n, budget):
    g = np.random.default_rng(n)
    for values in ([1.0], [0.0, -0.0], [0.5, 0.25, np.inf, -1.0, 0.0, -0.0], [np.nan, 1.0, np.inf, -np.inf],
                   [1e-45, 0.0, 3e-39, -1e-45]):
        w = g.choice(np.array(values, dtype=np.float32), (3, n + 5))
        run_evict([n], budget, 4, 16, 16, w=w, seed=n)


@pytest.mark.parametrize("lens", [[4091, 1000], [4092, 1025], [16384, 100], [16385, 4096, 0], [40961], [196608], [196609, 16384, 300], [300000]])
def test_long_requests(lens):
    # either side of every change of blocks and chunks, with equal weights across chunks
    g = np.random.default_rng(len(lens))
    w = (np.floor(g.random((len(lens) + 2, max(lens) + 5)) * 500) * 2.0 ** -10).astype(np.float32)
    run_evict(lens, 5000, 7, 300, 16, w=w)
    run_evict(lens, 400, 0, 400, 1, w=w, in_place=True)
    run_evict(lens, 401, 400, 0, 1, w=w)


def test_weights_that_differ_in_their_last_bits():
    for d in (1, 1 << 10, 1 << 21):
        bits = 0x3f800000 + d * np.random.default_rng(d).integers(0, 3000 if d < 1 << 21 else 3, (3, 5005))
        run_evict([5000], 1200, 4, 16, 64, w=bits.astype(np.int32).view(np.float32), seed=d)


def test_rows_columns_and_room_that_are_not_there():
    run_evict([300, 200, 100], 50, 4, 16, 16, reqs=[4, -1, 5])  # outside: all weights count as 0
    run_evict([300, 200], 50, 4, 16, 16, cols=256)  # positions past the columns take no part
    run_evict([300, 20000], 50, 4, 16, 16, max_kv_len=250)
    run_evict([300, 20000], 50, 4, 16, 16, max_kv_len=17000)
    run_evict([300, 200], 50, 4, 16, 16, freed_size=260)


def test_many_requests():
    g = np.random.default_rng(5)
    run_evict(g.integers(0, 400, 300).tolist(), 100, 4, 16, 8, seed=5)


def test_allocated_outputs():
    w = torch.rand(2, 64, device=DEV)
    kept, lens, freed = evict.evict(w, torch.tensor([0, 4, 8], dtype=torch.int32, device=DEV),
                                    torch.arange(1, 9, dtype=torch.int32, device=DEV), torch.tensor([60, 64], device=DEV),
                                    32, page_size=16)
    assert kept.shape == (2, 32) and lens.tolist() == [32, 32] and freed.numel() == 128
    both = torch.cat((kept.flatten(), freed[:60])).sort().values
    slots = torch.cat((torch.arange(16, 76), torch.arange(80, 144))).to(DEV)
    assert torch.equal(both.long(), slots)
