"""Captured calls that choose their parts on the device, replayed for other lengths, and two streams at once.

Results are those of the same call made eagerly, bit for bit.
"""

import pytest
import torch

from mla_kv_quant_amd import evict, expanded, rotary
from tests.test_gpu_mx4 import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
I32 = torch.int32


def offsets(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=I32, device=DEV)


def captured(call, outs, states, replays=2):
    """``call`` eagerly and from one graph for each of ``states`` (functions that change its inputs in place)."""
    states[0]()
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    seen = []
    for change in states:
        change()
        for t in outs:
            t.fill_(3)
        call()
        want = [t.clone() for t in outs]
        for _ in range(replays):
            for t in outs:
                t.fill_(3)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        seen.append(want)
    assert any(not torch.equal(a, b) for a, b in zip(seen[0], seen[-1]))


def test_expanded_attention_of_other_lengths():
    T, N, H, dn = 300, 9000, 2, 128
    g = torch.Generator().manual_seed(1)
    q, kv, pe = (torch.randn(*s, generator=g).to(BF).to(DEV) for s in ((T, H, 192), (N, H, 256), (N, 64)))
    qo, ki = torch.zeros(4, dtype=I32, device=DEV), torch.zeros(4, dtype=I32, device=DEV)
    o, lse = torch.zeros(T, H, dn, dtype=BF, device=DEV), torch.zeros(T, H, device=DEV)

    def lens(qs, ks):
        return lambda: (qo.copy_(offsets(qs)), ki.copy_(offsets(ks)))

    captured(lambda: expanded.expanded_attend_fwd(q, kv, pe, o, qo, ki, 200, dn ** -0.5, lse=lse), (o, lse),
             [lens([200, 99, 1], [200, 99, 1]), lens([1, 150, 40], [8000, 151, 800]), lens([0, 0, 3], [0, 0, 9000]),
              lens([0, 0, 0], [5, 5, 5]), lens([60, 200, 0], [4000, 5000, 0])])


@pytest.mark.parametrize("D,H", [(512, 64), (256, 40)])
def test_weights_and_eviction_of_other_lengths(D, H):
    b = Batch(D, H, [700, 400], [30, 30], 16, seed=3)
    q, lse = b.q.to(DEV), torch.full((b.T, H), 2.0, device=DEV)
    lens, acc = b.kv_lens.clone(), torch.zeros(2, 700, device=DEV)

    def set_lens(*n):
        return lambda: lens.copy_(torch.tensor(n))

    captured(lambda: evict.accumulate_weights(q, lse, b.pool, 0, acc, b.kv_indptr, b.kv_indices, lens, b.sm,
                                              qo_indptr=b.qo, max_q_len=30, page_size=16, add=False), (acc,),
             [set_lens(700, 400), set_lens(31, 33), set_lens(0, 400), set_lens(64, 1)])


@pytest.mark.parametrize("most", [3000, 50000])
def test_eviction_of_other_lengths(most):
    g = torch.Generator(device=DEV).manual_seed(4)
    acc = torch.rand(3, most, generator=g, device=DEV)
    ptr, idx = offsets([most] * 3), torch.randperm(3 * most, generator=g, device=DEV).to(I32)
    lens = torch.zeros(3, dtype=torch.int64, device=DEV)
    kept, kl = torch.zeros(3, 900, dtype=I32, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    freed, out = torch.zeros(3 * most, dtype=I32, device=DEV), torch.zeros_like(acc)

    def state(*n):
        return lambda: (lens.copy_(torch.tensor(n)), acc.uniform_(generator=g))

    captured(lambda: evict.evict(acc, ptr, idx, lens, 900, acc_out=out, kept=kept, kept_lens=kl, freed=freed),
             (kept, kl, freed, out), [state(most, most, most), state(0, 900, most - 1), state(901, 1, 17), state(most, 0, 2000)])


def test_rotary_of_other_positions():
    rope = rotary.Rotary(64, device=DEV)
    p, q, k = torch.arange(50, device=DEV), torch.randn(50, 4, 64, device=DEV).to(BF), torch.randn(50, 64, device=DEV).to(BF)
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    captured(lambda: rotary.apply_rotary(rope, p, q, k, qo, ko), (qo, ko),
             [lambda: None, lambda: p.add_(1 << 40), lambda: q.mul_(2)])


def test_two_streams_at_once():
    b = [Batch(512, 64, [300, 200], [40, 20], 16, seed=s) for s in (5, 6)]
    g = torch.Generator().manual_seed(7)
    xs = [[torch.randn(*s, generator=g).to(BF).to(DEV) for s in ((40, 2, 192), (6000, 2, 256), (6000, 64))] for _ in b]
    lse = torch.full((60, 64), 2.0, device=DEV)
    qs = [x.q.to(DEV) for x in b]

    def work(i):
        acc, o = torch.zeros(2, 300, device=DEV), torch.zeros(40, 2, 128, dtype=BF, device=DEV)
        evict.accumulate_weights(qs[i], lse, b[i].pool, 0, acc, b[i].kv_indptr, b[i].kv_indices, b[i].kv_lens, b[i].sm,
                                 qo_indptr=b[i].qo, max_q_len=40, page_size=16)
        expanded.expanded_attend_fwd(*xs[i], o, ptrs[0], ptrs[1], 40, 0.1)
        w = torch.linspace(0, 1, 40000, device=DEV)[None].contiguous()
        kept, _, freed = evict.evict(w, ptrs[2], ids, n, 1000 + i)
        return acc, o, kept, freed[:40000 - 1000 - i].clone()

    ptrs = [offsets([40]), offsets([6000]), offsets([40000])]
    ids, n = torch.arange(40000, dtype=I32, device=DEV), torch.tensor([40000], device=DEV)
    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in b]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))
