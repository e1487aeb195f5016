"""The operators around the caches together: a prompt's prefill in the expanded form, the weights of its last
queries, eviction, and decode steps over what stays -- eagerly and from a captured graph.

Tolerances: rows go through two bf16 roundings (the cache's values, then kv_b_proj's output) that
the float64 side makes too, so the attentions' own apply: 2^-8 for the weights' rounding and 2^-8 for
the output's, of the largest weighted values, times two for the rounded operands' products.
"""

import math

import pytest
import torch

from mla_kv_quant_amd import MX4MLAPool, evict, expanded, mx4, rotary

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def softmax64(s):
    return torch.exp(s - torch.logsumexp(s, -1, keepdim=True))


@pytest.mark.parametrize("D,R,dn,H", [(512, 64, 128, 16), (256, 32, 64, 40)])
def test_prefill_evict_decode(D, R, dn, H):
    g = torch.Generator().manual_seed(D)
    lens, window, budget, sink, recent = [400, 333], 8, 96, 4, 16
    T, sm = sum(lens), (dn + R) ** -0.5
    rand = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(BF).to(DEV)  # noqa: E731
    latent, k_pe, q_all = rand(T, D), rand(T, R), rand(T, H, dn + R, std=2.0)
    w_b = rand(H, 2 * dn, D, std=D ** -0.5)  # kv_b_proj: (k_nope | v) of each head
    rope = rotary.Rotary(R, scaling={"type": "yarn", "factor": 8, "original_max_position_embeddings": 4096}, device=DEV)
    pool = MX4MLAPool(1023, 1, D, R, device=DEV)
    perm = torch.randperm(1023, generator=g)[:T + 2].to(DEV) + 1
    slots = perm[:T]
    pos = torch.cat([torch.arange(n) for n in lens]).to(DEV)
    indptr = torch.tensor([0, lens[0], T], dtype=torch.int32, device=DEV)

    # prefill: rotate, store, read back, expand, attend
    plain_pe = k_pe.clone()
    rotary.apply_rotary(rope, pos, q_all[..., dn:], k_pe)
    assert not torch.equal(k_pe, plain_pe)
    mx4.write_rows(pool, 0, slots, latent, k_pe)
    rows = mx4.read_rows(pool, 0, slots)
    assert torch.equal(rows[:, D:], k_pe)
    kv = (rows[:, :D] @ w_b.reshape(-1, D).t()).view(T, H, 2 * dn)
    o = torch.empty(T, H, dn, dtype=BF, device=DEV)
    expanded.expanded_attend_fwd(q_all, kv, rows[:, D:], o, indptr, indptr, max(lens), sm)
    for b, n in enumerate(lens):
        i = sum(lens[:b])
        k = torch.cat((kv[i:i + n, :, :dn], rows[i:i + n, None, D:].expand(n, H, R)), -1).double()
        s = torch.einsum("thd,nhd->htn", q_all[i:i + n].double(), k) * sm
        w = softmax64(s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), float("-inf")))
        v = kv[i:i + n, :, dn:].double().transpose(0, 1)
        want, big = (w @ v).transpose(0, 1), (w @ v.abs()).transpose(0, 1)
        assert ((o[i:i + n].double() - want).abs() <= 2.0 ** -7 * big + 1e-6).all()

    # the weights of each prompt's last queries, in the absorbed form, over the cache
    last = torch.cat([torch.arange(sum(lens[:b + 1]) - window, sum(lens[:b + 1])) for b in range(2)]).to(DEV)
    absorb = lambda x: torch.cat((torch.matmul(x[..., :dn].float().transpose(0, 1), w_b[:, :dn].float())  # noqa: E731
                                  .transpose(0, 1).to(BF), x[..., dn:]), -1).contiguous()
    q = absorb(q_all[last])
    qo = torch.tensor([0, window, 2 * window], dtype=torch.int32, device=DEV)
    kv_lens = torch.tensor(lens, device=DEV)
    lse, ol = torch.empty(2 * window, H, device=DEV), torch.empty(2 * window, H, D, dtype=BF, device=DEV)
    indices = slots.to(torch.int32)
    mx4.attend_fwd(q, ol, pool, 0, indptr, indices, kv_lens, sm, qo_indptr=qo, max_q_len=window, lse=lse)
    acc = torch.full((4, 512), float("nan"), device=DEV)
    reqs = torch.tensor([3, 1], device=DEV)
    evict.accumulate_weights(q, lse, pool, 0, acc, indptr, indices, kv_lens, sm, qo_indptr=qo, max_q_len=window,
                             req_pool_indices=reqs, add=False)
    for b, n in enumerate(lens):
        i = sum(lens[:b])
        s = torch.einsum("thd,nd->thn", q[window * b:window * (b + 1)].double(), rows[i:i + n].double()) * sm
        s = s.masked_fill(torch.arange(n, device=DEV) > n - window + torch.arange(window, device=DEV)[:, None, None],
                          float("-inf"))
        want = softmax64(s).sum((0, 1))
        assert ((acc[reqs[b], :n].double() - want).abs() <= 2.0 ** -12 * want + 1e-9).all()
    assert torch.isnan(acc[[0, 2]]).all()

    # eviction: acc stays with the positions
    before = acc.clone()
    kept, kept_lens, freed = evict.evict(acc, indptr, indices, kv_lens, budget, sink, recent, req_pool_indices=reqs)
    assert kept_lens.tolist() == [budget, budget]
    gone = set(freed[:T - 2 * budget].tolist())
    assert gone | set(kept.flatten().tolist()) == set(indices.tolist()) and len(gone) == T - 2 * budget
    for b, n in enumerate(lens):
        where = {int(s): j for j, s in enumerate(indices[sum(lens[:b]):sum(lens[:b + 1])].tolist())}
        at = torch.tensor([where[int(s)] for s in kept[b].tolist()], device=DEV)
        assert (at[1:] > at[:-1]).all() and at[:sink].tolist() == list(range(sink))
        assert at[-recent:].tolist() == list(range(n - recent, n))
        assert torch.equal(acc[reqs[b], :budget], before[reqs[b]][at]) and (acc[reqs[b], budget:n] == 0).all()

    # a decode step over what stays and one new position, eagerly and as a graph
    lists = torch.zeros(2, budget + 1, dtype=torch.int32, device=DEV)
    lists[:, :budget] = kept
    lists[:, budget] = perm[T:].to(torch.int32)
    st = {"pos": torch.tensor(lens, device=DEV), "latent": rand(2, D), "pe": rand(2, R), "x": rand(2, H, dn + R, std=2.0)}
    ptr = torch.tensor([0, budget + 1, 2 * budget + 2], dtype=torch.int32, device=DEV)
    n1 = torch.full((2,), budget + 1, device=DEV)
    q1, pe1 = torch.empty(2, H, D + R, dtype=BF, device=DEV), torch.empty(2, R, dtype=BF, device=DEV)
    out, l1 = torch.empty(2, H, D, dtype=BF, device=DEV), torch.empty(2, H, device=DEV)
    w1 = torch.zeros(4, 512, device=DEV)
    small, small_lens = torch.empty(2, 64, dtype=torch.int32, device=DEV), torch.empty(2, dtype=torch.int64, device=DEV)
    rest, w2 = torch.zeros(2 * budget + 2, dtype=torch.int32, device=DEV), torch.zeros(4, 512, device=DEV)
    again = torch.empty(2, H, dn, dtype=BF, device=DEV)

    def step():
        q1[..., :D] = torch.matmul(st["x"][..., :dn].float().transpose(0, 1), w_b[:, :dn].float()).transpose(0, 1)
        rotary.apply_rotary(rope, st["pos"], st["x"][..., dn:], st["pe"], q1[..., D:], pe1)
        mx4.write_rows(pool, 0, perm[T:], st["latent"], pe1)
        mx4.attend_fwd(q1, out, pool, 0, ptr, lists.view(-1), n1, sm, lse=l1)
        evict.accumulate_weights(q1, l1, pool, 0, w1, ptr, lists.view(-1), n1, sm, add=False)
        evict.evict(w1, ptr, lists.view(-1), n1, 64, sink, recent, max_kv_len=budget + 1, acc_out=w2, kept=small,
                    kept_lens=small_lens, freed=rest)
        expanded.expanded_attend_fwd(st["x"], kv, rows[:, D:], again, qo1, indptr, 1, sm)

    qo1 = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    names = lambda: [t.clone() for t in (q1, pe1, out, l1, w1, w2, small, small_lens, rest, again)]  # noqa: E731
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        st["latent"].copy_(rand(2, D))
        st["pe"].copy_(rand(2, R))
        st["x"].copy_(rand(2, H, dn + R, std=2.0))
        st["pos"].add_(1)
        step()
        want = names()
        for t in (q1, pe1, out, l1, w1, w2, small, small_lens, rest, again):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(names(), want):
            assert torch.equal(a, b)
    k = mx4.read_rows(pool, 0, lists.view(-1).long(), unrotate=False).view(2, budget + 1, D + R).double()
    s = torch.einsum("bhd,bnd->bhn", q1.double(), k) * sm
    w = softmax64(s)
    want, big = w @ k[..., :D], w @ k[..., :D].abs()
    assert ((out.double() - want).abs() <= 2.0 ** -7 * big).all()
    assert ((w1[:2, :budget + 1].double() - w.sum(1)).abs() <= 2.0 ** -12 * w.sum(1) + 1e-9).all()
