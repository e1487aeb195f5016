"""Eviction's outputs beside its inputs in one storage, and where they may not lie."""

import pytest
import torch

from mla_kv_quant_amd import evict

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32


def batch(lens, cols, seed=1):
    """(acc, offsets, list, lengths) of requests with pages of one slot in shuffled order."""
    g = torch.Generator().manual_seed(seed)
    at = [sum(lens[:i]) for i in range(len(lens) + 1)]
    return (torch.rand(len(lens), cols, generator=g).to(DEV), torch.tensor(at, dtype=I32, device=DEV),
            torch.randperm(at[-1], generator=g).to(I32).to(DEV), torch.tensor(lens, device=DEV))


@pytest.mark.parametrize("most", [3000, 40000])
def test_outputs_beside_inputs_in_one_storage(most):
    lens, budget = [most, 50, most - 7], 60
    acc, ptr, ids, n = batch(lens, most)
    out = torch.full_like(acc, 7.0)
    kept, kept_lens, freed = evict.evict(acc, ptr, ids, n, budget, acc_out=out)
    count = sum(max(m - budget, 0) for m in lens)
    wide = torch.full((3, 2 * most), 7.0, device=DEV)  # acc and acc_out side by side in the same rows
    wide[:, most:] = acc
    total, room = ids.numel(), 3 * budget
    ints = torch.cat((torch.zeros(room, dtype=I32, device=DEV), ids, torch.zeros(count, dtype=I32, device=DEV)))
    longs = torch.cat((n, torch.zeros(3, dtype=torch.int64, device=DEV)))
    k, kl, f = evict.evict(wide[:, most:], ptr, ints[room:room + total], longs[:3], budget, acc_out=wide[:, :most],
                           kept=ints[:room].view(3, budget), kept_lens=longs[3:], freed=ints[room + total:])
    assert torch.equal(kl, kept_lens) and torch.equal(f, freed[:count])
    assert all(torch.equal(k[b, :m], kept[b, :m]) for b, m in enumerate(kept_lens.tolist()))
    assert torch.equal(wide[:, :most], out) and torch.equal(wide[:, most:], acc)
    assert torch.equal(ints[room:room + total], ids) and torch.equal(longs[:3], n)


def test_outputs_on_inputs_are_refused():
    acc, ptr, ids, n = batch([500, 300], 500)
    with pytest.raises(ValueError, match="kept_lens must not overlap kv_lens"):
        evict.evict(acc, ptr, ids, n, 60, kept_lens=n)
    with pytest.raises(ValueError, match="kept must not overlap kv_indices"):
        evict.evict(acc, ptr, ids, n, 60, kept=ids[100:220].view(2, 60))
    with pytest.raises(ValueError, match="freed must not overlap kv_indices"):
        evict.evict(acc, ptr, ids, n, 60, freed=ids)
    with pytest.raises(ValueError, match="acc_out must not overlap acc"):
        evict.evict(acc[:, :400], ptr, ids, n, 60, acc_out=acc[:, 100:])
    assert n.tolist() == [500, 300]


@pytest.mark.parametrize("lens,cols,kw,cut", [
    ([500, 90, 300], 500, {}, [500, 90, 300]), ([500, 90, 300], 200, {}, [200, 90, 200]),
    ([500, 90, 300], 500, {"max_kv_len": 250}, [250, 90, 250]), ([20000, 90], 18000, {}, [18000, 90]),
    ([20000, 400], 20000, {"max_kv_len": 17000}, [17000, 400]), ([30, 90], 100, {}, [30, 90]),
])
def test_how_many_are_freed(lens, cols, kw, cut):
    acc, ptr, ids, n = batch(lens, cols)
    torch.full((ids.numel(),), 5, dtype=I32, device=DEV)  # (what an allocation may find)
    kept, kept_lens, freed = evict.evict(acc, ptr, ids, n, 64, **kw)
    gone = freed[freed >= 0]
    assert gone.numel() == (torch.tensor(cut) - kept_lens.cpu()).sum() and (freed[gone.numel():] == -1).all()
    at, seen = 0, ids.tolist()
    for b, m in enumerate(cut):
        own = seen[sum(lens[:b]):sum(lens[:b]) + m]
        rest = m - int(kept_lens[b])
        assert sorted(kept[b, :int(kept_lens[b])].tolist() + gone[at:at + rest].tolist()) == sorted(own)
        at += rest


def test_requests_longer_than_their_lists():
    acc, ptr, ids, _ = batch([500, 300], 600)
    kept, kept_lens, freed = evict.evict(acc, ptr, ids, torch.tensor([600, 10 ** 9], device=DEV), 64)
    assert kept_lens.tolist() == [64, 64] and (freed >= 0).sum() == 800 - 128
