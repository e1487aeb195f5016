"""What eviction allocates when its caller gives no outputs (CPU only; the kernel's part is replaced)."""

import torch

from mla_kv_quant_amd import evict, kernels


def test_entries_of_freed_that_no_slot_takes_are_marked(monkeypatch):
    def some(acc, ptr, ids, lens, budget, sink, recent, page, req, most, out, kept, kept_lens, freed, ws):
        freed[:3] = torch.tensor([7, 8, 9])

    monkeypatch.setattr(kernels, "evict", some)
    args = (torch.zeros(2, 64), torch.tensor([0, 2, 4], dtype=torch.int32), torch.arange(4, dtype=torch.int32),
            torch.tensor([60, 64]), 32)
    freed = evict.evict(*args, page_size=16)[2]
    assert freed[:3].tolist() == [7, 8, 9] and freed.shape == (64,) and (freed[3:] == -1).all()
    given = torch.full((50,), 4, dtype=torch.int32)
    assert evict.evict(*args, page_size=16, freed=given)[2] is given and (given[3:] == 4).all()
