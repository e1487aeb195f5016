"""Accumulated weights and eviction with workspaces that their caller gives, whatever they hold, and keeps for the next call."""

import pytest
import torch

from mla_kv_quant_amd import evict, kernels
from tests.test_gpu_evict_outputs import batch
from tests.test_gpu_mx4 import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_of_weights():
    b = Batch(512, 64, [200, 333], [40, 9], 16, seed=15)
    n = kernels.accumulate_weights_workspace_bytes(b.T, 2, 64, 512, b.kv_indices.shape[0], 16, 40, DEV)
    assert n > 0
    q, lse = b.q.to(DEV), torch.full((b.T, 64), 2.0, device=DEV)

    def run(**kw):
        acc = torch.zeros(2, 333, device=DEV)
        return evict.accumulate_weights(q, lse, b.pool, 0, acc, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm, qo_indptr=b.qo,
                                        max_q_len=40, page_size=16, **kw)

    want, ws = run(), torch.full((n,), 255, dtype=torch.uint8, device=DEV)
    for _ in range(2):
        assert torch.equal(run(workspace=ws), want)
    with pytest.raises(ValueError, match="workspace"):
        run(workspace=ws[:n - 16])


@pytest.mark.parametrize("lens,cols", [([17000, 300], 17000), ([200, 300], 70000)])
def test_of_eviction(lens, cols):
    acc, ptr, ids, n = batch(lens, cols)
    size = kernels.evict_workspace_bytes(2, cols, DEV)
    ws = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    args, out = (acc, ptr, ids, n, 100), torch.zeros_like(acc)
    want = evict.evict(*args, acc_out=out)
    for kw in ({"workspace": ws}, {"workspace": ws}, {"max_kv_len": max(lens)}):
        again = torch.zeros_like(acc)
        got = evict.evict(*args, acc_out=again, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(again, out)
    with pytest.raises(ValueError, match="workspace"):
        evict.evict(*args, acc_out=out, workspace=ws[:size - 16])
