"""Rows with an LSE of -inf weigh nothing, whatever their queries hold: padding of a batch, queries without keys."""

import pytest
import torch

from mla_kv_quant_amd import evict
from tests.test_gpu_mx4 import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D,H,lens,qlens", [
    (512, 16, [300, 70], [1, 1]), (512, 16, [300, 70], [4, 2]), (256, 40, [300, 70], [1, 1]),  # rows kept in LDS
    (512, 16, [700, 170], [9, 13]), (256, 40, [2000, 300], [33, 8]), (512, 128, [170, 51], [51, 20]),  # streamed, parts
])
def test_rows_that_weigh_nothing(D, H, lens, qlens, what):
    b = Batch(D, H, lens, qlens, 16, seed=2)
    lse, q = torch.full((b.T, H), 2.0, device=DEV), b.q.to(DEV)
    rows = torch.rand(b.T, H, generator=torch.Generator().manual_seed(3)).to(DEV) < 0.2
    rows[qlens[0] - 1, :2] = rows[-1] = True
    lse[rows] = float("-inf")

    def run(q):
        acc = torch.full((2, max(lens)), 1.5, device=DEV)
        evict.accumulate_weights(q, lse, b.pool, 0, acc, b.kv_indptr, b.kv_indices, b.kv_lens, b.sm, qo_indptr=b.qo,
                                 max_q_len=max(qlens), page_size=16)
        return acc

    want = run(q)
    assert torch.isfinite(want).all() and (want[0, :lens[0]] > 1.5).any()
    q[rows] = what
    assert torch.equal(run(q), want)
    lse.fill_(float("-inf"))  # a batch of nothing else
    q.fill_(what)
    assert (run(q) == 1.5).all()
