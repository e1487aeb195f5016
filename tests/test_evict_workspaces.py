"""Workspaces that a caller gives to the accumulated weights and to eviction (CPU only)."""

import pytest
import torch

from mla_kv_quant_amd import evict, kernels
from mla_kv_quant_amd.mx4 import MX4MLAPool

I32 = torch.int32


def test_size_of_evictions():
    assert kernels.evict_workspace_bytes(4, 16384, "cpu") == 0 and kernels.evict_workspace_bytes(0, 1 << 20, "cpu") == 0
    one = kernels.evict_workspace_bytes(1, 16385, "cpu")
    assert one > 4 * 16385 and kernels.evict_workspace_bytes(4, 16385, "cpu") == 4 * one
    for bad in ((-1, 5), (1, -5), (1, (1 << 30) + 1)):
        with pytest.raises(ValueError, match="invalid"):
            kernels.evict_workspace_bytes(*bad, "cpu")


def test_the_weights_workspace_is_passed_on(monkeypatch):
    pool, seen = MX4MLAPool(7, 1, 256, 32, device="cpu"), []
    monkeypatch.setattr(kernels, "mx4_accumulate_weights", lambda *a, **kw: seen.append((a, kw)))
    ws = torch.zeros(64, dtype=torch.uint8)
    args = (torch.zeros(2, 4, 288, dtype=torch.bfloat16), torch.zeros(2, 4), pool, 0, torch.zeros(3, 10),
            torch.tensor([0, 1, 2], dtype=I32), torch.tensor([1, 2], dtype=I32), torch.tensor([1, 1]), 0.1)
    evict.accumulate_weights(*args, workspace=ws)
    evict.accumulate_weights(*args)
    assert any(v is ws for v in [*seen[0][0], *seen[0][1].values()])
    assert not any(v is ws for v in [*seen[1][0], *seen[1][1].values()])
    monkeypatch.undo()
    with pytest.raises(TypeError, match="workspace"):
        evict.accumulate_weights(*args, workspace=torch.zeros(64))
