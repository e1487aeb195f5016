"""Refusals of the MX4 entry points: by the tensor checks and by the C ABI, before any launch (CPU only)."""

import ctypes

import pytest
import torch

from mla_kv_quant_amd import MX4MLAPool, _lib, mx4

P = ctypes.c_void_p(4096)
BF = torch.bfloat16


def refused(fn, args, word):
    assert fn(*args) == _lib.ROLAQ_ERR_INVALID
    assert word in _lib.load().rolaq_last_error().decode(), _lib.load().rolaq_last_error()


def changed(args, **by_index):
    out = list(args)
    for k, v in by_index.items():
        out[int(k[1:])] = v
    return out


def test_write_rows_arguments():
    fn = _lib.load().rolaq_mx4_write_rows
    ok = [P, 512, P, 64, 1, P, P, 8, 512, 64, P, P, P, 100, None]
    assert fn(*changed(ok, i7=0)) == _lib.ROLAQ_OK  # no rows: nothing to do
    refused(fn, changed(ok, i7=-1), "n < 0")
    refused(fn, changed(ok, i8=384), "(D, R)")
    refused(fn, changed(ok, i9=32), "(D, R)")
    refused(fn, changed(ok, i13=0), "num_slots")
    refused(fn, changed(ok, i13=1 << 31), "num_slots")
    refused(fn, changed(ok, i1=504), "stride")
    refused(fn, changed(ok, i1=516), "stride")
    refused(fn, changed(ok, i0=ctypes.c_void_p(4104)), "16-byte")
    refused(fn, changed(ok, i5=ctypes.c_void_p(4104)), "rotation")
    refused(fn, changed(ok, i7=(1 << 31) + 1), "2^31")
    for i in (0, 2, 6, 10, 11, 12):
        refused(fn, changed(ok, **{f"i{i}": None}), "null")
    for i in (10, 11, 12):
        refused(fn, changed(ok, **{f"i{i}": ctypes.c_void_p(4104)}), "aligned")


def test_read_rows_arguments():
    fn = _lib.load().rolaq_mx4_read_rows
    ok = [P, 8, P, P, P, 100, None, 512, 64, P, 576, None]
    assert fn(*changed(ok, i1=0)) == _lib.ROLAQ_OK
    refused(fn, changed(ok, i1=-1), "n < 0")
    refused(fn, changed(ok, i7=128), "(D, R)")
    refused(fn, changed(ok, i10=568), "stride")
    refused(fn, changed(ok, i10=580), "stride")
    refused(fn, changed(ok, i9=ctypes.c_void_p(4100)), "16-byte")
    refused(fn, changed(ok, i6=ctypes.c_void_p(4104)), "rotation")
    for i in (0, 2, 3, 4, 9):
        refused(fn, changed(ok, **{f"i{i}": None}), "null")


def test_attend_arguments():
    lib = _lib.load()
    fn = lib.rolaq_mx4_attend_fwd
    n = ctypes.c_int64(0)
    assert lib.rolaq_mx4_attend_workspace(512, ctypes.byref(n)) == _lib.ROLAQ_OK and n.value > 1 << 20
    refused(lib.rolaq_mx4_attend_workspace, [128, ctypes.byref(n)], "D must be")
    refused(lib.rolaq_mx4_attend_workspace, [512, None], "null")
    ok = [P, 16 * 576, 576, P, P, P, 100, P, P, P, 50, 64, P, 8, 4, 16, 512, 64, 2, 0.07, P, 16 * 512, 512, None, P,
          n.value, None]
    for i in (13, 14, 18):  # no queries, no requests, none to look at
        assert fn(*changed(ok, **{f"i{i}": 0})) == _lib.ROLAQ_OK
        refused(fn, changed(ok, **{f"i{i}": -1}), "negative")
    refused(fn, changed(ok, i15=0), "H must be")
    refused(fn, changed(ok, i15=129), "H must be")
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        refused(fn, changed(ok, i19=bad), "sm_scale")
    refused(fn, changed(ok, i11=3), "power of two")
    refused(fn, changed(ok, i11=0), "power of two")
    refused(fn, changed(ok, i16=384), "(D, R)")
    refused(fn, changed(ok, i6=0), "num_slots")
    refused(fn, changed(ok, i10=-1), "n_indices")
    refused(fn, changed(ok, i13=(1 << 24) + 1), "queries")
    refused(fn, changed(ok, i13=1 << 24, i15=128), "query rows")
    refused(fn, changed(ok, i7=None), "qo_indptr")            # two queries each need offsets
    refused(fn, changed(ok, i7=None, i18=1, i13=3), "qo_indptr")  # fewer queries than requests
    refused(fn, changed(ok, i14=1 << 30, i13=1 << 24, i18=1 << 20), "too large")
    for i, v in ((0, ctypes.c_void_p(4104)), (1, 9220), (2, 572), (2, 568), (1, -9216)):
        refused(fn, changed(ok, **{f"i{i}": v}), "q must be")
    for i, v in ((20, ctypes.c_void_p(4100)), (21, 8190), (22, 510), (22, 508), (21, -8192)):
        refused(fn, changed(ok, **{f"i{i}": v}), "out must be")
    refused(fn, changed(ok, i25=n.value - 1), "workspace")
    refused(fn, changed(ok, i24=ctypes.c_void_p(4128)), "workspace")
    for i in (0, 8, 9, 12, 20, 24):
        refused(fn, changed(ok, **{f"i{i}": None}), "null")


def small_pool(**kw):
    return MX4MLAPool(32, 2, device="cpu", **kw)


def test_pool():
    with pytest.raises(ValueError):
        MX4MLAPool(32, 1, 512, 32, device="cpu")
    pool = small_pool(start_layer=5, rotations=[None, torch.eye(512)])
    assert pool.latent_rotation(5) is None and pool.latent_rotation(6).dtype == BF
    assert pool.get_kv_size_bytes() == 33 * 2 * 400
    held = sum(t.numel() * t.element_size() for t in pool.c_codes + pool.c_scales + pool.rope_buf)
    assert held == pool.get_kv_size_bytes()


def test_row_tensors():
    pool = small_pool()
    loc = torch.arange(1, 5)
    x, pe = torch.zeros(4, 512, dtype=BF), torch.zeros(4, 64, dtype=BF)
    for bad in ((loc[:3], x, pe), (loc, x[:3], pe), (loc, x, pe[:3])):
        with pytest.raises(ValueError):
            mx4.write_rows(pool, 0, *bad)
    with pytest.raises(TypeError):
        mx4.write_rows(pool, 0, loc, x.float(), pe)
    with pytest.raises(TypeError):
        mx4.write_rows(pool, 0, loc, x, pe.float())
    with pytest.raises(ValueError):
        mx4.write_rows(pool, 0, loc, torch.zeros(512, 4, dtype=BF).t(), pe)
    with pytest.raises(ValueError):
        mx4.read_rows(pool, 0, loc, out=torch.zeros(3, 576, dtype=BF))
    with pytest.raises(ValueError):
        mx4.read_rows(pool, 0, loc, out=torch.zeros(4, 512, dtype=BF))
    with pytest.raises(TypeError):
        mx4.read_rows(pool, 0, loc, out=torch.zeros(4, 576))
    pool.c_scales[0] = pool.c_scales[0][:-1]
    with pytest.raises(ValueError):
        mx4.read_rows(pool, 0, loc)


def test_attend_tensors():
    pool = small_pool()
    ws = torch.zeros(16, dtype=torch.uint8)
    q, o = torch.zeros(3, 16, 576, dtype=BF), torch.zeros(3, 16, 512, dtype=BF)
    ptr, idx, lens = torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.ones(3, dtype=torch.int64)

    def call(q=q, o=o, ptr=ptr, idx=idx, lens=lens, **kw):
        mx4.attend_fwd(q, o, pool, 0, ptr, idx, lens, 0.1, workspace=ws, **kw)

    for kw in (dict(q=q.float()), dict(o=o.float()), dict(ptr=ptr.long()), dict(idx=idx.long()),
               dict(qo_indptr=ptr.long()), dict(lse=torch.zeros(3, 16, dtype=BF)), dict(lse=[0.0])):
        with pytest.raises(TypeError):
            call(**kw)
    for kw in (dict(q=torch.zeros(3, 16, 512, dtype=BF)), dict(q=torch.zeros(3, 576, 16, dtype=BF).transpose(1, 2)),
               dict(o=o[:2]), dict(o=o[:, :8]), dict(o=o[..., :256]), dict(ptr=ptr[:3]), dict(lens=lens[:2]),
               dict(lse=torch.zeros(3, 8)), dict(lse=torch.zeros(3, 32)[:, ::2]),
               dict(qo_indptr=torch.zeros(0, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call(**kw)


# ---- the rotation that a write takes: the layer's as it is now ------------------------
def written(monkeypatch, pool, layer=0):
    """R_eff^T that a write of one row hands to the kernel."""
    got = []
    monkeypatch.setattr(mx4.kernels, "mx4_write_rows", lambda x, pe, rt, *rest: got.append(rt))
    D, R = pool.kv_lora_rank, pool.qk_rope_head_dim
    mx4.write_rows(pool, layer, torch.ones(1, dtype=torch.int64), torch.zeros(1, D, dtype=BF), torch.zeros(1, R, dtype=BF))
    return got[0]


def rotation(seed):
    return torch.randn(256, 256, generator=torch.Generator().manual_seed(seed))


def laid_out(r):
    return r.to(BF).t().contiguous()


def test_a_rotation_that_changes_is_laid_out_again(monkeypatch):
    pool = MX4MLAPool(32, 2, 256, 32, device="cpu", rotations=[rotation(1), rotation(2)], start_layer=3)
    first = written(monkeypatch, pool, 3)
    assert torch.equal(first, laid_out(rotation(1))) and written(monkeypatch, pool, 3) is first  # laid out once
    assert torch.equal(written(monkeypatch, pool, 4), laid_out(rotation(2)))
    # weights loaded into the tensor that is there
    pool.rotations[0].copy_(rotation(3))
    assert torch.equal(written(monkeypatch, pool, 3), laid_out(rotation(3)))
    # another tensor in its place, and what it replaces gone (another may get its id)
    for seed in range(4, 12):
        pool.rotations[0] = rotation(seed).to(BF)
        assert torch.equal(written(monkeypatch, pool, 3), laid_out(rotation(seed)))
    # all of this in one buffer, which captured calls hold
    assert written(monkeypatch, pool, 3) is first
    # none, and one again
    pool.rotations[0] = None
    assert written(monkeypatch, pool, 3) is None
    pool.rotations[0] = rotation(12)
    assert torch.equal(written(monkeypatch, pool, 3), laid_out(rotation(12)))
    assert torch.equal(written(monkeypatch, pool, 4), laid_out(rotation(2)))


def test_a_pool_that_builds_its_rotation_at_each_call(monkeypatch):
    pool = MX4MLAPool(32, 1, 256, 32, device="cpu")
    seeds = iter(range(20))
    pool.latent_rotation = lambda layer_id, local=True: rotation(next(seeds))
    for seed in range(20):
        assert torch.equal(written(monkeypatch, pool), laid_out(rotation(seed)))


def test_a_rotation_without_a_version(monkeypatch):
    """Inference tensors do not count their changes: laid out at each call."""
    with torch.inference_mode():
        pool = MX4MLAPool(32, 1, 256, 32, device="cpu")
        r = pool.rotations[0] = rotation(1).to(BF)
        assert torch.equal(written(monkeypatch, pool), laid_out(rotation(1)))
        r.copy_(rotation(2))
        assert torch.equal(written(monkeypatch, pool), laid_out(rotation(2)))


@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_a_pool_made_in_inference_mode_lays_out_once(monkeypatch, dtype):
    with torch.inference_mode():
        pool = MX4MLAPool(32, 1, 256, 32, device="cpu", rotations=[rotation(1).to(dtype)])
        first = written(monkeypatch, pool)
        assert torch.equal(first, laid_out(rotation(1))) and written(monkeypatch, pool) is first
        pool.rotations[0].copy_(rotation(2))
        assert torch.equal(written(monkeypatch, pool), laid_out(rotation(2)))


def test_a_rotation_in_and_out_of_inference_mode(monkeypatch):
    """What is kept serves both, and a parameter's layout has no graph."""
    pool = MX4MLAPool(32, 1, 256, 32, device="cpu", rotations=[rotation(1)])
    with torch.inference_mode():
        first = written(monkeypatch, pool)
    pool.rotations[0].copy_(rotation(2))
    assert torch.equal(written(monkeypatch, pool), laid_out(rotation(2)))
    pool.rotations[0] = torch.nn.Parameter(rotation(3).to(BF))
    for seed in (3, 4):
        with torch.no_grad():
            pool.rotations[0].copy_(rotation(seed))
        rt = written(monkeypatch, pool)
        assert rt is first and torch.equal(rt, laid_out(rotation(seed))) and not rt.requires_grad


# ---- two host threads on one stream ----------------------------------------------------
def test_calls_of_two_threads_take_turns_in_the_pool_s_workspace(monkeypatch):
    """A call is two launches with the workspace between them: no other call's may come in between."""
    import threading
    import time

    pool = small_pool()
    inside, met = [], []

    def launch(*args):
        inside.append(1)
        met.append(len(inside))
        time.sleep(0.002)  # (as ctypes does, lets other threads run)
        inside.pop()

    monkeypatch.setattr(mx4.kernels, "mx4_attend_fwd", launch)
    monkeypatch.setattr(mx4, "attend_workspace", lambda p: torch.zeros(16, dtype=torch.uint8))
    q, o = torch.zeros(3, 16, 576, dtype=BF), torch.zeros(3, 16, 512, dtype=BF)
    ptr, idx, lens = torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.ones(3, dtype=torch.int64)
    threads = [threading.Thread(target=lambda: [mx4.attend_fwd(q, o, pool, 0, ptr, idx, lens, 0.1) for _ in range(10)])
               for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(met) == 40 and max(met) == 1
