"""Rotary frequencies, and the refusals of the operators around the caches, before any launch (CPU only)."""

import ctypes
import math

import pytest
import torch

from mla_kv_quant_amd import _lib, evict, expanded, rotary
from mla_kv_quant_amd.mx4 import MX4MLAPool

P = ctypes.c_void_p(4096)
BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def refused(fn, args, word):
    assert fn(*args) == _lib.ROLAQ_ERR_INVALID
    assert word in _lib.load().rolaq_last_error().decode(), _lib.load().rolaq_last_error()


def changed(args, **by_index):
    out = list(args)
    for k, v in by_index.items():
        out[int(k[1:])] = v
    return out


# ---- rotary -----------------------------------------------------------------------------
def test_plain_and_linear_frequencies():
    f, s = rotary.frequencies(64)
    assert s == 1.0 and f[0] == 1.0 and f[16] == pytest.approx(0.01, rel=1e-14)
    g, s = rotary.frequencies(64, scaling={"rope_type": "linear", "factor": 4})
    assert s == 1.0 and all(a == b / 4 for a, b in zip(g, f))
    assert rotary.frequencies(64, scaling={"type": "default"})[0] == f


def test_yarn_frequencies():
    """Pairs that turn more than 32 times over the original length stay, those below one turn are slowed."""
    kw = {"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096}
    f, _ = rotary.frequencies(64)
    g, s = rotary.frequencies(64, scaling=kw)
    assert s == pytest.approx(0.1 * math.log(40) + 1)
    ratio = [b / a for a, b in zip(f, g)]
    for a, r in zip(f, ratio):
        turns = 4096 * a / (2 * math.pi)
        if turns > 40:
            assert r == pytest.approx(1)
        if turns < 0.7:
            assert r == pytest.approx(1 / 40)
    assert all(x >= y - 1e-15 for x, y in zip(ratio, ratio[1:]))
    # hand-computed ends of the ramp: 64 ln(4096 / (32 2 pi)) / (2 ln 10000) = 10.47, 64 ln(4096 / 2 pi) / (2 ln 10000) = 22.5
    assert ratio[10] == pytest.approx(1) and ratio[11] < 1 and ratio[22] > 1 / 40 and ratio[23] == pytest.approx(1 / 40)
    assert ratio[15] == pytest.approx(1 - 5 / 13 + 5 / 13 / 40)
    assert rotary.frequencies(64, scaling=dict(kw, mscale=0.707, mscale_all_dim=0.707))[1] == 1.0
    assert rotary.frequencies(64, scaling=dict(kw, attention_factor=1.5))[1] == 1.5


def test_longrope_frequencies():
    kw = {"type": "longrope", "factor": 4, "original_max_position_embeddings": 32768, "long_factor": [2.0] * 16,
          "short_factor": [1.0] * 16}
    f, _ = rotary.frequencies(32)
    g, s = rotary.frequencies(32, scaling=kw)
    assert s == pytest.approx(math.sqrt(1 + 2 / 15)) and all(a == 2 * b for a, b in zip(f, g))
    assert rotary.frequencies(32, scaling=dict(kw, long=False))[0] == f


@pytest.mark.parametrize("scaling,word", [
    ({"type": "dynamic"}, "unknown"), ({"type": "linear"}, "factor"), ({"type": "linear", "factor": 0}, "factor"),
    ({"type": "yarn", "factor": 4}, "original"), ({"type": "yarn", "factor": math.nan}, "factor"),
    ({"type": "longrope", "long_factor": [1.0] * 3}, "factors"), ({"type": "longrope", "long_factor": [0.0] * 32}, "factors"),
])
def test_scalings_that_are_refused(scaling, word):
    with pytest.raises(ValueError, match=word):
        rotary.frequencies(64, scaling=scaling)


def test_rotary_handles():
    r = rotary.Rotary(4, inv_freq=torch.tensor([math.pi, -math.pi / 2], dtype=torch.float64), device="cpu", scale=2.0)
    # half a turn and minus a quarter, to double's pi
    t = [v % 2 ** 64 / 2 ** 64 for v in r.turns.tolist()]
    assert t == pytest.approx([0.5, 0.75], abs=1e-15) and r.scale == 2.0
    for kw in ({"dim": 3}, {"dim": 0}, {"dim": 514}, {"dim": 4, "base": 1.0}, {"dim": 4, "scale": math.inf},
               {"dim": 4, "inv_freq": [1.0]}, {"dim": 4, "inv_freq": [1.0, math.nan]},
               {"dim": 4, "inv_freq": [1.0, 1.0], "scaling": {"type": "linear", "factor": 2}}):
        with pytest.raises(ValueError):
            rotary.Rotary(device="cpu", **kw)


def test_rotary_tensors():
    r = rotary.Rotary(32, device="cpu")
    p, q, k = torch.arange(5), torch.zeros(5, 3, 32, dtype=BF), torch.zeros(5, 32, dtype=BF)
    with pytest.raises(TypeError, match="integers"):
        rotary.apply_rotary(r, p.float(), q)
    with pytest.raises(TypeError):
        rotary.apply_rotary(r, p, q.double())
    with pytest.raises(TypeError):
        rotary.apply_rotary(r, p, q, k.float())
    with pytest.raises(TypeError):
        rotary.apply_rotary(r, p, q, q_out=q.float())
    with pytest.raises(ValueError):
        rotary.apply_rotary(r, p[:4], q)
    with pytest.raises(ValueError):
        rotary.apply_rotary(r, p, q[..., :30])
    with pytest.raises(ValueError, match="last dim"):
        rotary.apply_rotary(r, p, torch.zeros(5, 32, 3, dtype=BF).transpose(1, 2))
    with pytest.raises(ValueError):
        rotary.apply_rotary(r, p, q, q_out=q[:, :2])
    with pytest.raises(ValueError, match="without k"):
        rotary.apply_rotary(r, p, q, k_out=k)
    with pytest.raises(ValueError, match="repeat"):
        rotary.apply_rotary(r, p, q[:, :1].expand(5, 3, 32))
    fn = _lib.load().rolaq_rotary
    ok = [P, 0, P, 64, 1.0, 1, 0, P, 64, 64, P, 64, 64, 4, P, 64, 0, P, 64, 0, 1, None]
    assert fn(*ok) == _lib.ROLAQ_OK  # no tokens: nothing to do
    ok[1] = 4
    assert fn(*changed(ok, i13=0, i20=0)) == _lib.ROLAQ_OK
    refused(fn, changed(ok, i1=-1), "negative")
    refused(fn, changed(ok, i3=63), "dim")
    refused(fn, changed(ok, i3=514), "dim")
    refused(fn, changed(ok, i4=math.nan), "scale")
    refused(fn, changed(ok, i6=3), "type")
    refused(fn, changed(ok, i13=(1 << 20) + 1), "heads")
    refused(fn, changed(ok, i7=ctypes.c_void_p(4097)), "aligned")
    for i in (0, 2, 7, 10, 14, 17):
        refused(fn, changed(ok, **{f"i{i}": None}), "null")


# ---- expanded attention ---------------------------------------------------------------------
def test_expanded_tensors():
    q, kv, pe = torch.zeros(4, 2, 192, dtype=BF), torch.zeros(6, 2, 256, dtype=BF), torch.zeros(6, 64, dtype=BF)
    o, qo, ko = torch.zeros(4, 2, 128, dtype=BF), torch.tensor([0, 4], dtype=I32), torch.tensor([0, 6], dtype=I32)

    def bad(err, word=".", **kw):
        a = dict(q=q, kv=kv, k_pe=pe, o=o, qo_indptr=qo, kv_indptr=ko, max_q_len=4, sm_scale=0.1)
        a.update(kw)
        with pytest.raises(err, match=word):
            expanded.expanded_attend_fwd(**a)

    bad(TypeError, q=q.float())
    bad(TypeError, o=o.float())
    bad(TypeError, qo_indptr=qo.long())
    bad(ValueError, kv=kv[:5])
    bad(ValueError, kv=kv[:, :1])
    bad(ValueError, kv=kv[..., :192])
    bad(ValueError, o=o[:3])
    bad(ValueError, kv_indptr=ko[:1])
    bad(ValueError, lse=torch.zeros(3, 2))
    bad(TypeError, lse=torch.zeros(4, 2, dtype=torch.float64))
    bad(ValueError, "last dim", k_pe=torch.zeros(64, 6, dtype=BF).t())
    bad(TypeError, workspace=torch.zeros(10))


def test_expanded_arguments():
    lib = _lib.load()
    fn = lib.rolaq_expanded_attend_fwd
    ok = [P, 16 * 192, 192, P, 4096, 256, P, 64, P, P, 0, 6, 2, 16, 128, 64, 128, 4, 0.1, 1, P, 2048, 128, None, P, 1 << 30,
          None]
    assert fn(*ok) == _lib.ROLAQ_OK
    ok[10] = 4
    refused(fn, changed(ok, i10=-1), "negative")
    refused(fn, changed(ok, i13=0), "H must")
    refused(fn, changed(ok, i13=129), "H must")
    refused(fn, changed(ok, i14=64), "nope")
    refused(fn, changed(ok, i18=math.inf), "sm_scale")
    refused(fn, changed(ok, i10=(1 << 24) + 1), "2^24")
    refused(fn, changed(ok, i2=193), "q must")
    refused(fn, changed(ok, i5=252), "kv must")
    refused(fn, changed(ok, i7=60), "k_pe must")
    refused(fn, changed(ok, i22=120), "out must")
    refused(fn, changed(ok, i20=ctypes.c_void_p(4104)), "out must")
    refused(fn, changed(ok, i10=1 << 24, i13=128), "too large")
    refused(fn, changed(ok, i11=100000, i24=None), "workspace")
    refused(fn, changed(ok, i11=100000, i25=1024), "workspace")
    for i in (0, 3, 6, 8, 9, 20):
        refused(fn, changed(ok, **{f"i{i}": None}), "null")
    n = ctypes.c_int64(-1)
    assert lib.rolaq_expanded_attend_workspace(0, 0, 0, 1, 64, 0, ctypes.byref(n)) == 0 and n.value == 0
    refused(lib.rolaq_expanded_attend_workspace, [1, 1, 1, 1, 96, 1, ctypes.byref(n)], "invalid")
    refused(lib.rolaq_expanded_attend_workspace, [1, 1, 1, 1, 64, 1, None], "invalid")


# ---- accumulated weights and eviction --------------------------------------------------------
def test_weights_tensors():
    pool = MX4MLAPool(7, 1, 256, 32, device="cpu")
    q, lse, acc = torch.zeros(2, 4, 288, dtype=BF), torch.zeros(2, 4), torch.zeros(3, 10)
    ptr, idx, lens = torch.tensor([0, 1, 2], dtype=I32), torch.tensor([1, 2], dtype=I32), torch.tensor([1, 1])

    def bad(err, word=".", **kw):
        a = dict(q=q, lse=lse, pool=pool, layer_id=0, acc=acc, kv_indptr=ptr, kv_indices=idx, kv_lens=lens, sm_scale=0.1)
        a.update(kw)
        with pytest.raises(err, match=word):
            evict.accumulate_weights(**a)

    bad(TypeError, q=q.float())
    bad(ValueError, q=q[..., :256])
    bad(ValueError, lse=lse[:1])
    bad(TypeError, lse=lse.double())
    bad(ValueError, "contiguous", lse=torch.zeros(4, 2).t())
    bad(TypeError, acc=acc.double())
    bad(ValueError, "rows", acc=torch.zeros(10, 3).t())
    bad(ValueError, "rows", acc=acc[:1].expand(3, 10))
    bad(ValueError, kv_indptr=ptr[:2])
    bad(ValueError, kv_lens=lens[:1])
    bad(ValueError, req_pool_indices=torch.tensor([0]))


def test_weights_arguments():
    fn = _lib.load().rolaq_mx4_accumulate_weights
    ok = [P, 9216, 576, P, P, P, P, 100, P, P, P, 50, 64, P, P, 4, 0, 16, 512, 64, 4, 0.1, P, 1000, 10, 1000, 1, None]
    assert fn(*ok) == _lib.ROLAQ_OK
    ok[16] = 2
    refused(fn, changed(ok, i16=-1), "negative")
    refused(fn, changed(ok, i17=129), "H must")
    refused(fn, changed(ok, i18=384), "(D, R)")
    refused(fn, changed(ok, i23=999), "acc")
    refused(fn, changed(ok, i24=-1), "acc")
    refused(fn, changed(ok, i11=-1), "n_indices")
    refused(fn, changed(ok, i12=48), "page_size")
    refused(fn, changed(ok, i21=0.0), "sm_scale")
    refused(fn, changed(ok, i8=None, i20=2), "max_q_len")
    refused(fn, changed(ok, i1=9218), "q must")
    refused(fn, changed(ok, i15=1 << 24, i17=128), "2^29")
    for i in (0, 3, 9, 10, 13, 22):
        refused(fn, changed(ok, **{f"i{i}": None}), "null")


def test_weights_workspace_arguments():
    lib = _lib.load()
    fn = lib.rolaq_mx4_accumulate_weights_workspace
    n = ctypes.c_int64(7)
    ok = [100, 2, 128, 512, 40, 16, 50, ctypes.byref(n)]
    assert fn(*ok) == _lib.ROLAQ_OK
    assert fn(*changed(ok, i6=0)) == _lib.ROLAQ_OK and n.value == 0
    for i, v in ((0, -1), (1, -1), (2, 0), (2, 129), (3, 384), (4, -1), (5, 48), (5, 0), (6, -1), (7, None)):
        refused(fn, changed(ok, **{f"i{i}": v}), "invalid sizes")


def test_evict_tensors():
    acc, ptr = torch.zeros(3, 10), torch.tensor([0, 1, 2], dtype=I32)
    idx, lens = torch.tensor([1, 2], dtype=I32), torch.tensor([1, 1])

    def bad(err, word=".", **kw):
        a = dict(acc=acc, kv_indptr=ptr, kv_indices=idx, kv_lens=lens, budget=4, sink=1, recent=1)
        a.update(kw)
        with pytest.raises(err, match=word):
            evict.evict(**a)

    bad(ValueError, "budget", budget=0, sink=0, recent=0)
    bad(ValueError, "budget", sink=3, recent=2)
    bad(ValueError, "budget", sink=-1)
    bad(TypeError, acc=acc.double())
    bad(ValueError, "shape", acc_out=torch.zeros(3, 9))
    bad(ValueError, kept=torch.zeros(2, 5, dtype=I32))
    bad(TypeError, kept=torch.zeros(2, 4, dtype=I64))
    bad(ValueError, kept=torch.zeros(3, 4, dtype=I32))
    bad(ValueError, kept_lens=torch.zeros(1, dtype=I64))
    bad(TypeError, freed=torch.zeros(4, dtype=I64))
    bad(ValueError, req_pool_indices=torch.tensor([0]))


def test_evict_arguments():
    lib = _lib.load()
    fn = lib.rolaq_evict
    ok = [P, 1000, 10, 1000, P, 1000, P, P, P, 50, 64, P, 0, 1000, 64, 4, 16, P, P, P, 100, None, 0, None]
    assert fn(*ok) == _lib.ROLAQ_OK
    ok[12] = 2
    refused(fn, changed(ok, i12=-1), "invalid B")
    refused(fn, changed(ok, i1=999), "acc")
    refused(fn, changed(ok, i5=999), "acc")
    refused(fn, changed(ok, i14=0), "budget")
    refused(fn, changed(ok, i15=60), "budget")
    refused(fn, changed(ok, i10=0), "page_size")
    refused(fn, changed(ok, i13=1001), "max_kv_len")
    refused(fn, changed(ok, i9=-1), "n_indices")
    refused(fn, changed(ok, i1=20000, i3=20000, i5=20000, i13=20000), "workspace")
    refused(fn, changed(ok, i12=1 << 22), "too large")
    for i in (0, 4, 7, 8, 11, 17, 18, 19):
        refused(fn, changed(ok, **{f"i{i}": None}), "null")
    n = ctypes.c_int64(-1)
    assert lib.rolaq_evict_workspace(4, 16384, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.rolaq_evict_workspace(4, 16385, ctypes.byref(n)) == 0 and n.value > 0
    refused(lib.rolaq_evict_workspace, [-1, 5, ctypes.byref(n)], "invalid")
