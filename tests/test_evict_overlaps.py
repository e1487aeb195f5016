"""Eviction refuses outputs that lie on its inputs or on each other: a block reads other requests' lengths and lists while
those requests' blocks write. Made-up addresses, refused before any launch (CPU only)."""

import ctypes

import pytest

from mla_kv_quant_amd import _lib

M = 1 << 24  # apart from each other by default
NAMES = ["acc", "acc_out", "req_idx", "kv_indptr", "kv_indices", "kv_lens", "kept", "kept_lens", "freed", "workspace"]
# 4 requests, acc of 6 rows of 20000 columns, 9000 pages of 16, 64 kept, room for 1000 freed
BYTES = {"acc": 480000, "acc_out": 480000, "req_idx": 32, "kv_indptr": 20, "kv_indices": 36000, "kv_lens": 32, "kept": 1024,
         "kept_lens": 32, "freed": 4000}
OUTPUTS = ["acc_out", "kept", "kept_lens", "freed", "workspace"]


def call(stride=20000, out_stride=20000, most=20000, **places):
    at = {n: M * (i + 1) for i, n in enumerate(NAMES)}
    at.update(places)
    p = {n: ctypes.c_void_p(v) for n, v in at.items()}
    lib, n = _lib.load(), ctypes.c_int64(0)
    assert lib.rolaq_evict_workspace(4, most, ctypes.byref(n)) == _lib.ROLAQ_OK
    rc = lib.rolaq_evict(p["acc"], stride, 6, 20000, p["acc_out"], out_stride, p["req_idx"], p["kv_indptr"], p["kv_indices"],
                         9000, 16, p["kv_lens"], 4, most, 64, 4, 16, p["kept"], p["kept_lens"], p["freed"], 1000,
                         p["workspace"], n.value, None)
    return rc, lib.rolaq_last_error().decode()


def refused(a, b, **kw):
    rc, text = call(**kw)
    assert rc == _lib.ROLAQ_ERR_INVALID and "overlap" in text and a in text and b in text, (rc, text)


@pytest.mark.parametrize("out", OUTPUTS)
@pytest.mark.parametrize("other", [n for n in NAMES if n != "workspace"])
def test_outputs_on_inputs_and_on_each_other(out, other):
    if out == other:
        return
    place = M * (NAMES.index(other) + 1)
    if (out, other) != ("acc_out", "acc"):  # (that one is eviction in place)
        refused(out, other, **{out: place})
    # by their ends alone
    last = place + BYTES[other]
    refused(out, other, **{out: (last - 1) // 16 * 16 if out == "workspace" else last - (8 if out == "kept_lens" else 4)})


def test_lengths_in_place():
    refused("kept_lens", "kv_lens", kept_lens=M * 6)
    refused("kept_lens", "kv_lens", kept_lens=M * 6, most=300)  # (without a workspace, one block a request)


def test_rows_of_weights_that_share_columns():
    row = 4 * 50000  # parts of the columns of wider rows: 0 .. 19999 and others
    kw = dict(stride=50000, out_stride=50000)
    refused("acc_out", "acc", acc_out=M + 4 * 19999, **kw)
    refused("acc_out", "acc", acc_out=M + 4 * 30001, **kw)  # its rows end in acc's next ones
    refused("acc_out", "acc", acc_out=M + row * 5 + 4 * 19999, **kw)
    refused("acc_out", "acc", acc_out=M + row, **kw)
    refused("acc_out", "acc", acc=M * 20 + row * 3 + 4 * 10, acc_out=M * 20, **kw)
    refused("acc_out", "acc", acc_out=M, stride=20000, out_stride=20001)  # in place with another stride
    refused("acc_out", "acc", acc_out=M + 4 * 20000, stride=50000, out_stride=45000)
    refused("kept", "acc", kept=M + row * 2 + 4 * 19999, **kw)
    refused("freed", "acc", freed=M + row * 4 + 4 * 49001, **kw)
