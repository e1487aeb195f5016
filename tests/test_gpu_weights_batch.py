"""Accumulated weights through the C entry without a workspace: a request's sums are the same, bit for bit, alone and
in a batch, whatever share of the blocks it gets and whichever of the two kernels (rows kept in LDS, rows streamed) the
batch's longest request asks for.
"""

import pytest
import torch

from mla_kv_quant_amd import _lib
from tests.test_gpu_mx4 import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain(b, lse, max_q_len, request=None):
    """Weights of all requests, or of one by itself, in one part."""
    q, fn = b.q.to(DEV), _lib.load().rolaq_mx4_accumulate_weights
    first, count = (0, len(b.lens)) if request is None else (request, 1)
    qo, ptr, lens = (t[first:].contiguous() for t in (b.qo, b.kv_indptr, b.kv_lens))
    acc = torch.zeros(count, max(b.lens), device=DEV)
    codes, scales, rope = b.pool.c_codes[0], b.pool.c_scales[0], b.pool.rope_buf[0]
    _lib.check(fn(q.data_ptr(), q.stride(0), q.stride(1), lse.data_ptr(), codes.data_ptr(), scales.data_ptr(), rope.data_ptr(),
                  codes.shape[0], qo.data_ptr(), ptr.data_ptr(), b.kv_indices.data_ptr(), b.kv_indices.shape[0], b.page,
                  lens.data_ptr(), None, b.T, count, b.H, b.D, b.R, max_q_len, b.sm, acc.data_ptr(), acc.stride(0),
                  acc.shape[0], acc.shape[1], 0, torch.cuda.current_stream().cuda_stream))
    return acc


@pytest.mark.parametrize("D,H,lens,qlens", [
    (512, 16, [900, 333, 64, 5000], [9, 1, 20, 6]), (256, 40, [900, 333, 64, 5000], [9, 1, 20, 6]),
    (256, 16, [900, 333, 64, 5000], [4, 1, 20, 3]), (512, 16, [900, 333, 64, 5000], [4, 1, 20, 3]),
    (512, 128, [500, 17, 300], [3, 1, 17]), (256, 3, [700, 1000, 2500, 41, 90], [16, 21, 22, 33, 60]),
])
def test_a_request_alone_and_in_a_batch(D, H, lens, qlens):
    b = Batch(D, H, lens, qlens, 16, seed=8)
    lse = torch.full((b.T, H), 2.0, device=DEV)
    together = plain(b, lse, max(qlens))
    for i, n in enumerate(lens):
        assert together[i, :n].min() >= 0 and together[i, :n].max() > 0
        assert torch.equal(plain(b, lse, qlens[i], i)[0, :n], together[i, :n]), i


@pytest.mark.parametrize("D", [512, 256])
@pytest.mark.parametrize("H,lens,qlens,most", [(16, [500, 90], [9, 3], 4), (40, [300, 700, 64], [20, 5, 64], 7)])
def test_queries_past_the_most_of_a_request_are_left_out(D, H, lens, qlens, most):
    """Tolerance: a score is an FP32 sum of D + R exact products, off by ds = (D + R) 2^-24 sm sum |q k|; scale, difference
    and exponential add 2^-22 of the exponent's size and 2^-22; the sum of n weights n 2^-24."""
    b = Batch(D, H, lens, qlens, 16, seed=3)
    lse = torch.full((b.T, H), 2.0, device=DEV)
    got = plain(b, lse, most).double().cpu()
    t = 0
    for i, (n, m) in enumerate(zip(lens, qlens)):
        r = min(m, most)
        q, k = b.q[t:t + r].double(), torch.cat((b.x[i], b.pe[i].double()), -1)
        seen = torch.arange(n) <= n - m + torch.arange(r)[:, None, None]
        e = q @ k.t() * b.sm - 2.0
        w = torch.where(seen, torch.exp(e), 0.0)
        off = (D + b.R) * 2.0 ** -24 * b.sm * (q.abs() @ k.abs().t()) + 2.0 ** -22 * (e.abs() + 1) + r * H * 2.0 ** -24
        assert ((got[i, :n] - w.sum((0, 1))).abs() <= (w * off).sum((0, 1)) + 1e-30).all(), i
        t += m
