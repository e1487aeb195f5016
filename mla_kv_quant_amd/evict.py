"""Eviction from a latent cache by accumulated attention weight.

A cache that only grows is cut back to a budget for each request: the first positions, the
last ones, and those that queries have attended to most stay.

    mx4.attend_fwd(q, o, pool, layer, ..., lse=lse)
    accumulate_weights(q, lse, pool, layer, acc, ...)        # a decode step's, or a prompt's last queries'
    kept, kept_lens, freed = evict(acc, kv_indptr, kv_indices, kv_lens, budget=2048)

``kept`` is then the request's page list, with pages of one slot: rope keys are stored
rotated, so rows stay where and as they are. ``acc`` has a row for each request (by request
index, as the window rows have) and a column for each cached position. Weights come from
the 4-bit cache; the INT2 cache finds its window rows by position, so its
positions cannot be renumbered. The reference's caches only grow.
"""

from __future__ import annotations

import torch

from . import kernels
from .writer import _as_int64


def accumulate_weights(q, lse, pool, layer_id, acc, kv_indptr, kv_indices, kv_lens, sm_scale, qo_indptr=None,
                       max_q_len: int = 1, page_size: int = 1, req_pool_indices=None, add: bool = True, workspace=None):
    """Add to ``acc`` the attention weight that each cached position gets from ``q``, over all queries and heads.

    ``q``, the index lists, ``kv_lens``, ``qo_indptr`` and ``max_q_len`` as for ``mx4.attend_fwd``, and ``lse`` as it
    returned for these queries (rows with -inf count for nothing, whatever ``q`` holds there: a batch's padding).
    ``acc``: FP32 ``[rows, columns]``; position ``t`` of request ``b`` is column ``t`` of row ``req_pool_indices[b]`` (row
    ``b`` if not given). Rows of one call must differ; a request whose row does not exist is left out, as are
    positions past the columns. With ``add=False`` the sums
    take the place of what the cached positions' columns held. ``workspace``: uint8, of
    ``kernels.accumulate_weights_workspace_bytes`` and used by no other call at the same time; allocated on the
    current stream when not given and needed. Returns ``acc``.
    """
    li = layer_id - pool.start_layer
    req = None if req_pool_indices is None else _as_int64(req_pool_indices)
    return kernels.mx4_accumulate_weights(q, lse, pool.c_codes[li], pool.c_scales[li], pool.rope_buf[li], qo_indptr,
                                          kv_indptr, kv_indices, _as_int64(kv_lens), max_q_len, acc, sm_scale, page_size,
                                          req, add, workspace)


def evict(acc, kv_indptr, kv_indices, kv_lens, budget: int, sink: int = 4, recent: int = 16, page_size: int = 1,
          req_pool_indices=None, max_kv_len: int | None = None, acc_out=None, kept=None, kept_lens=None, freed=None,
          workspace=None):
    """Choose the positions that stay of every request: ``(kept, kept_lens, freed)``.

    A request of ``budget`` positions or fewer keeps all of them. Of a longer one stay the first ``sink``, the last
    ``recent`` and, of the others, those of largest ``acc`` (the earlier of equal ones; NaN counts as the largest).
    ``kept``: int32 ``[B, budget]`` slots in order of position, of which ``kept_lens`` (int64 ``[B]``) are set:
    a page list of pages of one slot, with ``b * budget`` as its offsets. ``freed``: int32, the other slots, request
    after request: ``n - kept_lens`` of each, ``n`` being its length, cut as below. Later entries of one that is given are
    left as they were (and slots past its end left out), of one that is allocated here they are -1.
    ``acc_out`` (``acc`` itself if not given) receives the weights of what stays in its new columns, and 0 in the
    others up to the old length. ``max_kv_len``: the most positions of a request (``acc``'s columns if not given, and at
    most those). A longer request is cut there, as one that is longer than its page list reaches is at that: the
    positions past it, its newest ones, are neither kept nor freed, and ``recent`` counts from the cut. Lists,
    lengths and rows as for
    :func:`accumulate_weights`. Outputs that are not given are allocated; none may overlap another or an input (``kept_lens``
    is not ``kv_lens``, ``kept`` no part of ``kv_indices``), ``acc_out`` on ``acc`` itself apart. ``workspace``: uint8, of
    ``kernels.evict_workspace_bytes`` for this ``max_kv_len``, used by no other call at the same time; allocated on the
    current stream when not given and needed. It follows from ``max_kv_len``, not from the lengths, as do the
    launches: one up to 16384, else four. Where ``acc`` has more columns than the batch is long, state it.
    """
    dev = acc.device
    kv_lens = _as_int64(kv_lens)
    B = kv_lens.shape[0] if kept is None else kept.shape[0]
    if budget < 1 or sink < 0 or recent < 0 or sink + recent > budget:
        raise ValueError(f"budget must be positive and hold sink + recent, got {budget}, {sink} + {recent}")
    if kept is None:
        kept = torch.empty(B, budget, dtype=torch.int32, device=dev)
    if kept_lens is None:
        kept_lens = torch.empty(B, dtype=torch.int64, device=dev)
    if freed is None:
        freed = torch.full((kv_indices.shape[0] * page_size,), -1, dtype=torch.int32, device=dev)
    req = None if req_pool_indices is None else _as_int64(req_pool_indices)
    kernels.evict(acc, kv_indptr, kv_indices, kv_lens, budget, sink, recent, page_size, req,
                  acc.shape[1] if max_kv_len is None else min(max_kv_len, acc.shape[1]), acc if acc_out is None else acc_out,
                  kept, kept_lens, freed, workspace)
    return kept, kept_lens, freed
