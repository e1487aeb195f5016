"""Attention over keys and values expanded from the latent (the prefill form of MLA).

For long prompts the expanded form costs fewer operations than the absorbed one: the
latent rows (a prompt's own, or those that ``mx4.read_rows`` / ``assemble.assemble_rows``
return of a cached prefix) go through ``kv_b_proj``, and every head attends over its own
keys and values, with one rope key for all heads. The reference leaves this attention
to its serving engine.
"""

from __future__ import annotations

from . import kernels


def expanded_attend_fwd(q, kv, k_pe, o, qo_indptr, kv_indptr, max_q_len: int, sm_scale, causal: bool = True, lse=None,
                        workspace=None):
    """Attention of a ragged batch over expanded keys and values.

    ``q``: bf16 ``[T, H, nope + rope]``; ``kv``: bf16 ``[N, H, nope + value]`` (``k_nope | v``, ``kv_b_proj``'s output
    viewed by heads); ``k_pe``: bf16 ``[N, rope]`` rotated rope keys (the last columns of read-back rows will do);
    ``o``: bf16 ``[T, H, value]``. Widths (nope, rope, value) are (128, 64, 128) or (64, 32, 64).
    ``qo_indptr`` / ``kv_indptr``: int32 ``[B + 1]`` offsets of the requests' queries and key rows. With ``causal``,
    query ``i`` of ``m`` sees the key rows up to ``n - m + i`` of the request's ``n``; else all of them (a prefix in
    parts, joined by ``lse``). ``max_q_len``: the most queries of a request (later ones are left out). ``lse``: FP32
    ``[T, H]``, receives the natural log of the sum of exponentials. A query that sees nothing gets 0 (and -inf).
    ``workspace``: uint8, of ``kernels.expanded_attend_workspace_bytes`` and used by no other call at the same
    time; allocated on the current stream when not given and needed.
    """
    return kernels.expanded_attend_fwd(q, kv, k_pe, qo_indptr, kv_indptr, max_q_len, o, sm_scale, causal, lse, workspace)
