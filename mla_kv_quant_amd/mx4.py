"""The 4-bit latent cache (MX4): pool, writer, read-back and attention.

For layers, or models, that do not stand INT2: a cached latent row is D 4-bit
floats (E2M1) with one power-of-two scale for 32 of them, beside the bf16 rope
key -- 400 bytes a token and layer at (512, 64), 200 at (256, 32), against
1152 and 576 in bf16 -- with no BF16 window and no quantizer parameters. The
matrix cores of gfx950 take the codes as they are stored. Rows may be rotated
by a layer's ``R_eff``, as in the INT2 cache; queries and outputs are then in the
rotated frame (``artifacts.fold_read_rotation``).

Every call launches on the current stream of its tensors' device, allocates
nothing but an output that was not given (and the attention's workspace, once
for a stream) and makes no synchronisation, so it can be captured in a HIP graph;
the one exception is a write that finds its layer's rotation new or changed
(``write_rows``). The reference has no 4-bit cache.
"""

from __future__ import annotations

import threading

import torch

from . import kernels
from .writer import SUPPORTED_DIMS, _as_int64, _rows

# A call of the attention is two launches, the first of which leaves in the workspace what the
# second joins: calls of several host threads on one stream must not get in between.
_turns = threading.Lock()


class MX4MLAPool:
    """Per-layer 4-bit cache buffers (layouts: ``include/rolaq_mla.h``).

    ``size`` token slots besides slot 0, which is for graph padding.
    ``rotations``: per-layer ``[D, D]`` rotations (or None), held in bf16
    (``R_eff = fp32(bf16(R))``). The functions of this module take any object
    with these attributes.
    """

    def __init__(self, size: int, layer_num: int, kv_lora_rank: int = 512, qk_rope_head_dim: int = 64, device="cuda",
                 rotations=None, start_layer: int = 0):
        if (kv_lora_rank, qk_rope_head_dim) not in SUPPORTED_DIMS:
            raise ValueError(f"(kv_lora_rank, qk_rope_head_dim) must be one of {sorted(SUPPORTED_DIMS)}")
        self.size = int(size)
        self.layer_num = int(layer_num)
        self.start_layer = int(start_layer)
        self.kv_lora_rank = D = int(kv_lora_rank)
        self.qk_rope_head_dim = int(qk_rope_head_dim)
        self.device = torch.device(device)
        slots, dev = self.size + 1, self.device

        def buf(width, dtype):
            return [torch.zeros(slots, width, dtype=dtype, device=dev) for _ in range(self.layer_num)]

        self.c_codes = buf(D // 2, torch.uint8)
        self.c_scales = buf(D // kernels.MX4_BLOCK, torch.uint8)
        self.rope_buf = buf(self.qk_rope_head_dim, torch.bfloat16)
        rotations = rotations or [None] * self.layer_num
        with torch.inference_mode(False):  # (a tensor of that mode does not count its changes: copied)
            held = [None if r is None else r.to(device=dev, dtype=torch.bfloat16) for r in rotations]
            self.rotations = [r.clone() if r is not None and r.is_inference() else r for r in held]

    def latent_rotation(self, layer_id: int, local: bool = True):
        return self.rotations[layer_id - self.start_layer if local else layer_id]

    def get_kv_size_bytes(self) -> int:
        D = self.kv_lora_rank
        return (self.size + 1) * self.layer_num * (D // 2 + D // kernels.MX4_BLOCK + 2 * self.qk_rope_head_dim)


def attend_workspace(pool) -> torch.Tensor:
    """The attention's workspace of ``pool`` for calls on the current stream (68 MB at width 512).

    One for each stream, allocated by its first call and used by every layer and batch
    on it: calls of two streams may overlap, and ``attend_fwd`` keeps those of several
    host threads on one stream apart. During a capture it is a new tensor
    of the graph's memory, so graphs that do not share their memory may be replayed
    side by side, and beside other calls.
    """
    like = pool.c_codes[0]
    if like.get_device() != torch.cuda.current_device():
        with torch.cuda.device(like.device):
            return attend_workspace(pool)
    kept = getattr(pool, "_mx4_workspaces", None)
    if kept is None:
        kept = pool._mx4_workspaces = {}
    capturing = torch.cuda.is_current_stream_capturing()
    stream = kernels._stream(like)
    ws = None if capturing else kept.get(stream)
    if ws is None:
        n = kernels.mx4_attend_workspace_bytes(pool.kv_lora_rank, like.device)
        ws = torch.empty(n, dtype=torch.uint8, device=like.device)
        if not capturing:
            kept[stream] = ws
    return ws


def _rotation_t(pool, layer_id):
    """bf16 R_eff^T of a layer as the writer takes it (None: no rotation).

    Kept for the pool with the tensor that it was laid out from, and laid out again,
    in the same buffer, when that is another tensor or torch has counted a change of
    it. Any stream may use what is kept: the layout waits for all that may still
    read the buffer, and is complete when this returns. During a capture, where nothing can be
    waited for, and for tensors that count no changes it is part of the call instead.
    """
    r = pool.latent_rotation(layer_id, local=True)
    if r is None:
        return None
    kept = getattr(pool, "_mx4_rotations_t", None)
    if kept is None:
        kept = pool._mx4_rotations_t = {}
    entry = kept.get(layer_id)
    try:
        version = r._version
    except RuntimeError:  # an inference tensor
        version = None
    if entry is not None and entry[0] is r and entry[1] == version and version is not None:
        return entry[2]
    if r.is_cuda:
        with torch.cuda.device(r.device):
            if version is None or torch.cuda.is_current_stream_capturing():
                return r.to(torch.bfloat16).t().contiguous()
            torch.cuda.synchronize()
            rt = _lay_out(r, entry)
            torch.cuda.current_stream().synchronize()
    elif version is None:
        return r.to(torch.bfloat16).t().contiguous()
    else:
        rt = _lay_out(r, entry)
    kept[layer_id] = (r, version, rt)
    return rt


def _lay_out(r, entry):
    with torch.inference_mode(False), torch.no_grad():  # (kept for calls of either mode)
        t = r.to(torch.bfloat16).t()
        if entry is None or entry[2].device != t.device or entry[2].shape != t.shape:
            return t.clone(memory_format=torch.contiguous_format)
        return entry[2].copy_(t)


def write_rows(pool, layer_id, loc, c_kv, k_pe) -> None:
    """Store rows of layer ``layer_id`` at slots ``loc``: a decode step's or a prefill chunk's.

    ``c_kv``: bf16 latents ``[n, D]`` (after ``kv_a_layernorm``; any shape with
    ``n * D`` elements), ``k_pe``: bf16 rope keys. One launch rotates (on a
    layer with a rotation), quantizes, packs and stores. Slots of one call must
    differ, except for the padding slot; one outside the cache is skipped.

    The kernel reads ``R_eff^T``, which the first write of a layer lays out and the pool
    keeps. The first write after the rotation has changed (another tensor, or the
    same one changed by a torch operation on it; a change through ``.data`` is not
    seen) lays it out again and, like the first, waits for the device; calls
    captured before follow from there on. A write that is captured before its layer has been laid
    out does it in the graph at each replay.
    """
    li = layer_id - pool.start_layer
    rt = _rotation_t(pool, layer_id)
    kernels.mx4_write_rows(_rows(c_kv, pool.kv_lora_rank), _rows(k_pe, pool.qk_rope_head_dim), rt, _as_int64(loc),
                           pool.c_codes[li], pool.c_scales[li], pool.rope_buf[li])


def read_rows(pool, layer_id, slots, out=None, unrotate: bool = True):
    """Rows at ``slots`` of layer ``layer_id``: bf16 ``[n, D + R]`` (latent | rope).

    With ``unrotate``, the latent of a rotated layer is multiplied back by
    ``R_eff^T`` (FP32 sums, one rounding); else it is returned as it is stored,
    exactly. A slot outside the cache reads as NaN.
    """
    li = layer_id - pool.start_layer
    s = _as_int64(slots)
    if out is None:
        out = torch.empty(s.shape[0], pool.kv_lora_rank + pool.qk_rope_head_dim, dtype=torch.bfloat16,
                          device=pool.c_codes[li].device)
    rot = pool.latent_rotation(layer_id, local=True) if unrotate else None
    if rot is not None and not (rot.dtype == torch.bfloat16 and rot.is_contiguous()):
        rot = rot.to(torch.bfloat16).contiguous()
    return kernels.mx4_read_rows(s, pool.c_codes[li], pool.c_scales[li], pool.rope_buf[li], rot, out)


def attend_fwd(q, o, pool, layer_id, kv_indptr, kv_indices, kv_lens, sm_scale, qo_indptr=None, max_q_len: int = 1,
               page_size: int = 1, lse=None, workspace=None):
    """Absorbed MLA attention over layer ``layer_id`` of ``pool``: decode, token verification, chunked prefill.

    ``q``: bf16 ``[T, H, D + R]`` (absorbed latent query | rope query), ``o``: bf16
    ``[T, H, D]``. ``kv_indptr``/``kv_indices``: int32 page (or token) lists;
    ``kv_lens``: ``[B]`` cached positions, those of the queries' own rows (written
    before) included. ``qo_indptr``: int32 ``[B + 1]`` query offsets, None for
    one query each; query ``i`` of ``n`` sees the positions up to
    ``kv_lens[b] - n + i``. ``max_q_len``: the most queries of a request (later
    ones are left out). ``lse``: FP32 ``[T, H]``, receives the natural log of the
    sum of exponentials. A query that sees nothing gets 0 (and -inf).
    ``workspace``: a tensor of ``attend_workspace``'s size that no call uses at the same
    time; that function's if not given.
    """
    li = layer_id - pool.start_layer
    args = (q, pool.c_codes[li], pool.c_scales[li], pool.rope_buf[li], qo_indptr, kv_indptr, kv_indices,
            _as_int64(kv_lens), max_q_len, o, sm_scale)
    if workspace is not None:
        return kernels.mx4_attend_fwd(*args, workspace, page_size, lse)
    with _turns:
        return kernels.mx4_attend_fwd(*args, attend_workspace(pool), page_size, lse)
