"""The 4-bit latent cache: its writer, its read-back and the attention over it.

A cached row holds the latent (``D`` values) as 4-bit floats (E2M1: 0, 0.5, 1,
1.5, 2, 3, 4, 6 and their negatives) with one power-of-two scale for every 32 of
them (a byte ``s`` stands for ``2^(s - 127)``, 255 for NaN), and the rope key
(``R`` values) in bf16. Three operators work on it:

* ``write``: rotate the latent rows by the layer's ``R_eff`` (or not, on a layer
  without a rotation), quantise, store at the rows' slots, and read the same
  slots back as bf16 ``[latent | rope]`` rows -- what a prefill that continues
  with dequantized rows does, and the only form in which 4-bit rows can be
  looked at;
* ``read``: cached rows as bf16, the latent rotated back to the model's frame
  where the layer has a rotation;
* ``attend``: absorbed multi-head latent attention over the cache, for decode
  (one query for each request), for verifying a few drafted tokens, and for
  chunked prefill whose own rows are in the cache already: query ``i`` of
  ``n`` sees the cached positions up to ``length - n + i``.

Widths (D, R) are (512, 64) and (256, 32). Inputs are synthetic, with the
distributions that the path meets: latent rows N(0, 1) with 1 % of the channels
x8 (the norm weight's outliers), orthogonal rotations, queries that give logits
of standard deviation about 2, pages in shuffled order.
"""

import math
import random
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LOWEST, HIGHEST, NAN = 63, 159, 255  # scale bytes: 2^-64 .. 2^32, and a block that is not finite


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a small decode batch writes its new rows: the smallest call of the path
        {"name": "write_b8", "op": "write", "D": 512, "batch": 8, "lo": 1, "hi": 1, "rotate": True, "mix": 1},
        # prefill write of a large chunked batch: 64 sequences x 2048 tokens
        {"name": "write_64x2048", "op": "write", "D": 512, "batch": 64, "lo": 2048, "hi": 2048, "rotate": True,
         "mix": 2},
        # ragged prompts on a layer without a rotation, small width
        {"name": "write_ragged_256_plain", "op": "write", "D": 256, "batch": 9, "lo": 200, "hi": 3000, "rotate": False,
         "mix": 3},
        # cached rows back in the model's frame for an MHA prefill over a cached prefix
        {"name": "read_16x4096", "op": "read", "D": 512, "batch": 16, "lo": 4096, "hi": 4096, "rotate": True, "mix": 4},
        # rows of a few ragged sequences as they are stored, small width
        {"name": "read_ragged_256_stored", "op": "read", "D": 256, "batch": 5, "lo": 100, "hi": 4001, "rotate": False,
         "mix": 5},
        # one request, token-level index lists: interactive decoding
        {"name": "decode_b1_3001", "op": "attend", "D": 512, "heads": 16, "batch": 1, "lo": 3001, "hi": 3001,
         "q_lo": 1, "q_hi": 1, "page": 1, "mix": 6},
        # the headline decode: batch 32 x 16384
        {"name": "decode_b32_16k", "op": "attend", "D": 512, "heads": 16, "batch": 32, "lo": 16384, "hi": 16384,
         "q_lo": 1, "q_hi": 1, "page": 64, "mix": 7},
        # a ragged batch at 128 heads
        {"name": "decode_b24_ragged_128h", "op": "attend", "D": 512, "heads": 128, "batch": 24, "lo": 2048, "hi": 12288,
         "q_lo": 1, "q_hi": 1, "page": 64, "mix": 8},
        # the small-width shape with 40 heads, batch 64 x 16384
        {"name": "decode_b64_16k_40h_256", "op": "attend", "D": 256, "heads": 40, "batch": 64, "lo": 16384, "hi": 16384,
         "q_lo": 1, "q_hi": 1, "page": 64, "mix": 9},
        # up to four drafted tokens verified for each request of a ragged batch
        {"name": "verify_b16_ragged", "op": "attend", "D": 512, "heads": 16, "batch": 16, "lo": 1024, "hi": 16384,
         "q_lo": 2, "q_hi": 4, "page": 64, "mix": 10},
        # chunked prefill over long prefixes, small width, 40 heads: the largest call
        {"name": "prefill_4x2048_14336_256", "op": "attend", "D": 256, "heads": 40, "batch": 4, "lo": 16384, "hi": 16384,
         "q_lo": 2048, "q_hi": 2048, "page": 64, "mix": 11},
        # a mixed prefill batch: ragged chunks over ragged prefixes, large width
        {"name": "prefill_ragged_512", "op": "attend", "D": 512, "heads": 16, "batch": 6, "lo": 2000, "hi": 9500,
         "q_lo": 100, "q_hi": 1500, "page": 64, "mix": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: rows, batch, lengths, heads, page size and width vary."""
    op = rng.choice(["write", "write", "read", "decode", "decode", "decode", "verify", "prefill"])
    D = rng.choice([512, 256])
    c = {"op": op, "D": D, "mix": rng.randrange(1 << 20)}
    if op in ("write", "read"):
        n = _log(rng, 1, 131072)  # rows in all
        batch = min(_log(rng, 1, 64), n)
        hi = max(1, n // batch)
        c.update(batch=batch, lo=max(1, int(hi * rng.uniform(0.2, 1.0))), hi=hi, rotate=rng.random() < 0.6)
        return c
    heads = rng.choice([16, 16, 8, 24, 32, 64, 128, 1, 20] if D == 512 else [40, 40, 16, 20, 24, 48, 8])
    c.update(op="attend", heads=heads, page=rng.choice([64, 64, 32, 16, 1]))
    if op == "prefill":
        batch = _log(rng, 1, 12)
        q_hi, hi = _log(rng, 8, 2048), _log(rng, 64, 16384)
        pairs = 1.2e9 / (heads * D / 256)  # below the largest listed call
        if batch * q_hi * (hi + q_hi) > pairs:
            q_hi = max(8, int(pairs / (batch * (hi + q_hi))))
        c.update(batch=batch, q_lo=max(1, int(q_hi * rng.uniform(0.2, 1.0))), q_hi=q_hi,
                 lo=q_hi + int(hi * rng.uniform(0.0, 1.0)), hi=q_hi + hi)
        return c
    n = _log(rng, 200, (1 << 20) if heads < 64 else (1 << 18))  # cached tokens in all
    batch = min(_log(rng, 1, 160), max(1, n // 20))
    hi = min(max(20, n // batch), 65536)
    q_hi = rng.randint(2, 8) if op == "verify" else 1
    c.update(batch=batch, lo=max(q_hi, int(hi * rng.uniform(0.1, 1.0))), hi=max(q_hi, hi), q_lo=1, q_hi=q_hi)
    return c


# ---------------------------------------------------------------------------
# sizes that follow from a case alone
# ---------------------------------------------------------------------------
def _lengths(case, lo="lo", hi="hi", salt=0):
    r = random.Random("%s %s" % (case["mix"], salt))
    return [r.randint(case[lo], case[hi]) for _ in range(case["batch"])]


def work(case):
    """Bytes and operations that one pass cannot do without."""
    D, R = case["D"], case["D"] // 8
    row = D // 2 + D // 32 + 2 * R  # a cached row
    lens = _lengths(case)
    n = sum(lens)
    if case["op"] == "attend":
        H, chunks = case["heads"], _lengths(case, "q_lo", "q_hi", 1)
        T = sum(chunks)
        pairs = sum(q * (m - q) + q * (q + 1) // 2 for m, q in zip(lens, chunks))
        return {"bytes": float(n * row + T * H * (2 * D + R) * 2 + 4 * (n // case["page"]) + 16 * case["batch"]),
                "flops": 2.0 * H * (2 * D + R) * pairs}
    b = n * (8 + row + 2 * (D + R)) + (2 * D * D if case["rotate"] else 0)
    f = 2.0 * n * D * D if case["rotate"] else 2.0 * n * D
    if case["op"] == "write":
        b += n * 2 * (D + R)
        f *= 2
    return {"bytes": float(b), "flops": f}


# ---------------------------------------------------------------------------
# inputs (plain torch, from the seed alone)
# ---------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)
    return g


def _normal(shape, g, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def _latents(n, D, g):
    x = torch.randn(n, D, generator=g, device=DEV)
    x[:, torch.randperm(D, generator=g, device=DEV)[:max(1, D // 100)]] *= 8.0
    return x.to(torch.bfloat16)


def _rotation(D, seed):
    g = torch.Generator()
    g.manual_seed((int(seed) * 7919 + 11) & 0x7FFFFFFF)
    q, r = torch.linalg.qr(torch.randn(D, D, generator=g, dtype=torch.float64))
    return (q * torch.sign(torch.diagonal(r))).to(DEV, torch.bfloat16).contiguous()


def _pool(slots, D, R, rotation):
    """One layer's cache, with the attributes that the package's entry points read of a pool."""
    p = SimpleNamespace(kv_lora_rank=D, qk_rope_head_dim=R, start_layer=0, rotation=rotation,
                        c_codes=[torch.zeros(slots, D // 2, dtype=torch.uint8, device=DEV)],
                        c_scales=[torch.full((slots, D // 32), LOWEST, dtype=torch.uint8, device=DEV)],
                        rope_buf=[torch.zeros(slots, R, dtype=torch.bfloat16, device=DEV)])
    p.latent_rotation = lambda layer_id, local=True: rotation
    return p


def prepare(case, seed):
    D, R = case["D"], case["D"] // 8
    lens = _lengths(case)
    n = sum(lens)
    g = _gen(seed, 1)
    page = case.get("page", 64)
    pages = [-(-m // page) for m in lens]
    # slots: every request's pages, shuffled over the pool; page 0 is the padding page
    order = torch.randperm(sum(pages), generator=g, device=DEV) + 1
    pool = _pool((sum(pages) + 1) * page, D, R, _rotation(D, seed) if case.get("rotate") else None)
    st = {"case": case, "pool": pool, "page": page, "max_len": max(lens)}
    starts = torch.tensor([0] + [sum(pages[:i + 1]) for i in range(len(pages))], device=DEV)
    row_page = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(lens, device=DEV))
    first = torch.tensor([0] + [sum(lens[:i + 1]) for i in range(len(lens) - 1)], device=DEV)
    pos = torch.arange(n, device=DEV) - first[row_page]
    slots = order[starts[row_page] + pos // page] * page + pos % page
    if case["op"] != "write":  # a cache that holds rows
        pool.c_codes[0][slots], pool.c_scales[0][slots] = _encode(_latents(n, D, g).float())
        pool.rope_buf[0][slots] = _normal((n, R), g)
    if case["op"] == "write":
        st.update(latent=_latents(n, D, g), k_pe=_normal((n, R), g), slots=slots)
    elif case["op"] == "read":
        st.update(slots=slots[torch.randperm(n, generator=g, device=DEV)])
    else:
        chunks = _lengths(case, "q_lo", "q_hi", 1)
        H, T = case["heads"], sum(chunks)
        st["sm_scale"] = (1.5 * D / 4) ** -0.5  # of the model's 128 + 64 (or 64 + 32) wide heads
        # logits of standard deviation about 2
        rms = math.sqrt(D * (1 + 63 / 100) + R)
        st["q"] = _normal((T, H, D + R), g, 2.0 / (st["sm_scale"] * rms))
        st["o"] = torch.zeros(T, H, D, dtype=torch.bfloat16, device=DEV)
        st["kv_indptr"] = starts.to(torch.int32)
        st["kv_indices"] = order.to(torch.int32)
        st["kv_lens"] = torch.tensor(lens, device=DEV)
        st["qo_indptr"] = torch.tensor([0] + [sum(chunks[:i + 1]) for i in range(len(chunks))], dtype=torch.int32,
                                       device=DEV)
        st["max_q"] = max(chunks)
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _encode(y):
    """(packed codes, scale bytes) of fp32 rows ``y``: the scale is the least power of two under which the
    block's largest magnitude is below 7 (so no value is off by more than half a step), codes round to nearest,
    ties to even, up to 6."""
    n, D = y.shape
    v = y.view(n, D // 32, 32)
    big = v.abs().amax(-1)
    b = ((big.view(torch.int32) + 0x200000) >> 23) - 2
    bad = ~torch.isfinite(big) | (b > HIGHEST)
    b = b.clamp(LOWEST, HIGHEST)
    w = torch.where(bad.unsqueeze(-1), torch.zeros_like(v), v * torch.exp2(127.0 - b.float()).unsqueeze(-1))
    m = w.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    m = (torch.round(m / step) * step).clamp(max=6.0)
    code = torch.where(m < 2, 2 * m, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(w).to(torch.uint8) << 3)).view(n, D // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), torch.where(bad, NAN, b).to(torch.uint8)


def _decode(codes, scales):
    """fp32 rows of packed codes and scale bytes."""
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    s = torch.where(scales == NAN, float("nan"), torch.exp2(scales.float() - 127.0))
    return v * s.repeat_interleave(32, -1)


def _read(pool, slots, rotation):
    x = _decode(pool.c_codes[0][slots], pool.c_scales[0][slots])
    if rotation is not None:
        x = x @ rotation.float().t()
    return torch.cat((x.to(torch.bfloat16), pool.rope_buf[0][slots]), -1)


def _attend(st):
    pool, q, page = st["pool"], st["q"], st["page"]
    T, H, _ = q.shape
    D = pool.kv_lora_rank
    B, L, Q = st["kv_lens"].numel(), st["max_len"], st["max_q"]
    pos = torch.arange(L, device=DEV)
    at = st["kv_indptr"][:-1, None] + torch.div(pos, page, rounding_mode="floor")
    slot = st["kv_indices"][at.clamp(max=st["kv_indices"].numel() - 1)].long() * page + pos % page
    slot = torch.where(pos < st["kv_lens"][:, None], slot, 0)
    k = torch.cat((_decode(pool.c_codes[0][slot], pool.c_scales[0][slot]), pool.rope_buf[0][slot].float()), -1)
    i = torch.arange(Q, device=DEV)
    chunk = (st["qo_indptr"][1:] - st["qo_indptr"][:-1]).long()
    rows = st["qo_indptr"][:-1, None].long() + i  # [B, Q]
    live = i < chunk[:, None]
    qq = q[rows.clamp(max=T - 1)].float().view(B, Q * H, -1)
    s = torch.matmul(qq, k.transpose(1, 2)).view(B, Q, H, L)
    s *= st["sm_scale"]
    last = st["kv_lens"][:, None] - chunk[:, None] + i  # the last position that a query sees
    s.masked_fill_((pos > last[..., None])[:, :, None], float("-inf"))
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, Q * H, L), k[..., :D]).view(B, Q, H, D)
    st["o"][rows[live]] = o[live].to(torch.bfloat16)
    return st["o"]


def run(st):
    case, pool = st["case"], st["pool"]
    rotation = pool.rotation
    if own:
        from mla_kv_quant_amd import mx4

        if case["op"] == "attend":
            mx4.attend_fwd(st["q"], st["o"], pool, 0, st["kv_indptr"], st["kv_indices"], st["kv_lens"], st["sm_scale"],
                           qo_indptr=st["qo_indptr"], max_q_len=st["max_q"], page_size=st["page"])
            return st["o"]
        if case["op"] == "write":
            mx4.write_rows(pool, 0, st["slots"], st["latent"], st["k_pe"])
        return mx4.read_rows(pool, 0, st["slots"])
    if case["op"] == "attend":
        return _attend(st)
    if case["op"] == "write":
        y = st["latent"].float()
        if rotation is not None:
            y = y @ rotation.float()
        pool.c_codes[0][st["slots"]], pool.c_scales[0][st["slots"]] = _encode(y)
        pool.rope_buf[0][st["slots"]] = st["k_pe"]
    return _read(pool, st["slots"], rotation)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _value64(codes, scales):
    """Stored rows in 64 bits, from the fields of the 4-bit format: sign, two exponent bits, one of the significand."""
    nib = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
    e, m = (nib // 2) % 4, (nib % 2).double()
    mag = torch.where(e == 0, m / 2, (1 + m / 2) * torch.ldexp(torch.ones_like(m), e - 1))
    v = torch.where(nib >= 8, -mag, mag).unflatten(-1, (-1, 32))
    s = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64, device=scales.device), scales.long() - 127)
    return (v * torch.where(scales == NAN, float("nan"), s)[..., None]).flatten(-2)


def _nearest64(y):
    """The values that rows in 64 bits are stored as: the nearest level (the even code on ties) at the block's scale."""
    v = y.unflatten(-1, (-1, 32))
    big = v.abs().amax(-1)
    e = torch.ceil(torch.log2(big / 7))
    e = torch.where(big >= 7 * torch.exp2(e), e + 1, e).clamp(LOWEST - 127, HIGHEST - 127)  # big < 7 * 2^e
    s = torch.exp2(e)[..., None]
    m, lv = (v / s).abs(), torch.tensor(LEVELS, dtype=torch.float64, device=y.device)
    code = torch.zeros_like(m)
    for c in range(7):
        mid = (lv[c] + lv[c + 1]) / 2
        code += ((m >= mid) if c % 2 else (m > mid)).double()
    return (torch.sign(v) * lv[code.long()] * s).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    pool, D = st["pool"], case["D"]
    rot = None if pool.rotation is None else pool.rotation.double()
    if case["op"] != "attend":
        out = []
        for at in st["slots"].split(8192):
            if case["op"] == "write":
                i = len(out) * 8192
                y = st["latent"][i:i + 8192].double()
                x, pe = _nearest64(y if rot is None else y @ rot), st["k_pe"][i:i + 8192]
            else:
                x, pe = _value64(pool.c_codes[0][at], pool.c_scales[0][at]), pool.rope_buf[0][at]
            out.append(torch.cat((x if rot is None else x @ rot.t(), pe.double()), -1))
        return torch.cat(out)
    H, page = case["heads"], st["page"]
    o = torch.zeros(st["o"].shape, dtype=torch.float64, device=DEV)
    qo, ptr = st["qo_indptr"].tolist(), st["kv_indptr"].tolist()
    for b, n in enumerate(st["kv_lens"].tolist()):
        t = torch.arange(n, device=DEV)
        at = st["kv_indices"][ptr[b]:ptr[b + 1]].long()[t // page] * page + t % page
        v = _value64(pool.c_codes[0][at], pool.c_scales[0][at])
        k = torch.cat((v, pool.rope_buf[0][at].double()), -1)
        step = max(1, (1 << 27) // (n * H))
        for i in range(qo[b], qo[b + 1], step):
            j = min(i + step, qo[b + 1])
            z = torch.einsum("thd,nd->thn", st["q"][i:j].double(), k) * st["sm_scale"]
            last = n - qo[b + 1] + torch.arange(i, j, device=DEV)
            z = z.where(t <= last[:, None, None], float("-inf"))
            o[i:j] = torch.einsum("thn,nd->thd", torch.exp(z - torch.logsumexp(z, -1, keepdim=True)), v)
    return o
