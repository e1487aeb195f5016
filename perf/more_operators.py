"""What a latent-attention serving loop does around the caches: rotary positions, the
expanded form of the attention, and eviction by accumulated attention weight.

* ``rotary``: the rope parts of the queries (``H`` heads) and of the one shared key of
  every token, rotated by the token's position, from where the projections left them
  (the last columns of the query heads) to where they are used (the rope columns of the
  absorbed query, the writer's ``k_pe``). Pairs are neighbours or halves apart; the
  frequencies are plain, or scaled for long contexts (linear, yarn, longrope). Angles
  are exact: positions go up to 131071 and angles are formed in 64 bits.
* ``expanded``: causal attention over keys and values that ``kv_b_proj`` expanded from
  the latent rows: per head ``k = (k_nope | k_pe)`` with one ``k_pe`` for all heads.
  Prompts from their start, chunks behind a prefix, a few tokens; widths
  (nope, rope, value) are (128, 64, 128) and (64, 32, 64).
* ``weights``: the attention weight that every cached position of the 4-bit latent cache
  gets from a request's queries, summed over heads and queries (their log sums of
  exponentials are in hand from the attention call).
* ``evict``: which positions of each request stay: the first ones, the last ones and
  those of largest accumulated weight, in order, with their slots and weights; the other
  slots are given back.

Inputs are synthetic: projections N(0, 1), queries that give logits of standard
deviation about 2, pages in shuffled order, accumulated weights that fall off as those of
trained models do (a few heavy positions, many that share the rest).
"""

import math
import random
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# rotary scalings as a model's configuration states them, by the rope width they are used with
SCALINGS = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "yarn": {"type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, "beta_fast": 32.0,
             "beta_slow": 1.0, "mscale": 1.0, "mscale_all_dim": 0.707},
    "longrope": {"type": "longrope", "factor": 4.0, "original_max_position_embeddings": 32768},
}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a decode step of a small batch: the smallest call, one launch for queries and keys
        {"name": "rotary_b8", "op": "rotary", "tokens": 8, "heads": 16, "dim": 64, "nope": 128, "wide": 512,
         "layout": "interleaved", "scaling": "yarn", "type": "bf16", "far": 16384, "mix": 1},
        # a large prefill batch, 16 x 2048 tokens
        {"name": "rotary_16x2048", "op": "rotary", "tokens": 32768, "heads": 16, "dim": 64, "nope": 128, "wide": 512,
         "layout": "interleaved", "scaling": "yarn", "type": "bf16", "far": 163840, "mix": 2},
        # the small width with 40 heads, halves, an odd number of far tokens
        {"name": "rotary_5003_40h_half", "op": "rotary", "tokens": 5003, "heads": 40, "dim": 32, "nope": 64,
         "wide": 256, "layout": "half", "scaling": "longrope", "type": "bf16", "far": 131072, "mix": 3},
        # one short prompt: latency
        {"name": "expanded_b1_333", "op": "expanded", "nope": 128, "heads": 16, "batch": 1, "q_lo": 333, "q_hi": 333,
         "p_lo": 0, "p_hi": 0, "causal": True, "mix": 4},
        # prompts from their start
        {"name": "expanded_4x4096", "op": "expanded", "nope": 128, "heads": 16, "batch": 4, "q_lo": 4096, "q_hi": 4096,
         "p_lo": 0, "p_hi": 0, "causal": True, "mix": 5},
        # chunked prefill over long prefixes, small width, 40 heads: the largest call
        {"name": "expanded_4x2048_14336_40h_64", "op": "expanded", "nope": 64, "heads": 40, "batch": 4, "q_lo": 2048,
         "q_hi": 2048, "p_lo": 14336, "p_hi": 14336, "causal": True, "mix": 6},
        # a mixed batch: ragged chunks over ragged prefixes, 128 heads
        {"name": "expanded_ragged_128h", "op": "expanded", "nope": 128, "heads": 128, "batch": 5, "q_lo": 1,
         "q_hi": 700, "p_lo": 100, "p_hi": 5000, "causal": True, "mix": 7},
        # one request, token-level index lists, the weights of one decode step
        {"name": "weights_b1_3001", "op": "weights", "D": 512, "heads": 16, "batch": 1, "lo": 3001, "hi": 3001,
         "q_lo": 1, "q_hi": 1, "page": 1, "mix": 8},
        # a decode step's weights of batch 32 x 16384
        {"name": "weights_b32_16k", "op": "weights", "D": 512, "heads": 16, "batch": 32, "lo": 16384, "hi": 16384,
         "q_lo": 1, "q_hi": 1, "page": 64, "mix": 9},
        # the last 32 queries of each prompt say which positions to keep: small width, 40 heads
        {"name": "weights_window_b8_40h_256", "op": "weights", "D": 256, "heads": 40, "batch": 8, "lo": 8192,
         "hi": 16384, "q_lo": 32, "q_hi": 32, "page": 64, "mix": 10},
        # 32 requests of 16384 positions down to 2048
        {"name": "evict_b32_16k", "op": "evict", "batch": 32, "lo": 16384, "hi": 16384, "budget": 2048, "sink": 4,
         "recent": 64, "page": 64, "mix": 11},
        # one long request down to a sixteenth, token-level index lists
        {"name": "evict_b1_128k", "op": "evict", "batch": 1, "lo": 131072, "hi": 131072, "budget": 8192, "sink": 4,
         "recent": 16, "page": 1, "mix": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges."""
    op = rng.choice(["rotary", "expanded", "expanded", "weights", "weights", "evict"])
    c = {"op": op, "mix": rng.randrange(1 << 20)}
    if op == "rotary":
        dim = rng.choice([64, 64, 32])
        tokens = _log(rng, 1, 32768)
        heads = rng.choice([16, 16, 40, 1, 8, 20, 128])
        heads = max(1, min(heads, (32768 * 16) // tokens))
        c.update(tokens=tokens, heads=heads, dim=dim, nope=2 * dim, wide=8 * dim,
                 layout=rng.choice(["interleaved", "half"]), scaling=rng.choice(sorted(SCALINGS)),
                 type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), far=_log(rng, max(2, tokens // 16), 163840))
        return c
    if op == "expanded":
        nope = rng.choice([128, 64])
        heads = rng.choice([16, 16, 8, 32, 128, 1, 20] if nope == 128 else [40, 40, 8, 16, 24])
        batch, q_hi, p_hi = _log(rng, 1, 12), _log(rng, 1, 4096), _log(rng, 1, 16384)
        scores = 4.0e9 / (nope / 64)  # below the largest listed call
        if batch * heads * q_hi * (p_hi + q_hi) > scores:
            q_hi = max(1, int(scores / (batch * heads * (p_hi + q_hi))))
        c.update(nope=nope, heads=heads, batch=batch, q_lo=max(1, int(q_hi * rng.uniform(0.1, 1.0))), q_hi=q_hi,
                 p_lo=int(p_hi * rng.uniform(0.0, 1.0)) if rng.random() < 0.7 else 0, p_hi=p_hi,
                 causal=rng.random() < 0.8)
        if rng.random() < 0.3:
            c.update(p_lo=0, p_hi=0)
        return c
    if op == "weights":
        D = rng.choice([512, 256])
        heads = rng.choice([16, 16, 8, 24, 32, 64, 128, 1, 20] if D == 512 else [40, 40, 16, 20, 24, 48, 8])
        n = _log(rng, 200, 1 << 19)  # cached positions in all
        batch = min(_log(rng, 1, 100), max(1, n // 20))
        hi = min(max(20, n // batch), 65536)
        q_hi = _log(rng, 1, 64) if rng.random() < 0.5 else 1
        q_hi = max(1, min(q_hi, hi, int(1.5e8 / (batch * hi * heads * D / 256))))
        c.update(D=D, heads=heads, batch=batch, lo=max(q_hi, int(hi * rng.uniform(0.1, 1.0))), hi=max(q_hi, hi),
                 q_lo=1, q_hi=q_hi, page=rng.choice([64, 64, 32, 16, 1]))
        return c
    n = _log(rng, 500, 1 << 19)
    batch = min(_log(rng, 1, 100), max(1, n // 50))
    hi = min(n // batch, 131072)
    sink, recent = rng.choice([0, 4, 4, 16]), rng.choice([1, 16, 64, 64])
    c.update(batch=batch, lo=max(1, int(hi * rng.uniform(0.1, 1.0))), hi=hi, sink=sink, recent=recent,
             budget=sink + recent + _log(rng, 1, max(2, hi // 2)), page=rng.choice([64, 32, 16, 1]))
    return c


# ---------------------------------------------------------------------------
# sizes that follow from a case alone
# ---------------------------------------------------------------------------
def _lengths(case, lo="lo", hi="hi", salt=0):
    r = random.Random("%s %s" % (case["mix"], salt))
    return [r.randint(case[lo], case[hi]) for _ in range(case["batch"])]


def _expanded_lengths(case):
    """(queries, keys) of each request."""
    q, p = _lengths(case, "q_lo", "q_hi", 1), _lengths(case, "p_lo", "p_hi", 2)
    return q, [a + b for a, b in zip(q, p)]


def work(case):
    """Bytes and operations that one pass cannot do without."""
    if case["op"] == "rotary":
        T, rows = case["tokens"], case["tokens"] * (case["heads"] + 1)
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": 2.0 * rows * case["dim"] * size + 8 * T, "flops": 4.0 * rows * case["dim"]}
    if case["op"] == "expanded":
        dn, dr, H = case["nope"], case["nope"] // 2, case["heads"]
        qs, ks = _expanded_lengths(case)
        pairs = sum(q * (k - q) + q * (q + 1) // 2 if case["causal"] else q * k for q, k in zip(qs, ks))
        b = 2.0 * (sum(qs) * H * (2 * dn + dr) + sum(ks) * (2 * H * dn + dr))
        return {"bytes": b, "flops": 2.0 * H * (2 * dn + dr) * pairs}
    lens = _lengths(case)
    n = sum(lens)
    if case["op"] == "weights":
        D, R, H = case["D"], case["D"] // 8, case["heads"]
        chunks = _lengths(case, "q_lo", "q_hi", 1)
        T = sum(chunks)
        pairs = sum(q * (m - q) + q * (q + 1) // 2 for m, q in zip(lens, chunks))
        row = D // 2 + D // 32 + 2 * R
        return {"bytes": float(n * (row + 4) + T * H * (2 * (D + R) + 4) + 4 * (n // case["page"])),
                "flops": 2.0 * H * (D + R) * pairs}
    kept = sum(min(m, case["budget"]) for m in lens)
    # the weights in, those of the kept positions and zeros out, every position's slot out
    return {"bytes": float(4 * n + 4 * n + 4 * n + 4 * (n // case["page"])), "flops": float(n + kept)}


# ---------------------------------------------------------------------------
# inputs (plain torch, from the seed alone)
# ---------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)
    return g


def _normal(shape, g, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _scaling(case):
    """The case's rotary scaling, with longrope's factors for its width."""
    s = SCALINGS[case["scaling"]]
    if s is not None and s["type"] == "longrope":
        n = case["dim"] // 2
        s = dict(s, long_factor=[1.0 + 30.0 * (i / n) ** 2 for i in range(n)],
                 short_factor=[1.0 + 0.5 * (i / n) for i in range(n)], long=case["far"] > 32768)
    return s


def _indptr(lens):
    at = [0]
    for m in lens:
        at.append(at[-1] + m)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def _pages(lens, page, g):
    """Shuffled pages of requests (page 0 is the padding page): offsets, numbers, how many."""
    counts = [-(-m // page) for m in lens]
    order = torch.randperm(sum(counts), generator=g, device=DEV) + 1
    return _indptr(counts), order.to(torch.int32), sum(counts) + 1


def _codes(n, D, g):
    """4-bit rows of normal values: packed codes and scale bytes."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    x = torch.randn(n, D, generator=g, device=DEV) * 2.0
    code = torch.bucketize(x.abs(), mids).to(torch.uint8) | (torch.signbit(x).to(torch.uint8) << 3)
    code = code.view(n, D // 2, 2)
    scales = torch.randint(125, 128, (n, D // 32), generator=g, device=DEV, dtype=torch.uint8)
    return code[..., 0] | (code[..., 1] << 4), scales


def prepare(case, seed):
    g = _gen(seed, 1)
    st = {"case": case}
    if case["op"] == "rotary":
        T, H, dim, nope, t = case["tokens"], case["heads"], case["dim"], case["nope"], TYPES[case["type"]]
        # requests' chunks at their places in long contexts
        starts = torch.randint(0, case["far"], (max(1, T // 2048),), generator=g, device=DEV)
        st["positions"] = (starts[torch.arange(T, device=DEV) * starts.numel() // T] + torch.arange(T, device=DEV)) \
            % case["far"]
        st["q"] = _normal((T, H, nope + dim), g, dtype=t)
        st["k_pe"] = _normal((T, dim), g, dtype=t)
        st["q_out"] = torch.zeros(T, H, case["wide"] + dim, dtype=t, device=DEV)
        st["k_out"] = torch.zeros(T, dim, dtype=t, device=DEV)
        st["inv_freq"], st["scale"] = _frequencies(case)
        if own:
            from mla_kv_quant_amd import rotary

            st["rope"] = rotary.Rotary(dim, 10000.0, interleaved=case["layout"] == "interleaved",
                                       scaling=_scaling(case), device=DEV)
        return st
    if case["op"] == "expanded":
        dn, dr, H = case["nope"], case["nope"] // 2, case["heads"]
        qs, ks = _expanded_lengths(case)
        st["sm_scale"] = (dn + dr) ** -0.5
        st["q"] = _normal((sum(qs), H, dn + dr), g, 2.0)
        st["kv"] = _normal((sum(ks), H, 2 * dn), g)
        st["k_pe"] = _normal((sum(ks), dr), g)
        st["o"] = torch.zeros(sum(qs), H, dn, dtype=torch.bfloat16, device=DEV)
        st["qo_indptr"], st["kv_indptr"] = _indptr(qs), _indptr(ks)
        st["max_q"], st["max_k"] = max(qs), max(ks)
        return st
    lens = _lengths(case)
    n, B, L = sum(lens), case["batch"], max(lens)
    st["kv_indptr"], st["kv_indices"], pages = _pages(lens, case["page"], g)
    st["kv_lens"] = torch.tensor(lens, device=DEV)
    st["max_len"] = L
    st["reqs"] = torch.randperm(B + 3, generator=g, device=DEV)[:B]  # rows of the accumulated weights
    if case["op"] == "evict":
        # heavy tails: exp of a normal with a standard deviation of 3
        st["acc"] = torch.exp(3.0 * torch.randn(B + 3, L + 64, generator=g, device=DEV))
        st["kept"] = torch.zeros(B, case["budget"], dtype=torch.int32, device=DEV)
        st["kept_lens"] = torch.zeros(B, dtype=torch.int64, device=DEV)
        st["freed"] = torch.zeros(st["kv_indices"].numel() * case["page"], dtype=torch.int32, device=DEV)
        st["acc_out"] = torch.zeros_like(st["acc"])
        return st
    D, H = case["D"], case["heads"]
    R, slots = D // 8, pages * case["page"]
    pool = SimpleNamespace(kv_lora_rank=D, qk_rope_head_dim=R, start_layer=0)
    codes, scales = _codes(slots, D, g)
    pool.c_codes, pool.c_scales, pool.rope_buf = [codes], [scales], [_normal((slots, R), g)]
    pool.latent_rotation = lambda layer_id, local=True: None
    chunks = _lengths(case, "q_lo", "q_hi", 1)
    st["pool"], st["max_q"], st["qo_indptr"] = pool, max(chunks), _indptr(chunks)
    st["sm_scale"] = (1.5 * D / 4) ** -0.5
    # logits of standard deviation about 2 (a value's mean square is about 4 * 7 / 16 / 3 * 4)
    rms = math.sqrt(D * 2.3 + R)
    st["q"] = _normal((sum(chunks), H, D + R), g, 2.0 / (st["sm_scale"] * rms))
    st["acc"] = torch.zeros(B + 3, L + 64, device=DEV)
    # what the attention call over the same queries returned
    s, live, rows = _scores(st)
    st["lse"] = torch.empty(sum(chunks), H, device=DEV)
    st["lse"][rows[live]] = torch.logsumexp(s, -1)[live]
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _frequencies(case):
    """Angle of a step of one position for each pair (64 bits), and the factor of sines and cosines."""
    dim, s = case["dim"], _scaling(case)
    i = torch.arange(dim // 2, dtype=torch.float64, device=DEV)
    f = torch.pow(torch.tensor(10000.0, dtype=torch.float64, device=DEV), -2.0 * i / dim)
    if s is None:
        return f, 1.0
    if s["type"] == "linear":
        return f / s["factor"], 1.0
    if s["type"] == "longrope":
        by = s["long_factor"] if s["long"] else s["short_factor"]
        scale = math.sqrt(1.0 + math.log(s["factor"]) / math.log(s["original_max_position_embeddings"]))
        return f / torch.tensor(by, dtype=torch.float64, device=DEV), scale
    # yarn: pairs that turn more than beta_fast times over the original length stay, those that turn less than
    # beta_slow times are slowed by the factor, a ramp over the pairs' numbers in between
    def pair(turns):
        return dim * math.log(s["original_max_position_embeddings"] / (turns * 2 * math.pi)) / (2 * math.log(10000.0))

    low = max(math.floor(pair(s["beta_fast"])), 0)
    high = min(math.ceil(pair(s["beta_slow"])), dim - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    m = [0.1 * s[k] * math.log(s["factor"]) + 1.0 for k in ("mscale", "mscale_all_dim")]
    return f / s["factor"] * ramp + f * (1.0 - ramp), m[0] / m[1]


def _rotate(x, cos, sin, interleaved):
    x = x.float()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
    ya, yb = a * cos - b * sin, b * cos + a * sin
    return torch.stack((ya, yb), -1).flatten(-2) if interleaved else torch.cat((ya, yb), -1)


def _rotary(st):
    case, t = st["case"], st["q"].dtype
    angle = st["positions"].double()[:, None] * st["inv_freq"]
    cos, sin = (torch.cos(angle) * st["scale"]).float(), (torch.sin(angle) * st["scale"]).float()
    two = case["layout"] == "interleaved"
    st["q_out"][..., case["wide"]:] = _rotate(st["q"][..., case["nope"]:], cos[:, None], sin[:, None], two).to(t)
    st["k_out"].copy_(_rotate(st["k_pe"], cos, sin, two).to(t))


def _rows(indptr, most):
    """Rows of every request, padded to `most`: their numbers and which of them there are."""
    i = torch.arange(most, device=DEV)
    live = i < (indptr[1:] - indptr[:-1])[:, None]
    return torch.where(live, indptr[:-1, None].long() + i, 0), live


def _expanded(st):
    case = st["case"]
    dn, H = case["nope"], case["heads"]
    at_q, live = _rows(st["qo_indptr"], st["max_q"])
    at_k, seen = _rows(st["kv_indptr"], st["max_k"])
    q = st["q"][at_q].float().transpose(1, 2)  # [B, H, Q, dn + dr]
    kv = st["kv"][at_k].float().transpose(1, 2)
    pe = st["k_pe"][at_k].float()[:, None]
    s = torch.matmul(q[..., :dn], kv[..., :dn].transpose(2, 3))
    s += torch.matmul(q[..., dn:], pe.transpose(2, 3))
    s *= st["sm_scale"]
    hidden = ~seen[:, None]
    if case["causal"]:
        n = (st["kv_indptr"][1:] - st["kv_indptr"][:-1]) - (st["qo_indptr"][1:] - st["qo_indptr"][:-1])
        last = n[:, None] + torch.arange(st["max_q"], device=DEV)  # the last position that a query sees
        hidden = hidden | (torch.arange(st["max_k"], device=DEV) > last[..., None])
    s.masked_fill_(hidden[:, None], float("-inf"))
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    o = torch.matmul(s, kv[..., dn:]).transpose(1, 2)
    st["o"][at_q[live]] = o[live].to(torch.bfloat16)
    return st["o"]


def _values(codes, scales):
    """fp32 rows of packed codes and scale bytes."""
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    return v * torch.exp2(scales.float() - 127.0).repeat_interleave(32, -1)


def _slots(st):
    """[B, L] slots of the positions (0 behind a request's last)."""
    page, pos = st["case"]["page"], torch.arange(st["max_len"], device=DEV)
    at = (st["kv_indptr"][:-1, None] + pos // page).clamp(max=st["kv_indices"].numel() - 1)
    slot = st["kv_indices"][at].long() * page + pos % page
    return torch.where(pos < st["kv_lens"][:, None], slot, 0)


def _scores(st):
    """Scaled scores [B, Q, H, L], -inf where a query does not see; which queries there are; their rows."""
    pool, slot = st["pool"], _slots(st)
    k = torch.cat((_values(pool.c_codes[0][slot], pool.c_scales[0][slot]), pool.rope_buf[0][slot].float()), -1)
    rows, live = _rows(st["qo_indptr"], st["max_q"])
    B, Q = rows.shape
    H = st["q"].shape[1]
    s = torch.matmul(st["q"][rows].float().view(B, Q * H, -1), k.transpose(1, 2)).view(B, Q, H, -1)
    s *= st["sm_scale"]
    chunk = (st["qo_indptr"][1:] - st["qo_indptr"][:-1]).long()
    last = st["kv_lens"][:, None] - chunk[:, None] + torch.arange(Q, device=DEV)
    hidden = (torch.arange(st["max_len"], device=DEV) > last[..., None]) | ~live[..., None]
    s.masked_fill_(hidden[:, :, None], float("-inf"))
    return s, live, rows


def _weights(st):
    s, live, rows = _scores(st)
    s -= torch.where(live[..., None], st["lse"][rows], 0.0)[..., None]
    s.exp_()
    w = s.sum((1, 2))
    there = torch.arange(st["max_len"], device=DEV) < st["kv_lens"][:, None]
    acc = st["acc"][st["reqs"], :st["max_len"]]
    st["acc"][st["reqs"], :st["max_len"]] = torch.where(there, w, acc)
    return st["acc"]


def _evict(st):
    case = st["case"]
    L, n = st["max_len"], st["kv_lens"][:, None]
    pos = torch.arange(L, device=DEV)
    w = st["acc"][st["reqs"], :L]
    there = pos < n
    safe = there & ((pos < case["sink"]) | (pos >= n - case["recent"]) | (n <= case["budget"]))
    open_ = there & ~safe
    # by weight, then the open ones before the others; both sorts keep the order of equals
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    order = order.gather(1, torch.sort(open_.gather(1, order).byte(), dim=-1, descending=True, stable=True).indices)
    rank = torch.empty_like(order).scatter_(1, order, pos.expand_as(order))
    keep = safe | (open_ & (rank < case["budget"] - case["sink"] - case["recent"]))
    slot = _slots(st).to(torch.int32)
    to = keep.cumsum(1) - 1
    b = torch.arange(case["batch"], device=DEV)[:, None].expand_as(to)
    st["kept"][b[keep], to[keep]] = slot[keep]
    st["kept_lens"].copy_(keep.sum(1))
    gone = there & ~keep
    st["freed"][gone.flatten().cumsum(0)[gone.flatten()] - 1] = slot[gone]
    out = torch.zeros_like(w)
    out[b[keep], to[keep]] = w[keep]
    st["acc_out"][st["reqs"], :L] = torch.where(there, out, st["acc_out"][st["reqs"], :L])
    return st["kept"], st["kept_lens"], st["freed"], st["acc_out"]


def run(st):
    case = st["case"]
    if case["op"] == "rotary":
        if own:
            from mla_kv_quant_amd import rotary

            rotary.apply_rotary(st["rope"], st["positions"], st["q"][..., case["nope"]:], st["k_pe"],
                                q_out=st["q_out"][..., case["wide"]:], k_out=st["k_out"])
        else:
            _rotary(st)
        return st["q_out"][..., case["wide"]:], st["k_out"]
    if case["op"] == "expanded":
        if not own:
            return _expanded(st)
        from mla_kv_quant_amd import expanded

        return expanded.expanded_attend_fwd(st["q"], st["kv"], st["k_pe"], st["o"], st["qo_indptr"], st["kv_indptr"],
                                            st["max_q"], st["sm_scale"], causal=case["causal"])
    if case["op"] == "weights":
        if not own:
            return _weights(st)
        from mla_kv_quant_amd import evict

        return evict.accumulate_weights(st["q"], st["lse"], st["pool"], 0, st["acc"], st["kv_indptr"],
                                        st["kv_indices"], st["kv_lens"], st["sm_scale"], qo_indptr=st["qo_indptr"],
                                        max_q_len=st["max_q"], page_size=case["page"], req_pool_indices=st["reqs"],
                                        add=False)
    if not own:
        return _evict(st)
    from mla_kv_quant_amd import evict

    kept, kept_lens, freed = evict.evict(st["acc"], st["kv_indptr"], st["kv_indices"], st["kv_lens"], case["budget"],
                                         sink=case["sink"], recent=case["recent"], page_size=case["page"],
                                         req_pool_indices=st["reqs"], max_kv_len=st["max_len"],
                                         acc_out=st["acc_out"], kept=st["kept"], kept_lens=st["kept_lens"],
                                         freed=st["freed"])
    return kept, kept_lens, freed, st["acc_out"]


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rotary(case, st):
    """Pairs as complex numbers, turned by position times frequency."""
    dim, s = case["dim"], _scaling(case) or {"type": "none"}
    freq, scale = [], 1.0
    if s["type"] == "longrope":
        scale = math.sqrt(1 + math.log(s["factor"], s["original_max_position_embeddings"]))
    if s["type"] == "yarn":
        scale = (1 + 0.1 * s["mscale"] * math.log(s["factor"])) / (1 + 0.1 * s["mscale_all_dim"] * math.log(s["factor"]))
        edge = [dim / 2 * math.log(s["original_max_position_embeddings"] / (2 * math.pi * b), 10000.0)
                for b in (s["beta_fast"], s["beta_slow"])]
        lo, hi = max(0, math.floor(edge[0])), min(dim - 1, math.ceil(edge[1]))
    for i in range(dim // 2):
        f = 10000.0 ** (-2.0 * i / dim)
        if s["type"] == "linear":
            f /= s["factor"]
        elif s["type"] == "longrope":
            f /= (s["long_factor"] if s["long"] else s["short_factor"])[i]
        elif s["type"] == "yarn":
            slowed = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f *= 1.0 - slowed + slowed / s["factor"]
        freq.append(f)
    turn = torch.polar(torch.full((case["tokens"], dim // 2), scale, dtype=torch.float64, device=DEV),
                       st["positions"].double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=DEV))

    def turned(x, turn):
        x = x.double()
        if case["layout"] == "interleaved":
            return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
        z = torch.complex(x[..., :dim // 2].contiguous(), x[..., dim // 2:].contiguous()) * turn
        return torch.cat((z.real, z.imag), -1)

    return turned(st["q"][..., case["nope"]:], turn[:, None]), turned(st["k_pe"], turn)


def _exact_expanded(case, st):
    dn, H = case["nope"], case["heads"]
    o = torch.zeros(st["o"].shape, dtype=torch.float64, device=DEV)
    qo, ko = st["qo_indptr"].tolist(), st["kv_indptr"].tolist()
    for b in range(case["batch"]):
        n, m = ko[b + 1] - ko[b], qo[b + 1] - qo[b]
        pe = st["k_pe"][ko[b]:ko[b + 1]].double()
        step = max(1, (1 << 28) // n)
        for h in range(H):
            kv = st["kv"][ko[b]:ko[b + 1], h].double()
            k = torch.cat((kv[:, :dn], pe), -1)
            for i in range(0, m, step):
                j = min(i + step, m)
                z = st["q"][qo[b] + i:qo[b] + j, h].double() @ k.t() * st["sm_scale"]
                if case["causal"]:
                    z = z.where(torch.arange(n, device=DEV) <= n - m + torch.arange(i, j, device=DEV)[:, None],
                                float("-inf"))
                o[qo[b] + i:qo[b] + j, h] = torch.exp(z - torch.logsumexp(z, -1, keepdim=True)) @ kv[:, dn:]
    return o


def _exact_weights(case, st):
    acc, pool, page = st["acc"].double(), st["pool"], case["page"]
    qo, ptr = st["qo_indptr"].tolist(), st["kv_indptr"].tolist()
    for b, n in enumerate(st["kv_lens"].tolist()):
        t = torch.arange(n, device=DEV)
        at = st["kv_indices"][ptr[b]:ptr[b + 1]].long()[t // page] * page + t % page
        codes = pool.c_codes[0][at]
        nib = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
        e, m = (nib // 2) % 4, (nib % 2).double()
        v = torch.where(e == 0, m / 2, (1 + m / 2) * torch.ldexp(torch.ones_like(m), e - 1))
        v = torch.where(nib >= 8, -v, v).unflatten(-1, (-1, 32))
        v = (v * torch.ldexp(torch.ones_like(v[..., 0]), pool.c_scales[0][at].long() - 127)[..., None]).flatten(-2)
        k = torch.cat((v, pool.rope_buf[0][at].double()), -1)
        w = torch.zeros(n, dtype=torch.float64, device=DEV)
        for i in range(qo[b], qo[b + 1]):
            z = k @ st["q"][i].double().t() * st["sm_scale"] - st["lse"][i].double()
            w += torch.exp(z).sum(-1).where(t <= n - qo[b + 1] + i, 0.0)
        acc[st["reqs"][b], :n] = w
    return acc


def _exact_evict(case, st):
    kept, freed = st["kept"].clone(), st["freed"].clone()
    out, page, used = st["acc_out"].double(), case["page"], 0
    ptr, counts = st["kv_indptr"].tolist(), []
    for b, n in enumerate(st["kv_lens"].tolist()):
        t = torch.arange(n, device=DEV)
        at = st["kv_indices"][ptr[b]:ptr[b + 1]].long()[t // page] * page + t % page
        w = st["acc"][st["reqs"][b], :n].double()
        stay = torch.ones(n, dtype=torch.bool, device=DEV)
        if n > case["budget"]:
            mid = torch.arange(case["sink"], n - case["recent"], device=DEV)
            best = mid[torch.argsort(-w[mid], stable=True)]
            stay[best[case["budget"] - case["sink"] - case["recent"]:]] = False
        kept[b, :int(stay.sum())] = at[stay].int()
        counts.append(int(stay.sum()))
        freed[used:used + n - counts[-1]] = at[~stay].int()
        used += n - counts[-1]
        out[st["reqs"][b], :n] = torch.nn.functional.pad(w[stay], (0, n - counts[-1]))
    return kept, torch.tensor(counts, device=DEV), freed, out


def exact(case, seed):
    st = prepare(case, seed)
    return {"rotary": _exact_rotary, "expanded": _exact_expanded, "weights": _exact_weights,
            "evict": _exact_evict}[case["op"]](case, st)
