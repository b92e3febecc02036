"""The attention half of a decode or prompt step, and the choice of the next token: cases, plain forms and calls.

Operators, each in a plain form (elementary torch operations, 32 bits, 64 where 32 lose what matters) and as the
library's own call (``own`` true):

* ``norm_rope``: RMS norm of each query and key head and the position rotation, in one pass;
* ``append``: keys (normed and rotated on the way) and values appended to a paged cache held in 8 bits with one scale for
  each block of 32 tokens and head; the pass ends with reading back every block that it touched;
* ``attention``: queries against that cache, ragged lengths, causal, optionally within a window;
* ``sample``: temperature, top-k, top-p and min-p from given random numbers.

Cache layout (the library's): values are bytes ``128 + q``, q in -127..127. A page holds, for each KV head, its blocks of
32 tokens; K blocks are ``[D/16][32 tokens][16]``, V blocks ``[D][32]`` with token t of a block at place
``(t & 3) | (t >> 3 & 3) << 2 | (t >> 2 & 1) << 4``. Scales are float32 ``[pages, heads, blocks of a page]``.
"""

import math

import numpy as np
import torch

own = False

BLOCK = 32
FLOOR = 2.0 ** -64   # the least scale of a block
KINDS = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


# ---- cases -------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one token of one request at the 27B-shaped head layout: the launch is the cost
        {"name": "norm_rope_decode_1", "op": "norm_rope", "tokens": 1, "q_heads": 40, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "kind": "bf16", "start": 40961},
        # a long prompt of odd length with wide heads of which a part is rotated
        {"name": "norm_rope_prompt_8191_d256", "op": "norm_rope", "tokens": 8191, "q_heads": 16, "kv_heads": 2, "dim": 256,
         "rotary": 64, "interleaved": False, "kind": "bf16", "start": 0},
        # one token for each of eight requests, each somewhere inside a block
        {"name": "append_decode_8", "op": "append", "batch": 8, "q_lo": 1, "q_hi": 1, "before": 100, "kv_heads": 8,
         "dim": 128, "page": 64, "norm": True, "rotary": 128, "interleaved": False, "kind": "bf16"},
        # ragged prompts appended in one call, some on top of a context that ends inside a block
        {"name": "append_prompts_8k", "op": "append", "batch": 6, "q_lo": 700, "q_hi": 2048, "before": 200, "kv_heads": 8,
         "dim": 128, "page": 64, "norm": True, "rotary": 128, "interleaved": False, "kind": "bf16"},
        # a single request early in its answer: latency
        {"name": "attention_decode_1x600", "op": "attention", "batch": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 601, "kv_hi": 601,
         "q_heads": 40, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "kind": "bf16"},
        # eight requests of very different lengths, the decode batch of the 27B-shaped step
        {"name": "attention_decode_8x32k", "op": "attention", "batch": 8, "q_lo": 1, "q_hi": 1, "kv_lo": 900, "kv_hi": 32767,
         "q_heads": 40, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "kind": "bf16"},
        # a large serving batch, narrow heads, fp16, drafts of three tokens verified at once
        {"name": "attention_decode_64x8k_d64", "op": "attention", "batch": 64, "q_lo": 1, "q_hi": 3, "kv_lo": 300, "kv_hi": 8192,
         "q_heads": 32, "kv_heads": 8, "dim": 64, "page": 32, "window": 0, "kind": "fp16"},
        # one long prompt
        {"name": "attention_prompt_8192", "op": "attention", "batch": 1, "q_lo": 8192, "q_hi": 8192, "kv_lo": 8192,
         "kv_hi": 8192, "q_heads": 40, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "kind": "bf16"},
        # chunks of three prompts on top of what is cached, wide heads
        {"name": "attention_chunks_3x512_d256", "op": "attention", "batch": 3, "q_lo": 333, "q_hi": 512, "kv_lo": 2000,
         "kv_hi": 6001, "q_heads": 16, "kv_heads": 2, "dim": 256, "page": 128, "window": 0, "kind": "bf16"},
        # one request's next token over the lm_head's vocabulary
        {"name": "sample_1x151936", "op": "sample", "rows": 1, "vocab": 151936, "spread": 2.5, "top_k": 50, "top_p": 0.95, "min_p": 0.0},
        # requests with settings of their own, odd vocabulary
        {"name": "sample_8x32003_mixed", "op": "sample", "rows": 8, "vocab": 32003, "spread": 3.0, "top_k": -1, "top_p": 0.9, "min_p": 0.02},
        # a large serving batch, nucleus over the whole vocabulary
        {"name": "sample_64x151936_top_p", "op": "sample", "rows": 64, "vocab": 151936, "spread": 2.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "attention", "attention", "sample"])
    if op == "sample":
        return {"op": op, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, 151936), "spread": rng.choice([1.0, 2.0, 3.0]),
                "top_k": rng.choice([-1, 0, 1, 20, 50, 1000]), "top_p": rng.choice([1.0, 0.95, 0.8, 0.5]),
                "min_p": rng.choice([0.0, 0.0, 0.05])}
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 4, 5, 8])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    rotary = rng.choice([dim, dim, dim // 4])
    if op == "norm_rope":
        return {"op": op, "tokens": _log(rng, 1, 8192), "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
                "interleaved": rng.random() < 0.3, "kind": rng.choice(["bf16", "fp16", "f32"]), "start": _log(rng, 1, 200000)}
    page = rng.choice([32, 64, 128])
    if op == "append":
        hi = _log(rng, 1, 2048)
        return {"op": op, "batch": _log(rng, 1, 16), "q_lo": max(1, hi // 3), "q_hi": hi, "before": _log(rng, 1, 500),
                "kv_heads": kv_heads, "dim": dim, "page": page, "norm": rng.random() < 0.7, "rotary": rng.choice([rotary, 0]),
                "interleaved": rng.random() < 0.3, "kind": kind}
    window = rng.choice([0, 0, 0, _log(rng, 50, 4000)])
    if rng.random() < 0.5:   # decode
        hi = _log(rng, 1, 32768)
        return {"op": op, "batch": _log(rng, 1, max(1, min(64, 262144 // hi))), "q_lo": 1, "q_hi": rng.choice([1, 1, 2, 4]),
                "kv_lo": max(1, hi // 8), "kv_hi": hi, "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "page": page, "window": window, "kind": kind}
    hi = _log(rng, 16, 2048)
    batch = _log(rng, 1, max(1, min(8, 4096 // hi)))
    more = rng.choice([0, _log(rng, 1, 900)])
    return {"op": op, "batch": batch, "q_lo": max(1, hi // 2), "q_hi": hi, "kv_lo": hi + more // 2, "kv_hi": hi + more,
            "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "kind": kind}


def _lengths(lo, hi, batch, salt):
    """`batch` lengths from lo to hi, both among them (hi alone for a batch of one): sizes, the same for every seed."""
    if batch == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * 7919 + salt) % batch) // (batch - 1) for i in range(batch)]


def _shape(case):
    """Host-side lengths of an append or attention case."""
    b = case["batch"]
    q = _lengths(case["q_lo"], case["q_hi"], b, 1)
    if case["op"] == "append":
        kv = [n + (case["before"] * (i + 1) // b if i % 3 else 0) for i, n in enumerate(q)]
    else:
        kv = _lengths(case["kv_lo"], case["kv_hi"], b, 2)
        q = [min(n, m) for n, m in zip(q, kv)]
    return q, kv


def work(case):
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    if op == "norm_rope":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * (4 if case["kind"] == "f32" else 2) + 8 * case["tokens"] + 8 * case["dim"], "flops": 8 * n}
    q, kv = _shape(case)
    heads, dim = case["kv_heads"], case["dim"]
    if op == "append":
        n = sum(q) * heads * dim
        back = sum(b - (b - a) // BLOCK * BLOCK for a, b in zip(q, kv))
        scales = sum((b + 31) // BLOCK - (b - a) // BLOCK for a, b in zip(q, kv)) * heads * 8
        return {"bytes": 2 * n * 3 + 2 * back * heads * dim * 3 + 2 * scales, "flops": 12 * n}
    w = case["window"]
    pairs = sum(min(m - n + i + 1, w or m) for n, m in zip(q, kv) for i in range(n))
    seen = sum(min(m, (n + w - 1) if w else m) for n, m in zip(q, kv))
    return {"bytes": 4 * sum(q) * case["q_heads"] * dim + seen * heads * (2 * dim + 8 / BLOCK), "flops": 4.0 * pairs * case["q_heads"] * dim}


# ---- inputs ------------------------------------------------------------------------------------------------------


def _tables(case, seed):
    """Page table (int32, pages in random order, -1 where unused), prefix of the query lengths and cached lengths."""
    q, kv = _shape(case)
    page = case["page"]
    need = [(m + page - 1) // page for m in kv]
    pages = sum(need) + 3
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table = np.full((len(kv), max(need)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    return q, kv, pages, torch.from_numpy(table).cuda(), torch.from_numpy(start).cuda(), torch.tensor(kv, dtype=torch.int32).cuda()


def _inv_freq(rotary):
    return (1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float().cuda() if rotary else None


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    op = case["op"]
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab) * case["spread"]
        logits[:, : vocab // 10] -= 8.0                                           # a part of the vocabulary that is never near
        logits.scatter_add_(1, torch.randint(0, vocab, (rows, 20), generator=g, device="cuda"), 4 + 2 * normal(rows, 20))
        s["logits"] = logits
        s["uniform"] = torch.rand(rows, generator=g, device="cuda")
        s["temperature"] = 0.6 + 0.8 * torch.rand(rows, generator=g, device="cuda")
        s["top_k"] = torch.full((rows,), max(case["top_k"], 0), dtype=torch.int32, device="cuda")
        if case["top_k"] < 0:                                                     # a mixed batch: some rows without top-k
            s["top_k"] = torch.randint(0, 3, (rows,), generator=g, device="cuda", dtype=torch.int32) * 20
            s["temperature"][: rows // 4] = 0.0                                   # and some greedy ones
        s["top_p"] = torch.full((rows,), case["top_p"], device="cuda")
        s["min_p"] = torch.full((rows,), case["min_p"], device="cuda")
        return s
    dim, kind = case["dim"], KINDS[case["kind"]]
    weight = lambda: 1 + 0.2 * normal(dim)  # noqa: E731
    if op == "norm_rope":
        # as a fused projection leaves them: q and k are columns of one [tokens, (q | k | v)] matrix
        t, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
        s["qkv"] = (normal(t, (hq + 2 * hk) * dim) * 1.7).to(kind)
        s["q_weight"], s["k_weight"] = weight(), weight()
        s["positions"] = torch.arange(case["start"], case["start"] + t, device="cuda")
        s["inv_freq"] = _inv_freq(case["rotary"])
        return s
    q, kv, pages, s["table"], s["q_start"], s["kv_lens"] = _tables(case, seed)
    heads, page = case["kv_heads"], case["page"]
    nb = page // BLOCK
    s["pages"], s["max_q"], s["max_kv"] = pages, max(q), max(kv)

    def cached():
        return (normal(pages, heads, nb, dim * BLOCK) * 32).round_().clamp_(-127, 127).add_(128).to(torch.uint8)

    def scales(level):
        return level / 32 * (0.7 + 0.6 * torch.rand(pages, heads, nb, generator=g, device="cuda"))

    s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"] = cached(), cached(), scales(1.3), scales(0.8)
    t = sum(q)
    if op == "attention":
        s["q"] = normal(t, case["q_heads"], dim).to(kind)
        return s
    s["k"], s["v"] = (normal(t, heads, dim) * 1.7).to(kind), normal(t, heads, dim).to(kind)
    s["k_weight"] = weight() if case["norm"] else None
    s["inv_freq"] = _inv_freq(case["rotary"])
    before = np.asarray(kv) - np.asarray(q)
    s["positions"] = torch.from_numpy(np.concatenate([np.arange(b, m) for b, m in zip(before, kv)]).astype(np.int64)).cuda()
    # what the read-back covers: from the first touched block of each sequence to its end
    back = np.asarray(kv) - before // BLOCK * BLOCK
    s["back"] = int(back.sum())
    s["back_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(back)]).astype(np.int32)).cuda()
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------


def _norm_rotate(x, weight, positions, inv_freq, interleaved, eps=1e-6):
    """x: float32 [tokens, heads, dim]."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    if inv_freq is None:
        return x
    angle = positions.double()[:, None] * inv_freq.double()          # far positions: 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    n = inv_freq.numel()
    head, rest = x[..., : 2 * n], x[..., 2 * n:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :n], head[..., n:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _places(device):
    t = torch.arange(BLOCK, device=device)
    return (t & 3) | ((t >> 3 & 3) << 2) | ((t >> 2 & 1) << 4)


def _unpack_k(blocks, dim):
    """[..., dim * 32] bytes of K blocks -> [..., 32 tokens, dim] whole numbers in float32."""
    lead = blocks.shape[:-1]
    return blocks.view(*lead, dim // 16, BLOCK, 16).transpose(-3, -2).reshape(*lead, BLOCK, dim).float() - 128


def _unpack_v(blocks, dim):
    lead = blocks.shape[:-1]
    return blocks.view(*lead, dim, BLOCK)[..., _places(blocks.device)].transpose(-2, -1).float() - 128


def _pack_k(x):
    lead, dim = x.shape[:-2], x.shape[-1]
    return (x + 128).to(torch.uint8).view(*lead, BLOCK, dim // 16, 16).transpose(-3, -2).reshape(*lead, dim * BLOCK)


def _pack_v(x):
    lead, dim = x.shape[:-2], x.shape[-1]
    return (x + 128).to(torch.uint8).transpose(-2, -1)[..., _places(x.device).argsort()].reshape(*lead, dim * BLOCK)


def _rows(start, lens, total):
    """For each row of a ragged batch: its sequence and its place in the sequence's cached tokens."""
    row = torch.arange(total, device=start.device)
    seq = torch.searchsorted(start[1:].long(), row, right=True)
    return seq, row - start[seq + 1].long() + lens[seq].long()


def _append_one(cache, scale, x, page, blk, off, unpack, pack):
    """Appends x [tokens, heads, dim] (float32) to one of the two caches; the bytes of tokens behind it stay."""
    heads, nb = scale.shape[1:]
    dim = x.shape[-1]
    gb = page * nb + blk                                                                   # block of every token
    touched = torch.unique(gb)
    at = torch.searchsorted(touched, gb)
    tp, tb = touched // nb, touched % nb
    first = torch.full((touched.numel(),), BLOCK, device=x.device).scatter_reduce_(0, at, off, "amin")   # tokens kept: off < first
    amax = torch.zeros(touched.numel(), heads, device=x.device).scatter_reduce_(
        0, at[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    old = torch.where(first[:, None] > 0, scale[tp, :, tb], torch.zeros((), device=x.device))
    new = torch.maximum(old, amax / 127).clamp_min(FLOOR)
    whole = unpack(cache[tp, :, tb], dim)                                                   # [touched, heads, 32, dim]
    kept = torch.arange(BLOCK, device=x.device)[None, :] < first[:, None]
    whole = torch.where(kept[:, None, :, None], (whole * (old / new)[..., None, None]).round(), whole)
    whole[at, :, off] = (x / new[at][..., None]).round().clamp_(-127, 127)
    cache[tp, :, tb] = pack(whole)
    scale[tp, :, tb] = new


def _read_one(cache, scale, page, blk, off, unpack, dim):
    """[rows, heads, dim]: the tokens' values, whole blocks unpacked once each."""
    gb = page * scale.shape[2] + blk
    touched = torch.unique(gb)
    tp, tb = touched // scale.shape[2], touched % scale.shape[2]
    values = unpack(cache[tp, :, tb], dim) * scale[tp, :, tb][..., None, None]
    return values[torch.searchsorted(touched, gb), :, off]


def _where(s, start, total):
    seq, place = _rows(start, s["kv_lens"], total)
    page = s["table"][seq, place // s["case"]["page"]].long()
    return page, place % s["case"]["page"] // BLOCK, place % BLOCK


def _plain_append(s):
    case, kind = s["case"], KINDS[s["case"]["kind"]]
    dim = case["dim"]
    page, blk, off = _where(s, s["q_start"], s["k"].shape[0])
    k = _norm_rotate(s["k"].float(), s["k_weight"], s["positions"], s["inv_freq"], case["interleaved"])
    _append_one(s["k_cache"], s["k_scale"], k, page, blk, off, _unpack_k, _pack_k)
    _append_one(s["v_cache"], s["v_scale"], s["v"].float(), page, blk, off, _unpack_v, _pack_v)
    page, blk, off = _where(s, s["back_start"], s["back"])
    return {"k": _read_one(s["k_cache"], s["k_scale"], page, blk, off, _unpack_k, dim).to(kind),
            "v": _read_one(s["v_cache"], s["v_scale"], page, blk, off, _unpack_v, dim).to(kind),
            "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attention(s):
    case = s["case"]
    dim, hk, group, b = case["dim"], case["kv_heads"], case["q_heads"] // case["kv_heads"], case["batch"]
    total, max_q, max_kv = s["q"].shape[0], s["max_q"], s["max_kv"]
    pages = s["table"].long().clamp_min(0)                                                 # [b, n]
    shape = (b, hk, pages.shape[1] * case["page"], dim)

    def gathered(cache, scale, unpack):
        x = unpack(cache[pages], dim) * scale[pages][..., None, None]                      # [b, n, hk, nb, 32, dim]
        return x.transpose(1, 2).reshape(shape)[:, :, :max_kv]

    seq, place = _rows(s["q_start"], s["kv_lens"], total)
    row = torch.arange(total, device=seq.device) - s["q_start"][seq].long()
    q = torch.zeros(b, max_q, hk, group, dim, device=seq.device)
    q[seq, row] = s["q"].view(total, hk, group, dim).float()
    q = q.permute(0, 2, 1, 3, 4).reshape(b, hk, max_q * group, dim)
    scores = torch.matmul(q, gathered(s["k_cache"], s["k_scale"], _unpack_k).transpose(-2, -1)).mul_(1 / math.sqrt(dim))
    lens, n_q = s["kv_lens"].long(), s["q_start"].diff().long()
    at = (lens - n_q)[:, None] + torch.arange(max_q, device=seq.device)                   # [b, max_q]: a query's place
    key = torch.arange(max_kv, device=seq.device)
    hidden = key > at[..., None]
    if case["window"]:
        hidden |= key <= at[..., None] - case["window"]
    hidden |= key >= lens[:, None, None]
    scores.view(b, hk, max_q, group, max_kv).masked_fill_(hidden[:, None, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = scores.sub_(top).exp_()
    o = torch.matmul(p, gathered(s["v_cache"], s["v_scale"], _unpack_v)) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.view(b, hk, max_q, group, dim).permute(0, 2, 1, 3, 4)[seq, row]
    return o.reshape(total, case["q_heads"], dim).to(s["q"].dtype)


def _plain_sample(s):
    vocab = s["logits"].shape[1]
    temperature = s["temperature"].double()[:, None]
    greedy = temperature <= 0
    z, order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)     # ties: the lowest index first
    z = (z - z[:, :1]) / torch.where(greedy, 1.0, temperature)
    w = z.exp()
    place = torch.arange(vocab, device=w.device)
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab).long()[:, None]
    w = torch.where((place < k) & (~greedy | (place < 1)), w, 0.0)
    total = w.sum(-1, keepdim=True)
    before = w.cumsum(-1) - w
    w = torch.where((before < s["top_p"].double()[:, None] * total) | (s["top_p"][:, None] >= 1) | (place < 1), w, 0.0)
    w = torch.where(w >= s["min_p"].double()[:, None].clamp_max(1.0), w, 0.0)
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    total = w.sum(-1, keepdim=True)
    run_up = by_index.cumsum(-1)
    ids = ((run_up > s["uniform"].double()[:, None] * total) & (by_index > 0)).int().argmax(-1)
    return {"ids": ids.int(), "logprobs": (by_index.gather(1, ids[:, None]) / total).log().float()[:, 0]}


def _plain(s):
    case = s["case"]
    if case["op"] == "sample":
        return _plain_sample(s)
    if case["op"] == "append":
        return _plain_append(s)
    if case["op"] == "attention":
        return _plain_attention(s)
    t, hq, hk, dim = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
    q, k = s["qkv"][:, : hq * dim].view(t, hq, dim), s["qkv"][:, hq * dim: (hq + hk) * dim].view(t, hk, dim)
    return {"q": _norm_rotate(q.float(), s["q_weight"], s["positions"], s["inv_freq"], case["interleaved"]).to(q.dtype),
            "k": _norm_rotate(k.float(), s["k_weight"], s["positions"], s["inv_freq"], case["interleaved"]).to(k.dtype)}


# ---- the library's calls -----------------------------------------------------------------------------------------


def _ptr(x):
    return None if x is None else x.data_ptr()


def _workspace(s, nbytes):
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")
    return {"workspace_ptr": s["workspace"].data_ptr(), "workspace_bytes": s["workspace"].numel()}


def _own(s):
    case = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "sample":
        from hipengine_amd.kernels.hip_gfx950.sampling import sample_rows as S

        rows, vocab = s["logits"].shape
        ids = torch.empty(rows, dtype=torch.int32, device="cuda")
        logprobs = torch.empty(rows, device="cuda")
        S.sample_f32_rows_i32(s["logits"].data_ptr(), s["uniform"].data_ptr(), ids.data_ptr(), rows, vocab,
                              temperature_ptr=_ptr(s["temperature"]), top_k_ptr=_ptr(s["top_k"]), top_p_ptr=_ptr(s["top_p"]),
                              min_p_ptr=_ptr(s["min_p"]), out_logprobs_ptr=_ptr(logprobs), stream=stream,
                              **_workspace(s, S.sample_workspace_bytes(rows, vocab)))
        return {"ids": ids, "logprobs": logprobs}
    if case["op"] == "norm_rope":
        from hipengine_amd.kernels.hip_gfx950.attention import qk_norm_rope as R

        t, hq, hk, dim = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
        x = s["qkv"]
        q, k = torch.empty(t, hq, dim, dtype=x.dtype, device="cuda"), torch.empty(t, hk, dim, dtype=x.dtype, device="cuda")
        R.qk_norm_rope(x.data_ptr(), x.data_ptr() + hq * dim * x.element_size(), q.data_ptr(), k.data_ptr(), t, hq, hk, dim,
                       q_weight_ptr=_ptr(s["q_weight"]), k_weight_ptr=_ptr(s["k_weight"]), positions_ptr=_ptr(s["positions"]),
                       inv_freq_ptr=_ptr(s["inv_freq"]), rotary_dim=case["rotary"], interleaved=case["interleaved"],
                       in_kind=case["kind"], out_kind=case["kind"], q_stride=x.stride(0), k_stride=x.stride(0), stream=stream)
        return {"q": q, "k": k}
    from hipengine_amd.kernels.hip_gfx950.attention import kv_cache_q8 as C

    cache = C.KVCacheQ8(s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), s["k_scale"].data_ptr(), s["v_scale"].data_ptr(),
                        s["pages"], case["page"], case["kv_heads"], case["dim"])
    table = (s["table"].data_ptr(), s["table"].stride(0))
    if case["op"] == "append":
        k, v = s["k"], s["v"]
        C.kv_append_q8(cache, k.data_ptr(), v.data_ptr(), *table, s["q_start"].data_ptr(), s["kv_lens"].data_ptr(), k.shape[0],
                       case["batch"], s["max_q"], k_weight_ptr=_ptr(s["k_weight"]), positions_ptr=_ptr(s["positions"]),
                       inv_freq_ptr=_ptr(s["inv_freq"]), rotary_dim=case["rotary"], interleaved=case["interleaved"],
                       in_kind=case["kind"], stream=stream)
        ko = torch.empty(s["back"], *k.shape[1:], dtype=k.dtype, device="cuda")
        vo = torch.empty_like(ko)
        C.kv_read_q8(cache, ko.data_ptr(), vo.data_ptr(), *table, s["back_start"].data_ptr(), s["kv_lens"].data_ptr(), s["back"],
                     case["batch"], out_kind=case["kind"], stream=stream)
        return {"k": ko, "v": vo, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    from hipengine_amd.kernels.hip_gfx950.attention import paged_attention_q8 as A

    q = s["q"]
    out = torch.empty_like(q)
    shape = (q.shape[0], case["batch"], s["max_q"], s["max_kv"], case["q_heads"])
    A.paged_attention_q8(cache, q.data_ptr(), out.data_ptr(), *table, s["q_start"].data_ptr(), s["kv_lens"].data_ptr(), *shape,
                         window=case["window"], kind=case["kind"], stream=stream,
                         **_workspace(s, A.paged_attention_q8_workspace_bytes(*shape, case["kv_heads"], case["dim"])))
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------


def _exact_turn(x, weight, positions, inv_freq, interleaved):
    x = x.double()
    if weight is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * weight.double()
    if inv_freq is None:
        return x
    n = inv_freq.numel()
    i = torch.arange(n, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    t = torch.outer(positions.double(), inv_freq.double()).unsqueeze(1)
    y = x.clone()
    z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.ones_like(t), t)
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_block(cache, scale, page, head, blk, dim, is_v):
    raw = cache[page, head, blk].cpu().numpy().astype(np.float64) - 128.0
    if is_v:
        t = np.arange(BLOCK)
        return raw.reshape(dim, 2, 4, 4)[:, t // 4 % 2, t // 8, t % 4].T.copy()
    return raw.reshape(dim // 16, BLOCK, 16).swapaxes(0, 1).reshape(BLOCK, dim).copy()


def _exact_append(s, case):
    q, kv = _shape(case)
    if sum(q) * case["kv_heads"] * case["dim"] > 1 << 24:
        return None
    table, page = s["table"].cpu().numpy(), case["page"]
    out = {}
    for key in ("k", "v"):
        x = s[key].double() if key == "v" else _exact_turn(s["k"], s["k_weight"], s["positions"], s["inv_freq"], case["interleaved"])
        x = x.cpu().numpy()
        scale = s[key + "_scale"].double().cpu().numpy()
        rows, at = [], 0
        for i, (n, m) in enumerate(zip(q, kv)):
            lo = m - n
            for b0 in range(lo // BLOCK * BLOCK, m, BLOCK):
                first, last = max(lo, b0), min(m, b0 + BLOCK)
                pg, blk = int(table[i, b0 // page]), b0 % page // BLOCK
                got = np.zeros((last - b0, case["kv_heads"], case["dim"]))
                for h in range(case["kv_heads"]):
                    new = x[at + first - lo: at + last - lo, h]
                    was = scale[pg, h, blk] if first > b0 else 0.0
                    now = max(was, np.abs(new).max() / 127.0, FLOOR)
                    if first > b0:
                        got[: first - b0, h] = np.rint(_exact_block(s[key + "_cache"], scale, pg, h, blk, case["dim"], key == "v")[: first - b0] * (was / now)) * now
                    got[first - b0:, h] = np.clip(np.rint(new / now), -127, 127) * now
                    scale[pg, h, blk] = now
                rows.append(got)
            at += n
        out[key] = torch.from_numpy(np.concatenate(rows))
        out[key + "_scale"] = torch.from_numpy(scale)
    return out


def _exact_attention(s, case):
    q, kv = _shape(case)
    if work(case)["flops"] > 2e12:
        return None
    dim, page, hk = case["dim"], case["page"], case["kv_heads"]
    group = case["q_heads"] // hk
    place = torch.tensor([[16 * (t >> 2 & 1) + 4 * (t >> 3) + (t & 3)] for t in range(BLOCK)]).flatten().cuda()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, m) in enumerate(zip(q, kv)):
        pages = s["table"][i, : (m + page - 1) // page].long()
        key = torch.arange(m, device="cuda")
        me = torch.arange(m - n, m, device="cuda")[:, None]
        seen = (key <= me) & ((key > me - case["window"]) if case["window"] else True)
        for h in range(hk):
            k = s["k_cache"][pages, h].double().view(-1, dim // 16, BLOCK, 16).permute(0, 2, 1, 3).reshape(-1, BLOCK, dim) - 128
            v = s["v_cache"][pages, h].double().view(-1, dim, BLOCK)[:, :, place].permute(0, 2, 1) - 128
            k = (k * s["k_scale"][pages, h].double().view(-1, 1, 1)).reshape(-1, dim)[:m]
            v = (v * s["v_scale"][pages, h].double().view(-1, 1, 1)).reshape(-1, dim)[:m]
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][at: at + n, j].double() @ k.T / dim ** 0.5).masked_fill(~seen, -math.inf)
                out[at: at + n, j] = torch.softmax(score, -1) @ v
        at += n
    return out


def _exact_sample(s):
    logits = s["logits"].cpu().numpy().astype(np.float64)
    set_ = {k: s[k].cpu().numpy().astype(np.float64) for k in ("uniform", "temperature", "top_k", "top_p", "min_p")}
    ids, logprobs = [], []
    for r, row in enumerate(logits):
        order = np.lexsort((np.arange(row.size), -row))
        if set_["temperature"][r] <= 0:
            order = order[:1]
        elif set_["top_k"][r] > 0:
            order = order[: int(set_["top_k"][r])]
        p = np.exp((row[order] - row[order[0]]) / (set_["temperature"][r] if set_["temperature"][r] > 0 else 1.0))
        if set_["top_p"][r] < 1:
            keep = 1 + int(np.searchsorted(np.cumsum(p), set_["top_p"][r] * p.sum(), side="left"))
            order, p = order[:keep], p[:keep]
        order, p = order[p >= min(1.0, set_["min_p"][r])], p[p >= min(1.0, set_["min_p"][r])]
        up = np.argsort(order)
        order, p = order[up], p[up]
        j = min(int(np.searchsorted(np.cumsum(p), set_["uniform"][r] * p.sum(), side="right")), p.size - 1)
        ids.append(order[j])
        logprobs.append(math.log(p[j] / p.sum()))
    return {"ids": torch.tensor(ids, dtype=torch.int32), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["op"] == "attention":
        return _exact_attention(s, case)
    t, hq, hk, dim = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
    x = s["qkv"].view(t, hq + 2 * hk, dim)
    return {"q": _exact_turn(x[:, :hq], s["q_weight"], s["positions"], s["inv_freq"], case["interleaved"]),
            "k": _exact_turn(x[:, hq: hq + hk], s["k_weight"], s["positions"], s["inv_freq"], case["interleaved"])}
