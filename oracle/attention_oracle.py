"""Plain float64 NumPy statements of the attention operators and of sampling, for the tests.

Caches are held here as whole numbers ``[pages, heads, page_size, dim]`` (int64) with scales ``[pages, heads, page_size /
32]`` and brought to and from the byte layout of the library by ``pack_cache`` / ``unpack_cache``.
"""

from __future__ import annotations

import numpy as np

BLOCK = 32
FLOOR = 2.0 ** -64
U = 2.0 ** -24                       # half a step of float32, relative
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def to_bits(x: np.ndarray, kind: str) -> np.ndarray:
    """Round float64 / float32 values to `kind` and return what goes to the device."""
    x = np.asarray(x, dtype=np.float32)
    if kind == "f32":
        return x
    if kind == "fp16":
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b: np.ndarray, kind: str) -> np.ndarray:
    if kind == "f32":
        return b.astype(np.float64)
    if kind == "fp16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def round_to(x: np.ndarray, kind: str) -> np.ndarray:
    return from_bits(to_bits(x, kind), kind)


def place(t):
    return (t & 3) | ((t >> 3 & 3) << 2) | ((t >> 2 & 1) << 4)


def pack_cache(k: np.ndarray, v: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    pages, heads, size, dim = k.shape
    nb = size // BLOCK
    kb = (k + 128).astype(np.uint8).reshape(pages, heads, nb, BLOCK, dim // 16, 16).swapaxes(3, 4)
    vb = np.empty((pages, heads, nb, dim, BLOCK), np.uint8)
    vb[..., place(np.arange(BLOCK))] = (v + 128).astype(np.uint8).reshape(pages, heads, nb, BLOCK, dim).swapaxes(3, 4)
    return np.ascontiguousarray(kb).reshape(pages, heads, nb, -1), vb.reshape(pages, heads, nb, -1)


def unpack_cache(kb: np.ndarray, vb: np.ndarray, dim: int) -> tuple[np.ndarray, np.ndarray]:
    pages, heads, nb = kb.shape[:3]
    k = kb.reshape(pages, heads, nb, dim // 16, BLOCK, 16).swapaxes(3, 4).reshape(pages, heads, nb * BLOCK, dim)
    v = vb.reshape(pages, heads, nb, dim, BLOCK)[..., place(np.arange(BLOCK))].swapaxes(3, 4).reshape(pages, heads, nb * BLOCK, dim)
    return k.astype(np.int64) - 128, v.astype(np.int64) - 128


def norm_rotate(x, weight, positions, inv_freq, *, eps=1e-6, interleaved=False, rope_scale=1.0):
    """(value, magnitude): the operator on x [tokens, heads, dim], and for each value the sum of the magnitudes of the
    terms that it is the sum of (what its rounding errors are relative to)."""
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    y, mag = x.copy(), np.abs(x)
    if inv_freq is not None:
        n = len(inv_freq)
        t = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)[None, :]
        c, s = (np.cos(t) * rope_scale)[:, None], (np.sin(t) * rope_scale)[:, None]
        i = np.arange(n)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        xa, xb = x[..., a], x[..., b]
        y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
        mag[..., a] = mag[..., b] = (np.abs(xa) + np.abs(xb)) * abs(rope_scale)
    return y, mag


def rows_of(q_start, kv_lens, b):
    """(first row, rows, place of the first row) of sequence b."""
    n = int(q_start[b + 1] - q_start[b])
    return int(q_start[b]), n, int(kv_lens[b]) - n


def append(k, v, k_int, v_int, k_scale, v_scale, table, q_start, kv_lens):
    """Appends float64 k, v [tokens, heads, dim] in place. Returns the unrounded quotients ``{(page, head, which):
    (places, x / scale)}`` of every byte that the call determines, for a test of roundings."""
    page_size = k_int.shape[2]
    touched = {}
    for which, (x, ints, scales) in enumerate(((k, k_int, k_scale), (v, v_int, v_scale))):
        for b in range(len(kv_lens)):
            row, n, at = rows_of(q_start, kv_lens, b)
            lo, hi = max(at, 0), int(kv_lens[b])
            for base in range(lo // BLOCK * BLOCK, hi, BLOCK):
                first, last = max(lo, base), min(hi, base + BLOCK)
                slot = base // page_size
                page = int(table[b, slot]) if slot < table.shape[1] else -1
                if first >= last or not 0 <= page < ints.shape[0]:
                    continue
                off = base % page_size
                for h in range(ints.shape[1]):
                    new = x[row + first - at: row + last - at, h]
                    old = float(counts_as(scales[page, h, off // BLOCK])) if first > base else 0.0
                    with np.errstate(invalid="ignore"):
                        bad = not np.isfinite(new).all() or np.isnan(old)
                        scale = np.nan if bad else max(old, np.abs(new).max() / 127.0, FLOOR)
                    scales[page, h, off // BLOCK] = scale
                    if bad:
                        continue
                    kept = ints[page, h, off: off + first - base]
                    quotients = np.concatenate([kept * (old / scale), new / scale])
                    if old == scale:
                        quotients[: first - base] = kept
                    ints[page, h, off: off + last - base] = np.clip(np.rint(quotients), -127, 127)
                    touched[(page, h, off, which)] = quotients
    return touched


def counts_as(scale):
    """A block's scale as it counts: at least FLOOR; a NaN stays one."""
    return np.where(scale < FLOOR, FLOOR, scale)


def gather(ints, scales, table_row, length):
    """The cached values of a sequence [heads, length, dim] and which of its tokens are there."""
    pages, heads, size, dim = ints.shape
    out, there = np.zeros((heads, length, dim)), np.zeros(length, bool)
    for slot in range((length + size - 1) // size):
        page = int(table_row[slot]) if slot < len(table_row) else -1
        a, b = slot * size, min(length, (slot + 1) * size)
        if 0 <= page < pages:
            out[:, a:b] = (ints[page] * np.repeat(counts_as(scales[page]), BLOCK, axis=1)[..., None])[:, : b - a]
            there[a:b] = True
    return out, there


def attention(q, k_int, v_int, k_scale, v_scale, table, q_start, kv_lens, *, scale, window=0):
    """(out, deviation, magnitude, argument error per unit) of q [tokens, q_heads, dim]: the attention, sum p |v - o|, sum
    p |v|, and the largest sum |q k| * scale of a visible key, all float64, for rows that belong to a sequence."""
    heads, dim = k_int.shape[1], q.shape[-1]
    group = q.shape[1] // heads
    out, dev, mag, arg = (np.zeros(q.shape) for _ in range(4))
    for b in range(len(kv_lens)):
        row, n, at = rows_of(q_start, kv_lens, b)
        m = int(kv_lens[b])
        if n == 0 or m <= 0:
            continue
        ks, there = gather(k_int, k_scale, table[b], m)
        vs, _ = gather(v_int, v_scale, table[b], m)
        me, key = at + np.arange(n)[:, None], np.arange(m)[None, :]
        seen = (key <= me) & there
        if window:
            seen &= key > me - window
        for h in range(q.shape[1]):
            kk, vv = ks[h // group], vs[h // group]
            x = q[row: row + n, h]
            s = np.where(seen, x @ kk.T * scale, -np.inf)
            top = s.max(-1, keepdims=True)
            p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
            total = p.sum(-1, keepdims=True)
            p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
            o = p @ vv
            out[row: row + n, h] = o
            mag[row: row + n, h] = p @ np.abs(vv)
            for i in range(n):
                dev[row + i, h] = p[i] @ np.abs(vv - o[i])
            arg[row: row + n, h] = np.where(seen, np.abs(x) @ np.abs(kk).T * scale, 0.0).max(-1, keepdims=True)
    return out, dev, mag, arg


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, accuracy=0.0):
    """{id: (lowest, highest log-probability)} of one row: with accuracy 0 the one token of the definition. With accuracy e
    every token that it gives if prefix sums (around top-p's border, and around the token's) are moved by up to e of
    themselves, and min-p by 2^-20 of that: what such arithmetic may answer, nearly always one token too."""
    l = np.minimum(np.asarray(logits, np.float64) + 0.0, np.finfo(np.float32).max)
    there = np.flatnonzero(~np.isnan(l) & (l > -np.inf))
    if not there.size:
        return {-1: (-np.inf, -np.inf)}
    order = there[np.lexsort((there, -l[there]))]
    if not temperature > 0:
        return {int(order[0]): (0.0, 0.0)}
    temperature = max(float(temperature), 2.0 ** -124)
    if top_k > 0:
        order = order[:top_k]
    w = np.exp(np.maximum((l[order] - l[order[0]]) / np.float64(temperature), -5000))
    u = min(float(uniform), 1.0) if uniform > 0 else 0.0
    cum, found = np.cumsum(w), {}
    for a in {-accuracy, 0.0, accuracy}:
        n = 1 + int(np.sum(cum[:-1] < max(float(top_p), 0.0) * cum[-1] * (1 + a))) if top_p < 1 else len(w)
        for b in {-accuracy, 0.0, accuracy}:
            m = min(float(min_p), 1.0) * (1 + b * 2.0 ** -20) if min_p > 0 else 0.0   # (an argument in float64 decides)
            keep = (np.arange(len(w)) < n) & ((w >= m) | (w == 1))
            ids, v = order[keep], w[keep]
            by = np.argsort(ids)
            ids, v = ids[by], v[by]
            run = np.cumsum(v)
            for c in {-accuracy, 0.0, accuracy}:
                i = min(int(np.searchsorted(run, (u + c) * run[-1], side="right")), len(v) - 1)
                while v[i] == 0:
                    i -= 1
                p = float(np.log(v[i]) - np.log(run[-1]))
                lo, hi = found.get(int(ids[i]), (p, p))
                found[int(ids[i])] = (min(lo, p), max(hi, p))
    return found
