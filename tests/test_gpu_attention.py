"""The attention operators on one MI355X against their float64 statements (oracle/attention_oracle.py), through the raw
pointer wrappers. Every tolerance is a sum of the roundings of the arithmetic in question; U is half a float32 step."""

from __future__ import annotations

import numpy as np
import pytest

from hipengine_amd.core.hip import HipError
from hipengine_amd.kernels.hip_gfx950.attention import kv_cache_q8 as C
from hipengine_amd.kernels.hip_gfx950.attention import paged_attention_q8 as A
from hipengine_amd.kernels.hip_gfx950.attention import qk_norm_rope as R
from oracle import attention_oracle as O

pytestmark = pytest.mark.gpu

U = O.U
# Roundings of a normed, rotated value, in U of the magnitude of its terms: the sum of squares (8 in a lane, 5 levels) and
# the mean at half weight 7, eps, root and quotient 2, two products 2, the fraction of a turn 2 pi, cos and sin 2, the
# product and the fma 2: 21.3, and never more than this:
NORM_ROPE = 24 * U
ITEM = {"f32": 4, "bf16": 2, "fp16": 2}
NP = {"f32": np.float32, "bf16": np.uint16, "fp16": np.uint16}


def inv_freq(rotary, theta=1e6):
    return (theta ** (-np.arange(0, rotary, 2) / rotary)).astype(np.float32)


# ---- q / k norm and rotation ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,interleaved,kind,out,start", [
    (1, 40, 8, 128, 128, False, "bf16", "bf16", 40961),
    (3, 5, 1, 64, 64, False, "f32", "f32", 1000003),
    (7, 16, 2, 256, 64, False, "fp16", "fp16", 5),
    (2, 3, 3, 128, 32, True, "f32", "f32", 262143),
    (33, 9, 1, 64, 16, True, "bf16", "f32", 0),
    (5, 64, 16, 256, 256, False, "f32", "bf16", 77),      # more heads than one pass of a workgroup holds
    (4, 8, 0, 128, 128, False, "bf16", "fp16", 9),        # only queries
    (4, 0, 8, 128, 0, False, "fp16", "f32", 0),           # only keys, no rotation
    (3, 1, 0, 256, 256, False, "bf16", "f32", 12345),     # more pairs than lanes that hold the heads
    (2, 1, 1, 256, 144, True, "f32", "bf16", 99),
    (5, 1, 0, 64, 64, False, "bf16", "bf16", 31),
])
def test_qk_norm_rope(dev, tokens, hq, hk, dim, rotary, interleaved, kind, out, start):
    rng = np.random.default_rng(tokens * 131 + dim + hq)
    width = (hq + 2 * hk) * dim + 24                       # columns of a wider matrix
    x = O.round_to(rng.standard_normal((tokens, width)) * 1.7, kind)
    qw, kw = (rng.uniform(0.5, 1.5, dim).astype(np.float32) for _ in range(2))
    pos = start + rng.permutation(tokens).astype(np.int64) * 17
    freq = inv_freq(rotary) if rotary else None
    dx, dqw, dkw, dpos = dev.put(O.to_bits(x, kind)), dev.put(qw), dev.put(kw), dev.put(pos)
    df = dev.put(freq) if rotary else None
    pad = 8                                                # padded output rows, whose padding must stay
    bufs = [dev.empty(tokens * (h * dim + pad) * ITEM[out]) for h in (hq, hk)]
    R.qk_norm_rope(dx.ptr, dx.ptr + hq * dim * ITEM[kind], bufs[0].ptr, bufs[1].ptr, tokens, hq, hk, dim,
                   q_weight_ptr=dqw.ptr, k_weight_ptr=dkw.ptr, positions_ptr=dpos.ptr, inv_freq_ptr=df.ptr if df else None,
                   rotary_dim=rotary, interleaved=interleaved, in_kind=kind, out_kind=out, q_stride=width, k_stride=width,
                   q_out_stride=hq * dim + pad, k_out_stride=hk * dim + pad, rope_scale=1.25)
    for h, w, c0, buf in ((hq, qw, 0, bufs[0]), (hk, kw, hq * dim, bufs[1])):
        raw = dev.get(buf, NP[out], (tokens, h * dim + pad))
        assert (raw[:, h * dim:].view(np.uint8) == 0xA5).all()
        if not h:
            continue
        got = O.from_bits(np.ascontiguousarray(raw[:, : h * dim]), out).reshape(tokens, h, dim)
        want, mag = O.norm_rotate(x[:, c0: c0 + h * dim].reshape(tokens, h, dim), w, pos, freq, interleaved=interleaved,
                                  rope_scale=1.25)
        tol = NORM_ROPE * mag + O.HALF_STEP[out] * (np.abs(want) + NORM_ROPE * mag) + (2.0 ** -25 if out == "fp16" else 0)
        assert (np.abs(got - want) <= tol).all()
    dev.free(dx, dqw, dkw, dpos, *bufs, *([df] if df else []))


def test_qk_norm_rope_in_place_and_without_norm(dev):
    rng = np.random.default_rng(5)
    t, hq, hk, dim = 6, 4, 2, 128
    x = O.round_to(rng.standard_normal((t, hq + hk, dim)), "bf16")
    pos, freq = np.arange(t, dtype=np.int64) + 3, inv_freq(dim)
    dx, dpos, df = dev.put(O.to_bits(x, "bf16")), dev.put(pos), dev.put(freq)
    k = dx.ptr + hq * dim * 2
    s = (hq + hk) * dim
    R.qk_norm_rope(dx.ptr, k, dx.ptr, k, t, hq, hk, dim, positions_ptr=dpos.ptr, inv_freq_ptr=df.ptr, rotary_dim=dim,
                   q_stride=s, k_stride=s, q_out_stride=s, k_out_stride=s)
    got = O.from_bits(dev.get(dx, np.uint16, x.shape), "bf16")
    want, mag = O.norm_rotate(x, None, pos, freq)
    assert (np.abs(got - want) <= NORM_ROPE * mag + 2.0 ** -8 * (np.abs(want) + NORM_ROPE * mag)).all()
    dev.free(dx, dpos, df)


def test_qk_norm_rope_odd_alignment(dev):
    """Rows that begin at odd multiples of the element: the vector accesses need no more than that."""
    rng = np.random.default_rng(6)
    t, h, dim = 3, 2, 64
    x = O.round_to(rng.standard_normal(1 + t * (h * dim + 3)), "bf16")
    w = rng.uniform(0.5, 1.5, dim).astype(np.float32)
    dx, dw, out = dev.put(O.to_bits(x, "bf16")), dev.put(np.concatenate([[0], w]).astype(np.float32)), dev.empty(2 + t * (h * dim + 1) * 2)
    R.qk_norm_rope(dx.ptr + 2, None, out.ptr + 2, None, t, h, 0, dim, q_weight_ptr=dw.ptr + 4, q_stride=h * dim + 3,
                   q_out_stride=h * dim + 1)
    got = O.from_bits(dev.get(out, np.uint16, (1 + t * (h * dim + 1),))[1:].reshape(t, -1)[:, : h * dim].copy(), "bf16").reshape(t, h, dim)
    want, mag = O.norm_rotate(x[1:].reshape(t, -1)[:, : h * dim].reshape(t, h, dim), w, None, None)
    assert (np.abs(got - want) <= NORM_ROPE * mag + 2.0 ** -8 * (np.abs(want) + NORM_ROPE * mag)).all()
    dev.free(dx, dw, out)


# ---- the cache -----------------------------------------------------------------------------------------------------


class Cache:
    """A cache on the device and its float64 statement beside it."""

    def __init__(self, dev, rng, kv_lens, page, heads, dim, spare=2, stride=None):
        self.dev, self.page, self.heads, self.dim = dev, page, heads, dim
        need = [(max(int(n), 0) + page - 1) // page for n in kv_lens]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(kv_lens), stride or max(max(need), 1)), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at: at + n]
            at += n
        shape = (self.pages, heads, page, dim)
        self.k, self.v = (np.clip(np.rint(rng.standard_normal(shape) * 32), -127, 127).astype(np.int64) for _ in range(2))
        self.ks, self.vs = (rng.uniform(0.02, 0.06, (self.pages, heads, page // 32)).astype(np.float32).astype(np.float64) for _ in range(2))
        self.upload()

    def upload(self):
        kb, vb = O.pack_cache(self.k, self.v)
        put = self.dev.put
        self.bufs = [put(kb), put(vb), put(self.ks.astype(np.float32)), put(self.vs.astype(np.float32)), put(self.table)]
        self.handle = C.KVCacheQ8(*(b.ptr for b in self.bufs[:4]), self.pages, self.page, self.heads, self.dim)

    def download(self):
        n = self.page // 32
        kb, vb = (self.dev.get(b, np.uint8, (self.pages, self.heads, n, self.dim * 32)) for b in self.bufs[:2])
        ks, vs = (self.dev.get(b, np.float32, (self.pages, self.heads, n)) for b in self.bufs[2:4])
        return *O.unpack_cache(kb, vb, self.dim), ks, vs

    @property
    def where(self):
        return self.bufs[4].ptr, self.table.shape[1]

    def free(self):
        self.dev.free(*self.bufs)


APPEND = [
    # dim, heads, page, rows, lengths behind the call, kind
    (128, 8, 64, [1, 1, 1], [1, 33, 64], "bf16"),
    (64, 2, 32, [1, 0, 5, 40], [32, 7, 5, 71], "fp16"),
    (256, 1, 128, [33, 64, 31], [33, 200, 63], "bf16"),
    (128, 3, 64, [100, 3], [163, 3], "f32"),
    (64, 1, 1024, [2, 2, 2, 2, 2], [2, 1000, 31, 32, 33], "f32"),
    (128, 2, 32, [1] * 70, list(range(1, 71)), "bf16"),
    (128, 2, 64, [3, 260] + [1] * 300, [2, 260] + [9] * 300, "bf16"),     # more rows than tokens; more sequences than threads
]


def _ragged(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


@pytest.mark.parametrize("dim,heads,page,rows,lens,kind", APPEND)
def test_append_without_norm_or_rotation_is_exact(dev, dim, heads, page, rows, lens, kind):
    """Scale and bytes are float32 expressions of the inputs and the cache: equal to the same expressions here."""
    rng = np.random.default_rng(dim + heads + len(rows))
    c = Cache(dev, rng, lens, page, heads, dim)
    t, start, kv = sum(rows), _ragged(rows), np.array(lens, np.int32)
    k, v = (O.round_to(rng.standard_normal((t + 1, heads, dim)) * rng.choice([0.3, 1.0, 3.0], (t + 1, 1, 1)), kind) for _ in range(2))
    bufs = [dev.put(O.to_bits(k, kind)), dev.put(O.to_bits(v, kind)), dev.put(start), dev.put(kv)]
    C.kv_append_q8(c.handle, bufs[0].ptr, bufs[1].ptr, *c.where, bufs[2].ptr, bufs[3].ptr, t, len(rows), max(rows), in_kind=kind)
    gk, gv, gks, gvs = c.download()
    f = np.float32
    for x, ints, scales, g, gs in ((k, c.k, c.ks, gk, gks), (v, c.v, c.vs, gv, gvs)):
        for b in range(len(rows)):
            row, n, at = O.rows_of(start, kv, b)
            lo, hi = max(at, 0), int(kv[b])
            for base in range(lo // 32 * 32, hi if n else 0, 32):
                first, last = max(lo, base), min(hi, base + 32)
                pg, off = c.table[b, base // page], base % page
                for h in range(heads):
                    new = x[row + first - at: row + last - at, h].astype(f)
                    old = f(scales[pg, h, off // 32]) if first > base else f(0)
                    scale = max(old, np.abs(new).max() / f(127), f(O.FLOOR))
                    kept = ints[pg, h, off: off + first - base]
                    if scale != old:
                        kept = np.rint(kept.astype(f) * (old / scale))
                    ints[pg, h, off: off + first - base] = kept
                    ints[pg, h, off + first - base: off + last - base] = np.clip(np.rint(new / scale), -127, 127)
                    scales[pg, h, off // 32] = scale
        assert np.array_equal(gs, scales.astype(f))
        assert np.array_equal(g, ints)                    # whole cache: other pages and bytes behind the tokens too
    dev.free(*bufs)
    c.free()


@pytest.mark.parametrize("dim,heads,page,rows,lens,kind", APPEND)
@pytest.mark.parametrize("rotary,interleaved,norm", [(1.0, False, True), (0.25, True, True), (0.5, False, False)])
def test_append_with_norm_and_rotation(dev, dim, heads, page, rows, lens, kind, rotary, interleaved, norm):
    rng = np.random.default_rng(dim * 3 + heads + len(rows))
    rotary = int(dim * rotary)
    c = Cache(dev, rng, lens, page, heads, dim)
    t, start, kv = sum(rows), _ragged(rows), np.array(lens, np.int32)
    width = heads * dim + 40
    k, v = (O.round_to(rng.standard_normal((t, width)) * 1.5, kind) for _ in range(2))
    w = rng.uniform(0.5, 1.5, dim).astype(np.float32) if norm else None
    pos = np.concatenate([np.arange(m - n, m) for n, m in zip(rows, lens)]).astype(np.int64) + (100000 if norm else 0)
    freq = inv_freq(rotary)
    bufs = [dev.put(O.to_bits(k, kind)), dev.put(O.to_bits(v, kind)), dev.put(start), dev.put(kv), dev.put(pos), dev.put(freq)]
    if norm:
        bufs.append(dev.put(w))
    C.kv_append_q8(c.handle, bufs[0].ptr, bufs[1].ptr, *c.where, bufs[2].ptr, bufs[3].ptr, t, len(rows), max(rows) + 5, in_kind=kind,
                   k_weight_ptr=bufs[6].ptr if norm else None, positions_ptr=bufs[4].ptr if norm else None,
                   inv_freq_ptr=bufs[5].ptr, rotary_dim=rotary, interleaved=interleaved, k_stride=width, v_stride=width)
    gk, gv, gks, gvs = c.download()
    cut = lambda x: x[:, : heads * dim].reshape(t, heads, dim)  # noqa: E731
    turned, _ = O.norm_rotate(cut(k), w, pos, freq, interleaved=interleaved)
    untouched = [a.copy() for a in (c.k, c.v)]
    quotients = O.append(turned, cut(v), c.k, c.v, c.ks, c.vs, c.table, start, kv)
    # the scale is a value over 127: a value of a pair is at least half of the pair's terms' magnitude where it is the
    # largest, so 2 NORM_ROPE relative, and the division
    for g, want in ((gks, c.ks), (gvs, c.vs)):
        assert (np.abs(g - want) <= (2 * NORM_ROPE + 2 * U) * np.abs(want)).all()
    # a byte is off by at most the rounding to whole numbers and its quotient's error: 127 times that of value and scale
    slack = 127 * (4 * NORM_ROPE + 6 * U)
    for (page_, h, off, which), x in quotients.items():
        got = (gk, gv)[which][page_, h, off: off + len(x)]
        assert (np.abs(got - x) <= 0.5 + slack).all()
        untouched[which][page_, h, off: off + len(x)] = got
    assert np.array_equal(untouched[0], gk) and np.array_equal(untouched[1], gv)
    dev.free(*bufs)
    c.free()


@pytest.mark.parametrize("kind", ["f32", "bf16", "fp16"])
def test_read_back(dev, kind):
    rng = np.random.default_rng(3)
    rows, lens, dim, heads, page = [5, 0, 33, 70, 1, 3], [5, 40, 65, 70, 96, 2], 64, 3, 32
    c = Cache(dev, rng, lens, page, heads, dim)
    c.table[3, 1] = c.pages                               # a page that is not there reads as zeros
    c.table[4, 2] = -7
    dev.free(*c.bufs)
    c.upload()
    t, start, kv = sum(rows), _ragged(rows), np.array(lens, np.int32)
    stride = heads * dim + 8
    bufs = [dev.put(start), dev.put(kv), dev.empty((t + 2) * stride * ITEM[kind]), dev.empty((t + 2) * stride * ITEM[kind])]
    C.kv_read_q8(c.handle, bufs[2].ptr, bufs[3].ptr, *c.where, bufs[0].ptr, bufs[1].ptr, t, len(rows), out_kind=kind,
                 k_out_stride=stride, v_out_stride=stride)
    for buf, ints, scales in ((bufs[2], c.k, c.ks), (bufs[3], c.v, c.vs)):
        raw = dev.get(buf, NP[kind], (t + 2, stride))
        fill = np.frombuffer(b"\xa5" * 4, NP[kind])[0]
        same = raw.view(np.uint32 if kind == "f32" else np.uint16) == np.array(fill).view(np.uint32 if kind == "f32" else np.uint16)
        assert same[t:].all() and same[:, heads * dim:].all()
        for b in range(len(rows)):
            row, n, at = O.rows_of(start, kv, b)
            values, _ = O.gather(ints, scales, c.table[b], lens[b])
            skip = max(-at, 0)                             # rows at negative places stay as they were
            assert same[row: row + skip].all()
            got = raw[row + skip: row + n, : heads * dim]
            want = O.to_bits((values.astype(np.float32))[:, max(at, 0):].swapaxes(0, 1).reshape(n - skip, heads * dim), kind)
            assert np.array_equal(got, want)
    # one output alone
    C.kv_read_q8(c.handle, None, bufs[3].ptr, *c.where, bufs[0].ptr, bufs[1].ptr, t, len(rows), out_kind=kind)
    dev.sync()
    dev.free(*bufs)
    c.free()


def test_append_token_by_token_follows_the_statement(dev):
    """70 calls of one token each: blocks start anew over stale pages, scales grow and earlier tokens are rescaled."""
    rng = np.random.default_rng(8)
    dim, heads, page, n = 128, 2, 32, 70
    c = Cache(dev, rng, [n], page, heads, dim)
    k, v = (O.round_to(rng.standard_normal((n, heads, dim)) * np.linspace(0.2, 4, n)[:, None, None], "f32") for _ in range(2))
    start = dev.put(np.array([0, 1], np.int32))
    f = np.float32
    for i in range(n):
        bufs = [dev.put(k[i].astype(f)), dev.put(v[i].astype(f)), dev.put(np.array([i + 1], np.int32))]
        C.kv_append_q8(c.handle, bufs[0].ptr, bufs[1].ptr, *c.where, start.ptr, bufs[2].ptr, 1, 1, 1, in_kind="f32")
        dev.sync()
        dev.free(*bufs)
        for x, ints, scales in ((k, c.k, c.ks), (v, c.v, c.vs)):
            pg, o = c.table[0, i // 32], i % 32
            for h in range(heads):
                old = f(scales[pg, h, 0]) if o else f(0)
                new = x[i, h].astype(f)
                scale = max(old, np.abs(new).max() / f(127))
                if scale != old:
                    ints[pg, h, :o] = np.rint(ints[pg, h, :o].astype(f) * (old / scale))
                ints[pg, h, o] = np.rint(new / scale)
                scales[pg, h, 0] = scale
    gk, gv, gks, gvs = c.download()
    assert np.array_equal(gks, c.ks.astype(f)) and np.array_equal(gvs, c.vs.astype(f))
    assert np.array_equal(gk, c.k) and np.array_equal(gv, c.v)
    dev.free(start)
    c.free()


def test_append_nonfinite_bad_pages_and_zeros(dev):
    rng = np.random.default_rng(9)
    dim, heads, page = 64, 2, 32
    rows, lens = [40, 2, 3, 32], [40, 34, 3, 32]
    c = Cache(dev, rng, lens, page, heads, dim)
    c.table[0, 1] = c.pages + 5                            # its second block goes nowhere
    dev.free(*c.bufs)
    c.upload()
    t, start, kv = sum(rows), _ragged(rows), np.array(lens, np.int32)
    k, v = (rng.standard_normal((t, heads, dim)).astype(np.float32) for _ in range(2))
    k[40, 0, 5] = np.nan                                   # sequence 1, head 0: block 1, whose scale becomes NaN
    v[42, 1, 0] = np.inf                                   # sequence 2, head 1
    k[45:], v[45:] = 0, 0                                  # sequence 3: zeros, the least scale
    bufs = [dev.put(k), dev.put(v), dev.put(start), dev.put(kv)]
    call = lambda: C.kv_append_q8(c.handle, bufs[0].ptr, bufs[1].ptr, *c.where, bufs[2].ptr, bufs[3].ptr, t, 4, 40, in_kind="f32")  # noqa: E731
    call()
    gk, gv, gks, gvs = c.download()
    untouched = c.k.copy()
    O.append(k.astype(np.float64), v.astype(np.float64), c.k, c.v, c.ks, c.vs, c.table, start, kv)
    for g, want in ((gks, c.ks), (gvs, c.vs)):
        assert np.array_equal(np.isnan(g), np.isnan(want))
        assert (np.abs(g - want)[~np.isnan(want)] <= 4 * U * want[~np.isnan(want)]).all()
    assert gks[c.table[3, 0], 0, 0] == np.float32(2.0 ** -64) and (gk[c.table[3, 0]] == 0).all() and (gv[c.table[3, 0]] == 0).all()
    spare = [p for p in range(c.pages) if p not in c.table]
    assert np.array_equal(gk[spare], untouched[spare])
    # a finite token behind it: the block stays NaN; a new start of the block makes it good again
    k[40, 0, 5] = 1.0
    again = [dev.put(k), dev.put(kv)]
    C.kv_append_q8(c.handle, again[0].ptr, bufs[1].ptr, *c.where, bufs[2].ptr, bufs[3].ptr, t, 4, 40, in_kind="f32")
    assert np.isnan(c.download()[2][c.table[1, 1], 0, 0]) == (lens[1] - rows[1] > 32)
    dev.free(*bufs, *again)
    c.free()


# ---- attention -----------------------------------------------------------------------------------------------------


def run_attention(dev, c, q, start, kv, max_q, max_kv, hq, kind, *, window=0, scale=None, pad=0, rows_behind=2):
    t = q.shape[0]
    width = hq * c.dim + pad
    wide = np.zeros((t, width))
    wide[:, : hq * c.dim] = q.reshape(t, -1)
    n = A.paged_attention_q8_workspace_bytes(t, len(kv), max_q, max_kv, hq, c.heads, c.dim)
    bufs = [dev.put(O.to_bits(wide, kind)), dev.put(start), dev.put(kv), dev.empty((t + rows_behind) * width * 2), dev.empty(max(n, 16))]
    A.paged_attention_q8(c.handle, bufs[0].ptr, bufs[3].ptr, *c.where, bufs[1].ptr, bufs[2].ptr, t, len(kv), max_q, max_kv, hq,
                         workspace_ptr=bufs[4].ptr if n else None, workspace_bytes=n, scale=scale, window=window, kind=kind,
                         q_stride=width, out_stride=width)
    raw = dev.get(bufs[3], np.uint16, (t + rows_behind, width))
    dev.free(*bufs)
    assert (raw[t:] == 0xA5A5).all() and (raw[:, hq * c.dim:] == 0xA5A5).all()
    return raw[:t, : hq * c.dim].reshape(t, hq, c.dim)


def attention_tolerance(want, deviation, magnitude, argument, kind, n, dim, v_max):
    """Roundings of one output: P to fp16 (2^-11 of every weight, and the sum takes the rounded ones, so it moves the
    output by at most 2^-11 sum p |v - o|), weights under fp16's range (2^-31 of the largest each); the softmax argument
    (dim products and sums of magnitude `argument`, plus its own size, in U, and exp2) acts like a relative error of the
    weights too; float32 sums over n keys in steps of 16; the output's rounding."""
    weights = 2.0 ** -11 + 2 * (dim + 8) * U * argument + 2 * U * (np.abs(argument) * 2 + 40)
    sums = (n / 16 + 64) * U
    inner = weights * deviation + sums * magnitude * 2 + n * 2.0 ** -31 * v_max
    return inner + O.HALF_STEP[kind] * (np.abs(want) + inner) + (2.0 ** -25 if kind == "fp16" else 0)


ATTENTION = [
    # dim, kv heads, group, page, rows, lengths, window, kind
    (128, 8, 5, 64, [1], [1], 0, "bf16"),
    (128, 8, 5, 64, [1, 1, 1, 1, 1], [31, 32, 33, 600, 0], 0, "bf16"),
    (64, 2, 8, 32, [1, 3, 2, 4], [700, 3, 65, 4], 0, "fp16"),
    (256, 2, 8, 128, [1, 2], [129, 300], 0, "bf16"),
    (128, 1, 1, 32, [1, 1], [513, 40], 0, "fp16"),
    (64, 1, 40, 64, [1, 3], [100, 200], 0, "bf16"),               # one KV head, more than one tile of rows
    (128, 2, 5, 64, [40, 0, 130, 1], [40, 17, 400, 90], 0, "bf16"),
    (64, 2, 4, 32, [257], [257], 0, "bf16"),
    (256, 1, 8, 64, [65, 33], [65, 290], 0, "fp16"),
    (128, 2, 4, 64, [5, 70], [3, 50], 0, "bf16"),                 # more rows than tokens: rows that see nothing
    (128, 2, 4, 64, [1, 1, 1], [1000, 70, 20], 64, "bf16"),       # windows
    (64, 2, 4, 32, [100, 33], [300, 33], 50, "fp16"),
    (128, 2, 8, 32, [90], [500], 1, "bf16"),
    (256, 2, 2, 128, [50], [700], 333, "bf16"),
    (128, 1, 8, 64, [1], [9000], 0, "bf16"),                      # chunks of keys and their joining
    (64, 1, 4, 1024, [2, 1], [7001, 40], 0, "fp16"),
    (256, 1, 8, 256, [1, 1], [5000, 4999], 0, "bf16"),
    (128, 1, 8, 64, [1], [9000], 4000, "bf16"),
    (128, 1, 8, 64, [150], [4000], 0, "bf16"),
    (128, 1, 8, 64, [150], [4000], 2500, "fp16"),
    (256, 2, 8, 128, [200, 64, 0, 331], [200, 1100, 0, 1331], 0, "bf16"),              # workgroups of eight waves, in parts
    (256, 4, 8, 32, [20] * 63 + [9], list(range(15, 78)) + [9], 0, "fp16"),            # and undivided
    (256, 4, 8, 32, [20] * 63 + [9], list(range(15, 78)) + [9], 17, "bf16"),
]


@pytest.mark.parametrize("dim,heads,group,page,rows,lens,window,kind", ATTENTION)
def test_paged_attention(dev, dim, heads, group, page, rows, lens, window, kind):
    rng = np.random.default_rng(dim + sum(lens) + group)
    c = Cache(dev, rng, lens, page, heads, dim)
    t, hq, start, kv = sum(rows), heads * group, _ragged(rows), np.array(lens, np.int32)
    q = O.round_to(rng.standard_normal((t, hq, dim)) * 2.0, kind)
    scale = dim ** -0.5
    got = O.from_bits(run_attention(dev, c, q, start, kv, max(rows), max(lens), hq, kind, window=window, pad=16), kind)
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=scale, window=window)
    tol = attention_tolerance(want, dv, mag, arg, kind, max(lens), dim, 127 * c.vs.max())
    worst = np.abs(got - want) - tol
    assert (worst <= 0).all(), (worst.max(), np.unravel_index(worst.argmax(), worst.shape))
    empty = [start[b] + i for b in range(len(rows)) for i in range(rows[b]) if lens[b] - rows[b] + i < 0]
    assert (got[empty] == 0).all()
    c.free()


def test_attention_larger_announced_lengths_and_own_scale(dev):
    """max_q_len and max_kv_len are upper bounds: larger ones, and lengths behind a table's end, change nothing."""
    rng = np.random.default_rng(77)
    rows, lens, dim, heads, group = [1, 2], [300, 70], 128, 2, 4
    c = Cache(dev, rng, lens, 64, heads, dim)
    start, kv = _ragged(rows), np.array(lens, np.int32)
    q = O.round_to(rng.standard_normal((3, heads * group, dim)), "bf16")
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=0.3)
    for max_q, max_kv in ((2, 300), (3, 5000), (64, 100000)):
        got = O.from_bits(run_attention(dev, c, q, start, kv, max_q, max_kv, heads * group, "bf16", scale=0.3), "bf16")
        assert (np.abs(got - want) <= attention_tolerance(want, dv, mag, arg, "bf16", 300, dim, 127 * c.vs.max())).all()
    c.free()


def test_attention_bad_pages_are_not_attended_to(dev):
    rng = np.random.default_rng(78)
    rows, lens, dim, heads, group = [1, 40], [300, 200], 128, 2, 4
    c = Cache(dev, rng, lens, 32, heads, dim)
    c.table[0, 3], c.table[0, 9], c.table[1, 0], c.table[1, 5] = -1, c.pages, 2**31 - 1, -(2**31)
    dev.free(*c.bufs)
    c.upload()
    start, kv = _ragged(rows), np.array(lens, np.int32)
    q = O.round_to(rng.standard_normal((41, heads * group, dim)), "bf16")
    got = O.from_bits(run_attention(dev, c, q, start, kv, 40, 300, heads * group, "bf16"), "bf16")
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=dim ** -0.5)
    assert (np.abs(got - want) <= attention_tolerance(want, dv, mag, arg, "bf16", 300, dim, 127 * c.vs.max())).all()
    c.free()


@pytest.mark.parametrize("rows,lens", [([1], [200]), ([150], [200])])
def test_attention_poisoned_blocks_reach_only_who_sees_them(dev, rows, lens):
    """A block whose scale is NaN makes NaN of the queries that see any of it, of no other; NaN in one query stays there;
    stale bytes behind the last token count for nothing."""
    rng = np.random.default_rng(79)
    dim, heads, group = 64, 2, 4
    for which in ("ks", "vs"):
        c = Cache(dev, rng, lens, 32, heads, dim)
        getattr(c, which)[c.table[0, 5], 1, 0] = np.nan                     # tokens 160 .. 191 of KV head 1
        dev.free(*c.bufs)
        c.upload()
        start, kv = _ragged(rows), np.array(lens, np.int32)
        q = O.round_to(rng.standard_normal((rows[0], heads * group, dim)), "bf16")
        q[0, 0, 3] = np.nan
        got = O.from_bits(run_attention(dev, c, q, start, kv, rows[0], lens[0], heads * group, "bf16"), "bf16")
        place = lens[0] - rows[0] + np.arange(rows[0])
        nan = np.zeros(got.shape[:2], bool)
        nan[place >= 160, group:] = True
        nan[0, 0] = True
        assert np.array_equal(np.isnan(got).all(-1), nan) and np.array_equal(np.isnan(got).any(-1), nan)
        c.free()


def test_attention_ranges(dev):
    """Scales far apart, values at the ends of the types, queries of very different size, all-zero blocks."""
    rng = np.random.default_rng(80)
    rows, lens, dim, heads, group = [3], [400], 128, 1, 4
    c = Cache(dev, rng, lens, 32, heads, dim)
    c.vs *= 2.0 ** rng.integers(-60, 60, c.vs.shape)
    c.ks *= 2.0 ** rng.integers(-6, 2, c.ks.shape)
    c.v[c.table[0, 2]] = 0
    c.vs[c.table[0, 2]] = O.FLOOR
    dev.free(*c.bufs)
    c.upload()
    start, kv = _ragged(rows), np.array(lens, np.int32)
    q = rng.standard_normal((3, group, dim))
    q[0] *= 2.0 ** -100
    q[1, 0] = 0
    q[1, 1] *= 3.0
    q[2, :, ::7] *= 2.0 ** -30
    q = O.round_to(q, "bf16")
    got = O.from_bits(run_attention(dev, c, q, start, kv, 3, 400, group, "bf16"), "bf16")
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=dim ** -0.5)
    # weights are relative to p * v_scale here: one under 2^-31 of the largest such product may be lost from the sum too
    tol = attention_tolerance(want, dv, mag, arg, "bf16", 400, dim, 127 * c.vs.max())
    assert (np.abs(got - want) <= tol).all()
    c.free()


def test_attention_refuses_a_small_workspace(dev):
    rng = np.random.default_rng(81)
    c = Cache(dev, rng, [9000], 64, 1, 128)
    n = A.paged_attention_q8_workspace_bytes(1, 1, 1, 9000, 8, 1, 128)
    assert n > 0
    bufs = [dev.empty(8 * 128 * 2), dev.empty(8 * 128 * 2), dev.put(np.array([0, 1], np.int32)), dev.put(np.array([9000], np.int32)), dev.empty(n)]
    for ptr, size in ((None, 0), (bufs[4].ptr, 1024), (bufs[4].ptr + 4, n)):
        with pytest.raises(HipError):
            A.paged_attention_q8(c.handle, bufs[0].ptr, bufs[1].ptr, *c.where, bufs[2].ptr, bufs[3].ptr, 1, 1, 1, 9000, 8,
                                 workspace_ptr=ptr, workspace_bytes=size)
    assert (dev.get(bufs[1], np.uint8, (8 * 128 * 2,)) == 0xA5).all()
    dev.free(*bufs)
    c.free()


@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("announced", [3000, 1 << 20])
def test_prompts_that_share_the_chip(dev, window, announced):
    """150 short prompts, some without rows, without keys, or with fewer keys than rows, a few behind thousands of keys: every
    sequence is cut into a number of parts of its own."""
    rng = np.random.default_rng(92)
    dim, heads, group, batch = 64, 1, 4, 150
    rows = [int(x) for x in rng.integers(0, 21, batch)]
    lens = [int(n + x) for n, x in zip(rows, rng.integers(0, 90, batch))]
    rows[3], lens[3], rows[70], lens[70], rows[71], lens[71], rows[149], lens[149] = 20, 3000, 17, 2500, 20, 0, 20, 2999
    rows[5], lens[5], rows[64], lens[64] = 20, 7, 0, 1500
    c = Cache(dev, rng, lens, 64, heads, dim)
    start, kv = _ragged(rows), np.array(lens, np.int32)
    q = O.round_to(rng.standard_normal((sum(rows), heads * group, dim)), "bf16")
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=dim ** -0.5, window=window)
    got = O.from_bits(run_attention(dev, c, q, start, kv, 20, announced, heads * group, "bf16", window=window), "bf16")
    assert (np.abs(got - want) <= attention_tolerance(want, dv, mag, arg, "bf16", 3000, dim, 127 * c.vs.max())).all()
    c.free()


@pytest.mark.parametrize("rows,lens", [([1, 2], [3000, 70]), ([3, 150], [40, 2100])])
def test_attention_announced_for_a_longer_cache_than_there_is(dev, rows, lens):
    """As a graph does that was captured for the longest cache: the keys are cut into parts by the lengths that there are."""
    rng = np.random.default_rng(78)
    dim, heads, group = 128, 1, 4
    c = Cache(dev, rng, lens, 64, heads, dim)
    start, kv = _ragged(rows), np.array(lens, np.int32)
    q = O.round_to(rng.standard_normal((sum(rows), heads * group, dim)), "fp16")
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=dim ** -0.5)
    for max_kv in (max(lens), 20000, 1 << 20, 1 << 30):
        got = O.from_bits(run_attention(dev, c, q, start, kv, max(rows), max_kv, heads * group, "fp16"), "fp16")
        assert (np.abs(got - want) <= attention_tolerance(want, dv, mag, arg, "fp16", max(lens), dim, 127 * c.vs.max())).all()
    c.free()


@pytest.mark.parametrize("dim,kv_len", [(128, 1024), (128, 1055), (64, 2048), (256, 512)])
def test_attention_workspace_is_enough_for_every_window(dev, dim, kv_len):
    """The size that is asked for without a window, at lengths that are a whole number of parts and windows around them."""
    rng = np.random.default_rng(91)
    c = Cache(dev, rng, [kv_len], 64, 1, dim)
    q = O.round_to(rng.standard_normal((1, 2, dim)), "bf16")
    start, kv = np.array([0, 1], np.int32), np.array([kv_len], np.int32)
    for window in (kv_len - 64, kv_len - 34, kv_len - 33, kv_len - 32, kv_len - 1, kv_len, kv_len + 1, 2 * kv_len):
        want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=dim ** -0.5, window=window)
        got = O.from_bits(run_attention(dev, c, q, start, kv, 1, kv_len, 2, "bf16", window=window), "bf16")
        assert (np.abs(got - want) <= attention_tolerance(want, dv, mag, arg, "bf16", kv_len, dim, 127 * c.vs.max())).all()
    c.free()


def test_append_then_attend_as_a_request_runs(dev):
    """A prompt in two chunks and then tokens one by one, q / k norm and rotation included: every step against attention
    over the values that the cache then holds, and the cache against the keys that went in."""
    rng = np.random.default_rng(82)
    dim, heads, group, page, kind = 128, 2, 5, 64, "bf16"
    hq, total = heads * group, 150
    c = Cache(dev, rng, [total], page, heads, dim)
    w = rng.uniform(0.5, 1.5, dim).astype(np.float32)
    freq = inv_freq(dim)
    fixed = [dev.put(w), dev.put(freq)]
    x = O.round_to(rng.standard_normal((total, (hq + 2 * heads) * dim)), kind)
    done = 0
    for n in (70, 59, 1, 1, 1, 18):
        rows = x[done: done + n]
        s = rows.shape[1]
        bufs = [dev.put(O.to_bits(rows, kind)), dev.put(np.arange(done, done + n)), dev.put(np.array([0, n], np.int32)),
                dev.put(np.array([done + n], np.int32)), dev.empty(n * hq * dim * 2), dev.empty(n * hq * dim * 2), dev.empty(1 << 22)]
        k, v = bufs[0].ptr + hq * dim * 2, bufs[0].ptr + (hq + heads) * dim * 2
        R.qk_norm_rope(bufs[0].ptr, None, bufs[4].ptr, None, n, hq, 0, dim, q_weight_ptr=fixed[0].ptr, positions_ptr=bufs[1].ptr,
                       inv_freq_ptr=fixed[1].ptr, rotary_dim=dim, q_stride=s)
        C.kv_append_q8(c.handle, k, v, *c.where, bufs[2].ptr, bufs[3].ptr, n, 1, n, k_weight_ptr=fixed[0].ptr, positions_ptr=bufs[1].ptr,
                       inv_freq_ptr=fixed[1].ptr, rotary_dim=dim, k_stride=s, v_stride=s)
        A.paged_attention_q8(c.handle, bufs[4].ptr, bufs[5].ptr, *c.where, bufs[2].ptr, bufs[3].ptr, n, 1, n, done + n, hq,
                             workspace_ptr=bufs[6].ptr, workspace_bytes=1 << 22)
        done += n
        q = O.from_bits(dev.get(bufs[4], np.uint16, (n, hq, dim)), kind)
        got = O.from_bits(dev.get(bufs[5], np.uint16, (n, hq, dim)), kind)
        ki, vi, ks, vs = c.download()
        want, dv, mag, arg = O.attention(q, ki, vi, ks.astype(np.float64), vs.astype(np.float64), c.table, np.array([0, n]),
                                         np.array([done]), scale=dim ** -0.5)
        assert (np.abs(got - want) <= attention_tolerance(want, dv, mag, arg, kind, done, dim, 127 * vs.max())).all()
        dev.free(*bufs)
    keys, _ = O.norm_rotate(x[:, hq * dim: (hq + heads) * dim].reshape(total, heads, dim), w, np.arange(total), freq)
    ki, _, ks, _ = c.download()
    values, _ = O.gather(ki, ks.astype(np.float64), c.table[0], total)
    # a byte carries half a step from its own rounding and at most half a (smaller) step from each of the rescalings
    steps = np.repeat(ks[c.table[0]].swapaxes(0, 1).reshape(heads, -1), 32, axis=1)[:, :total, None]
    assert (np.abs(values - keys.swapaxes(0, 1)) <= steps * 3.5).all()
    dev.free(*fixed)
    c.free()


@pytest.mark.parametrize("dim,heads,group,rows,kv_len", [(64, 2, 4, 3, 200), (128, 1, 8, 60, 300), (256, 2, 8, 40, 200)])
def test_weights_on_a_block_of_small_scale_are_counted_as_rounded(dev, dim, heads, group, rows, kv_len):
    """Every query's weight lies nearly all on one key of block 4, whose V is small beside that of block 0: the output is that
    key's value, and the rounding of its weight to fp16 leaves it there because the sum takes the weight as rounded. (With the
    sum over unrounded weights it is off by up to 2^-11 of itself more than its own rounding.) A key of block 0 is there to set
    the reference: at the reference a weight is a power of two."""
    rng = np.random.default_rng(dim)
    c = Cache(dev, rng, [kv_len], 32, heads, dim)
    c.vs[c.table[0, 0]] *= 30
    c.vs = c.vs.astype(np.float32).astype(np.float64)
    dev.free(*c.bufs)
    c.upload()
    start, kv = np.array([0, rows], np.int32), np.array([kv_len], np.int32)
    keys, _ = O.gather(c.k, c.ks, c.table[0], kv_len)
    q = np.zeros((rows, heads * group, dim))
    for i in range(rows):
        for h in range(heads * group):
            pair = keys[h // group][[128 + rng.integers(0, 32), rng.integers(0, 32)]]
            logit = 45 + rng.uniform(0, 8)                 # in log2; the other's w is 1 to 6 octaves less
            other = logit - np.log2(c.vs[c.table[0, 0], h // group, 0] / c.vs[c.table[0, 4], h // group, 0]) - rng.uniform(1, 6)
            q[i, h] = pair.T @ np.linalg.solve(pair @ pair.T, np.array([logit, other]) * np.log(2) * dim ** 0.5)
    q = O.round_to(q, "fp16")
    got = O.from_bits(run_attention(dev, c, q, start, kv, rows, kv_len, heads * group, "fp16"), "fp16")
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=dim ** -0.5)
    assert (np.abs(got - want) <= attention_tolerance(want, dv, mag, arg, "fp16", kv_len, dim, 127 * c.vs.max())).all()
    c.free()


@pytest.mark.parametrize("dim,heads,group,page,rows,lens,window,kind", [
    # 64 sequences of 8 heads: undivided, and the longest have 272 blocks for four waves, more than 64 each
    (64, 8, 1, 32, [1] * 64, [8700, 8300] + [3 + i for i in range(62)], 0, "bf16"),
    (128, 8, 1, 64, [1] * 64, [40] * 63 + [8500], 0, "fp16"),
    (256, 4, 2, 64, [1] * 128, [17] * 127 + [8400], 8300, "bf16"),
    # prompts of more than 64 rows a KV head, undivided: workgroups that walk over 72 to 150 blocks
    (64, 8, 8, 32, [9] * 32, [2300] + [9 + 5 * i for i in range(30)] + [4800], 0, "fp16"),
    (128, 8, 8, 64, [9] * 32, [2300] + [9] * 31, 0, "bf16"),
    (128, 8, 8, 64, [9] * 32, [3000] + [9] * 31, 2200, "bf16"),
    (256, 4, 8, 64, [20] * 63 + [9], [20] * 62 + [2300, 9], 0, "bf16"),              # eight waves
])
def test_attention_over_more_blocks_than_one_list_holds(dev, dim, heads, group, page, rows, lens, window, kind):
    """A wave keeps the numbers and scales of 64 blocks at a time: sequences that need two and three such lists in one
    workgroup, every block with scales of its own, some pages missing around the lists' ends."""
    rng = np.random.default_rng(dim + group)
    c = Cache(dev, rng, lens, page, heads, dim)
    c.ks *= 2.0 ** rng.uniform(-1.5, 0.5, c.ks.shape)
    c.vs *= 2.0 ** rng.uniform(-3, 3, c.vs.shape)
    c.ks, c.vs = (x.astype(np.float32).astype(np.float64) for x in (c.ks, c.vs))
    longest = int(np.argmax(lens))
    for block in (63, 64, 255, 257, 260):                 # (of 32 tokens: the page that it lies on)
        if block * 32 // page < c.table.shape[1]:
            c.table[longest, block * 32 // page] = -1
    dev.free(*c.bufs)
    c.upload()
    t, hq, start, kv = sum(rows), heads * group, _ragged(rows), np.array(lens, np.int32)
    q = O.round_to(rng.standard_normal((t, hq, dim)) * 2.0, kind)
    assert A.paged_attention_q8_workspace_bytes(t, len(lens), max(rows), max(lens), hq, heads, dim) == 0        # undivided
    got = O.from_bits(run_attention(dev, c, q, start, kv, max(rows), max(lens), hq, kind, window=window), kind)
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=dim ** -0.5, window=window)
    tol = attention_tolerance(want, dv, mag, arg, kind, max(lens), dim, 127 * c.vs.max())
    worst = np.abs(got - want) - tol
    assert (worst <= 0).all(), (worst.max(), np.unravel_index(worst.argmax(), worst.shape))
    c.free()


@pytest.mark.parametrize("window", [300, 700, 1])
def test_shares_of_eight_waves_within_a_window(dev, window):
    """Prompts of D 256 that share the workgroups, each cut into parts of its own, seeing a window only."""
    rng = np.random.default_rng(96)
    rows, lens, dim, heads, group = [200, 64, 0, 331], [200, 1100, 0, 1331], 256, 2, 8
    c = Cache(dev, rng, lens, 128, heads, dim)
    start, kv = _ragged(rows), np.array(lens, np.int32)
    q = O.round_to(rng.standard_normal((sum(rows), heads * group, dim)), "fp16")
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=dim ** -0.5, window=window)
    for max_q, max_kv in ((331, 1331), (400, 1 << 20)):
        got = O.from_bits(run_attention(dev, c, q, start, kv, max_q, max_kv, heads * group, "fp16", window=window), "fp16")
        assert (np.abs(got - want) <= attention_tolerance(want, dv, mag, arg, "fp16", 1331, dim, 127 * c.vs.max())).all()
    c.free()


def test_scales_under_the_least_count_as_the_least(dev):
    """A scale below 2^-64 (0, negative, subnormal) stands for 2^-64 wherever the cache is looked at: reading back, the
    earlier tokens of a block that is appended to, and attention. A NaN stays one."""
    rng = np.random.default_rng(21)
    dim, heads, page, lens = 64, 2, 32, [40, 20, 5]
    c = Cache(dev, rng, lens, page, heads, dim)
    for s in (c.ks, c.vs):
        s[...] = np.array([0.0, 2.0 ** -70, -1.0, 2.0 ** -140])[rng.integers(0, 4, s.shape)]
        s[c.table[2, 0], 1] = np.nan
    dev.free(*c.bufs)
    c.upload()
    least = np.float32(O.FLOOR)
    start, kv = _ragged(lens), np.array(lens, np.int32)
    out = [dev.empty(sum(lens) * heads * dim * 4) for _ in range(2)]
    ints = [dev.put(start), dev.put(kv)]
    C.kv_read_q8(c.handle, out[0].ptr, out[1].ptr, *c.where, ints[0].ptr, ints[1].ptr, sum(lens), 3, out_kind="f32")
    for buf, held, scales in ((out[0], c.k, c.ks), (out[1], c.v, c.vs)):
        got = dev.get(buf, np.float32, (sum(lens), heads, dim))
        for b, n in enumerate(lens):
            for t in range(n):
                pg, off = c.table[b, t // page], t % page
                want = held[pg, :, off].astype(np.float32) * np.where(np.isnan(scales[pg, :, 0]), np.nan, least)[:, None].astype(np.float32)
                assert np.array_equal(got[start[b] + t], want, equal_nan=True)
    # one more token each: zeros to sequence 0, values of two steps of 2^-64 at most to sequence 1, anything to sequence 2
    new = np.zeros((3, heads, dim), np.float32)
    new[1] = np.float32(2.0 ** -63) * rng.integers(-127, 128, (heads, dim))
    new[1, :, 0] = np.float32(127 * 2.0 ** -63)
    new[2] = rng.standard_normal((heads, dim))
    more = [dev.put(new), dev.put(_ragged([1, 1, 1])), dev.put(kv + 1)]
    C.kv_append_q8(c.handle, more[0].ptr, more[0].ptr, *c.where, more[1].ptr, more[2].ptr, 3, 3, 1, in_kind="f32")
    gk, gv, gks, gvs = c.download()
    for got, gs, held in ((gk, gks, c.k), (gv, gvs, c.v)):
        at = c.table[0, 1]
        assert (gs[at] == least).all() and np.array_equal(got[at, :, :8], held[at, :, :8]) and (got[at, :, 8] == 0).all()
        at = c.table[1, 0]
        assert (gs[at] == 2 * least).all() and np.array_equal(got[at, :, :20], np.rint(held[at, :, :20] * 0.5))
        assert np.array_equal(got[at, :, 20], np.rint(new[1] / np.float32(2.0 ** -63)))
        assert np.isnan(gs[c.table[2, 0], 1]).all() and not np.isnan(gs[c.table[2, 0], 0]).any()
    dev.free(*out, *ints, *more)
    c.free()


@pytest.mark.parametrize("dim,interleaved", [(128, False), (256, True), (64, False)])
def test_rotation_into_float32_is_rounded_once(dev, dim, interleaved):
    """Pairs (1, 0): the outputs are cos and sin of position * inv_freq as they are. A value of at most 1 rounded once is off
    by half a step, 2^-25; the angle, up to 2^20 radians in float64 with three roundings of 2^-53 here and on the device each,
    by 2^20 * 6 * 2^-53 < 2^-30."""
    rng = np.random.default_rng(dim)
    t = 700
    freq = inv_freq(dim)
    pos = np.sort(rng.integers(0, 1 << 20, t)).astype(np.int64)
    x = np.zeros((t, dim), np.float32)
    first = np.arange(0, dim, 2) if interleaved else np.arange(dim // 2)
    x[:, first] = 1
    bufs = [dev.put(x), dev.put(pos), dev.put(freq), dev.empty(x.nbytes)]
    R.qk_norm_rope(bufs[0].ptr, None, bufs[3].ptr, None, t, 1, 0, dim, positions_ptr=bufs[1].ptr, inv_freq_ptr=bufs[2].ptr,
                   rotary_dim=dim, interleaved=interleaved, in_kind="f32", out_kind="f32")
    got = dev.get(bufs[3], np.float32, (t, dim)).astype(np.float64)
    angle = pos[:, None].astype(np.float64) * freq.astype(np.float64)
    for cols, want in ((first, np.cos(angle)), (first + (1 if interleaved else dim // 2), np.sin(angle))):
        assert np.abs(got[:, cols] - want).max() <= 2.0 ** -25 + 2.0 ** -30
    dev.free(*bufs)


@pytest.mark.parametrize("dim,heads,group,rows,kv_len,window,longer", [
    (128, 2, 8, 100, 4000, 0, (9000, 1 << 17, 1 << 30)),
    (64, 8, 4, 64, 3000, 0, (1 << 15, 1 << 20)),
    (256, 2, 8, 60, 2500, 0, (5000, 10000)),
    (128, 2, 8, 100, 300, 0, (4000, 1 << 17)),            # fewer blocks than two parts have
    (128, 2, 8, 100, 6000, 2500, (1 << 17,)),
    (128, 2, 8, 100, 60, 0, (1 << 17,)),                  # rows that see nothing
])
def test_one_prompt_is_cut_by_the_keys_that_there_are(dev, dim, heads, group, rows, kv_len, window, longer):
    """The parts that a prompt's keys are cut into follow the length at run time: announced for a longer cache the call gives
    the same bits, being joined from the same parts."""
    rng = np.random.default_rng(95)
    c = Cache(dev, rng, [kv_len], 64, heads, dim)
    start, kv = np.array([0, rows], np.int32), np.array([kv_len], np.int32)
    q = O.round_to(rng.standard_normal((rows, heads * group, dim)), "bf16")
    exact = run_attention(dev, c, q, start, kv, rows, kv_len, heads * group, "bf16", window=window)
    want, dv, mag, arg = O.attention(q, c.k, c.v, c.ks, c.vs, c.table, start, kv, scale=dim ** -0.5, window=window)
    tol = attention_tolerance(want, dv, mag, arg, "bf16", kv_len, dim, 127 * c.vs.max())
    assert (np.abs(O.from_bits(exact, "bf16") - want) <= tol).all()
    for max_kv in longer:
        assert np.array_equal(run_attention(dev, c, q, start, kv, rows, max_kv, heads * group, "bf16", window=window), exact)
    c.free()


def test_attention_announced_for_more_rows_than_there_are(dev):
    """max_q_len counts as the batch's tokens at most."""
    rng = np.random.default_rng(98)
    rows, lens, dim, heads, group = [1, 30], [300, 70], 128, 2, 40
    c = Cache(dev, rng, lens, 64, heads, dim)
    start, kv = _ragged(rows), np.array(lens, np.int32)
    q = O.round_to(rng.standard_normal((31, heads * group, dim)), "bf16")
    want = run_attention(dev, c, q, start, kv, 31, 300, heads * group, "bf16")
    for max_q in (1 << 20, 1 << 30, 1 << 40):
        assert np.array_equal(run_attention(dev, c, q, start, kv, max_q, 300, heads * group, "bf16"), want)
    c.free()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_poisoned_block_stays_so_until_it_starts_anew(dev, which, bad):
    """A NaN or infinity in one token of K or V: finite tokens behind it leave the scale NaN, whatever their size, and reading
    gives NaN; once its first token is appended again the block is as good as any."""
    rng = np.random.default_rng(23)
    dim, heads, page = 64, 2, 32
    c = Cache(dev, rng, [70], page, heads, dim)
    start, one = dev.put(np.array([0, 2], np.int32)), dev.put(np.array([0, 1], np.int32))

    def append(x, end, rows):
        bufs = [dev.put(y.astype(np.float32)) for y in x] + [dev.put(np.array([end], np.int32))]
        C.kv_append_q8(c.handle, bufs[0].ptr, bufs[1].ptr, *c.where, (start if rows == 2 else one).ptr, bufs[2].ptr, rows, 1, rows, in_kind="f32")
        dev.sync()
        dev.free(*bufs)
        return c.download()

    x = rng.standard_normal((2, 2, heads, dim))
    x[which, 1, 1, 7] = bad
    append(x, 34, 2)                                       # places 32, 33
    pg = c.table[0, 1]
    for end, size in ((35, 1.0), (36, 0.0), (37, 1e30)):
        got = append(rng.standard_normal((2, 1, heads, dim)) * size, end, 1)
        scales, other = got[2 + which], got[3 - which]
        assert np.isnan(scales[pg, 1, 0]) and np.isfinite(scales[pg, 0, 0]) and np.isfinite(other[pg]).all()
    out, lens, full = dev.empty(37 * heads * dim * 4), dev.put(np.array([37], np.int32)), dev.put(np.array([0, 37], np.int32))
    C.kv_read_q8(c.handle, *((out.ptr, None) if which == 0 else (None, out.ptr)), *c.where, full.ptr, lens.ptr, 37, 1, out_kind="f32")
    nan = np.isnan(dev.get(out, np.float32, (37, heads, dim)))
    assert nan[32:, 1].all() and not nan[:32].any() and not nan[:, 0].any()
    x = rng.standard_normal((2, 1, heads, dim))
    gk, gv, gks, gvs = append(x, 33, 1)
    for g, gs, y in ((gk, gks, x[0, 0]), (gv, gvs, x[1, 0])):
        scale = np.abs(y.astype(np.float32)).max(-1) / np.float32(127)
        assert np.array_equal(gs[pg, :, 0], scale)
        assert np.array_equal(g[pg, :, 0], np.rint(y.astype(np.float32) / scale[:, None]))
    dev.free(start, one, out, lens, full)
    c.free()
