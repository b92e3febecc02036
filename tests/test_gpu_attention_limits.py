"""The attention operators and the sampler where offsets pass 32 bits, on buffers that are aligned to an element only, in
padded batches, over shared pages, and with the largest strides; mostly against the same call in ordinary circumstances,
whose results other tests hold against float64."""

from __future__ import annotations

import numpy as np
import pytest

from hipengine_amd.kernels.hip_gfx950.attention import kv_cache_q8 as C
from hipengine_amd.kernels.hip_gfx950.attention import paged_attention_q8 as A
from hipengine_amd.kernels.hip_gfx950.attention import qk_norm_rope as R
from hipengine_amd.kernels.hip_gfx950.sampling import sample_rows as S
from oracle import attention_oracle as O

pytestmark = pytest.mark.gpu


class Space:
    """A cache of so many pages, uninitialized."""

    def __init__(self, dev, pages, page, heads, dim):
        self.dev, self.page, self.heads, self.dim, self.pages = dev, page, heads, dim, pages
        self.k, self.v = (dev.empty(C.KVCacheQ8.value_bytes(pages, page, heads, dim), fill=None) for _ in range(2))
        self.ks, self.vs = (dev.empty(C.KVCacheQ8.scale_bytes(pages, page, heads)) for _ in range(2))
        self.handle = C.KVCacheQ8(self.k.ptr, self.v.ptr, self.ks.ptr, self.vs.ptr, pages, page, heads, dim)

    def free(self):
        self.dev.free(self.k, self.v, self.ks, self.vs)


def request(dev, space, table, rows, lens, k, v, q, hq, *, tokens=None, shift=0, pad=0, kind="bf16", window=0):
    """Append k, v in one call, attend with q, read all back. Buffers begin `shift` elements behind an allocation's start, rows
    are `pad` elements longer, and the batch has `tokens` rows of which those behind the sequences' are nobody's."""
    dim, heads, n = space.dim, space.heads, sum(rows)
    tokens = tokens or n
    start, kv = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32), np.array(lens, np.int32)
    full = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    table = np.array(table, np.int32)

    def put(x, width):
        raw = np.full(shift + tokens * (width + pad), 0x7FC0, np.uint16)          # (NaN where nobody is to look)
        raw[shift:].reshape(tokens, -1)[:n, :width] = O.to_bits(x, kind).reshape(n, width)
        return dev.put(raw)

    at = [put(k, heads * dim), put(v, heads * dim), put(q, hq * dim)]
    ints = [dev.put(table), dev.put(start), dev.put(kv), dev.put(full)]
    where, ks = (ints[0].ptr, table.shape[1]), heads * dim + pad
    size = A.paged_attention_q8_workspace_bytes(tokens, len(rows), max(rows), max(lens), hq, heads, dim)
    outs = [dev.empty(2 * (shift + tokens * (hq * dim + pad)))] + [dev.empty(2 * (shift + (full[-1] + 3) * ks)) for _ in range(2)]
    work = dev.empty(max(size, 16))
    C.kv_append_q8(space.handle, at[0].ptr + 2 * shift, at[1].ptr + 2 * shift, *where, ints[1].ptr, ints[2].ptr, tokens, len(rows), max(rows),
                   in_kind=kind, k_stride=ks, v_stride=ks)
    A.paged_attention_q8(space.handle, at[2].ptr + 2 * shift, outs[0].ptr + 2 * shift, *where, ints[1].ptr, ints[2].ptr, tokens,
                         len(rows), max(rows), max(lens), hq, workspace_ptr=work.ptr, workspace_bytes=size, kind=kind, window=window,
                         q_stride=hq * dim + pad, out_stride=hq * dim + pad)
    C.kv_read_q8(space.handle, outs[1].ptr + 2 * shift, outs[2].ptr + 2 * shift, *where, ints[3].ptr, ints[2].ptr, int(full[-1]) + 3,
                 len(rows), out_kind=kind, k_out_stride=ks, v_out_stride=ks)
    got = []
    for buf, r, m, width in ((outs[0], tokens, n, hq * dim), (outs[1], full[-1] + 3, full[-1], heads * dim), (outs[2], full[-1] + 3, full[-1], heads * dim)):
        raw = dev.get(buf, np.uint16, (buf.nbytes // 2,))
        x = raw[shift:].reshape(r, width + pad)
        assert (raw[:shift] == 0xA5A5).all() and (x[m:] == 0xA5A5).all() and (x[:, width:] == 0xA5A5).all()
        got.append(x[:m, :width].copy())
    dev.free(*at, *ints, *outs, work)
    return got


def draw(rng, rows, heads, hq, dim, kind="bf16"):
    n = sum(rows)
    return [O.round_to(rng.standard_normal((n, h, dim)), kind) for h in (heads, heads, hq)]


def same(a, b):
    for x, y in zip(a, b):
        assert np.array_equal(x, y)


@pytest.mark.parametrize("rows", [[150], [3]])
def test_pages_past_32_bits(dev, rows):
    """33000 pages of 64 tokens, 8 heads of 256: 4.3 GB of K and of V, more than 2^32 bytes. What lies on the last pages is
    what lies on the first ones of a small cache."""
    rng = np.random.default_rng(1)
    heads, hq, dim, page = 8, 16, 256, 64
    k, v, q = draw(rng, rows, heads, hq, dim)
    big, small = Space(dev, 33000, page, heads, dim), Space(dev, 4, page, heads, dim)
    assert big.k.nbytes > 1 << 32
    want = request(dev, small, [[0, 2, 1]], rows, rows, k, v, q, hq)
    got = request(dev, big, [[32999, 32769, 1]], rows, rows, k, v, q, hq)
    same(got, want)
    big.free()
    small.free()


@pytest.mark.parametrize("shift,pad", [(1, 3), (3, 1), (4, 4), (7, 0)])
@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("fp16", 64), ("bf16", 256)])
def test_element_alignment(dev, kind, dim, shift, pad):
    rng = np.random.default_rng(2)
    rows, heads, hq = [1, 70, 2], 2, 6
    k, v, q = draw(rng, rows, heads, hq, dim, kind)
    table = [[0, 5], [1, 2], [4, 3]]
    space = Space(dev, 6, 64, heads, dim)
    want = request(dev, space, table, rows, rows, k, v, q, hq, kind=kind)
    same(request(dev, space, table, rows, rows, k, v, q, hq, kind=kind, shift=shift, pad=pad), want)
    space.free()


@pytest.mark.parametrize("rows", [[1, 1, 1], [1, 0, 90]])
def test_rows_of_no_sequence(dev, rows):
    """A batch padded to more rows than its sequences have: the padding is neither read (it is NaN) nor written."""
    rng = np.random.default_rng(3)
    heads, hq, dim = 2, 8, 128
    k, v, q = draw(rng, rows, heads, hq, dim)
    table = [[0, 5], [1, 2], [4, 3]]
    space = Space(dev, 6, 64, heads, dim)
    want = request(dev, space, table, rows, rows, k, v, q, hq)
    for tokens in (sum(rows) + 1, sum(rows) + 61):
        same(request(dev, space, table, rows, rows, k, v, q, hq, tokens=tokens), want)
    space.free()


def test_shared_prefix_pages(dev):
    """Two sequences whose tables begin with the same two pages: each reads what a sequence with pages of its own reads."""
    rng = np.random.default_rng(4)
    heads, hq, dim, page = 2, 8, 128, 32
    prefix, tails = draw(rng, [64], heads, hq, dim), [draw(rng, [20], heads, hq, dim) for _ in range(2)]
    shared, own = Space(dev, 8, page, heads, dim), Space(dev, 8, page, heads, dim)
    request(dev, shared, [[6, 1]], [64], [64], *prefix, hq)
    both = [np.concatenate([t[i] for t in tails]) for i in range(3)]
    got = request(dev, shared, [[6, 1, 3], [6, 1, 0]], [20, 20], [84, 84], *both, hq)
    for b, tail in enumerate(tails):
        request(dev, own, [[2, 5]], [64], [64], *prefix, hq)
        want = request(dev, own, [[2, 5, 7]], [20], [84], *tail, hq)
        same([got[0][20 * b: 20 * b + 20], got[1][84 * b: 84 * b + 84], got[2][84 * b: 84 * b + 84]], want)
    shared.free()
    own.free()


def test_strides_past_32_bits(dev):
    """Three rows 2^30 elements apart (6.4 GB each in bf16) against the same rows packed."""
    rng = np.random.default_rng(5)
    t, hq, hk, dim, far = 3, 4, 2, 128, 1 << 30
    x = O.to_bits(rng.standard_normal((t, hq + 2 * hk, dim)), "bf16")
    near = dev.put(x)
    wide = dev.empty(2 * (2 * far + (hq + 2 * hk) * dim), fill=None)
    for i in range(t):
        dev.runtime.memcpy(wide.ptr + 2 * i * far, x[i].ctypes.data, x[i].nbytes, 1)
    w, pos = dev.put(rng.uniform(0.5, 1.5, dim).astype(np.float32)), dev.put(np.arange(t, dtype=np.int64) + 7)
    freq = dev.put((1e4 ** (-np.arange(0, dim, 2) / dim)).astype(np.float32))
    start, kv, table = dev.put(np.array([0, t], np.int32)), dev.put(np.array([t], np.int32)), dev.put(np.array([[1]], np.int32))
    out = dev.empty(2 * (2 * far + (hq + 2 * hk) * dim), fill=None)
    spaces, results = [Space(dev, 2, 32, hk, dim) for _ in range(2)], []
    for src, dst, stride, space in ((near, dev.empty(x.nbytes), x[0].size, spaces[0]), (wide, out, far, spaces[1])):
        k, v = src.ptr + 2 * hq * dim, src.ptr + 2 * (hq + hk) * dim
        R.qk_norm_rope(src.ptr, k, src.ptr, dst.ptr + 2 * hq * dim, t, hq, hk, dim, q_weight_ptr=w.ptr, k_weight_ptr=w.ptr,
                       positions_ptr=pos.ptr, inv_freq_ptr=freq.ptr, rotary_dim=dim, q_stride=stride, k_stride=stride,
                       q_out_stride=stride, k_out_stride=stride)
        C.kv_append_q8(space.handle, dst.ptr + 2 * hq * dim, v, table.ptr, 1, start.ptr, kv.ptr, t, 1, t, k_stride=stride, v_stride=stride)
        A.paged_attention_q8(space.handle, src.ptr, dst.ptr, table.ptr, 1, start.ptr, kv.ptr, t, 1, t, t, hq, q_stride=stride, out_stride=stride)
        C.kv_read_q8(space.handle, dst.ptr + 2 * hq * dim, dst.ptr + 2 * (hq + hk) * dim, table.ptr, 1, start.ptr, kv.ptr, t, 1,
                     k_out_stride=stride, v_out_stride=stride)
        dev.sync()
        rows = np.zeros_like(x)
        for i in range(t):
            dev.runtime.memcpy(rows[i].ctypes.data, dst.ptr + 2 * i * stride, rows[i].nbytes, 2)
        results.append(rows)
        if dst is not out:
            dev.free(dst)
    assert np.isfinite(O.from_bits(results[0], "bf16")).all()
    same([results[1]], [results[0]])
    for s in spaces:
        s.free()
    dev.free(near, wide, out, w, pos, freq, start, kv, table)


def test_logits_past_32_bits(dev):
    rng = np.random.default_rng(6)
    rows, vocab, far = 3, 5000, 1 << 30
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    near, wide = dev.put(x), dev.empty(4 * (2 * far + vocab), fill=None)
    for i in range(rows):
        dev.runtime.memcpy(wide.ptr + 4 * i * far, x[i].ctypes.data, x[i].nbytes, 1)
    size = S.sample_workspace_bytes(rows, vocab)
    u, p, work, ids, lp = dev.put(rng.random(rows).astype(np.float32)), dev.put(np.full(rows, 0.9, np.float32)), dev.empty(size), dev.empty(12), dev.empty(12)
    got = []
    for src, stride in ((near, 0), (wide, far)):
        S.sample_f32_rows_i32(src.ptr, u.ptr, ids.ptr, rows, vocab, workspace_ptr=work.ptr, workspace_bytes=size, top_p_ptr=p.ptr,
                              out_logprobs_ptr=lp.ptr, logits_stride=stride)
        got.append([dev.get(ids, np.int32, (rows,)).copy(), dev.get(lp, np.uint32, (rows,)).copy()])
    same(*got)
    assert (got[0][0] >= 0).all()
    dev.free(near, wide, u, p, work, ids, lp)
