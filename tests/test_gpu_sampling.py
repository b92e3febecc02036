"""Sampling on one MI355X against its float64 statement (oracle/attention_oracle.py sample).

A weight on the device is good to 2^-22 of itself (argument in float64, exp2 of its fraction in float32, 24 bits kept) and
2^-40 of the largest, so a prefix sum is good to 2^-22 of the total: the id has to be one that the statement gives when its
sums are moved by that much, which nearly always is one id (and in half the rows at least has to be: asserted)."""

from __future__ import annotations

import numpy as np
import pytest

from hipengine_amd.core.hip import HipError
from hipengine_amd.kernels.hip_gfx950.sampling import sample_rows as S
from oracle import attention_oracle as O

pytestmark = pytest.mark.gpu

ACCURACY = 2.0 ** -22


def run(dev, logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None, stride=None, logprobs=True):
    rows, vocab = logits.shape
    wide = np.full((rows, stride or vocab), 1e30, np.float32)      # behind a row's end: what would win if it were read
    wide[:, :vocab] = logits
    n = S.sample_workspace_bytes(rows, vocab)
    given = {"temperature_ptr": (temperature, np.float32), "top_k_ptr": (top_k, np.int32), "top_p_ptr": (top_p, np.float32), "min_p_ptr": (min_p, np.float32)}
    put = {k: dev.put(np.broadcast_to(np.asarray(v, t), (rows,)).copy()) for k, (v, t) in given.items() if v is not None}
    bufs = [dev.put(wide), dev.put(np.asarray(uniform, np.float32)), dev.empty(rows * 4), dev.empty(rows * 4), dev.empty(n)]
    S.sample_f32_rows_i32(bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, rows, vocab, workspace_ptr=bufs[4].ptr, workspace_bytes=n,
                          out_logprobs_ptr=bufs[3].ptr if logprobs else None, logits_stride=stride or 0, **{k: b.ptr for k, b in put.items()})
    got = dev.get(bufs[2], np.int32, (rows,)), dev.get(bufs[3], np.float32, (rows,))
    dev.free(*bufs, *put.values())
    return got


def check(dev, logits, uniform, **settings):
    stride, borders = settings.pop("stride", None), settings.pop("borders", 0)
    ids, logprobs = run(dev, logits, uniform, stride=stride, **settings)
    at = lambda v, r: v if v is None or np.ndim(v) == 0 else v[r]  # noqa: E731
    open_rows = 0
    for r in range(len(logits)):
        kw = {k: at(v, r) for k, v in settings.items() if v is not None}
        kw = {k: (float(np.float32(v)) if k != "top_k" else int(v)) for k, v in kw.items()}
        want = O.sample(logits[r], float(np.float32(uniform[r])), accuracy=ACCURACY, **kw)
        assert ids[r] in want, (r, ids[r], want, kw)
        open_rows += len(want) > 1
        lo, hi = want[int(ids[r])]
        if np.isfinite(lo):
            assert lo - 2.0 ** -21 - 2.0 ** -24 * abs(lo) <= logprobs[r] <= hi + 2.0 ** -21 + 2.0 ** -24 * abs(lo)
        else:
            assert logprobs[r] == lo
    # of the statement alone: the test decides. In a flat row of 10^5 tokens 2^-22 of the total is a fortieth of a token, at
    # top-p's border and at the token's, above and below: a tenth of such rows is open
    assert open_rows <= max(1, len(logits) // 2, borders)


SETTINGS = [
    dict(),
    dict(temperature=0.7),
    dict(top_k=1),
    dict(top_k=50, top_p=0.95, temperature=0.8),
    dict(top_p=0.9),
    dict(top_p=0.999, temperature=1.5),
    dict(min_p=0.05),
    dict(top_k=40, top_p=0.8, min_p=0.1, temperature=1.3),
    dict(top_k=1000, min_p=0.001),
    dict(top_p=0.0),
    dict(min_p=1.0),
    dict(min_p=7.0, top_p=0.5),
    dict(temperature=0.0),
    dict(temperature=100.0),
    dict(temperature=100.0, top_k=777),
    dict(temperature=1e-3),
    dict(top_k=10**9, top_p=2.0, min_p=-1.0),
]


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4096, 4097, 32003, 151936])
@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: ",".join(f"{k}={v}" for k, v in s.items()) or "none")
def test_rows_against_the_statement(dev, vocab, settings):
    rows = 5
    rng = np.random.default_rng(vocab * 7 + 1)
    logits = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    check(dev, logits, rng.random(rows), stride=vocab + 3, **settings)


def test_every_row_has_its_own_settings(dev):
    rng = np.random.default_rng(11)
    rows, vocab = 70, 5003
    logits = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    check(dev, logits, rng.random(rows), temperature=rng.choice([0.0, 0.5, 1.0, 2.0], rows), top_k=rng.choice([0, 1, 7, 300, -3], rows),
          top_p=rng.choice([1.0, 0.9, 0.3], rows), min_p=rng.choice([0.0, 0.02, 0.5], rows))


def test_ties_go_to_the_lowest_index(dev):
    """Logits of few distinct values: borders fall inside runs of equal tokens."""
    rng = np.random.default_rng(12)
    rows, vocab = 12, 9001
    logits = rng.integers(-3, 3, (rows, vocab)).astype(np.float32)
    logits[0] = 1.0
    logits[1, ::2], logits[1, 1::2] = 0.0, -0.0                        # the same number
    for settings in (dict(top_k=100), dict(top_k=3000), dict(top_p=0.0123), dict(top_p=0.77), dict(top_k=2000, top_p=0.333)):
        check(dev, logits, rng.random(rows), **settings)


def test_flat_rows_whose_border_bin_does_not_fit_the_list(dev):
    rng = np.random.default_rng(13)
    rows, vocab = 4, 100003
    logits = (rng.standard_normal((rows, vocab)) * 0.01).astype(np.float32)
    logits[0] = 0.25
    for settings in (dict(top_k=30000), dict(top_p=0.5003), dict(top_k=50000, top_p=0.7001), dict(top_p=0.9003, min_p=0.95), dict(min_p=0.99)):
        check(dev, logits, rng.random(rows), **settings)


def test_masked_infinite_and_nan_logits(dev):
    rng = np.random.default_rng(14)
    rows, vocab = 8, 4500
    logits = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, :] = -np.inf
    logits[2, 4400] = -3.0                                             # one token left
    logits[3, ::3] = -np.inf
    logits[4, 5], logits[4, 4444] = np.inf, np.inf                     # two equal tokens of all weight
    logits[5, 100:4000] = np.nan
    logits[6] = np.finfo(np.float32).min                               # masks by the type's lowest value: tokens like others
    logits[6, 77] = 0.0
    logits[7, :] = np.finfo(np.float32).min
    u = np.array([0.3, 0.3, 0.9, 0.51, 0.7, 0.2, 0.99, 0.613], np.float32)
    for settings in (dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.9), dict(min_p=0.01), dict(temperature=0.0)):
        check(dev, logits, u, **settings)


@pytest.mark.parametrize("temperature", [1e-45, 1e-38, 2.0 ** -124, 3e38, np.inf])
@pytest.mark.parametrize("settings", [dict(), dict(min_p=0.5), dict(top_p=0.5), dict(top_k=2)], ids=str)
def test_extreme_temperatures(dev, temperature, settings):
    """Rows whose logits differ by the least there is, by ordinary amounts and by the most."""
    rows = np.zeros((3, 5), np.float32)
    rows[0] = np.float32(2.0 ** -126) - np.arange(5, dtype=np.float32) * np.float32(2.0 ** -149)
    rows[1] = [1.0, 3.0, 3.0, -2.0, 0.5]
    rows[2] = [3e38, -3e38, 0.0, 3e38, 1.0]
    for u in (0.1, 0.45, 0.8):
        # (float32(0.8) is 4/5 + 2^-26: at the border of five equal weights, which the rows have at the highest
        # temperatures, both answers are within 2^-22)
        check(dev, rows, [u] * 3, temperature=temperature, borders=3 if u == 0.8 else 0, **settings)


def test_uniform_ends(dev):
    logits = np.log(np.array([[1, 2, 4, 1]], np.float32)).repeat(5, 0)
    ids, _ = run(dev, logits, [0.0, 1.0, 2.0, np.nan, np.nextafter(np.float32(1), np.float32(0))])
    assert list(ids) == [0, 3, 3, 0, 3]


def test_frequencies_follow_the_distribution(dev):
    """4096 evenly spaced uniforms: every token is chosen as often as its share says, to one count at each of its ends."""
    rng = np.random.default_rng(15)
    rows, vocab = 4096, 50
    row = (rng.standard_normal(vocab) * 2).astype(np.float32)
    ids, _ = run(dev, np.broadcast_to(row, (rows, vocab)), (np.arange(rows) + 0.5) / rows, temperature=0.9, top_p=0.95)
    w = np.exp(row.astype(np.float64) / np.float64(np.float32(0.9)))
    order = np.argsort(-row, kind="stable")
    n = 1 + int(np.sum(np.cumsum(w[order])[:-1] < float(np.float32(0.95)) * w.sum()))
    kept = np.zeros(vocab)
    kept[order[:n]] = w[order[:n]]
    assert (np.abs(np.bincount(ids, minlength=vocab) - rows * kept / kept.sum()) <= 1.0).all()


def test_two_runs_are_equal_and_logprobs_are_optional(dev):
    rng = np.random.default_rng(16)
    logits = (rng.standard_normal((3, 151936)) * 2).astype(np.float32)
    u = rng.random(3)
    a, b = (run(dev, logits, u, top_p=0.9) for _ in range(2))
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1].view(np.uint32), b[1].view(np.uint32))
    c = run(dev, logits, u, top_p=0.9, logprobs=False)
    assert np.array_equal(a[0], c[0]) and (c[1].view(np.uint32) == 0xA5A5A5A5).all()


def test_small_workspace_is_refused(dev):
    n = S.sample_workspace_bytes(2, 1000)
    bufs = [dev.empty(8000), dev.empty(8), dev.empty(8), dev.empty(n + 8)]
    for ptr, size in ((bufs[3].ptr, n - 1), (bufs[3].ptr + 4, n)):
        with pytest.raises(HipError):
            S.sample_f32_rows_i32(bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, 2, 1000, workspace_ptr=ptr, workspace_bytes=size)
    assert (dev.get(bufs[2], np.uint8, (8,)) == 0xA5).all()
    dev.free(*bufs)


@pytest.mark.parametrize("vocab", [262145, 400003, 1 << 20, 1 << 22])
@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.9, temperature=0.8), dict(top_k=50, top_p=0.95), dict(top_k=3000, min_p=0.001)],
                         ids=lambda s: ",".join(f"{k}={v}" for k, v in s.items()) or "none")
def test_vocabularies_of_many_chunks(dev, vocab, settings):
    """More chunks than a wave has lanes, and than the borders' kernel adds up at once, up to the 1024 that there can be."""
    rng = np.random.default_rng(vocab + len(settings))
    rows = 2 if vocab < 1 << 20 else 1
    logits = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    for u in (0.02, 0.985):
        check(dev, logits, [u] * rows, borders=rows, **settings)


@pytest.mark.parametrize("vocab", [400003, 1 << 22])
def test_flat_rows_of_many_chunks(dev, vocab):
    """The largest sums that there are: every weight is the largest, 2^40, and the answer is known."""
    logits = np.full((1, vocab), -3.5, np.float32)
    for u in (0.0, 0.25, 0.7501, 0.99999):
        u = float(np.float32(u))
        ids, logprobs = run(dev, logits, [u])
        assert ids[0] == int(u * vocab) and abs(logprobs[0] + np.log(vocab)) <= 2.0 ** -20
        kept = int(np.ceil(0.5 * vocab))                   # by top-p, then by top-k: the first so many by index
        assert run(dev, logits, [u], top_p=0.5)[0][0] == int(u * kept)
        assert run(dev, logits, [u], top_k=300000)[0][0] == int(u * 300000)
