"""Where ah_paged_attention cuts and joins, and values that are not finite among those that a token sees; cases, loops and tolerances of
tests/test_gpu_paged.py."""
import math

import numpy as np
import pytest

from alpha2_amd import _ffi as ffi
from test_gpu_paged import TYPES, B, Case, check_attention, dev, run_attention, values  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,D", [(4, 2, 64), (2, 2, 128), (8, 1, 40)])
@pytest.mark.parametrize("news", [[1] * 10, [1, 0, 3, 1, 1, 1, 0, 2, 1, 1], [33, 1, 0, 64, 1, 90, 1, 128, 3, 40]])
def test_lengths_around_what_is_cut(B, dev, dtype, heads, kv_heads, D, news):
    """One batch with sequences of one part, just cut, of several parts and of none, some idle: every tile's parts are found where they were left."""
    lens = [511, 512, 513, 640, 1, 769, 1025, 128, 2050, 257]
    c = Case(dtype, heads, kv_heads, D, 48, lens, news, seed=D, entries=2)
    check_attention(c, *run_attention(B, dev, c, 0.15, 0.0), 0.15, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,D,length,new", [(1, 1, 64, 9000, 1), (4, 4, 128, 20000, 1), (2, 1, 32, 33000, 2), (1, 1, 128, 6000, 40)])
def test_one_sequence_in_many_parts(B, dev, dtype, heads, kv_heads, D, length, new):
    c = Case(dtype, heads, kv_heads, D, 128, [length], [new], seed=length, entries=1, spare=1)
    check_attention(c, *run_attention(B, dev, c, 0.2, 0.0), 0.2, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_sequences_than_a_wave_looks_at_together(B, dev, dtype):
    """200 sequences, most of them idle, long ones among the last."""
    rs = np.random.RandomState(3)
    lens = [int(n) for n in rs.randint(0, 40, 200)]
    news = [int(min(n, rs.randint(0, 2))) for n in lens]
    for s, n, m in ((70, 1500, 1), (150, 900, 30), (199, 2000, 1)):
        lens[s], news[s] = n, m
    c = Case(dtype, 2, 1, 64, 32, lens, news, seed=4)
    check_attention(c, *run_attention(B, dev, c, 0.125, 30.0), 0.125, 30.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("heads,kv_heads,D,length,new", [(1, 1, 64, 200, 200), (2, 1, 128, 300, 170), (4, 1, 64, 90, 5), (2, 2, 32, 1400, 130), (3, 1, 128, 700, 1)])
def test_infinite_values_reach_those_who_see_them_and_nobody_else(B, dev, dtype, cap, heads, kv_heads, D, length, new):
    """Infinite values at some positions, the first and last new ones among them: the features there are infinite for the tokens from those positions on, NaN
    where both signs or a NaN are seen; all else is what it is without them.  (Weights stay above 2^-126: no 0 x infinity.)"""
    c = Case(dtype, heads, kv_heads, D, 16, [length], [new], seed=length + new)
    first = length - new
    put = [(first, 3, np.inf), (length - 1, 5, -np.inf), (first + new // 2, 3, -np.inf), (first + new // 3, 7, np.nan), (first // 2, 6, np.inf), (first + 2 * new // 3, 6, np.inf)]
    bits = {"inf": 0x7f80, "-inf": 0xff80, "nan": 0x7fc0}
    clean = c.v.copy()
    for p, f, x in put:
        at = int(c.places(0, p)) + f
        clean[at] = 0
        c.v[at] = np.uint16(bits[str(x)]) if dtype == ffi.BF16 else np.float32(x)
    out, lse = run_attention(B, dev, c, 0.1, cap)
    out = values(out).astype(np.float64).copy()
    with np.errstate(invalid="ignore"):
        for r in range(new):
            extra = np.zeros(D)
            for (p, f), x in {(p, f): x for p, f, x in put}.items():        # (of two put in one place the later one lies there)
                if p <= first + r:
                    extra[f] += x
            for h in range(heads):
                mine = out[r, h * D:(h + 1) * D] if out.ndim == 2 else out[r, h]
                odd = ~np.isfinite(extra)
                if h * kv_heads // heads == 0:
                    assert np.array_equal(mine[odd], extra[odd], equal_nan=True), (r, h, mine[odd], extra[odd])
                    assert np.all(np.isfinite(mine[~odd])), (r, h)
                else:
                    assert np.all(np.isfinite(mine))
    # with 0 in their place the finite features are the same, but for sums taken in another order
    c.v = clean
    again, sums = run_attention(B, dev, c, 0.1, cap)
    check_attention(c, again, sums, 0.1, cap)
    assert np.array_equal(lse, sums)
    again = values(again).astype(np.float64)
    fine = np.isfinite(out)
    h = 2.0 ** -8 if dtype == ffi.BF16 else 0.0
    assert np.all(abs(out - again)[fine] <= (2 * h + 400 * 2.0 ** -24) * np.maximum(abs(again[fine]), 4.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [[1, 3, 1], [40, 3, 70]])
@pytest.mark.parametrize("scale,cap", [(-0.2, 0.0), (-0.3, 20.0), (-0.3, 90.0), (0.0, 0.0), (0.0, 5.0), (0.2, 41.0), (3.0, 60.0), (3.0, 0.0)])
def test_scales_of_every_sign_and_size(B, dev, dtype, news, scale, cap):
    c = Case(dtype, 4, 2, 64, 16, [120, 60, 90], news, seed=5)
    check_attention(c, *run_attention(B, dev, c, scale, cap), scale, cap)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [[1, 3, 1], [40, 3, 70]])
@pytest.mark.parametrize("cap", [50.0, 3000.0, 1e7, 2.0 ** 45])
def test_a_large_cap_costs_no_last_places_of_its_own(B, dev, dtype, news, cap):
    """The bound of tests/test_gpu_paged.py with the cap's share relative to the score: tanh to 1.63 last places (3.3 u), its argument and the product with the cap, u each
    (scores here are below half the cap, where a relative error of the argument is no larger in tanh): 6 u |s| in place of 8 u cap."""
    c, scale = Case(dtype, 4, 2, 64, 16, [120, 60, 90], news, seed=6), 0.2
    out, lse = run_attention(B, dev, c, scale, cap)
    q, h, u = c.part("q"), 2.0 ** -8 if dtype == ffi.BF16 else 0.0, 2.0 ** -24
    for s, length in enumerate(c.lens):
        k, v = (c.seen(name, s, np.arange(length)) for name in "kv")
        for r in range(int(c.starts[s]), int(c.starts[s + 1])):
            n = length - c.news[s] + r - int(c.starts[s]) + 1
            for head in range(4):
                raw = scale * (k[:n, head // 2] @ q[r, head])
                x, size = cap * np.tanh(raw / cap), scale * (abs(k[:n, head // 2]) @ abs(q[r, head]))
                assert abs(raw).max() < cap / 2
                e = float(((c.D + 3) * u * size + 10 * u * abs(x)).max())
                w = np.exp(x - x.max())
                want, around = (w @ v[:n, head // 2]) / w.sum(), (w @ abs(v[:n, head // 2])) / w.sum()
                bound = (math.expm1(2 * e + 4 * u) + (n + 16) * u + 2 * h * (1 + h)) * around * (1 + h) + (h + 2 * u) * abs(want)
                assert np.all(abs(values(out[r]).reshape(4, 64)[head] - want) <= bound), (s, r, head)
                want_l = x.max() + math.log(w.sum())
                assert abs(lse[r, head] - want_l) <= e + (n + 16) * u + 4 * u * abs(want_l) + 8 * u, (s, r, head)


@pytest.mark.parametrize("cap", [0.0, 30.0, 60.0])
@pytest.mark.parametrize("page", [64, 128, 192])
@pytest.mark.parametrize("heads,kv_heads,lens,news", [(4, 2, [300, 64, 129, 1000], [200, 64, 129, 40]), (2, 1, [63, 65, 2500], [63, 60, 50]), (8, 1, [700, 3, 640], [9, 3, 20])])
def test_pages_that_hold_whole_tiles(B, dev, cap, page, heads, kv_heads, lens, news):
    """bf16 heads of 128 in pages of a multiple of 64 positions, whose tiles are fetched by one address: ends inside a tile, at its end, and cut contexts."""
    c = Case(ffi.BF16, heads, kv_heads, 128, page, lens, news, seed=page + heads, heads_first=page == 128, entries=2)
    check_attention(c, *run_attention(B, dev, c, 0.09, cap), 0.09, cap)


@pytest.mark.parametrize("page", [64, 192])
def test_missing_pages_that_hold_whole_tiles(B, dev, page):
    c = Case(ffi.BF16, 4, 2, 128, page, [500, 400, 2100], [100, 90, 40], seed=2, entries=2)
    c.table[0, 1], c.table[2, 3] = c.pages, -1
    c.table[1, -(-400 // page):] = 2 ** 31 - 1           # behind what the sequence has: nobody reads them
    pages = c.upload(dev)
    c.table = np.where((c.table < 0) | (c.table >= c.pages), 0, c.table).astype(np.int32)
    check_attention(c, *run_attention(B, dev, c, 0.09, 0.0, pages=pages), 0.09, 0.0, bad={(0, 1), (2, 3)})
