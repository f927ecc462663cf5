"""Pages and sampling at the ends of what they take: the smallest caps, the largest vocabulary, pages filled from the host, a sequence alone and beside others."""
import numpy as np
import pytest

from alpha2_amd import _ffi as ffi
from test_gpu_paged import TYPES, B, Case, check_attention, dev, run_attention, to_bf16  # noqa: F401 (fixtures)
from test_gpu_sample import check as check_sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [[1, 3, 1], [40, 3, 70]])
@pytest.mark.parametrize("cap", [2.0 ** -149, 1e-40, 2.0 ** -126, 1e-30, 2.0 ** -41, 2.0 ** -40, 1e-6])
def test_the_smallest_caps(B, dev, dtype, news, cap):
    """Every position weighs the same to the last place, whatever its score is (below 0, above, 0 itself).  The bounds of tests/test_gpu_paged.py: a cap may
    be taken for one of up to 2^-40, which moves a score by 2^-39 at most, less than the 4 u that they have for an exponential."""
    c = Case(dtype, 4, 2, 64, 16, [120, 60, 90], news, seed=12)
    c.qkv[1] = 0                                 # (a query of zeros: its scores are 0)
    check_attention(c, *run_attention(B, dev, c, 0.125, cap), 0.125, cap)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,news", [
    ([3000] + [40] * 9, [1] * 10),               # in other parts than by itself
    ([3000] + [30] * 140, [1] * 141),            # 564 tiles of the four heads: not cut at all
    ([2000, 300, 350], [1, 300, 350]),           # one token in a tile of 128 columns (32 in fp32)
    ([700] + [20] * 70, [60] + [1] * 70),        # a chunk through tiles of 16 columns
])
def test_a_sequence_alone_and_beside_others(B, dev, dtype, lens, news):
    """How the positions are cut and which kernel runs follow from the whole batch, so sums are taken in other orders: within the bounds, both times."""
    c = Case(dtype, 4, 4, 64, 16, lens, news, seed=13, spare=0)
    out, lse = run_attention(B, dev, c, 0.125, 30.0)
    check_attention(c, out, lse, 0.125, 30.0)
    pages = c.upload(dev)
    pages.seqs = 1
    c.lens, c.news, c.starts = c.lens[:1], c.news[:1], c.starts[:2]
    alone, sums = run_attention(B, dev, c, 0.125, 30.0, pages=pages)
    check_attention(c, alone, sums, 0.125, 30.0)
    again = run_attention(B, dev, c, 0.125, 30.0, pages=pages)
    assert np.array_equal(alone, again[0]) and np.array_equal(sums, again[1])            # the same call gives the same bits


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("news", [[1, 1], [50, 20]])
def test_pages_filled_from_the_host(B, head_dim, news):
    """bf16 pages that are given their contents as f32: what the same numbers cast on the device give, bit by bit."""
    from alpha2_amd import Pages, TensorData
    rs = np.random.RandomState(14)
    i32 = lambda x: TensorData(np.shape(x), "i32", np.asarray(x, np.int32))
    host = [rs.standard_normal(6 * 16 * 2 * head_dim).astype(np.float32) for _ in range(2)]
    starts = np.cumsum([0] + news)
    q = B.castStore(TensorData((int(starts[-1]), 4 * head_dim), "f32", rs.standard_normal(int(starts[-1]) * 4 * head_dim)), "bf16")
    results = []
    for by_hand in (False, True):
        if by_hand:
            k, v = B.newPages(6, 16, 2, head_dim, "bf16")
            k.data, v.data = host
        else:
            k, v = (B.castStore(TensorData((6, 16, 2, head_dim), "f32", x), "bf16") for x in host)
        r = B.pagedAttention(Pages(k, v, i32([[3, 0, 5, 2], [1, 4, 0, 3]]), i32(starts), i32([60, 40])), q, 4, 0.1, 0.0)
        results.append((r["output"].data.copy(), r["lse"].data.copy(), k.data.copy(), v.data.copy()))
    for a, b in zip(*results):
        assert np.array_equal(a, b)
    assert np.array_equal(results[0][2].view(np.uint32) >> 16, to_bf16(host[0]).astype(np.uint32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at", [0, 1])
def test_the_largest_vocabulary(B, dev, dtype, at):
    """2^20 logits, at a whole 16 bytes and one logit behind it.  All equal: their weights add up to 2^63 units, and the numbers lie half way between borders.
    A thousand that count among others 60 below: borders a thousandth apart, the first and the last logit among them."""
    V, rs = 1 << 20, np.random.RandomState(15)
    half = lambda *n: ((np.array(n) + 0.5) / V).astype(np.float32)
    equal = np.zeros((4, V), np.float32)
    flat = to_bf16(equal) if dtype == ffi.BF16 else equal
    e = (4 if dtype == ffi.F32 else 2) * at
    check_sample(B, dev, dtype, flat, np.ones(4), np.array([0, 40, V // 2, 0]), np.array([1.0, 1.0, float(half(70000)[0]), float(half(3)[0])]), None,
                 half(0, V - 1, V // 3, V // 2), at=e, ld=V + 8)
    x = np.full((5, V), -60.0, np.float32)
    for r in range(5):
        ids = np.concatenate([[0, V - 1], rs.choice(np.arange(1, V - 1), 998, replace=False)])
        x[r, ids] = rs.standard_normal(1000)
    logits = to_bf16(x) if dtype == ffi.BF16 else x
    check_sample(B, dev, dtype, logits, np.array([0.0, 1.0, 0.8, 0.9, 1.2]), np.array([0, 0, 40, 0, 700]), np.array([1.0, 1.0, 1.0, 0.9, 1.0]),
                 np.array([0.0, 0.0, 0.0, 0.0, 0.05]), np.array([0.5, 0.71, 0.33, 0.64, 0.97], np.float32), at=e, ld=V + 8)
