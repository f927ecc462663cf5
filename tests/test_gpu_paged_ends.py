"""Pages and sampling at the ends of what they take: caps, vocabularies, rows and tables, other strides, pages filled from the host, a sequence alone and beside others, two contexts at once."""
import numpy as np
import pytest

from alpha2_amd import _ffi as ffi
from test_gpu_paged import TYPES, B, Case, check_attention, dev, run_append, run_attention, to_bf16, values  # noqa: F401 (fixtures)
from test_gpu_sample import check as check_sample, run as run_sample

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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [[1, 2, 1], [40, 3, 70]])
def test_heads_before_rows(B, dev, dtype, news):
    """q, k, v, rotated and o as [heads][rows][D], rows apart by more than D: the bits of [rows][heads][D]."""
    c = Case(dtype, 4, 2, 64, 16, [120, 60, 90], news, seed=16)
    want_o, want_l = run_attention(B, dev, c, 0.125, 30.0)
    D, apart = c.D, c.D + 16
    raw = c.qkv[:, :8 * D].reshape(c.rows, 8, D)
    heads_first = np.zeros((8, c.rows, apart), raw.dtype)
    heads_first[:, :, :D] = raw.transpose(1, 0, 2)
    at = dev.put(heads_first)
    out, sums = np.full((4, c.rows, apart), 7, raw.dtype), np.full((c.rows, 4), 7, np.float32)
    o, l = dev.put(out), dev.put(sums)
    pages = c.upload(dev)
    ffi.check(B.lib.ah_paged_attention(pages, ffi.AhPagedAttention(c.rows, 4, 0.125, 30.0, apart, c.rows * apart, apart, c.rows * apart, at, o, l)))
    got, n = dev.get(o, out), int(c.starts[-1])
    assert np.array_equal(got[:, :n, :D].transpose(1, 0, 2), want_o[:n]) and np.array_equal(dev.get(l, sums)[:n], want_l[:n])
    assert (got[:, n:] == 7).all() and (got[:, :, D:] == 7).all()
    for rot, neighbours in ((32, False), (32, True), (20, False)):
        k, v, turned, table = run_append(B, dev, c, rot, neighbours)
        pages = c.upload(dev)
        row, head = apart, c.rows * apart
        r, e = dev.put(out), head * raw.itemsize
        ffi.check(B.lib.ah_paged_append(pages, ffi.AhPagedAppend(c.rows, 4, rot, len(table), int(neighbours), 0, row, head, row, head, row, head, row, head,
                                                                  at, at + 4 * e, at + 6 * e, r, dev.put(table))))
        got = dev.get(r, out)
        assert np.array_equal(got[:, :n, :D].transpose(1, 0, 2), turned[:n]) and (got[:, n:] == 7).all() and (got[:, :, D:] == 7).all()
        assert np.array_equal(dev.get(c.at["k"], c.k), k) and np.array_equal(dev.get(c.at["v"], c.v), v)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("none", ["table_pages", "pages"])
def test_a_table_of_no_entries_and_a_cache_of_no_pages(B, dev, dtype, new, none):
    """Nothing is read or written there: the tokens that have a position get NaN, those that have none 0."""
    c = Case(dtype, 2, 2, 64, 16, [60, 0], [new, 2], seed=17)
    pages = c.upload(dev)
    setattr(pages, none, 0)
    pages.k = pages.v = pages.table = 0
    out, lse = run_attention(B, dev, c, 0.125, 0.0, pages=pages)
    assert np.isnan(values(out[:new])).all() and np.isnan(lse[:new]).all()
    assert (values(out[new:new + 2]) == 0).all() and (lse[new:new + 2] == -np.inf).all() and (values(out[new + 2:]) == 7).all()
    q, k, v = c.offsets()
    ffi.check(B.lib.ah_paged_append(pages, ffi.AhPagedAppend(c.rows, 0, 0, 0, 0, 0, 0, 0, c.pitch, c.D, c.pitch, c.D, 0, 0, 0, k, v, 0, 0)))
    assert np.array_equal(dev.get(c.at["k"], c.k), c.k) and np.array_equal(dev.get(c.at["v"], c.v), c.v)


def test_more_rows_than_16_bits_count(B, dev):
    rs = np.random.RandomState(18)
    rows = 70001
    logits = rs.randint(-8, 8, (rows, 8)).astype(np.float32)
    tokens, _ = run_sample(B, dev, ffi.F32, logits, t=np.zeros(rows), u=np.zeros(rows))
    assert np.array_equal(tokens, logits.argmax(1))
    low = np.where(logits == logits.max(1, keepdims=True), 0.0, -200.0).astype(np.float32)        # (as good as none: 2^-43 of the others is nothing)
    tokens, logp = run_sample(B, dev, ffi.F32, low, u=np.zeros(rows))
    assert np.array_equal(tokens, low.argmax(1)) and np.allclose(logp, -np.log((low == 0).sum(1)), rtol=2.0 ** -23, atol=2.0 ** -40)


def test_step_plans_around_generation_on_the_fast_backend():
    from alpha2_amd import FastHipBackend
    from alpha2_amd.rng import SeededRng
    from alpha2_amd.sample import SampleConfig, sampleTokensBatch
    from test_gpu_decode import _model
    F = FastHipBackend(0)
    cfg, params = _model(F, 80, 90, 2, 64, 2)
    run = lambda: sampleTokensBatch(cfg, params, F, [SeededRng(i) for i in range(3)], [[1], [2, 3], [4, 5, 6]], SampleConfig(steps=40), F.releaseGpuTensor, F.flush)
    want = run()
    F.enableStepGraphs(True)
    try:
        got = [run() for _ in range(3)]
    finally:
        F.enableStepGraphs(False)
    for tokens in got:
        assert all(np.array_equal(a, b) for a, b in zip(tokens, want))


def test_two_generations_side_by_side(B):
    """Two contexts whose passes alternate, over the library's one scratch: each gives the bits that it gives alone."""
    from alpha2_amd.decode import PagedContext
    from test_gpu_decode import _model
    cfg, params = _model(B, 50, 700, 2, 64, 2)
    rs = np.random.RandomState(19)
    texts = [[rs.randint(0, 50, n).astype(np.int32) for n in lens] for lens in ((650, 30), (10, 690, 600))]

    def passes(kept, prompts):
        new = [p[:-4] for p in prompts]
        yield kept.forward(range(len(prompts)), [p.size for p in new], np.concatenate(new), range(len(prompts)), B.releaseGpuTensor).data.copy()
        for i in range(-4, 0):
            yield kept.forward(range(len(prompts)), [1] * len(prompts), np.array([p[i] for p in prompts]), range(len(prompts)), B.releaseGpuTensor).data.copy()
    kept = [[PagedContext.of(cfg, params, B, [p.size for p in prompts]) for prompts in texts] for _ in range(2)]
    alone = [list(passes(k, prompts)) for k, prompts in zip(kept[0], texts)]
    together = list(zip(*(passes(k, prompts) for k, prompts in zip(kept[1], texts))))
    for k in kept[0] + kept[1]:
        k.close()
    for i, both in enumerate(together):
        assert all(np.array_equal(x, alone[j][i]) for j, x in enumerate(both))
