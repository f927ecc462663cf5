"""Several sequences through one model: HipBackend's operators on pages as a model calls them, and the generation that is built on them."""
import math

import numpy as np
import pytest

from test_gpu_decode import _logits64, _model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def B():
    from alpha2_amd import HipBackend
    return HipBackend(0)


@pytest.fixture(scope="module")
def F():
    from alpha2_amd import FastHipBackend
    return FastHipBackend(0)


def _rows(B, cfg, params, prompts, passes, release=True):
    """The logits behind the last token of every sequence that a pass has: `passes` is a list of {sequence: tokens of it}."""
    from alpha2_amd.decode import PagedContext
    kept = PagedContext.of(cfg, params, B, [len(p) for p in prompts])
    at, out = [0] * len(prompts), []
    for counts in passes:
        seqs, new = list(counts), []
        for s in seqs:
            new.append(prompts[s][at[s]:at[s] + counts[s]])
            at[s] += counts[s]
        logits = kept.forward(seqs, [counts[s] for s in seqs], np.concatenate(new), range(len(seqs)), B.releaseGpuTensor if release else None)
        out.append([(s, at[s], row) for s, row in zip(seqs, logits.data.reshape(len(seqs), -1).copy())])
    kept.close()
    return out


# sequences of one token, shorter and longer than a page, one that ends with it; passes with prompts, pieces of them and single tokens, in other orders
LENGTHS = [1, 64, 150, 65, 130]
PASSES = [{0: 1, 1: 63, 2: 70}, {3: 64}, {2: 1, 1: 1}, {2: 60, 4: 129, 3: 1}, {4: 1, 2: 19}]


@pytest.mark.parametrize("vocab,layers,width,heads,more", [
    (7, 1, 8, 1, dict()),
    (97, 2, 64, 4, dict(softCap=0.0)),
    (256, 2, 256, 8, dict(ffnActivation="swiglu")),
    (301, 2, 768, 12, dict(ffnActivation="kan_spline")),
    (64, 1, 1024, 8, dict(ffnActivation="relu")),
])
def test_logits_of_several_sequences(B, vocab, layers, width, heads, more):
    """fp32: as near to 64 bits as the pass over each whole context is (one bound for both: the same terms are summed in fp32, in other
    orders; root mean square over the rows, 1.5 times for the scatter, and the bound of single roundings that tests/test_gpu_decode.py
    derives for sums that are short)."""
    from alpha2_amd.sample import _lastRow
    cfg, params = _model(B, vocab, 160, layers, width, heads, **more)
    rs = np.random.RandomState(1)
    prompts = [rs.randint(0, vocab, n).astype(np.int32) for n in LENGTHS]
    exact = [_logits64(cfg, params, p) for p in prompts]
    off = lambda row, want: np.linalg.norm(row.astype(np.float64) - want) / np.linalg.norm(want)
    ours, theirs = [], []
    for rows in _rows(B, cfg, params, prompts, PASSES):
        for s, n, row in rows:
            ours.append(off(row, exact[s][n - 1]))
            theirs.append(off(_lastRow(cfg, params, B, prompts[s][:n], B.releaseGpuTensor), exact[s][n - 1]))
    ours, theirs = (math.sqrt(np.mean(np.square(e))) for e in (ours, theirs))
    print("off 64 bits: in pages %.2e, by itself %.2e" % (ours, theirs))
    assert ours <= max(1.5 * theirs, 8 * (layers + 1) * 2.0 ** -24)


@pytest.mark.parametrize("width,heads", [(64, 4), (256, 2)])
def test_logits_in_bf16(F, width, heads):
    """The fast backend keeps bf16 in the pages: as near to 64 bits as its own pass over the whole context, whose projections, weights of
    the softmax and outputs are rounded to bf16 in the same places."""
    from alpha2_amd.sample import _lastRow
    cfg, params = _model(F, 101, 160, 2, width, heads)
    rs = np.random.RandomState(2)
    prompts = [rs.randint(0, 101, n).astype(np.int32) for n in LENGTHS]
    off = lambda row, want: np.linalg.norm(row.astype(np.float64) - want) / np.linalg.norm(want)
    exact = [_logits64(cfg, params, p) for p in prompts]
    ours, theirs = [], []
    for rows in _rows(F, cfg, params, prompts, PASSES):
        for s, n, row in rows:
            ours.append(off(row, exact[s][n - 1]))
            theirs.append(off(_lastRow(cfg, params, F, prompts[s][:n], F.releaseGpuTensor), exact[s][n - 1]))
    ours, theirs = (math.sqrt(np.mean(np.square(e))) for e in (ours, theirs))
    print("off 64 bits: in pages %.2e, by itself %.2e" % (ours, theirs))
    assert ours <= 1.5 * theirs


def test_released_or_collected(B):
    """The same bits whether tensors are released as they are done with or collected."""
    cfg, params = _model(B, 50, 160, 1, 64, 2)
    rs = np.random.RandomState(3)
    prompts = [rs.randint(0, 50, n).astype(np.int32) for n in LENGTHS]
    a, b = (_rows(B, cfg, params, prompts, PASSES, release) for release in (True, False))
    for x, y in zip(a, b):
        for (_, _, p), (_, _, q) in zip(x, y):
            assert np.array_equal(p, q)


GENERATE = [(0.0, 0, 1.0), (0.8, 40, 1.0), (1.0, 5, 0.9), (1.2, 0, 0.6), (0.7, 0, None)]


def test_generated_tokens_are_those_of_each_by_itself(B):
    """fp32 roundings move a choice only where a draw lands within about 1e-6 of a boundary."""
    from alpha2_amd.rng import SeededRng
    from alpha2_amd.sample import SampleConfig, sampleTokens, sampleTokensBatch
    cfg, params = _model(B, 80, 90, 2, 64, 2)
    rs = np.random.RandomState(4)
    prompts = [rs.randint(0, 80, n).tolist() for n in (1, 4, 70, 64, 30, 90, 9)]
    configs = [SampleConfig(steps=n, temperature=t, topk=k, topp=p) for n, (t, k, p) in zip((40, 3, 40, 26, 1, 5, 0), GENERATE + GENERATE)]
    want = [sampleTokens(cfg, params, B, SeededRng(20 + i), p, c, B.releaseGpuTensor, B.flush) for i, (p, c) in enumerate(zip(prompts, configs))]
    rngs = [SeededRng(20 + i) for i in range(len(prompts))]
    got = sampleTokensBatch(cfg, params, B, rngs, prompts, configs, B.releaseGpuTensor, B.flush)
    assert [t.size for t in got] == [41, 7, 90, 90, 31, 90, 9]
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == np.int32 and np.array_equal(a, b), i
    # each rng has been asked as often: what it gives next is the same
    for i, c in enumerate(configs):
        other = SeededRng(20 + i)
        for _ in range(got[i].size - len(prompts[i]) if c.temperature > 0 else 0):
            other.next()
        assert rngs[i].next() == other.next()
    # one sequence; and nothing to do
    one = sampleTokensBatch(cfg, params, B, [SeededRng(21)], prompts[1:2], configs[1])
    assert np.array_equal(one[0], want[1])
    assert sampleTokensBatch(cfg, params, B, [], [], SampleConfig()) == []


def test_prompts_in_pieces(B, monkeypatch):
    """Fewer rows to a pass than the prompts have: the same tokens."""
    from alpha2_amd.decode import PagedContext
    from alpha2_amd.rng import SeededRng
    from alpha2_amd.sample import SampleConfig, sampleTokensBatch
    cfg, params = _model(B, 80, 200, 1, 64, 2)
    rs = np.random.RandomState(5)
    prompts = [rs.randint(0, 80, n).tolist() for n in (100, 1, 150, 20)]
    run = lambda: sampleTokensBatch(cfg, params, B, [SeededRng(i) for i in range(4)], prompts, SampleConfig(steps=12, temperature=1.0, topk=0), B.releaseGpuTensor)
    whole = run()
    monkeypatch.setattr(PagedContext, "MOST_ROWS", 48)
    for a, b in zip(run(), whole):
        assert np.array_equal(a, b)


def test_generation_on_the_fast_backend(F):
    """Greedy, bf16: the logits differ by roundings, so a token may be another one where two are as likely; each token chosen is, by the
    pass over its whole context, within those roundings of the largest logit: 2^-8 for each of the eight roundings to bf16 that follow
    one another in a block and before the head, of the row's norm."""
    from alpha2_amd.rng import SeededRng
    from alpha2_amd.sample import SampleConfig, _lastRow, sampleTokensBatch
    cfg, params = _model(F, 80, 90, 2, 64, 2)
    rs = np.random.RandomState(6)
    prompts = [rs.randint(0, 80, n).astype(np.int32) for n in (3, 64, 70)]
    got = sampleTokensBatch(cfg, params, F, [SeededRng(1)] * 3, prompts, SampleConfig(steps=8, temperature=0.0, topk=0), F.releaseGpuTensor, F.flush)
    for t, p in zip(got, prompts):
        assert t.size == p.size + 8 and np.array_equal(t[:p.size], p)
        for n in range(p.size, t.size):
            row = _lastRow(cfg, params, F, t[:n], F.releaseGpuTensor)
            assert row[t[n]] >= row.max() - 8 * (cfg.nLayer + 1) * 2.0 ** -8 * np.linalg.norm(row)


def test_memory_goes_back(B):
    from alpha2_amd.rng import SeededRng
    from alpha2_amd.sample import SampleConfig, sampleTokensBatch
    cfg, params = _model(B, 80, 90, 2, 64, 2)
    run = lambda: sampleTokensBatch(cfg, params, B, [SeededRng(i) for i in range(3)], [[1], [2, 3], [4, 5, 6]], SampleConfig(steps=20), B.releaseGpuTensor, B.flush)
    run()
    live = B.gpuMemStats()["liveAllocs"]
    run()
    assert B.gpuMemStats()["liveAllocs"] <= live


def test_step_plans_around_generation(B):
    """With the steps recorded and replayed between flushes: the same tokens."""
    from alpha2_amd.rng import SeededRng
    from alpha2_amd.sample import SampleConfig, sampleTokensBatch
    cfg, params = _model(B, 80, 90, 1, 64, 2)
    run = lambda: sampleTokensBatch(cfg, params, B, [SeededRng(i) for i in range(3)], [[1], [2, 3], [4, 5, 6]], SampleConfig(steps=60), B.releaseGpuTensor, B.flush)
    want = run()
    B.enableStepGraphs(True)
    try:
        got = run()
        again = run()
    finally:
        B.enableStepGraphs(False)
    for a, b, c in zip(want, got, again):
        assert np.array_equal(a, b) and np.array_equal(a, c)


def test_parameters_that_move(B):
    """flushGpu of the caller's own may move the parameters: their places are looked up in every pass."""
    from alpha2_amd.model import collectParamEntries
    from alpha2_amd.rng import SeededRng
    from alpha2_amd.sample import SampleConfig, sampleTokensBatch
    cfg, params = _model(B, 80, 90, 1, 64, 2)
    config = SampleConfig(steps=30, temperature=1.0, topk=0)
    run = lambda flush: sampleTokensBatch(cfg, params, B, [SeededRng(i) for i in range(2)], [[1], [2, 3]], config, B.releaseGpuTensor, flush)
    want = run(None)

    def move():
        for _, v in collectParamEntries(params):
            host = v.data.data.copy()
            B.releaseGpuTensor(v.data)
            v.data.data = host
    for a, b in zip(run(move), want):
        assert np.array_equal(a, b)


# ------------------------------------------------------------------------------------ the operators by themselves
def _tensor(x, dtype="f32"):
    from alpha2_amd import TensorData
    return TensorData(x.shape, dtype, x)


@pytest.mark.parametrize("store", ["f32", "bf16"])
@pytest.mark.parametrize("neighbours", [False, True])
def test_rotated_grouped_and_sampled(B, F, store, neighbours):
    """Rotation, heads that share keys and selection in one run, against loops in 64 bits, on the backend's methods.  Tolerances: those
    of tests/test_gpu_paged.py, loosened to the worst over a row (the scores here stay below 8, sums below 40 terms: 2^-24 times a few
    hundred; bf16: 2^-8 for q, k, v as stored, the weights, and the result, against what was stored)."""
    backend = B if store == "f32" else F
    H, KH, D, R, page, rs = 6, 2, 16, 8, 5, np.random.RandomState(7)
    from alpha2_amd import Pages
    lens, news = [9, 1, 23], [4, 1, 7]
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    rows, width = int(starts[-1]), 5
    table = rs.permutation(3 * width).astype(np.int32).reshape(3, width)
    angles = np.arange(32)[:, None] * 10.0 ** -np.arange(R // 2)
    rotary = np.concatenate([np.cos(angles), np.sin(angles)], 1).astype(np.float32)
    k, v = backend.newPages(3 * width, page, KH, D, store)
    for t in (k, v):                             # earlier positions hold what was written there before
        host = np.round(rs.standard_normal(t.size) * 64).astype(np.float32) / 64        # (exact in bf16)
        src = backend.castStore(_tensor(host.reshape(t.shape)), store)
        backend._ptr(src)
        t._buf, t._host_valid = src._buf, False
        src._buf.refs += 1
    qkv = np.round(rs.standard_normal((rows, (H + 2 * KH) * D)) * 32).astype(np.float32) / 32
    pages = Pages(k, v, _tensor(table, "i32"), _tensor(starts, "i32"), _tensor(np.array(lens, np.int32), "i32"))
    before_k, before_v = (t.data.reshape(t.shape).astype(np.float64).copy() for t in (k, v))
    x = backend.castStore(_tensor(qkv), store)
    q = backend.pagedAppend(pages, x, H, _tensor(rotary), neighbours)
    r = backend.pagedAttention(pages, q, H, 0.25, 20.0)
    assert q.store == r["output"].store == store and q.shape == r["output"].shape == (rows, H * D) and r["lse"].shape == (rows, H)
    after_k, after_v = (t.data.reshape(t.shape).astype(np.float64) for t in (k, v))
    h = 2.0 ** -8 if store == "bf16" else 2.0 ** -23

    def turn(x, p):                              # [heads, D]
        c, s = rotary[p, :R // 2].astype(np.float64), rotary[p, R // 2:].astype(np.float64)
        y = x.copy()
        i, j = (np.arange(0, R, 2), np.arange(1, R, 2)) if neighbours else (np.arange(R // 2), np.arange(R // 2, R))
        y[:, i], y[:, j] = x[:, i] * c - x[:, j] * s, x[:, j] * c + x[:, i] * s
        return y
    want_k, want_v = before_k.copy(), before_v.copy()
    got_q, out, lse = (t.data.reshape(rows, H, -1).astype(np.float64) for t in (q, r["output"], r["lse"]))
    for s in range(3):
        for row in range(starts[s], starts[s + 1]):
            p = lens[s] - starts[s + 1] + row
            parts = qkv[row].astype(np.float64).reshape(-1, D)
            assert np.abs(got_q[row] - turn(parts[:H], p)).max() <= 2 * h * 5
            want_k[table[s, p // page], p % page], want_v[table[s, p // page], p % page] = turn(parts[H:H + KH], p), parts[H + KH:]
    assert np.abs(after_k - want_k).max() <= 2 * h * 5 and np.array_equal(after_v, want_v)
    for s in range(3):
        for row in range(starts[s], starts[s + 1]):
            seen = np.arange(lens[s] - starts[s + 1] + row + 1)
            K, V = (t[table[s, seen // page], seen % page] for t in (after_k, after_v))
            for i in range(H):
                z = 20 * np.tanh(0.25 * K[:, i * KH // H] @ got_q[row, i] / 20)
                w = np.exp(z - z.max())
                o = w @ V[:, i * KH // H] / w.sum()
                near = (w @ np.abs(V[:, i * KH // H]) / w.sum()).max()
                assert np.abs(out[row, i] - o).max() <= (3 * h + 2.0 ** -15) * near
                assert abs(lse[row, i, 0] - (z.max() + math.log(w.sum()))) <= 2.0 ** -15 + (0 if store == "f32" else 2 * h)
    logits = backend.castStore(_tensor(qkv), store)
    n = rows
    picks = backend.sampleRows(logits, _tensor(np.full(n, 0.5, np.float32)), _tensor(np.linspace(0, 1, n).astype(np.float32)), _tensor(np.arange(n, dtype=np.int32), "i32"))
    for i, (token, logprob) in enumerate(zip(picks["tokens"].data, picks["logprobs"].data)):
        row, t = qkv[i].astype(np.float64), np.linspace(0, 1, n).astype(np.float32)[i]
        if t == 0:
            assert token == row.argmax()
            continue
        w = np.exp((row - row.max()) / t) * (row >= (np.sort(row)[-i] if i else -np.inf))
        run = np.cumsum(w) / w.sum()
        assert run[token] >= 0.5 - 1e-6 and (token == 0 or run[token - 1] <= 0.5 + 1e-6) and w[token] > 0
        assert abs(logprob - math.log(w[token] / w.sum())) < 1e-5


def test_a_clone_of_the_pages_stays(B):
    from alpha2_amd import Pages
    k, v = B.newPages(2, 4, 1, 8)
    for t in (k, v):
        B.scaleInplace(t, 0.0)
    held = B.clone(k)
    before = held.data.copy()
    i32 = lambda *x: _tensor(np.array(x, np.int32), "i32")
    pages = Pages(k, v, _tensor(np.array([[1]], np.int32), "i32"), i32(0, 2), i32(2))
    B.pagedAppend(pages, _tensor(np.ones((2, 24), np.float32)), 1)
    assert np.array_equal(held.data, before)
    assert np.array_equal(B.clone(held).data, before) and (k.data.reshape(2, 4, 8)[1, :2] == 1).all()
