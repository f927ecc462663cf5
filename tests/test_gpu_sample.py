"""The next token from logits and given random numbers (ah_sample) against the definition in 64 bits.

Tokens have to be equal.  The kernel's weights are whole numbers of 2^-43 of the largest, from an exponential good to 2^-43, so a running sum of n of them is off by n (2^-44 + 2^-43)
at most: where the given number falls nearer than 2 n 2^-43 to a border between two tokens, or the
nucleus ends that near to one, either may be chosen; the cases below are looked at for that (`margin`) and are never so near.
logprob: its exponent and the logarithm of the sum are taken in 64 bits and rounded once, 2^-24 of its value, and the sum is off by the above."""
import ctypes as C
import math

import numpy as np
import pytest

from alpha2_amd import _ffi as ffi
from test_gpu_paged import Device, to_bf16, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def B():
    from alpha2_amd import HipBackend
    return HipBackend(0)


@pytest.fixture()
def dev(B):
    d = Device(B)
    yield d
    d.close()


def choose(logits, t, k, p, m, u):
    """(token, logprob, margin) of one row in 64 bits."""
    l = logits.astype(np.float64)
    V, ids = l.size, np.arange(l.size)
    fine = l > -np.inf                            # NaN is not
    if not fine.any():
        return 0, math.nan, math.inf
    top = l[fine].max()
    if not t > 0:
        return int(np.nonzero(l == top)[0][0]), 0.0, math.inf
    with np.errstate(invalid="ignore"):
        w = np.where(fine, np.where(l == top, 1.0, np.exp((l - top) / t)), 0.0)
    order = ids[fine][np.argsort(-l[fine], kind="stable")]
    keep, margin = fine.copy(), math.inf
    if 0 < k < V and order.size > k:
        keep &= l >= l[order[k - 1]]
    order = order[keep[order]]
    nucleus = 0 < p < 1
    if nucleus:
        mass = np.cumsum(w[order])
        target = float(p) * mass[-1]
        n = int(np.searchsorted(mass, target))
        margin = min(margin, abs(mass - target).min())
        keep[order[n + 1:]] = False
    if m > 0:
        keep &= w >= min(float(m), 1.0)
    order = order[keep[order]]
    if not nucleus:
        order = np.sort(order)
    mass = np.cumsum(w[order])
    target = min(max(float(u), 0.0) if u == u else 0.0, 1.0) * mass[-1]
    n = int(np.searchsorted(mass, target, side="right"))
    if 0 < target < mass[-1]:
        margin = min(margin, abs(mass - target).min())
    weighs = np.nonzero(w[order] > 2.0 ** -44)[0]
    token = int(order[min(n, weighs[-1])])
    with np.errstate(divide="ignore"):
        return token, (0.0 if l[token] == top else (l[token] - top) / t) - math.log(mass[-1]), margin


def run(B, dev, dtype, logits, t=None, k=None, p=None, m=None, u=None, ld=None, at=0, logprobs=True):
    """`logits`: as they are stored.  None: no such array."""
    rows, V = logits.shape
    ld = V if ld is None else ld
    wide = np.zeros((rows, ld), logits.dtype)
    wide[:] = np.float32(50).astype(np.float32) if dtype == ffi.F32 else 0x4248      # what lies between the rows must not be read
    wide[:, :V] = logits
    tokens, logp = np.full(rows + 1, 77, np.int32), np.full(rows + 1, 7, np.float32)
    put = lambda x, kind: 0 if x is None else dev.put(np.asarray(x, kind))
    a, b = dev.put(tokens), dev.put(logp)
    ffi.check(B.lib.ah_sample(ffi.AhSample(dtype, V, rows, ld, dev.put(wide, at), put(t, np.float32), put(k, np.int32), put(p, np.float32), put(m, np.float32),
                                           put(u, np.float32), a, b if logprobs else 0)))
    tokens, logp = dev.get(a, tokens), dev.get(b, logp)
    assert tokens[-1] == 77 and logp[-1] == 7
    return tokens[:-1], logp[:-1]


def check(B, dev, dtype, logits, t, k, p, m, u, **more):
    rows, V = logits.shape
    full = lambda x, off: np.broadcast_to(np.asarray(off if x is None else x), (rows,))
    got, logp = run(B, dev, dtype, logits, t, k, p, m, u, **more)
    for r in range(rows):
        want, lp, margin = choose(values(logits[r]), *(np.float32(x[r]) if i != 1 else int(x[r]) for i, x in enumerate((full(t, 1.0), full(k, 0), full(p, 1.0), full(m, 0.0), full(u, 0.0)))))
        assert margin > 2 * V * 2.0 ** -43, (r, margin)
        assert got[r] == want, (r, got[r], want, margin)
        assert (math.isnan(lp) and math.isnan(logp[r])) or abs(logp[r] - lp) <= 2.0 ** -24 * abs(lp) + V * 2.0 ** -42, (r, logp[r], lp)


def model_logits(rs, rows, V, dtype, spread=1.1):
    rank = np.argsort(rs.random_sample((rows, V)), 1)
    x = (rs.standard_normal((rows, V)) - spread * np.log1p(rank)).astype(np.float32)
    return to_bf16(x) if dtype == ffi.BF16 else x


TYPES = [ffi.F32, ffi.BF16]
SETTINGS = {"greedy": (0.0, None, None, None), "plain": (1.0, None, None, None), "default": (0.8, 40, None, None), "nucleus": (0.9, None, 0.9, None),
            "least": (1.2, None, None, 0.05), "all": (0.7, 50, 0.8, 0.01), "wide": (1.5, 500, 0.99, None), "narrow": (0.3, 1, 0.05, 1.0)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 63, 64, 256, 257, 1000, 4096, 50304, 53249, 131072])
@pytest.mark.parametrize("name", list(SETTINGS))
def test_tokens_are_those_of_the_definition(B, dev, dtype, V, name):
    t, k, p, m = SETTINGS[name]
    rs = np.random.RandomState(V + len(name))
    rows = 7 if V <= 4096 else 3
    logits = model_logits(rs, rows, V, dtype)
    every = lambda x: None if x is None else np.full(rows, x)
    check(B, dev, dtype, logits, every(t), every(k), every(p), every(m), rs.random_sample(rows).astype(np.float32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,rows", [(300, 300), (5000, 40)])
def test_every_row_has_its_own_choice(B, dev, dtype, V, rows):
    rs = np.random.RandomState(1)
    on = lambda p, x, off: np.where(rs.random_sample(rows) < p, x, off)
    check(B, dev, dtype, model_logits(rs, rows, V, dtype), on(0.8, 0.2 + 2 * rs.random_sample(rows), 0.0), on(0.5, rs.randint(1, V + 2, rows), 0),
          on(0.5, rs.random_sample(rows), 1.0), on(0.3, 0.3 * rs.random_sample(rows), 0.0), rs.random_sample(rows).astype(np.float32), ld=V + 3, at=12 if dtype == ffi.F32 else 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 2500, 60000])
def test_equal_logits(B, dev, dtype, V):
    """All equal, few values, and the k-th among many equal ones: those stay, a nucleus takes the lower indices."""
    rs = np.random.RandomState(2)
    rows = 12
    x = np.stack([np.full(V, 1.5), rs.randint(0, 3, V), np.where(rs.random_sample(V) < 0.5, 2.0, -1.0), -np.arange(V) // 7] * 3).astype(np.float32)
    x[4:8] = np.where(x[4:8] == 0, -0.0, x[4:8])
    logits = to_bf16(x) if dtype == ffi.BF16 else x
    u = (rs.randint(0, 1000, rows) / 1000 + 0.00037).astype(np.float32)
    check(B, dev, dtype, logits, np.full(rows, 0.9), np.array([0] * 4 + [10] * 4 + [V // 2] * 4), np.array([1.0] * 2 + [0.7013] * 6 + [1.0, 0.4007, 0.9011, 1.0]),
          np.array([0.0] * 6 + [0.2] * 6), u)


def test_the_ends_of_the_random_numbers(B, dev):
    """0 gives the first of what is kept, 1 (and what is nearest below it) the last that weighs, NaN and negative ones count as 0, larger ones as 1."""
    rs = np.random.RandomState(3)
    x = model_logits(rs, 1, 600, ffi.F32)[0]
    u = np.array([0.0, -0.5, np.nan, 1.0, 2.0, np.inf, -np.inf], np.float32)
    for k, p in ((None, None), (30, None), (30, 0.8), (None, 0.9)):
        logits = np.stack([x] * u.size)
        check(B, dev, ffi.F32, logits, np.full(u.size, 0.8), None if k is None else np.full(u.size, k), None if p is None else np.full(u.size, p), None, u)


@pytest.mark.parametrize("V", [50, 5000])
def test_infinite_and_missing_logits(B, dev, V):
    rs = np.random.RandomState(4)
    x = np.stack([model_logits(rs, 1, V, ffi.F32)[0] for _ in range(10)])
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, 1:] = -np.inf
    x[3, :V - 3] = np.nan
    x[4, 7] = np.inf
    x[5, [3, V - 5]] = np.inf
    x[6, ::2] = -np.inf
    x[7, ::3] = np.nan
    x[8, :] = -3.402823466e38
    x[8, 11] = 3.402823466e38
    x[9, 1:] = -3.402823466e38
    for t, k, p, m in ((0.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.0), (0.7, 20, 1.0, 0.0), (0.7, 20, 0.9, 0.0), (1.3, 0, 0.8, 0.02), (1e-30, 0, 1.0, 0.0), (1e30, 5, 0.999, 0.0)):
        every = lambda v: np.full(10, v)
        check(B, dev, ffi.F32, x, every(t), every(k), every(p), every(m), rs.random_sample(10).astype(np.float32))


def test_settings_that_switch_off(B, dev):
    """NaN and what is outside their ranges: a temperature that is not above 0 is greedy, the others are off."""
    rs = np.random.RandomState(5)
    rows = 12
    x = np.repeat(model_logits(rs, 1, 400, ffi.F32), rows, 0)
    t = np.array([np.nan, -1.0, -np.inf, 0.0] + [0.8] * 8)
    k = np.array([0] * 4 + [-3, 400, 401, 2 ** 31 - 1, 0, 0, 0, 0])
    p = np.array([1.0] * 4 + [np.nan, 0.0, -1.0, 1.0, 1.5, 1.0, 1.0, np.inf])
    m = np.array([0.0] * 4 + [0.0, 0.0, 0.0, 0.0, np.nan, -1.0, 2.0, 0.0])
    check(B, dev, ffi.F32, x, t, k, p, m, rs.random_sample(rows).astype(np.float32))


@pytest.mark.parametrize("dtype", TYPES)
def test_peaked_and_flat_rows(B, dev, dtype):
    """A row that is one token, rows as flat as they come, outliers far below and far above the rest."""
    rs = np.random.RandomState(6)
    V = 20000
    x = np.stack([rs.standard_normal(V) * s for s in (1e-3, 0.1, 1.0, 10.0, 100.0, 1e4)] + [rs.standard_normal(V)] * 2).astype(np.float32)
    x[6, 123] = 1e6
    x[7, 55] = -1e30
    logits = to_bf16(x) if dtype == ffi.BF16 else x
    for k, p in ((0, 1.0), (0, 0.9013), (100, 1.0), (3000, 0.7003)):
        u = (rs.randint(0, 4000, 8) / 4000 + 0.0001237).astype(np.float32)
        check(B, dev, dtype, logits, np.full(8, 0.9), np.full(8, k), np.full(8, p), None, u)


@pytest.mark.parametrize("dtype", TYPES)
def test_logits_that_lie_closer_or_wider_than_bins_can_tell(B, dev, dtype):
    """Neighbouring numbers, the smallest ones and the largest ones, thousands of each; a step of a row's temperature is none of theirs."""
    rs = np.random.RandomState(9)
    V = 9001
    pick = lambda *v: np.asarray(v, np.float32)[rs.randint(0, len(v), V)]
    x = np.stack([pick(0.0, 1e-45, -1e-45), pick(3.4e38, -3.4e38, 0.0), pick(1.0, 1.0 + 2.0 ** -23, 1.0 - 2.0 ** -24), pick(-np.inf, 5.0, 5.0 + 2.0 ** -21),
                  np.where(rs.random_sample(V) < 0.001, 1e5, rs.standard_normal(V) * 1e-3).astype(np.float32), pick(7.0, -1e30, 7.0 - 1e-3)])
    logits = to_bf16(x) if dtype == ffi.BF16 else x
    if dtype == ffi.BF16:
        logits[3] = np.where(np.isneginf(x[3]), 0xff80, logits[3])
    for t, k, p in ((1.0, 0, 0.6007), (1e-3, 0, 0.9003), (1.0, 3000, 1.0), (1e-3, 4500, 0.7013), (1.0, 30, 0.5003)):
        u = (rs.randint(0, 4000, 6) / 4000 + 0.0001237).astype(np.float32)
        check(B, dev, dtype, logits, np.full(6, t, np.float32), np.full(6, k), np.full(6, p), None, u)


def test_the_choice_is_that_of_the_sampling_loop(B, dev):
    """selectToken on the same logits and random numbers (it rounds the scaled logits to fp32: a number within 1e-6 of a border may fall on the other side)."""
    from alpha2_amd.sample import selectToken
    rs = np.random.RandomState(7)

    class Given:
        def __init__(self, u):
            self.u = u

        def next(self):
            return float(self.u)
    rows, V, same = 64, 3001, 0
    logits = model_logits(rs, rows, V, ffi.F32)
    u = rs.random_sample(rows).astype(np.float32)
    t, k, p = np.where(np.arange(rows) % 8 == 0, 0.0, 0.8).astype(np.float32), rs.choice([0, 40, 200], rows), rs.choice([1.0, 0.9, 0.5], rows).astype(np.float32)
    got, _ = run(B, dev, ffi.F32, logits, t, k, p, None, u)
    for r in range(rows):
        _, _, margin = choose(logits[r], t[r], int(k[r]), p[r], 0.0, u[r])
        row = (logits[r].astype(np.float64) / t[r]).astype(np.float32) if t[r] > 0 else logits[r].copy()
        want = selectToken(row, Given(u[r]), float(t[r]), int(k[r]), float(p[r]))
        if margin > 1e-4:
            assert got[r] == want, r
            same += 1
    assert same > 0.8 * rows


def test_a_captured_call_follows_its_arrays_and_no_row_depends_on_another(B, dev):
    rs = np.random.RandomState(8)
    logits = model_logits(rs, 5, 50304, ffi.F32)
    u = rs.random_sample((4, 5)).astype(np.float32)
    t, p = np.full(5, 0.9, np.float32), np.array([1.0, 0.9, 1.0, 0.95, 1.0], np.float32)
    x, uu, tokens = dev.put(logits), dev.put(u[0]), dev.put(np.zeros(5, np.int32))
    d = ffi.AhSample(ffi.F32, 50304, 5, 50304, x, dev.put(t), 0, dev.put(p), 0, uu, tokens, 0)
    ffi.check(B.lib.ah_sample(d))
    g = C.c_uint64()
    ffi.check(B.lib.ah_graph_begin())
    ffi.check(B.lib.ah_sample(d))
    ffi.check(B.lib.ah_graph_end(C.byref(g)))
    try:
        for i in range(4):
            ffi.check(B.lib.ah_upload(uu, u[i].ctypes.data_as(C.c_void_p), 20))
            ffi.check(B.lib.ah_graph_launch(g))
            got = dev.get(tokens, np.zeros(5, np.int32))
            for r in range(5):                    # one row alone
                one = dev.put(np.zeros(1, np.int32))
                ffi.check(B.lib.ah_sample(ffi.AhSample(ffi.F32, 50304, 1, 50304, x + r * 50304 * 4, d.temperature + 4 * r, 0, d.top_p + 4 * r, 0, uu + 4 * r, one, 0)))
                assert dev.get(one, np.zeros(1, np.int32))[0] == got[r]
    finally:
        ffi.check(B.lib.ah_sync())
        ffi.check(B.lib.ah_graph_destroy(g))


def test_no_rows(B, dev):
    ffi.check(B.lib.ah_sample(ffi.AhSample(ffi.F32, 10, 0, 10, 0, 0, 0, 0, 0, 0, 0, 0)))
