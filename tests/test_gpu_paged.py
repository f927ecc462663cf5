"""Keys and values in pages (ah_paged_append, ah_paged_attention) against plain loops in 64 bits.

Tolerances are worst cases of the roundings.  u = 2^-24 (fp32) and, where something is rounded to bf16, h = 2^-8, of its value:
  append     a turned feature x c - y s: two products and a sum, 2 u (|x c| + |y s|), and its own rounding to bf16; anything else is a copy.
  a score    D products and their sum, then the scale: (D + 3) u |scale| sum |q k|; with a cap, whose slope is at most 1, tanh by an
             exponential and a reciprocal to one last place each, 8 u cap more; going over to powers of two and back, 4 u |s|.  Call it e.
  o          a weight is off by e^(2 e) (score and maximum), 4 u for its exponential; the sums over L positions and the joining of parts by
             (L + 16) u; bf16: weights rounded, h, in the product and at most once more in the sum it is divided by, and the result, h.
             All relative to sum w |v|.
  lse        e, (L + 16) u for the sum, 4 u of its value and 4 u for the logarithm's."""
import ctypes as C
import math

import numpy as np
import pytest

from alpha2_amd import _ffi as ffi

pytestmark = pytest.mark.gpu
U, H8 = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module")
def B():
    from alpha2_amd import HipBackend
    return HipBackend(0)


def to_bf16(x):
    """f32 -> bf16 bits, to nearest even (finite values)."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def values(raw):
    return (raw.astype(np.uint32) << 16).view(np.float32) if raw.dtype == np.uint16 else raw


class Device:
    """Arrays on the device, freed at the end."""

    def __init__(self, B):
        self.lib, self.held = B.lib, []

    def put(self, array, at=0):
        """The address of a copy that begins `at` bytes into a block."""
        array = np.ascontiguousarray(array)
        p = C.c_uint64()
        ffi.check(self.lib.ah_alloc(array.nbytes + at + 16, C.byref(p)))
        self.held.append(p.value)
        if array.nbytes:
            ffi.check(self.lib.ah_upload(p.value + at, array.ctypes.data_as(C.c_void_p), array.nbytes))
        return p.value + at

    def get(self, address, like):
        out = np.empty_like(like)
        if out.nbytes:
            ffi.check(self.lib.ah_download(out.ctypes.data_as(C.c_void_p), address, out.nbytes))
        return out

    def close(self):
        for p in self.held:
            ffi.check(self.lib.ah_free(p))


@pytest.fixture()
def dev(B):
    d = Device(B)
    yield d
    d.close()


class Case:
    """Pages, tables and new tokens on the host; `lens` and `news` per sequence."""

    def __init__(self, dtype, heads, kv_heads, D, page, lens, news, seed=0, heads_first=False, spare=2, gap=0, scale=1.0, entries=0, share=None):
        rs = np.random.RandomState(seed)
        self.dtype, self.heads, self.kv_heads, self.D, self.page, self.lens, self.news = dtype, heads, kv_heads, D, page, list(lens), list(news)
        self.store = (lambda x: to_bf16(x)) if dtype == ffi.BF16 else (lambda x: np.asarray(x, np.float32))
        need = [-(-max(n, 0) // page) for n in lens]
        self.pages = sum(need) + 2
        order = rs.permutation(self.pages)
        self.width = max(need + [1]) + entries
        self.table = rs.randint(0, self.pages, (len(lens), self.width)).astype(np.int32)         # entries behind the last are some page or other
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        if share:                                # a first page that two sequences have in common
            self.table[share[1], 0] = self.table[share[0], 0]
        self.starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + spare
        self.pitch = (heads + 2 * kv_heads) * D + gap
        self.qkv = self.store(rs.standard_normal((self.rows, self.pitch)) * scale)
        self.strides = (page * kv_heads * D + 16, D * kv_heads, D) if not heads_first else (page * kv_heads * D + 16, D, page * D)
        size = self.pages * self.strides[0]
        self.k, self.v = (self.store(rs.standard_normal(size) * scale) for _ in range(2))

    def places(self, s, positions):
        """Elements from the start to (position, head 0)."""
        positions = np.asarray(positions)
        return self.table[s, positions // self.page].astype(np.int64) * self.strides[0] + positions % self.page * self.strides[1]

    def part(self, name):
        a = {"q": 0, "k": self.heads, "v": self.heads + self.kv_heads}[name] * self.D
        n = (self.heads if name == "q" else self.kv_heads) * self.D
        return values(self.qkv)[:, a:a + n].reshape(self.rows, -1, self.D).astype(np.float64)

    def seen(self, name, s, positions):
        """[positions, kv_heads, D] of the pages, in 64 bits."""
        at = self.places(s, positions)[:, None, None] + (np.arange(self.kv_heads) * self.strides[2])[:, None] + np.arange(self.D)
        return values(getattr(self, name))[at].astype(np.float64)

    def upload(self, dev):
        self.at = {n: dev.put(getattr(self, n)) for n in ("k", "v", "qkv", "table", "starts")}
        self.at["lens"] = dev.put(np.asarray(self.lens, np.int32))
        return ffi.AhPages(self.dtype, self.kv_heads, self.D, self.page, len(self.lens), self.width, self.pages, *self.strides, self.at["k"], self.at["v"],
                           self.at["table"], self.at["starts"], self.at["lens"])

    def offsets(self):
        e = self.qkv.itemsize * self.D
        return self.at["qkv"], self.at["qkv"] + self.heads * e, self.at["qkv"] + (self.heads + self.kv_heads) * e


def rotary_table(rows, rot):
    angles = np.outer(np.arange(rows), 10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1)))
    return np.concatenate([np.cos(angles), np.sin(angles)], 1).astype(np.float32)


def turn64(x, table, position, rot, neighbours):
    """(turned x, sum of the terms' sizes) of [heads, D] at a position."""
    y, size = x.copy(), np.zeros_like(x)
    half = rot // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        c, s = (float(table[position, i]), float(table[position, half + i])) if 0 <= position < len(table) else (math.nan, math.nan)
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
        size[:, a], size[:, b] = abs(x[:, a] * c) + abs(x[:, b] * s), abs(x[:, b] * c) + abs(x[:, a] * s)
    return y, size


def run_append(B, dev, c, rot=0, neighbours=False, rot_rows=None, in_place=False):
    """What the call leaves of k, v and rotated."""
    pages = c.upload(dev)
    q, k, v = c.offsets()
    table = rotary_table(max(c.lens + [1]) if rot_rows is None else rot_rows, rot)
    out = c.store(np.full((c.rows, c.heads, c.D), 7.0))
    where, st, sh = (q, c.pitch, c.D) if in_place else (dev.put(out), c.heads * c.D, c.D)
    ffi.check(B.lib.ah_paged_append(pages, ffi.AhPagedAppend(c.rows, c.heads, rot, len(table) if rot else 0, int(neighbours), 0, c.pitch, c.D, c.pitch, c.D, c.pitch, c.D,
                                                              st, sh, q if rot else 0, k, v, where if rot else 0, dev.put(table) if rot else 0)))
    if in_place:
        out = dev.get(c.at["qkv"], c.qkv)[:, :c.heads * c.D].reshape(c.rows, c.heads, c.D)
    elif rot:
        out = dev.get(where, out)
    return dev.get(c.at["k"], c.k), dev.get(c.at["v"], c.v), out, table


def check_append(c, k, v, out, table, rot, neighbours, written=lambda s, p: True, in_place=False):
    want_k, want_v = c.k.copy(), c.v.copy()
    new_q, new_k, new_v = (c.part(n) for n in "qkv")
    h = H8 if c.dtype == ffi.BF16 else 0.0
    before = c.qkv[:, :c.heads * c.D].reshape(c.rows, c.heads, c.D) if in_place else c.store(np.full((c.rows, c.heads, c.D), 7.0))
    for r in range(c.rows):
        s = int(np.searchsorted(c.starts, r, side="right")) - 1
        if s >= len(c.lens):                     # behind the last sequence: left as they were
            assert np.array_equal(out[r], before[r])
            continue
        p = c.lens[s] - c.news[s] + r - int(c.starts[s])
        if rot:
            q64, size = turn64(new_q[r], table, p, rot, neighbours)
            got = values(out[r])
            assert np.array_equal(np.isnan(got), np.isnan(q64))
            assert np.all(np.where(np.isnan(q64), 0, abs(got - q64) - 2 * U * size * (1 + h) - h * abs(q64)) <= 1e-37), (r, s, p)
        if p < 0 or not written(s, p):
            continue
        k64, size = turn64(new_k[r], table, p, rot, neighbours)
        for g in range(c.kv_heads):
            at = int(c.places(s, p)) + g * c.strides[2]
            got = values(k[at:at + c.D])
            assert np.array_equal(np.isnan(got), np.isnan(k64[g]))
            assert np.all(np.where(np.isnan(k64[g]), 0, abs(got - k64[g]) - 2 * U * size[g] * (1 + h) - h * abs(k64[g]) * (rot > 0)) <= 1e-37), (r, s, p, g)
            assert np.array_equal(got[rot:], new_k[r, g, rot:])
            want_k[at:at + c.D] = k[at:at + c.D]
            want_v[at:at + c.D] = c.store(new_v[r, g])
    bits = lambda x: x.view(np.uint32 if x.itemsize == 4 else np.uint16)
    assert np.array_equal(bits(k), bits(want_k)) and np.array_equal(bits(v), bits(want_v))       # and nothing else


TYPES = [ffi.F32, ffi.BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,D,page,lens,news", [
    (2, 2, 64, 16, [1], [1]), (8, 8, 32, 16, [250], [1]), (3, 1, 8, 1, [5, 3, 9], [2, 0, 9]), (8, 2, 128, 33, [70, 1, 40, 33], [70, 1, 0, 5]),
    (6, 3, 48, 7, [3, 20, 7], [5, 20, 1]), (4, 4, 120, 65536, [100, 12], [3, 12]), (1, 1, 16, 64, [64] * 130, [1] * 130)])
@pytest.mark.parametrize("rot", ["none", "half", "neighbours", "odd"])
def test_new_keys_and_values_lie_where_their_positions_do(B, dev, dtype, heads, kv_heads, D, page, lens, news, rot):
    """`odd`: pairs whose halves are no whole 16 bytes; [3, .., ..] with 5 new tokens: two of them have no position and go nowhere."""
    if page == 65536:
        lens = [min(n, 100) for n in lens]
    c = Case(dtype, heads, kv_heads, D, page, lens, news, seed=D + page, heads_first=len(lens) % 2 == 0, gap=16)
    r, n = {"none": (0, False), "half": (D, False), "neighbours": (D - 4 if D > 8 else D, True), "odd": (D // 2 // 2 * 2 - 2 or 2, False)}[rot]
    check_append(c, *run_append(B, dev, c, r, n), r, n)


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_are_turned_in_place_too_and_positions_past_the_angles_give_nan(B, dev, dtype):
    for rot, neighbours in ((64, False), (64, True), (20, False)):
        c = Case(dtype, 4, 2, 64, 16, [30, 9], [30, 4], seed=3)
        got = run_append(B, dev, c, rot, neighbours, rot_rows=22, in_place=True)
        check_append(c, *got, rot, neighbours, in_place=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_without_a_place_are_not_written(B, dev, dtype):
    """Pages that the table names outside the array, positions past the table, starts that name rows outside."""
    c = Case(dtype, 2, 2, 64, 8, [40, 24, 16], [40, 24, 16], seed=5)
    c.table[0, 1], c.table[0, 3], c.table[1, 0] = -1, c.pages, 2 ** 31 - 1
    bad = {(0, 1), (0, 3), (1, 0)}
    check_append(c, *run_append(B, dev, c), 0, False, written=lambda s, p: (s, p // 8) not in bad)
    c = Case(dtype, 2, 2, 64, 8, [40, 24], [40, 24], seed=6)
    c.width = 3                                  # the table has 24 positions
    c.table = np.ascontiguousarray(c.table[:, :3])
    check_append(c, *run_append(B, dev, c), 0, False, written=lambda s, p: p < 24)
    c = Case(dtype, 2, 2, 64, 8, [6, 8], [6, 8], seed=7, spare=0)
    c.starts[2] = 2 ** 31 - 1                    # the second sequence: rows 6 .. 13, of as many as it says: the last positions of 8 are theirs all the same
    check_append(c, *run_append(B, dev, c), 0, False)


# ---------------------------------------------------------------------------------------------- attention
def run_attention(B, dev, c, scale, cap, pages=None, lse=True):
    pages = pages or c.upload(dev)
    out, sums = c.store(np.full((c.rows, c.heads, c.D), 7.0)), np.full((c.rows, c.heads), 7.0, np.float32)
    o, l = dev.put(out), dev.put(sums)
    ffi.check(B.lib.ah_paged_attention(pages, ffi.AhPagedAttention(c.rows, c.heads, scale, cap, c.pitch, c.D, c.heads * c.D, c.D, c.offsets()[0], o, l if lse else 0)))
    return dev.get(o, out), dev.get(l, sums)


def check_attention(c, out, lse, scale, cap, bad=(), past=()):
    """bad: (sequence, page entry) pairs that name no page; past: sequences longer than the table."""
    q = c.part("q")
    h = H8 if c.dtype == ffi.BF16 else 0.0
    for s in range(len(c.lens)):
        first, n, length = int(c.starts[s]), c.news[s], c.lens[s]
        reach = min(length, c.width * c.page)
        k, v = (c.seen(name, s, np.arange(reach)) for name in "kv")
        entries = np.arange(reach) // c.page
        lost = np.isin(entries, [e for t, e in bad if t == s])
        for r in range(first, first + n):
            p = length - n + r - first
            got_o, got_l = values(out[r]).astype(np.float64), lse[r].astype(np.float64)
            if p < 0:
                assert np.all(got_o == 0) and np.all(got_l == -np.inf), (s, p)
                continue
            if lost[:p + 1].any() or p >= reach:
                assert np.all(np.isnan(got_o)) and np.all(np.isnan(got_l)), (s, p)
                continue
            for head in range(c.heads):
                g = head // (c.heads // c.kv_heads)
                x, size = scale * (k[:p + 1, g] @ q[r, head]), abs(scale) * (abs(k[:p + 1, g]) @ abs(q[r, head]))
                if cap > 0:
                    x = cap * np.tanh(x / cap)
                e = float(((c.D + 3) * U * size + 4 * U * abs(x)).max()) + 8 * U * cap
                top = x.max()
                w = np.exp(x - top)
                total = w.sum()
                want, want_l = (w @ v[:p + 1, g]) / total, top + math.log(total)
                around = (w @ abs(v[:p + 1, g])) / total
                bound = (math.expm1(2 * e + 4 * U) + (p + 1 + 16) * U + 2 * h * (1 + h)) * around * (1 + h) + (h + 2 * U) * abs(want)
                assert np.all(abs(got_o[head] - want) <= bound), (s, p, head, float((abs(got_o[head] - want) / bound).max()))
                assert abs(got_l[head] - want_l) <= e + (p + 1 + 16) * U + 4 * U * abs(want_l) + 8 * U, (s, p, head)
    end = int(c.starts[-1])
    assert np.all(values(out[end:]) == 7.0) and np.all(lse[end:] == 7.0)


SHAPES = [  # heads, kv_heads, D, page, lens, news
    (1, 1, 8, 16, [1], [1]),
    (12, 12, 64, 16, [777], [1]),
    (8, 8, 48, 16, [17, 512, 1, 33], [1, 1, 1, 1]),
    (8, 2, 128, 33, [100, 31, 64, 1], [1, 5, 0, 1]),
    (4, 1, 32, 7, [40, 9, 130], [40, 9, 2]),
    (6, 2, 80, 64, [300, 65], [150, 65]),
    (3, 3, 64, 13, [2, 3, 200], [4, 3, 129]),
    (8, 1, 120, 100, [257], [33]),
    (16, 8, 16, 1, [20] * 70, [1] * 70),
    (2, 2, 128, 256, [1030, 700], [1, 1]),
    (4, 2, 64, 16, [600, 290], [300, 290]),
    (64, 1, 24, 32, [90, 31], [1, 3]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 30.0, 60.0, 0.5])
@pytest.mark.parametrize("shape", SHAPES)
def test_new_tokens_attend_to_their_sequences_positions(B, dev, dtype, cap, shape):
    heads, kv_heads, D, page, lens, news = shape
    c = Case(dtype, heads, kv_heads, D, page, lens, news, seed=heads + D, heads_first=page % 2 == 1, gap=8 if dtype == ffi.F32 else 16, scale=1.3)
    check_attention(c, *run_attention(B, dev, c, 1 / math.sqrt(D), cap), 1 / math.sqrt(D), cap)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,D,lens,news", [(4, 1, 64, [5000, 40, 2600], [1, 1, 1]), (2, 2, 128, [4100], [3]), (8, 4, 32, [3000, 100], [200, 50]),
                                                          (1, 1, 64, [2500], [140])])
def test_long_contexts(B, dev, dtype, heads, kv_heads, D, lens, news):
    """Few rows, many positions: the axis is cut and the parts are joined."""
    c = Case(dtype, heads, kv_heads, D, 16, lens, news, seed=1, entries=3)
    check_attention(c, *run_attention(B, dev, c, 0.2, 30.0), 0.2, 30.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [30, 2, 20, 70]])
def test_pages_that_do_not_exist_give_nan_to_those_who_read_them_and_to_nobody_else(B, dev, dtype, news):
    c = Case(dtype, 4, 2, 64, 8, [60, 30, 41, 70], news, seed=2, entries=2)
    c.table[0, 5], c.table[2, 0], c.table[3, 8] = c.pages, -1, -2 ** 31
    c.table[1, 4:], c.table[3, 9:] = -7, 2 ** 31 - 1                     # behind what the sequences have: nobody reads them
    bad = {(0, 5), (2, 0), (3, 8)}
    pages = c.upload(dev)
    c.table = np.where((c.table < 0) | (c.table >= c.pages), 0, c.table).astype(np.int32)
    check_attention(c, *run_attention(B, dev, c, 0.125, 0.0, pages=pages), 0.125, 0.0, bad=bad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 9])
def test_lengths_past_the_table_and_below_the_number_of_new_tokens(B, dev, dtype, new):
    c = Case(dtype, 2, 1, 32, 16, [40, 64, 0, 3], [new, new, new, new], seed=4)
    c.width = 3
    c.table = np.ascontiguousarray(c.table[:, :3])                       # 48 positions: the second sequence's 64 are not all there
    check_attention(c, *run_attention(B, dev, c, 0.3, 0.0), 0.3, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,D,news", [(2, 64, [1, 1]), (2, 64, [40, 64]), (8, 128, [3, 5]), (4, 32, [100, 130])])
def test_what_lies_behind_a_position_weighs_nothing_whatever_it_is(B, dev, dtype, heads, D, news):
    """Infinities and NaN in rows of a page behind a sequence's end, and in keys and values of later new tokens."""
    lens = [max(n, 70) for n in news]
    c = Case(dtype, heads, 2, D, 16, lens, news, seed=8, entries=1)
    kinds = [np.inf, -np.inf, np.nan]
    poison = [np.uint16(b) for b in (0x7f80, 0xff80, 0x7fc0)] if dtype == ffi.BF16 else [np.float32(x) for x in kinds]
    clean_k, clean_v = c.k.copy(), c.v.copy()
    used = np.zeros(c.k.size, bool)
    for s, n in enumerate(lens):
        at = c.places(s, np.arange(n))[:, None, None] + (np.arange(2) * c.strides[2])[:, None] + np.arange(D)
        used[at.reshape(-1)] = True
    for i, (x, y) in enumerate(((c.k, clean_k), (c.v, clean_v))):
        free = np.nonzero(~used)[0]
        x[free] = np.array([poison[(j + i) % 3] for j in range(free.size)], x.dtype)
    # the last new token of each sequence with more than one: keys and values that only it sees
    spoilt = []
    for s, n in enumerate(lens):
        if news[s] > 1:
            at = int(c.places(s, n - 1))
            c.k[at:at + D], c.v[at + 1:at + D:3] = poison[2], poison[s % 3]
            spoilt.append(int(c.starts[s + 1]) - 1)
    out, lse = run_attention(B, dev, c, 0.125, 0.0)
    for r in spoilt:                              # head 0 of that token reads it itself
        group = heads // 2
        assert np.all(np.isnan(values(out[r, :group]))) and np.all(np.isnan(lse[r, :group]))
    c.k, c.v = clean_k, clean_v
    again, sums = run_attention(B, dev, c, 0.125, 0.0)
    check_attention(c, again, sums, 0.125, 0.0)
    rest = [r for r in range(c.rows) if r not in spoilt]
    ref, refs = values(again[rest]).astype(np.float64), sums[rest].astype(np.float64)
    # the same weights and values, perhaps summed in another way around the poisoned places: within the rounding of both
    h = H8 if dtype == ffi.BF16 else 0.0
    assert np.allclose(values(out[rest]), ref, rtol=2 * h + 200 * U, atol=(2 * h + 200 * U) * 4) and np.allclose(lse[rest], refs, rtol=200 * U, atol=200 * U)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_page_may_be_shared_and_rows_do_not_depend_on_the_batch(B, dev, dtype):
    """Two sequences with the same first page; and the output is the same with and without the lse."""
    c = Case(dtype, 4, 2, 64, 32, [50, 45, 64], [3, 1, 2], seed=9, share=(0, 1))
    first = run_attention(B, dev, c, 0.125, 30.0)
    check_attention(c, *first, 0.125, 30.0)
    assert np.array_equal(first[0], run_attention(B, dev, c, 0.125, 30.0, lse=False)[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_past_32_bits(B, dev, dtype):
    """Pages 2^31 elements and more into the arrays (strides as wide as that: a page of one array lies between those of others)."""
    size = 4 if dtype == ffi.F32 else 2
    c = Case(dtype, 2, 1, 64, 16, [40], [2], seed=10, spare=0)
    far = (1 << 31) // 4 + 64                     # elements between pages
    block = C.c_uint64()
    ffi.check(B.lib.ah_alloc(2 * (c.pages * far) * size, C.byref(block)))
    try:
        pages = c.upload(dev)
        for i, x in enumerate((c.k, c.v)):
            for p in range(c.pages):
                ffi.check(B.lib.ah_copy(block.value + (i * c.pages + p) * far * size, (c.at["k"], c.at["v"])[i] + p * c.strides[0] * size, 16 * 64 * size))
        assert (c.pages - 1) * far > 1 << 31
        pages.k, pages.v, pages.page_stride = block.value, block.value + c.pages * far * size, far
        check_attention(c, *run_attention(B, dev, c, 0.125, 0.0, pages=pages), 0.125, 0.0)
        q, k, v = c.offsets()
        ffi.check(B.lib.ah_paged_append(pages, ffi.AhPagedAppend(c.rows, 0, 0, 0, 0, 0, 0, 0, c.pitch, c.D, c.pitch, c.D, 0, 0, 0, k, v, 0, 0)))
        got = dev.get(block.value + (int(c.table[0, 2]) * far + (39 % 16) * 64) * size, c.qkv[1, :64])
        assert np.array_equal(got, c.qkv[1, 128:192])
    finally:
        ffi.check(B.lib.ah_sync())
        ffi.check(B.lib.ah_free(block.value))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_captured_call_follows_tables_starts_and_lengths(B, dev, dtype):
    c = Case(dtype, 4, 2, 64, 16, [900, 50, 333], [1, 1, 1], seed=11, entries=60, spare=0)
    pages = c.upload(dev)
    out, lse = dev.put(np.zeros_like(c.qkv[:, :256])), dev.put(np.zeros((3, 4), np.float32))
    q, k, v = c.offsets()
    d = ffi.AhPagedAttention(3, 4, 0.125, 30.0, c.pitch, 64, 256, 64, q, out, lse)
    a = ffi.AhPagedAppend(3, 0, 0, 0, 0, 0, 0, 0, c.pitch, 64, c.pitch, 64, 0, 0, 0, k, v, 0, 0)

    def both():
        ffi.check(B.lib.ah_paged_append(pages, a))
        ffi.check(B.lib.ah_paged_attention(pages, d))
    both()
    graphs = []
    for _ in range(2):
        g = C.c_uint64()
        ffi.check(B.lib.ah_graph_begin())
        both()
        ffi.check(B.lib.ah_graph_end(C.byref(g)))
        graphs.append(g.value)
    try:
        for step in range(4):
            lens = np.asarray([900 + 3 * step, 50 * (step + 1), 333 - 100 * step], np.int32)
            ffi.check(B.lib.ah_upload(c.at["lens"], lens.ctypes.data_as(C.c_void_p), lens.nbytes))
            both()
            want = dev.get(out, c.qkv[:, :256]), dev.get(lse, np.zeros((3, 4), np.float32)), dev.get(c.at["k"], c.k)
            ffi.check(B.lib.ah_fill_f32(lse, 5.0, 12))
            ffi.check(B.lib.ah_graph_launch(graphs[step % 2]))
            ffi.check(B.lib.ah_graph_launch(graphs[(step + 1) % 2]))
            got = dev.get(out, c.qkv[:, :256]), dev.get(lse, np.zeros((3, 4), np.float32)), dev.get(c.at["k"], c.k)
            assert all(np.array_equal(x, y) for x, y in zip(got, want)), step
    finally:
        ffi.check(B.lib.ah_sync())
        for g in graphs:
            ffi.check(B.lib.ah_graph_destroy(g))


def test_nothing_to_do(B, dev):
    c = Case(ffi.F32, 2, 2, 64, 16, [5], [0], spare=3)
    pages = c.upload(dev)
    out, lse = run_attention(B, dev, c, 0.1, 0.0, pages=pages)
    assert np.all(out == 7.0) and np.all(lse == 7.0)
    pages.seqs = 0
    out, lse = run_attention(B, dev, c, 0.1, 0.0, pages=pages)
    assert np.all(out == 7.0) and np.all(lse == 7.0)
