"""What generation from several prompts refuses, and what runs where nothing is kept in pages, without a GPU."""
import numpy as np
import pytest

from alpha2_amd import FastHipBackend, HipBackend, Pages, TensorData
from alpha2_amd import sample
from alpha2_amd.decode import PagedContext
from alpha2_amd.model import ModelConfig
from alpha2_amd.sample import SampleConfig, sampleTokensBatch


def T(*shape, dtype="f32", store=None):
    t = TensorData(shape, dtype, np.zeros(shape))
    t.store = store or dtype
    return t


def I(*shape):
    return T(*shape, dtype="i32")


def pages(store="f32", **other):
    parts = dict(k=T(4, 16, 2, 8, store=store), v=T(4, 16, 2, 8, store=store), table=I(3, 5), starts=I(4), lens=I(3))
    return Pages(**{**parts, **other})


@pytest.fixture(params=[HipBackend, FastHipBackend])
def backend(request):
    return request.param.__new__(request.param)         # what is refused here is so before the library is called


@pytest.mark.parametrize("other", [dict(k=T(4, 16, 16)), dict(v=T(4, 16, 2, 16)), dict(v=T(4, 16, 2, 8, store="bf16")), dict(table=I(15)),
                                   dict(table=I(2, 5)), dict(starts=I(3)), dict(lens=I(4))])
def test_pages_that_do_not_fit(other):
    with pytest.raises(ValueError):
        pages(**other)


@pytest.mark.parametrize("name", ["table", "starts", "lens"])
def test_indices_of_another_type(name):
    with pytest.raises(TypeError):
        pages(**{name: T(*getattr(pages(), name).shape)})


@pytest.mark.parametrize("shape,heads,rotary", [((5, 64), 3, None), ((5, 48), 0, None), ((80,), 6, None), ((5, 80), 6, (32,)), ((5, 32), -2, None)])
def test_projections_that_do_not_fit(backend, shape, heads, rotary):
    with pytest.raises(ValueError):
        backend.pagedAppend(pages(), T(*shape), heads, rotary and T(*rotary))


@pytest.mark.parametrize("shape,heads", [((5, 40), 6), ((5, 48), 0), ((48,), 6)])
def test_queries_that_do_not_fit(backend, shape, heads):
    with pytest.raises(ValueError):
        backend.pagedAttention(pages(), T(*shape), heads, 1.0)


def test_tensors_of_another_type(backend):
    with pytest.raises(TypeError):
        backend.pagedAppend(pages(), I(5, 80), 6)
    with pytest.raises(TypeError):
        backend.pagedAttention(pages(), I(5, 48), 6, 1.0)
    with pytest.raises(TypeError):
        backend.sampleRows(I(5, 48), T(5))
    if type(backend) is HipBackend:                      # (the fast one makes a copy of the pages' type)
        with pytest.raises(TypeError):
            backend.pagedAppend(pages("bf16"), T(5, 80), 6)
        with pytest.raises(TypeError):
            backend.pagedAttention(pages(), T(5, 48, store="bf16"), 6, 1.0)


@pytest.mark.parametrize("which", ["k", "v"])
def test_pages_whose_storage_has_changed_since(backend, which):
    """FastHipBackend's ops that take f32 alone give a bf16 tensor f32 storage in place: keys of one type are not read beside values of another."""
    def nothing(*a):
        raise AssertionError("the library has been called")
    backend.lib = type("Lib", (), {"__getattr__": lambda self, name: nothing})()
    backend._launch_flash = backend._ptr = lambda *a: 0
    kept = pages("bf16")
    getattr(kept, which).store = "f32"
    new = lambda n: T(5, n, store=kept.k.store)
    backend._new = lambda shape, dtype="f32", store=None: T(*shape, store=store)
    with pytest.raises(TypeError, match="one type"):
        backend._pages_desc(kept)
    with pytest.raises(TypeError, match="one type"):
        backend.pagedAppend(kept, new(80), 6)


@pytest.mark.parametrize("name,t,error", [("uniform", T(4), ValueError), ("uniform", I(5), TypeError), ("temperature", T(5, 1), ValueError),
                                          ("temperature", T(5, store="bf16"), TypeError), ("topk", T(5), TypeError), ("topk", I(6), ValueError),
                                          ("topp", I(5), TypeError), ("minp", T(1), ValueError)])
def test_options_that_do_not_fit(backend, name, t, error):
    with pytest.raises(error):
        backend.sampleRows(T(5, 48), **{"uniform": T(5), name: t})
    with pytest.raises(ValueError):
        backend.sampleRows(T(48), T(48))


CFG = dict(vocabSize=20, blockSize=12, nLayer=1, nEmbd=16, nHead=2)


@pytest.mark.parametrize("prompts,rngs,configs", [([[]], 1, SampleConfig()), ([[1] * 13], 1, SampleConfig()), ([[1, 20]], 1, SampleConfig()), ([[-1]], 1, SampleConfig()),
                                                  ([[1], [2]], 1, SampleConfig()), ([[1], [2]], 2, [SampleConfig()])])
def test_prompts_that_are_refused(prompts, rngs, configs):
    with pytest.raises(ValueError):
        sampleTokensBatch(ModelConfig(**CFG), {}, None, [None] * rngs, prompts, configs)


@pytest.mark.parametrize("more", [dict(attention="unfused"), dict(attention="reference-flash"), dict(dropout=0.1), dict(nEmbd=24, nHead=2), dict(nEmbd=15), dict(nEmbd=512, nHead=2)])
def test_models_whose_sequences_are_run_one_by_one(monkeypatch, more):
    cfg, calls = ModelConfig(**{**CFG, **more}), []
    assert PagedContext.of(cfg, {}, HipBackend.__new__(HipBackend), [3]) is None
    assert PagedContext.of(ModelConfig(**CFG), {}, object(), [3]) is None
    monkeypatch.setattr(sample, "sampleTokens", lambda *a: calls.append(a) or np.array(a[4]))
    configs = [SampleConfig(steps=3), SampleConfig(steps=4)]
    got = sampleTokensBatch(cfg, "params", object(), ["a", "b"], [[1], [2, 3]], configs, "release", "flush")
    assert [g.tolist() for g in got] == [[1], [2, 3]]
    assert [(a[3], a[5], a[6], a[7]) for a in calls] == [("a", configs[0], "release", "flush"), ("b", configs[1], "release", "flush")]


def test_parameters_of_another_model_are_run_one_by_one():
    cfg, backend = ModelConfig(**CFG), HipBackend.__new__(HipBackend)
    wpe = lambda rows: type("V", (), {"data": T(rows, 16)})()
    assert PagedContext.of(cfg, {"layers": [], "wpe": wpe(12)}, backend, [3]) is None
    assert PagedContext.of(cfg, {"layers": [{}], "wpe": wpe(2)}, backend, [3]) is None


def test_more_tokens_than_a_sequence_was_given_room_for():
    kept = PagedContext(ModelConfig(**CFG), {}, None, [3, 12])
    kept.lens[:] = 2, 12
    for seqs, counts in (([0], [2]), ([1], [1]), ([0, 0], [1, 1]), ([0], [0])):
        with pytest.raises(ValueError):
            kept.forward(seqs, counts, np.zeros(sum(counts), np.int32), [], None)


def test_every_sequence_has_pages_of_its_own():
    kept = PagedContext(ModelConfig(**{**CFG, "blockSize": 300}), {}, None, [1, 64, 65, 300, 128])
    need = [1, 1, 2, 5, 2]
    owned = [set(kept.table[i, :n].tolist()) for i, n in enumerate(need)]
    assert sorted(p for s in owned for p in s) == list(range(sum(need)))
    for i, s in enumerate(owned):
        assert set(kept.table[i].tolist()) == s


class OneTokenEach:
    """In PagedContext's place: logits of nothing; `asked` holds the options that sampleRows was given with each row."""
    MOST_ROWS = 8192

    def __init__(self):
        self.asked = []

    def forward(self, seqs, counts, tokens, wanted, release):
        return T(len(wanted), 20)

    def close(self):
        pass

    def sampleRows(self, logits, uniform, temperature, topk, topp):
        self.asked.append([t.data.copy() for t in (uniform, temperature, topk, topp)])
        return {"tokens": I(logits.shape[0])}


class Draw:
    def __init__(self, *draws):
        self.draws = list(draws)

    def next(self):
        return self.draws.pop(0)


@pytest.mark.parametrize("config,temperature,topk,topp", [
    # selectToken: 0 < topP < 1 cuts and walks from the largest down, whatever of it f32 can hold; 0, 1, NaN and what lies outside do not
    (dict(topp=1 - 1e-12), lambda t: t == np.float32(0.8), lambda k: k == 20 or k == 0, lambda p: 1 - 1e-7 < p < 1),
    (dict(topp=1e-60), None, None, lambda p: 0 < p < 1e-30),
    (dict(topp=0.9), None, None, lambda p: p == np.float32(0.9)),
    (dict(topp=0.0), None, None, lambda p: not 0 < p < 1),
    (dict(topp=1.0), None, None, lambda p: not 0 < p < 1),
    (dict(topp=float("nan")), None, None, lambda p: not 0 < p < 1),
    (dict(topp=None), None, None, lambda p: not 0 < p < 1),
    # 0 < topk < vocabulary keeps so many; others keep all, those that 32 bits do not hold among them
    (dict(topk=2 ** 32 + 5), None, lambda k: not 0 < k < 20, None),
    (dict(topk=2 ** 70), None, lambda k: not 0 < k < 20, None),
    (dict(topk=-2 ** 70), None, lambda k: not 0 < k < 20, None),
    (dict(topk=20), None, lambda k: not 0 < k < 20, None),
    (dict(topk=19), None, lambda k: k == 19, None),
    # a temperature above 0 samples, 0 and below take the largest, NaN counts as 1
    (dict(temperature=1e-60), lambda t: 0 < t < 1e-30, None, None),
    (dict(temperature=1e60), lambda t: 1e30 < t, None, None),
    (dict(temperature=float("inf")), lambda t: 1e30 < t, None, None),
    (dict(temperature=float("nan")), lambda t: t == 1, None, None),
    (dict(temperature=0.0), lambda t: t == 0, None, None),
    (dict(temperature=-1e-60), lambda t: t <= 0, None, None),
])
def test_options_keep_their_side_of_what_switches_them_off(monkeypatch, config, temperature, topk, topp):
    """SampleConfig's numbers have 64 bits, the kernel's 32: none of them may be rounded to one that means something else."""
    kept = OneTokenEach()
    monkeypatch.setattr(sample.PagedContext, "of", staticmethod(lambda *a: kept))
    with np.errstate(over="raise", invalid="raise"):
        sampleTokensBatch(ModelConfig(**CFG), {}, kept, [Draw(0.25)], [[1]], SampleConfig(**{"steps": 1, **config}))
    (_, t, k, p), = kept.asked
    assert t.dtype == p.dtype == np.float32 and k.dtype == np.int32
    for got, right in ((t, temperature), (k, topk), (p, topp)):
        assert right is None or right(got[0]), got[0]


def test_draws_stay_below_one(monkeypatch):
    kept = OneTokenEach()
    monkeypatch.setattr(sample.PagedContext, "of", staticmethod(lambda *a: kept))
    sampleTokensBatch(ModelConfig(**CFG), {}, kept, [Draw(1 - 2.0 ** -53), Draw(0.0)], [[1], [2]], SampleConfig(steps=1))
    assert kept.asked[0][0].tolist() == [1 - 2.0 ** -24, 0.0]


def test_fewer_than_no_steps(monkeypatch):
    """Refused by sampleTokens: here too, whether the sequences are run together or one by one."""
    with pytest.raises(ValueError):
        sample.sampleTokens(ModelConfig(**CFG), {}, None, None, [1, 2], SampleConfig(steps=-1))
    for of in (lambda *a: OneTokenEach(), lambda *a: None):
        monkeypatch.setattr(sample.PagedContext, "of", staticmethod(of))
        monkeypatch.setattr(sample, "sampleTokens", lambda *a: np.array(a[4]))
        for steps in ([-1, 3], [0, -5]):
            with pytest.raises(ValueError, match="steps"):
                sampleTokensBatch(ModelConfig(**CFG), {}, OneTokenEach(), [Draw(), Draw(0.1, 0.2, 0.3)], [[1, 2], [3]], [SampleConfig(steps=n) for n in steps])


@pytest.mark.parametrize("longest", [[], [0], [0, 0]])
def test_no_sequences_or_none_with_a_token(longest):
    params = {"layers": [{}], "wpe": type("V", (), {"data": T(12, 16)})()}
    assert PagedContext.of(ModelConfig(**CFG), params, HipBackend.__new__(HipBackend), longest) is None
