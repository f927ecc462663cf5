"""Host contents given to a tensor: as many as its shape says, and in bf16 where it is stored so (a page of keys filled by hand, a cached activation put back)."""
import ctypes as C

import numpy as np
import pytest

from alpha2_amd import FastHipBackend, HipBackend, TensorData


class Lib:
    """Blocks of host memory, with a guard behind each."""

    def __init__(self):
        self.blocks, self.uploads = {}, []

    def ah_alloc(self, nbytes, out):
        block = np.full(nbytes + 64, 0xA5, np.uint8)
        self.blocks[block.ctypes.data] = (block, nbytes)
        C.cast(out, C.POINTER(C.c_uint64))[0] = block.ctypes.data
        return 0

    def ah_free(self, ptr):
        return 0

    def ah_upload(self, dst, src, nbytes):
        self.uploads.append(nbytes)
        block, room = self.blocks[dst]
        assert nbytes <= room, "past the block's end"
        C.memmove(dst, src, nbytes)
        return 0

    def ah_download(self, dst, src, nbytes):
        C.memmove(dst, src, nbytes)
        return 0


@pytest.fixture(params=[HipBackend, FastHipBackend])
def backend(request):
    b = request.param.__new__(request.param)
    b.lib = Lib()
    b._adam_q = b._wgrads = []
    b._scatters = b._lazy = b._orphans = b._ln_unwritten = {}
    b._held = b._held_ln = b._held_ce = b._pending_flash = None
    b._launch_weight_grads = lambda: None
    return b


# f32 and the bf16 next to it, ties to the even one: exact, below and above half a step, ties both ways, past the largest, the smallest f32
VALUES = [(0.0, 0x0000), (-0.0, 0x8000), (1.0, 0x3F80), (-2.5, 0xC020), (1.0 + 2.0 ** -8, 0x3F80), (1.0 + 3 * 2.0 ** -8, 0x3F82), (1.0 + 2.0 ** -8 + 2.0 ** -20, 0x3F81),
          (1.0 + 2.0 ** -9, 0x3F80), (3.4028235e38, 0x7F80), (np.inf, 0x7F80), (-np.inf, 0xFF80), (2.0 ** -149, 0x0000), (2.0 ** -126, 0x0080)]


@pytest.mark.parametrize("released", [False, True])
def test_host_contents_are_rounded_to_what_is_stored(backend, released):
    want = np.array([b for _, b in VALUES], np.uint16)
    t = backend._new((len(VALUES),), "f32", "bf16")
    if released:
        backend.releaseGpuTensor(t)
    t.data = np.array([v for v, _ in VALUES], np.float32)
    ptr = backend._ptr(t)
    block, room = backend.lib.blocks[ptr]
    assert t.store == "bf16" and room == 2 * len(VALUES) and backend.lib.uploads == [room]
    assert np.array_equal(block[:room].view(np.uint16), want) and (block[room:] == 0xA5).all()
    assert np.array_equal(t.data.view(np.uint32), want.astype(np.uint32) << 16)          # and that is what is read back
    assert backend._ptr(t) == ptr and len(backend.lib.uploads) == 1


def test_nan_stays_nan(backend):
    t = backend._new((4,), "f32", "bf16")
    t.data = np.array([0x7F800001, 0xFF800001, 0x7FFFFFFF, 0xFFFFFFFF], np.uint32).view(np.float32)
    backend._ptr(t)
    assert np.isnan(t.data).all()


@pytest.mark.parametrize("dtype", ["f32", "i32"])
def test_other_storage_is_uploaded_as_it_is(backend, dtype):
    t = TensorData((3,), dtype, np.array([1, -2, 3]))
    ptr = backend._ptr(t)
    block, room = backend.lib.blocks[ptr]
    assert room == 12 and block[:12].view(t.data.dtype).tolist() == [1, -2, 3] and t._host_valid


@pytest.mark.parametrize("dtype,store", [("i32", "i32"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("n", [0, 5, 7, 13])
def test_host_contents_of_another_size_are_refused(backend, dtype, store, n):
    """A kernel goes by the shape: a table, a list of tokens or a page with fewer numbers than that would be read past its end, with more written past its block's."""
    t = TensorData((2, 3), dtype, np.zeros(n))
    t.store = store
    with pytest.raises(ValueError, match=r"\(2, 3\)"):
        backend._ptr(t)
    t = backend._new((2, 3), dtype, store)
    t.data = np.zeros(n)
    with pytest.raises(ValueError, match=r"\(2, 3\)"):
        backend._ptr(t)
    assert backend.lib.uploads == []
    t.data = np.arange(6)
    backend._ptr(t)
    assert t.data.tolist() == [0, 1, 2, 3, 4, 5]


def test_tokens_of_another_number_than_asked_for(backend):
    from alpha2_amd.decode import PagedContext
    from alpha2_amd.model import ModelConfig
    kept = PagedContext(ModelConfig(vocabSize=20, blockSize=12, nLayer=0, nEmbd=16, nHead=2), {"wte": type("V", (), {"data": TensorData((20, 16), "f32", np.zeros(320)), "requiresGrad": False})()}, backend, [12])
    backend.lib.ah_embedding = lambda *a: pytest.fail("the kernel has been called")
    for tokens in (np.zeros(2, np.int32), np.zeros(4, np.int32), TensorData((2,), "i32", np.zeros(2))):
        with pytest.raises(ValueError):
            kept.forward([0], [3], tokens, [0], None)
    assert kept.lens.tolist() == [0]
