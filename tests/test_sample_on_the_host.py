"""The sampling kernel's own source on the CPU, a fiber to a thread (wave_host.h), with the undefined-behaviour checks of the compiler: it ends, and chooses as the
definition in 64 bits does, on the rows that its loops are most likely to go wrong on."""
import os
import struct
import subprocess

import numpy as np
import pytest

import test_gpu_sample as gpu
from alpha2_amd import _ffi as ffi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MAIN = r"""
#include <vector>
int main() {   // rows, vocab, row stride, bytes of a logit; logits, temperature, top_k, top_p, min_p, uniform in; tokens and logprobs out
  int h[4];
  if (fread(h, 4, 4, stdin) != 4) return 2;
  const int rows = h[0], V = h[1], ld = h[2];
  std::vector<char> x((size_t)rows * ld * h[3] + 32);
  std::vector<float> t(rows), p(rows), m(rows), u(rows), lp(rows);
  std::vector<int> k(rows), tok(rows);
  auto get = [](void *q, size_t n) { if (fread(q, 1, n, stdin) != n) exit(2); };
  char *base = (char *)(((uintptr_t)x.data() + 15) / 16 * 16);
  get(base, (size_t)rows * ld * h[3]); get(t.data(), 4 * rows); get(k.data(), 4 * rows); get(p.data(), 4 * rows); get(m.data(), 4 * rows); get(u.data(), 4 * rows);
  SampleArgs a{base, t.data(), p.data(), m.data(), u.data(), k.data(), tok.data(), lp.data(), ld, V};
  for (int r = 0; r < rows; r++) {
    blockIdx.x = r;
    const bool ended = V > LONG ? host::run(1024, [&] { if (h[3] == 2) k_sample<uint16_t, 1024>(a); else k_sample<float, 1024>(a); })
                                : host::run(512, [&] { if (h[3] == 2) k_sample<uint16_t, 512>(a); else k_sample<float, 512>(a); });
    if (!ended) { fprintf(stderr, "row %d: nobody can go on\n", r); return 3; }
  }
  fwrite(tok.data(), 4, rows, stdout); fwrite(lp.data(), 4, rows, stdout);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    src = open(os.path.join(ROOT, "alpha2_amd", "csrc", "sample.hip")).read()
    src = src[:src.index('extern "C"')].replace('#include "common.h"', '#include "wave_host.h"')
    d = tmp_path_factory.mktemp("sample")
    (d / "sample.cpp").write_text(src + MAIN)
    subprocess.run(["g++", "-std=c++20", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-Wno-unknown-pragmas", "-I", os.path.join(ROOT, "tests"),
                    str(d / "sample.cpp"), "-o", str(d / "sample")], check=True)
    return str(d / "sample")


@pytest.fixture()
def on_the_host(program, monkeypatch):
    def run(B, dev, dtype, logits, t=None, k=None, p=None, m=None, u=None, ld=None, at=0, logprobs=True):
        rows, V = logits.shape
        wide = np.zeros((rows, ld or V), logits.dtype)
        wide[:, :V] = logits
        every = lambda x, off, kind: np.broadcast_to(np.asarray(off if x is None else x), (rows,)).astype(kind).tobytes()
        data = struct.pack("4i", rows, V, ld or V, logits.itemsize) + wide.tobytes() + every(t, 1.0, np.float32) + every(k, 0, np.int32) \
            + every(p, 1.0, np.float32) + every(m, 0.0, np.float32) + every(u, 0.0, np.float32)
        r = subprocess.run([program], input=data, capture_output=True, timeout=300)
        assert r.returncode == 0, r.stderr.decode()
        return np.frombuffer(r.stdout[:4 * rows], np.int32), np.frombuffer(r.stdout[4 * rows:], np.float32)
    monkeypatch.setattr(gpu, "run", run)


@pytest.mark.parametrize("dtype", gpu.TYPES)
@pytest.mark.parametrize("V", [40, 2500])
def test_equal_logits(on_the_host, dtype, V):
    gpu.test_equal_logits(None, None, dtype, V)


@pytest.mark.parametrize("dtype", gpu.TYPES)
def test_logits_that_lie_closer_or_wider_than_bins_can_tell(on_the_host, dtype):
    gpu.test_logits_that_lie_closer_or_wider_than_bins_can_tell(None, None, dtype)


def test_infinite_and_missing_logits(on_the_host):
    gpu.test_infinite_and_missing_logits(None, None, 50)
    gpu.test_infinite_and_missing_logits(None, None, 5000)


def test_settings_and_random_numbers_at_their_ends(on_the_host):
    gpu.test_settings_that_switch_off(None, None)
    gpu.test_the_ends_of_the_random_numbers(None, None)


@pytest.mark.parametrize("dtype", gpu.TYPES)
@pytest.mark.parametrize("V,rows", [(300, 40), (5000, 24)])
def test_every_row_has_its_own_choice(on_the_host, dtype, V, rows):
    gpu.test_every_row_has_its_own_choice(None, None, dtype, V, rows)


@pytest.mark.parametrize("name", list(gpu.SETTINGS))
def test_a_long_row(on_the_host, name):
    gpu.test_tokens_are_those_of_the_definition(None, None, ffi.F32, 53249, name)
