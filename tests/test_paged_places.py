"""What needs no GPU of the operators on pages and of sampling: where positions lie (csrc/paged.h, compiled for the host), and the calls that are
refused, which they are before a device is asked for."""
import ctypes as C
import os
import subprocess

import pytest

from alpha2_amd import _ffi as ffi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "paged.h"
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
using namespace ah;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
  // quotients: all divisors, the numerators next to multiples and to the ends
  for (uint32_t d = 1; d <= 65536; d++) {
    const Quotient q = quotient_by(d);
    CHECK(q.shift <= 47 && (q.shift == 31 || (1u << (q.shift - 31)) >= d));
    const uint32_t most = 0x7fffffffu / d;
    for (uint32_t k : {0u, 1u, 2u, most / 3, most / 2, most - 1, most})
      for (int e = -1; e <= 1; e++) {
        const int64_t n = (int64_t)k * d + e;
        if (n >= 0 && n <= 0x7fffffff) CHECK(quotient((uint32_t)n, q) == (uint32_t)n / d);
      }
    CHECK(quotient(0x7fffffffu, q) == 0x7fffffffu / d);
  }
  for (uint32_t d : {65537u, 98304u, 131071u, 1000003u, 1u << 26, 134217727u, 0x7fffffffu}) {
    const Quotient q = quotient_by(d);
    for (uint32_t n : {0u, d - 1, d, d + 1 < 0x7fffffffu ? d + 1 : d, 0x7fffffffu / d * d, 0x7fffffffu / d * d - 1, 0x7fffffffu}) CHECK(quotient(n, q) == n / d);
  }
  // places: pages of 5 rows, two sequences of 3 entries; a page outside the array and a position past the table have none
  const int32_t table[6] = {2, 0, 7, -1, 1, 2147483647};
  PagedCache c{};
  c.table = table; c.pages = 4; c.page_stride = int64_t(1) << 33; c.row_stride = 96; c.page_rows = quotient_by(5); c.seqs = 2; c.table_pages = 3; c.capacity = 15;
  for (int s = 0; s < 2; s++)
    for (int p = -2; p < 20; p++) {
      const int32_t page = p >= 0 && p < 15 ? table[3 * s + p / 5] : -1;
      CHECK(position_place(c, s, p) == (page >= 0 && page < 4 ? page * (int64_t(1) << 33) + (p % 5) * 96 : -1));
    }
  // sequences: starts that go back, or past the rows, name nothing outside them
  const int32_t values[] = {-2147483647 - 1, -1, 0, 1, 4, 5, 6, 2147483647};
  for (int32_t start : values) for (int32_t next : values) for (int32_t len : values) {
    const Sequence s = sequence_of(start, next, len, 5);
    CHECK(s.first >= 0 && s.count >= 0 && s.first + s.count <= 5 && s.len >= 0);
    if (start >= 0 && start <= next && next <= 5) CHECK(s.first == start && s.count == next - start);
    if (len >= 0) CHECK(s.len == len);
  }
  puts("ok");
  return 0;
}
"""


def test_positions_lie_where_the_table_says(tmp_path):
    src, exe = tmp_path / "places.cpp", tmp_path / "places"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "alpha2_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


P = 1 << 20                  # an address: these calls never get to a device


def pages(**more):
    d = dict(dtype=ffi.BF16, kv_heads=2, head_dim=64, page_rows=16, seqs=3, table_pages=4, pages=10, page_stride=2048, row_stride=128, head_stride=64,
             k=P, v=P, table=P, starts=P, lens=P)
    d.update(more)
    return ffi.AhPages(**d)


def append(**more):
    d = dict(rows=5, heads=4, rot_dim=64, rot_rows=100, q_st=512, q_sh=64, k_st=512, k_sh=64, v_st=512, v_sh=64, r_st=256, r_sh=64,
             q=P, k=P, v=P, rotated=P, rotary=P)
    d.update(more)
    return ffi.AhPagedAppend(**d)


def attention(**more):
    d = dict(rows=5, heads=4, scale=0.125, soft_cap=0.0, q_st=512, q_sh=64, o_st=256, o_sh=64, q=P, o=P, lse=P)
    d.update(more)
    return ffi.AhPagedAttention(**d)


def sample(**more):
    d = dict(dtype=ffi.F32, vocab=100, rows=3, ld=100, logits=P, temperature=P, top_k=P, top_p=P, min_p=P, uniform=P, tokens=P, logprobs=P)
    d.update(more)
    return ffi.AhSample(**d)


def _refused(rc, word):
    assert rc == 2 and word in ffi.load().ah_last_error().decode(), (rc, ffi.load().ah_last_error())


BAD_PAGES = [(dict(dtype=ffi.F16), "dtype"), (dict(dtype=9), "dtype"), (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=1 << 20), "kv_heads"),
             (dict(head_dim=0), "head_dim"), (dict(head_dim=60), "head_dim"), (dict(head_dim=136), "head_dim"), (dict(page_rows=0), "page_rows"),
             (dict(page_rows=65537), "page_rows"), (dict(seqs=-1), "sequences"), (dict(seqs=1 << 21), "sequences"), (dict(table_pages=-1), "pages"),
             (dict(pages=-1), "pages"), (dict(pages=1 << 31), "pages"), (dict(page_stride=2044), "strides"), (dict(row_stride=132), "strides"),
             (dict(head_stride=1), "strides"), (dict(head_stride=-64), "strides"), (dict(page_stride=1 << 35), "strides"), (dict(k=P + 8), "aligned"), (dict(v=P + 2), "aligned"),
             (dict(table=P + 2), "aligned"), (dict(lens=P + 1), "aligned"), (dict(starts=0), "null"), (dict(lens=0), "null"), (dict(k=0), "null"),
             (dict(v=0), "null"), (dict(table=0), "null")]


@pytest.mark.parametrize("more,word", BAD_PAGES)
def test_pages_that_are_refused(more, word):
    lib = ffi.load()
    _refused(lib.ah_paged_append(pages(**more), append()), word)
    _refused(lib.ah_paged_attention(pages(**more), attention()), word)


@pytest.mark.parametrize("more,word", [
    (dict(rows=-1), "rows"), (dict(rot_dim=63), "rot_dim"), (dict(rot_dim=-2), "rot_dim"), (dict(rot_dim=66), "rot_dim"), (dict(heads=-1), "heads"),
    (dict(rot_rows=-1), "positions"), (dict(q_st=4), "16 bytes"), (dict(q_sh=63), "16 bytes"), (dict(k_st=4), "16 bytes"), (dict(v_sh=2), "16 bytes"),
    (dict(r_st=9), "16 bytes"), (dict(k=P + 4), "16 bytes"), (dict(q=P + 2), "16 bytes"), (dict(rotary=P + 4), "16 bytes"), (dict(k=0), "null"), (dict(v=0), "null"),
    (dict(q=0), "null"), (dict(rotated=0), "null"), (dict(rotary=0), "null"), (dict(rot_dim=0), "rotation"), (dict(rot_dim=0, q=0, rotated=0), "rotation")])
def test_new_tokens_that_are_refused(more, word):
    _refused(ffi.load().ah_paged_append(pages(), append(**more)), word)


@pytest.mark.parametrize("more,word", [
    (dict(rows=-1), "rows"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"), (dict(heads=1 << 17), "multiple"), (dict(q_st=4), "16 bytes"),
    (dict(o_sh=4), "16 bytes"), (dict(q=P + 8), "16 bytes"), (dict(o=P + 8), "16 bytes"), (dict(lse=P + 2), "16 bytes"), (dict(soft_cap=-1.0), "soft_cap"),
    (dict(soft_cap=float("inf")), "soft_cap"), (dict(soft_cap=float("nan")), "soft_cap"), (dict(scale=float("nan")), "scale"), (dict(q=0), "null"),
    (dict(o=0), "null")])
def test_queries_that_are_refused(more, word):
    _refused(ffi.load().ah_paged_attention(pages(), attention(**more)), word)


@pytest.mark.parametrize("more,word", [
    (dict(dtype=ffi.F16), "dtype"), (dict(vocab=0), "vocabulary"), (dict(vocab=(1 << 20) + 1, ld=1 << 21), "vocabulary"), (dict(rows=-1), "rows"),
    (dict(rows=1 << 31), "rows"), (dict(ld=99), "apart"), (dict(logits=0), "null"), (dict(uniform=0), "null"), (dict(tokens=0), "null"),
    (dict(logits=P + 2), "multiple"), (dict(top_k=P + 1), "multiple"), (dict(logprobs=P + 3), "multiple")])
def test_logits_that_are_refused(more, word):
    _refused(ffi.load().ah_sample(sample(**more)), word)


def test_missing_structs_are_refused_and_nothing_else_is_before_a_device_is_asked_for():
    lib = ffi.load()
    for rc in (lib.ah_paged_append(None, append()), lib.ah_paged_append(pages(), None), lib.ah_paged_attention(None, attention()),
               lib.ah_paged_attention(pages(), None), lib.ah_sample(None)):
        assert rc == 2
    if lib.ah_sync() == 3:                       # no device initialised in this process
        for rc in (lib.ah_paged_append(pages(), append()), lib.ah_paged_attention(pages(), attention()), lib.ah_sample(sample()),
                   lib.ah_paged_append(pages(seqs=0, starts=0, k=0), append(rows=0, q=0))):
            assert rc == 3, lib.ah_last_error()
