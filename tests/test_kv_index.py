"""Index arithmetic of the quantised cache on the CPU: csrc/kv_cache.h compiled
by the host compiler, and the C entry points' refusals (no GPU needed)."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "kv_cache.h"
using namespace phew::kv;
#define CHECK(x) do { if (!(x)) { std::printf("failed: %s line %d\n", #x, __LINE__); return 1; } } while (0)
int main() {
  // division by every small and some large divisors, at the borders of the quotient
  std::vector<uint32_t> ds;
  for (uint32_t d = 1; d < 700; ++d) ds.push_back(d);
  for (uint32_t d : {1023u, 1024u, 1025u, 65535u, 65536u, 65537u, 1000003u, (1u << 30), (1u << 30) + 1, 0x7fffffffu}) ds.push_back(d);
  for (uint32_t d : ds) {
    const FastDiv f = fast_div(d);
    for (uint64_t q = 0; q < 50; ++q)
      for (int64_t e = -1; e <= 1; ++e) {
        const int64_t n = static_cast<int64_t>(q * d) + e;
        if (n >= 0 && n < (1ll << 31)) CHECK(div_by(f, static_cast<uint32_t>(n)) == static_cast<uint32_t>(n) / d);
      }
    for (uint32_t n : {0x7fffffffu, 0x7ffffffeu, 0x40000000u, 0x3fffffffu}) CHECK(div_by(f, n) == n / d);
    for (int i = 0; i < 2000; ++i) {
      const uint32_t n = ((static_cast<uint32_t>(std::rand()) << 16) ^ static_cast<uint32_t>(std::rand())) & 0x7fffffffu;
      CHECK(div_by(f, n) == n / d);
    }
  }
  // rows of good tables are distinct and inside the cache; bad entries and positions give none
  for (int page : {1, 3, 8, 16, 24, 700}) {
    const int pages = 11, heads = 3, columns = 4, batch = 2;
    int32_t table[2 * 5] = {4, 0, 10, 7, 99, 1, 2, -1, 11, 99};  // rows 5 apart; sequence 1 has two bad pages
    PageMap m{table, 5, columns, pages, heads, page, fast_div(static_cast<uint32_t>(page))};
    std::vector<int> hit(static_cast<size_t>(pages) * heads * page, 0);
    for (int b = 0; b < batch; ++b)
      for (int h = 0; h < heads; ++h)
        for (int64_t pos = -3; pos < capacity(m) + 3; ++pos) {
          const uint32_t r = row_of(m, b, h, pos);
          const bool in = pos >= 0 && pos < capacity(m);
          const int want = in ? table[b * 5 + pos / page] : -1;
          if (!in || want < 0 || want >= pages) {
            CHECK(r == kNoRow);
            continue;
          }
          CHECK(r == static_cast<uint32_t>((want * heads + h) * page + pos % page));
          CHECK(hit[r]++ == 0);
        }
    PageMap n{nullptr, 0, 1, pages, heads, page, fast_div(static_cast<uint32_t>(page))};
    CHECK(row_of(n, 10, 2, page - 1) == static_cast<uint32_t>(pages * heads * page - 1));
    CHECK(row_of(n, 10, 2, page) == kNoRow && row_of(n, 11, 0, 0) == kNoRow);
  }
  // rows past 2^31
  PageMap far{nullptr, 0, 1, 1 << 20, 4, 1000, fast_div(1000)};
  CHECK(row_of(far, (1 << 20) - 1, 3, 999) == 4194304000u - 1u);
  // lengths and masks
  CHECK(clamp_count(-5, 10) == 0 && clamp_count(11, 10) == 10 && clamp_count(7, 10) == 7 && clamp_count(0x7fffffff, 1ll << 40) == 0x7fffffff);
  CHECK(seen_end(10, 3, 0, true) == 8 && seen_end(10, 3, 2, true) == 10 && seen_end(10, 3, 3, true) == 0);
  CHECK(seen_end(2, 5, 0, true) == 0 && seen_end(2, 5, 3, true) == 1 && seen_end(2, 5, 1, false) == 2);
  std::puts("ok");
  return 0;
}
"""


def test_index_arithmetic(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    src, exe = tmp_path / "h.cpp", tmp_path / "h"
    src.write_text(HARNESS)
    subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    str(ROOT / "phew_b200" / "csrc"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


@pytest.fixture(scope="module")
def lib():
    from phew_b200 import _native
    from phew_b200.build import build

    build()
    return _native.load()


FAKE = 4096  # never dereferenced: every check below runs before a launch


def cache(**over):
    from phew_b200 import _native

    f = dict(k_codes=FAKE, k_scales=FAKE, k_biases=FAKE, v_codes=FAKE, v_scales=FAKE, v_biases=FAKE, pages=8,
             page_size=16, kv_heads=2, head_dim=128, group_size=64, bits=4, dtype=_native.PHEW_BF16)
    f.update(over)
    return _native.KVCache(**f)


@pytest.mark.parametrize("over,message", [
    (dict(v_scales=None), "null cache array"),
    (dict(bits=2), "bits must be 4 or 8"),
    (dict(head_dim=96), "head_dim must be"),
    (dict(group_size=16), "group_size must be"),
    (dict(head_dim=64, group_size=128), "group_size must be"),
    (dict(dtype=9), "bad dtype"),
    (dict(pages=0), "empty cache"),
    (dict(pages=1 << 30, page_size=16), "too many rows"),
    (dict(k_codes=FAKE + 4), "16-byte aligned"),
])
def test_entry_points_refuse_bad_caches(lib, over, message):
    from phew_b200 import _native

    st = (ctypes.c_int64 * 3)(128, 128, 128)
    c = cache(**over)
    for status in (
        lib.phew_kv_update(c, FAKE, FAKE, st, st, 2, 1, FAKE, None, FAKE, 4, 4, None, None, FAKE, None),
        lib.phew_kv_fetch(c, FAKE, FAKE, 2, 16, FAKE, FAKE, 4, 4, FAKE, None),
        lib.phew_kv_attention(c, FAKE, st, FAKE, 2, 4, 1, FAKE, None, FAKE, 4, 4, 1.0, 0, FAKE, 1 << 40, FAKE, None),
    ):
        assert status == _native.PHEW_ERR_INVALID
        assert message in _native.last_error()


def test_entry_points_refuse_bad_arguments(lib):
    from phew_b200 import _native

    c, ok = cache(), (ctypes.c_int64 * 3)(128, 128, 128)
    odd = (ctypes.c_int64 * 3)(128, 129, 128)
    big = 1 << 40

    def refused(status, message):
        assert status == _native.PHEW_ERR_INVALID and message in _native.last_error(), _native.last_error()

    refused(lib.phew_kv_update(c, FAKE, FAKE, ok, odd, 2, 1, FAKE, None, FAKE, 4, 4, None, None, FAKE, None), "strides")
    refused(lib.phew_kv_update(c, FAKE, FAKE, ok, ok, 2, 1, FAKE, None, FAKE, 4, 4, FAKE, None, FAKE, None), "go together")
    refused(lib.phew_kv_update(c, FAKE, FAKE, ok, ok, 2, 1, FAKE, None, FAKE, 4, 4, None, None, None, None), "null pointer")
    refused(lib.phew_kv_update(c, FAKE, FAKE, ok, ok, 9, 1, FAKE, None, None, 0, 1, None, None, FAKE, None), "page per sequence")
    refused(lib.phew_kv_update(c, FAKE, FAKE, ok, ok, 2, 1, FAKE, None, FAKE, 4, 1 << 28, None, None, FAKE, None), "bad block table")
    refused(lib.phew_kv_fetch(c, FAKE, FAKE + 2, 2, 16, FAKE, FAKE, 4, 4, FAKE, None), "aligned")
    refused(lib.phew_kv_fetch(c, FAKE, FAKE, 2, 0, FAKE, FAKE, 4, 4, FAKE, None), "output length")
    attend = lambda cc, heads, tokens, st, ws: lib.phew_kv_attention(  # noqa: E731
        cc, FAKE, st, FAKE, 2, heads, tokens, FAKE, None, FAKE, 4, 4, 1.0, 0, FAKE, ws, FAKE, None)
    refused(attend(cache(bits=8), 4, 1, ok, big), "4-bit")
    refused(attend(c, 3, 1, ok, big), "multiple of the cache's kv_heads")
    refused(attend(c, 4, 0, ok, big), "token count")
    refused(attend(c, 4, 1, odd, big), "strides")
    wide = lambda cc, heads, columns: lib.phew_kv_attention(  # noqa: E731
        cc, FAKE, ok, FAKE, 2, heads, 1, FAKE, None, FAKE, columns, columns, 1.0, 0, FAKE, big, FAKE, None)
    refused(wide(cache(page_size=16), 4, (1 << 27) - 1), "too many tokens")  # 2^31 - 16
    refused(wide(cache(page_size=16, kv_heads=128), 128, (1 << 27) - 64), "too many tokens")  # 2^26 tiles of 128 heads
