"""The index arithmetic that the key-value cache's kernels read and write by
(scriptonait_amd/csrc/kv_index.h), compiled for the host: no length, page id
or slot, right or wrong, leads outside its range."""
import subprocess
import textwrap
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "scriptonait_amd" / "csrc"

MAIN = textwrap.dedent(r"""
    #include <stdint.h>
    #include <stdio.h>
    #include <initializer_list>
    #include "kv_index.h"
    using namespace llmhip;
    static long bad_cases = 0;
    #define CHECK(c) do { if (!(c)) { ++bad_cases; printf("line %d\n", __LINE__); } } while (0)
    int main() {
      const uint32_t top = 0x7fffffffu;
      uint64_t x = 1;
      for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 8u, 16u, 20u, 24u, 31u, 64u, 100u, 255u, 256u, 4095u, 65537u, 1u << 30, top - 1u, top}) {
        const FastDiv f = FastDiv::of(d);
        for (uint32_t n : {0u, 1u, d - 1u, d, d + 1u, 2u * d - 1u, top - 1u, top}) if (n <= top) CHECK(f.div(n) == n / d && f.mod(n) == n % d);
        for (int i = 0; i < 100000; ++i) {
          x = x * 6364136223846793005ull + 1442695040888963407ull;
          const uint32_t n = (uint32_t)(x >> 33);
          CHECK(f.div(n) == n / d);
        }
      }
      for (int32_t len : {INT32_MIN, -5, -1, 0, 1, 99, 100, 101, INT32_MAX}) {
        bool bad = false;
        const uint32_t n = clamp_len(len, 100u, bad);
        CHECK(n <= 100u && bad == (len < 0 || len > 100) && (bad || n == (uint32_t)len));
      }
      const uint32_t pages = 2000000000u, page = 24u;
      const int64_t end = (int64_t)pages * page;
      for (int64_t s : {INT64_MIN, (int64_t)-1, (int64_t)0, (int64_t)23, (int64_t)24, end - 1, end, end + 1, (int64_t)1 << 33, INT64_MAX}) {
        uint32_t p = 7, t = 7;
        bool bad = false;
        const bool live = split_slot(s, pages, page, p, t, bad);
        CHECK(live == (s >= 0 && s < end) && bad == (s >= end));
        if (live) CHECK(p < pages && t < page && (int64_t)p * page + t == s);
      }
      CHECK(window_start(0, 0) == 0 && window_start(10, 0) == 0 && window_start(10, 10) == 0 && window_start(10, 3) == 7);
      CHECK(window_start(0, 5) == 0 && window_start(5, 0x7fffffff) == 0);
      printf("%ld\n", bad_cases);
    }
""")


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(d / "main.cpp"), "-o", str(d / "main")], check=True)
    return d / "main"


def test_no_input_leaves_the_ranges(exe):
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "0\n"
