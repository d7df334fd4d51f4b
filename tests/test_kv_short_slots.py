"""A slot's page and token without 64-bit divisions (scriptonait_amd/csrc/kv_index.h),
compiled for the host: the same as with them, for pools below 2^31 tokens."""
import subprocess
import textwrap
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "scriptonait_amd" / "csrc"

MAIN = textwrap.dedent(r"""
    #include <stdint.h>
    #include <stdio.h>
    #include <initializer_list>
    #include "kv_index.h"
    using namespace llmhip;
    int main() {
      long wrong = 0;
      uint64_t x = 1;
      for (uint32_t page : {1u, 2u, 3u, 7u, 16u, 20u, 24u, 64u, 100u, 256u, 65537u, 0x7fffffffu}) {
        for (uint32_t pages : {1u, 2u, 77u, 0x7fffffffu / page}) {
          const int64_t end = (int64_t)pages * page;
          if (end > 0x7fffffff) continue;
          const FastDiv by = FastDiv::of(page);
          const auto check = [&](int64_t slot) {
            uint32_t p = 9, t = 9, q = 9, u = 9;
            bool bad = false, worse = false;
            const bool a = split_slot(slot, pages, page, p, t, bad), b = split_short_slot(slot, pages, by, q, u, worse);
            wrong += a != b || bad != worse || p != q || t != u || (b && (q >= pages || u >= page));
          };
          for (int64_t s : {INT64_MIN, (int64_t)-1, (int64_t)0, end - 1, end, end + 1, (int64_t)1 << 31, (int64_t)1 << 32, INT64_MAX}) check(s);
          for (int i = 0; i < 20000; ++i) {
            x = x * 6364136223846793005ull + 1442695040888963407ull;
            check((int64_t)((x >> 32) % (uint64_t)(end + 3)));
          }
        }
      }
      printf("%ld\n", wrong);
    }
""")


def test_both_ways_agree(tmp_path):
    (tmp_path / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")], check=True)
    assert subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True).stdout == "0\n"
