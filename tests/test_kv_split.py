"""How attention is split over workgroups (scriptonait_amd/csrc/kv_split.h),
compiled for the host: whatever the call, waves, teams and ranges fit the
launch, the workspace and the cuts that lie before its partial answers."""
import subprocess
import textwrap
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "scriptonait_amd" / "csrc"

MAIN = textwrap.dedent(r"""
    #include <stdio.h>
    #include <initializer_list>
    #include "kv_split.h"
    using namespace llmhip;
    static long bad_cases = 0, cut = 0, whole = 0;
    #define CHECK(c) do { if (!(c)) { if (++bad_cases < 20) printf("line %d: %u %u %u %u %u %u %u %u\n", __LINE__, waves, tile, bytes, cus, B, vheads, tokens, window); } } while (0)
    int main() {
      for (uint32_t waves : {4u, 8u})
        for (uint32_t tile : {16u, 32u})
          for (uint32_t bytes : {16u, 48u, 320u, 512u, 2048u})
            for (uint32_t cus : {1u, 3u, 80u, 256u, 304u, 1000u, 5000u})
              for (uint32_t B : {1u, 2u, 37u, 300u, 2048u, 2049u, 65535u})
                for (uint32_t vheads : {1u, 2u, 3u, 5u, 8u, 12u, 96u, 1001u, 65535u})
                  for (uint32_t tokens : {0u, 1u, 16u, 700u, 4096u, 1000000u, 0x7ffffe00u})
                    for (uint32_t window : {0u, 1u, 512u, 0x7ffffffeu}) {
                      const AttendSplit s = attend_split(waves, tile, bytes, cus, B, vheads, tokens, window);
                      CHECK(s.team >= 1 && s.team * s.splits == waves && vheads % s.team == 0);
                      if (s.ranges) {
                        ++cut;
                        CHECK(s.ranges <= kMaxRanges && B <= kMaxSplitBatch);
                        const unsigned long long most = vheads > 8ull * cus ? vheads : 8ull * cus;
                        CHECK((unsigned long long)s.ranges * vheads <= most);  // partial answers, half of them
                        CHECK(s.ranges == 1 || (unsigned long long)s.ranges * (vheads / s.team) <= cus * (8ull / waves));
                      } else {
                        ++whole;
                      }
                    }
      printf("%ld %d %d\n", bad_cases, cut > 10000, whole > 10000);
    }
""")


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_split")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(d / "main.cpp"), "-o", str(d / "main")], check=True)
    return d / "main"


def test_every_split_fits(exe):
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "0 1 1\n"
