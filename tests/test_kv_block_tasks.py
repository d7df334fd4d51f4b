"""Sizes of the block append's tables (scriptonait_amd/csrc/kv_block_tasks.h),
compiled for the host: over all head sizes, rotations, types and blocks they fit
what a workgroup has."""
import subprocess
import textwrap
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "scriptonait_amd" / "csrc"

MAIN = textwrap.dedent(r"""
    #include <stdio.h>
    #include "kv_block_tasks.h"
    using namespace llmhip;
    int main() {
      uint32_t most_tokens = 0, most_bytes = 0, most_steps = 0, wrong = 0;
      for (uint32_t dim = 8; dim <= 256; dim += 8)
        for (uint32_t dims = 0; dims <= dim; dims += 2)
          for (uint32_t elem : {2u, 4u})
            for (int neighbours = 0; neighbours < 2; ++neighbours) {
              const uint32_t vec = append_vec(elem, neighbours, dims, dim);
              // Vectors of a row's two parts are whole, and so are pairs' places.
              wrong += dims % (2 * vec) != 0 || (dim - dims) % (2 * vec) != 0 || vec * elem > 16 || dim % (2 * vec) != 0;
              const uint32_t half = dims / 2, row = dim / (2 * vec), units = kAppendThreads * append_held(vec);
              if (!half) continue;
              for (uint32_t longest = 1; longest <= 256; ++longest) {
                const uint32_t tokens = append_turn_tokens(longest, vec, dim);
                // A step's tokens (of one block, begun and ended inside a token) are among them.
                wrong += tokens < std::min(longest, (units - 1) / row + 2);
                most_tokens = std::max(most_tokens, tokens);
                most_bytes = std::max(most_bytes, half * std::max(tokens, kMaxQueryTokens) * 8u);
                // The turns that a thread makes out of the one before, from its first token on.
                const uint32_t stride = kAppendThreads / half;
                most_steps = std::max(most_steps, (std::max(tokens, kMaxQueryTokens) - 1) / stride);
              }
            }
      printf("%u %u %u %u\n", wrong, most_tokens, most_bytes, most_steps);
    }
""")


def test_tables_fit(tmp_path):
    (tmp_path / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")],
                   check=True)
    out = subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True).stdout
    wrong, tokens, size, steps = map(int, out.split())
    assert wrong == 0
    assert tokens <= 256 + 15  # what the kernel has positions for
    # 64 KiB of LDS, with 64 runs of 16 bytes, the positions and four maxima beside the table.
    assert size + 64 * 16 + 4 * 271 + 16 <= 64 * 1024
    assert steps == 31  # as the kernel's comment on its error says
