"""The host's side of the 8-bit paged cache's calls, without a GPU: the index
arithmetic that kernels and host share, compiled here."""

import os
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def compiled(tmp_path, body):
    """Runs `body` as a C++ main over the kernels' shared header."""
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text('#include "kv8.h"\n#include <cstdio>\n#include <initializer_list>\nusing namespace grx;\n'
                   "int main() {\n" + body + "\nreturn 0;\n}\n")
    cuda = Path(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")).parents[1] / "include"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(ROOT / "gorelaxor_b200/csrc"), "-I", str(cuda), str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()


def test_append_groups_past_2_to_the_24_blocks(tmp_path):
    """A launch's groups of threads are numbered from 0 up without a gap or a
    repeat, however many blocks there are: the first and the last groups of a
    block, and of the largest launch that the entry point takes."""
    out = compiled(tmp_path, """
  for (int threads : {8, 16, 32, 256}) {
    const uint32_t per = 256 / threads;
    for (int64_t groups : {int64_t(1), int64_t(per) + 1, int64_t(16842495), int64_t(268697600), int64_t(2147483647)}) {
      const uint32_t grid = kv8_append_grid(groups, threads);
      if (int64_t(grid) * per < groups || int64_t(grid - 1) * per >= groups || grid > 2147483647u) std::puts("grid");
      for (uint32_t block : {0u, 1u, (1u << 24) - 1, 1u << 24, (1u << 24) + 1, 1u << 27, grid - 1}) {
        if (block >= grid) continue;
        for (uint32_t thread : {0u, 255u})
          if (kv8_append_group(block, thread, threads) != int64_t(block) * per + thread / threads)
            std::printf("group:%d:%u\\n", threads, block);
      }
    }
  }
  // pages that a sequence's new tokens can touch
  for (int page : {16, 32, 64})
    for (int64_t t : {int64_t(1), int64_t(2), int64_t(page), int64_t(page) + 1, int64_t(4096), int64_t(2147483647)})
      if (kv8_append_pages(int(t), page) != (page - 1 + t - 1) / page + 1) std::puts("pages");""")
    assert out == []
