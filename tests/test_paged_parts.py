"""The numbers of parts that test_gpu_paged_parts.py counts on, from instantllm_amd/csrc/ill_paged_plan.h on the CPU, with the
limits that ill_paged_host.h gives the prompt kernel."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from test_gpu_paged_parts import SHAPES

CSRC = Path(__file__).resolve().parents[1] / "instantllm_amd" / "csrc"

COUNT = r"""
#include <cstdio>
#include <cstdlib>
#include "ill_paged_plan.h"
int main(int argc, char** argv) {   // log, least, query heads of a key/value head, key/value heads, then length and rows of each sequence
  const int G = atoi(argv[3]), kv = atoi(argv[4]);
  PgCut c{(uint32_t)G, (uint32_t)kv, 128, 64, 0, 0, atoi(argv[1]), atoi(argv[2]), 0, PG_MOST, 1};
  long long tiles = 0, work = 0;
  for (int i = 5; i < argc; i += 2) tiles += pg_prompt_tiles(atoi(argv[i + 1]), G, kv);
  pg_share(c, tiles);
  for (int i = 5; i < argc; i += 2) work += (long long)pg_qtiles(atoi(argv[i + 1]), c) * kv * pg_most(atoi(argv[i]), 1 << 20, c);
  printf("%d %d\n", pg_qtiles(atoi(argv[6]), c), pg_splits(pg_most(atoi(argv[5]), 1 << 20, c), pg_part(work, c)));
}
"""


@pytest.mark.parametrize("seqs,heads,kv,parts", SHAPES, ids=[str(s[3]) for s in SHAPES])
def test_parts_of_the_first_sequence(tmp_path, seqs, heads, kv, parts):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no host compiler")
    body = re.search(r"PgCut prompt_cut\(.*?\{(.*?)\n\}", (CSRC / "ill_paged_host.h").read_text(), re.S).group(1)
    log, least = re.search(r"128, 64, window, sinks, (\d+), (\d+), 0, PG_MOST, 0", body).groups()
    fan = int(re.search(r"#define PG_FAN (\d+)", (CSRC / "ill_paged_plan.h").read_text()).group(1))
    src, exe = tmp_path / "count.cpp", tmp_path / "count"
    src.write_text(COUNT)
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    args = [log, least, heads // kv, kv] + [x for s in seqs for x in s]
    tiles, splits = map(int, subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, check=True).stdout.split())
    assert tiles > 0 and splits == parts > fan
