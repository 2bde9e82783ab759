"""Work division of the paged-cache attention (instantllm_amd/csrc/ill_paged_plan.h), compiled with the host compiler and
evaluated on the CPU: every visible key belongs to exactly one tile of exactly one part, and what the workspace and the launch
assume holds."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "instantllm_amd" / "csrc"

SEARCH = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "ill_paged_plan.h"
#define CHECK(x) do { if (!(x)) { printf("failed: %s (line %d)\n", #x, __LINE__); return 1; } } while (0)

static unsigned long long state = 88172645463325252ull;
static int draw(int lo, int hi) {   // lo .. hi
  state ^= state << 13; state ^= state >> 7; state ^= state << 17;
  return lo + (int)(state % (unsigned long long)(hi - lo + 1));
}

int main() {
  // sequences: rows stay inside the buffers and stand at the last positions
  for (int i = 0; i < 200000; i++) {
    const int rows = draw(0, 50), begin = draw(-5, 60), end = draw(-5, 60), len = draw(-10, 100);
    const PgSeq q = pg_seq(begin, end, len, rows);
    CHECK(q.n >= 0 && q.first >= 0 && q.first + q.n <= rows);
    if (q.n) CHECK(q.first >= begin && q.first + q.n <= end && q.p0 == (len > 0 ? len : 0) - (end - q.first));
  }
  CHECK(pg_seq(-2147483647 - 1, 2147483647, 5, 1 << 30).n == 1 << 30);
  CHECK(pg_seq(0, 2147483647, 2147483647, 1 << 30).p0 == (1 << 30) - 2147483647 || pg_seq(0, 2147483647, 2147483647, 1 << 30).p0 == -PG_MOST);

  for (int i = 0; i < 30000; i++) {
    PgCut c{};
    c.G = draw(1, 20); c.kv = draw(1, 4); c.M = draw(0, 1) ? 16 : 128; c.KT = draw(0, 1) ? 64 : 32;
    c.window = draw(0, 2) ? 0 : draw(1, 300); c.sinks = draw(0, 1) ? 0 : draw(0, 200);
    if (draw(0, 50) == 0) c.window = PG_MOST, c.sinks = PG_MOST;
    c.log = draw(0, 6); c.least = draw(1, 5); c.lo = draw(0, 1) ? 0 : draw(0, 64); c.hi = draw(0, 3) ? PG_MOST : draw(1, 64);
    const int seqs = draw(1, 6), width = draw(1, 40), log = 4;
    std::vector<PgSeq> seq(seqs);
    int rows = 0, most_rows = 0;
    for (auto& q : seq) {
      const int n = draw(0, 3) ? draw(0, 3) : draw(0, 70), len = draw(0, 5) ? draw(0, 700) : draw(0, 4);
      q = pg_seq(rows, rows + n, len, 1 << 20);
      CHECK(q.n == n);
      rows += n;
      most_rows = pg_max(most_rows, n);
    }
    const int cap = width << log;
    long long work = 0;
    for (auto& q : seq) { const int t = pg_qtiles(q.n, c) * c.kv; work += (long long)t * pg_most(q.p0 + q.n, cap, c); }
    const int part = pg_part(work, c);
    CHECK(part >= 1);
    long long units = 0, parts = 0, cut = 0;
    for (auto& q : seq) {
      const int t = pg_qtiles(q.n, c), most = pg_most(q.p0 + q.n, cap, c), splits = pg_splits(most, part);
      const long long flat = (long long)q.n * c.G;
      CHECK((t > 0) == (flat > c.lo && flat <= c.hi));
      if (t) CHECK((long long)t * c.M >= flat && (long long)(t - 1) * c.M < flat);
      units += (long long)t * c.kv * splits;
      if (splits > 1) { parts += (long long)t * c.kv * splits; cut += t * c.kv; }
      for (int k = 0; k < t; k++) {
        const int f0 = k * c.M, live = pg_min(c.M, (int)flat - f0);
        const int G = c.G, p0 = q.p0 + f0 / G, p1 = q.p0 + (f0 + live - 1) / G;
        const PgRange r = pg_range(p0, p1, cap, c);
        CHECK(r.n >= 0 && r.n <= most && r.sink <= r.n);
        // the tiles are distinct, ascending, and inside the cache
        for (int x = 0, before = -1; x < r.n; x++) {
          const int kt = pg_key_tile(r, x);
          CHECK(kt > before && kt * c.KT < pg_min(p1 + 1, cap));
          before = kt;
        }
        // every key that a row sees is in one of them
        for (int p = pg_max(p0, 0); p <= p1; p += pg_max(1, (p1 - p0) / 3))
          for (int j = 0; j <= pg_min(p, cap - 1); j++)
            if (pg_sees(p, j, c.window, c.sinks)) {
              const int kt = j / c.KT;
              CHECK(kt < r.sink || (kt >= r.lo && kt < r.lo + r.n - r.sink));
            }
        // the parts cover the tiles once
        const int per = pg_up(r.n, splits);
        int next = 0;
        for (int x = 0; x < splits; x++) {
          const int a = pg_min(x * per, r.n), b = pg_min(a + per, r.n);
          CHECK(a == next || a == b);
          next = b;
        }
        CHECK(next == r.n);
      }
    }
    CHECK(parts <= 2ll << c.log && cut <= 1ll << c.log);
    // the launch has a workgroup for every unit, where the sizes that the host knows hold
    CHECK(units <= pg_grid(seqs, rows, false, cap, c));
    if (most_rows <= 1 && rows == seqs) CHECK(units <= pg_grid(seqs, rows, true, cap, c));
  }
  // rows of sequences in any order (which is not allowed): nothing is cut where the units are more than the launch has, and
  // else the workspace holds the parts
  for (int i = 0; i < 20000; i++) {
    PgCut c{};
    c.G = draw(1, 20); c.kv = draw(1, 4); c.M = draw(0, 1) ? 16 : 128; c.KT = 64;
    c.log = draw(0, 6); c.least = draw(1, 5); c.hi = PG_MOST;
    const int seqs = draw(1, 6), rows = draw(1, 200), cap = 16 * draw(1, 40);
    long long work = 0, parts = 0, cut = 0;
    std::vector<PgSeq> seq(seqs);
    for (auto& q : seq) {
      q = pg_seq(draw(-5, 220), draw(-5, 220), draw(-10, 700), rows);
      work += (long long)pg_qtiles(q.n, c) * c.kv * pg_most(q.p0 + q.n, cap, c);
    }
    const int part = pg_part(work, c);
    for (auto& q : seq) {
      const int t = pg_qtiles(q.n, c) * (int)c.kv, most = pg_most(q.p0 + q.n, cap, c);
      if (pg_splits(most, part) > 1) { parts += (long long)t * pg_splits(most, part); cut += t; }
      CHECK(pg_splits(most, PG_MOST) == 1);
    }
    CHECK(parts <= 2ll << c.log && cut <= 1ll << c.log);
  }
  // two kernels: every sequence with rows is exactly one's
  for (int i = 0; i < 20000; i++) {
    PgCut step{}, prompt{};
    step.G = prompt.G = draw(1, 20); step.kv = prompt.kv = draw(1, 8); step.M = 16; prompt.M = 128;
    step.hi = prompt.hi = PG_MOST;
    int n[5];
    long long tiles = 0;
    for (int& x : n) { x = draw(0, 2) ? draw(0, 10) : draw(0, 900); tiles += pg_prompt_tiles(x, step.G, step.kv); }
    pg_share(step, tiles);
    pg_share(prompt, tiles);
    long long taken = 0, units = 0;
    int rows = 0;
    for (int x : n) { units += pg_qtiles(x, step) * (int)step.kv; rows += x; }
    step.shared = 1; step.KT = 64; step.least = 8; step.log = 8;
    CHECK(units <= pg_grid(5, rows, false, 64, step));   // (one tile of keys: no parts)
    for (int x : n) {
      CHECK((pg_qtiles(x, step) > 0) + (pg_qtiles(x, prompt) > 0) == (x > 0));
      taken += pg_qtiles(x, prompt) * (int)prompt.kv;
    }
    CHECK(taken == (tiles >= PG_MANY ? tiles : 0));
  }
  printf("ok\n");
  return 0;
}
"""


def test_work_division(tmp_path):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(SEARCH)
    subprocess.run([cxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.stdout.strip() == "ok" and out.returncode == 0, out.stdout + out.stderr
