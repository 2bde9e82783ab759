"""Which workspace a call of the paged-cache operators takes (instantllm_amd/csrc/ill_paged_claims.h), compiled with the host
compiler and evaluated on the CPU."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "instantllm_amd" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "ill_paged_claims.h"
#define CHECK(x) do { if (!(x)) { printf("failed: %s (line %d)\n", #x, __LINE__); return 1; } } while (0)
int main() {
  const char at[16] = {};
  const void *a = at, *b = at + 1, *c = at + 2, *none = nullptr;
  illp::Workspaces w;
  w.count = 3;
  // a stream and each of its captures have their own, always the same
  CHECK(w.claim(a, 0) == 0 && w.claim(a, 7) == 1 && w.claim(a, 0) == 0 && w.claim(none, 0) == 2 && w.claim(a, 7) == 1);
  CHECK(w.claim(a, 8) == -1 && w.claim(b, 0) == -1 && w.claim(none, 0) == 2);
  // what unbound calls hold cannot be bound, not by the stream itself either
  CHECK(!w.bind(b, 0) && !w.bind(a, 0) && w.bound_to(b) == -1 && w.bound_to(a) == -1);
  // a stream forgotten: its own and its captures' are free, no one else's
  w.forget(a);
  CHECK(w.claim(none, 0) == 2 && w.bind(b, 1) && w.bound_to(b) == 1 && w.bind(c, 1) && w.bind(b, 1));
  CHECK(!w.bind(b, 0) && w.bound_to(b) == 1);
  // calls of others pass a bound workspace over, for as long as a stream is bound to it
  CHECK(w.claim(a, 0) == 0 && w.claim(a, 9) == -1);
  w.forget(b);
  CHECK(w.bound_to(b) == -1 && w.claim(a, 9) == -1);
  w.forget(c);
  CHECK(w.claim(a, 9) == 1 && w.claim(b, 0) == -1);
  w.forget(none);
  CHECK(w.claim(b, 0) == 2);
  w.forget(at + 9);   // (never seen)
  w.clear();
  for (int i = 0; i < 3; i++) CHECK(w.claim(a, i) == i);
  w.clear();
  for (int i = 0; i < 16; i++) CHECK(w.bind(at + i, 2) && w.bound_to(at + i) == 2);
  CHECK(w.claim(none, 0) == 0 && w.claim(none, 1) == 1 && w.claim(none, 2) == -1);
  printf("ok\n");
  return 0;
}
"""


def test_claims_and_bindings(tmp_path):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "claims.cpp", tmp_path / "claims"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.stdout.strip() == "ok" and out.returncode == 0, out.stdout + out.stderr


def test_null_handle_is_refused():
    from instantllm_amd.engine import ILL_E_ARG, load_library
    if not (CSRC.parent / "libillhip.so").exists():
        pytest.skip("libillhip.so not built")
    assert load_library().ill_paged_bind(None, None, 0) == ILL_E_ARG
