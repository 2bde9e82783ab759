"""Registers, scratch and LDS of kernels as the compiler reports them, without a GPU: limits that a change of a neighbouring kernel
must not pass unseen."""
from __future__ import annotations

import re
import subprocess
from pathlib import Path

import pytest

from instantllm_amd import build

CSRC = Path(__file__).resolve().parents[1] / "instantllm_amd" / "csrc"


def _resources(tmp_path, header: str, kernels: list[str]) -> list[dict[str, int]]:
    """What the compiler says of each kernel, in their order."""
    if not Path(build.HIPCC).exists():
        pytest.skip("no hipcc")
    src = tmp_path / "k.hip"
    src.write_text(f'#include <hip/hip_runtime.h>\n#include "{CSRC / header}"\n' + "".join(f"template __global__ void {k};\n" for k in kernels))
    cmd = [build.HIPCC, *build.FLAGS, "-w", "-Rpass-analysis=kernel-resource-usage", "--cuda-device-only", "-c", str(src), "-o", str(tmp_path / "k.o")]
    said = subprocess.run(cmd, capture_output=True, text=True)
    assert said.returncode == 0, said.stderr
    got = [{k.strip(): int(v) for k, v in re.findall(r"remark: [^\n]*?    ([A-Z][\w ]*?)(?: \[[\w/]+\])?: (\d+) \[-Rpass", part)}
           for part in said.stderr.split("Function Name: ")[1:]]
    assert len(got) == len(kernels), said.stderr
    return got


# What the 16-bit caches' kernels took before microscaled caches came: (kernel, spilled scalar registers, spilled vector registers,
# bytes of scratch, bytes of LDS)
PAGED = [("pg_step_kernel<PG_F16, 64, false, false>(PgStep)", 2, 0, 0, 66208), ("pg_step_kernel<PG_BF16, 128, true, false>(PgStep)", 2, 0, 0, 66208),
         ("pg_prompt_kernel<PG_F16, 64, false, false>(PgStep)", 16, 0, 0, 32944), ("pg_prompt_kernel<PG_BF16, 128, false, false>(PgStep)", 9, 19, 80, 65712),
         ("pg_both_kernel<PG_F16, 64, false, false>(PgBoth)", 28, 0, 0, 66208), ("pg_both_kernel<PG_BF16, 128, true, false>(PgBoth)", 29, 14, 60, 66208)]


def test_attention_over_16_bit_caches(tmp_path):
    """Pays nothing for what only microscaled caches use."""
    for got, (kernel, sgprs, vgprs, scratch, lds) in zip(_resources(tmp_path, "ill_paged.h", [k[0] for k in PAGED]), PAGED):
        assert got["SGPRs Spill"] <= sgprs and got["VGPRs Spill"] <= vgprs and got["ScratchSize"] <= scratch, (kernel, got)
        assert got["LDS Size"] <= lds and got["Occupancy"] >= 2, (kernel, got)


JOINS = r"""
#include <hip/hip_runtime.h>
#include <cstddef>
#include "%s/ill_paged.h"
// What a join of PG_FAN parts of M rows of D dims reads and writes, in bytes: weights and sums of the parts, references and sums of the rows, and
// the states that groups of threads hand to the first one, for every number of rows.
template <int M>
constexpr size_t need(int D) {
  size_t most = 0;
  for (int live = 1; live <= M; live++) {
    const int items = live * (D / 4), groups = items <= PG_THREADS / 4 ? 4 : items <= PG_THREADS / 2 ? 2 : 1, width = PG_THREADS / groups;
    const size_t states = (size_t)(groups - 1) * (groups > 1 ? (width > items ? width : items) : 0);
    most = states > most ? states : most;
  }
  return (2 * PG_FAN * M + 2 * M) * sizeof(float) + most * sizeof(v4f);
}
template <int M, class L>
constexpr bool fits(int D) { return sizeof(L::join) >= need<M>(D) && offsetof(L, join) + sizeof(L::join) <= offsetof(L, last); }
static_assert(fits<16, PgStepLds<false>>(64) && fits<16, PgStepLds<true>>(64) && fits<16, PgStepLds<false>>(128) && fits<16, PgStepLds<true>>(128));
static_assert(fits<128, PgPromptLds<64, false>>(64) && fits<128, PgPromptLds<64, true>>(64));
static_assert(fits<128, PgPromptLds<128, false>>(128) && fits<128, PgPromptLds<128, true>>(128));
"""


def test_joins_have_their_lds(tmp_path):
    """The area of a join holds all that it touches, and ends before what lives on beside it."""
    if not Path(build.HIPCC).exists():
        pytest.skip("no hipcc")
    (tmp_path / "j.hip").write_text(JOINS % CSRC)
    said = subprocess.run([build.HIPCC, "--offload-arch=gfx950", "-std=c++17", "--cuda-host-only", "-fsyntax-only", "-w", "-Wno-invalid-offsetof", str(tmp_path / "j.hip")],
                          capture_output=True, text=True)
    assert said.returncode == 0, said.stderr
