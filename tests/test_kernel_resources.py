"""Registers, scratch and LDS of kernels as the compiler reports them, without a GPU: limits that a change of a neighbouring kernel
must not pass unseen."""
from __future__ import annotations

import re
import subprocess
from pathlib import Path

import pytest

from instantllm_amd import build

CSRC = Path(__file__).resolve().parents[1] / "instantllm_amd" / "csrc"


def _compile(tmp_path, text: str, *flags: str) -> str:
    """What the compiler says."""
    if not Path(build.HIPCC).exists():
        pytest.skip("no hipcc")
    src = tmp_path / "k.hip"
    src.write_text(text)
    said = subprocess.run([build.HIPCC, *build.FLAGS, "-w", *flags, str(src)], capture_output=True, text=True)
    assert said.returncode == 0, said.stderr
    return said.stderr


def _resources(tmp_path, text: str) -> dict[str, dict[str, int]]:
    """What the compiler says of each kernel, by its name, in their order."""
    said = _compile(tmp_path, text, "-Rpass-analysis=kernel-resource-usage", "--cuda-device-only", "-c", "-o", str(tmp_path / "k.o"))
    names, found = [], []
    for part in said.split("Function Name: ")[1:]:
        names.append(part.split(" ")[0])
        found.append({k.strip(): int(v) for k, v in re.findall(r"remark: [^\n]*?    ([A-Z][\w ]*?)(?: \[[\w/]+\])?: (\d+) \[-Rpass", part)})
    plain = subprocess.run(["c++filt"], input="\n".join(names), capture_output=True, text=True, check=True).stdout.split("\n")
    return {re.sub(r"^void ", "", name): f for name, f in zip(plain, found)}


# What the 16-bit caches' kernels took before microscaled caches came: (kernel, spilled scalar registers, spilled vector registers,
# bytes of scratch, bytes of LDS)
PAGED = [("pg_step_kernel<PG_F16, 64, false, false>(PgStep)", 2, 0, 0, 66208), ("pg_step_kernel<PG_BF16, 128, true, false>(PgStep)", 2, 0, 0, 66208),
         ("pg_prompt_kernel<PG_F16, 64, false, false>(PgStep)", 16, 0, 0, 32944), ("pg_prompt_kernel<PG_BF16, 128, false, false>(PgStep)", 9, 19, 80, 65712),
         ("pg_both_kernel<PG_F16, 64, false, false>(PgBoth)", 28, 0, 0, 66208), ("pg_both_kernel<PG_BF16, 128, true, false>(PgBoth)", 29, 14, 60, 66208)]


def test_attention_over_16_bit_caches(tmp_path):
    """Pays nothing for what only microscaled caches use."""
    text = f'#include <hip/hip_runtime.h>\n#include "{CSRC}/ill_paged.h"\n' + "".join(f"template __global__ void {k[0]};\n" for k in PAGED)
    found = _resources(tmp_path, text)
    assert len(found) == len(PAGED)
    for got, (kernel, sgprs, vgprs, scratch, lds) in zip(found.values(), PAGED):
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
    _compile(tmp_path, JOINS % CSRC, "--cuda-host-only", "-fsyntax-only")


def test_products(tmp_path):
    """No kernel of the microscaled operators spills, and slices are launched with as many workgroups for a CU as it holds."""
    found = _resources(tmp_path, f'#include "{CSRC}/ill_mx.hip"\n')
    assert len(found) > 30 and not {k: v for k, v in found.items() if v["VGPRs Spill"] or v["SGPRs Spill"] or v["ScratchSize"]}
    slices = [(re.fullmatch(r"mx_slice_kernel<(\d), (true|false), (\d)>.*", k), v["Occupancy"]) for k, v in found.items() if k.startswith("mx_slice")]
    held = "".join(f"static_assert(MxSlice<{m[2]}, {m[3]}>::EACH * MxSlice<{m[2]}, {m[3]}>::WAVES <= {4 * waves}, \"{m[0]}\");\n" for m, waves in slices)
    assert len(slices) >= 8
    _compile(tmp_path, f'#include <hip/hip_runtime.h>\n#include "{CSRC}/ill_mx.h"\n{held}', "--cuda-host-only", "-fsyntax-only")
