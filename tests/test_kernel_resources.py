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
# bytes of scratch, bytes of LDS but for 16)
PAGED = [("pg_step_kernel<PG_F16, 64, false, false>(PgStep)", 2, 0, 0, 66208), ("pg_step_kernel<PG_BF16, 128, true, false>(PgStep)", 2, 0, 0, 66208),
         ("pg_prompt_kernel<PG_F16, 64, false, false>(PgStep)", 16, 0, 0, 32944), ("pg_prompt_kernel<PG_BF16, 128, false, false>(PgStep)", 9, 19, 80, 65712),
         ("pg_both_kernel<PG_F16, 64, false, false>(PgBoth)", 28, 0, 0, 66208), ("pg_both_kernel<PG_BF16, 128, true, false>(PgBoth)", 29, 14, 60, 66208)]


def test_attention_over_16_bit_caches(tmp_path):
    """Pays nothing for what only microscaled caches use."""
    for got, (kernel, sgprs, vgprs, scratch, lds) in zip(_resources(tmp_path, "ill_paged.h", [k[0] for k in PAGED]), PAGED):
        assert got["SGPRs Spill"] <= sgprs and got["VGPRs Spill"] <= vgprs and got["ScratchSize"] <= scratch, (kernel, got)
        assert got["LDS Size"] <= lds + 16 and got["Occupancy"] >= 2, (kernel, got)
