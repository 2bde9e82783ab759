"""Builds the HIP engine library in-tree: instantllm_amd/libillhip.so (gfx950).

Flags: -O3, -ffp-contract=off (every multiply-add in the kernels is written as an explicit
fmaf, so the per-row arithmetic is the same instruction sequence in every T-instantiation),
and packed-FP32 instruction selection disabled.
"""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
SRCS = [HERE / "csrc" / f"{name}.hip" for name in ("ill_engine", "ill_mx", "ill_paged_mx")]
OUT = HERE / "libillhip.so"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result", "-Wno-unused-value",
]
LINK = ["-shared", f"-Wl,--version-script={HERE / 'csrc' / 'exports.map'}"]


def _run(cmd: list[str]) -> str:
    r = subprocess.run(cmd, capture_output=True, text=True)
    out = "\n".join(line for line in (r.stdout + r.stderr).splitlines()
                    if "packed-fp32-ops" not in line)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed ({r.returncode}):\n{out}")
    return out


def build(verbose: bool = False) -> Path:
    """Compiles the sources side by side and links them."""
    tmp = OUT.with_suffix(".so.tmp")
    with tempfile.TemporaryDirectory() as d, ThreadPoolExecutor(len(SRCS)) as pool:
        objects = [str(Path(d) / f"{src.stem}.o") for src in SRCS]
        said = list(pool.map(_run, [[HIPCC, *FLAGS, "-c", str(src), "-o", o] for src, o in zip(SRCS, objects)]))
        said.append(_run([HIPCC, *FLAGS, *LINK, *objects, "-o", str(tmp)]))
    if verbose and "".join(said).strip():
        print("\n".join(s for s in said if s.strip()))
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    p = build(verbose=True)
    print("built", p, p.stat().st_size, "bytes")
    sys.exit(0)
