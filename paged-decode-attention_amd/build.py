"""Build `pagedattn/libpagedattn_hip.so` from csrc/ with hipcc for gfx950.

Usage: python paged-decode-attention_amd/build.py   (or __graft_entry__.build())
The library is written in-tree next to the Python package that loads it.
"""

from __future__ import annotations

import os
import pathlib
import subprocess
import sys
import tempfile

PKG_ROOT = pathlib.Path(__file__).resolve().parent
REPO_ROOT = PKG_ROOT.parent
SOURCES = [PKG_ROOT / "csrc" / name
           for name in ("paged_decode.hip", "cache_write.hip", "paged_prefill.hip", "paged_stream.hip", "step_tables.hip")]
OUTPUT = PKG_ROOT / "pagedattn" / "libpagedattn_hip.so"
ARCH = os.environ.get("PAGEDATTN_ARCH", "gfx950")

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    # packed-FP32 VALU forms are kept out of the generated code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def hipcc() -> str:
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    cand = pathlib.Path(rocm) / "bin" / "hipcc"
    return str(cand) if cand.exists() else "hipcc"


def build(verbose: bool = True) -> pathlib.Path:
    """Compile every source (all at once: one process each) and link the library."""
    noise = "is not a recognized feature for this target"
    compile_flags = [f for f in HIPCC_FLAGS if f != "-shared"]
    with tempfile.TemporaryDirectory() as tmp:
        objects = [pathlib.Path(tmp) / (src.stem + ".o") for src in SOURCES]
        cmds = [[hipcc(), *compile_flags, f"-I{REPO_ROOT / 'include'}", "-c", str(src), "-o", str(obj)]
                for src, obj in zip(SOURCES, objects)]
        if verbose:
            for cmd in cmds:
                print("[build]", " ".join(cmd), flush=True)
        procs = [subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True) for cmd in cmds]
        outs = [p.communicate() for p in procs]
        for src, proc, (_, stderr) in zip(SOURCES, procs, outs):
            err = "\n".join(l for l in stderr.splitlines() if noise not in l)
            if proc.returncode != 0:
                raise RuntimeError(f"hipcc failed on {src.name} ({proc.returncode}):\n{err}")
            if verbose and err.strip():
                print(err, file=sys.stderr)
        lib = OUTPUT.with_suffix(".so.tmp")
        link = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objects), "-o", str(lib)]
        if verbose:
            print("[build]", " ".join(link), flush=True)
        res = subprocess.run(link, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"hipcc failed to link ({res.returncode}):\n{res.stderr}")
    os.replace(lib, OUTPUT)
    return OUTPUT


if __name__ == "__main__":
    print(build())
