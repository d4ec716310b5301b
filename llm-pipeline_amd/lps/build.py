"""In-tree build of ``liblps.so`` for gfx950 with hipcc: the translation units
of ``csrc/`` side by side, then one link.

Flags: ``-ffp-contract=off`` and correctly rounded fp32 division keep the
penalty / temperature arithmetic bit-identical to IEEE fp32; packed-fp32 ops
are disabled (``-packed-fp32-ops``)."""

from __future__ import annotations

import os
import subprocess
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
PKG_ROOT = os.path.dirname(HERE)                    # llm-pipeline_amd/
REPO = os.path.dirname(PKG_ROOT)
CSRC = os.path.join(PKG_ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
OUT = os.path.join(HERE, "liblps.so")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
    "-ffp-contract=off", "-fhip-fp32-correctly-rounded-divide-sqrt",
    "-Wall", "-Werror=return-type", "-Werror=uninitialized",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # a private array moved to LDS is addressed by the flat work-item id, which
    # makes every wave read the dispatch packet (host memory) first
    "-mllvm", "-disable-promote-alloca-to-lds",
]


UNITS = ("lps.hip", "lps_table.hip", "lps_mx4head.hip")


def _finish(cmd, proc) -> None:
    out, err = proc.communicate()
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{' '.join(cmd)}\n{out}\n{err}")


def _start(cmd):
    return cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)


def build(verbose: bool = False) -> str:
    """Compile the units of ``csrc`` into ``lps/liblps.so`` (always recompiles)."""
    tmp = OUT + ".tmp"
    with tempfile.TemporaryDirectory() as objs:
        made = [os.path.join(objs, u + ".o") for u in UNITS]
        cmds = [[HIPCC, *FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", os.path.join(CSRC, u), "-o", o]
                for u, o in zip(UNITS, made)]
        running = [_start(c) for c in cmds]
        try:
            for cmd, proc in running:
                _finish(cmd, proc)
        finally:
            for _, proc in running:
                if proc.poll() is None:
                    proc.kill()
                    proc.communicate()
        link = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *made]
        _finish(*_start(link))
        cmds.append(link)
    os.replace(tmp, OUT)
    if verbose:
        for cmd in cmds:
            print(" ".join(cmd))
    return OUT


if __name__ == "__main__":
    print(build(verbose=True))
