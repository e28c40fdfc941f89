"""Build the sm_100a shared library picolm_b200/libpl_attn.so in tree.

    python -m picolm_b200.build            # or: make -C picolm_b200

nvcc compiles csrc/pl_attn.cu (the FP16 cache and everything around it) and
csrc/pl_kv8.cu (rotary positions and the 8-bit paged cache), which include
the kernel headers, for sm_100a only and links the CUDA runtime statically.
The driver API entry point the module needs (cuTensorMapEncodeTiled) is looked
up at run time through cudaGetDriverEntryPoint, so the library has no link-time dependency
on libcuda and loads on a host without a GPU (its calls then fail with
PL_EDEVICE).  ptxas' resource report (registers, spills per kernel) is
kept beside the library in libpl_attn.resources.json, and the build fails if
the kernels that split their registers between warpgroups do not have the
count the split needs.
"""
from __future__ import annotations

import json
import os
import re
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = [os.path.join(HERE, "csrc", f) for f in ("pl_attn.cu", "pl_kv8.cu")]
OUT = os.path.join(HERE, "libpl_attn.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O2",
    "-cudart", "static",
    "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    csrc = os.path.join(HERE, "csrc")
    out = [os.path.join(csrc, f) for f in sorted(os.listdir(csrc))]
    out.append(os.path.join(INCLUDE, "pl_attn.h"))
    return out


def up_to_date() -> bool:
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(s) <= t for s in sources())


RESOURCES = os.path.join(HERE, "libpl_attn.resources.json")

# The prefill kernels split the registers of their launch allocation between
# warpgroups with setmaxnreg: they need exactly this many per thread at
# launch (65536 / 384 threads, rounded down to 8), or the increase of the
# softmax warpgroups can never be granted.
PREFILL_LAUNCH_REGS = 168
# The same for the 8-bit cache's chunk attention: 65536 / 512 threads.
CHUNK_LAUNCH_REGS = 128


def parse_ptxas(text: str) -> dict:
    """{mangled kernel name: {"registers": n, "spill_stores": b, "spill_loads": b}}
    from nvcc -Xptxas=-v output."""
    out, cur = {}, None
    for line in text.splitlines():
        m = re.search(r"Compiling entry function '([^']+)'", line)
        if m:
            cur = m.group(1)
            out[cur] = {}
            continue
        if cur is None:
            continue
        m = re.search(r"(\d+) bytes spill stores, (\d+) bytes spill loads", line)
        if m:
            out[cur]["spill_stores"] = int(m.group(1))
            out[cur]["spill_loads"] = int(m.group(2))
        m = re.search(r"Used (\d+) registers", line)
        if m:
            out[cur]["registers"] = int(m.group(1))
    return out


def check_resources(res: dict) -> None:
    """Fail the build, not a later launch, when a toolkit change moves the
    prefill kernels off the register count their warpgroup split needs."""
    for name, regs in (("prefill_attn_kernel", PREFILL_LAUNCH_REGS),
                       ("kv8_chunk_kernel", CHUNK_LAUNCH_REGS)):
        of = {k: v for k, v in res.items() if name in k}
        if not of:
            raise RuntimeError(f"ptxas reported no {name}")
        bad = {k: v.get("registers") for k, v in of.items() if v.get("registers") != regs}
        if bad:
            raise RuntimeError(f"{name} needs {regs} registers per thread at launch, "
                               f"ptxas gave {bad}")


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date() and os.path.exists(RESOURCES):
        return OUT
    with tempfile.TemporaryDirectory() as tmp:
        # the translation units side by side, each with its own ptxas report
        objs, cmds = [], []
        for src in SRC:
            objs.append(os.path.join(tmp, os.path.basename(src) + ".o"))
            cmds.append([nvcc(), "-Xptxas=-v", *NVCC_FLAGS, "-I", INCLUDE, "-c", "-o", objs[-1], src])
        runs = [subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
                for c in cmds]
        text = [r.communicate()[0] for r in runs]
        cmds.append([nvcc(), *NVCC_FLAGS, "-shared", "-o", OUT, *objs])
        codes = [r.returncode for r in runs]
        if not any(codes):
            r = subprocess.run(cmds[-1], capture_output=True, text=True)
            text.append(r.stdout + r.stderr)
            codes.append(r.returncode)
    for cmd, out, rc in zip(cmds, text, codes):
        if verbose:
            print(" ".join(cmd))
        if verbose or rc:
            sys.stderr.write(out)
        if rc:
            raise subprocess.CalledProcessError(rc, cmd)
    res = {}
    for out in text:
        res.update(parse_ptxas(out))
    with open(RESOURCES, "w") as f:
        json.dump(res, f, indent=1, sort_keys=True)
    check_resources(res)
    return OUT


if __name__ == "__main__":
    build(force=True, verbose="-v" in sys.argv)
    print(OUT)
