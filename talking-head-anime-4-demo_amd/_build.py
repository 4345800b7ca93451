"""Build the gfx950 shared library in-tree with hipcc (no JIT cache: the .so must travel with the tree)."""
from __future__ import annotations

import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(_HERE), "include")
LIB = os.path.join(CSRC, "libtha4_hip.so")
RESOURCES = os.path.join(CSRC, "libtha4_hip.resources.txt")
# The same source compiled with every memory wait forced to zero (-mllvm -amdgpu-waitcnt-forcezero=1): identical arithmetic, so a byte
# that differs from the shipped library is a memory-ordering / hazard fault in one of them (how round 3 found the faulty level-2
# geometry).  TEST ARTEFACT: only tests/test_twin_gpu.py and tools/compare_libs.py load it, through THA4_HIP_LIB.
TWIN = os.path.join(CSRC, "libtha4_hip_wait0.so")
# One object per source (kept under csrc/build/), so that a change to one family of kernels does not recompile the others (the posers' take minutes).
# The order is the link order: the posers' code object is the first of the library.
SOURCES = ["tha4_capi.hip", "tha4_transformer.hip"]
OBJECTS = os.path.join(CSRC, "build")
# No packed-fp32 VALU instructions (v_pk_mul / v_pk_fma / v_pk_add_f32) in any kernel of the library: the compiler's packed arithmetic is
# what made level2_16p_kernel<8,.,2> produce run-to-run varying pixels on gfx950 once the sine shrank to one instruction
# (profiles/r03_sin_cliff.md: wait states in front of every v_pk_* all but cure it, a build without them equals its forced-wait twin
# bit for bit), and it buys nothing here (a v_pk_fma_f32 costs two v_fma_f32).  THA4_NO_PACKED_FP32 tells the sources so.
DEVICE_FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-DTHA4_NO_PACKED_FP32=1"]


def is_transformer_header(name: str) -> bool:
    return name.startswith("transformer_")


def _dependencies(source: str):
    """Headers a source includes: transformer_*.h belong to tha4_transformer.hip alone, which includes nothing of the posers' kernels."""
    own = source == "tha4_transformer.hip"
    shared = ("tha4_platform.h", "tha4_tuning.h", "tha4_host.h")
    heads = [f for f in sorted(os.listdir(CSRC)) if f.endswith(".h") and (f in shared or is_transformer_header(f) == own)]
    return [os.path.join(CSRC, f) for f in [source] + heads] + [os.path.join(INCLUDE, "tha4_hip.h"), os.path.abspath(__file__)]


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def hipcc_path() -> str:
    p = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(p):
        raise RuntimeError("hipcc not found (ROCm toolchain required to build libtha4_hip.so)")
    return p


def _compile(source: str, tag: str, extra, force: bool, verbose: bool = False) -> str:
    """One source -> csrc/build/<name>.<tag>.o, with the resource report of its kernels beside it."""
    os.makedirs(OBJECTS, exist_ok=True)
    obj = os.path.join(OBJECTS, f"{os.path.splitext(source)[0]}.{tag}.o")
    report = obj[:-2] + ".resources.txt"
    if not force and not _stale(obj, _dependencies(source)) and os.path.exists(report):
        return obj
    cmd = [hipcc_path(), "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-c", "-Rpass-analysis=kernel-resource-usage"] + extra + DEVICE_FLAGS + \
          ["-I", CSRC, "-I", INCLUDE, os.path.join(CSRC, source), "-o", obj]
    if verbose:
        print(" ".join(cmd))
    r = subprocess.run(cmd, stderr=subprocess.PIPE, text=True)
    if r.returncode != 0:
        raise RuntimeError("hipcc failed:\n" + r.stderr[-4000:])
    with open(report, "w") as f:             # per-kernel VGPR / scratch / LDS report (tests/test_api_surface.py gates on it)
        f.write(parse_resource_remarks(r.stderr))
    return obj


def _link(target: str, tag: str, extra, force: bool, verbose: bool = False):
    with ThreadPoolExecutor(len(SOURCES)) as pool:
        objs = list(pool.map(lambda s: _compile(s, tag, extra, force, verbose), SOURCES))
    if force or _stale(target, objs):
        r = subprocess.run([hipcc_path(), "--offload-arch=gfx950", "-fPIC", "-shared"] + objs + ["-o", target], stderr=subprocess.PIPE, text=True)
        if r.returncode != 0:
            raise RuntimeError("hipcc failed (link):\n" + r.stderr[-4000:])
    return objs


def _current(target: str, tag: str) -> bool:
    """Whether the library is newer than every source and holds no object that is older than its own (a source edited while the others compiled)."""
    for s in SOURCES:
        obj = os.path.join(OBJECTS, f"{os.path.splitext(s)[0]}.{tag}.o")
        if _stale(target, _dependencies(s)) or (os.path.exists(obj) and _stale(obj, _dependencies(s))):
            return False
    return True


def build_native(force: bool = False, verbose: bool = False) -> str:
    if not force and _current(LIB, "product") and os.path.exists(RESOURCES):
        return LIB
    objs = _link(LIB, "product", [], force, verbose)
    with open(RESOURCES, "w") as f:
        for o in objs:
            f.write(open(o[:-2] + ".resources.txt").read())
    return LIB


def build_forced_wait_twin(force: bool = False) -> str:
    if not force and _current(TWIN, "wait0"):
        return TWIN
    _link(TWIN, "wait0", ["-mllvm", "-amdgpu-waitcnt-forcezero=1"], force)
    return TWIN


def parse_resource_remarks(stderr: str) -> str:
    """`-Rpass-analysis=kernel-resource-usage` remarks -> one line per kernel: name vgprs vgpr_spill scratch_bytes occupancy."""
    out, cur = [], {}
    for line in stderr.splitlines():
        if "remark:" not in line:
            continue
        body = line.split("remark:", 1)[1].split("[-Rpass", 1)[0].strip()
        if body.startswith("Function Name:"):
            if cur:
                out.append(cur)
            cur = {"name": body.split(":", 1)[1].strip()}
        elif ":" in body and cur:
            k, v = body.split(":", 1)
            cur[k.strip()] = v.strip()
    if cur:
        out.append(cur)
    return "".join(f"{c['name']} vgprs={c.get('VGPRs', '?')} vgpr_spill={c.get('VGPRs Spill', '?')} "
                   f"scratch={c.get('ScratchSize [bytes/lane]', '?')} occupancy={c.get('Occupancy [waves/SIMD]', '?')} "
                   f"sgpr_spill={c.get('SGPRs Spill', '?')}\n" for c in out)
