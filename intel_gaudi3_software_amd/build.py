"""Builds ``csrc/libmme_hip.so`` with hipcc for gfx950 (cross-compiles without a GPU)."""
import os
import subprocess
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
SOURCES = ["cast_kernels.hip", "gemm_kernels.hip", "gemm_inst_bf16.hip", "gemm_inst_fp16.hip", "gemm_inst_fp32.hip", "gemm_inst_fp8_00.hip", "gemm_inst_fp8_10.hip", "gemm_inst_fp8_01.hip", "gemm_inst_fp8_11.hip", "gemm_large_tile.hip", "gemm_large_tile_f16.hip", "gemm_large_tile_128.hip", "gemm_large_tile_ragged.hip", "gemm_large_tile_conv_fp8.hip", "gemm_large_tile_fp8_at.hip", "gemm_large_tile_ragged_conv.hip", "gemm_large_tile_persistent.hip", "gemm_large_tile_chk.hip", "gemm_large_tile_persistent_chk.hip", "gemm_large_tile_w4.hip", "conv_fwd_fast.hip", "diagnostics.hip", "row_quant.hip", "scaled_gemm.hip", "scaled_gemm_few.hip", "scaled_gemm_tile.hip", "scaled_gemm_large.hip", "mme_api.hip"]
LIB = os.path.join(CSRC, "libmme_hip.so")

# -packed-fp32-ops is switched off: some packed fp32 forms have produced wrong results on this hardware pool
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wno-unused-command-line-argument", "-Wno-unknown-attributes", "-Rpass-analysis=kernel-resource-usage"]


def _includes(path, seen=None):
    """The files a source includes from this directory, transitively (for the only_changed mode)."""
    import re
    seen = set() if seen is None else seen
    with open(path) as f:
        names = re.findall(r'#include\s+"([^"]+)"', f.read())
    for name in names:
        dep = os.path.normpath(os.path.join(os.path.dirname(path), name))
        if os.path.exists(dep) and dep not in seen:
            seen.add(dep)
            _includes(dep, seen)
    return seen


def build_library(verbose=False, jobs=8, only_changed=False):
    """Compile every HIP source and link the shared library.  Recompiles everything unless only_changed is set (then a
    source is skipped when its object is newer than the source and every header it includes)."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    objs, procs = [], []
    for src in SOURCES:
        obj = os.path.join(CSRC, src.replace(".hip", ".o"))
        objs.append(obj)
        if only_changed and os.path.exists(obj):
            deps = [os.path.join(CSRC, src)] + sorted(_includes(os.path.join(CSRC, src)))
            if all(os.path.getmtime(d) <= os.path.getmtime(obj) for d in deps):
                continue
        cmd = [hipcc] + FLAGS + ["-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        if len(procs) >= jobs:
            _wait(procs)
    _wait(procs)
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return LIB


def build_cpp_tests():
    """Compile the C++ programs over the calculator header (host code only, g++): the known-answer program (needs a GPU to
    run) and the planner's and the 8-bit linear layer's (run anywhere).  Returns the path of the first."""
    root = os.path.dirname(_HERE)
    exes = []
    for name in ("kat_calculator", "plan_calculator", "linear8_calculator"):
        src = os.path.join(root, "tests", "cpp", name + ".cpp")
        exe = os.path.join(root, "tests", "cpp", name)
        cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-I" + os.path.join(root, "include"), src, "-o", exe, "-L" + CSRC,
               "-lmme_hip", "-Wl,-rpath,$ORIGIN/../../intel_gaudi3_software_amd/csrc"]
        subprocess.check_call(cmd)
        exes.append(exe)
    return exes[0]


def _resource_report(text):
    """The compiler's per-kernel resource remarks, reduced to what matters here: kernels whose vector registers spill to
    scratch memory.  The large-tile kernels sit a few registers under the limit of 256 and a change that tips one over costs a
    factor of five to ten in run time while every test stays green, so a spill is reported loudly at build time."""
    import re
    name, spilled = None, []
    for line in text.splitlines():
        m = re.search(r"remark: Function Name: (\S+)", line)
        if m:
            name = m.group(1)
        m = re.search(r"remark:\s+VGPRs Spill: (\d+)", line)
        if m and int(m.group(1)) > 0:
            spilled.append((name, int(m.group(1))))
    return spilled


def _wait(procs):
    while procs:
        cmd, p = procs.pop(0)
        out, _ = p.communicate()
        text = out.decode(errors="replace")
        for name, n in _resource_report(text):
            sys.stderr.write("WARNING: %d vector registers of kernel %s spill to scratch memory (%s)\n" % (n, name, os.path.basename(cmd[-3])))
        # the host pass warns that it does not know the packed-fp32 target feature: harmless; the resource remarks have been read
        text = "\n".join(l for l in text.splitlines() if "packed-fp32-ops" not in l and "kernel-resource-usage" not in l and l.strip())
        if p.returncode != 0:
            raise RuntimeError("hipcc failed: %s\n%s" % (" ".join(cmd), text))
        if text:
            sys.stderr.write(text + "\n")


if __name__ == "__main__":
    print(build_library(verbose=True, only_changed="--changed" in sys.argv))
    print(build_cpp_tests())
