"""Builds libvsloss.so in-tree with hipcc for gfx950, and the torch binding of the class losses (no GPU needed to compile)."""
from __future__ import annotations

import os
import re
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libvsloss.so")
RESOURCES = os.path.join(HERE, "libvsloss.resources.txt")
SOURCES = ["vsl_loss.hip", "vsl_layers.hip", "vsl_pose.hip", "vsl_metrics.hip", "vsl_vocab.hip", "vsl_linear_ce.hip"]
BINDING_SOURCE = os.path.join(CSRC, "vsl_vocab_binding.cpp")
BINDING = os.path.join(HERE, "vsl_vocab_binding.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def needs_build() -> bool:
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if not f.endswith(".cpp")]
    deps.append(os.path.join(HERE, "..", "include", "vsloss.h"))
    return any(os.path.getmtime(d) > t for d in deps if os.path.isfile(d))


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return OUT
    # -ffp-contract=on: fuse a*b+c only inside one expression.  The default (fast) also fuses
    # across statements, which measurably moves the pose/disparity gradients away from the
    # reference's float32 results (1.5e-5 instead of 1e-6 relative on the golden fixtures).
    # -fno-slp-vectorize: packed f32 math has no rate advantage on gfx950 and its operand pairing costs
    # register moves (measured 3 % slower with it).  -packed-fp32-ops keeps the compiler from forming it in other passes.
    flags = ["-Rpass-analysis=kernel-resource-usage", "-O3", "--offload-arch=gfx950", "-std=c++17", "-ffp-contract=on",
             "-fno-slp-vectorize", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-fPIC",
             "-I", os.path.join(HERE, "..", "include")]
    with tempfile.TemporaryDirectory() as tmp:  # the sources side by side, the longest takes 80 s
        objects = [os.path.join(tmp, s + ".o") for s in SOURCES]
        compile_ = [[HIPCC] + flags + ["-c", os.path.join(CSRC, s), "-o", o] for s, o in zip(SOURCES, objects)]
        link = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", OUT] + objects
        if verbose:
            print("\n".join(" ".join(c) for c in compile_ + [link]), file=sys.stderr)
        with ThreadPoolExecutor(len(SOURCES)) as pool:
            done = list(pool.map(lambda c: subprocess.run(c, stderr=subprocess.PIPE, text=True), compile_))
        if all(p.returncode == 0 for p in done):
            done.append(subprocess.run(link, stderr=subprocess.PIPE, text=True))
    text = "".join(p.stderr for p in done)
    table = kernel_resources(text)
    other, after_remark = [], False  # everything but the remarks and the source excerpts printed under them
    for ln in text.splitlines():
        if "-Rpass-analysis=kernel-resource-usage" in ln:
            after_remark = True
        elif not (after_remark and re.match(r"\s*\d*\s*\|", ln)):
            after_remark = False
            other.append(ln)
    if other:
        print("\n".join(other), file=sys.stderr)
    for proc in done:
        if proc.returncode != 0:
            raise subprocess.CalledProcessError(proc.returncode, proc.args)
    with open(RESOURCES, "w") as f:
        f.write("# kernel  VGPRs  SGPR-spills  VGPR-spills  scratch-bytes-per-lane  LDS-bytes\n")
        for k in table:
            f.write("%s %d %d %d %d %d\n" % (k["name"], k["vgprs"], k["sgpr_spill"], k["vgpr_spill"], k["scratch"], k["lds"]))
    if verbose:
        print(open(RESOURCES).read(), file=sys.stderr)
    # A private array that the compiler cannot keep in registers lands in scratch memory and is written back to HBM
    # by every wave (one such array of 16 B per lane doubled the tile kernel's HBM writes without changing a result):
    # no kernel of this library may have any.
    bad = [k["name"] for k in table if k["scratch"] or k["vgpr_spill"]]
    if bad:
        os.remove(OUT)
        raise RuntimeError("kernels with scratch memory or vector-register spills: " + ", ".join(bad))
    return OUT


def build_binding(force: bool = False) -> str:
    """The extension module behind vocab_losses: include/vsloss_vocab_torch.h against the installed torch, with g++.  The
    library's functions stay undefined in it; the package loads them first."""
    include = os.path.join(HERE, "..", "include")
    deps = [BINDING_SOURCE] + [os.path.join(include, f) for f in os.listdir(include)]
    if not force and os.path.exists(BINDING) and all(os.path.getmtime(BINDING) >= os.path.getmtime(d) for d in deps):
        return BINDING
    import sysconfig

    import torch
    tdir = os.path.dirname(torch.__file__)
    subprocess.check_call(
        ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
         "-DTORCH_EXTENSION_NAME=vsl_vocab_binding", "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch.compiled_with_cxx11_abi()),
         "-I", include, "-I", os.path.join(tdir, "include"),
         "-I", os.path.join(tdir, "include", "torch", "csrc", "api", "include"), "-I", "/opt/rocm/include",
         "-I", sysconfig.get_paths()["include"], BINDING_SOURCE, "-o", BINDING, "-L", os.path.join(tdir, "lib"),
         "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip",
         "-Wl,-rpath," + os.path.join(tdir, "lib")])
    return BINDING


def kernel_resources(remarks: str):
    """The compiler's per-kernel resource remarks as a list of dicts."""
    out, cur = [], None
    keys = {"VGPRs": "vgprs", "SGPRs Spill": "sgpr_spill", "VGPRs Spill": "vgpr_spill",
            "ScratchSize [bytes/lane]": "scratch", "LDS Size [bytes/block]": "lds"}
    for ln in remarks.splitlines():
        m = re.search(r"remark:\s+(.*?):\s+(\S+) \[-Rpass-analysis", ln)
        if not m:
            continue
        key, val = m.group(1).strip(), m.group(2)
        if key == "Function Name":
            cur = {"name": val, "vgprs": 0, "sgpr_spill": 0, "vgpr_spill": 0, "scratch": 0, "lds": 0}
            out.append(cur)
        elif cur is not None and key in keys:
            cur[keys[key]] = int(val)
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_binding(force="--force" in sys.argv))
