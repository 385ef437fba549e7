"""Builds libfklhip.so: the C-ABI runtime plus the ahead-of-time compiled gfx950 kernels of every chain
signature listed in csrc/aot_signatures.txt and the attention kernels under csrc/attention, and _attention.so, the
attention operators' torch binding.  `python -m fusedkernellibrary_amd.build` rebuilds it in place."""
from __future__ import annotations

import concurrent.futures as cf
import hashlib
import importlib.util
import os
import shlex
import subprocess
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(os.path.dirname(PKG), "include")
AOT_DIR = os.path.join(CSRC, "aot")
OBJ_DIR = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libfklhip.so")
N_UNITS = 8

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# -ffp-contract=off: every + - * / is one IEEE rounding, as on the CPU backend the results are checked against.
# packed-fp32-ops off: keep hipcc from forming packed fp32 instructions.
HIP_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++20", "-fPIC", "-ffp-contract=off", "-Wno-unused-value",
    # the SLP vectoriser glues byte lanes into <N x i8> vectors that the backend then legalises through scratch memory
    "-fno-slp-vectorize",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # a per-thread array the optimiser cannot take apart would otherwise be moved to LDS without a word (a 1080p chain
    # ran 18.6 us instead of 5.3 us that way); left in scratch memory it trips the no-scratch gate below
    "-mllvm", "-disable-promote-alloca-to-lds=true",
]
# Extra compiler flags (for example -DFKD_GATHER_XI=4 to try another tile shape) and an alternative output path.
HIP_FLAGS += shlex.split(os.environ.get("FKLHIP_HIPCC_FLAGS", ""))
LIB = os.environ.get("FKLHIP_OUT", LIB)


def read_signatures(path: str | None = None) -> list[str]:
    path = path or os.path.join(CSRC, "aot_signatures.txt")
    sigs = []
    with open(path) as f:
        for line in f:
            line = line.strip()
            if line and not line.startswith("#") and line not in sigs:
                sigs.append(line)
    return sigs


def generate_units(sigs: list[str]) -> list[str]:
    os.makedirs(AOT_DIR, exist_ok=True)
    units = [[] for _ in range(min(N_UNITS, max(1, len(sigs))))]
    # heaviest chains (longest signatures) first, dealt round-robin, so compile time spreads evenly
    for i, s in enumerate(sorted(sigs, key=len, reverse=True)):
        units[i % len(units)].append(s)
    paths = []
    for k, chunk in enumerate(units):
        path = os.path.join(AOT_DIR, f"aot_{k}.hip")
        body = ["// Generated by fusedkernellibrary_amd/build.py from aot_signatures.txt -- do not edit.",
                '#include "../aot_common.hpp"', "using namespace fkd;", ""]
        body += [f"FKD_AOT_CHAIN({s})" for s in chunk]
        text = "\n".join(body) + "\n"
        if not os.path.exists(path) or open(path).read() != text:
            with open(path, "w") as f:
                f.write(text)
        paths.append(path)
    for name in os.listdir(AOT_DIR):
        if name.endswith(".hip") and os.path.join(AOT_DIR, name) not in paths:
            os.remove(os.path.join(AOT_DIR, name))
    return paths


# Device headers embedded into the library for run-time compilation, under the names they are included by.
JIT_HEADERS = [
    ("fkd_kernels.hpp", os.path.join(CSRC, "fkd_kernels.hpp")),
    ("fkd/launch_info.hpp", os.path.join(INCLUDE, "fkd", "launch_info.hpp")),
    ("fkd/ops.hpp", os.path.join(INCLUDE, "fkd", "ops.hpp")),
    ("fkd/types.hpp", os.path.join(INCLUDE, "fkd", "types.hpp")),
    ("types.hpp", os.path.join(INCLUDE, "fkd", "types.hpp")),
]


def generate_jit_sources() -> str:
    """aot/jit_sources.cpp: the device headers as string constants plus the compiler flags of this build, so chains
    compiled at run time get exactly the code generation of the chains compiled here."""
    os.makedirs(AOT_DIR, exist_ok=True)
    path = os.path.join(AOT_DIR, "jit_sources.cpp")
    flags = [f for f in HIP_FLAGS if not f.startswith("--offload-arch") and f != "-fPIC"]
    out = ["// Generated by fusedkernellibrary_amd/build.py -- do not edit.", '#include "../registry.hpp"', "namespace fklhip {"]
    texts = []
    for i, (_, src) in enumerate(JIT_HEADERS):
        text = open(src).read()
        assert ')FKDSRC"' not in text
        # string literals are limited to 64 KiB by some compilers: emit each header in chunks that are concatenated
        chunks = [text[k:k + 12000] for k in range(0, len(text), 12000)]
        out.append(f"static const char kText{i}[] =")
        out += [f'R"FKDSRC({c})FKDSRC"' for c in chunks]
        out.append(";")
        texts.append(f"kText{i}")
    out.append("const char* const kJitHeaderNames[] = {" + ", ".join(f'"{n}"' for n, _ in JIT_HEADERS) + "};")
    out.append("const char* const kJitHeaderTexts[] = {" + ", ".join(texts) + "};")
    out.append(f"const int kJitHeaderCount = {len(JIT_HEADERS)};")
    out.append("const char* const kJitFlags[] = {" + ", ".join('"' + f.replace('"', '\\"') + '"' for f in flags) + "};")
    out.append(f"const int kJitFlagCount = {len(flags)};")
    out.append("} // namespace fklhip")
    text = "\n".join(out) + "\n"
    if not os.path.exists(path) or open(path).read() != text:
        with open(path, "w") as f:
            f.write(text)
    return path


def _compile(src: str) -> str:
    obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
    device_code = src.endswith(".hip")
    # for device code the compiler reports each kernel's resources; a kernel that needs scratch memory (a private
    # array the optimiser could not keep in registers, or spills) is a build error here, not a silent 20x slowdown
    cmd = [HIPCC, *HIP_FLAGS, *(["-Rpass-analysis=kernel-resource-usage"] if device_code else []), "-I", INCLUDE, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    err = "\n".join(l for l in r.stderr.splitlines() if "packed-fp32-ops" not in l and "kernel-resource-usage" not in l)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{err}")
    if device_code:
        name = "?"
        for line in r.stderr.splitlines():
            if "Function Name:" in line:
                name = line.split("Function Name:")[1].split("[")[0].strip()
            for key in ("ScratchSize [bytes/lane]:", "SGPRs Spill:", "VGPRs Spill:"):
                if key in line and int(line.split(key)[1].split("[")[0].strip()) != 0:
                    raise RuntimeError(f"{src}: kernel {name} uses scratch memory ({line.split('remark:')[1].strip()})")
    return obj


def build_library(verbose: bool = True) -> str:
    if not os.path.exists(HIPCC):
        raise RuntimeError(f"hipcc not found at {HIPCC}")
    sigs = read_signatures()
    units = generate_units(sigs)
    os.makedirs(OBJ_DIR, exist_ok=True)
    attention = [os.path.join(CSRC, "attention", name) for name in sorted(os.listdir(os.path.join(CSRC, "attention"))) if name.endswith((".hip", ".cpp")) and name != "torch_binding.cpp"]
    srcs = attention + units + [os.path.join(CSRC, "fklhip_runtime.cpp"), os.path.join(CSRC, "jit.cpp"), generate_jit_sources()]
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(_compile, srcs))
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB + ".tmp", *objs, "-lhiprtc"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(LIB + ".tmp", LIB)
    if verbose:
        print(f"built {LIB}: {len(sigs)} chain signatures in {len(units)} translation units")
    return LIB


def build_torch_binding(verbose: bool = True) -> str | None:
    """_attention.so: host code only, so the host compiler builds it. Without torch, or with one that is not ROCm's, there is
    nothing to bind, and libfklhip.so does not need it."""
    spec = importlib.util.find_spec("torch")
    torch_dir = spec.submodule_search_locations[0] if spec else ""
    if not spec or not os.path.exists(os.path.join(torch_dir, "lib", "libc10_hip.so")):
        if verbose:
            print("no torch for ROCm: fusedkernellibrary_amd.attention is not built")
        return None
    out = os.path.join(PKG, "_attention.so")
    rocm = os.path.join(os.path.dirname(os.path.dirname(HIPCC)), "include")
    include = [INCLUDE, os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"), rocm,
               sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-std=c++20", "-O2", "-fPIC", "-shared", "-fvisibility=hidden", "-w", "-DUSE_ROCM=1", "-D__HIP_PLATFORM_AMD__=1",
           *[f"-I{d}" for d in include], os.path.join(CSRC, "attention", "torch_binding.cpp"), "-o", out + ".tmp",
           "-L", PKG, "-lfklhip", "-L", os.path.join(torch_dir, "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on torch_binding.cpp:\n{r.stderr}")
    os.replace(out + ".tmp", out)
    if verbose:
        print(f"built {out}")
    return out


if __name__ == "__main__":
    build_library()
    build_torch_binding()
