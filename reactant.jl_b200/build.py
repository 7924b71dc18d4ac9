"""Builds librx_b200.so (sm_100a) in-tree with nvcc, and the extension module _call with the host compiler.

Run as `python reactant.jl_b200/build.py`; `__graft_entry__.build()` calls
`build()` below.  Objects are rebuilt only when a source or header is newer.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "librx_b200.so")
OBJ = os.path.join(HERE, "build")

SOURCES = [
    "rx_parser.cpp", "rx_plan.cpp", "rx_kernels.cu", "rx_wide.cu", "rx_gemm.cu", "rx_gemm_tc.cu",
    "rx_stencil.cu", "rx_stencil_tma.cu", "rx_collective.cu", "rx_runtime.cu", "rx_noalloc.cu", "rx_abi_extra.cu", "rx_jit.cpp",
    "rx_embedding.cu", "rx_dropout.cu", "rx_logprobs.cu",
]

# Device headers handed to NVRTC by name when a fused chain is specialised at run time.
EMBEDDED = ["rx_vm.h", "rx_device.cuh", "rx_chain_kernels.cuh", "rx_tma_device.cuh", "rx_gemm_pair.cuh"]
EMBED_OUT = os.path.join(CSRC, "rx_jit_embed.inc")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC,-Wall,-Wno-unused-function,-fvisibility=default",
    "-gencode", "arch=compute_100a,code=sm_100a", "-I", os.path.join(HERE, "..", "include"), "-I", CSRC,
    "--expt-relaxed-constexpr",
]


def _stale(obj: str, deps: list[str]) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(d) > t for d in deps)


def write_embedded_headers() -> None:
    """Writes csrc/rx_jit_embed.inc: the device headers as C++ raw string literals."""
    parts = ["// generated by build.py from " + ", ".join(EMBEDDED) + "; do not edit\n"]
    parts.append("static const int kEmbedCount = %d;\n" % len(EMBEDDED))
    parts.append("static const char* const kEmbedNames[] = {" + ", ".join('"%s"' % n for n in EMBEDDED) + "};\n")
    parts.append("static const char* const kEmbedSrc[] = {\n")
    for n in EMBEDDED:
        text = open(os.path.join(CSRC, n)).read()
        assert ')RXEMBED"' not in text
        # a raw string literal is limited to 64 KiB by some compilers: split into concatenated pieces
        chunks = [text[i:i + 12000] for i in range(0, len(text), 12000)]
        parts.append("".join('R"RXEMBED(%s)RXEMBED"\n' % c for c in chunks) + ",\n")
    parts.append("};\n")
    new = "".join(parts)
    if not os.path.exists(EMBED_OUT) or open(EMBED_OUT).read() != new:
        with open(EMBED_OUT, "w") as f:
            f.write(new)


def build_call(verbose: bool = False) -> str:
    """The extension module of the Python package's call path, named for the interpreter that builds it (another version
    does not load it).  It links against nothing: _lib.py hands it the library's entry points."""
    src, out = os.path.join(CSRC, "rx_python.cpp"), os.path.join(HERE, "_call" + sysconfig.get_config_var("EXT_SUFFIX"))
    if _stale(out, [src, os.path.join(CSRC, "rx_dlpack.h"), os.path.join(HERE, "..", "include", "rx_b200.h")]):
        cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-Wall", "-Wno-missing-field-initializers", "-shared", "-fPIC", "-fvisibility=hidden", "-I", sysconfig.get_paths()["include"],
               src, "-o", out]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or r.returncode:
            sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
        if r.returncode:
            raise RuntimeError("failed: " + " ".join(cmd))
    return out


def build(verbose: bool = False, ptxas_info: bool = False, bounds: bool = False) -> str:
    """bounds=True builds librx_b200_bounds.so instead: the same library with -DRX_BOUNDS=1 (every element access of
    the chain kernels, the fused GEMM epilogues and the stencil stores checked against its buffer; select it with
    RX_B200_LIB=<path> in the environment of the process that loads the package)."""
    out_path = OUT.replace(".so", "_bounds.so") if bounds else OUT
    obj_dir = OBJ + "_bounds" if bounds else OBJ
    flags = FLAGS + (["-DRX_BOUNDS=1"] if bounds else [])
    os.makedirs(obj_dir, exist_ok=True)
    write_embedded_headers()
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    headers.append(os.path.join(HERE, "..", "include", "rx_b200.h"))
    headers.append(EMBED_OUT)
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    objs, jobs = [], []
    for s in srcs:
        src = os.path.join(CSRC, s)
        obj = os.path.join(obj_dir, s + ".o")
        objs.append(obj)
        if _stale(obj, [src] + headers):
            cmd = [NVCC, *flags, "-x", "cu", "-c", src, "-o", obj]
            if ptxas_info:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or r.returncode:
            sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
        if r.returncode:
            raise RuntimeError("nvcc failed: " + " ".join(cmd))
        return r.stderr

    with ThreadPoolExecutor(max_workers=8) as ex:
        logs = list(ex.map(run, jobs))
    if jobs or not os.path.exists(out_path):
        link = [NVCC, "-shared", "-o", out_path, *objs, "-cudart", "static", "-ldl", "-lpthread",
                "-gencode", "arch=compute_100a,code=sm_100a"]
        run(link)
    if ptxas_info:
        sys.stderr.write("\n".join(logs))
    build_call(verbose)
    return out_path


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, ptxas_info="--ptxas" in sys.argv, bounds="--bounds" in sys.argv))
